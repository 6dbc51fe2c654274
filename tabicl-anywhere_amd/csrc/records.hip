// The fit-time side of the stored cache: keys and values of every training row, laid out in the reference's chunk
// records and quantised on the card.
//
// * k_to_records: a layer's keys and values as the projection wrote them, row-major [rows][2d], to f32 chunk
//   records [K: d][rc][V: d][rc] per chunk (src/fit.rs:633-647). 64 x 64 tiles are transposed through LDS so both
//   the reads (along coordinates) and the writes (along rows of a chunk) are coalesced.
// * k_pack: f32 records to i16/i8 records, bit for bit as the reference's quantiser (src/fit.rs:549-576): per chunk
//   and coordinate row, big = max |v| (NaN ignored, as f32::max does), s = big > 0 ? big / top : 1 with top 32767
//   or 127, inv = 1 / s, code = round-half-away(v * inv) saturated to the integer range; the 2d scales first.
//   One wavefront per coordinate row. Division is the correctly rounded one (__fdiv_rn), so the same f32 input
//   gives the same scales and codes as the CPU.
// * k_pack4: f32 records to i4 records (kv4.hpp).
// * k_unpack: records of i16, i8 or i4 to f32 records.
#include <algorithm>

#include "common.hpp"
#include "device_math.hpp"
#include "kv4.hpp"

namespace tah {

__global__ __launch_bounds__(256) void k_to_records(int rows, int d2, int chunk, const float *__restrict__ kv,
                                                     float *__restrict__ rec) {
    __shared__ float tile[64][65];
    const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int i = ty; i < 64; i += 4) {
        const int m = m0 + i, n = n0 + tx;
        tile[i][tx] = (m < rows && n < d2) ? kv[(size_t)m * d2 + n] : 0.0f;
    }
    __syncthreads();
    const int n_chunks = (rows + chunk - 1) / chunk;
    const int last_rc = rows - (n_chunks - 1) * chunk;
    for (int j = ty; j < 64; j += 4) {
        const int n = n0 + j, m = m0 + tx;
        if (m >= rows || n >= d2) continue;
        const int ci = m / chunk, r = m - ci * chunk;
        const int rc = ci == n_chunks - 1 ? last_rc : chunk;
        rec[(size_t)ci * d2 * chunk + (size_t)n * rc + r] = tile[tx][j];
    }
}

template <int FMT>
__global__ __launch_bounds__(256) void k_pack(int rows, int d, int chunk, const float *__restrict__ rec32,
                                               uint8_t *__restrict__ recq) {
    const int ci = blockIdx.x, j = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (j >= 2 * d) return;
    const int n_chunks = (rows - 1) / chunk + 1;
    const int rc = ci == n_chunks - 1 ? rows - (n_chunks - 1) * chunk : chunk;
    const float *src = rec32 + (size_t)ci * 2 * d * chunk + (size_t)j * rc;
    constexpr size_t W = FMT == TAH_KV_I16 ? 2 : 1;
    uint8_t *rec = recq + (size_t)ci * (2 * (size_t)d * chunk * W + 8 * (size_t)d);
    float big = 0.0f;
    for (int r = lane; r < rc; r += 64) big = fmaxf(big, fabsf(src[r]));
    big = wave_max(big);
    const float top = FMT == TAH_KV_I16 ? 32767.0f : 127.0f;
    const float s = big > 0.0f ? __fdiv_rn(big, top) : 1.0f;
    const float inv = __fdiv_rn(1.0f, s);
    if (lane == 0) reinterpret_cast<float *>(rec)[j] = s;
    uint8_t *body = rec + 8 * (size_t)d;
    for (int r = lane; r < rc; r += 64) {
        const float v = roundf(__fmul_rn(src[r], inv));
        if (FMT == TAH_KV_I16) {
            const int16_t code = v != v ? 0 : (v >= 32767.0f ? 32767 : (v <= -32768.0f ? -32768 : (int16_t)v));
            reinterpret_cast<int16_t *>(body)[(size_t)j * rc + r] = code;
        } else {
            const int8_t code = v != v ? 0 : (v >= 127.0f ? 127 : (v <= -128.0f ? -128 : (int8_t)v));
            reinterpret_cast<int8_t *>(body)[(size_t)j * rc + r] = code;
        }
    }
}

// ---- i4 records and back ------------------------------------------------------------------------------------------------
// Both are bound by memory (a number is 4 bytes and 9/16 of one), so the numbers move 16 bytes a lane where the records
// allow it: a lane takes four consecutive rows of a coordinate, 16 lanes a group of 64, UNITS groups in turn with their
// loads issued together. Records whose rows do not start on whole words (odd chunks) take the same path by single loads.
constexpr int UNITS = 4;

// grid (groups of a full chunk / 64, chunks); 256 threads.
__global__ __launch_bounds__(256) void k_pack4(int rows, int d, int chunk, const float *__restrict__ rec32,
                                               uint8_t *__restrict__ rec4) {
    const int n_chunks = (rows - 1) / chunk + 1;
    for (int ci = blockIdx.y; ci < n_chunks; ci += gridDim.y) {
        const int rc = min(chunk, rows - ci * chunk), G = groups4(rc), half = (rc + 1) / 2, in16 = 4 * (threadIdx.x & 15);
        const float *src = rec32 + (size_t)ci * 2 * d * chunk;
        uint8_t *rec = rec4 + (size_t)ci * record_bytes(TAH_KV_I4, d, chunk), *codes = rec + 8 * (size_t)d * G;
        const bool fours = rc % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
        const bool pairs = half % 2 == 0 && (reinterpret_cast<uintptr_t>(codes) & 1) == 0;
        float v[UNITS][4];
        int j[UNITS], g[UNITS];
        // the units of a thread are 16 apart
        const int unit = blockIdx.x * UNITS * 16 + (threadIdx.x >> 4), over = 16 / G, past = 16 - over * G;
        j[0] = unit / G;
        g[0] = unit - j[0] * G;
#pragma unroll
        for (int u = 1; u < UNITS; u++) {
            g[u] = g[u - 1] + past;
            j[u] = j[u - 1] + over + (g[u] >= G);
            g[u] -= g[u] >= G ? G : 0;
        }
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int r = 64 * g[u] + in16;
            const float *at = src + (size_t)j[u] * rc + r;
#pragma unroll
            for (int t = 0; t < 4; t++) v[u][t] = NAN;  // what is past the end takes no part
            if (j[u] >= 2 * d) continue;
            if (fours && r < rc) {
                const float4 x = *reinterpret_cast<const float4 *>(at);
                v[u][0] = x.x; v[u][1] = x.y; v[u][2] = x.z; v[u][3] = x.w;
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++)
                    if (r + t < rc) v[u][t] = at[t];
            }
        }
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            // the group's least and largest number (NaN passed over); again without the infinities where there are any
            auto range = [&](bool all, float &lo, float &hi) {
                lo = INFINITY;
                hi = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const float x = all || fabsf(v[u][t]) < INFINITY ? v[u][t] : NAN;
                    lo = fminf(lo, x);
                    hi = fmaxf(hi, x);
                }
                lo = row16_reduce(lo, fminf);
                hi = row16_reduce(hi, fmaxf);
            };
            float lo, hi;
            range(true, lo, hi);
            if (__any(fmaxf(fabsf(lo), fabsf(hi)) == INFINITY)) range(false, lo, hi);
            const Step4 st = step_for4(lo, hi);
            if (j[u] >= 2 * d) continue;
            const int r = 64 * g[u] + in16, left = rc - r;
            if (in16 == 0) {
                uint16_t *sp = reinterpret_cast<uint16_t *>(rec) + 2 * ((size_t)j[u] * G + g[u]);
                sp[0] = (uint16_t)(__float_as_uint(st.s) >> 16);
                sp[1] = (uint16_t)(__float_as_uint(st.z) >> 16);
            }
            if (left <= 0) continue;
            int code[4];
            codes4(st, v[u], code);
            uint32_t word = 0;
#pragma unroll
            for (int t = 0; t < 4; t++) word |= (t < left ? (uint32_t)(code[t] + 8) : 0u) << 4 * t;
            uint8_t *cp = codes + (size_t)j[u] * half + r / 2;
            if (pairs && left > 2) {
                *reinterpret_cast<uint16_t *>(cp) = (uint16_t)word;
            } else {
                cp[0] = (uint8_t)word;
                if (left > 2) cp[1] = (uint8_t)(word >> 8);
            }
        }
    }
}

// What four consecutive rows (from a multiple of 4) of coordinate j of a chunk's record stand for; rows past the end not
// looked at.
template <int FMT>
__device__ __forceinline__ void values_of(const uint8_t *rec, int d, int rc, int j, int r, bool whole, float (&v)[4]) {
    if constexpr (FMT == TAH_KV_I4) {
        Step4 st;
        if (whole) {
            const uint32_t sz = reinterpret_cast<const uint32_t *>(rec)[(size_t)j * groups4(rc) + r / GROUP4];
            st = {__uint_as_float(sz << 16), __uint_as_float(sz & 0xFFFF0000u)};
        } else {
            st = step_at4(rec, rc, j, r / GROUP4);
        }
        const int half = (rc + 1) / 2;
        const uint8_t *cp = rec + 8 * (size_t)d * groups4(rc) + (size_t)j * half + r / 2;
        uint32_t word;
        if (whole) word = *reinterpret_cast<const uint16_t *>(cp);
        else word = cp[0] | (r + 2 < rc ? cp[1] : 0) << 8;
#pragma unroll
        for (int t = 0; t < 4; t++) v[t] = value4(st, (int)(word >> 4 * t & 15) - 8);
    } else {
        const float s = reinterpret_cast<const float *>(rec)[j];
        const size_t at = (size_t)j * rc + r;
        const uint8_t *body = rec + 8 * (size_t)d;
#pragma unroll
        for (int t = 0; t < 4; t++)
            if (r + t < rc)
                v[t] = s * (FMT == TAH_KV_I16 ? (float)reinterpret_cast<const int16_t *>(body)[at + t]
                                              : (float)reinterpret_cast<const int8_t *>(body)[at + t]);
    }
}

// grid (fours of rows of a full chunk / 1,024, chunks); 256 threads.
template <int FMT>
__global__ __launch_bounds__(256) void k_unpack(int rows, int d, int chunk, const uint8_t *__restrict__ rec,
                                                float *__restrict__ rec32) {
    const int n_chunks = (rows - 1) / chunk + 1;
    for (int ci = blockIdx.y; ci < n_chunks; ci += gridDim.y) {
        const int rc = min(chunk, rows - ci * chunk), Q = (rc + 3) / 4;
        const uint8_t *src = rec + (size_t)ci * record_bytes(FMT, d, chunk);
        float *dst = rec32 + (size_t)ci * 2 * d * chunk;
        const bool fours = rc % 4 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
        const bool whole = rc % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & 3) == 0;  // steps and codes by whole words
        float v[UNITS][4];
        int j[UNITS], r[UNITS];
        // the fours of a thread are 256 apart
        const int unit = blockIdx.x * UNITS * 256 + threadIdx.x, over = 256 / Q, past = 256 - over * Q;
        j[0] = unit / Q;
        r[0] = unit - j[0] * Q;
#pragma unroll
        for (int u = 1; u < UNITS; u++) {
            r[u] = r[u - 1] + past;
            j[u] = j[u - 1] + over + (r[u] >= Q);
            r[u] -= r[u] >= Q ? Q : 0;
        }
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            r[u] *= 4;
            if (j[u] < 2 * d) values_of<FMT>(src, d, rc, j[u], r[u], whole, v[u]);
        }
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            if (j[u] >= 2 * d) continue;
            float *to = dst + (size_t)j[u] * rc + r[u];
            if (fours) {
                *reinterpret_cast<float4 *>(to) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++)
                    if (r[u] + t < rc) to[t] = v[u][t];
            }
        }
    }
}

void to_records(hipStream_t s, int rows, int d, int chunk, const float *kv, float *rec32) {
    if (rows <= 0) return;
    dim3 grid((rows + 63) / 64, (2 * d + 63) / 64);
    hipLaunchKernelGGL(k_to_records, grid, dim3(256), 0, s, rows, 2 * d, chunk, kv, rec32);
    TAH_LAUNCHED();
}

void pack(hipStream_t s, int rows, int d, int chunk, int fmt, const float *rec32, uint8_t *recq) {
    if (rows <= 0 || fmt == TAH_KV_F32) return;
    const int n_chunks = (rows - 1) / chunk + 1;
    dim3 grid(n_chunks, (2 * d + 3) / 4);
    if (fmt == TAH_KV_I4) {
        const size_t units = 2 * (size_t)d * groups4(std::min(chunk, rows));
        hipLaunchKernelGGL(k_pack4, dim3((units + 16 * UNITS - 1) / (16 * UNITS), std::min(n_chunks, 65535)), dim3(256), 0, s,
                           rows, d, chunk, rec32, recq);
    } else if (fmt == TAH_KV_I16)
        hipLaunchKernelGGL(k_pack<TAH_KV_I16>, grid, dim3(256), 0, s, rows, d, chunk, rec32, recq);
    else if (fmt == TAH_KV_I8)
        hipLaunchKernelGGL(k_pack<TAH_KV_I8>, grid, dim3(256), 0, s, rows, d, chunk, rec32, recq);
    else
        throw ArgError{"pack: unknown key/value format"};
    TAH_LAUNCHED();
}

void unpack(hipStream_t s, int rows, int d, int chunk, int fmt, const uint8_t *rec, float *rec32) {
    if (rows <= 0) return;
    const int n_chunks = (rows - 1) / chunk + 1;
    const size_t fours = 2 * (size_t)d * ((std::min(chunk, rows) + 3) / 4);
    const dim3 grid((fours + 256 * UNITS - 1) / (256 * UNITS), std::min(n_chunks, 65535));
    if (fmt == TAH_KV_F32)
        TAH_HIP(hipMemcpyAsync(rec32, rec, sizeof(float) * 2 * (size_t)rows * d, hipMemcpyDeviceToDevice, s));
    else if (fmt == TAH_KV_I16)
        hipLaunchKernelGGL(k_unpack<TAH_KV_I16>, grid, dim3(256), 0, s, rows, d, chunk, rec, rec32);
    else if (fmt == TAH_KV_I8)
        hipLaunchKernelGGL(k_unpack<TAH_KV_I8>, grid, dim3(256), 0, s, rows, d, chunk, rec, rec32);
    else
        hipLaunchKernelGGL(k_unpack<TAH_KV_I4>, grid, dim3(256), 0, s, rows, d, chunk, rec, rec32);
    TAH_LAUNCHED();
}

}  // namespace tah

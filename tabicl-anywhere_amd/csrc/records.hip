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
    const int n_chunks = (rows - 1) / chunk + 1;
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
// A number is 4 bytes and 9/16 of one. It moves 16 bytes at a time: a lane takes four consecutive rows of a coordinate, 16
// lanes a group of 64, UNITS groups in turn with their loads issued together (10,000 x 512 in chunks of 256 unpacked with 1, 2
// and 4: 11.9, 9.2 and 9.9 us; packed 12.5, 11.0 and 12.0). Chunks of any length do so: fours that start off a 16-byte line
// are loads and stores of 4-byte alignment, only a coordinate's last rows go one by one. Unpacked numbers are written past the
// caches, which hold the records and would be turned over (40,000 x 512: 61.7 -> 30.4 us).
//
// 10,000 x 512 (46.7 MB): unpacked 8.2 us, 5.7 TB/s, a large copy's rate; packed 11.0 us, bound by its instructions, about 120
// a lane's four numbers: the range of 16 lanes, the step, four quotients, their ties.
constexpr int UNITS = 2;
typedef float Four __attribute__((ext_vector_type(4), aligned(4)));

// The least lo and largest hi of 16 lanes (neither a NaN), in all of them: lanes 1, 2, 4 and 8 apart. Written out because the
// compiler moves and cleans a lane's neighbour in two instructions of their own before each comparison; a register written
// is read across lanes two instructions later at the soonest.
__device__ __forceinline__ void row16_range(float &lo, float &hi) {
    asm("s_nop 1\n\t"
        "v_min_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
        "v_max_f32_dpp %1, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 0\n\t"
        "v_min_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
        "v_max_f32_dpp %1, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 0\n\t"
        "v_min_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "v_max_f32_dpp %1, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 0\n\t"
        "v_min_f32_dpp %0, %0, %0 row_mirror row_mask:0xf bank_mask:0xf\n\t"
        "v_max_f32_dpp %1, %1, %1 row_mirror row_mask:0xf bank_mask:0xf"
        : "+v"(lo), "+v"(hi));
}

// grid (groups of a full chunk / 64, chunks); 256 threads.
__global__ __launch_bounds__(256) void k_pack4(int rows, int d, int chunk, const float *__restrict__ rec32,
                                               uint8_t *__restrict__ rec4) {
    const int n_chunks = (rows - 1) / chunk + 1;
    for (int ci = blockIdx.y; ci < n_chunks; ci += gridDim.y) {
        const int rc = min(chunk, rows - ci * chunk), G = groups4(rc), half = (rc + 1) / 2, in16 = 4 * (threadIdx.x & 15);
        const float *src = rec32 + (size_t)ci * 2 * d * chunk;
        uint8_t *rec = rec4 + (size_t)ci * record_bytes(TAH_KV_I4, d, chunk), *codes = rec + 8 * (size_t)d * G;
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
            if (r + 4 <= rc) {
                const Four x = *reinterpret_cast<const Four *>(at);
#pragma unroll
                for (int t = 0; t < 4; t++) v[u][t] = x[t];
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
                row16_range(lo, hi);
            };
            float lo, hi;
            range(true, lo, hi);
            if (__any(fmaxf(fabsf(lo), fabsf(hi)) == INFINITY)) range(false, lo, hi);
            const Step4 st = step_for4(lo, hi);
            if (j[u] >= 2 * d) continue;
            const int r = 64 * g[u] + in16, left = rc - r;
            if (in16 == 0) {
                const uint32_t sz = __float_as_uint(st.s) >> 16 | __float_as_uint(st.z);
                __builtin_memcpy(rec + 4 * ((size_t)j[u] * G + g[u]), &sz, 4);
            }
            if (left <= 0) continue;
            uint32_t word = codes4(st, v[u]);
            if (left < 4) word &= (1u << 4 * left) - 1;
            uint8_t *cp = codes + (size_t)j[u] * half + r / 2;
            if (left > 2) __builtin_memcpy(cp, &word, 2);
            else cp[0] = (uint8_t)word;
        }
    }
}

// What four consecutive rows (from a multiple of 4) of coordinate j of a chunk's record stand for; rows past the end not
// looked at.
template <int FMT>
__device__ __forceinline__ void values_of(const uint8_t *rec, int d, int rc, int j, int r, float (&v)[4]) {
    if constexpr (FMT == TAH_KV_I4) {
        const Step4 st = step_at4(rec, rc, j, r / GROUP4);
        const int half = (rc + 1) / 2;
        const uint8_t *cp = rec + 8 * (size_t)d * groups4(rc) + (size_t)j * half + r / 2;
        uint32_t word = 0;
        if (r + 2 < rc) __builtin_memcpy(&word, cp, 2);
        else word = cp[0];
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
            if (j[u] < 2 * d) values_of<FMT>(src, d, rc, j[u], r[u], v[u]);
        }
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            if (j[u] >= 2 * d) continue;
            float *to = dst + (size_t)j[u] * rc + r[u];
            if (r[u] + 4 <= rc) {
                __builtin_nontemporal_store(Four{v[u][0], v[u][1], v[u][2], v[u][3]}, reinterpret_cast<Four *>(to));
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

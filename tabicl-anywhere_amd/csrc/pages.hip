// Rows of many tables into pages of a pool and back (tah_pages_write, tah_pages_read): the step of a row's head, the ints, and
// the values' transposition.
#include "device_math.hpp"
#include "pages.hpp"

namespace tah {

namespace {

constexpr int TILE = 64;      // rows a workgroup
constexpr int QUADS = 17;     // fours of rows in one table's order: 16, and one more where they begin between two
constexpr int IN_LDS = 1024;  // tables whose offsets a workgroup looks through in LDS

template <int FMT>
struct Number;
template <>
struct Number<TAH_KV_F32> {
    typedef float T;
    typedef floatx4 V;
};
template <>
struct Number<TAH_KV_I16> {
    typedef int16_t T;
    typedef int16_t V __attribute__((ext_vector_type(4)));
    static constexpr float top = 32767.0f;
};
template <>
struct Number<TAH_KV_I8> {
    typedef int8_t T;
    typedef int8_t V __attribute__((ext_vector_type(4)));
    static constexpr float top = 127.0f;
};

// Where a workgroup's rows lie: page (-1: none, -2: a row of no table) and slot of each, and for each four of rows from `first` on whether they are one
// aligned four of a page. Fours begin where the first row that lies anywhere makes them aligned.
struct Places {
    int page[TILE], slot[TILE];
    int whole[QUADS], first;
};

__device__ void find_places(const PageSet &p, const int32_t *starts, const int32_t *offsets, int r0, int rows, int *offs,
                            Places &pl) {
    const int tid = threadIdx.x;
    const bool in_lds = p.tables < IN_LDS;
    if (in_lds) {
        for (int i = tid; i <= p.tables; i += 256) offs[i] = offsets[i];
        __syncthreads();
    }
    if (tid < TILE) {
        const int r = r0 + tid;
        int page = -2, slot = 0;
        if (r < rows) {
            const int32_t *o = in_lds ? offs : offsets;
            const int t = table_of(o, p.tables, r);
            if (r >= o[t] && r < o[t + 1]) {
                const long at = (long)starts[t] + (r - o[t]);
                page = page_of(p, t, at);
                slot = (int)(at & (p.rows - 1));
            }
        }
        pl.page[tid] = page;
        pl.slot[tid] = slot;
        const uint64_t some = __ballot(page >= 0);
        const int lead = some ? __ffsll((unsigned long long)some) - 1 : 0;
        const int at = __shfl(slot, lead);
        if (tid == 0) pl.first = ((lead - at) & 3) - 4;
    }
    __syncthreads();
    if (tid < QUADS) {
        const int a = pl.first + 4 * tid;
        bool ok = a >= 0 && a + 3 < TILE;
        if (ok) {
            ok = pl.page[a] >= 0 && (pl.slot[a] & 3) == 0;
            for (int i = 1; i < 4; i++) ok = ok && pl.page[a + i] == pl.page[a] && pl.slot[a + i] == pl.slot[a] + i;
        }
        pl.whole[tid] = ok;
    }
    __syncthreads();
}

__device__ __forceinline__ float finite_abs(float x) { return __uint_as_float(finite_bits(__float_as_uint(x))); }

// x / s rounded to the nearest int, ties to even, within the top; inv is about 1 / s. The product's rounding may miss by one
// where x / s is next to a tie: its residual x - c s is exact in f32 (a multiple of half an ulp of s, below 2^24 of them), and
// says which side of the tie x is on.
__device__ __forceinline__ int code_of(float x, float s, float inv, float top) {
    if (!(s > 0.0f)) return 0;
    if (x != x) return 0;
    if (finite_abs(x) != fabsf(x)) return x > 0.0f ? (int)top : -(int)top;
    float c = rintf(x * inv);
    const float r = fmaf(-c, s, x), half = 0.5f * s;
    if (fabsf(r) > half)
        c += copysignf(1.0f, r);
    else if (fabsf(r) == half && ((int)c & 1))
        c += copysignf(1.0f, r);
    return (int)fminf(fmaxf(c, -top), top);
}

// grid (rows / 64, heads, keys and values); 256 threads: sixteen lanes a row, four numbers a lane at a time. Values go through
// LDS, so that a page's rows of one coordinate are stored four at a time.
template <int FMT>
__global__ __launch_bounds__(256) void k_pages_write(PageSet p, const int32_t *__restrict__ starts,
                                                     const int32_t *__restrict__ offsets, const float *__restrict__ k,
                                                     const float *__restrict__ v, int rows, size_t row_ld) {
    typedef typename Number<FMT>::T T;
    typedef typename Number<FMT>::V V;
    __shared__ T tile[128][TILE + 4];
    __shared__ int offs[IN_LDS + 1];
    __shared__ Places pl;
    const int tid = threadIdx.x, l16 = tid & 15, h = blockIdx.y;
    const bool values = blockIdx.z == 1;
    const int r0 = blockIdx.x * TILE, hd = p.hd, P = p.rows;
    find_places(p, starts, offsets, r0, rows, offs, pl);
    const float *src = (values ? v : k) + (size_t)h * hd;
    uint8_t *head = p.pool + (size_t)h * p.head_bytes;
#pragma unroll
    for (int pass = 0; pass < TILE / 16; pass++) {
        const int i = 16 * pass + (tid >> 4), page = pl.page[i], slot = pl.slot[i];
        floatx4 x[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int dim = 64 * c + 4 * l16;
            x[c] = page >= 0 && dim < hd ? (floatx4) * reinterpret_cast<const floatx4u *>(src + (size_t)(r0 + i) * row_ld + dim)
                                         : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float s = 0.0f, inv = 0.0f;
        if constexpr (FMT != TAH_KV_F32) {
            float big = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) big = fmaxf(big, finite_abs(x[c][j]));
            big = row16_reduce(big, fmaxf);
            s = big / Number<FMT>::top;
            if (s < 0x1p-126f) s = 0.0f;
            inv = 1.0f / s;
        }
        uint8_t *base = head + (size_t)max(page, 0) * p.page_bytes;
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int dim = 64 * c + 4 * l16;
            V w;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (FMT == TAH_KV_F32)
                    w[j] = x[c][j];
                else
                    w[j] = (T)code_of(x[c][j], s, inv, Number<FMT>::top);
            }
            if (dim >= hd) continue;
            if (values) {
#pragma unroll
                for (int j = 0; j < 4; j++) tile[dim + j][i] = w[j];
            } else if (page >= 0) {
                *reinterpret_cast<V *>(reinterpret_cast<T *>(base) + (size_t)slot * hd + dim) = w;
            }
        }
        if constexpr (FMT != TAH_KV_F32)
            if (page >= 0 && l16 == 0)
                reinterpret_cast<float *>(base + 2 * (size_t)P * hd * sizeof(T))[(values ? P : 0) + slot] = s;
    }
    if (!values) return;
    __syncthreads();
    const int first = pl.first;
    for (int u = tid; u < hd * QUADS; u += 256) {
        const int dim = u / QUADS, q = u - dim * QUADS, a = first + 4 * q;
        if (pl.whole[q]) {
            T *dst = reinterpret_cast<T *>(head + (size_t)pl.page[a] * p.page_bytes) + (size_t)P * hd + (size_t)dim * P + pl.slot[a];
            V w;
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = tile[dim][a + j];
            *reinterpret_cast<V *>(dst) = w;
        } else {
            for (int i = max(a, 0); i < min(a + 4, TILE); i++)
                if (pl.page[i] >= 0)
                    reinterpret_cast<T *>(head + (size_t)pl.page[i] * p.page_bytes)[(size_t)P * hd + (size_t)dim * P + pl.slot[i]] =
                        tile[dim][i];
        }
    }
}

// grid as k_pages_write's: the same the other way, rows on no page as zeros.
template <int FMT>
__global__ __launch_bounds__(256) void k_pages_read(PageSet p, const int32_t *__restrict__ starts,
                                                    const int32_t *__restrict__ offsets, float *__restrict__ k,
                                                    float *__restrict__ v, int rows, size_t row_ld) {
    typedef typename Number<FMT>::T T;
    typedef typename Number<FMT>::V V;
    __shared__ T tile[128][TILE + 4];
    __shared__ int offs[IN_LDS + 1];
    __shared__ Places pl;
    const int tid = threadIdx.x, l16 = tid & 15, h = blockIdx.y;
    const bool values = blockIdx.z == 1;
    const int r0 = blockIdx.x * TILE, hd = p.hd, P = p.rows;
    find_places(p, starts, offsets, r0, rows, offs, pl);
    float *dst = (values ? v : k) + (size_t)h * hd;
    const uint8_t *head = p.pool + (size_t)h * p.head_bytes;
    if (values) {
        const int first = pl.first;
        for (int u = tid; u < hd * QUADS; u += 256) {
            const int dim = u / QUADS, q = u - dim * QUADS, a = first + 4 * q;
            if (pl.whole[q]) {
                const V w = *reinterpret_cast<const V *>(reinterpret_cast<const T *>(head + (size_t)pl.page[a] * p.page_bytes) +
                                                         (size_t)P * hd + (size_t)dim * P + pl.slot[a]);
#pragma unroll
                for (int j = 0; j < 4; j++) tile[dim][a + j] = w[j];
            } else {
                for (int i = max(a, 0); i < min(a + 4, TILE); i++)
                    if (pl.page[i] >= 0)
                        tile[dim][i] = reinterpret_cast<const T *>(head + (size_t)pl.page[i] * p.page_bytes)[(size_t)P * hd + (size_t)dim * P + pl.slot[i]];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int pass = 0; pass < TILE / 16; pass++) {
        const int i = 16 * pass + (tid >> 4), page = pl.page[i], slot = pl.slot[i];
        const uint8_t *base = head + (size_t)max(page, 0) * p.page_bytes;
        float s = 1.0f;
        if constexpr (FMT != TAH_KV_F32)
            if (page >= 0) s = reinterpret_cast<const float *>(base + 2 * (size_t)P * hd * sizeof(T))[(values ? P : 0) + slot];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int dim = 64 * c + 4 * l16;
            if (dim >= hd) continue;
            floatx4 x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (page >= 0) {
                V w;
                if (values) {
#pragma unroll
                    for (int j = 0; j < 4; j++) w[j] = tile[dim + j][i];
                } else {
                    w = *reinterpret_cast<const V *>(reinterpret_cast<const T *>(base) + (size_t)slot * hd + dim);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = (float)w[j] * s;
            }
            if (page >= -1) *reinterpret_cast<floatx4u *>(dst + (size_t)(r0 + i) * row_ld + dim) = x;
        }
    }
}

template <int FMT>
void launch_rows(hipStream_t s, const PageSet &p, const int32_t *starts, const int32_t *offsets, float *k, float *v, int rows,
                 size_t row_ld, bool write) {
    const dim3 grid((rows + TILE - 1) / TILE, p.heads, 2);
    if (write)
        hipLaunchKernelGGL(k_pages_write<FMT>, grid, dim3(256), 0, s, p, starts, offsets, k, v, rows, row_ld);
    else
        hipLaunchKernelGGL(k_pages_read<FMT>, grid, dim3(256), 0, s, p, starts, offsets, k, v, rows, row_ld);
    TAH_LAUNCHED();
}

}  // namespace

void pages_rows(hipStream_t s, int fmt, const PageSet &p, const int32_t *starts, const int32_t *offsets, float *k, float *v,
                int rows, size_t row_ld, bool write) {
    if (rows <= 0) return;
    if (fmt == TAH_KV_F32)
        launch_rows<TAH_KV_F32>(s, p, starts, offsets, k, v, rows, row_ld, write);
    else if (fmt == TAH_KV_I16)
        launch_rows<TAH_KV_I16>(s, p, starts, offsets, k, v, rows, row_ld, write);
    else
        launch_rows<TAH_KV_I8>(s, p, starts, offsets, k, v, rows, row_ld, write);
}

}  // namespace tah

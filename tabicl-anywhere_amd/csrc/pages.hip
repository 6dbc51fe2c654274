// Rows of many tables into pages of a pool and back (tah_pages_write, tah_pages_read): the step of a row's head, the ints, and
// the values' transposition.
#include "device_math.hpp"
#include "pages.hpp"

namespace tah {

namespace {

constexpr int TILE = 64;      // rows a workgroup
constexpr int IN_LDS = 256;   // tables whose offsets a workgroup looks through in LDS
constexpr int MOST_TILES = (1 << 24) - 1;  // workgroups of 256 threads in a dimension of a launch

template <int FMT>
struct Number;
template <>
struct Number<TAH_KV_F32> {
    typedef float T;
};
template <>
struct Number<TAH_KV_I16> {
    typedef int16_t T;
    static constexpr float top = 32767.0f;
};
template <>
struct Number<TAH_KV_I8> {
    typedef int8_t T;
    static constexpr float top = 127.0f;
};

// 16 bytes of which no alignment is known (a page's row of a coordinate, from any row on)
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(1)));

// Where a workgroup's rows lie: page (-1: none, -2: a row of no table) and slot of each, and which rows (bits) lie behind the row
// before them in a page.
struct Places {
    int page[TILE], slot[TILE];
    uint64_t follows;
    int ahead;  // rows from a multiple of sixteen rows of its page to where row 0 is, or would be before the first that is on one
    int offs[IN_LDS + 1], starts[IN_LDS];
};

__device__ __forceinline__ void find_places(const PageSet &p, const int32_t *starts, const int32_t *offsets, int r0, int rows,
                                            Places &pl) {
    const int tid = threadIdx.x;
    const bool in_lds = p.tables < IN_LDS;
    if (in_lds) {
        for (int i = tid; i <= p.tables; i += 256) {
            pl.offs[i] = offsets[i];
            pl.starts[min(i, p.tables - 1)] = starts[min(i, p.tables - 1)];
        }
        __syncthreads();
    }
    if (tid < TILE) {
        const int r = r0 + tid;
        int page = -2, slot = 0;
        if (r < rows) {
            const int32_t *o = in_lds ? pl.offs : offsets;
            const int t = table_of(o, p.tables, r);
            if (r >= o[t] && r < o[t + 1]) {
                const long at = (long)(in_lds ? pl.starts : starts)[t] + (r - o[t]);
                page = page_of(p, t, at);
                slot = (int)(at & (p.rows - 1));
            }
        }
        pl.page[tid] = page;
        pl.slot[tid] = slot;
        const int page_before = __shfl_up(page, 1), slot_before = __shfl_up(slot, 1);
        const uint64_t follows = __ballot(tid > 0 && page >= 0 && page == page_before && slot == slot_before + 1);
        const uint64_t some = __ballot(page >= 0);
        const int lead = some ? __ffsll((unsigned long long)some) - 1 : 0;
        const int ahead = (__shfl(slot, lead) - lead) & 15;
        if (tid == 0) {
            pl.follows = follows;
            pl.ahead = ahead;
        }
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

// The ints of sixteen lanes' 4 C numbers of a row, in the low bits, and the row's step. Nearly always a number's residual is
// below half a step, and the rounding by adding 1.5 2^23 (whose low bits are the int) right; a lane where one is not, or where a number
// is not finite, takes code_of.
template <int FMT, int C>
__device__ __forceinline__ float quantise(const floatx4 (&x)[C], uint32_t (&code)[4 * C]) {
    constexpr float TOP = Number<FMT>::top, MAGIC = 12582912.0f;
    uint32_t raw = 0;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float f = x[c][j];
            raw = max(raw, __float_as_uint(f) & 0x7fffffffu);
        }
    float big = __uint_as_float(raw);
    if (raw >= 0x7f800000u) {
        big = 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) big = fmaxf(big, finite_abs(x[c][j]));
    }
    big = row16_reduce(big, fmaxf);
    float s = big / TOP;
    if (s < 0x1p-126f) s = 0.0f;
    const float inv = s > 0.0f ? 1.0f / s : 0.0f, half = s > 0.0f ? 0.5f * s : INFINITY;
    bool near = false;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float f = x[c][j], t = fmaf(f, inv, MAGIC), r = fmaf(MAGIC - t, s, f);
            near = near || !(fabsf(r) < half);
            code[4 * c + j] = __float_as_uint(t);
        }
    if (near) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) code[4 * c + j] = (uint32_t)code_of(x[c][j], s, inv, TOP);
    }
    return s;
}

// low bytes (FMT i8) or halves (i16) of four ints, in order; four floats (f32)
template <int FMT>
__device__ __forceinline__ void pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t *to) {
    if constexpr (FMT == TAH_KV_I8) {
        const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
        to[0] = lo | hi;
    } else if constexpr (FMT == TAH_KV_I16) {
        to[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        to[1] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    } else {
        to[0] = a;
        to[1] = b;
        to[2] = c;
        to[3] = d;
    }
}
// number j of four so packed
template <int FMT>
__device__ __forceinline__ float number4(const uint32_t *from, int j) {
    if constexpr (FMT == TAH_KV_I8)
        return (float)(int8_t)(from[0] >> (8 * j));
    else if constexpr (FMT == TAH_KV_I16)
        return (float)(int16_t)(from[j >> 1] >> (16 * (j & 1)));
    else
        return __uint_as_float(from[j]);
}

// words of four numbers, and of a coordinate's row of 64 in LDS (apart so that neither four lanes' fours nor the next coordinates'
// fall on the same banks)
template <int FMT>
struct Words {
    static constexpr int N = page_width(FMT), ROW = TILE * N / 4 + (N == 4 ? 4 : N);
};

// the first row of a workgroup: grid (rows / 64 of a part, heads, keys and values of each part), parts of part_rows where rows are too
// many for one dimension. The last ones may have none: all are looked at as rows behind the last.
__device__ __forceinline__ int first_row(int part_rows) { return (int)((blockIdx.z >> 1) * (uint32_t)part_rows + blockIdx.x * TILE); }

// grid (rows / 64, heads, keys and values); 256 threads: four rows and four of each 64 coordinates a lane, sixteen lanes a row.
// Bound by bytes: 40 tables of up to 1,500 rows, 4 heads of 128 to i16 (180 MB) take 43 us at least (median 47), at the rate of a large
// copy 35; without its stores the kernel takes 25 us (the reads at 4.7 TB/s), without its arithmetic 2 to 4 less. Values are turned in
// LDS, so that a page's rows of one coordinate are stored 16 bytes at a time. The floats pass the caches by, here and in k_pages_read
// (written and read back 92 -> 78 us, 10,000 rows of 8 heads of 64 in i8 24.3 -> 24.0): what is wanted next is the pages.
template <int FMT, int C>
__global__ __launch_bounds__(256) void k_pages_write(PageSet p, const int32_t *__restrict__ starts,
                                                     const int32_t *__restrict__ offsets, const float *__restrict__ k,
                                                     const float *__restrict__ v, int rows, size_t row_ld, int part_rows) {
    typedef typename Number<FMT>::T T;
    constexpr int N = Words<FMT>::N, ROW = Words<FMT>::ROW, W = page_width(FMT), RUN = 16 / W;
    __shared__ uint32_t tile[64 * C][ROW];
    __shared__ Places pl;
    const int tid = threadIdx.x, l16 = tid & 15, quad = tid >> 4, h = blockIdx.y;
    const bool values = blockIdx.z & 1;
    const int r0 = first_row(part_rows), hd = p.hd, P = p.rows;
    const float *src = (values ? v : k) + (size_t)h * hd;
    floatx4 x[4][C];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int dim = 64 * c + 4 * l16;
            x[i][c] = __builtin_nontemporal_load(
                reinterpret_cast<const floatx4u *>(src + (size_t)min(r0 + 4 * quad + i, rows - 1) * row_ld + (dim < hd ? dim : 0)));
            if (dim >= hd) x[i][c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    find_places(p, starts, offsets, r0, rows, pl);
    uint8_t *head = p.pool + (size_t)h * p.head_bytes;
    uint32_t code[4][4 * C];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int page = pl.page[4 * quad + i], slot = pl.slot[4 * quad + i];
        uint8_t *base = head + (size_t)max(page, 0) * p.page_bytes;
        if constexpr (FMT == TAH_KV_F32) {
#pragma unroll
            for (int j = 0; j < 4 * C; j++) {
                const float f = x[i][j >> 2][j & 3];
                code[i][j] = __float_as_uint(f);
            }
        } else {
            const float s = quantise<FMT, C>(x[i], code[i]);
            if (page >= 0 && l16 == 0) reinterpret_cast<float *>(base + 2 * (size_t)P * hd * W)[(values ? P : 0) + slot] = s;
        }
        if (values || page < 0) continue;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int dim = 64 * c + 4 * l16;
            if (dim >= hd) continue;
            uint32_t w[N];
            pack4<FMT>(code[i][4 * c], code[i][4 * c + 1], code[i][4 * c + 2], code[i][4 * c + 3], w);
            uint32_t *to = reinterpret_cast<uint32_t *>(base + ((size_t)slot * hd + dim) * W);
#pragma unroll
            for (int n = 0; n < N; n++) to[n] = w[n];
        }
    }
    if (!values) return;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t w[N];
            pack4<FMT>(code[0][4 * c + j], code[1][4 * c + j], code[2][4 * c + j], code[3][4 * c + j], w);
#pragma unroll
            for (int n = 0; n < N; n++) tile[64 * c + 4 * l16 + j][N * quad + n] = w[n];
        }
    __syncthreads();
    // runs of 16 bytes that are so aligned in their page, where the rows are one table's: from `ahead` rows before one on
    const uint64_t follows = pl.follows;
    const int ahead = pl.ahead & (RUN - 1), runs = TILE / RUN + (ahead ? 1 : 0);  // of a coordinate
    const uint32_t per_dim = (65536 + runs - 1) / runs;  // u / runs as a product, exact for every u here
    for (int u = tid; u < hd * runs; u += 256) {
        const int dim = (int)((u * per_dim) >> 16), a = RUN * (u - dim * runs) - ahead;
        T *part = reinterpret_cast<T *>(head) + (size_t)P * hd + (size_t)dim * P;  // of page 0
        const uint64_t behind = a >= 0 ? (((uint64_t)1 << RUN) - 2) << a : 0;
        if (a >= 0 && a + RUN <= TILE && pl.page[a] >= 0 && (follows & behind) == behind) {
            // from anywhere in the row's words: the run lies between five of them
            const int at = a * W >> 2;
            uint32_t w[5];
#pragma unroll
            for (int n = 0; n < 5; n++) w[n] = tile[dim][at + n];  // at most the row's padding
            u32x4 o;
#pragma unroll
            for (int n = 0; n < 4; n++) o[n] = __builtin_amdgcn_alignbyte(w[n + 1], w[n], a * W & 3);
            *reinterpret_cast<u32x4u *>(reinterpret_cast<uint8_t *>(part + pl.slot[a]) + (size_t)pl.page[a] * p.page_bytes) = o;
        } else {
#pragma unroll
            for (int i = 0; i < RUN; i++) {
                const int r = a + i;
                if (r >= 0 && r < TILE && pl.page[r] >= 0)
                    *reinterpret_cast<T *>(reinterpret_cast<uint8_t *>(part + pl.slot[r]) + (size_t)pl.page[r] * p.page_bytes) =
                        reinterpret_cast<const T *>(tile[dim])[r];
            }
        }
    }
}

// grid and lanes as k_pages_write's: the same the other way, rows on no page as zeros.
template <int FMT, int C>
__global__ __launch_bounds__(256) void k_pages_read(PageSet p, const int32_t *__restrict__ starts,
                                                    const int32_t *__restrict__ offsets, float *__restrict__ k,
                                                    float *__restrict__ v, int rows, size_t row_ld, int part_rows) {
    typedef typename Number<FMT>::T T;
    constexpr int N = Words<FMT>::N, ROW = Words<FMT>::ROW, W = page_width(FMT), RUN = 16 / W, RUNS = TILE / RUN;
    __shared__ uint32_t tile[64 * C][ROW];
    __shared__ Places pl;
    const int tid = threadIdx.x, l16 = tid & 15, quad = tid >> 4, h = blockIdx.y;
    const bool values = blockIdx.z & 1;
    const int r0 = first_row(part_rows), hd = p.hd, P = p.rows;
    find_places(p, starts, offsets, r0, rows, pl);
    const uint8_t *head = p.pool + (size_t)h * p.head_bytes;
    if (values) {
        const uint64_t follows = pl.follows;
#pragma unroll 4
        for (int u = tid; u < hd * RUNS; u += 256) {
            const int dim = u / RUNS, a = RUN * (u % RUNS);
            const uint64_t behind = (((uint64_t)1 << RUN) - 2) << a;
            const T *part = reinterpret_cast<const T *>(head) + (size_t)P * hd + (size_t)dim * P;
            uint32_t *to = &tile[dim][4 * (u % RUNS)];
            if (pl.page[a] >= 0 && (follows & behind) == behind) {
                const u32x4 w = *reinterpret_cast<const u32x4u *>(reinterpret_cast<const uint8_t *>(part + pl.slot[a]) +
                                                                  (size_t)pl.page[a] * p.page_bytes);
#pragma unroll
                for (int n = 0; n < 4; n++) to[n] = w[n];
            } else {
                T w[RUN];
#pragma unroll
                for (int i = 0; i < RUN; i++)  // rows on no page: page 0's, not used
                    w[i] = *reinterpret_cast<const T *>(reinterpret_cast<const uint8_t *>(part + pl.slot[a + i]) +
                                                        (size_t)max(pl.page[a + i], 0) * p.page_bytes);
#pragma unroll
                for (int i = 0; i < RUN; i++) reinterpret_cast<T *>(to)[i] = w[i];
            }
        }
        __syncthreads();
    }
    uint32_t w[4][C][N];
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int page = pl.page[4 * quad + i], slot = pl.slot[4 * quad + i];
        const uint8_t *base = head + (size_t)max(page, 0) * p.page_bytes;
        s[i] = FMT == TAH_KV_F32 ? 1.0f : reinterpret_cast<const float *>(base + 2 * (size_t)P * hd * W)[(values ? P : 0) + slot];
        if (values) continue;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int dim = 64 * c + 4 * l16;
            const uint32_t *from = reinterpret_cast<const uint32_t *>(base + ((size_t)slot * hd + (dim < hd ? dim : 0)) * W);
#pragma unroll
            for (int n = 0; n < N; n++) w[i][c][n] = from[n];
        }
    }
    uint32_t t[C][4][N];  // values: four rows of a coordinate
    if (values) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int n = 0; n < N; n++) t[c][j][n] = tile[64 * c + 4 * l16 + j][N * quad + n];
    }
    float *dst = (values ? v : k) + (size_t)h * hd;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int page = pl.page[4 * quad + i];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int dim = 64 * c + 4 * l16;
            floatx4 x;
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[j] = page >= 0 ? (values ? number4<FMT>(t[c][j], i) : number4<FMT>(w[i][c], j)) * s[i] : 0.0f;
            if (dim < hd && page >= -1)
                __builtin_nontemporal_store((floatx4u)x, reinterpret_cast<floatx4u *>(dst + (size_t)(r0 + 4 * quad + i) * row_ld + dim));
        }
    }
}

template <int FMT, int C>
void launch_rows(hipStream_t s, const PageSet &p, const int32_t *starts, const int32_t *offsets, float *k, float *v, int rows,
                 size_t row_ld, bool write) {
    // fewer than 2^32 threads in a dimension
    const int tiles = (rows + TILE - 1) / TILE, parts = tiles / MOST_TILES + 1;
    const dim3 grid((tiles + parts - 1) / parts, p.heads, 2 * parts);
    const int part_rows = (int)grid.x * TILE;
    if (write)
        hipLaunchKernelGGL((k_pages_write<FMT, C>), grid, dim3(256), 0, s, p, starts, offsets, k, v, rows, row_ld, part_rows);
    else
        hipLaunchKernelGGL((k_pages_read<FMT, C>), grid, dim3(256), 0, s, p, starts, offsets, k, v, rows, row_ld, part_rows);
    TAH_LAUNCHED();
}

template <int FMT>
void launch_width(hipStream_t s, const PageSet &p, const int32_t *starts, const int32_t *offsets, float *k, float *v, int rows,
                  size_t row_ld, bool write) {
    if (p.hd <= 64)
        launch_rows<FMT, 1>(s, p, starts, offsets, k, v, rows, row_ld, write);
    else
        launch_rows<FMT, 2>(s, p, starts, offsets, k, v, rows, row_ld, write);
}

}  // namespace

void pages_rows(hipStream_t s, int fmt, const PageSet &p, const int32_t *starts, const int32_t *offsets, float *k, float *v,
                int rows, size_t row_ld, bool write) {
    if (rows <= 0) return;
    if (fmt == TAH_KV_F32)
        launch_width<TAH_KV_F32>(s, p, starts, offsets, k, v, rows, row_ld, write);
    else if (fmt == TAH_KV_I16)
        launch_width<TAH_KV_I16>(s, p, starts, offsets, k, v, rows, row_ld, write);
    else
        launch_width<TAH_KV_I8>(s, p, starts, offsets, k, v, rows, row_ld, write);
}

}  // namespace tah

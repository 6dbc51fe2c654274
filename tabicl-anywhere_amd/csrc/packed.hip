// Attention of packed tables (tah_attend_packed): every table's queries over its own rows, causal or not, grouped heads, at f32's
// precision on the fp16 matrix cores.
//
// Keys and values become split-fp16 tiles first, one per (block of 64 of a table's rows, key/value head), laid out as the LDS
// images that the attention reads: tables begin at tiles of their own, short blocks are filled with zeros. The attention then
// takes a tile of queries of one table and head a workgroup.
#include "common.hpp"
#include "device_math.hpp"
#include "tiles.hpp"

namespace tah {

namespace {

struct Packed {
    const float *q, *k, *v;
    const int32_t *qo, *ko;
    int tables, nq, nkv, heads, kv_heads, hd, causal;
    size_t q_ld, kv_ld;
    float *out;
    // working memory: the tiles, per tile the keys' and the values' power of two (twice it, and 1 if a value is not finite), which
    // keys of each coordinate hold values that are not, the tables' first blocks, the key ranges' states
    int blocks;  // room for so many
    uint8_t *tiles;
    int *shifts;
    uint64_t *odd;
    uint32_t *first;
    int splits;
    float *part_o;
    float2 *part_ml;
};

// rows [a, a + n) of table t, cut to what there are
__device__ __forceinline__ int rows_of(const int32_t *offsets, int t, int rows, int &a) {
    a = min(max(offsets[t], 0), rows);
    return min(max(offsets[t + 1], a), rows) - a;
}

// The table whose units (size units of its rows) hold unit `at` of all: its number (-1 if there are fewer), and `at` within it.
// Every lane of a wavefront calls it.
__device__ __forceinline__ int table_with(const int32_t *offsets, int tables, int rows, int size, uint32_t at, uint32_t &within) {
    const int lane = threadIdx.x & 63;
    uint64_t before = 0;
    for (int t0 = 0; t0 < tables; t0 += 64) {
        int a = 0;
        const uint32_t c = t0 + lane < tables ? (uint32_t)((rows_of(offsets, t0 + lane, rows, a) + size - 1) / size) : 0;
        const uint64_t sum = before + wave_scan(c);  // of 64 tables: below 2^32
        const uint64_t past = __ballot(sum > at);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            within = at - (uint32_t)__shfl(sum - c, l);
            return __builtin_amdgcn_readfirstlane(t0 + l);
        }
        before = __shfl(sum, 63);
    }
    return -1;
}

// Bytes of a tile of C x 64 coordinates: keys by 64 coordinates, hi then lo [64 keys][64] each, then values, hi then lo [64 C][64
// keys], rows of 128 bytes in swizzled chunks of 16 (swz).
template <int C>
constexpr int TILE_BYTES = C * 32768;

// grid (blocks, key/value heads, keys and values); 256 threads: one half tile. Scaled by the power of two that brings its own
// largest finite number below 2^14. A value that is not finite is a zero in the tile, and its bit is set in `odd`.
template <int C>
__global__ __launch_bounds__(256) void k_packed_tiles(Packed p) {
    constexpr int HD = 64 * C;
    __shared__ float x[KB][HD + 1];
    __shared__ float most[4];
    __shared__ int some[4];
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.y;
    const bool values = blockIdx.z == 1;
    if (blockIdx.x == 0 && h == 0 && !values && tid < 64) {  // the tables' first blocks, for the attention
        uint64_t before = 0;
        for (int t0 = 0; t0 < p.tables; t0 += 64) {
            int a = 0;
            const uint32_t c = t0 + lane < p.tables ? (uint32_t)((rows_of(p.ko, t0 + lane, p.nkv, a) + KB - 1) / KB) : 0;
            const uint64_t sum = before + wave_scan(c);
            if (t0 + lane < p.tables) p.first[t0 + lane] = (uint32_t)min(sum - c, (uint64_t)0x7fffffff);
            before = __shfl(sum, 63);
        }
    }
    uint32_t kb = 0;
    const int t = table_with(p.ko, p.tables, p.nkv, KB, blockIdx.x, kb);
    if (t < 0) return;
    int a = 0;
    const int n = min(rows_of(p.ko, t, p.nkv, a) - (int)kb * KB, KB);
    const float *src = (values ? p.v : p.k) + (size_t)(a + (int)kb * KB) * p.kv_ld + (size_t)h * p.hd;
    uint32_t big = 0, raw = 0;
#pragma unroll
    for (int i = 0; i < KB * HD / 4 / 256; i++) {
        const int u = tid + 256 * i, r = u / (HD / 4), dim = 4 * (u % (HD / 4));
        const floatx4 w = r < n && dim < p.hd ? (floatx4) * reinterpret_cast<const floatx4u *>(src + (size_t)r * p.kv_ld + dim)
                                              : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float f = w[j];
            const uint32_t b = __float_as_uint(f);
            big = max(big, finite_bits(b));
            raw = max(raw, b & 0x7fffffffu);
            x[r][dim + j] = f;
        }
    }
    const float m = wave_max(__uint_as_float(big));
    const bool any = __any(raw >= 0x7f800000u);
    if (lane == 0) {
        most[tid >> 6] = m;
        some[tid >> 6] = any;
    }
    __syncthreads();
    const int shift = min(shift_for_max(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]))), 126);
    const bool odd = values && (some[0] | some[1] | some[2] | some[3]);
    const float f = pow2(shift);
    const size_t at = (size_t)blockIdx.x * p.kv_heads + h;
    if (tid == 0) p.shifts[2 * at + (values ? 1 : 0)] = values ? 2 * shift + (odd ? 1 : 0) : shift;
    uint8_t *tile = p.tiles + at * TILE_BYTES<C>;
    if (odd && tid < HD) {
        uint64_t bits = 0;
        for (int r = 0; r < KB; r++) {
            const bool b = (__float_as_uint(x[r][tid]) & 0x7fffffffu) >= 0x7f800000u;
            bits |= (uint64_t)b << r;
        }
        p.odd[at * HD + tid] = bits;
    }
#pragma unroll
    for (int i = 0; i < HD * 8 / 256; i++) {
        const int u = tid + 256 * i, c = u & 7;
        float w[8];
        uint8_t *hi;
        if (values) {
            const int r = u >> 3;  // coordinate r, keys 8 c ..
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = x[8 * c + e][r];
                w[e] = odd && (__float_as_uint(y) & 0x7fffffffu) >= 0x7f800000u ? 0.0f : y;
            }
            hi = tile + C * 16384 + r * 128 + swz(r, c) * 16;
        } else {
            const int part = u >> 9, r = (u >> 3) & 63;  // key r, coordinates 64 part + 8 c ..
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = x[r][64 * part + 8 * c + e];
            hi = tile + part * 16384 + r * 128 + swz(r, c) * 16;
        }
        halfx8 wh, wl;
        split8(w, f, wh, wl);
        *reinterpret_cast<halfx8 *>(hi) = wh;
        *reinterpret_cast<halfx8 *>(hi + (values ? C * 8192 : 8192)) = wl;
    }
}

// grid (query tiles x heads x key ranges); 64 WAVES threads, 32 queries of one table and head a wavefront.
//
// S^T = K Q^T and O^T += V^T P^T by v_mfma_f32_32x32x16_f16, three products of halves a term, the keys in sigma32 order so that
// the weights of a block are the values' operand where they stand. Tiles come by DMA into two LDS buffers each for keys and
// values. The softmax is in log2 units against a reference that is raised when a block passes it by more than 3; weights stay
// below 2^15. The sums are held in units of the least power of two that the values' tiles so far have; a block with a larger one
// has its weights smaller by the difference (at most 2^60: what is cut off there is below 2^-60 of the largest value).
template <int C, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void k_packed(Packed p) {
    constexpr int QT = 32 * WAVES, HALF = C * 16384, HD = 64 * C;
    __shared__ __align__(16) uint8_t kt[2][HALF], vt[2][HALF];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r32 = lane & 31, g = lane >> 5;
    const int per_tile = p.heads * p.splits, tile_at = blockIdx.x / per_tile, rest = blockIdx.x - tile_at * per_tile;
    const int split = rest / p.heads, hpos = rest - split * p.heads;
    // heads that share keys on the same XCD (workgroup i runs on XCD i % 8)
    const int h = p.heads % 8 == 0 ? (hpos % 8) * (p.heads / 8) + hpos / 8 : hpos, hk = h / (p.heads / p.kv_heads);
    uint32_t tile = 0;
    const int t = table_with(p.qo, p.tables, p.nq, QT, tile_at, tile);
    if (t < 0) return;
    int qa = 0, ka = 0;
    const int n_q = rows_of(p.qo, t, p.nq, qa), n_t = rows_of(p.ko, t, p.nkv, ka);
    const uint32_t first = p.first[t];
    // a table past the room that the offsets' promise gives has no rows
    const int n_k = (uint64_t)first + (n_t + KB - 1) / KB <= (uint64_t)p.blocks ? n_t : 0;
    // causal: a table's last tile first, which has the most to do
    const int q0 = (p.causal ? (n_q + QT - 1) / QT - 1 - (int)tile : (int)tile) * QT, w0 = q0 + 32 * wave, qi = w0 + r32;
    auto limit_of = [&](int i) { return p.causal ? max(0, n_k - (n_q - 1 - i)) : n_k; };
    const bool live = qi < n_q;
    const int limit = live ? limit_of(qi) : n_k, least = w0 < n_q ? limit_of(w0) : n_k;
    const int nb = (limit_of(min(n_q, q0 + QT) - 1) + KB - 1) / KB;
    const int kb0 = (int)((long)nb * split / p.splits), kb1 = (int)((long)nb * (split + 1) / p.splits);
    const uint8_t *tiles = p.tiles + ((size_t)first * p.kv_heads + hk) * TILE_BYTES<C>;
    const int *shifts = p.shifts + 2 * ((size_t)first * p.kv_heads + hk);
    const size_t kb_bytes = (size_t)p.kv_heads * TILE_BYTES<C>;
    auto keys_to = [&](int kb, int s) { half_image_to_lds<WAVES, HALF>(tiles + kb * kb_bytes, kt[s], tid); };
    auto values_to = [&](int kb, int s) { half_image_to_lds<WAVES, HALF>(tiles + kb * kb_bytes + HALF, vt[s], tid); };
    if (kb0 < kb1) {
        keys_to(kb0, 0);
        values_to(kb0, 0);
    }
    // this lane's query coordinates 16 dc + 8 g + t, at a maximum near 2^14, split
    halfx8 qh[4 * C], ql[4 * C];
    float to_log2;
    {
        float qv[4 * C][8], most = 0.0f;
        const float *src = p.q + (size_t)(qa + (live ? qi : 0)) * p.q_ld + (size_t)h * p.hd;
#pragma unroll
        for (int dc = 0; dc < 4 * C; dc++) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const floatx4 w = live && 16 * dc < p.hd ? (floatx4) * reinterpret_cast<const floatx4u *>(src + 16 * dc + 8 * g + 4 * j)
                                                         : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float f = w[e];
                    qv[dc][4 * j + e] = f;
                    most = fmaxf(most, __uint_as_float(finite_bits(__float_as_uint(f))));
                }
            }
        }
        most = half_max(most);
        const int eq = min(shift_for_max(most), 126);
        const float f = pow2(eq);
#pragma unroll
        for (int dc = 0; dc < 4 * C; dc++) split8(qv[dc], f, qh[dc], ql[dc]);
        to_log2 = LOG2E * pow2(-eq);
    }
    const int krow = sigma32(r32);
    float ref = -INFINITY, l = 0.0f;
    int ev = 1000;  // the sums are in units of 2^-ev
    floatx16 acc[2 * C];
#pragma unroll
    for (int db = 0; db < 2 * C; db++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[db][v] = 0.0f;
    floatx16 zero;
#pragma unroll
    for (int v = 0; v < 16; v++) zero[v] = 0.0f;

    auto scores = [&](const uint8_t *buf, floatx16 (&sc)[2]) {
#pragma unroll
        for (int dc = 0; dc < 4 * C; dc++)
#pragma unroll
            for (int kh = 0; kh < 2; kh++) {
                const int r = 32 * kh + krow;
                const uint8_t *at = buf + (dc >> 2) * 16384 + r * 128 + swz(r, 2 * (dc & 3) + g) * 16;
                const halfx8 hi = *reinterpret_cast<const halfx8 *>(at), lo = *reinterpret_cast<const halfx8 *>(at + 8192);
                sc[kh] = mfma16(hi, qh[dc], dc == 0 ? zero : sc[kh]);
                sc[kh] = mfma16(hi, ql[dc], sc[kh]);
                sc[kh] = mfma16(lo, qh[dc], sc[kh]);
            }
    };
    auto step = [&](int kb) {
        const int sl = (kb - kb0) & 1;
        __builtin_amdgcn_s_waitcnt(0);  // this wavefront's copies of block kb have landed
        __syncthreads();                // everyone's have, and block kb - 1's buffers are no longer read
        if (kb + 1 < kb1) {
            keys_to(kb + 1, sl ^ 1);
            values_to(kb + 1, sl ^ 1);
        }
        const int *sh = shifts + 2 * (size_t)kb * p.kv_heads;
        const int ek = sh[0], evo = sh[1], eb = evo >> 1;
        floatx16 sc[2];
        scores(kt[sl], sc);
        const float f = fminf(fmaxf(to_log2 * pow2(-ek), 0x1p-126f), 0x1p126f);
        if ((kb + 1) * KB > least) {
            const int lim = limit - kb * KB - 8 * g;  // accumulator v of half kh is seen while 32 kh + 16 (v / 8) + v % 8 < lim
#pragma unroll
            for (int kh = 0; kh < 2; kh++)
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (32 * kh + 16 * (v >> 3) + (v & 7) >= lim) sc[kh][v] = -INFINITY;
        }
        float mb = -INFINITY;
#pragma unroll
        for (int kh = 0; kh < 2; kh++)
#pragma unroll
            for (int v = 0; v < 16; v++) mb = fmaxf(mb, sc[kh][v]);
        mb = half_max(mb) * f;
        const bool grow = mb > ref + 3.0f;
        if (__any(grow)) {
            const float nref = grow ? mb : ref;
            const float alpha = grow ? exp2_hw(ref - nref) : 1.0f;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < 2 * C; db++) acc[db] *= alpha;
            ref = nref;
        }
        if (eb < ev) {
            const float beta = ev < 1000 ? pow2(eb - ev) : 0.0f;
#pragma unroll
            for (int db = 0; db < 2 * C; db++) acc[db] *= beta;
            ev = eb;
        }
        const int less = max(ev - eb, -60);
        const float off = (ref == -INFINITY ? 0.0f : 12.0f - ref) + (float)less;
        halfx8 ph[2][2], pl[2][2];
        float ps = 0.0f;
#pragma unroll
        for (int kh = 0; kh < 2; kh++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
                u32x4 hw, lw;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p0 = exp2_hw(fmaf(sc[kh][8 * hh + 2 * i], f, off));
                    const float p1 = exp2_hw(fmaf(sc[kh][8 * hh + 2 * i + 1], f, off));
                    ps += p0 + p1;
                    uint32_t hi, lo;
                    split2(p0, p1, hi, lo);
                    hw[i] = hi;
                    lw[i] = lo;
                }
                ph[kh][hh] = __builtin_bit_cast(halfx8, hw);
                pl[kh][hh] = __builtin_bit_cast(halfx8, lw);
            }
        l += ps * pow2(-less);
        const uint8_t *vb = vt[sl];
#pragma unroll
        for (int kh = 0; kh < 2; kh++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++)
#pragma unroll
                for (int db = 0; db < 2 * C; db++) {
                    const int r = 32 * db + r32;
                    const uint8_t *at = vb + r * 128 + swz(r, 4 * kh + 2 * hh + g) * 16;
                    const halfx8 hi = *reinterpret_cast<const halfx8 *>(at), lo = *reinterpret_cast<const halfx8 *>(at + C * 8192);
                    acc[db] = mfma16(hi, ph[kh][hh], acc[db]);
                    acc[db] = mfma16(hi, pl[kh][hh], acc[db]);
                    acc[db] = mfma16(lo, ph[kh][hh], acc[db]);
                }
        if (evo & 1) {  // values that are not finite, zeros in the tile: what sees one is no number
            const int left = limit - kb * KB;
            const uint64_t sees = left >= 64 ? ~uint64_t(0) : (left > 0 ? (uint64_t(1) << left) - 1 : 0);
            const uint64_t *odd = p.odd + (((size_t)first + kb) * p.kv_heads + hk) * HD;
#pragma unroll
            for (int db = 0; db < 2 * C; db++)
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (odd[32 * db + 8 * (v >> 2) + 4 * g + (v & 3)] & sees) acc[db][v] = NAN;
        }
    };
    for (int kb = kb0; kb < kb1; kb++) step(kb);
    l = half_sum(l);  // lanes l and l ^ 32 have the same queries' sums over different keys
    if (!live) return;
    const float inv = l > 0.0f ? 1.0f / l : l, unit = pow2(-min(ev, 149));  // 0 and NaN stay
    const size_t row = (size_t)(qa + qi) * p.heads + h;
    float *dst = p.splits == 1 ? p.out + row * p.hd : p.part_o + ((size_t)split * p.nq * p.heads + row) * p.hd;
#pragma unroll
    for (int db = 0; db < 2 * C; db++)
#pragma unroll
        for (int v4 = 0; v4 < 4; v4++) {
            const int dim = 32 * db + 8 * v4 + 4 * g;
            if (dim < p.hd) {
                floatx4 o;
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = acc[db][4 * v4 + e] * inv * unit;
                *reinterpret_cast<floatx4u *>(dst + dim) = o;
            }
        }
    if (p.splits > 1 && g == 0) p.part_ml[(size_t)split * p.nq * p.heads + row] = make_float2(ref, l);
}

// grid (queries x heads / 4); 256 threads: a wavefront joins the key ranges' states of one query and head.
constexpr int MOST_SPLITS = 32;
__global__ __launch_bounds__(256) void k_packed_join(Packed p) {
    const int lane = threadIdx.x & 63, items = p.nq * p.heads, i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= items) return;
    if (i / p.heads >= p.qo[p.tables]) return;  // of no table
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < p.splits) ml = p.part_ml[(size_t)lane * items + i];
    const float top = wave_max(ml.y > 0.0f ? ml.x : -INFINITY);
    const float f = ml.y > 0.0f ? ml.y * exp2_hw(ml.x - top) : ml.y;
    const float sum = wave_sum(f);
    float o[2] = {0.0f, 0.0f};
    for (int s = 0; s < p.splits; s++) {
        const float fs = __shfl(f, s), ls = __shfl(ml.y, s);
        if (ls == 0.0f) continue;
        const float *src = p.part_o + ((size_t)s * items + i) * p.hd;
        if (lane < p.hd) o[0] += fs * src[lane];
        if (64 + lane < p.hd) o[1] += fs * src[64 + lane];
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum;
    if (lane < p.hd) p.out[(size_t)i * p.hd + lane] = o[0] * inv;
    if (64 + lane < p.hd) p.out[(size_t)i * p.hd + 64 + lane] = o[1] * inv;
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// Wavefronts a workgroup, key ranges, workgroups and the working memory's parts.
struct Plan {
    int waves, splits, blocks, c;
    int64_t grid;
    size_t tiles, shifts, odd, first, part_o, part_ml;
    size_t bytes() const { return tiles + shifts + odd + first + part_o + part_ml; }
};

Plan plan(const PackedShape &a) {
    Plan r;
    r.c = a.hd <= 64 ? 1 : 2;
    r.waves = r.c == 2 ? 8 : 4;
    const int qt = 32 * r.waves;
    const int64_t tiles = a.nq / qt + (int64_t)std::min(a.tables, a.nq);
    const int64_t blocks = a.nkv / KB + (int64_t)std::min(a.tables, a.nkv);
    r.blocks = (int)blocks;
    // few query tiles: several key ranges each, so that every compute unit has a workgroup
    const int64_t each = std::max<int64_t>(1, blocks / std::max<int64_t>(1, std::min(a.tables, a.nkv)));
    r.splits = (int)std::max<int64_t>(1, std::min<int64_t>({MOST_SPLITS, 256 / std::max<int64_t>(1, tiles * a.heads), each / 2}));
    r.grid = tiles * a.heads * r.splits;
    const size_t halves = (size_t)blocks * a.kv_heads;
    r.tiles = up256(halves * r.c * 32768);
    r.shifts = up256(halves * 2 * sizeof(int));
    r.odd = up256(halves * 64 * r.c * sizeof(uint64_t));
    r.first = up256((size_t)a.tables * sizeof(uint32_t));
    const size_t items = r.splits > 1 ? (size_t)r.splits * a.nq * a.heads : 0;
    r.part_o = up256(items * a.hd * sizeof(float));
    r.part_ml = up256(items * sizeof(float2));
    return r;
}

template <int C, int WAVES>
void launch(hipStream_t s, const Packed &p, const Plan &r) {
    if (r.blocks > 0) {
        hipLaunchKernelGGL(k_packed_tiles<C>, dim3(r.blocks, p.kv_heads, 2), dim3(256), 0, s, p);
        TAH_LAUNCHED();
    }
    hipLaunchKernelGGL((k_packed<C, WAVES>), dim3((unsigned)r.grid), dim3(64 * WAVES), 0, s, p);
    TAH_LAUNCHED();
    if (r.splits > 1) {
        hipLaunchKernelGGL(k_packed_join, dim3(((unsigned)p.nq * p.heads + 3) / 4), dim3(256), 0, s, p);
        TAH_LAUNCHED();
    }
}

}  // namespace

size_t packed_work_bytes(const PackedShape &a) {
    const Plan r = plan(a);
    if (r.grid > 0x7FFFFFFF || r.blocks > 0x7FFFFF) throw ArgError{"attend_packed: more rows than a call takes: fewer tables a call"};
    return r.bytes();
}

void packed_attention(hipStream_t s, const PackedShape &a, const float *q, const float *k, const float *v, const int32_t *q_offsets,
                      const int32_t *kv_offsets, bool causal, size_t q_ld, size_t kv_ld, float *out, void *work) {
    const Plan r = plan(a);
    uint8_t *at = static_cast<uint8_t *>(work);
    auto carve = [&](size_t bytes) {
        uint8_t *here = at;
        at += bytes;
        return here;
    };
    Packed p{q, k, v, q_offsets, kv_offsets, a.tables, a.nq, a.nkv, a.heads, a.kv_heads, a.hd, causal ? 1 : 0, q_ld, kv_ld, out};
    p.blocks = r.blocks;
    p.tiles = carve(r.tiles);
    p.shifts = reinterpret_cast<int *>(carve(r.shifts));
    p.odd = reinterpret_cast<uint64_t *>(carve(r.odd));
    p.first = reinterpret_cast<uint32_t *>(carve(r.first));
    p.splits = r.splits;
    p.part_o = reinterpret_cast<float *>(carve(r.part_o));
    p.part_ml = reinterpret_cast<float2 *>(carve(r.part_ml));
    if (r.c == 2)
        launch<2, 8>(s, p, r);
    else
        launch<1, 4>(s, p, r);
}

}  // namespace tah

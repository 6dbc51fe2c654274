// The classification head's reading of a row of class scores as a distribution at a softmax temperature, the counterpart of
// the quantile head's (quantiles.hip): its entropy, the log probabilities of given classes and the most probable classes.
//
// With m the row's largest score, u_i = (x_i - m) / T and S = sum exp(u_i):
//     log p_i = u_i - log S,    H = log S - sum exp(u_i) u_i / S.
// S is carried without the maximum's own 1 (s = S - 1, log S = log1p(s)), so that a confident row's log probabilities and
// entropy keep their relative precision; every term of s and of t = sum exp(u_i) (-u_i) is positive, so neither cancels.
// (m, s, t) of two parts join as the online softmax's do: with m1 >= m2 and g = (m1 - m2) / T,
//     s = s1 + e^-g (s2 + 1),    t = t1 + e^-g (t2 + g (s2 + 1)).
// Classes in order: larger scores first, the lower id among equals (-0 and 0 are equal), NaN after every number.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "device_math.hpp"

namespace tah {

constexpr float LN2 = 0.69314718055994530942f;

struct ClassDist {
    float m, s, t;
    bool bad;  // a NaN among the scores
};

// e^x for x <= 0 on the hardware's exp2 (1 ulp; x log2 e rounded: 2^-24 of it in the exponent)
__device__ __forceinline__ float exp_below(float x) { return exp2_hw(x * LOG2E); }

// (x - m) / T as (part x - part m) inv: at temperatures over 1 the halves' difference, which is finite for all finite scores
// (elsewhere a difference past float's largest has a quotient past it too). Scaling by 2 is exact: no result changes.
struct ClassScale {
    float part, inv;
    explicit ClassScale(float temperature) : part(temperature > 1.0f ? 0.5f : 1.0f), inv(1.0f / temperature / part) {}
    __device__ __forceinline__ float below(float x, float m) const { return fmaf(part, x, -(part * m)) * inv; }
    // a row's scores, where that is the kernel's time: f(part, inv), in halves only where m is large enough for them to matter
    // (below 2^100, float's least less m rounds to float's least; in halves always 64 x 100,000 18.8 -> 19.2 us; up to 256
    // classes the choice itself takes longer, 200,000 x 7 5.76 -> 5.83)
    template <class F>
    __device__ __forceinline__ void over(float m, F &&f) const {
        if (m < 0x1p100f) f(1.0f, part * inv);
        else f(part, inv);
    }
};

__device__ __forceinline__ ClassDist join(ClassDist a, ClassDist b, ClassScale by) {
    const bool swap = b.m > a.m;
    const float m = swap ? b.m : a.m, m2 = swap ? a.m : b.m;
    const float s1 = swap ? b.s : a.s, t1 = swap ? b.t : a.t, s2 = (swap ? a.s : b.s) + 1.0f, t2 = swap ? a.t : b.t;
    const float g = by.below(m, m2), f = exp_below(-g);
    // nothing but -inf in the lesser part, or too far below to count (g times 0 would be NaN where g is infinite)
    const bool none = m2 == -INFINITY || f == 0.0f;
    return {m, none ? s1 : fmaf(f, s2, s1), none ? t1 : fmaf(f, fmaf(g, s2, t2), t1), a.bad || b.bad};
}

__device__ __forceinline__ ClassDist join_lane(ClassDist a, int mask, ClassScale by) {
    const ClassDist b{__shfl_xor(a.m, mask), __shfl_xor(a.s, mask), __shfl_xor(a.t, mask), (bool)__shfl_xor((int)a.bad, mask)};
    return join(a, b, by);
}

// a score as a number that orders as the scores do: a NaN 1, and 0 is left for none
__device__ __forceinline__ uint32_t score_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return x != x ? 1u : u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t k) {
    return k == 1u ? NAN : __uint_as_float((k >> 31) ? (k ^ 0x80000000u) : ~k);
}
// with its class: a number that orders as the classes do
__device__ __forceinline__ uint64_t class_key(uint32_t k, int id) { return (uint64_t)k << 32 | (0xFFFFFFFFu - (uint32_t)id); }
__device__ __forceinline__ int class_of(uint64_t key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

struct ClassOut {
    const int32_t *given;  // [rows][n_given]
    int n_given, top;
    float *stats;   // [rows][1 + n_given + top]
    int32_t *ids;   // [rows][top]
    ClassOut from(size_t row) const {
        return {given + row * n_given, n_given, top, stats + row * (1 + n_given + top), ids + row * top};
    }
};

// What a row's distribution says: its entropy, and of one score.
struct ClassLogs {
    float entropy, from, logs;  // log p = (x - from) / T - logs
    __device__ __forceinline__ ClassLogs(const ClassDist &c) : from(c.m), logs(log1pf(c.s)) {
        entropy = logs + c.t / (1.0f + c.s);
        if (c.m == -INFINITY) {
            // every class ruled out: -inf - 0
            entropy = from = logs = 0.0f;
        }
        if (c.bad || !(c.m < INFINITY)) entropy = logs = NAN;
    }
    __device__ __forceinline__ float log_p(float x, ClassScale by) const { return by.below(x, from) - logs; }
};

// ---- up to 256 classes: one to 32 lanes a row ----------------------------------------------------------------------------
// v combined over the L lanes of a row (neighbours, L a power of two up to 32).
template <int L, class T, class F>
__device__ __forceinline__ T row_lanes(T v, F &&f) {
    static_assert(sizeof(T) == 4, "one register");
    auto there = [](T x, auto ctrl) {
        return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    if (L > 1) v = f(v, there(v, std::integral_constant<int, 0xb1>()));   // lanes 1 apart
    if (L > 2) v = f(v, there(v, std::integral_constant<int, 0x4e>()));   // 2 apart
    if (L > 4) v = f(v, there(v, std::integral_constant<int, 0x141>()));  // mirrored in eights: of the other four
    if (L > 8) v = f(v, there(v, std::integral_constant<int, 0x140>()));  // mirrored in sixteens: of the other eight
    if (L > 16) {
        const auto both = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v),
                                                           false, false);
        const unsigned a = both[0], b = both[1];  // a bit cast of a vector's element takes its first
        v = f(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
    }
    return v;
}

// grid ceil(rows / (64 / L)); 64 threads. Each of a row's L lanes keeps N / L of its N >= n scores in registers, read where
// they lie: a wavefront's loads meet the same few lines again and again, in L1 (turned in LDS first, whole lines at a time:
// 200,000 x 7 6.9 us for 5.8, 100,000 x 20 10.9 for 8.9). A wavefront or a workgroup a row spent most of its instructions on
// reductions (200,000 x 7: 664 us a workgroup a row). The most probable classes by one scan of the keys each. 200,000 x 7 with
// three best takes 460 instructions a wavefront of 64 rows, 2.7 us of issue; its wavefronts wait for memory 56% of their time.
// 100,000 x 50 with five best, 14.6 us, 1.4 TB/s, is bound by its instructions (724 for eight rows).
template <int N, int L>
__global__ __launch_bounds__(64) void k_class_stats_rows(int rows, int n, size_t ld, const float *__restrict__ x,
                                                         ClassScale by, ClassOut o) {
    constexpr int R = 64 / L, E = N / L;
    const int part = threadIdx.x % L;
    const size_t row = (size_t)blockIdx.x * R + threadIdx.x / L;
    if (row >= (size_t)rows) return;
    const float *mine = x + row * ld;
    // entry i of a lane: class L i + part
    float v[E];
    uint32_t k[E];
    ClassDist c{-INFINITY, 0.0f, 0.0f, false};
    int bad = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int at = L * i + part;
        v[i] = -INFINITY;
        if (L * (i + 1) <= n || at < n) v[i] = mine[at];  // the first is the same for all lanes
    }
#pragma unroll
    for (int i = 0; i < E; i++) {
        k[i] = L * i + part < n ? score_key(v[i]) : 0u;
        bad |= v[i] != v[i];
        c.m = fmaxf(c.m, v[i]);
    }
    c.m = row_lanes<L>(c.m, [](float a, float b) { return fmaxf(a, b); });
    c.bad = row_lanes<L>(bad, [](int a, int b) { return a | b; }) != 0;
    // in units of log 2; the largest scores' terms are exactly 1 and are counted apart. From 2^-200 down a term is 0
    const float inv2 = by.inv * LOG2E, pm = by.part * c.m;
    int tops = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const float u = fmaxf(fmaf(by.part, v[i], -pm) * inv2, -200.0f);
        const bool is_top = v[i] == c.m;
        const float w = is_top ? 0.0f : exp2_hw(u);
        tops += is_top;
        c.s += w;
        c.t = fmaf(-w, u, c.t);
    }
    const auto add = [](auto a, auto b) { return a + b; };
    c.s = row_lanes<L>(c.s, add) + (float)(row_lanes<L>(tops, add) - 1);
    c.t = row_lanes<L>(c.t, add) * LN2;
    float *st = o.stats + row * (1 + o.n_given + o.top);
    const ClassLogs says(c);
    if (part == 0) st[0] = says.entropy;
    for (int i = part; i < o.n_given; i += L) {
        const int id = o.given[row * o.n_given + i];
        st[1 + i] = id >= 0 && id < n ? says.log_p(mine[id], by) : NAN;
    }
    for (int r = 0; r < o.top; r++) {
        uint32_t best = 0;
        int id = 0;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const bool more = k[i] > best;
            best = more ? k[i] : best;
            id = more ? L * i + part : id;
        }
        const uint32_t most = row_lanes<L>(best, [](uint32_t a, uint32_t b) { return max(a, b); });
        id = row_lanes<L>(best == most ? id : N, [](int a, int b) { return min(a, b); });
#pragma unroll
        for (int i = 0; i < E; i++) k[i] = L * i + part == id ? 0u : k[i];
        if (r % L == part) {
            st[1 + o.n_given + r] = says.log_p(score_of(most), by);
            o.ids[row * o.top + r] = id;
        }
    }
}

// ---- a wavefront's scores, E a lane -----------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    // as floats' bit patterns would not do: an unsigned maximum in pairs of lanes 1, 2, 4, 8, 16 and 32 apart
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, false));
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)a[0], (uint32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((uint32_t)b[0], (uint32_t)b[1]);
}

// the largest of the lanes' keys
__device__ __forceinline__ uint64_t wave_best(uint64_t key) {
    const uint32_t hi = wave_max_u32((uint32_t)(key >> 32));
    const uint32_t lo = wave_max_u32((uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
    return (uint64_t)hi << 32 | lo;
}

// The distribution of a wavefront's scores v (E a lane, -inf past the last), in every lane.
template <int E>
__device__ __forceinline__ ClassDist wave_dist(const float (&v)[E], ClassScale by) {
    float own = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int r = 0; r < E; r++) {
        own = fmaxf(own, v[r]);
        bad = bad || v[r] != v[r];
    }
    ClassDist c{wave_max(own), 0.0f, 0.0f, __any(bad) != 0};
    if (c.m == -INFINITY) return c;
    // in units of log 2; the terms of the largest score are exactly 1 and are counted apart. From 2^-200 down a term is 0
    int tops = 0;
    float s = 0.0f, t = 0.0f;
    by.over(c.m, [&](float part, float inv) {
        const float inv2 = inv * LOG2E, pm = part * c.m;
#pragma unroll
        for (int r = 0; r < E; r++) {
            const float u = fmaxf(fmaf(part, v[r], -pm) * inv2, -200.0f), e = exp2_hw(u);
            const bool is_top = v[r] == c.m;
            tops += __popcll(__ballot(is_top));
            const float w = is_top ? 0.0f : e;
            s += w;
            t = fmaf(-w, u, t);
        }
    });
    c.s = wave_sum(s) + (float)(tops - 1);
    c.t = wave_sum(t) * LN2;
    return c;
}

// The top largest scores of a wavefront as keys in order: lane r's result is the r-th (top at most 64). live: how many
// entries of a lane are scores. Class ids: id(r) of entry r. Taken one by one: each lane keeps its own largest left, and
// the one whose key is taken looks for its next.
template <int E, class Id>
__device__ __forceinline__ uint64_t wave_top_each(const float (&v)[E], int live, int top, int lane, Id &&id) {
    uint32_t k[E];
#pragma unroll
    for (int r = 0; r < E; r++) k[r] = r < live ? score_key(v[r]) : 0u;
    uint64_t mine = 0, got = 0;
    auto next = [&] {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int r = 0; r < E; r++) {
            const bool more = k[r] > best;
            best = more ? k[r] : best;
            at = more ? r : at;
        }
#pragma unroll
        for (int r = 0; r < E; r++) k[r] = r == at ? 0u : k[r];
        mine = best ? class_key(best, id(at)) : 0;
    };
    next();
    for (int r = 0; r < top; r++) {
        const uint64_t best = wave_best(mine);
        if (lane == r) got = best;
        if (mine == best && best) next();
    }
    return got;
}

// The largest key that at least top of the lanes' keys (two a lane) reach, or a little less: halved ten times between the
// least and the largest of them (hi). 14 times are a finer bound and take longer (3,000 x 1,001 with ten best 7.9 us for 7.6,
// 1,000 x 5,000 with five 14.2 for 13.5), eight let too many past where the keys span zero (8.7 and 13.1).
__device__ __forceinline__ uint32_t bound_of(uint32_t key, uint32_t other, uint32_t hi, int top) {
    uint32_t lo = ~wave_max_u32(~min(key, other));
    for (int i = 0; i < 10 && lo < hi; i++) {
        const uint32_t mid = hi - (hi - lo) / 2;
        if (__popcll(__ballot(key >= mid)) + __popcll(__ballot(other >= mid)) >= top) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// The same sooner. A bound that top lanes' own largest scores reach, and few more (bound_of): top scores reach it, so nothing
// below it is among the top. What reaches it goes into a list in LDS, whose entries are placed by counting the larger ones.
// Where that does not serve (too many equal scores, or rising ones in few lanes; a bound of -inf; NaN among the top) the keys
// are taken one by one (3,000 x 1,001 with ten best: 15.2 us for all rows so, 7.6 by the bound).
constexpr int LIST = 256;
template <int E, class Id>
__device__ __forceinline__ uint64_t wave_top(const float (&v)[E], const ClassDist &c, int live, int top, int lane,
                                             uint64_t *list, Id &&id) {
    float own = -INFINITY;
#pragma unroll
    for (int r = 0; r < E; r++) own = fmaxf(own, v[r]);
    const uint32_t lo = bound_of(score_key(own), 0xFFFFFFFFu, score_key(c.m), top + 64);  // one a lane: 64 that always do
    if (lo > score_key(-INFINITY)) {
        const float bound = score_of(lo);
        int n = 0;
#pragma unroll
        for (int r = 0; r < E; r++) {
            const bool in = v[r] >= bound;
            const uint64_t who = __ballot(in);
            if (who) {
                const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
                if (in && at < LIST) list[at] = class_key(score_key(v[r]), id(r));
                n += __popcll(who);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (n >= top && n <= LIST) {
            uint64_t mine[LIST / 64];
            int place[LIST / 64];
#pragma unroll
            for (int u = 0; u < LIST / 64; u++) {
                if (64 * u >= n) break;
                mine[u] = 64 * u + lane < n ? list[64 * u + lane] : 0;
                place[u] = 0;
#pragma unroll 4
                for (int j = 0; j < n; j++) place[u] += list[j] > mine[u];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();  // every entry is read before the first is written over
#pragma unroll
            for (int u = 0; u < LIST / 64; u++) {
                if (64 * u >= n) break;
                if (mine[u] && place[u] < top) list[place[u]] = mine[u];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            return lane < top ? list[lane] : 0;
        }
    }
    return wave_top_each(v, live, top, lane, id);
}

// ---- up to 1,024 classes, many of them wanted: a wavefront a row ------------------------------------------------------------------------------
// grid ceil(rows / 4); 256 threads. Entry r of a lane is class 64 r + lane: the row is read once, in whole lines, and kept.
template <int E>
__global__ __launch_bounds__(256) void k_class_stats_wave(int rows, int n, size_t ld, const float *__restrict__ x,
                                                          ClassScale by, ClassOut o) {
    __shared__ uint64_t list[4][LIST];
    const int lane = threadIdx.x & 63;
    const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (size_t)rows) return;
    const float *src = x + row * ld;
    float v[E];
#pragma unroll
    for (int r = 0; r < E; r++) v[r] = 64 * r + lane < n ? src[64 * r + lane] : -INFINITY;
    const ClassDist c = wave_dist(v, by);
    float *st = o.stats + row * (1 + o.n_given + o.top);
    const ClassLogs says(c);
    if (lane == 0) st[0] = says.entropy;
    if (lane < o.n_given) {
        const int id = o.given[row * o.n_given + lane];
        st[1 + lane] = id >= 0 && id < n ? says.log_p(src[id], by) : NAN;
    }
    if (o.top == 0) return;
    const uint64_t key = wave_top(v, c, (n - lane + 63) / 64, o.top, lane, list[threadIdx.x >> 6],
                                  [&](int r) { return 64 * r + lane; });
    if (lane < o.top) {
        st[1 + o.n_given + lane] = says.log_p(score_of((uint32_t)(key >> 32)), by);
        o.ids[row * o.top + lane] = class_of(key);
    }
}

// ---- more classes: a workgroup a segment of a row ------------------------------------------------------------------------
// A segment's state: its distribution, then its top keys in order.
struct SegState {
    ClassDist c;
};
constexpr int SEG_T = 512, SEG = 32 * SEG_T, SEG_LIST = 1024;

__host__ __device__ inline size_t seg_bytes(int top) { return sizeof(SegState) + 8 * (size_t)top; }

__device__ __forceinline__ void write_row(const ClassLogs &says, const ClassOut &o, size_t row, int n, const float *src,
                                          ClassScale by, int tid) {
    float *st = o.stats + row * (1 + o.n_given + o.top);
    if (tid == 0) st[0] = says.entropy;
    if (tid < o.n_given) {
        const int id = o.given[row * o.n_given + tid];
        st[1 + tid] = id >= 0 && id < n ? says.log_p(src[id], by) : NAN;
    }
}

// The place of key among `lists` lists of `each` falling keys (in LDS, 0 past a list's end): how many are larger.
__device__ __forceinline__ int place_of(uint64_t key, const uint64_t *keys, int lists, int each) {
    int place = 0;
    for (int l = 0; l < lists; l++) {
        int lo = 0, hi = each;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (keys[l * each + mid] > key) lo = mid + 1;
            else hi = mid;
        }
        place += lo;
    }
    return place;
}

// grid (segments, rows); 512 threads: each keeps up to E scores of its segment (len, a multiple of 4) in registers, so that
// the row is read once. The wavefronts' distributions are joined in LDS, the segments of a row by k_class_stats_join (a row of
// one segment is written here). The most probable classes as wave_top has them, but of the workgroup: the bound from the
// largest scores of its 128 groups of four lanes, one list (a list a wavefront, then joined: 64 x 100,000 with 20 best
// 22 us for 18). Loads and arithmetic hardly overlap, since all workgroups start together.
template <int E>
__global__ __launch_bounds__(SEG_T) void k_class_stats_seg(int n, int len, size_t ld, const float *__restrict__ x,
                                                           ClassScale by, uint8_t *__restrict__ state, ClassOut o) {
    constexpr int W = SEG_T / 64;
    __shared__ ClassDist part[W];
    __shared__ float group[SEG_T / 4];
    __shared__ uint64_t list[SEG_LIST];
    __shared__ int listed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, seg = blockIdx.x, segs = gridDim.x;
    const size_t row = blockIdx.y;
    const float *src = x + row * ld;
    const int base = seg * len, end = min(n, base + len);
    if (tid == 0) listed = 0;
    float v[E];
    // entry 4 r + j of a thread: class base + 4 (512 r + tid) + j
    auto id = [&](int e) { return base + 4 * (SEG_T * (e >> 2) + tid) + (e & 3); };
    const bool fours = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
#pragma unroll
    for (int r = 0; r < E / 4; r++) {
        const int i = id(4 * r);
        if (fours && i + 4 <= end) {
            const float4 x4 = *reinterpret_cast<const float4 *>(src + i);
            v[4 * r] = x4.x;
            v[4 * r + 1] = x4.y;
            v[4 * r + 2] = x4.z;
            v[4 * r + 3] = x4.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[4 * r + j] = i + j < end ? src[i + j] : -INFINITY;
        }
    }
    if (o.top > 0) {
        float own = -INFINITY;
#pragma unroll
        for (int r = 0; r < E; r++) own = fmaxf(own, v[r]);
        own = fmaxf(own, dpp<0xb1>(own));   // lanes 1 apart
        own = fmaxf(own, dpp<0x4e>(own));   // 2 apart
        if ((lane & 3) == 0) group[tid >> 2] = own;
    }
    const ClassDist w = wave_dist(v, by);
    if (lane == 0) part[wave] = w;
    __syncthreads();
    ClassDist c = part[0];
#pragma unroll
    for (int i = 1; i < W; i++) c = join(c, part[i], by);
    uint8_t *mine = state + (row * segs + seg) * seg_bytes(o.top);
    const ClassLogs says(c);
    if (segs == 1) write_row(says, o, row, n, src, by, tid);
    else if (tid == 0) reinterpret_cast<SegState *>(mine)->c = c;
    if (o.top == 0) return;
    auto put = [&](uint64_t key, int place) {
        if (segs == 1) {
            o.stats[row * (1 + o.n_given + o.top) + 1 + o.n_given + place] = says.log_p(score_of((uint32_t)(key >> 32)), by);
            o.ids[row * o.top + place] = class_of(key);
        } else {
            reinterpret_cast<uint64_t *>(mine + sizeof(SegState))[place] = key;
        }
    };
    static_assert(SEG_T / 4 == 128, "two groups a lane");
    const uint32_t lo = bound_of(score_key(group[lane]), score_key(group[64 + lane]), score_key(c.m), o.top);
    const bool bounded = lo > score_key(-INFINITY);
    if (bounded) {
        const float bound = score_of(lo);
#pragma unroll
        for (int r = 0; r < E; r++) {
            const bool in = v[r] >= bound;
            const uint64_t who = __ballot(in);
            if (who) {
                int from = 0;
                if (lane == 0) from = atomicAdd(&listed, __popcll(who));
                from = __builtin_amdgcn_readfirstlane(from);
                const int at = from + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
                if (in && at < SEG_LIST) list[at] = class_key(score_key(v[r]), id(r));
            }
        }
    }
    __syncthreads();
    const int got = listed;
    if (bounded && got >= o.top && got <= SEG_LIST) {
        for (int i = tid; i < got; i += SEG_T) {
            const uint64_t key = list[i];
            int place = 0;
#pragma unroll 8
            for (int j = 0; j < got; j++) place += list[j] > key;
            if (place < o.top) put(key, place);
        }
        return;
    }
    __syncthreads();  // the list is free
    // entries of this thread that are scores: those of its whole fours, then what its last one has
    const int left = max(0, end - base - 4 * tid), live = left / (4 * SEG_T) * 4 + min(4, left % (4 * SEG_T));
    static_assert(W * 64 <= SEG_LIST, "every wavefront's keys fit the list");
    const uint64_t key = wave_top_each(v, live, o.top, lane, id);
    if (lane < o.top) list[wave * o.top + lane] = key;
    __syncthreads();
    if (tid < W * o.top) {
        const uint64_t k = list[tid];
        const int place = k ? place_of(k, list, W, o.top) : o.top;
        if (place < o.top) put(k, place);
    }
}

// grid rows; 512 threads: the segments of a row joined; segs (at most 64) lists of top falling keys, in LDS, placed by
// counting the larger ones: up to 192 all of them (64 x 30,000 with 20 best 14.6 us by a bound, 13.1 so), else those that reach a
// bound: with j = ceil(top / segs), the ceil(top / j)-th largest of the lists' j-th entries, which top keys reach (all 960 keys
// of one row took 25 us of LDS reads).
constexpr int JOIN_LIST = 512, JOIN_ALL = 192;
__global__ __launch_bounds__(512) void k_class_stats_join(int n, size_t ld, const float *__restrict__ x, ClassScale by,
                                                          int segs, const uint8_t *__restrict__ state, ClassOut o) {
    extern __shared__ uint64_t all[];
    __shared__ uint64_t list[JOIN_LIST];
    __shared__ int listed;
    const int tid = threadIdx.x, lane = tid & 63, total = segs * o.top;
    const size_t row = blockIdx.x;
    const uint8_t *rows_state = state + row * segs * seg_bytes(o.top);
    if (tid == 0) listed = 0;
    for (int i = tid; i < total; i += 512) {
        const int s = i / o.top;
        all[i] = reinterpret_cast<const uint64_t *>(rows_state + s * seg_bytes(o.top) + sizeof(SegState))[i - s * o.top];
    }
    ClassDist c{-INFINITY, 0.0f, 0.0f, false};
    if (lane < segs) c = reinterpret_cast<const SegState *>(rows_state + lane * seg_bytes(o.top))->c;
    for (int mask = 1; mask < 64; mask <<= 1) c = join_lane(c, mask, by);
    const ClassLogs says(c);
    write_row(says, o, row, n, x + row * ld, by, tid);
    if (o.top == 0) return;
    __syncthreads();
    const bool all_of_them = total <= JOIN_ALL;
    if (!all_of_them) {
        const int j = (o.top + segs - 1) / segs, need = (o.top + j - 1) / j;
        // lanes past the lists count as reaching any bound
        const uint32_t entry = lane < segs ? (uint32_t)(all[lane * o.top + j - 1] >> 32) : 0xFFFFFFFFu;
        const uint32_t bound = bound_of(entry, 0xFFFFFFFFu, wave_max_u32(lane < segs ? entry : 0u), need + 64 + 64 - segs);
        for (int i = tid; i < total; i += 512) {
            const uint64_t key = all[i];
            if ((uint32_t)(key >> 32) >= bound) {
                const int at = atomicAdd(&listed, 1);
                if (at < JOIN_LIST) list[at] = key;
            }
        }
        __syncthreads();
    }
    const int got = all_of_them ? total : listed;
    const bool few = all_of_them || got <= JOIN_LIST;  // else equal scores without end
    const uint64_t *keys = few && !all_of_them ? list : all;
    for (int i = tid; i < (few ? got : total); i += 512) {
        const uint64_t key = keys[i];
        int place = 0;
        if (few) {
#pragma unroll 8
            for (int u = 0; u < got; u++) place += keys[u] > key;
        } else {
            place = place_of(key, all, segs, o.top);
        }
        if (place < o.top) {
            o.stats[row * (1 + o.n_given + o.top) + 1 + o.n_given + place] = says.log_p(score_of((uint32_t)(key >> 32)), by);
            o.ids[row * o.top + place] = class_of(key);
        }
    }
}

// Rows of more than 1,024 classes: how they are cut. As few segments as registers hold them in: more of them, to fill whole
// rounds of the compute units, gave the join more to do than they saved (1 x 100,000 with 20 best in 7 and in 48 segments 14.0
// and 14.8 us, 64 x 16,384 in 1 and in 4 8.9 and 14.9, 64 x 100,000 in 7 and in 8 alike). Rows at a time whose segments'
// states fit 32 MB (and a launch's grid). Every segment has the top classes that it hands over: the last one has n / segs
// less 4 (segs - 1) of them or more.
static_assert(SEG / 2 - 4 * ((1 << 20) / SEG - 1) >= 64, "a last segment of 2^20 classes or fewer has 64");
struct ClassCut {
    int segs, len, rows;
};
static ClassCut cut(int n, int top) {
    ClassCut c;
    c.segs = (n + SEG - 1) / SEG;
    c.len = ((n + c.segs - 1) / c.segs + 3) / 4 * 4;
    c.segs = (n + c.len - 1) / c.len;
    c.rows = (int)std::max<size_t>(1, std::min<size_t>(65535, (size_t(32) << 20) / (c.segs * seg_bytes(top))));
    return c;
}

size_t class_stats_work_bytes(int rows, int n, int top) {
    if (n <= 1024) return 0;
    const ClassCut c = cut(n, top);
    return c.segs == 1 ? 0 : (size_t)std::min(rows, c.rows) * c.segs * seg_bytes(top);
}

template <int N, int L>
static void launch_rows(hipStream_t s, int rows, int n, size_t ld, const float *x, ClassScale by, const ClassOut &o) {
    constexpr int R = 64 / L, MOST = 1 << 26;  // rows a launch: a grid holds fewer than 2^32 threads
    for (int r0 = 0; r0 < rows; r0 += std::min(MOST, rows - r0)) {
        const int here = std::min(MOST, rows - r0);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_class_stats_rows<N, L>), dim3((here + R - 1) / R), dim3(64), 0, s, here, n, ld,
                           x + r0 * ld, by, o.from(r0));
    }
}
template <int E>
static void launch_wave(hipStream_t s, int rows, int n, size_t ld, const float *x, ClassScale by, const ClassOut &o) {
    constexpr int MOST = 1 << 24;  // rows a launch: a grid holds fewer than 2^32 threads
    for (int r0 = 0; r0 < rows; r0 += std::min(MOST, rows - r0)) {
        const int here = std::min(MOST, rows - r0);
        hipLaunchKernelGGL(k_class_stats_wave<E>, dim3((here + 3) / 4), dim3(256), 0, s, here, n, ld, x + r0 * ld, by,
                           o.from(r0));
    }
}

// the fewest scores a thread that hold a segment (1,000 x 2,000 by 32 a thread 17.8 us, by 8 10.8;
// 1,000 x 5,000 by 32 18.7, by 16 14.1)
static void launch_seg(hipStream_t s, int segs, int rows, int n, int len, size_t ld, const float *x, ClassScale by,
                       uint8_t *state, const ClassOut &o) {
    const dim3 grid(segs, rows), block(SEG_T);
    if (len <= 8 * SEG_T) hipLaunchKernelGGL(k_class_stats_seg<8>, grid, block, 0, s, n, len, ld, x, by, state, o);
    else if (len <= 16 * SEG_T) hipLaunchKernelGGL(k_class_stats_seg<16>, grid, block, 0, s, n, len, ld, x, by, state, o);
    else hipLaunchKernelGGL(k_class_stats_seg<32>, grid, block, 0, s, n, len, ld, x, by, state, o);
}

// work: class_stats_work_bytes(rows, n, top) bytes.
void class_stats(hipStream_t s, int rows, int n, size_t ld, const float *x, float temperature, const int32_t *given,
                 int n_given, int top, float *stats, int32_t *ids, void *work) {
    if (rows <= 0) return;
    const ClassScale by(temperature);
    ClassOut o{given, n_given, top, stats, ids};
    // Eight scores a lane (sixteen: 1,000 x 50 4.0 -> 5.1 us, 100,000 x 50 14.6 -> 15.0; four: 200,000 x 7 5.8 -> 6.7, 100,000 x
    // 20 8.9 -> 11.3), up to 256 classes while few of them are wanted one by one (20,000 x 100, a wavefront a row against this:
    // five best 15.5 -> 7.7 us, 20 best 16.9 and 16.1; 20,000 x 200: 17.2 -> 12.9, 18.7 and 29.2; 200 x 100, 20 best 4.7 and
    // 7.2). Else a wavefront a row, the fewest entries a lane that hold it.
    if (n <= 8) launch_rows<8, 1>(s, rows, n, ld, x, by, o);
    else if (n <= 16) launch_rows<16, 2>(s, rows, n, ld, x, by, o);
    else if (n <= 32) launch_rows<32, 4>(s, rows, n, ld, x, by, o);
    else if (n <= 64) launch_rows<64, 8>(s, rows, n, ld, x, by, o);
    else if (n <= 128 && top <= 8) launch_rows<128, 16>(s, rows, n, ld, x, by, o);
    else if (n <= 256 && top <= 8) launch_rows<256, 32>(s, rows, n, ld, x, by, o);
    else if (n <= 128) launch_wave<2>(s, rows, n, ld, x, by, o);
    else if (n <= 256) launch_wave<4>(s, rows, n, ld, x, by, o);
    else if (n <= 512) launch_wave<8>(s, rows, n, ld, x, by, o);
    else if (n <= 1024) launch_wave<16>(s, rows, n, ld, x, by, o);
    else {
        const ClassCut c = cut(n, top);
        const int segs = c.segs;
        for (int r0 = 0; r0 < rows; r0 += c.rows) {
            const int here = std::min(c.rows, rows - r0);
            const float *xr = x + r0 * ld;
            const ClassOut at = o.from(r0);
            launch_seg(s, segs, here, n, c.len, ld, xr, by, static_cast<uint8_t *>(work), at);
            if (segs > 1)
                hipLaunchKernelGGL(k_class_stats_join, dim3(here), dim3(512), (size_t)segs * top * 8, s, n, ld, xr, by, segs,
                                   static_cast<const uint8_t *>(work), at);
        }
    }
    TAH_LAUNCHED();
}

}  // namespace tah

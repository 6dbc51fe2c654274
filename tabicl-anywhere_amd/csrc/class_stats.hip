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
#include <cmath>

#include "common.hpp"
#include "device_math.hpp"

namespace tah {

struct ClassDist {
    float m, s, t;
    bool bad;  // a NaN among the scores
};

__device__ __forceinline__ ClassDist join(ClassDist a, ClassDist b, float inv) {
    const bool swap = b.m > a.m;
    const float m = swap ? b.m : a.m, m2 = swap ? a.m : b.m;
    const float s1 = swap ? b.s : a.s, t1 = swap ? b.t : a.t, s2 = (swap ? a.s : b.s) + 1.0f, t2 = swap ? a.t : b.t;
    const float g = (m - m2) * inv, f = __expf(-g);
    // nothing but -inf in the lesser part, or too far below to count (g times 0 would be NaN where g is infinite)
    const bool none = m2 == -INFINITY || f == 0.0f;
    return {m, none ? s1 : fmaf(f, s2, s1), none ? t1 : fmaf(f, fmaf(g, s2, t2), t1), a.bad || b.bad};
}

__device__ __forceinline__ ClassDist join_lane(ClassDist a, int mask, float inv) {
    return join(a, {__shfl_xor(a.m, mask), __shfl_xor(a.s, mask), __shfl_xor(a.t, mask), (bool)__shfl_xor((int)a.bad, mask)}, inv);
}

// a score and its id as a number that orders as the classes do; never 0
__device__ __forceinline__ uint64_t class_key(float x, int id) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t k = x != x ? 0u : u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
    return (uint64_t)k << 32 | (0xFFFFFFFFu - (uint32_t)id);
}

struct ClassOut {
    const int32_t *given;  // [rows][n_given]
    int n_given, top;
    float *stats;   // [rows][1 + n_given + top]
    int32_t *ids;   // [rows][top]
};

// What a row's distribution says of one score.
__device__ __forceinline__ float log_p(const ClassDist &c, float x, float inv) {
    if (c.bad || !(c.m < INFINITY)) return NAN;
    if (c.m == -INFINITY) return -INFINITY;  // every class ruled out
    return (x - c.m) * inv - log1pf(c.s);
}
__device__ __forceinline__ float entropy(const ClassDist &c) {
    if (c.bad || !(c.m < INFINITY)) return NAN;
    return c.m == -INFINITY ? 0.0f : log1pf(c.s) + c.t / (1.0f + c.s);
}

// grid rows; 256 threads.
__global__ __launch_bounds__(256) void k_class_stats(int n, size_t ld, const float *__restrict__ x, float inv, ClassOut o) {
    __shared__ ClassDist part[4];
    __shared__ uint64_t best[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x;
    const float *src = x + row * ld;
    ClassDist c{-INFINITY, 0.0f, 0.0f, false};
    for (int i = tid; i < n; i += 256) c = join(c, {src[i], 0.0f, 0.0f, src[i] != src[i]}, inv);
    for (int mask = 1; mask < 64; mask <<= 1) c = join_lane(c, mask, inv);
    if (lane == 0) part[wave] = c;
    __syncthreads();
    c = join(join(part[0], part[1], inv), join(part[2], part[3], inv), inv);
    float *st = o.stats + row * (1 + o.n_given + o.top);
    if (tid == 0) st[0] = entropy(c);
    for (int i = tid; i < o.n_given; i += 256) {
        const int id = o.given[row * o.n_given + i];
        st[1 + i] = id >= 0 && id < n ? log_p(c, src[id], inv) : NAN;
    }
    uint64_t last = ~0ull;
    for (int r = 0; r < o.top; r++) {
        uint64_t k = 0;
        for (int i = tid; i < n; i += 256) {
            const uint64_t u = class_key(src[i], i);
            if (u < last && u > k) k = u;
        }
        for (int mask = 1; mask < 64; mask <<= 1) {
            const uint64_t u = __shfl_xor(k, mask);
            k = u > k ? u : k;
        }
        __syncthreads();
        if (lane == 0) best[wave] = k;
        __syncthreads();
        for (int w = 0; w < 4; w++) k = best[w] > k ? best[w] : k;
        last = k;
        if (tid == 0) {
            const int id = (int)(0xFFFFFFFFu - (uint32_t)k);
            st[1 + o.n_given + r] = log_p(c, src[id], inv);
            o.ids[row * o.top + r] = id;
        }
    }
}

void class_stats(hipStream_t s, int rows, int n, size_t ld, const float *x, float temperature, const int32_t *given,
                 int n_given, int top, float *stats, int32_t *ids) {
    if (rows <= 0) return;
    hipLaunchKernelGGL(k_class_stats, dim3(rows), dim3(256), 0, s, n, ld, x, 1.0f / temperature,
                       ClassOut{given, n_given, top, stats, ids});
    TAH_LAUNCHED();
}

}  // namespace tah

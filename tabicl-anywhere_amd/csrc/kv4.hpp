// The 4-bit stored form of keys and values (TAH_KV_I4, include/tah.h): per coordinate and group of 64 rows of a chunk a
// bfloat16 step s and offset z, per number a code c of -8 .. 7; value = z + s c rounded to eleven significant bits.
//
// Why so. A group's sixteen levels span its own range about its own middle: keys and values have a mean of their own per
// coordinate (the median coordinate's is 0.2 to 0.75 of its spread in the published classifier), which levels about zero
// would spend codes on (64 test rows of a fitted 900 x 12 table: probabilities move by 0.0012 on average and 0.010 at
// worst; by 0.0018 and 0.014 with levels about zero and groups of 64, by 0.0019 and 0.021 with groups of 32 at the same
// bits; in i8 by 0.0002 and 0.002). Groups are key blocks of the attention kernels, which then see one step and one offset
// a coordinate. And eleven bits are what an fp16 operand of the matrix cores holds: a value times its head's power of two
// goes in as one operand, exact, where an f32 or i16 value goes in as two halves; that rounding is 2^-12 of a value, far
// below half a step.
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"
#include "device_math.hpp"

namespace tah {

struct Step4 {
    float s, z;  // bfloat16 values
};

// v rounded to eleven significant bits, ties to even (infinities stay)
__device__ __forceinline__ float eleven_bits(float v) {
    const uint32_t u = __float_as_uint(v);
    return __uint_as_float((u + 0xFFFu + ((u >> 13) & 1u)) & 0xFFFFE000u);
}

// s c is exact in f32 (at most eleven bits)
__device__ __forceinline__ float value4(Step4 st, int code) { return eleven_bits(fmaf(st.s, (float)code, st.z)); }

// the step and offset of a group whose finite values lie from lo to hi (hi < lo: it has none)
__device__ __forceinline__ Step4 step_for4(float lo, float hi) {
#pragma clang fp contract(off)
    Step4 st{0.0f, 0.0f};
    if (!(lo <= hi)) return st;
    lo = fminf(fmaxf(lo, -0x1p126f), 0x1p126f);  // so that no difference overflows
    hi = fminf(fmaxf(hi, -0x1p126f), 0x1p126f);
    const float mid = lo * (7.0f / 15.0f) + hi * (8.0f / 15.0f) + 0.0f;  // a zero is +0, whichever zeros lo and hi are
    const uint32_t u = __float_as_uint(mid);
    st.z = __uint_as_float((u + 0x7FFFu + ((u >> 16) & 1u)) & 0xFFFF0000u);
    const float s = fmaxf((hi - st.z) * (1.0f / 7.0f), (st.z - lo) * 0.125f);
    st.s = s < 0x1p-100f ? 0.0f : __uint_as_float((__float_as_uint(s) + 0xFFFFu) & 0xFFFF0000u);
    return st;
}

// The code of a value: the nearest level of (v - z) / s, a tie to the even one. The quotient correctly rounded never meets a
// tie that the exact one does not: a tie is a product of twelve bits with s, and a float beside it is off by more than half
// the quotient's last place.
__device__ __forceinline__ int code4(Step4 st, float v) {
    if (!(st.s > 0.0f) || v != v) return 0;
    return (int)fminf(fmaxf(rintf(__fdiv_rn(v - st.z, st.s)), -8.0f), 7.0f);
}

// The same of four values, eight more than each in four bits, with one reciprocal: it is off by 2^-22 of the quotient at
// most, so that away from a tie the nearest level is the same; where a lane of the wavefront is near one (one in 2^15
// values), by the division.
__device__ __forceinline__ uint32_t codes4(Step4 st, const float (&v)[4]) {
    const float inv = st.s > 0.0f ? __builtin_amdgcn_rcpf(st.s) : 0.0f;
    float far = 0.0f;  // from the nearest level, a NaN passed over
    int code[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const float x = (v[t] - st.z) * inv, q = rintf(x);
        far = fmaxf(far, fabsf(x - q));
        // the instruction takes a NaN to 0 and clamps what does not fit, which the language leaves open
        asm("v_cvt_i32_f32 %0, %1" : "=v"(code[t]) : "v"(q));
        code[t] = min(max(code[t], -8), 7);
    }
    if (__any(far > 0.5f - 0x1p-16f)) {
#pragma unroll
        for (int t = 0; t < 4; t++) code[t] = code4(st, v[t]);
    }
    return (uint32_t)(code[0] + 16 * (code[1] + 16 * (code[2] + 16 * code[3])) + 0x8888);
}

__device__ __forceinline__ Step4 step_at4(const uint8_t *rec, int rc, int j, int g) {
    uint32_t sz;  // a record starts on an even byte
    __builtin_memcpy(&sz, rec + 4 * ((size_t)j * groups4(rc) + g), 4);
    return {__uint_as_float(sz << 16), __uint_as_float(sz & 0xFFFF0000u)};
}

// number (stacked coordinate j of 2d, row r) of a chunk's record
__device__ __forceinline__ float record_value4(const uint8_t *rec, int d, int rc, int j, int r) {
    const uint8_t b = rec[8 * (size_t)d * groups4(rc) + (size_t)j * ((rc + 1) / 2) + (r >> 1)];
    return value4(step_at4(rec, rc, j, r / GROUP4), (int)(b >> 4 * (r & 1) & 15) - 8);
}

// A tile word's eight codes (code t at bits 4 (t / 2) + 16 (t % 2), 8 more than it is) as the fp16 numbers z + s c, each
// rounded once. The conversion is the published one by exponent: bits or'ed into the significand of a power of two are that
// power and their number (for 4-bit weights in fp16: Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run", 2022).
// Four bits in 1024 are 1024 + n, or 1024 + 16 n from the next four, so that a pair of codes is a half each in two
// instructions (one shift for the second two pairs), exact; then one packed multiply-add.
__device__ __forceinline__ halfx8 values4(uint32_t word, halfx8 s, halfx8 z) {
    const halfx2 down = {(_Float16)-1032.0f, (_Float16)-1032.0f}, down16 = {(_Float16)-72.0f, (_Float16)-72.0f};
    const halfx2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    // in registers: as literals the and and the or would be an instruction each
    uint32_t low = 0x000F000Fu, up = 0x00F000F0u, base = 0x64006400u;
    asm("" : "+s"(low), "+s"(up), "+v"(base));
    const uint32_t high = word >> 8;
    halfx2 c[4];
    c[0] = __builtin_bit_cast(halfx2, (word & low) | base) + down;
    c[1] = __builtin_elementwise_fma(__builtin_bit_cast(halfx2, (word & up) | base), sixteenth, down16);
    c[2] = __builtin_bit_cast(halfx2, (high & low) | base) + down;
    c[3] = __builtin_elementwise_fma(__builtin_bit_cast(halfx2, (high & up) | base), sixteenth, down16);
    halfx8 v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const halfx2 x = __builtin_elementwise_fma(c[i], halfx2{s[2 * i], s[2 * i + 1]}, halfx2{z[2 * i], z[2 * i + 1]});
        v[2 * i] = x[0];
        v[2 * i + 1] = x[1];
    }
    return v;
}

}  // namespace tah

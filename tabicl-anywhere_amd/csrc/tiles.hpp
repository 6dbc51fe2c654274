// What the attention kernels over split-fp16 tiles of 64 keys share.
#pragma once

#include "device_math.hpp"

namespace tah {

constexpr int KB = 64;   // keys per block

// rows r and r + 1 already sit in different bank halves (128-byte rows); rows of one parity among 16 consecutive ones
// get eight different chunks
__device__ __forceinline__ int swz(int r, int c) { return c ^ ((r >> 1) & 7); }

// Half an image (its keys or its values: BYTES, 16 KB of split values or 8 KB of codes) into an LDS buffer, 16 bytes
// a lane: in copy i, wavefront w fills the 1 KB at chunk 64 (WAVES i + w) (a wavefront-uniform LDS base; the lanes'
// offsets are implicit).
template <int WAVES, int BYTES>
__device__ __forceinline__ void half_image_to_lds(const uint8_t *src, uint8_t *dst, int tid) {
    constexpr int T = 64 * WAVES, CHUNKS = BYTES / 16;
    static_assert(BYTES % 16 == 0, "whole 16-byte copies");
    const int w = tid >> 6;
#pragma unroll
    for (int i = 0; i < (CHUNKS + T - 1) / T; i++) {
        const int base = i * T + 64 * w;
        // lanes past the last copy stay idle (a copy a lane: each writes its own 16 bytes at dst + 16 (base + lane))
        if (CHUNKS % T == 0 || base + (tid & 63) < CHUNKS)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint4 *>(src) + base + (tid & 63), dst + 16 * base, 16,
                                             0, 0);
    }
}

template <bool B>
struct Flag {
    static constexpr bool value = B;
};

}  // namespace tah

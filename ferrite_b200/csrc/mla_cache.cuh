// Rows of a latent cache in 4 or 8 bits. A token's row: codes of its L latent values | R = 64 rotated key values in bf16 | scale bytes | zeros up to 16 bytes.
//
//   4 bits   groups of 16 share a scale (8 + f) / 8 * 2^(e - 20), byte e << 3 | f: their largest magnitude / 7 to four significant bits. Code c in
//            -7..7 is held as the nibble c + 8; of eight values' word, nibble i is value 2 i and nibble 4 + i value 2 i + 1, so that a shift and a mask
//            leave neighbours in the halves of a register.
//   8 bits   groups of 32 share a power of two 2^k, byte k + 127, k in -15..7: the smallest that brings their largest magnitude to 448 or less; codes
//            are e4m3.
//   A group with a value that is no finite number has scale byte 255 and reads back as NaN.
//
// code * scale has at most seven significant bits and no bit below 2^-24: it is exact in bf16 and in fp16. Scale bytes lie half by half of every 64
// values (of the lower 32 of all 64s, then of the upper 32), so that a thread with 32 of every 64 values finds its own side by side.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace fb {

constexpr int LC_R = 64;               // width of the rotated key part
constexpr int LC_MAX_L = 512;          // latent widths: multiples of 64 up to this
constexpr int LC_NAN = 255;

template <int BITS>
struct LatentRow {
  static constexpr int group = BITS == 4 ? 16 : 32;              // values to a scale
  static constexpr int per_half = 32 / group;                    // scales to 32 values
  __host__ __device__ static constexpr int rope_at(int L) { return L * BITS / 8; }
  __host__ __device__ static constexpr int scale_at(int L) { return rope_at(L) + 2 * LC_R; }
  __host__ __device__ static constexpr int bytes(int L) { return (scale_at(L) + L / group + 15) / 16 * 16; }
  // byte of the scale of value e
  __host__ __device__ static constexpr int scale_of(int L, int e) {
    return scale_at(L) + (e / 32 % 2) * (L / 64 * per_half) + e / 64 * per_half + e % 32 / group;
  }
};
__host__ __device__ inline int latent_row_bytes(int L, int bits) { return bits == 4 ? LatentRow<4>::bytes(L) : LatentRow<8>::bytes(L); }

// the scale that a byte stands for (the caller looks for LC_NAN)
template <int BITS>
__device__ __forceinline__ float latent_scale(uint32_t byte) {
  return BITS == 4 ? __uint_as_float((byte << 20) + (107u << 23)) : __uint_as_float(byte << 23);
}
template <int BITS>
__device__ __forceinline__ bool latent_scale_nan(uint32_t byte) { return byte >= (BITS == 4 ? 248u : 135u); }

}  // namespace fb

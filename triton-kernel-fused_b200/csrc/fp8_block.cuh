// e4m3 codes with an fp32 scale per block of 128 values: shared by the quantiser and by the products that requantise their result.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "common.cuh"
#include "mxfp8_quant.cuh"
#include "ptx.cuh"

namespace b200moe {

constexpr int kBlockK = 128;                            // values that share a scale
constexpr uint32_t kAmaxFloor = 0x0d800000u;            // 2^-100: a block below it (of zeros) still has a scale
constexpr float kE4m3Max = 448.0f;

// scale = max(amax, 2^-100) / 448, correctly rounded, and the factor 448 / amax that codes are made with; amax as the bits of |x|, so that NaN
// is above all.  The quotient a / 448 = a / 7 / 64 is never nearer than 1/14 of a step to the middle between two fp32 numbers, so a product
// with 1 / 448, corrected once by its remainder, rounds to the right one.
__device__ __forceinline__ void block_scale_factor(uint32_t amax_bits, float& scale, float& factor) {
  const float a = __uint_as_float(max(amax_bits, kAmaxFloor));
  if (a < 1e30f) {
    constexpr float kInv = 1.0f / kE4m3Max;
    const float s = a * kInv;
    scale = fmaf(fmaf(-s, kE4m3Max, a), kInv, s);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    factor = kE4m3Max * r;
  } else {                 // the reciprocal may be too small for a normal number; infinity and NaN
    scale = __fdiv_rn(a, kE4m3Max);
    factor = __fdiv_rn(kE4m3Max, a);
  }
}

// A code is the e4m3 value nearest to 448 x / amax.  For bf16 x and amax, both of 8 bits, that quotient is either exactly half way between
// two codes or at least 2^-13 away from there (relative), while x * (448 / amax) is off by 2^-23: rounded to 20 bits first, it is half
// way exactly where the quotient is, and ties go to even as they should.  (Without, one value in some hundred goes the other way.)
__device__ __forceinline__ float block_snap(float q) { return __uint_as_float((__float_as_uint(q) + 8u) & ~15u); }

// 8 bf16 values -> their codes; and the larger of m and their |x|, as bits, in each half of a word
__device__ __forceinline__ uint2 block_codes8(const uint4& v, float factor, bool finite) {
  const uint32_t words[4] = {v.x, v.y, v.z, v.w};
  float a[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[2 * i] = bf16_lo(words[i]) * factor;
    a[2 * i + 1] = bf16_hi(words[i]) * factor;
  }
  if (finite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = block_snap(a[i]);
  }
  return make_uint2(cvt4_e4m3(a[0], a[1], a[2], a[3]), cvt4_e4m3(a[4], a[5], a[6], a[7]));
}
__device__ __forceinline__ uint32_t absmax8(uint32_t m, const uint4& v) {
  return __vmaxu2(m, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
}

// First row of scales of k-block kb: scales lie block by block, rows in order (a warp's rows are one line)
__device__ __forceinline__ long long scale_at(int kb, long long pitch, long long row) { return kb * pitch + row; }

// Elements between the scales of two k-blocks: rows rounded up so that a bulk copy of the last rows stays inside
inline int64_t scale_pitch(int64_t rows) { return (rows + 127) / 128 * 128; }
// Bytes between rows of codes
inline int64_t code_pitch(int64_t K) { return (K + 15) / 16 * 16; }

// fp8_block.cu
int fp8_block_quant(const void* x, int64_t rows, int64_t K, int64_t out_rows, const int32_t* slot_row, int k, void* q, int64_t ldq, float* scale,
                    int64_t pitch, b200moe_stream_t stream);

}  // namespace b200moe

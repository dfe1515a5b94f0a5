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

// scale = max(amax, 2^-100) / 448 and the factor 448 / amax that codes are made with; amax as the bits of |x|, so that NaN is above all
__device__ __forceinline__ float block_scale(uint32_t amax_bits) { return __fdiv_rn(__uint_as_float(max(amax_bits, kAmaxFloor)), kE4m3Max); }
__device__ __forceinline__ float block_factor(uint32_t amax_bits) { return __fdiv_rn(kE4m3Max, __uint_as_float(max(amax_bits, kAmaxFloor))); }

// A code is the e4m3 value nearest to 448 x / amax.  For bf16 x and amax, both of 8 bits, that quotient is either exactly half way between
// two codes or at least 2^-13 away from there (relative), while x * (448 / amax) is off by 2^-23: rounded to 20 bits first, it is half
// way exactly where the quotient is, and ties go to even as they should.  (Without, one value in some hundred goes the other way.)
__device__ __forceinline__ float block_snap(float q) { return __uint_as_float((__float_as_uint(q) + 8u) & ~15u); }

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

// Quantiser of activations: bf16 rows -> e4m3 codes with an fp32 scale per row and block of 128 values.
//
//   scale = max(|x|) / 448 (a block's largest value becomes 448, e4m3's largest), code = nearest e4m3 to 448 x / max(|x|)
//
// Sixteen lanes a block, eight values each: one 16-byte load and one 8-byte store a lane.  Bound by HBM: 2 bytes in and one out a value.
// With a table of rows (experts) a token's codes are made once and written to each of its rows.
#include <algorithm>

#include "fp8_block.cuh"

namespace b200moe {

__global__ void __launch_bounds__(256)
fp8_block_quant_kernel(const __nv_bfloat16* x, long long rows, int K, const int* slot_row, int k, uint8_t* q, long long ldq, float* scale,
                       long long pitch) {
  grid_dep_begin();
  const int lane16 = threadIdx.x & 15;
  const unsigned half = 0xffffu << (threadIdx.x & 16);      // the lanes of this block
  const int blocks = (K + kBlockK - 1) / kBlockK;
  const long long total = rows * blocks;
  for (long long i = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 4; i < total;
       i += (static_cast<long long>(gridDim.x) * blockDim.x) >> 4) {
    const long long r = i / blocks;
    const int kb = static_cast<int>(i - r * blocks), c = kb * kBlockK + 8 * lane16;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (c < K) v = *reinterpret_cast<const uint4*>(x + r * K + c);       // K is a multiple of 8
    uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    m = max(m & 0xffffu, m >> 16) << 16;                                 // the bits of the largest |x|
    m = __reduce_max_sync(half, m);
    const float f = block_factor(m);
    const bool finite = m < 0x7f800000u;
    auto code = [&](uint32_t w, float& a, float& b) {
      a = bf16_lo(w) * f;
      b = bf16_hi(w) * f;
      if (finite) {
        a = block_snap(a);
        b = block_snap(b);
      }
    };
    float a[8];
    code(v.x, a[0], a[1]);
    code(v.y, a[2], a[3]);
    code(v.z, a[4], a[5]);
    code(v.w, a[6], a[7]);
    const uint2 o = make_uint2(cvt4_e4m3(a[0], a[1], a[2], a[3]), cvt4_e4m3(a[4], a[5], a[6], a[7]));
    const float s = block_scale(m);
    if (slot_row == nullptr) {
      if (c < K) *reinterpret_cast<uint2*>(q + r * ldq + c) = o;
      if (lane16 == 0) scale[scale_at(kb, pitch, r)] = s;
    } else {
      for (int j = 0; j < k; ++j) {
        const long long to = slot_row[r * k + j];
        if (to < 0) continue;            // a pick that names no expert has no row
        if (c < K) *reinterpret_cast<uint2*>(q + to * ldq + c) = o;
        if (lane16 == 0) scale[scale_at(kb, pitch, to)] = s;
      }
    }
  }
}

int fp8_block_quant(const void* x, int64_t rows, int64_t K, int64_t out_rows, const int32_t* slot_row, int k, void* q, int64_t ldq, float* scale,
                    int64_t pitch, b200moe_stream_t stream) {
  B200_CHECK_ARG(x && q && scale, B200MOE_E_NULL, "fp8_block_quant: null pointer");
  B200_CHECK_ARG(rows >= 0 && K > 0 && K % 8 == 0 && K < (1LL << 31), B200MOE_E_BAD_SHAPE,
                 "fp8_block_quant: rows = %lld, K = %lld (a positive multiple of 8)", (long long)rows, (long long)K);
  B200_CHECK_ARG(ldq >= K && ldq % 8 == 0 && pitch >= out_rows, B200MOE_E_BAD_SHAPE, "fp8_block_quant: rows of codes %lld bytes apart, scales %lld",
                 (long long)ldq, (long long)pitch);
  B200_CHECK_ARG(aligned16(x) && reinterpret_cast<uintptr_t>(q) % 8 == 0, B200MOE_E_ALIGN, "fp8_block_quant: x must be 16-byte, q 8-byte aligned");
  if (rows == 0) return 0;
  const int64_t blocks = (rows * ((K + kBlockK - 1) / kBlockK) + 15) / 16;
  B200_LAUNCH(fp8_block_quant_kernel, static_cast<int>(std::min<int64_t>(blocks, static_cast<int64_t>(num_sms()) * 16)), 256, 0, stream,
              reinterpret_cast<const __nv_bfloat16*>(x), static_cast<long long>(rows), static_cast<int>(K), slot_row, k,
              reinterpret_cast<uint8_t*>(q), static_cast<long long>(ldq), scale, static_cast<long long>(pitch));
  return 0;
}

// Weights, once: codes and one scale of a block of 128 x 128 values.  One CTA a block, 64 values a thread, all loaded before the
// largest is known.
__global__ void __launch_bounds__(256)
fp8_block_quant_weight_kernel(const __nv_bfloat16* w, long long N, int K, uint8_t* q, float* scale) {
  grid_dep_begin();
  __shared__ uint32_t warp_max_s[8];
  const int kb = (K + kBlockK - 1) / kBlockK;
  const long long nb = (N + kBlockK - 1) / kBlockK;
  const long long g = blockIdx.x / (nb * kb);
  const long long rem = blockIdx.x - g * nb * kb, bn = rem / kb;
  const int c = static_cast<int>(rem - bn * kb) * kBlockK + 8 * (threadIdx.x & 15);
  const long long r0 = bn * kBlockK + (threadIdx.x >> 4);
  uint4 v[8];
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (c < K && r0 + 16 * i < N) v[i] = *reinterpret_cast<const uint4*>(w + (g * N + r0 + 16 * i) * K + c);
    m = __vmaxu2(m, __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu), __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu)));
  }
  m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16) << 16);
  if ((threadIdx.x & 31) == 0) warp_max_s[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, warp_max_s[i]);
  const float f = block_factor(m);
  const bool finite = m < 0x7f800000u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (c >= K || r0 + 16 * i >= N) continue;
    const uint32_t words[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    uint32_t o[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float a[4] = {bf16_lo(words[2 * h]) * f, bf16_hi(words[2 * h]) * f, bf16_lo(words[2 * h + 1]) * f, bf16_hi(words[2 * h + 1]) * f};
      if (finite)
        for (int j = 0; j < 4; ++j) a[j] = block_snap(a[j]);
      o[h] = cvt4_e4m3(a[0], a[1], a[2], a[3]);
    }
    *reinterpret_cast<uint2*>(q + (g * N + r0 + 16 * i) * K + c) = make_uint2(o[0], o[1]);
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = block_scale(m);
}

}  // namespace b200moe

using namespace b200moe;

extern "C" {

int b200moe_fp8_block_quant_weight(const void* w, int64_t groups, int64_t N, int64_t K, void* q, float* scale, b200moe_stream_t stream) {
  B200_CHECK_ARG(w && q && scale, B200MOE_E_NULL, "fp8_block_quant_weight: null pointer");
  const int64_t blocks = groups * ((N + kBlockK - 1) / kBlockK) * ((K + kBlockK - 1) / kBlockK);
  B200_CHECK_ARG(groups >= 1 && N > 0 && K > 0 && K % 8 == 0 && K < (1LL << 31) && blocks < (1LL << 31), B200MOE_E_BAD_SHAPE,
                 "fp8_block_quant_weight: %lld matrices of %lld x %lld (a positive multiple of 8)", (long long)groups, (long long)N, (long long)K);
  B200_CHECK_ARG(aligned16(w) && reinterpret_cast<uintptr_t>(q) % 8 == 0, B200MOE_E_ALIGN,
                 "fp8_block_quant_weight: w must be 16-byte, q 8-byte aligned");
  B200_LAUNCH(fp8_block_quant_weight_kernel, static_cast<int>(blocks), 256, 0, stream, reinterpret_cast<const __nv_bfloat16*>(w),
              static_cast<long long>(N), static_cast<int>(K), reinterpret_cast<uint8_t*>(q), scale);
  return 0;
}

int b200moe_fp8_block_quant(const void* x, int64_t rows, int64_t K, void* q, int64_t ldq, float* scale, int64_t scale_pitch_,
                            b200moe_stream_t stream) {
  return fp8_block_quant(x, rows, K, rows, nullptr, 1, q, ldq, scale, scale_pitch_, stream);
}

}  // extern "C"

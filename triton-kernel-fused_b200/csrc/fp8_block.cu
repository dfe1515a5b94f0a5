// Quantiser of activations: bf16 rows -> e4m3 codes with an fp32 scale per row and block of 128 values.
//
//   scale = max(|x|) / 448 (a block's largest value becomes 448, e4m3's largest), code = nearest e4m3 to 448 x / max(|x|)
//
// Eight lanes a block, sixteen values each, kQuantAhead blocks of a lane on their way.  Bound by HBM, 2 bytes in and one out a value, and close
// behind by issue: 8192 x 14336 in 59.5 us, 5.4 TB/s (with sixteen lanes a block and quotients by division 120).  With a table of rows (experts) a
// token's codes are made once and written to each of its rows.
#include <algorithm>

#include "fp8_block.cuh"

namespace b200moe {

constexpr int kQuantAhead = 3;

// 16 values -> their codes
__device__ __forceinline__ void block_codes(const uint4 (&v)[2], float factor, bool finite, uint2 (&o)[2]) {
  o[0] = block_codes8(v[0], factor, finite);
  o[1] = block_codes8(v[1], factor, finite);
}

__global__ void __launch_bounds__(256)
fp8_block_quant_kernel(const __nv_bfloat16* x, long long rows, int K, const int* slot_row, int k, uint8_t* q, long long ldq, float* scale,
                       long long pitch) {
  grid_dep_begin();
  const int lane8 = threadIdx.x & 7;
  const int blocks = (K + kBlockK - 1) / kBlockK;
  // the first block of these eight lanes and their step, as (row, block of the row)
  const long long begin = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 3;
  const long long step = (static_cast<long long>(gridDim.x) * blockDim.x) >> 3;
  const long long step_r = step / blocks;
  const int step_b = static_cast<int>(step - step_r * blocks);
  long long r = begin / blocks;
  int b = static_cast<int>(begin - r * blocks);
  while (__any_sync(0xffffffffu, r < rows)) {      // all four blocks of a warp, for the shuffles
    uint4 v[kQuantAhead][2];
    long long row[kQuantAhead];
    int kb[kQuantAhead];
#pragma unroll
    for (int u = 0; u < kQuantAhead; ++u) {
      row[u] = r;
      kb[u] = b;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = b * kBlockK + 64 * h + 8 * lane8;
        v[u][h] = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows && c < K) v[u][h] = *reinterpret_cast<const uint4*>(x + r * K + c);       // K is a multiple of 8
      }
      r += step_r;
      b += step_b;
      if (b >= blocks) {
        b -= blocks;
        ++r;
      }
    }
#pragma unroll
    for (int u = 0; u < kQuantAhead; ++u) {
      uint32_t m = absmax8(absmax8(0u, v[u][0]), v[u][1]);
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, off));
      m = max(m & 0xffffu, m >> 16) << 16;                                 // the bits of the largest |x|
      if (row[u] >= rows) continue;
      float s, f;
      block_scale_factor(m, s, f);
      uint2 o[2];
      block_codes(v[u], f, m < 0x7f800000u, o);
      const int c = kb[u] * kBlockK + 8 * lane8;
      if (slot_row == nullptr) {
        uint8_t* to = q + row[u] * ldq + c;
        if (c < K) *reinterpret_cast<uint2*>(to) = o[0];
        if (c + 64 < K) *reinterpret_cast<uint2*>(to + 64) = o[1];
        if (lane8 == 0) scale[scale_at(kb[u], pitch, row[u])] = s;
      } else {
        for (int j = 0; j < k; ++j) {
          const long long rr = slot_row[row[u] * k + j];
          if (rr < 0) continue;            // a pick that names no expert has no row
          uint8_t* to = q + rr * ldq + c;
          if (c < K) *reinterpret_cast<uint2*>(to) = o[0];
          if (c + 64 < K) *reinterpret_cast<uint2*>(to + 64) = o[1];
          if (lane8 == 0) scale[scale_at(kb[u], pitch, rr)] = s;
        }
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
  OpScope scope("fp8_block_quant", 1);
  // three blocks of 128 for each eight lanes, but a CTA an SM where there is work for them
  const int64_t blocks = rows * ((K + kBlockK - 1) / kBlockK);
  const int64_t ctas = std::max<int64_t>((blocks + 32 * kQuantAhead - 1) / (32 * kQuantAhead), std::min<int64_t>((blocks + 31) / 32, num_sms()));
  B200_LAUNCH(fp8_block_quant_kernel, static_cast<int>(std::min<int64_t>(ctas, static_cast<int64_t>(num_sms()) * 16)), 256, 0, stream,
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
    m = absmax8(m, v[i]);
  }
  m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16) << 16);
  if ((threadIdx.x & 31) == 0) warp_max_s[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, warp_max_s[i]);
  float sc, f;
  block_scale_factor(m, sc, f);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint4 two[2] = {v[i], v[i + 1]};
    uint2 o[2];
    block_codes(two, f, m < 0x7f800000u, o);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (c < K && r0 + 16 * (i + h) < N) *reinterpret_cast<uint2*>(q + (g * N + r0 + 16 * (i + h)) * K + c) = o[h];
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = sc;
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
  OpScope scope("fp8_block_quant_weight", 1);
  B200_LAUNCH(fp8_block_quant_weight_kernel, static_cast<int>(blocks), 256, 0, stream, reinterpret_cast<const __nv_bfloat16*>(w),
              static_cast<long long>(N), static_cast<int>(K), reinterpret_cast<uint8_t*>(q), scale);
  return 0;
}

int b200moe_fp8_block_quant(const void* x, int64_t rows, int64_t K, void* q, int64_t ldq, float* scale, int64_t scale_pitch_,
                            b200moe_stream_t stream) {
  return fp8_block_quant(x, rows, K, rows, nullptr, 1, q, ldq, scale, scale_pitch_, stream);
}

}  // extern "C"

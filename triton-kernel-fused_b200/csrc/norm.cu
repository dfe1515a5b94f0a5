// Root-mean-square norm of rows, with the residual's addition before it and its result as rows, as e4m3 codes with a scale per 128 values, or both:
//
//   h = x + residual, rounded to the rows' type      rstd = 1 / sqrt(mean(h^2) + eps)      n = h rstd      y = n w
//
// and its gradient: d = grad_y w,  grad_x = rstd (d - n mean(d n)) + grad_h  (of x and of the residual alike),  grad_w = sum over the rows of grad_y n.
//
// The norm is taken of h as it goes on, rounded, so that the backward, which has h alone, computes the gradient of what the forward computed; rstd
// is computed again there, from a row that is read anyway.  Codes are made from y in fp32, not from its rounding.  All sums are fp32.
//
// Bound by HBM: a row is read once and stays in registers between the sum and what is made of it.
#include <algorithm>

#include "fp8_block.cuh"
#include "logits.cuh"

namespace b200moe {

constexpr int kNormMaxK = 16384;

// Eight neighbouring values of a row as they lie in memory: what a thread holds of each 8 x (threads of the row) values
template <class T>
struct Eight {
  uint4 raw[sizeof(T) == 4 ? 2 : 1];
};
// left: values of the row from p on.  VEC: p is 16-byte aligned and left a multiple of 8.
template <bool VEC, class T>
__device__ __forceinline__ Eight<T> load8(const T* p, int left) {
  Eight<T> v;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(v.raw) / 16); ++i)
      v.raw[i] = left > 0 ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0u, 0u, 0u, 0u);
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < left ? p[i] : from_f32<T>(0.0f);
    memcpy(&v, e, sizeof(v));
  }
  return v;
}
template <class T>
__device__ __forceinline__ void values8(const Eight<T>& v, float (&f)[8]) {
  T e[8];
  memcpy(e, &v, sizeof(v));
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32(e[i]);
}
template <bool VEC, class T>
__device__ __forceinline__ void store8(T* p, int left, const float (&f)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(f[i]);
  if constexpr (VEC) {
    if (left <= 0) return;
    Eight<T> v;
    memcpy(&v, e, sizeof(v));
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(v.raw) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = v.raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = e[i];
  }
}

// Sums over the threads of a row: a warp's, or a CTA's by way of `part`, which two rows in turn use
template <int N, bool WARP>
__device__ __forceinline__ void row_sums(float (&s)[N], float (&part)[2][N][32], int flip) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = warp_sum(s[i]);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0)
      for (int i = 0; i < N; ++i) part[flip][i][warp] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = warp_sum(lane < warps ? part[flip][i][lane] : 0.0f);
  }
}

struct NormFwd {
  const void *x, *residual, *w;      // residual: nullable
  long long ldx, ldr;                // elements between rows
  void *y, *h;                       // nullable, contiguous
  uint8_t* q;                        // nullable: codes (rows, K) and scales [block of 128][pitch]
  float* scale;
  long long pitch, rows;
  int K;
  float eps;
};

// WARP: a warp a row, else a CTA.  NV: groups of eight values a thread.
template <class T, class W, int NV, bool VEC, bool WARP, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_fwd_kernel(const NormFwd a) {
  grid_dep_begin();
  __shared__ float part[2][1][32];
  const int tpr = WARP ? 32 : static_cast<int>(blockDim.x);
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int rows_cta = WARP ? blockDim.x >> 5 : 1;
  const T *x = static_cast<const T*>(a.x), *r = static_cast<const T*>(a.residual);
  Eight<W> w[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = 8 * (j * tpr + t);
    w[j] = load8<VEC>(static_cast<const W*>(a.w) + c, a.K - c);
  }
  int flip = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * rows_cta + (WARP ? threadIdx.x >> 5 : 0); row < a.rows;
       row += static_cast<long long>(gridDim.x) * rows_cta, flip ^= 1) {
    Eight<T> xv[NV], rv[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 8 * (j * tpr + t);
      xv[j] = load8<VEC>(x + row * a.ldx + c, a.K - c);
      if (r != nullptr) rv[j] = load8<VEC>(r + row * a.ldr + c, a.K - c);
    }
    float v[NV][8], ss[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      values8(xv[j], v[j]);
      if (r != nullptr) {
        float o[8];
        values8(rv[j], o);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = to_f32(from_f32<T>(v[j][i] + o[i]));
        const int c = 8 * (j * tpr + t);
        if (a.h != nullptr) store8<VEC>(static_cast<T*>(a.h) + row * a.K + c, a.K - c, v[j]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss[0] = fmaf(v[j][i], v[j][i], ss[0]);
    }
    row_sums<1, WARP>(ss, part, flip);
    const float rstd = 1.0f / sqrtf(ss[0] / static_cast<float>(a.K) + a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 8 * (j * tpr + t);
      float o[8];
      values8(w[j], o);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * rstd * o[i];
      if (a.y != nullptr) store8<VEC>(static_cast<T*>(a.y) + row * a.K + c, a.K - c, v[j]);
      if (a.q != nullptr) {        // sixteen threads hold a block of 128
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[j][i]) & 0x7fffffffu);
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
        float s, f;
        block_scale_factor(m, s, f);
        if (c < a.K) {
          uint2 o2;
          o2.x = cvt4_e4m3(v[j][0] * f, v[j][1] * f, v[j][2] * f, v[j][3] * f);
          o2.y = cvt4_e4m3(v[j][4] * f, v[j][5] * f, v[j][6] * f, v[j][7] * f);
          *reinterpret_cast<uint2*>(a.q + row * a.K + c) = o2;
          if ((t & 15) == 0) a.scale[scale_at(c / kBlockK, a.pitch, row)] = s;
        }
      }
    }
  }
}

struct NormBwd {
  const void *gy, *gh, *h, *w;       // gh: nullable
  long long ldh;                     // elements between rows of h
  void* gx;                          // nullable
  float* part;                       // nullable: (CTAs, K), each CTA's rows' share of grad_w
  long long rows;
  int K;
  float eps;
};

template <class T, class W, int NV, bool VEC, bool WARP, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_bwd_kernel(const NormBwd a) {
  grid_dep_begin();
  __shared__ float part[2][2][32];
  __shared__ float s_sum[WARP ? 8 * 32 * NV : 1];
  const int tpr = WARP ? 32 : static_cast<int>(blockDim.x);
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int rows_cta = WARP ? blockDim.x >> 5 : 1;
  const T *gy = static_cast<const T*>(a.gy), *gh = static_cast<const T*>(a.gh), *h = static_cast<const T*>(a.h);
  Eight<W> w[NV];
  float acc[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = 8 * (j * tpr + t);
    w[j] = load8<VEC>(static_cast<const W*>(a.w) + c, a.K - c);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[j][i] = 0.0f;
  }
  int flip = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * rows_cta + (WARP ? threadIdx.x >> 5 : 0); row < a.rows;
       row += static_cast<long long>(gridDim.x) * rows_cta, flip ^= 1) {
    Eight<T> hv[NV], gv[NV], ov[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 8 * (j * tpr + t);
      hv[j] = load8<VEC>(h + row * a.ldh + c, a.K - c);
      gv[j] = load8<VEC>(gy + row * a.K + c, a.K - c);
      if (gh != nullptr) ov[j] = load8<VEC>(gh + row * a.K + c, a.K - c);
    }
    float s[2] = {0.0f, 0.0f};       // of h^2 and of h d
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float hf[8], gf[8], wf[8];
      values8(hv[j], hf);
      values8(gv[j], gf);
      values8(w[j], wf);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[0] = fmaf(hf[i], hf[i], s[0]);
        s[1] = fmaf(hf[i], gf[i] * wf[i], s[1]);
      }
    }
    row_sums<2, WARP>(s, part, flip);
    const float rstd = 1.0f / sqrtf(s[0] / static_cast<float>(a.K) + a.eps);
    const float back = s[1] * rstd / static_cast<float>(a.K);       // mean(d n)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 8 * (j * tpr + t);
      float hf[8], gf[8], wf[8], of[8];
      values8(hv[j], hf);
      values8(gv[j], gf);
      values8(w[j], wf);
      if (gh != nullptr) values8(ov[j], of);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = hf[i] * rstd;
        acc[j][i] = fmaf(gf[i], n, acc[j][i]);
        hf[i] = rstd * (gf[i] * wf[i] - n * back);
        if (gh != nullptr) hf[i] += of[i];
      }
      if (a.gx != nullptr) store8<VEC>(static_cast<T*>(a.gx) + row * a.K + c, a.K - c, hf);
    }
  }
  if (a.part == nullptr) return;
  if constexpr (WARP) {              // the warps' sums one after another
    for (int u = 0; u < rows_cta; ++u) {
      __syncthreads();
      if (static_cast<int>(threadIdx.x >> 5) == u) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float* to = s_sum + (8 * j + i) * 32 + t;
            *to = u == 0 ? acc[j][i] : *to + acc[j][i];
          }
      }
    }
    __syncthreads();
    if (threadIdx.x < 32) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j][i] = s_sum[(8 * j + i) * 32 + t];
    } else {
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = 8 * (j * tpr + t) + i;
      if (c < a.K) a.part[static_cast<long long>(blockIdx.x) * a.K + c] = acc[j][i];
    }
}

// out (K) = the sum of part (P, K) over P, 32 columns a CTA, always in the same order
template <class W>
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float* part, int P, int K, W* out) {
  grid_dep_begin();
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (c < K)
    for (int p = warp; p < P; p += 32) v += part[static_cast<long long>(p) * K + c];
  s[warp][lane] = v;
  __syncthreads();
  v = warp_sum(s[lane][warp]);
  if (lane == 0 && blockIdx.x * 32 + warp < K) out[blockIdx.x * 32 + warp] = from_f32<W>(v);
}

static bool same_or_f32(int type, int w_type) { return w_type == type || w_type == B200MOE_F32; }
// f(T, W) for rows of T and a weight of the same type or fp32
template <class F>
static int by_types(int type, int w_type, F f) {
  if (type == B200MOE_F32) return f(float(), float());
  if (type == B200MOE_BF16) return w_type == type ? f(__nv_bfloat16(), __nv_bfloat16()) : f(__nv_bfloat16(), float());
  return w_type == type ? f(__half(), __half()) : f(__half(), float());
}
// rows at `p`, `ld` elements apart, that vectors of 16 bytes can be read from
static bool vectors(const void* p, int64_t ld, int type) { return aligned16(p) && (ld * type_bytes(type)) % 16 == 0; }

static int row_threads(int64_t K, int nv) { return static_cast<int>((K + 8 * nv * 32 - 1) / (8 * nv * 32)) * 32; }
static int64_t norm_ctas(int64_t rows, int rows_cta, int threads, int threads_sm) {
  return std::max<int64_t>(1, std::min<int64_t>((rows + rows_cta - 1) / rows_cta, static_cast<int64_t>(num_sms()) * (threads_sm / threads)));
}

constexpr int kBwdThreadsSm = 768;
static int bwd_threads(int64_t K) { return K <= 1024 ? 256 : row_threads(K, 2); }
static int64_t bwd_ctas(int64_t rows, int64_t K) {
  const int threads = bwd_threads(K);
  return norm_ctas(rows, K <= 1024 ? 8 : 1, threads, std::max(kBwdThreadsSm, threads));
}

}  // namespace b200moe

using namespace b200moe;

static int check_norm(const char* who, int type, int w_type, int64_t rows, int64_t K, float eps) {
  B200_CHECK_ARG(known_logits(type) && same_or_f32(type, w_type), B200MOE_E_UNSUPPORTED, "%s: rows of type %d with a weight of type %d", who, type,
                 w_type);
  B200_CHECK_ARG(rows >= 0 && rows < (1LL << 31) - 256, B200MOE_E_BAD_SHAPE, "%s: %lld rows", who, (long long)rows);
  B200_CHECK_ARG(K >= 1 && K <= kNormMaxK, B200MOE_E_BAD_SHAPE, "%s: rows of %lld values, supported 1..%d", who, (long long)K, kNormMaxK);
  B200_CHECK_ARG(eps >= 0.0f, B200MOE_E_BAD_SHAPE, "%s: eps = %g must not be negative", who, (double)eps);
  return 0;
}

extern "C" {

int b200moe_rms_norm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, int type, const void* weight, int weight_type, int64_t rows,
                         int64_t K, float eps, void* y, void* h, void* q, float* scale, int64_t scale_pitch_, b200moe_stream_t stream) {
  const int rc = check_norm("rms_norm_fwd", type, weight_type, rows, K, eps);
  if (rc) return rc;
  B200_CHECK_ARG(ldx >= K && (residual == nullptr || ldr >= K), B200MOE_E_BAD_SHAPE, "rms_norm_fwd: rows %lld and %lld apart, shorter than K = %lld",
                 (long long)ldx, (long long)ldr, (long long)K);
  B200_CHECK_ARG(q == nullptr || (K % 8 == 0 && scale_pitch_ >= rows), B200MOE_E_BAD_SHAPE,
                 "rms_norm_fwd: codes of K = %lld (a multiple of 8), scales %lld apart", (long long)K, (long long)scale_pitch_);
  if (rows == 0) return 0;
  B200_CHECK_ARG(x && weight && (y || h || q) && (q == nullptr || scale) && (h == nullptr || residual), B200MOE_E_NULL, "rms_norm_fwd: null pointer");
  B200_CHECK_ARG(reinterpret_cast<uintptr_t>(q) % 8 == 0, B200MOE_E_ALIGN, "rms_norm_fwd: q must be 8-byte aligned");
  const bool vec = K % 8 == 0 && vectors(x, ldx, type) && (residual == nullptr || vectors(residual, ldr, type)) && aligned16(weight) &&
                   (y == nullptr || vectors(y, K, type)) && (h == nullptr || vectors(h, K, type));
  const NormFwd a{x, residual, weight, ldx, ldr, y, h, static_cast<uint8_t*>(q), scale, scale_pitch_, rows, static_cast<int>(K), eps};
  OpScope scope("rms_norm_fwd", 1);
  return by_types(type, weight_type, [&](auto t, auto w) -> int {
    using T = decltype(t);
    using W = decltype(w);
    auto run = [&](auto kernel, int rows_cta, int threads) -> int {
      B200_LAUNCH(kernel, static_cast<int>(norm_ctas(rows, rows_cta, threads, 1024)), threads, 0, stream, a);
      return 0;
    };
    if (rows <= num_sms() && K > 256 && K <= 8192)
      return vec ? run(rms_norm_fwd_kernel<T, W, 1, true, false, 1024>, 1, row_threads(K, 1))
                 : run(rms_norm_fwd_kernel<T, W, 1, false, false, 1024>, 1, row_threads(K, 1));
    if (K <= 1024) return vec ? run(rms_norm_fwd_kernel<T, W, 4, true, true, 256>, 8, 256) : run(rms_norm_fwd_kernel<T, W, 4, false, true, 256>, 8, 256);
    return vec ? run(rms_norm_fwd_kernel<T, W, 4, true, false, 512>, 1, row_threads(K, 4))
               : run(rms_norm_fwd_kernel<T, W, 4, false, false, 512>, 1, row_threads(K, 4));
  });
}

size_t b200moe_rms_norm_bwd_ws_bytes(int64_t rows, int64_t K) {
  if (rows <= 0 || K < 1 || K > kNormMaxK) return 0;
  return static_cast<size_t>(bwd_ctas(rows, K)) * K * sizeof(float);
}

int b200moe_rms_norm_bwd(const void* grad_y, const void* grad_h, const void* h, int64_t ldh, int type, const void* weight, int weight_type, int64_t rows,
                         int64_t K, float eps, void* ws, void* grad_x, void* grad_weight, b200moe_stream_t stream) {
  const int rc = check_norm("rms_norm_bwd", type, weight_type, rows, K, eps);
  if (rc) return rc;
  B200_CHECK_ARG(ldh >= K, B200MOE_E_BAD_SHAPE, "rms_norm_bwd: rows of h %lld apart, K = %lld", (long long)ldh, (long long)K);
  if (rows == 0 && grad_weight == nullptr) return 0;
  B200_CHECK_ARG((rows == 0 || (grad_y && h && weight)) && (grad_x || grad_weight), B200MOE_E_NULL, "rms_norm_bwd: null pointer");
  B200_CHECK_ARG(rows == 0 || grad_weight == nullptr || (ws && reinterpret_cast<uintptr_t>(ws) % 4 == 0), B200MOE_E_NULL,
                 "rms_norm_bwd: no workspace for the weight's gradient");
  const bool vec = K % 8 == 0 && vectors(grad_y, K, type) && vectors(h, ldh, type) && aligned16(weight) &&
                   (grad_h == nullptr || vectors(grad_h, K, type)) && (grad_x == nullptr || vectors(grad_x, K, type));
  const NormBwd a{grad_y, grad_h, h, weight, ldh, grad_x, grad_weight != nullptr ? static_cast<float*>(ws) : nullptr, rows, static_cast<int>(K), eps};
  const int64_t ctas = rows == 0 ? 0 : bwd_ctas(rows, K);
  OpScope scope("rms_norm_bwd", (rows > 0) + (grad_weight != nullptr));
  return by_types(type, weight_type, [&](auto t, auto w) -> int {
    using T = decltype(t);
    using W = decltype(w);
    auto run = [&](auto kernel) -> int {
      B200_LAUNCH(kernel, static_cast<int>(ctas), bwd_threads(K), 0, stream, a);
      return 0;
    };
    if (rows > 0) {
      const int rc2 = K <= 1024 ? (vec ? run(rms_norm_bwd_kernel<T, W, 4, true, true, 256>) : run(rms_norm_bwd_kernel<T, W, 4, false, true, 256>))
                      : K <= 4096 ? (vec ? run(rms_norm_bwd_kernel<T, W, 2, true, false, 256>) : run(rms_norm_bwd_kernel<T, W, 2, false, false, 256>))
                                  : (vec ? run(rms_norm_bwd_kernel<T, W, 2, true, false, 1024>) : run(rms_norm_bwd_kernel<T, W, 2, false, false, 1024>));
      if (rc2) return rc2;
    }
    if (grad_weight != nullptr)
      B200_LAUNCH(norm_weight_grad_kernel<W>, static_cast<int>((K + 31) / 32), 1024, 0, stream, static_cast<const float*>(ws), static_cast<int>(ctas),
                  static_cast<int>(K), static_cast<W*>(grad_weight));
    return 0;
  });
}

}  // extern "C"

// Root-mean-square norm of rows, with the residual's addition before it and its result as rows, as e4m3 codes with a scale per 128 values, or both:
//
//   h = x + residual, rounded to the rows' type      rstd = 1 / sqrt(mean(h^2) + eps)      n = h rstd      y = n w
//
// and its gradient: d = grad_y w,  grad_x = rstd (d - n mean(d n)) + grad_h  (of x and of the residual alike),  grad_w = sum over the rows of grad_y n.
//
// The norm is taken of h as it goes on, rounded, so that the backward, which has h alone, computes the gradient of what the forward computed; rstd
// is computed again there, from a row that is read anyway.  Codes are made from y in fp32, not from its rounding.  All sums are fp32.
//
// Bound by HBM: a row is read once.  Three forms: rows through shared memory, which a ring of bulk copies keeps full (rms_norm_*_rows_kernel); few rows of a
// forward, where latency counts, as vectors through registers (rms_norm_fwd_kernel with VEC); and rows off a vector's boundary value by value through registers
// (rms_norm_*_kernel without).  The last is bound by its loads: 16384 x 2047 forward and backward 315 us, 16384 x 2048 through shared memory 85, of 82.
#include <algorithm>
#include <limits>

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

// a + b, each sum rounded to T, as values.  Where a sum of two 16-bit numbers lies near the middle between two others it has at most 24 bits, so that
// rounding it at once, as the packed addition does, and by way of fp32 are the same.
template <class T>
__device__ __forceinline__ void sum8(const Eight<T>& a, const Eight<T>& b, Eight<T>& h, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    float o[8];
    values8(a, f);
    values8(b, o);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += o[i];
    memcpy(&h, f, sizeof(h));
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 p[4], q[4];
    memcpy(p, &a, 16);
    memcpy(q, &b, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __hadd2(p[i], q[i]);
    memcpy(&h, p, 16);
    values8(h, f);
  }
}
template <class T>
__device__ __forceinline__ void put8(T* p, int left, const Eight<T>& v) {
  if (left <= 0) return;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(v.raw) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = v.raw[i];
}
// 1 / sqrt(a): the approximation and a step of Newton's method, off by a rounding or two
__device__ __forceinline__ float inverse_root(float a) {
  const float r = rsqrtf(a);
  return a > 0.0f && a < 1e38f ? fmaf(r, 0.5f * fmaf(-a * r, r, 1.0f), r) : r;
}
// the larger, NaN where one is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
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

// a thread's eight values y at column c of a row -> codes and, once a block of 128 (sixteen threads), their scale
__device__ __forceinline__ void codes_of_pairs(const NormFwd& a, const float2 (&v)[4], long long row, int c, int t) {
  float most = fabsf(v[0].x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i > 0) most = max_nan(most, fabsf(v[i].x));
    most = max_nan(most, fabsf(v[i].y));
  }
  uint32_t m = __float_as_uint(most);
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
  float s, f;
  block_scale_factor(m, s, f);
  if (c < a.K) {
    uint2 o;
    o.x = cvt4_e4m3(v[0].x * f, v[0].y * f, v[1].x * f, v[1].y * f);
    o.y = cvt4_e4m3(v[2].x * f, v[2].y * f, v[3].x * f, v[3].y * f);
    *reinterpret_cast<uint2*>(a.q + row * a.K + c) = o;
    if ((t & 15) == 0) a.scale[scale_at(c / kBlockK, a.pitch, row)] = s;
  }
}
// ... and h -> y, codes or both
template <bool VEC, class T, class W>
__device__ __forceinline__ void finish8(const NormFwd& a, const Eight<W>& w, float (&v)[8], float rstd, long long row, int c, int t) {
  float o[8];
  values8(w, o);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = v[i] * rstd * o[i];
  if (a.y != nullptr) store8<VEC>(static_cast<T*>(a.y) + row * a.K + c, a.K - c, v);
  if (a.q != nullptr) {
    const float2 pairs[4] = {make_float2(v[0], v[1]), make_float2(v[2], v[3]), make_float2(v[4], v[5]), make_float2(v[6], v[7])};
    codes_of_pairs(a, pairs, row, c, t);
  }
}

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
    const float rstd = inverse_root(ss[0] / static_cast<float>(a.K) + a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 8 * (j * tpr + t);
      finish8<VEC, T>(a, w[j], v[j], rstd, row, c, t);
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
    const float rstd = inverse_root(s[0] / static_cast<float>(a.K) + a.eps);
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

// ------------------------------------------------------------------------------------------------ rows through shared memory
// A CTA takes up to `group` rows a turn.  Bulk copies keep a ring of `stages` turns full; `tpr` threads share the columns of a row, NV vectors each, and
// have R rows of a turn at once, so that what is done once a turn (shuffles, a barrier, roots, addresses) is spread over 32
// values a thread: what bounds these kernels next to HBM is the number of instructions a value.  us from a cold cache, and the floor at the rate of a plain copy:
// 16384 x 4096 with residual to codes 75.7 (72), 16384 x 2048 forward 40 (41: part of the result is still in L2), backward 44.5 (41).  With one vector of one row a
// thread 113, 49 and 85; with rows in registers and no ring 97, 42 and 74.  fp32, 16384 x 2048, forward, backward and the weight's sum 175 (164).
struct NormPlan {
  int threads, tpr, group, stages;
  long long ctas;
};
constexpr int kNormRing = 196 << 10;    // of all CTAs of an SM
template <class T, int NV> constexpr int kNormR = NV >= 4 ? 1 : (sizeof(T) == 4 ? 2 : 4) / NV;

// the ring: `tensors` of the sources, `group` rows of each a stage
template <int MOST, class T>
struct NormRows {
  uint32_t ring, bars;           // bars: full [8], empty [8]
  volatile int* abort_flag;
  const void* src[MOST];
  long long ld[MOST];
  long long rows;
  int tensors, K, group, stages;

  // one thread: the rows of a turn that begins at `row` into a stage, which every warp has read
  __device__ __forceinline__ void fetch(long long row, int stage) const {
    if (row >= rows) return;
    const uint32_t bytes = K * static_cast<int>(sizeof(T)), bar = bars + 8 * stage;
    const int n = static_cast<int>(min(static_cast<long long>(group), rows - row));
    mbar_arrive_expect_tx(bar, tensors * n * bytes);
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      if (i >= tensors) break;
      const T* from = static_cast<const T*>(src[i]) + row * ld[i];
      const uint32_t to = ring + (stage * tensors + i) * group * bytes;
      if (ld[i] == K) bulk_load_1d(to, from, n * bytes, bar);
      else
        for (int r = 0; r < n; ++r) bulk_load_1d(to + r * bytes, from + r * ld[i], bytes, bar);
    }
  }
  __device__ __forceinline__ void refill(long long row, int stage, uint32_t phase) const {
    if (row < rows && mbar_wait(bars + 64 + 8 * stage, phase, abort_flag, ST_WAIT_ROWS)) fetch(row, stage);
  }
  __device__ __forceinline__ void init(const NormPlan& p, uint8_t* smem, uint64_t* b, int* word) {
    ring = smem_u32(smem);
    bars = smem_u32(b);
    abort_flag = word;
    group = p.group;
    stages = p.stages;
    if (threadIdx.x == 0) {
      for (int s = 0; s < stages; ++s) {
        mbar_init(bars + 8 * s, 1);
        mbar_init(bars + 64 + 8 * s, p.threads >> 5);
      }
      *word = 0;
      fence_mbar_init();
    }
    __syncthreads();
  }
  __device__ __forceinline__ void wait(int stage, uint32_t phase) const { mbar_wait(bars + 8 * stage, phase, abort_flag, ST_WAIT_ROWS); }
  __device__ __forceinline__ void release(int stage) const {      // this warp has read the stage
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bars + 64 + 8 * stage);
  }
};
// two products or multiply-adds in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 twice(float a) { return make_float2(a, a); }
// eight values in pairs
template <class T>
__device__ __forceinline__ void pairs8(const Eight<T>& v, float2 (&f)[4]) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const uint32_t w[4] = {v.raw[0].x, v.raw[0].y, v.raw[0].z, v.raw[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(bf16_lo(w[i]), bf16_hi(w[i]));
  } else {
    float e[8];
    values8(v, e);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(e[2 * i], e[2 * i + 1]);
  }
}
template <class T>
__device__ __forceinline__ Eight<T> from_pairs8(const float2 (&f)[4]) {
  Eight<T> v;
  if constexpr (sizeof(T) == 4) {
    v.raw[0] = make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
    v.raw[1] = make_uint4(__float_as_uint(f[2].x), __float_as_uint(f[2].y), __float_as_uint(f[3].x), __float_as_uint(f[3].y));
  } else if constexpr (std::is_same_v<T, __half>) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __float22half2_rn(f[i]);
    memcpy(&v, h, 16);
  } else {
    v.raw[0] = make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y), pack_bf16x2(f[3].x, f[3].y));
  }
  return v;
}
template <class T>
__device__ __forceinline__ Eight<T> shared8(uint32_t at) {
  Eight<T> v;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(v.raw) / 16); ++i)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.raw[i].x), "=r"(v.raw[i].y), "=r"(v.raw[i].z), "=r"(v.raw[i].w)
                 : "r"(at + 16 * i)
                 : "memory");
  return v;
}
template <class T>
__device__ __forceinline__ Eight<T> zeros8() {
  Eight<T> v;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(v.raw) / 16); ++i) v.raw[i] = make_uint4(0u, 0u, 0u, 0u);
  return v;
}

// The sums of V values (a power of two) over a row's threads: value i ends up in lanes i * 32 / V ..., by halving first what the lanes exchange; rows
// of several warps by way of part[value][warp] and a barrier
template <int V>
__device__ __forceinline__ float turn_sums(float (&s)[V], float (*part)[16], int warps_row, int warp_row) {
  const int lane = threadIdx.x & 31;
  int off = 16;
#pragma unroll
  for (int n = V / 2; n >= 1; n >>= 1, off >>= 1) {
    const bool upper = (lane & off) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = upper ? s[i] : s[i + n], keep = upper ? s[i + n] : s[i];
      s[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
    }
  }
  constexpr int L = 32 / V;      // lanes of a value
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
  if (warps_row == 1) return s[0];
  const int value = lane / L, mine = lane % L;
  if (mine == 0) part[value][warp_row] = s[0];
  __syncthreads();
  float v = 0.0f;
  for (int w = mine; w < warps_row; w += L) v += part[value][w];
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// of a value of turn_sums, to all lanes
template <int V>
__device__ __forceinline__ float turn_value(float v, int i) { return __shfl_sync(0xffffffffu, v, i * (32 / V)); }

template <class T, class W, int NV>
__global__ void __launch_bounds__(512, 1) rms_norm_fwd_rows_kernel(const NormFwd a, const NormPlan p, int* status) {
  constexpr int R = kNormR<T, NV>, SIZE = static_cast<int>(sizeof(T));
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float part[2][8][R][16];
  __shared__ __align__(8) uint64_t bars[16];
  __shared__ int abort_word;
  NormRows<2, T> ring;
  ring.init(p, smem, bars, &abort_word);
  grid_dep_begin();
  ring.src[0] = a.x;
  ring.src[1] = a.residual;
  ring.ld[0] = a.ldx;
  ring.ld[1] = a.ldr;
  ring.tensors = a.residual != nullptr ? 2 : 1;
  ring.rows = a.rows;
  ring.K = a.K;
  const long long step = static_cast<long long>(gridDim.x) * p.group;
  long long first = static_cast<long long>(blockIdx.x) * p.group;
  if (threadIdx.x == 0)
    for (int s = 0; s < p.stages; ++s) ring.fetch(first + s * step, s);
  {
    const int g = threadIdx.x / p.tpr, t = threadIdx.x - g * p.tpr, groups = p.threads / p.tpr;
    const int warps_row = p.tpr >> 5, warp_row = t >> 5;
    const uint32_t row_bytes = a.K * SIZE, tensor_bytes = p.group * row_bytes, stage_bytes = ring.tensors * tensor_bytes;
    const bool add = a.residual != nullptr;
    float2 w[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 8 * (j * p.tpr + t);
      pairs8(load8<true>(static_cast<const W*>(a.w) + c, a.K - c), w[j]);
    }
    const uint32_t from = smem_u32(smem) + g * row_bytes + 8 * SIZE * t;
    int stage = 0, flip = 0;
    uint32_t phase = 0;
    for (; first < a.rows; first += step) {
      const int n = static_cast<int>(min(static_cast<long long>(p.group), a.rows - first));
      const long long at = (first + g) * a.K + 8 * t;
      ring.wait(stage, phase);
      float2 v[R][NV][4];
      float ss[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool live = g + r * groups < n;
        const uint32_t x = from + stage * stage_bytes + r * groups * row_bytes;
        float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const bool in = live && 8 * (j * p.tpr + t) < a.K;
          Eight<T> e = in ? shared8<T>(x + 8 * SIZE * j * p.tpr) : zeros8<T>();
          if (add && in) {
            float unused[8];
            sum8(e, shared8<T>(x + tensor_bytes + 8 * SIZE * j * p.tpr), e, unused);
            if (a.h != nullptr) put8(static_cast<T*>(a.h) + at + static_cast<long long>(r * groups) * a.K + 8 * j * p.tpr, 8, e);
          }
          pairs8(e, v[r][j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) s2 = fma2(v[r][j][i], v[r][j][i], s2);
        }
        ss[r] = s2.x + s2.y;
      }
      ring.release(stage);
      float mine = turn_sums<R>(ss, part[flip][g], warps_row, warp_row);
      if (threadIdx.x == 0) ring.refill(first + p.stages * step, stage, phase);
      mine = inverse_root(mine / static_cast<float>(a.K) + a.eps);
      flip ^= 1;
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float2 rstd = twice(turn_value<R>(mine, r));
        if (g + r * groups >= n) break;
        const long long row = first + g + r * groups;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int c = 8 * (j * p.tpr + t);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[r][j][i] = mul2(mul2(v[r][j][i], rstd), w[j][i]);
          if (a.y != nullptr) put8(static_cast<T*>(a.y) + row * a.K + c, a.K - c, from_pairs8<T>(v[r][j]));
          if (a.q != nullptr) codes_of_pairs(a, v[r][j], row, c, t);
        }
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && abort_word != 0) *status = abort_word;
}

template <class T, class W, int NV>
__global__ void __launch_bounds__(512, 1) rms_norm_bwd_rows_kernel(const NormBwd a, const NormPlan p, int* status) {
  constexpr int R = kNormR<T, NV>, SIZE = static_cast<int>(sizeof(T));
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float part[2][8][2 * R][16];
  __shared__ __align__(8) uint64_t bars[16];
  __shared__ int abort_word;
  NormRows<3, T> ring;
  ring.init(p, smem, bars, &abort_word);
  grid_dep_begin();
  ring.src[0] = a.h;
  ring.src[1] = a.gy;
  ring.src[2] = a.gh;
  ring.ld[0] = a.ldh;
  ring.ld[1] = ring.ld[2] = a.K;
  ring.tensors = a.gh != nullptr ? 3 : 2;
  ring.rows = a.rows;
  ring.K = a.K;
  const long long step = static_cast<long long>(gridDim.x) * p.group;
  long long first = static_cast<long long>(blockIdx.x) * p.group;
  const int g = threadIdx.x / p.tpr, t = threadIdx.x - g * p.tpr, groups = p.threads / p.tpr;
  float2 acc[NV][4];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = make_float2(0.0f, 0.0f);
  if (threadIdx.x == 0)
    for (int s = 0; s < p.stages; ++s) ring.fetch(first + s * step, s);
  {
    const int warps_row = p.tpr >> 5, warp_row = t >> 5;
    const uint32_t row_bytes = a.K * SIZE, tensor_bytes = p.group * row_bytes, stage_bytes = ring.tensors * tensor_bytes;
    const bool add = a.gh != nullptr;
    float2 w[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 8 * (j * p.tpr + t);
      pairs8(load8<true>(static_cast<const W*>(a.w) + c, a.K - c), w[j]);
    }
    const uint32_t from = smem_u32(smem) + g * row_bytes + 8 * SIZE * t;
    int stage = 0, flip = 0, before = -1;      // before: the stage of the turn before
    uint32_t phase = 0, before_phase = 0;
    for (; first < a.rows; first += step) {
      const int n = static_cast<int>(min(static_cast<long long>(p.group), a.rows - first));
      ring.wait(stage, phase);
      float s[2 * R];                  // of h^2 and of h d
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool live = g + r * groups < n;
        const uint32_t x = from + stage * stage_bytes + r * groups * row_bytes;
        float2 s2 = make_float2(0.0f, 0.0f), d2 = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const bool in = live && 8 * (j * p.tpr + t) < a.K;
          float2 hf[4], gf[4];
          pairs8(in ? shared8<T>(x + 8 * SIZE * j * p.tpr) : zeros8<T>(), hf);
          pairs8(in ? shared8<T>(x + tensor_bytes + 8 * SIZE * j * p.tpr) : zeros8<T>(), gf);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s2 = fma2(hf[i], hf[i], s2);
            d2 = fma2(mul2(gf[i], w[j][i]), hf[i], d2);
          }
        }
        s[2 * r] = s2.x + s2.y;
        s[2 * r + 1] = d2.x + d2.y;
      }
      const float mine = turn_sums<2 * R>(s, part[flip][g], warps_row, warp_row) / static_cast<float>(a.K);
      if (threadIdx.x == 0 && before >= 0 && p.stages > 1) ring.refill(first + (p.stages - 1) * step, before, before_phase);
      const float other = __shfl_xor_sync(0xffffffffu, mine, 32 / (2 * R));
      // in a row's first lanes: rstd, and what n is multiplied with, -rstd mean(d n)
      const float root = inverse_root(mine + a.eps), slope = -root * (root * other);
      flip ^= 1;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float2 rstd = twice(turn_value<2 * R>(root, 2 * r)), back = twice(turn_value<2 * R>(slope, 2 * r));
        if (g + r * groups >= n) break;
        const uint32_t x = from + stage * stage_bytes + r * groups * row_bytes;
        const long long row = first + g + r * groups;
#pragma unroll
        for (int j = 0; j < NV; ++j) {       // read a second time, which takes fewer registers
          const int c = 8 * (j * p.tpr + t);
          if (c >= a.K) break;
          float2 hf[4], gf[4], of[4];
          pairs8(shared8<T>(x + 8 * SIZE * j * p.tpr), hf);
          pairs8(shared8<T>(x + tensor_bytes + 8 * SIZE * j * p.tpr), gf);
          pairs8(add ? shared8<T>(x + 2 * tensor_bytes + 8 * SIZE * j * p.tpr) : zeros8<T>(), of);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 m = mul2(hf[i], rstd);
            acc[j][i] = fma2(gf[i], m, acc[j][i]);
            of[i] = fma2(mul2(gf[i], w[j][i]), rstd, fma2(m, back, of[i]));
          }
          if (a.gx != nullptr) put8(static_cast<T*>(a.gx) + row * a.K + c, a.K - c, from_pairs8<T>(of));
        }
      }
      ring.release(stage);
      if (threadIdx.x == 0 && p.stages == 1) ring.refill(first + step, 0, phase);
      before = stage;
      before_phase = phase;
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && abort_word != 0) *status = abort_word;
  if (a.part == nullptr) return;
  // the groups' sums one after another, in the ring: all copies have arrived
  float* sum = reinterpret_cast<float*>(smem);
  for (int u = 0; u < groups; ++u) {
    if (g == u) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = 8 * (j * p.tpr + t);
        if (c >= a.K) continue;
        float4* to = reinterpret_cast<float4*>(u + 1 < groups ? sum + c : a.part + static_cast<long long>(blockIdx.x) * a.K + c);
        const float4* old = reinterpret_cast<const float4*>(sum + c);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float4 v = make_float4(acc[j][2 * i].x, acc[j][2 * i].y, acc[j][2 * i + 1].x, acc[j][2 * i + 1].y);
          if (u > 0) {
            const float4 o = old[i];
            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
          }
          to[i] = v;
        }
      }
    }
    __syncthreads();
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
// `sms`: gemm_cta_budget() of the call, since these grids stay until their rows are done and SMs reserved for an exchange are not theirs.  The workspace of the
// weight's gradient is sized for num_sms().
static int64_t norm_ctas(int64_t rows, int rows_cta, int threads, int threads_sm, int sms) {
  return std::max<int64_t>(1, std::min<int64_t>((rows + rows_cta - 1) / rows_cta, static_cast<int64_t>(sms) * (threads_sm / threads)));
}

// Threads, rows a turn and turns in the ring for rows through shared memory: a vector of a row a thread up to 2048 values, two up to 4096, else four; as many
// CTAs an SM as have two turns in the ring and 512 threads between them
static int rows_nv(int64_t K) { return K <= 2048 ? 1 : K <= 4096 ? 2 : 4; }
static NormPlan norm_plan(int64_t rows, int64_t K, int64_t row_bytes, int size, int sms) {
  const int nv = rows_nv(K), r = nv >= 4 ? 1 : (size == 4 ? 2 : 4) / nv;      // kNormR
  NormPlan p;
  p.tpr = row_threads(K, nv);
  const int groups = std::max(1, 256 / p.tpr);
  p.threads = p.tpr * groups;
  p.group = groups * r;
  int ctas = std::max(1, 512 / p.threads);
  while (p.group > 1 && p.group * static_cast<int64_t>(ctas) * sms > rows) p.group = (p.group + 1) / 2;
  while (ctas > 1 && 2 * p.group * row_bytes * ctas > kNormRing) --ctas;
  p.stages = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, kNormRing / ctas / (p.group * row_bytes))));
  p.ctas = std::max<int64_t>(1, std::min<int64_t>((rows + p.group - 1) / p.group, static_cast<int64_t>(ctas) * sms));
  return p;
}
template <class F>
static int by_rows_nv(int64_t K, F f) {
  const int nv = rows_nv(K);
  return nv == 1 ? f(std::integral_constant<int, 1>()) : nv == 2 ? f(std::integral_constant<int, 2>()) : f(std::integral_constant<int, 4>());
}
// of the backward through registers
static int bwd_threads(int64_t K) { return K <= 512 ? 256 : row_threads(K, K > 8192 ? 4 : 2); }
static int64_t bwd_ctas(int64_t rows, int64_t K, int sms) {
  const int threads = bwd_threads(K);
  return norm_ctas(rows, K <= 512 ? 8 : 1, threads, std::max(512, threads), sms);
}

}  // namespace b200moe

using namespace b200moe;

static int check_norm(const char* who, int type, int w_type, int64_t rows, int64_t K, float eps) {
  B200_CHECK_ARG(known_logits(type) && same_or_f32(type, w_type), B200MOE_E_UNSUPPORTED, "%s: rows of type %d with a weight of type %d", who, type,
                 w_type);
  B200_CHECK_ARG(rows >= 0 && rows < (1LL << 31) - 256, B200MOE_E_BAD_SHAPE, "%s: %lld rows", who, (long long)rows);
  B200_CHECK_ARG(K >= 1 && K <= kNormMaxK, B200MOE_E_BAD_SHAPE, "%s: rows of %lld values, supported 1..%d", who, (long long)K, kNormMaxK);
  B200_CHECK_ARG(eps >= 0.0f && eps <= std::numeric_limits<float>::max(), B200MOE_E_BAD_SHAPE, "%s: eps = %g must be finite and not negative", who, (double)eps);
  return 0;
}

extern "C" {

int b200moe_rms_norm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, int type, const void* weight, int weight_type, int64_t rows,
                         int64_t K, float eps, void* y, void* h, void* q, float* scale, int64_t scale_pitch_, int32_t* status,
                         b200moe_stream_t stream) {
  const int rc = check_norm("rms_norm_fwd", type, weight_type, rows, K, eps);
  if (rc) return rc;
  B200_CHECK_ARG(ldx >= K && (residual == nullptr || ldr >= K), B200MOE_E_BAD_SHAPE, "rms_norm_fwd: rows %lld and %lld apart, shorter than K = %lld",
                 (long long)ldx, (long long)ldr, (long long)K);
  B200_CHECK_ARG(q == nullptr || (K % 8 == 0 && scale_pitch_ >= rows), B200MOE_E_BAD_SHAPE,
                 "rms_norm_fwd: codes of K = %lld (a multiple of 8), scales %lld apart", (long long)K, (long long)scale_pitch_);
  if (rows == 0) return 0;
  B200_CHECK_ARG(x && weight && status && (y || h || q) && (q == nullptr || scale) && (h == nullptr || residual), B200MOE_E_NULL, "rms_norm_fwd: null pointer");
  B200_CHECK_ARG(reinterpret_cast<uintptr_t>(q) % 8 == 0, B200MOE_E_ALIGN, "rms_norm_fwd: q must be 8-byte aligned");
  const bool vec = K % 8 == 0 && vectors(x, ldx, type) && (residual == nullptr || vectors(residual, ldr, type)) && aligned16(weight) &&
                   (y == nullptr || vectors(y, K, type)) && (h == nullptr || vectors(h, K, type));
  const NormFwd a{x, residual, weight, ldx, ldr, y, h, static_cast<uint8_t*>(q), scale, scale_pitch_, rows, static_cast<int>(K), eps};
  const int sms = gemm_cta_budget();
  OpScope scope("rms_norm_fwd", 1);
  return by_types(type, weight_type, [&](auto t, auto w) -> int {
    using T = decltype(t);
    using W = decltype(w);
    auto run = [&](auto kernel, int rows_cta, int threads) -> int {
      B200_LAUNCH(kernel, static_cast<int>(norm_ctas(rows, rows_cta, threads, 1024, sms)), threads, 0, stream, a);
      return 0;
    };
    auto run_rows = [&](auto nv) -> int {
      constexpr int NV = decltype(nv)::value;
      static PerDevice allowed;
      B200_CUDA(allow_smem(allowed, rms_norm_fwd_rows_kernel<T, W, NV>, kNormRing));
      const int64_t row_bytes = K * static_cast<int64_t>(sizeof(T)) * (residual != nullptr ? 2 : 1);
      const NormPlan p = norm_plan(rows, K, row_bytes, type_bytes(type), sms);
      B200_LAUNCH((rms_norm_fwd_rows_kernel<T, W, NV>), static_cast<int>(p.ctas), p.threads, p.stages * p.group * row_bytes, stream, a, p, status);
      return 0;
    };
    if (rows <= num_sms() && K > 256 && K <= 8192)
      return vec ? run(rms_norm_fwd_kernel<T, W, 1, true, false, 1024>, 1, row_threads(K, 1))
                 : run(rms_norm_fwd_kernel<T, W, 1, false, false, 1024>, 1, row_threads(K, 1));
    if (vec) return by_rows_nv(K, run_rows);
    return K <= 1024 ? run(rms_norm_fwd_kernel<T, W, 4, false, true, 256>, 8, 256) : run(rms_norm_fwd_kernel<T, W, 4, false, false, 512>, 1, row_threads(K, 4));
  });
}

size_t b200moe_rms_norm_bwd_ws_bytes(int64_t rows, int64_t K) {
  if (rows <= 0 || K < 1 || K > kNormMaxK) return 0;
  return static_cast<size_t>(std::max(bwd_ctas(rows, K, num_sms()), static_cast<int64_t>(8) * num_sms())) * K * sizeof(float);
}

int b200moe_rms_norm_bwd(const void* grad_y, const void* grad_h, const void* h, int64_t ldh, int type, const void* weight, int weight_type, int64_t rows,
                         int64_t K, float eps, void* ws, void* grad_x, void* grad_weight, int32_t* status, b200moe_stream_t stream) {
  const int rc = check_norm("rms_norm_bwd", type, weight_type, rows, K, eps);
  if (rc) return rc;
  B200_CHECK_ARG(ldh >= K, B200MOE_E_BAD_SHAPE, "rms_norm_bwd: rows of h %lld apart, K = %lld", (long long)ldh, (long long)K);
  if (rows == 0 && grad_weight == nullptr) return 0;
  B200_CHECK_ARG((rows == 0 || (grad_y && h && weight && status)) && (grad_x || grad_weight), B200MOE_E_NULL, "rms_norm_bwd: null pointer");
  B200_CHECK_ARG(rows == 0 || grad_weight == nullptr || ws, B200MOE_E_NULL, "rms_norm_bwd: no workspace for the weight's gradient");
  B200_CHECK_ARG(aligned16(ws), B200MOE_E_ALIGN, "rms_norm_bwd: the workspace must be 16-byte aligned");
  const bool vec = K % 8 == 0 && vectors(grad_y, K, type) && vectors(h, ldh, type) && aligned16(weight) &&
                   (grad_h == nullptr || vectors(grad_h, K, type)) && (grad_x == nullptr || vectors(grad_x, K, type));
  const NormBwd a{grad_y, grad_h, h, weight, ldh, grad_x, grad_weight != nullptr ? static_cast<float*>(ws) : nullptr, rows, static_cast<int>(K), eps};
  const int64_t row_bytes = K * type_bytes(type) * (grad_h != nullptr ? 3 : 2);
  const int sms = gemm_cta_budget();
  const NormPlan p = norm_plan(rows, K, row_bytes, type_bytes(type), sms);
  const int64_t ctas = rows == 0 ? 0 : vec ? p.ctas : bwd_ctas(rows, K, sms);
  OpScope scope("rms_norm_bwd", (rows > 0) + (grad_weight != nullptr));
  return by_types(type, weight_type, [&](auto t, auto w) -> int {
    using T = decltype(t);
    using W = decltype(w);
    auto run = [&](auto kernel) -> int {
      B200_LAUNCH(kernel, static_cast<int>(ctas), bwd_threads(K), 0, stream, a);
      return 0;
    };
    auto run_rows = [&](auto nv) -> int {
      constexpr int NV = decltype(nv)::value;
      static PerDevice allowed;
      B200_CUDA(allow_smem(allowed, rms_norm_bwd_rows_kernel<T, W, NV>, kNormRing));
      B200_LAUNCH((rms_norm_bwd_rows_kernel<T, W, NV>), static_cast<int>(ctas), p.threads, p.stages * p.group * row_bytes, stream, a, p, status);
      return 0;
    };
    if (rows > 0) {
      const int rc2 = vec ? by_rows_nv(K, run_rows)
                      : K <= 512 ? run(rms_norm_bwd_kernel<T, W, 2, false, true, 256>)
                      : K <= 8192 ? run(rms_norm_bwd_kernel<T, W, 2, false, false, 512>) : run(rms_norm_bwd_kernel<T, W, 4, false, false, 512>);
      if (rc2) return rc2;
    }
    if (grad_weight != nullptr)
      B200_LAUNCH(norm_weight_grad_kernel<W>, static_cast<int>((K + 31) / 32), 1024, 0, stream, static_cast<const float*>(ws), static_cast<int>(ctas),
                  static_cast<int>(K), static_cast<W*>(grad_weight));
    return 0;
  });
}

}  // extern "C"

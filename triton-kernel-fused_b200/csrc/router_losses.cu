// Losses of a router and their gradient: the balance loss over the experts and the z loss, with the gradient of the logits.
//
//   p = softmax(z), or sigmoid(z) / sum sigmoid(z);  over the n tokens of a segment (the batch, or each sequence)
//   f_e = E / (k n) * picks of e,  P_e = 1/n sum p_e;  balance = sum_e f_e P_e, averaged over the segments that have tokens
//   z loss = mean over all tokens of lse^2, lse = log sum exp z
//   dz = g_b / (live n) p (f - <f, p>) [(1 - s) for sigmoid scores] + g_z 2 lse softmax(z) / N
//
// A token counts unless its mask is 0 or all its logits are -inf; one that does not count has zero gradient.  f counts picks, so it has
// no gradient.  Bound: at small batches the launches, at large ones the issue of instructions, 349 a token forward and 364 backward at 256 experts
// (a warp's exponentials and its sums over the lanes), which take 69 % of the cycles: 32 768 tokens in bf16 22.7 us forward, 16 backward, where the bytes
// take 2.9 and 5.1.  Sums:
// a warp's tokens in registers, a CTA's warps in shared memory, the CTAs' in order in a second kernel (a batch that one CTA
// takes needs none): no atomics on floats, so the same bits every time.
#include <algorithm>

#include "logits.cuh"
#include "ptx.cuh"

namespace b200moe {

constexpr int kLossWarps = 32;

struct LossParams {
  const void* logits;
  const long long* idx;     // (rows, k)
  const uint8_t* mask;      // (rows), nullable
  long long S;              // rows of a segment
  int segs, E, k, vec, sigmoid;
  int blocks;               // CTAs of a segment
  // per (segment, CTA): sums of p (E), then [sum lse^2, tokens] as doubles, and picks (E)
  float* part_p;
  int* part_hits;
  double* part_z;
  float* coef;              // (segs, E): f / n, then [1 / live segments, 1 / N]
  double* seg_out;          // per segment: balance, sum lse^2, tokens
  float *balance, *z;       // the two losses
  int* status;
};

// p of a lane's experts, lse, and whether the token counts; soft: softmax(z), SIGMOID only (else it is p)
template <bool SIGMOID, int V>
__device__ __forceinline__ bool loss_row(const float (&z)[V], int live, float (&p)[V], float (&soft)[V], float& lse) {
  float m = z[0];
#pragma unroll
  for (int i = 1; i < V; ++i) m = fmaxf(m, z[i]);
  m = warp_max(m);
  bool nan = false;        // fmaxf passes over NaN
#pragma unroll
  for (int i = 0; i < V; ++i) nan = nan || z[i] != z[i];
  if (m == -INFINITY && !__any_sync(0xffffffffu, nan)) {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = soft[i] = 0.0f;
    lse = 0.0f;
    return false;
  }
  float sum = 0.0f, ssum = 0.0f;
  const float below = fminf(m, 0.0f);     // rows far below zero: every sigmoid times exp(-m), which leaves p as it is
#pragma unroll
  for (int i = 0; i < V; ++i) {
    soft[i] = i < live ? expf(z[i] - m) : 0.0f;
    sum += soft[i];
    if constexpr (SIGMOID) {
      p[i] = i >= live ? 0.0f : below < 0.0f ? expf(z[i] - below) / (1.0f + expf(z[i])) : 1.0f / (1.0f + expf(-z[i]));
      ssum += p[i];
    }
  }
  sum = warp_sum(sum);
  lse = m + logf(sum);
  const float inv = 1.0f / sum;
  if constexpr (SIGMOID) ssum = 1.0f / warp_sum(ssum);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    soft[i] *= inv;
    p[i] = SIGMOID ? p[i] * ssum : soft[i];
  }
  return true;
}

// One segment's f, coefficients and balance from its sums, by one CTA.  n: its tokens; P(e), hits(e): its sums
template <class FP, class FH>
__device__ __forceinline__ double segment_balance(const LossParams& p, int seg, double n, double* red, FP P, FH hits) {
  double acc = 0.0;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    const double f = n > 0.0 ? static_cast<double>(p.E) * hits(e) / (p.k * n) : 0.0;
    const double c = n > 0.0 ? f / n : 0.0;
    p.coef[static_cast<long long>(seg) * p.E + e] = static_cast<float>(c);
    acc += c * P(e);
  }
  acc = warp_sum(acc);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) total += red[i];
  __syncthreads();
  return total;
}
__device__ __forceinline__ void put_losses(const LossParams& p, double balance, double z, double n, double live) {
  float* scalars = p.coef + static_cast<long long>(p.segs) * p.E;
  scalars[0] = live > 0.0 ? static_cast<float>(1.0 / live) : 0.0f;
  scalars[1] = n > 0.0 ? static_cast<float>(1.0 / n) : 0.0f;
  *p.balance = live > 0.0 ? static_cast<float>(balance / live) : 0.0f;
  *p.z = n > 0.0 ? static_cast<float>(z / n) : 0.0f;
}

template <class T, bool SIGMOID, int V>
__global__ void __launch_bounds__(32 * kLossWarps, 1)
router_losses_kernel(const LossParams p) {
  grid_dep_begin();
  __shared__ float sum_s[kLossWarps][32 * V];
  __shared__ int hist[32 * V];
  __shared__ double z_s[kLossWarps], n_s[kLossWarps], red[kLossWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = lane * V, live = max(0, min(V, p.E - first));
  const int seg = blockIdx.y;
  for (int e = threadIdx.x; e < 32 * V; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  float P[V];
  double z2 = 0.0;
  long long n = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) P[i] = 0.0f;
  // of 32 768 tokens each warp has 7, one after the other (logits fetched while the token before is summed gave nothing at 32 warps an SM: 23.6 us
  // against 22.7 in bf16, 22.9 against 22.8 in fp32)
  const long long step = static_cast<long long>(gridDim.x) * kLossWarps;
  for (long long r = static_cast<long long>(blockIdx.x) * kLossWarps + warp; r < p.S; r += step) {
    const long long t = seg * p.S + r;
    if (p.mask != nullptr && p.mask[t] == 0) continue;
    float z[V], pr[V], soft[V], lse;
    load_values<T, V>(reinterpret_cast<const T*>(p.logits) + t * p.E + (live > 0 ? first : 0), live, p.vec, z);
    const long long e = lane < p.k ? p.idx[t * p.k + lane] : 0;
    if (!loss_row<SIGMOID, V>(z, live, pr, soft, lse)) continue;
    if (lane < p.k) {
      if (e >= 0 && e < p.E) atomicAdd(&hist[e], 1);
      else if (p.status != nullptr) atomicCAS(p.status, 0, ST_BAD_EXPERT_INDEX);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) P[i] += pr[i];
    z2 += static_cast<double>(lse) * lse;
    ++n;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) sum_s[warp][first + i] = P[i];
  if (lane == 0) {
    z_s[warp] = z2;
    n_s[warp] = static_cast<double>(n);
  }
  __syncthreads();
  const long long at = static_cast<long long>(seg) * p.blocks + blockIdx.x;
  double zt = 0.0, nt = 0.0;
  for (int i = 0; i < kLossWarps; ++i) {
    zt += z_s[i];
    nt += n_s[i];
  }
  auto column = [&](int e) {
    float s = 0.0f;
    for (int i = 0; i < kLossWarps; ++i) s += sum_s[i][e];
    return s;
  };
  if (p.blocks == 1 && p.segs == 1) {      // nothing to wait for
    const double b = segment_balance(p, 0, nt, red, column, [&](int e) { return hist[e]; });
    if (threadIdx.x == 0) put_losses(p, b, zt, nt, nt > 0.0 ? 1.0 : 0.0);
    return;
  }
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    p.part_p[at * p.E + e] = column(e);
    p.part_hits[at * p.E + e] = hist[e];
  }
  if (threadIdx.x == 0) {
    p.part_z[2 * at] = zt;
    p.part_z[2 * at + 1] = nt;
  }
}

// the CTAs' sums of each segment, in order; 1024 threads, `parts` of them a column
__global__ void __launch_bounds__(1024)
router_losses_segments_kernel(const LossParams p) {
  grid_dep_begin();
  __shared__ double part[1024], red[32], zn[2];
  __shared__ int hits[1024];
  const int parts = 1024 / p.E, c = threadIdx.x / p.E, e = threadIdx.x - c * p.E;
  for (int seg = blockIdx.x; seg < p.segs; seg += gridDim.x) {
    const long long at = static_cast<long long>(seg) * p.blocks;
    double s = 0.0;
    int h = 0;
    if (c < parts) {
#pragma unroll 8
      for (int b = c; b < p.blocks; b += parts) {
        s += p.part_p[(at + b) * p.E + e];
        h += p.part_hits[(at + b) * p.E + e];
      }
    }
    part[threadIdx.x] = s;
    hits[threadIdx.x] = h;
    if (threadIdx.x < 64) {      // warp 0: lse^2, warp 1: tokens
      const int w = threadIdx.x >> 5;
      double v = 0.0;
      for (int b = threadIdx.x & 31; b < p.blocks; b += 32) v += p.part_z[2 * (at + b) + w];
      v = warp_sum(v);
      if ((threadIdx.x & 31) == 0) zn[w] = v;
    }
    __syncthreads();
    const double z = zn[0], n = zn[1];
    const double b = segment_balance(
        p, seg, n, red,
        [&](int x) {
          double v = 0.0;
          for (int i = 0; i < parts; ++i) v += part[i * p.E + x];
          return v;
        },
        [&](int x) {
          int v = 0;
          for (int i = 0; i < parts; ++i) v += hits[i * p.E + x];
          return v;
        });
    if (threadIdx.x == 0) {
      if (p.segs == 1) {
        put_losses(p, b, z, n, n > 0.0 ? 1.0 : 0.0);
      } else {
        p.seg_out[3 * seg] = b;
        p.seg_out[3 * seg + 1] = z;
        p.seg_out[3 * seg + 2] = n;
      }
    }
    __syncthreads();
  }
}

// the segments' results, in order: one CTA
__global__ void __launch_bounds__(256)
router_losses_total_kernel(const LossParams p) {
  grid_dep_begin();
  __shared__ double red[4][8];
  double v[4] = {0.0, 0.0, 0.0, 0.0};      // balance, lse^2, tokens, segments that have some
  for (int s = threadIdx.x; s < p.segs; s += 256) {
    v[0] += p.seg_out[3 * s];
    v[1] += p.seg_out[3 * s + 1];
    v[2] += p.seg_out[3 * s + 2];
    v[3] += p.seg_out[3 * s + 2] > 0.0 ? 1.0 : 0.0;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = warp_sum(v[i]);
    if ((threadIdx.x & 31) == 0) red[i][threadIdx.x >> 5] = v[i];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      v[i] = 0.0;
      for (int w = 0; w < 8; ++w) v[i] += red[i][w];
    }
    put_losses(p, v[0], v[1], v[2], v[3]);
  }
}

template <class T, bool SIGMOID, int V>
__global__ void __launch_bounds__(256)
router_losses_bwd_kernel(const T* logits, const uint8_t* mask, const float* coef, const float* grad_balance, const float* grad_z,
                         long long rows, long long S, int segs, int E, int vec, T* grad) {
  grid_dep_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = lane * V, live = max(0, min(V, E - first));
  const float* scalars = coef + static_cast<long long>(segs) * E;
  const float gb = grad_balance != nullptr ? *grad_balance * scalars[0] : 0.0f;
  const float gz = grad_z != nullptr ? 2.0f * *grad_z * scalars[1] : 0.0f;
  long long have = -1;
  float f[V];
  for (long long t = static_cast<long long>(blockIdx.x) * 8 + warp; t < rows; t += static_cast<long long>(gridDim.x) * 8) {
    float z[V], p[V], soft[V], d[V], lse = 0.0f;
    bool counts = mask == nullptr || mask[t] != 0;
    if (counts) {
      load_values<T, V>(logits + t * E + (live > 0 ? first : 0), live, vec, z);
      counts = loss_row<SIGMOID, V>(z, live, p, soft, lse);
    }
    if (counts) {
      const long long seg = segs == 1 ? 0 : t / S;
      if (seg != have) {
        have = seg;
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = i < live ? coef[seg * E + first + i] : 0.0f;
      }
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) dot += f[i] * p[i];
      dot = warp_sum(dot);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] = gb * p[i] * (f[i] - dot);
        if constexpr (SIGMOID) d[i] *= 1.0f / (1.0f + expf(z[i]));
        d[i] += gz * lse * soft[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = 0.0f;
    }
    if (live > 0) store_values<T, V>(grad + t * E + first, live, vec, d);
  }
}

// CTAs of a segment: four tokens a warp at least, all segments together one wave.  (512 tokens of 8 experts, forward and backward: four CTAs and
// a second kernel 13.6 us, one CTA for all 19.4.)
static int loss_blocks(int64_t S, int segs) {
  const int64_t most = std::max<int64_t>(1, num_sms() / segs);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((S + 4 * kLossWarps - 1) / (4 * kLossWarps), most)));
}

}  // namespace b200moe

using namespace b200moe;

#define CHECK_LOSSES(name)                                                                                                             \
  B200_CHECK_ARG(known_logits(logits_type), B200MOE_E_UNSUPPORTED, name ": unknown type %d of the logits", logits_type);               \
  B200_CHECK_ARG(E >= 1 && E <= B200MOE_MAX_EXPERTS, B200MOE_E_UNSUPPORTED, name ": E = %d, supported 1..%d", E, B200MOE_MAX_EXPERTS); \
  B200_CHECK_ARG(segs >= 1 && segs <= 65535 && S >= 0, B200MOE_E_BAD_SHAPE, name ": %d segments (1..65535) of %lld tokens", segs,      \
                 (long long)S);                                                                                                        \
  B200_CHECK_ARG(scoring == B200MOE_SIGMOID || scoring == B200MOE_SOFTMAX, B200MOE_E_UNSUPPORTED, name ": unknown scoring %d", scoring)

extern "C" {

size_t b200moe_router_losses_ws_bytes(int64_t S, int segs, int E) {
  if (S < 0 || segs < 1 || E < 1) return 0;
  const size_t n = static_cast<size_t>(loss_blocks(S, segs)) * segs;
  return n * (16 + 8 * static_cast<size_t>(E)) + 24 * static_cast<size_t>(segs);
}

int b200moe_router_losses_fwd(const void* logits, int logits_type, const int64_t* idx, const uint8_t* mask, int64_t S, int segs, int E, int k,
                              int scoring, void* ws, float* coef, float* balance, float* z, int32_t* status, b200moe_stream_t stream) {
  B200_CHECK_ARG(ws && coef && balance && z && (S == 0 || (logits && idx)), B200MOE_E_NULL, "router_losses_fwd: null pointer");
  CHECK_LOSSES("router_losses_fwd");
  B200_CHECK_ARG(k >= 1 && k <= B200MOE_MAX_TOPK, B200MOE_E_BAD_SHAPE, "router_losses_fwd: top_k = %d, supported 1..%d", k, B200MOE_MAX_TOPK);
  LossParams p{};
  p.logits = logits; p.idx = reinterpret_cast<const long long*>(idx); p.mask = mask; p.S = S; p.segs = segs; p.E = E; p.k = k;
  p.sigmoid = scoring == B200MOE_SIGMOID; p.blocks = loss_blocks(S, segs);
  const long long n = static_cast<long long>(p.blocks) * segs;
  p.part_z = reinterpret_cast<double*>(ws);
  p.seg_out = p.part_z + 2 * n;
  p.part_p = reinterpret_cast<float*>(p.seg_out + 3 * static_cast<long long>(segs));
  p.part_hits = reinterpret_cast<int*>(p.part_p + n * E);
  p.coef = coef; p.balance = balance; p.z = z; p.status = status;
  OpScope scope("router_losses_fwd", p.blocks == 1 && segs == 1 ? 1 : segs == 1 ? 2 : 3);
  cudaError_t err = cudaSuccess;
  by_values((E + 31) / 32, [&](auto v) {
    constexpr int V = v.value;
    if constexpr (V <= 8) {
      p.vec = E % V == 0 && reinterpret_cast<uintptr_t>(logits) % std::min(16, V * type_bytes(logits_type)) == 0;
      by_logits(logits_type, [&](auto type) {
        using T = decltype(type);
        err = launch_chained(p.sigmoid ? router_losses_kernel<T, true, V> : router_losses_kernel<T, false, V>, dim3(p.blocks, segs),
                             32 * kLossWarps, 0, (cudaStream_t)stream, 1, p);
      });
    }
  });
  B200_CUDA(err);
  if (p.blocks == 1 && segs == 1) return 0;
  B200_LAUNCH(router_losses_segments_kernel, std::min(segs, num_sms()), 1024, 0, stream, p);
  if (segs > 1) B200_LAUNCH(router_losses_total_kernel, 1, 256, 0, stream, p);
  return 0;
}

int b200moe_router_losses_bwd(const void* logits, int logits_type, const uint8_t* mask, const float* coef, const float* grad_balance,
                              const float* grad_z, int64_t S, int segs, int E, int scoring, void* grad_logits, b200moe_stream_t stream) {
  B200_CHECK_ARG(coef && (S == 0 || (logits && grad_logits)), B200MOE_E_NULL, "router_losses_bwd: null pointer");
  CHECK_LOSSES("router_losses_bwd");
  const int64_t rows = S * segs;
  if (rows == 0) return 0;
  const int grid = static_cast<int>(std::min<int64_t>((rows + 7) / 8, static_cast<int64_t>(num_sms()) * 8));
  OpScope scope("router_losses_bwd", 1);
  cudaError_t err = cudaSuccess;
  by_values((E + 31) / 32, [&](auto v) {
    constexpr int V = v.value;
    if constexpr (V <= 8) {
      const int bytes = std::min(16, V * type_bytes(logits_type));
      const int vec = E % V == 0 && reinterpret_cast<uintptr_t>(logits) % bytes == 0 && reinterpret_cast<uintptr_t>(grad_logits) % bytes == 0;
      by_logits(logits_type, [&](auto type) {
        using T = decltype(type);
        err = launch_chained(scoring == B200MOE_SIGMOID ? router_losses_bwd_kernel<T, true, V> : router_losses_bwd_kernel<T, false, V>, grid,
                             256, 0, (cudaStream_t)stream, 1, reinterpret_cast<const T*>(logits), mask, coef, grad_balance, grad_z,
                             static_cast<long long>(rows), static_cast<long long>(S), segs, E, vec, reinterpret_cast<T*>(grad_logits));
      });
    }
  });
  B200_CUDA(err);
  return 0;
}

}  // extern "C"

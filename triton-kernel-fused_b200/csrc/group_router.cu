// Group-limited top-k routing: softmax or sigmoid scores, a selection bias, the best groups of experts, the best experts of those,
// renormalised weights; and the gradient of the weights.
//
//   s = sigmoid(z) or softmax(z);  v = s + b;  a group's value = its largest v, or the sum of its two largest;  the `open` groups of
//   largest value;  the k largest v inside them, equal values to the lowest index;  w = s / (sum s + 1e-20) * scale
//
// A pick is a comparison of real numbers, and two of 256 experts are often closer than fp32 resolves (32 768 tokens, 8 of 256: some
// hundred picks a step), so which one an fp32 kernel takes is left to its rounding.  Here the picks are those of the real numbers:
// without a bias s rises with z, and z itself is compared; with one, values closer than the error of the fp32 ones (kNear) are
// computed again in 64 bits and compared there, unless logit and bias are the same, which is a tie.
//
// One warp a token.  A lane holds V neighbouring experts of one group (groups own lanes, so a group's value is a reduction over
// neighbouring lanes).  Instead of k dependent rounds of argmax: the k-th largest of the lanes' maxima bounds the k-th largest value
// from below, so the experts above it, ten or so, are all that can be picked; they are collected in shared memory, and
// each lane counts how many of them are larger than its own.
#include <algorithm>

#include "logits.cuh"
#include "ptx.cuh"

namespace b200moe {

constexpr int kGroupWarps = 8;
// At least twice the error of an fp32 value v = s + b, relative to 1 + |b|.  In steps of 2^-23: the exponential of x is off by
// 2 + 1.17 |x| of its own, of which a sigmoid keeps the share s (1 - s), 0.7 at most, the quotient 2, the sums 0.5 and 0.5 (1 + |b|):
// below 4 and 8.  A softmax keeps 2 of the exponentials, 2 of those in its sum, 6.5 of 13 additions, 1.5 of the quotient: 12.5 and 32.
template <bool SOFTMAX>
constexpr float kNear = SOFTMAX ? 3.814697265625e-6f : 1.9073486328125e-6f;   // 2^-18, 2^-19

// A value as a key of the same order: 0 lies below every value, NaN above infinity, the zeros are one
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ unsigned long long key_of(double v) {
  const unsigned long long u = __double_as_longlong(v + 0.0);
  return v != v ? ~0ull : (u >> 63) ? ~u : (u | (1ull << 63));
}

struct GroupParams {
  const void* logits;
  const float* bias;
  long long T;
  int E, k, groups, open, per_group, lanes_log;    // experts of a group; log2 of a group's lanes
  int top2, norm, vec;
  float scale;
  long long* idx;
  float* w;
  int* counts;        // nullable
  int count_direct;   // one CTA does all: counts are written, not added to
};

// The scores of a lane's experts in 64 bits; m: the row's largest logit
template <bool SOFTMAX, int V>
__device__ __forceinline__ void scores64(const float (&z)[V], int live, float m, double (&s)[V]) {
  if constexpr (SOFTMAX) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = i < live ? exp(static_cast<double>(z[i]) - static_cast<double>(m)) : 0.0;
      sum += s[i];
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = m == -INFINITY ? 0.0 : s[i] / sum;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 1.0 / (1.0 + exp(-static_cast<double>(z[i])));
  }
}

// The two largest of a group's values, over the lanes it owns; NaN counts as infinity
template <class F, int V>
__device__ __forceinline__ void group_best(const F (&v)[V], int live, int lanes_log, F& a, F& b) {
  a = b = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const F x = i >= live ? static_cast<F>(-INFINITY) : v[i] != v[i] ? static_cast<F>(INFINITY) : v[i];
    b = x > a ? a : (x > b ? x : b);
    a = x > a ? x : a;
  }
  for (int off = 1; off < (1 << lanes_log); off <<= 1) {
    const F oa = __shfl_xor_sync(0xffffffffu, a, off), ob = __shfl_xor_sync(0xffffffffu, b, off);
    const F lo = oa > a ? a : oa;
    a = oa > a ? oa : a;
    b = b > ob ? b : ob;
    b = b > lo ? b : lo;
  }
}
// Whether a lane's group is among the `open` best.  close: the last one that is and one that is not lie within `near` of one another
template <class F>
__device__ __forceinline__ bool group_open(F value, int g, int groups, int lanes_log, int open, F near, bool& close) {
  int rank = 0;
  bool below = false;
  for (int j = 0; j < groups; ++j) {
    const F o = __shfl_sync(0xffffffffu, value, j << lanes_log);
    const bool ahead = o > value || (o == value && j < g);
    rank += ahead ? 1 : 0;
    below = below || (!ahead && j != g && value - o <= near);
  }
  close = __any_sync(0xffffffffu, g < groups && rank == open - 1 && below);
  return g < groups && rank < open;
}

template <class T, bool SOFTMAX, int V>
__global__ void __launch_bounds__(32 * kGroupWarps)
group_topk_kernel(const GroupParams p) {
  grid_dep_begin();
  __shared__ int hist[B200MOE_MAX_EXPERTS];
  __shared__ float4 cand_s[kGroupWarps][32];     // value, logit, bias, expert
  __shared__ float2 pick_s[kGroupWarps][32];     // expert, logit
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned lower = (1u << lane) - 1u;
  if (p.counts != nullptr) {
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) hist[e] = 0;
    __syncthreads();
  }
  const int g = lane >> p.lanes_log, sub = lane & ((1 << p.lanes_log) - 1);
  const int live = g < p.groups ? max(0, min(V, p.per_group - sub * V)) : 0;
  const int first = live > 0 ? g * p.per_group + sub * V : 0;
  float bias[V], span = 1.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = p.bias != nullptr && i < live ? p.bias[first + i] : 0.0f;
    span = fmaxf(span, 1.0f + fabsf(bias[i]));
  }
  const bool by_logit = p.bias == nullptr;
  const float near = by_logit ? -1.0f : kNear<SOFTMAX> * warp_max(span);
  float4* cand = cand_s[warp];
  float2* pick = pick_s[warp];

  for (long long t = static_cast<long long>(blockIdx.x) * kGroupWarps + warp; t < p.T;
       t += static_cast<long long>(gridDim.x) * kGroupWarps) {
    float z[V], v[V];
    load_values<T, V>(reinterpret_cast<const T*>(p.logits) + t * p.E + first, live, p.vec, z);
    // ---- scores and selection values
    float m = 0.0f, inv = 0.0f;
    if constexpr (SOFTMAX) {
      m = z[0];
#pragma unroll
      for (int i = 1; i < V; ++i) m = fmaxf(m, z[i]);
      m = warp_max(m);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[i] = i < live ? __expf(z[i] - m) : 0.0f;
        sum += v[i];
      }
      sum = warp_sum(sum);
      inv = m == -INFINITY ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = m == -INFINITY ? bias[i] : v[i] * inv + bias[i];
    } else if (!by_logit || p.top2) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __fdividef(1.0f, 1.0f + __expf(-z[i])) + bias[i];
    }
    // ---- the open groups
    bool mine = live > 0;
    if (p.open < p.groups) {
      float a, b;
      const bool direct = by_logit && !p.top2;           // the largest logit decides
      if (direct) group_best(z, live, p.lanes_log, a, b);
      else group_best(v, live, p.lanes_log, a, b);
      bool close;
      mine = group_open(p.top2 && p.per_group > 1 ? a + b : a, g, p.groups, p.lanes_log, p.open,
                        direct ? -1.0f : 2.0f * (by_logit ? kNear<SOFTMAX> : near), close) && live > 0;
      if (close) {                                        // two groups that fp32 does not tell apart
        double s[V], a2, b2;
        scores64<SOFTMAX, V>(z, live, m, s);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] += static_cast<double>(bias[i]);
        group_best(s, live, p.lanes_log, a2, b2);
        mine = group_open(p.top2 && p.per_group > 1 ? a2 + b2 : a2, g, p.groups, p.lanes_log, p.open, -1.0, close) && live > 0;
      }
    }
    // ---- candidates: every expert that reaches the k-th largest of the lanes' maxima (less `near`)
    uint32_t key[V], best = 0u;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      key[i] = mine && i < live ? key_of(by_logit ? z[i] : v[i]) : 0u;
      best = max(best, key[i]);
    }
    uint32_t floor_key = 1u;
    for (int n = 0;;) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      if (top == 0u) {       // fewer than k lanes with an expert: all of them
        floor_key = 1u;
        break;
      }
      const bool at = best == top;
      n += __popc(__ballot_sync(0xffffffffu, at));
      if (at) best = 0u;
      floor_key = top;
      if (n >= p.k) break;
    }
    if (!by_logit && floor_key != 1u) {
      const float f = value_of(floor_key);
      floor_key = f == f && fabsf(f) < INFINITY ? key_of(f - near) : floor_key;
    }
    int n = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool in = key[i] >= floor_key;
      const unsigned b = __ballot_sync(0xffffffffu, in);
      const int at = n + __popc(b & lower);
      if (in && at < 32) cand[at] = make_float4(by_logit ? z[i] : v[i], z[i], bias[i], __int_as_float(first + i));
      n += __popc(b);
    }
    __syncwarp();
    if (n <= 32) {
      const float4 c = lane < n ? cand[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
      const uint32_t ck = key_of(c.x);
      const int ce = __float_as_int(c.w);
      int rank = 0;
      bool close = false;
      for (int j = 0; j < n; ++j) {
        const float4 o = cand[j];
        const uint32_t ok = key_of(o.x);
        rank += ok > ck || (ok == ck && __float_as_int(o.w) < ce) ? 1 : 0;
        close = close || (fabsf(o.x - c.x) <= near && (o.y != c.y || o.z != c.z));
      }
      if (__any_sync(0xffffffffu, lane < n && rank < p.k && close)) {     // picks that fp32 does not tell apart
        double d;
        if constexpr (SOFTMAX) {
          double s[V], sum = 0.0;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            s[i] = i < live ? exp(static_cast<double>(z[i]) - static_cast<double>(m)) : 0.0;
            sum += s[i];
          }
          sum = warp_sum(sum);
          d = m == -INFINITY ? 0.0 : exp(static_cast<double>(c.y) - static_cast<double>(m)) / sum;
        } else {
          d = 1.0 / (1.0 + exp(-static_cast<double>(c.y)));
        }
        const unsigned long long dk = key_of(d + static_cast<double>(c.z));
        rank = 0;
        for (int j = 0; j < n; ++j) {
          const unsigned long long ok = __shfl_sync(0xffffffffu, dk, j);
          const int oe = __shfl_sync(0xffffffffu, ce, j);
          rank += ok > dk || (ok == dk && oe < ce) ? 1 : 0;
        }
      }
      if (lane < n && rank < p.k) pick[rank] = make_float2(__int_as_float(ce), c.y);
    } else {
      // more than 32 candidates (rows of equal logits): k rounds of argmax, in 64 bits where there is a bias
      unsigned long long k64[V];
      double s[V];
      if (!by_logit) scores64<SOFTMAX, V>(z, live, m, s);
#pragma unroll
      for (int i = 0; i < V; ++i)
        k64[i] = mine && i < live ? key_of(by_logit ? static_cast<double>(z[i]) : s[i] + static_cast<double>(bias[i])) : 0ull;
      for (int j = 0; j < p.k; ++j) {
        unsigned long long bk = k64[0];
        int bi = 0;
#pragma unroll
        for (int i = 1; i < V; ++i)
          if (k64[i] > bk) {
            bk = k64[i];
            bi = i;
          }
        const uint32_t hi = static_cast<uint32_t>(bk >> 32), lo = static_cast<uint32_t>(bk);
        const uint32_t th = __reduce_max_sync(0xffffffffu, hi);
        const uint32_t tl = __reduce_max_sync(0xffffffffu, hi == th ? lo : 0u);
        const int owner = __ffs(__ballot_sync(0xffffffffu, hi == th && lo == tl)) - 1;   // lanes hold ascending experts
        if (lane == owner) {
          float zi = z[0];
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (i == bi) {
              zi = z[i];
              k64[i] = 0ull;
            }
          pick[j] = make_float2(__int_as_float(first + bi), zi);
        }
      }
    }
    __syncwarp();
    // ---- lane j < k: pick j and its weight
    int e = 0;
    float s = 0.0f;
    if (lane < p.k) {
      const float2 c = pick[lane];
      e = __float_as_int(c.x);
      if constexpr (SOFTMAX) s = m == -INFINITY ? 0.0f : expf(c.y - m) * inv;
      else s = 1.0f / (1.0f + expf(-c.y));
    }
    if (p.norm && p.k > 1) s /= warp_sum(s) + 1e-20f;
    if (lane < p.k) {
      p.idx[t * p.k + lane] = e;
      p.w[t * p.k + lane] = s * p.scale;
      if (p.counts != nullptr) atomicAdd(&hist[e], 1);
    }
    __syncwarp();      // the picks and candidates have been read
  }
  if (p.counts != nullptr) {
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
      const int c = hist[e];
      if (p.count_direct) p.counts[e] = c;
      else if (c != 0) atomicAdd(&p.counts[e], c);
    }
  }
}

// dz of w = s[idx] scale, or of w = s[idx] / (sum + 1e-20) scale: ds at the picks, then dz = ds s (1 - s), or s (ds - <ds, s>).
// Bound by the one write of dz (and, softmax, the one read of z; sigmoid reads its k logits alone).  The k values meet their
// experts in a row of shared memory.
template <class T, bool SOFTMAX, int V>
__global__ void __launch_bounds__(32 * kGroupWarps)
group_topk_bwd_kernel(const T* logits, const long long* idx, const float* grad_w, long long T_, int E, int k, int norm, int vec,
                      float scale, T* grad) {
  grid_dep_begin();
  __shared__ __align__(16) float row_s[kGroupWarps][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = lane * V, live = max(0, min(V, E - first));
  float* row = row_s[warp];
#pragma unroll
  for (int i = 0; i < V; ++i) row[first + i] = 0.0f;
  __syncwarp();
  for (long long t = static_cast<long long>(blockIdx.x) * kGroupWarps + warp; t < T_;
       t += static_cast<long long>(gridDim.x) * kGroupWarps) {
    const T* zr = logits + t * E;
    int e = -1;
    float g = 0.0f, zk = 0.0f, sk = 0.0f;
    if (lane < k) {
      const long long i = idx[t * k + lane];
      e = i >= 0 && i < E ? static_cast<int>(i) : -1;
      g = grad_w[t * k + lane] * scale;
      if (e >= 0) zk = to_f32(zr[e]);
    }
    const bool has = lane < k && e >= 0;      // a pick; one that names no expert gets no gradient
    float s[V], m = 0.0f, inv = 0.0f;
    if constexpr (SOFTMAX) {
      load_values<T, V>(zr + (live > 0 ? first : 0), live, vec, s);
      m = s[0];
#pragma unroll
      for (int i = 1; i < V; ++i) m = fmaxf(m, s[i]);
      m = warp_max(m);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[i] = i < live && m != -INFINITY ? expf(s[i] - m) : 0.0f;
        sum += s[i];
      }
      sum = warp_sum(sum);
      inv = m == -INFINITY ? 0.0f : 1.0f / sum;
      if (has) sk = m == -INFINITY ? 0.0f : expf(zk - m) * inv;
    } else if (has) {
      sk = 1.0f / (1.0f + expf(-zk));
    }
    float ds = g;
    if (norm && k > 1) {
      const float total = warp_sum(sk) + 1e-20f;
      ds = (g - warp_sum(g * sk) / total) / total;
    }
    float dot = 0.0f;
    if constexpr (SOFTMAX) {
      dot = warp_sum(has ? ds * sk : 0.0f);
    } else {
      const float x = expf(-fabsf(zk));
      ds *= x / ((1.0f + x) * (1.0f + x));      // s (1 - s), without the cancellation of 1 - s
    }
    if (has) row[e] = ds;
    __syncwarp();
    float d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      d[i] = row[first + i];
      if constexpr (SOFTMAX) d[i] = s[i] * inv * (d[i] - dot);
    }
    if (live > 0) store_values<T, V>(grad + t * E + first, live, vec, d);
    __syncwarp();
    if (has) row[e] = 0.0f;
    __syncwarp();
  }
}

static int group_grid(int64_t T) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((T + kGroupWarps - 1) / kGroupWarps, static_cast<int64_t>(num_sms()) * 8)));
}

}  // namespace b200moe

using namespace b200moe;

extern "C" {

int b200moe_group_topk_fwd(const void* logits, int logits_type, const float* bias, int64_t T, int E, int k, int groups, int open, int scoring,
                           int group_top2, int norm_topk, float scale, int64_t* idx, float* w, int32_t* counts, b200moe_stream_t stream) {
  B200_CHECK_ARG(logits && idx && w, B200MOE_E_NULL, "group_topk_fwd: null pointer");
  B200_CHECK_ARG(known_logits(logits_type), B200MOE_E_UNSUPPORTED, "group_topk_fwd: unknown type %d of the logits", logits_type);
  B200_CHECK_ARG(E >= 1 && E <= B200MOE_MAX_EXPERTS, B200MOE_E_UNSUPPORTED, "group_topk_fwd: E = %d, supported 1..%d", E,
                 B200MOE_MAX_EXPERTS);
  B200_CHECK_ARG(groups >= 1 && groups <= 32 && E % groups == 0, B200MOE_E_BAD_SHAPE,
                 "group_topk_fwd: %d groups must be 1..32 and divide E = %d", groups, E);
  B200_CHECK_ARG(open >= 1 && open <= groups, B200MOE_E_BAD_SHAPE, "group_topk_fwd: %d open groups of %d", open, groups);
  B200_CHECK_ARG(k >= 1 && k <= B200MOE_MAX_TOPK && k <= open * (E / groups), B200MOE_E_BAD_SHAPE,
                 "group_topk_fwd: top_k = %d must be in 1..min(%d experts of the open groups, %d)", k, open * (E / groups), B200MOE_MAX_TOPK);
  B200_CHECK_ARG(scoring == B200MOE_SIGMOID || scoring == B200MOE_SOFTMAX, B200MOE_E_UNSUPPORTED, "group_topk_fwd: unknown scoring %d",
                 scoring);
  B200_CHECK_ARG(T >= 0, B200MOE_E_BAD_SHAPE, "group_topk_fwd: T = %lld", (long long)T);
  cudaStream_t st = (cudaStream_t)stream;
  const int grid = group_grid(T);
  if (counts != nullptr && (T == 0 || grid > 1)) B200_CUDA(cudaMemsetAsync(counts, 0, sizeof(int32_t) * E, st));
  if (T == 0) return 0;
  GroupParams p{};
  p.logits = logits; p.bias = bias; p.T = T; p.E = E; p.k = k; p.groups = groups; p.open = open; p.per_group = E / groups;
  while ((2 << p.lanes_log) * groups <= 32) ++p.lanes_log;
  p.top2 = group_top2; p.norm = norm_topk; p.scale = scale;
  p.idx = reinterpret_cast<long long*>(idx); p.w = w; p.counts = counts; p.count_direct = grid == 1;
  const int lanes = 1 << p.lanes_log;
  cudaError_t err = cudaSuccess;
  by_values((p.per_group + lanes - 1) / lanes, [&](auto v) {
    constexpr int V = v.value;
    const int bytes = std::min(16, V * type_bytes(logits_type));
    p.vec = p.per_group % V == 0 && reinterpret_cast<uintptr_t>(logits) % bytes == 0;
    by_logits(logits_type, [&](auto type) {
      using T_ = decltype(type);
      err = launch_chained(scoring == B200MOE_SOFTMAX ? group_topk_kernel<T_, true, V> : group_topk_kernel<T_, false, V>, grid,
                           32 * kGroupWarps, 0, st, 1, p);
    });
  });
  B200_CUDA(err);
  return 0;
}

int b200moe_group_topk_bwd(const void* logits, int logits_type, const int64_t* idx, const float* grad_w, int64_t T, int E, int k, int scoring,
                           int norm_topk, float scale, void* grad_logits, b200moe_stream_t stream) {
  B200_CHECK_ARG(logits && idx && grad_w && grad_logits, B200MOE_E_NULL, "group_topk_bwd: null pointer");
  B200_CHECK_ARG(known_logits(logits_type), B200MOE_E_UNSUPPORTED, "group_topk_bwd: unknown type %d of the logits", logits_type);
  B200_CHECK_ARG(E >= 1 && E <= B200MOE_MAX_EXPERTS, B200MOE_E_UNSUPPORTED, "group_topk_bwd: E = %d, supported 1..%d", E,
                 B200MOE_MAX_EXPERTS);
  B200_CHECK_ARG(k >= 1 && k <= E && k <= B200MOE_MAX_TOPK, B200MOE_E_BAD_SHAPE, "group_topk_bwd: top_k = %d", k);
  B200_CHECK_ARG(scoring == B200MOE_SIGMOID || scoring == B200MOE_SOFTMAX, B200MOE_E_UNSUPPORTED, "group_topk_bwd: unknown scoring %d",
                 scoring);
  if (T <= 0) return 0;
  cudaError_t err = cudaSuccess;
  by_values((E + 31) / 32, [&](auto v) {
    constexpr int V = v.value;
    if constexpr (V <= 8) {
      const int bytes = std::min(16, V * type_bytes(logits_type));
      const int vec = E % V == 0 && reinterpret_cast<uintptr_t>(logits) % bytes == 0 && reinterpret_cast<uintptr_t>(grad_logits) % bytes == 0;
      by_logits(logits_type, [&](auto type) {
        using T_ = decltype(type);
        err = launch_chained(scoring == B200MOE_SOFTMAX ? group_topk_bwd_kernel<T_, true, V> : group_topk_bwd_kernel<T_, false, V>,
                             group_grid(T), 32 * kGroupWarps, 0, (cudaStream_t)stream, 1, reinterpret_cast<const T_*>(logits),
                             reinterpret_cast<const long long*>(idx), grad_w, static_cast<long long>(T), E, k, norm_topk, vec, scale,
                             reinterpret_cast<T_*>(grad_logits));
      });
    }
  });
  B200_CUDA(err);
  return 0;
}

}  // extern "C"

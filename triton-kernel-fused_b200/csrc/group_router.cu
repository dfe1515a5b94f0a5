// Group-limited top-k routing: softmax or sigmoid scores, a selection bias, the best groups of experts, the best experts of those,
// renormalised weights; and the gradient of the weights.
//
//   s = sigmoid(z) or softmax(z);  v = s + b;  a group's value = its largest v, or the sum of its two largest;  the `open` groups of
//   largest value;  the k largest v inside them, equal values to the lowest index;  w = s / (sum s + 1e-20) * scale
//
// A pick is a comparison of real numbers, and two of 256 experts are often closer than fp32 resolves (32 768 tokens, 8 of 256: some
// hundred picks a step), so which one an fp32 kernel takes is left to its rounding.  Here the picks are those of the real numbers:
// without a bias s rises with z, and z itself is compared; with one, values closer than the error of the fp32 ones (kErr) are
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
// Two fp32 values v = s + b whose distance is above the sum of their kErr * max(1, |v|) are in the order of the real numbers.  In steps of 2^-23,
// relative to max(1, |v|): a sigmoid is off by 0.7 (its exponential, 2 + 1.17 |x| of itself, times s (1 - s)), 2 (quotient) and 0.5 (sum), v by 0.5 more and
// the sum of a group's two values by 0.5: 4.2, and 8 are allowed.  A softmax value is off by 2 (the exponential of x <= 0: 2 + 1.67 |x| of itself with the
// rounding of x, times at most e^x), 0.5 (product), 0.5 and 0.5: 3.5 of its own.  What the denominator is off by is common to the two values and
// counts with their distance, below 1: 0.5 (quotient), 2 + 2.5 (its exponentials; the mean of 1.67 |x|, times the largest share), 6 or 10 (12 or 20 additions, at
// 8 or 16 values a lane): 15 a pair.  7 + 15 = 22, and 32 are allowed.
template <bool SOFTMAX>
constexpr float kErr = SOFTMAX ? 1.9073486328125e-6f : 9.5367431640625e-7f;   // 2^-19, 2^-20
// of v, finite for an infinite one too (a sum with infinity is exact)
template <bool SOFTMAX>
__device__ __forceinline__ float err_of(float v) {
  return kErr<SOFTMAX> * fminf(fmaxf(fabsf(v), 1.0f), 3.402823466e38f);
}

// A value (no NaN) as a signed integer of the same order, and back; kNone lies below every value
constexpr int kNone = static_cast<int>(0x80000000u);
__device__ __forceinline__ int key_of(float v) {
  const int i = __float_as_int(v);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float value_of(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }
// ... and in 64 bits, with NaN above infinity; 0 lies below every value, the zeros are one
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

// The two largest of a group's values, over the lanes it owns; NaN counts as infinity
__device__ __forceinline__ void best_of(float x, float& a, float& b) {      // no NaN
  b = fmaxf(b, fminf(a, x));
  a = fmaxf(a, x);
}
__device__ __forceinline__ void best_of(double x, double& a, double& b) {
  x = x != x ? static_cast<double>(INFINITY) : x;
  b = x > a ? a : (x > b ? x : b);
  a = x > a ? x : a;
}
// A group's value from them, halved, so that the sum of two finite values is finite; infinity less infinity counts as infinity too
template <class F>
__device__ __forceinline__ F group_value(F a, F b) {
  const F v = static_cast<F>(0.5) * a + static_cast<F>(0.5) * b;
  return v != v ? static_cast<F>(INFINITY) : v;
}
template <class F>
__device__ __forceinline__ void group_best(int lanes_log, F& a, F& b) {
  for (int off = 1; off < (1 << lanes_log); off <<= 1) {
    const F oa = __shfl_xor_sync(0xffffffffu, a, off), ob = __shfl_xor_sync(0xffffffffu, b, off);
    const F lo = oa > a ? a : oa;
    a = oa > a ? oa : a;
    b = b > ob ? b : ob;
    b = b > lo ? b : lo;
  }
}
// Whether a lane's group is among the `open` best
template <class F>
__device__ __forceinline__ bool group_open(F value, int g, int groups, int lanes_log, int open) {
  int rank = 0;
  for (int j = 0; j < groups; ++j) {
    const F o = __shfl_sync(0xffffffffu, value, j << lanes_log);
    rank += o > value || (o == value && j < g) ? 1 : 0;
  }
  return g < groups && rank < open;
}
// Whether an open and a closed group may be the other way round, each value off by `err` at most.  (Infinite ones are equal as they are.)
__device__ __forceinline__ bool groups_close(float value, float err, bool opened, bool closed) {
  const float lo = value_of(__reduce_min_sync(0xffffffffu, opened ? key_of(value - err) : 0x7fffffff));
  const float hi = value_of(__reduce_max_sync(0xffffffffu, closed ? key_of(value + err) : kNone));
  return hi >= lo && fabsf(lo) < INFINITY;
}

// The rest is for tokens that fp32 does not decide.  Out of line, with the logits read again one by one: inlined, its 64-bit arithmetic
// doubled the kernel's registers (32 768 tokens, 8 of 256 experts in 4 of 8 groups: 128 us with it inside, whether it ran or not).
template <class T, bool SOFTMAX>
struct Exact {
  const GroupParams& p;
  const T* z;          // the lane's logits
  int first, live;
  double m, sum;       // softmax: the row's largest logit, its denominator
  __device__ __forceinline__ Exact(const GroupParams& p_, long long t, int first_, int live_, float m_)
      : p(p_), z(reinterpret_cast<const T*>(p_.logits) + t * p_.E + first_), first(first_), live(live_), m(m_), sum(1.0) {
    if constexpr (SOFTMAX) {
      double s = 0.0;
#pragma unroll 1
      for (int i = 0; i < live; ++i) s += exp(static_cast<double>(to_f32(z[i])) - m);
      sum = warp_sum(s);
    }
  }
  __device__ __forceinline__ double score(float logit) const {
    if constexpr (SOFTMAX) return m == -INFINITY ? 0.0 : exp(static_cast<double>(logit) - m) / sum;
    else return 1.0 / (1.0 + exp(-static_cast<double>(logit)));
  }
  __device__ __forceinline__ double value(int i) const {      // what selection compares
    if (p.bias == nullptr) return score(to_f32(z[i]));
    return score(to_f32(z[i])) + static_cast<double>(p.bias[first + i]);
  }
};

template <class T, bool SOFTMAX>
__device__ __noinline__ bool open_exactly(const GroupParams& p, long long t, int g, int first, int live, float m) {
  const Exact<T, SOFTMAX> x(p, t, first, live, m);
  double a = -INFINITY, b = -INFINITY;
#pragma unroll 1
  for (int i = 0; i < live; ++i) best_of(x.value(i), a, b);
  group_best(p.lanes_log, a, b);
  return group_open(group_value(a, p.top2 ? b : a), g, p.groups, p.lanes_log, p.open);
}

// the rank of a lane's candidate (its logit and bias) among n
template <class T, bool SOFTMAX>
__device__ __noinline__ int rank_exactly(const GroupParams& p, long long t, int first, int live, float m, int n, float logit, float bias) {
  const Exact<T, SOFTMAX> x(p, t, first, live, m);
  const unsigned long long key = key_of(x.score(logit) + static_cast<double>(bias));
  const int lane = threadIdx.x & 31;
  int rank = 0;
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const unsigned long long o = __shfl_sync(0xffffffffu, key, j);
    rank += o > key || (o == key && j < lane) ? 1 : 0;
  }
  return rank;
}

// More than 32 candidates (rows of equal logits): k rounds of argmax over keys in shared memory.  live: 0 for a closed group
template <class T, bool SOFTMAX>
__device__ __noinline__ void pick_exactly(const GroupParams& p, long long t, int first, int live, int open_live, float m, unsigned long long* keys,
                                          float2* pick) {
  const Exact<T, SOFTMAX> x(p, t, first, live, m);
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int i = 0; i < open_live; ++i)
    keys[first + i] = key_of(p.bias == nullptr ? static_cast<double>(to_f32(x.z[i])) : x.value(i));
#pragma unroll 1
  for (int j = 0; j < p.k; ++j) {
    unsigned long long best = 0ull;
    int at = 0;
#pragma unroll 1
    for (int i = 0; i < open_live; ++i)
      if (keys[first + i] > best) {
        best = keys[first + i];
        at = i;
      }
    const uint32_t hi = static_cast<uint32_t>(best >> 32), lo = static_cast<uint32_t>(best);
    const uint32_t th = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t tl = __reduce_max_sync(0xffffffffu, hi == th ? lo : 0u);
    const int owner = __ffs(__ballot_sync(0xffffffffu, hi == th && lo == tl)) - 1;   // lanes hold ascending experts
    if (lane == owner) {
      pick[j] = make_float2(__int_as_float(first + at), to_f32(x.z[at]));
      keys[first + at] = 0ull;
    }
    __syncwarp();
  }
}

// (At four CTAs an SM the softmax form spills: 48 bytes a thread at eight values a lane, 16 at four.)
template <class T, bool SOFTMAX, int V>
__global__ void __launch_bounds__(32 * kGroupWarps, V > 8 ? 1 : 4)
group_topk_kernel(const __grid_constant__ GroupParams p) {
  grid_dep_begin();
  __shared__ int hist[B200MOE_MAX_EXPERTS];
  __shared__ int2 cand_s[kGroupWarps][32];       // key, expert
  __shared__ float2 pick_s[kGroupWarps][32];     // expert, logit
  __shared__ unsigned long long key_s[kGroupWarps][B200MOE_MAX_EXPERTS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.counts != nullptr) {
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) hist[e] = 0;
    __syncthreads();
  }
  const int g = lane >> p.lanes_log, sub = lane & ((1 << p.lanes_log) - 1);
  const int live = g < p.groups ? max(0, min(V, p.per_group - sub * V)) : 0;
  const int first = live > 0 ? g * p.per_group + sub * V : 0;
  float bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) bias[i] = p.bias != nullptr && i < live ? p.bias[first + i] : 0.0f;
  const bool by_logit = p.bias == nullptr;
  int2* cand = cand_s[warp];
  float2* pick = pick_s[warp];

  for (long long t = static_cast<long long>(blockIdx.x) * kGroupWarps + warp; t < p.T;
       t += static_cast<long long>(gridDim.x) * kGroupWarps) {
    const T* row = reinterpret_cast<const T*>(p.logits) + t * p.E;
    float v[V];
    load_values<T, V>(row + first, live, p.vec, v);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < V; ++i) odd = odd || v[i] != v[i];
    odd = __any_sync(0xffffffffu, odd);          // a row with NaN, or with scores or sums that are NaN (below)
    // ---- what selection compares: the logits, or scores + bias (groups by two: the scores, until a group is chosen)
    const bool sums = p.open < p.groups && p.top2;
    int key[V];
    float m = 0.0f, inv = 0.0f;
    if constexpr (SOFTMAX) {
      m = v[0];
#pragma unroll
      for (int i = 1; i < V; ++i) m = fmaxf(m, v[i]);
      m = warp_max(m);
    }
    if (by_logit) {
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = i < live ? key_of(v[i] + 0.0f) : kNone;
    }
    if (SOFTMAX || !by_logit || sums) {
      if constexpr (SOFTMAX) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[i] = m == -INFINITY ? 0.0f : __expf(v[i] - m);       // a value that does not exist is -inf
          sum += v[i];
        }
        sum = warp_sum(sum);
        inv = m == -INFINITY ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = v[i] * inv + bias[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __fdividef(1.0f, 1.0f + __expf(-v[i])) + bias[i];
      }
      // a softmax over +infinity, a bias of NaN: NaN is neither above nor below a value, and fp32 finds no pick
      bool nan = odd;
#pragma unroll
      for (int i = 0; i < V; ++i) nan = nan || v[i] != v[i];
      odd = __any_sync(0xffffffffu, nan);
    }
    if (!by_logit) {
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = i < live ? key_of(v[i]) : kNone;
    }
    // ---- the open groups
    bool mine = live > 0;
    if (p.open < p.groups) {
      bool close = odd;
      if (!odd) {
        float a = -INFINITY, b = -INFINITY;
        const bool direct = by_logit && !p.top2;           // the largest logit decides
        if (direct) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (i < live) a = fmaxf(a, value_of(key[i]));
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (i < live) best_of(v[i], a, b);
        }
        group_best(p.lanes_log, a, b);
        if (!p.top2) b = a;
        const float value = direct ? a : group_value(a, b);
        const bool opened = group_open(value, g, p.groups, p.lanes_log, p.open);
        close = !direct && groups_close(value, 0.5f * (err_of<SOFTMAX>(a) + err_of<SOFTMAX>(b)), opened, g < p.groups && !opened);
        mine = mine && opened;
      }
      if (close) mine = open_exactly<T, SOFTMAX>(p, t, g, first, live, m) && live > 0;
      if (!mine) {
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = kNone;
      }
    }
    // ---- candidates: every expert that reaches the k-th largest of the lanes' maxima (less what the two may be off by)
    int best = key[0];
#pragma unroll
    for (int i = 1; i < V; ++i) best = max(best, key[i]);
    int floor_key = kNone + 1;
    for (int n = 0; n < p.k;) {
      const int top = __reduce_max_sync(0xffffffffu, best);
      floor_key = top;
      if (top == kNone) break;
      const unsigned at = __ballot_sync(0xffffffffu, best == top);
      n += __popc(at);
      if (best == top) best = kNone;
    }
    // fewer than k lanes with an expert: all of them; else what may be hidden below it too
    if (floor_key == kNone) floor_key = kNone + 1;
    else if (!by_logit) floor_key = min(floor_key, key_of(value_of(floor_key) - 2.0f * err_of<SOFTMAX>(value_of(floor_key))));
    // collected in the order of the experts, so that of equal ones the first collected wins
    int have = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) have += key[i] >= floor_key ? 1 : 0;
    int at = have;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, at, off);
      if (lane >= off) at += o;
    }
    const int n = __shfl_sync(0xffffffffu, at, 31);
    if (n <= 32 && !odd) {
      at -= have;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (key[i] >= floor_key) cand[at++] = make_int2(key[i], first + i);
      __syncwarp();
      const int2 c = lane < n ? cand[lane] : make_int2(kNone, 0);
      const float logit = to_f32(row[c.y]);
      const float value = lane < n ? value_of(c.x) : -INFINITY;
      const float near = 2.0f * err_of<SOFTMAX>(value);      // values this close are of one size
      int rank = 0, level = 0;                     // level: candidates within `near` of this one, itself among them
      if (by_logit) {
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
          const int o = __shfl_sync(0xffffffffu, c.x, j);
          rank += o > c.x || (o == c.x && j < lane) ? 1 : 0;
        }
      } else {
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
          const float o = __shfl_sync(0xffffffffu, value, j);
          rank += o > value || (o == value && j < lane) ? 1 : 0;
          level += fabsf(o - value) <= near ? 1 : 0;
        }
        if (__any_sync(0xffffffffu, lane < n && rank < p.k && level > 1)) {
          // the same logit and bias is a tie; others are compared in 64 bits
          const float b = p.bias[c.y];
          bool close = false;
          for (int j = 0; j < n; ++j) {
            const float o = __shfl_sync(0xffffffffu, value, j), oz = __shfl_sync(0xffffffffu, logit, j), ob = __shfl_sync(0xffffffffu, b, j);
            close = close || (fabsf(o - value) <= near && (oz != logit || ob != b));
          }
          if (__any_sync(0xffffffffu, lane < n && rank < p.k && close)) rank = rank_exactly<T, SOFTMAX>(p, t, first, live, m, n, logit, b);
        }
      }
      if (lane < n && rank < p.k) pick[rank] = make_float2(__int_as_float(c.y), logit);
    } else {
      pick_exactly<T, SOFTMAX>(p, t, first, live, mine ? live : 0, m, key_s[warp], pick);
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
// Bound by the issue of instructions and by one token's loads at a time in a warp (the picks, then their logits): 32 768 tokens, 8 of 256 experts, bf16
// 11.8 us by sigmoid scores, 184 warp instructions a token in 72 % of the cycles, where dz, the picks and their logits' sectors take 4.3; softmax, which reads
// and sums the whole row, 400 in 61 %.  The k values meet their experts in a row of shared memory.
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
  p.top2 = group_top2 && p.per_group > 1; p.norm = norm_topk; p.scale = scale;
  p.idx = reinterpret_cast<long long*>(idx); p.w = w; p.counts = counts; p.count_direct = grid == 1;
  const int lanes = 1 << p.lanes_log;
  OpScope scope("group_topk_fwd", 1);
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
  OpScope scope("group_topk_bwd", 1);
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

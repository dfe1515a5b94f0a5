// Low-rank adapters of many requests beside a shared projection: row t of x has the adapter l = index[t], or none,
//
//   v[t] = s_l x[t] A_l^T          out[t] = base[t] + v[t] B_l^T           A (L,R,K), B (L,N,R)
//
// and backward   u[t] = s_l g[t] B_l,   grad_x[t] = u[t] A_l,   grad_A_l = sum_t u[t]^T x[t],   grad_B_l = sum_t g[t]^T v[t].
//
// Four products with one short side (R of at most 128), all bound by HBM: `shrink` (T,D) -> (T,R) reads x or g, `expand` (T,R) -> (T,D) reads
// base and writes out or grad_x, `wgrad` reads x or g again.  Each is a tcgen05 kernel.  The first two take tiles of 128 rows as they come, without sorting
// them: a tile's distinct adapters are found by a kernel before, each is multiplied with all rows of the tile into tensor memory of its own, and a
// row takes the result of its adapter.  `wgrad` takes the rows of an adapter's list.  Rows of other adapters are never added to anything, not even times
// zero, so an infinity or a NaN stays with its own adapter or row.  Few rows (a decoding batch) run in one kernel of their own, a cluster for up to sixteen rows of an adapter.
//
// v and u, which go from one product to the next, are two bf16 numbers each, the nearest and what that leaves, side by side: 16 bits, so that results are as
// exact as those of an fp32 v.  (Rounded to one number the error of a result without a base was 0.0024 in the norm in place of 0.0017.)  All sums are fp32.
#include <cuda.h>

#include <algorithm>

#include "gemm_common.cuh"

namespace b200moe {

constexpr int kLTile = 128;                      // rows of a tile
constexpr int kLBox = 128 * 64 * 2;              // 128 rows x 64 values, 128-byte swizzle

struct LoraIndex {
  const void* index;      // T adapters, or nullptr: adapter 0 for every row
  int bytes;              // of one: 4 or 8
  int T, L;
  int* status;
};

__device__ __forceinline__ int lora_adapter(const LoraIndex& p, long long t) {
  if (t >= p.T) return -1;
  if (p.index == nullptr) return 0;
  const long long l = p.bytes == 8 ? static_cast<const long long*>(p.index)[t] : static_cast<const int*>(p.index)[t];
  if (l >= p.L) {
    *p.status = ST_BAD_ADAPTER_INDEX;
    return -1;
  }
  return l < 0 ? -1 : static_cast<int>(l);
}

// The adapters of each tile of 128 rows, each named once, in the order of its first row.  nullptr: adapter 0 for every row
struct LoraTiles {
  int* n;                    // (tiles): adapters of a tile
  int* adapter;              // (tiles, 128)
  short* slot;               // (tiles, 128): of a row, its adapter's place among them, -1: none
  int T, tiles;
};
__device__ __forceinline__ int tile_n(const LoraTiles& p, int tile) { return p.n == nullptr ? 1 : p.n[tile]; }
__device__ __forceinline__ int tile_adapter(const LoraTiles& p, int tile, int i) {
  return p.n == nullptr ? 0 : p.adapter[static_cast<long long>(tile) * kLTile + i];
}
__device__ __forceinline__ int tile_slot(const LoraTiles& p, int tile, int row) {
  const long long t = static_cast<long long>(tile) * kLTile + row;
  return p.n == nullptr ? (t < p.T ? 0 : -1) : p.slot[t];
}

// The same for the lists, which the tiles' CTAs report for: no store between the loads, so that several are on their way
__device__ __forceinline__ int named_adapter(const LoraIndex& p, long long t) {
  const long long l = p.bytes == 8 ? static_cast<const long long*>(p.index)[t] : static_cast<const int*>(p.index)[t];
  return l < 0 || l >= p.L ? -1 : static_cast<int>(l);
}
// The rows of each adapter, in their order, one adapter after another: those of l are order[bounds[l]] ... order[bounds[l + 1] - 1].
struct LoraLists {
  int* order;                // (T), nullptr: not asked for
  int* bounds;               // (L + 1)
};
constexpr int kTilesThreads = 512, kTilesEach = kTilesThreads / kLTile;

// one CTA: the list of adapter l.  Each warp counts in a stretch of the rows of its own, and then writes behind those before it.
__device__ __forceinline__ void lora_list(const LoraIndex& ix, const LoraLists& p, int l) {
  constexpr int WARPS = kTilesThreads / 32, U = 8;
  __shared__ int found[2][WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long each = (static_cast<long long>(ix.T) + 32 * WARPS - 1) / (32 * WARPS) * 32, r0 = warp * each, r1 = min(static_cast<long long>(ix.T), r0 + each);
  int here = 0, below = 0;
  for (long long r = r0 + lane; r - lane < r1; r += 32 * U) {
    int of[U];
#pragma unroll
    for (int u = 0; u < U; ++u) of[u] = r + 32 * u < r1 ? named_adapter(ix, r + 32 * u) : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      here += of[u] == l;
      below += of[u] >= 0 && of[u] < l;
    }
  }
  here = __reduce_add_sync(0xffffffffu, here);
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) {
    found[0][warp] = here;
    found[1][warp] = below;
  }
  __syncthreads();
  int first = 0, at = 0, all = 0;
  for (int w = 0; w < WARPS; ++w) {
    first += found[1][w];
    if (w < warp) at += found[0][w];
    all += found[0][w];
  }
  at += first;
  if (threadIdx.x == 0) {
    p.bounds[l] = first;
    if (l == ix.L - 1) p.bounds[l + 1] = first + all;
  }
  for (long long r = r0 + lane; here > 0 && r - lane < r1; r += 32 * U) {
    int of[U];
#pragma unroll
    for (int u = 0; u < U; ++u) of[u] = r + 32 * u < r1 ? named_adapter(ix, r + 32 * u) : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned m = __ballot_sync(0xffffffffu, of[u] == l);
      if (of[u] == l) p.order[at + __popc(m & ((1u << lane) - 1u))] = static_cast<int>(r + 32 * u);
      at += __popc(m);
    }
  }
}

// The first CTAs make a list each, where lists are asked for; the others take kTilesEach tiles each, 128 threads a tile.
__global__ void __launch_bounds__(kTilesThreads) lora_tiles_kernel(const LoraIndex ix, const LoraTiles p, const LoraLists lists) {
  grid_dep_wait();
  __shared__ __align__(16) int all_rows[kTilesEach][kLTile];
  __shared__ int slots[kTilesEach][kLTile], all_warps[kTilesEach][kLTile / 32];
  const int n_lists = lists.order != nullptr ? ix.L : 0;
  const int g = threadIdx.x / kLTile, t = threadIdx.x % kLTile;
  const int tile = (static_cast<int>(blockIdx.x) - n_lists) * kTilesEach + g;
  if (static_cast<int>(blockIdx.x) < n_lists) {
    lora_list(ix, lists, blockIdx.x);
  } else if (tile < p.tiles) {
    auto sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(g + 1), "n"(kLTile) : "memory"); };
    int *of_row = all_rows[g], *slot = slots[g], *warps = all_warps[g];
    const long long row = static_cast<long long>(tile) * kLTile + t;
    const int l = lora_adapter(ix, row);
    of_row[t] = l;
    sync();
    // the first row of this thread's adapter: in this warp, or in one before
    const unsigned same = __match_any_sync(0xffffffffu, l);
    int at = (t & ~31) + __ffs(same) - 1;
    for (int j = 0; j < (t >> 5) * 8; ++j) {
      const int4 o = reinterpret_cast<const int4*>(of_row)[j];
      const int i = o.x == l ? 0 : o.y == l ? 1 : o.z == l ? 2 : o.w == l ? 3 : 4;
      if (i < 4) {
        at = 4 * j + i;
        break;
      }
    }
    __syncwarp();
    const bool first = l >= 0 && at == t;
    const unsigned firsts = __ballot_sync(0xffffffffu, first);
    if ((t & 31) == 0) warps[t >> 5] = __popc(firsts);
    sync();
    int n = __popc(firsts & ((1u << (t & 31)) - 1u));
    for (int w = 0; w < (t >> 5); ++w) n += warps[w];
    if (first) {
      slot[t] = n;
      p.adapter[static_cast<long long>(tile) * kLTile + n] = l;
    }
    if (t == 0) p.n[tile] = warps[0] + warps[1] + warps[2] + warps[3];
    sync();
    p.slot[row] = static_cast<short>(l >= 0 ? slot[at] : -1);
  }
  grid_dep_launch();
}

// Where a cluster's share of the units of work begins and ends: tile t has weight f(its adapters), and a place is a tile and what of its weight is
// before.  All threads of the CTA; barriers inside.
struct LoraShare {
  long long warps[32], rest[2];
  int tile[2];
};
template <int THREADS, class F>
__device__ __forceinline__ void lora_share(const LoraTiles& p, long long share, long long shares, F weight, LoraShare& s) {
  const int t = threadIdx.x;
  if (p.n == nullptr) {
    if (t < 2) {
      const long long w = weight(1), at = (share + t) * (p.tiles * w) / shares;
      s.tile[t] = static_cast<int>(at / w);
      s.rest[t] = at % w;
    }
    __syncthreads();
    return;
  }
  const int per = (p.tiles + THREADS - 1) / THREADS, t0 = min(p.tiles, t * per), t1 = min(p.tiles, t0 + per);
  long long sum = 0;
  for (int i = t0; i < t1; ++i) sum += weight(p.n[i]);
  long long incl = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, off);
    if ((t & 31) >= off) incl += o;
  }
  if ((t & 31) == 31) s.warps[t >> 5] = incl;
  __syncthreads();
  long long before = incl - sum, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < (t >> 5)) before += s.warps[w];
    total += s.warps[w];
  }
  for (int e = 0; e < 2; ++e) {
    const long long at = (share + e) * total / shares;
    if (at >= before && at < before + sum) {
      long long rest = at - before;
      int i = t0;
      for (; rest >= weight(p.n[i]); ++i) rest -= weight(p.n[i]);
      s.tile[e] = i;
      s.rest[e] = rest;
    }
    if (at == total && t == 0) {
      s.tile[e] = p.tiles;
      s.rest[e] = 0;
    }
  }
  __syncthreads();
}

// two fp32 numbers as bf16 and what that leaves of them, as bf16 too (nothing of an infinity)
__device__ __forceinline__ void split_bf16x2(float2 f, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(f.x, f.y);
  const float2 h = unpack_bf16x2(hi);
  lo = pack_bf16x2(fabsf(h.x) == INFINITY ? 0.0f : f.x - h.x, fabsf(h.y) == INFINITY ? 0.0f : f.y - h.y);
}

// columns of tensor memory -> registers, 32 or 16 at a time
template <int N>
__device__ __forceinline__ void lora_fetch(uint32_t taddr, bool mine, float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 16) {
    uint32_t r[16];
    tmem_ld16(taddr + c, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[c + i] = mine ? __uint_as_float(r[i]) : v[c + i];
  }
}

// four neighbouring sums of every CTA of the cluster, added up in their order: all loads on their way at once
__device__ __forceinline__ float4 cluster_sum4(uint32_t at, int ctas) {
  float4 v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (k < ctas)
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w)
                   : "r"(mapa_shared(at, k))
                   : "memory");
  }
#pragma unroll
  for (int k = 1; k < 8; ++k) {
    v[0].x += v[k].x; v[0].y += v[k].y; v[0].z += v[k].z; v[0].w += v[k].w;
  }
  return v[0];
}

// ------------------------------------------------------------------------------------------------ shrink
// v[t, r] = s_l sum_d X[t, d] W_l[r, d].  A unit of work is a row tile and as many of its adapters as fit 128 accumulator columns; a cluster of `split`
// CTAs shares a unit's columns d and adds up its partial sums through distributed shared memory.  WMN: W_l lies (D, R), reduction index first (the
// backward's B).
// 8192 x 4096 to rank 32 takes 20 us, 10.3 of them at the rate of a plain copy: there is one wave of CTAs, so nothing runs while they set up, find
// their share and add up (5.5 us with a single block of columns).  One remote sum at a time in place of all at once made it 3 us more.
constexpr int kShrinkMost = 5, kShrinkThreads = 192, kShrinkRing = 96 << 10;      // stages: of X and of the adapters that a unit can have
constexpr int kShrinkSmem = kShrinkRing + (2 * kShrinkMost + 2) * 8 + 16 + 1024;

struct ShrinkParams {
  LoraTiles tiles;
  int D, R, split;
  int stages, stage;         // of the ring, bytes of one
  const float* scales;       // (L,), or nullptr: `scale` for all
  float scale;
  __nv_bfloat16* v;          // (T, 2 RP): nearest, rests
  int* counter;              // of the expand behind it, set to zero
  int* status;
};

// one CTA of share `part` of `parts`, of a cluster or not
template <int RP, bool WMN>
__device__ __forceinline__ void shrink_rows(const CUtensorMap& tmX, const CUtensorMap& tmW, const ShrinkParams& p, int part, int parts, uint8_t* smem,
                                            LoraShare& share) {
  constexpr int NB = WMN && RP < 64 ? 64 : RP;       // accumulator columns of an adapter: whole swizzle atoms where W is MN-major
  constexpr int SLOTS = 128 / NB;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kShrinkRing);
  const uint32_t bar_full = smem_u32(bars), bar_empty = smem_u32(bars + kShrinkMost);
  const uint32_t bar_tfull = smem_u32(bars + 2 * kShrinkMost), bar_tempty = bar_tfull + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kShrinkMost + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(bar_full + 8 * s, 2);        // X, and the adapters
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_tfull, 1);
    mbar_init(bar_tempty, 4);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 128);
    tmem_relinquish();
  }
  grid_dep_wait();
  if (part == 0 && rank == 0 && threadIdx.x == 0) *p.counter = 0;
  tc_fence_before();
  lora_share<kShrinkThreads>(p.tiles, part, parts, [](int n) { return max(1, (n + SLOTS - 1) / SLOTS); }, share);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int nkb = (p.D + 63) / 64;
  const int kb0 = static_cast<int>(static_cast<long long>(rank) * nkb / p.split), kb1 = static_cast<int>(static_cast<long long>(rank + 1) * nkb / p.split);
  int done = 0;              // blocks of the units before: the place in the ring
  uint32_t unit_ph = 0;
  bool ok = true;

  for (int tile = share.tile[0], pass = static_cast<int>(share.rest[0]); tile < share.tile[1] || (tile == share.tile[1] && pass < static_cast<int>(share.rest[1]));) {
    const int all = tile_n(p.tiles, tile), first = pass * SLOTS, n = min(SLOTS, all - first);      // n = 0: a tile without adapters
    const int row0 = tile * kLTile;
    float v[RP];
#pragma unroll
    for (int i = 0; i < RP; ++i) v[i] = 0.0f;
    int mine = -1;
    if (warp == 0) {
      if (n > 0 && elect_one()) {
        int s = done % p.stages;
        uint32_t ph = done / p.stages & 1;
        int of[SLOTS];
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) of[j] = j < n ? tile_adapter(p.tiles, tile, first + j) : 0;
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          ok = mbar_wait(bar_empty + 8 * s, ph ^ 1, abort_flag, ST_WAIT_PRODUCER);
          if (!ok) break;
          const uint32_t full = bar_full + 8 * s, sx = smem_u32(smem + s * p.stage), sw = sx + kLBox;
          mbar_arrive_expect_tx(full, kLBox);
          tma_load_3d(sx, &tmX, full, kb * 64, row0, 0);
          mbar_arrive_expect_tx(full, n * NB * 128);
#pragma unroll
          for (int j = 0; j < SLOTS; ++j) {
            if (j >= n) break;
            if constexpr (WMN) {
#pragma unroll
              for (int h = 0; h < NB / 64; ++h) tma_load_3d(sw + (j * (NB / 64) + h) * 8192, &tmW, full, 64 * h, kb * 64, of[j]);
            } else {
              tma_load_3d(sw + j * NB * 128, &tmW, full, kb * 64, 0, of[j]);
            }
          }
          if (++s == p.stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    } else if (warp == 1) {
      if (n > 0 && elect_one()) {
        int s = done % p.stages;
        uint32_t ph = done / p.stages & 1;
        const uint32_t idesc = umma_idesc_bf16(n * NB, 0, WMN);
        ok = ok && mbar_wait(bar_tempty, unit_ph ^ 1, abort_flag, ST_WAIT_MMA_TMEM);
        tc_fence_after();
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          ok = mbar_wait(bar_full + 8 * s, ph, abort_flag, ST_WAIT_MMA_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sx = smem_u32(smem + s * p.stage), sw = sx + kLBox;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16(tmem, umma_desc_sw128(sx + 32 * k, 0, 1024), umma_desc_sw128(sw + (WMN ? 2048 : 32) * k, WMN ? 8192 : 0, 1024), idesc,
                      kb != kb0 || k != 0);
          umma_commit(bar_empty + 8 * s);
          if (++s == p.stages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (ok) umma_commit(bar_tfull);
      }
    } else {
      const int q = warp & 3, row = 32 * q + lane;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(32 * q) << 16);
      mine = tile_slot(p.tiles, tile, row);
      if (n > 0) {
        ok = ok && mbar_wait(bar_tfull, unit_ph, abort_flag, ST_WAIT_EPILOGUE);
        __syncwarp();
        tc_fence_after();
        for (int j = 0; j < n; ++j) {
          const bool me = mine == first + j;
          if (__any_sync(0xffffffffu, me)) lora_fetch<RP>(taddr + j * NB, me, v);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_tempty);
      }
      const long long t = static_cast<long long>(row0) + row;
      if (p.split == 1) {
        // a row is written by the unit of its adapter, or without one by the tile's first
        if (t < p.tiles.T && (mine < 0 ? pass == 0 : mine >= first && mine < first + n)) {
          const float s = mine < 0 ? 0.0f : p.scales != nullptr ? p.scales[tile_adapter(p.tiles, tile, mine)] : p.scale;
#pragma unroll
          for (int i = 0; i < RP; i += 8) {
            uint32_t hi[4] = {0u, 0u, 0u, 0u}, lo[4] = {0u, 0u, 0u, 0u};
            if (mine >= 0 && i < p.R) {      // R a multiple of 8
#pragma unroll
              for (int h = 0; h < 4; ++h) split_bf16x2(make_float2(s * v[i + 2 * h], s * v[i + 2 * h + 1]), hi[h], lo[h]);
            }
            *reinterpret_cast<uint4*>(p.v + t * (2 * RP) + i) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(p.v + t * (2 * RP) + RP + i) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        }
      } else {      // every load of this CTA has been used: its stages are free
        float4* to = reinterpret_cast<float4*>(smem + row * (RP + 4) * 4);
#pragma unroll
        for (int i = 0; i < RP; i += 4) to[i / 4] = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
    __syncwarp();
    if (p.split > 1) {
      cluster_sync_all();
      const int rows = kLTile / p.split;
      for (int i = threadIdx.x; i < rows * (RP / 4); i += kShrinkThreads) {
        const int row = rank * rows + i / (RP / 4), c = 4 * (i % (RP / 4)), slot = tile_slot(p.tiles, tile, row);
        const long long t = static_cast<long long>(row0) + row;
        if (t >= p.tiles.T || (slot < 0 ? pass > 0 : slot < first || slot >= first + n)) continue;
        const float4 v4 = cluster_sum4(smem_u32(smem) + 4 * (row * (RP + 4) + c), p.split);
        const float s = slot < 0 ? 0.0f : p.scales != nullptr ? p.scales[tile_adapter(p.tiles, tile, slot)] : p.scale;
        uint2 hi = make_uint2(0u, 0u), lo = make_uint2(0u, 0u);
        if (slot >= 0 && c < p.R) {
          split_bf16x2(make_float2(s * v4.x, s * v4.y), hi.x, lo.x);
          split_bf16x2(make_float2(s * v4.z, s * v4.w), hi.y, lo.y);
        }
        *reinterpret_cast<uint2*>(p.v + t * (2 * RP) + c) = hi;
        *reinterpret_cast<uint2*>(p.v + t * (2 * RP) + RP + c) = lo;
      }
      fence_proxy_async_smem();      // before the next unit's rows land there
      __syncwarp();
      cluster_sync_all();            // nobody goes on while another reads its sums
    }
    if (n > 0) {
      done += kb1 - kb0;
      unit_ph ^= 1;
    }
    if (++pass * SLOTS >= all) {
      pass = 0;
      ++tile;
    }
  }
  if (warp == 0) grid_dep_launch();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 128);
  if (threadIdx.x == 0 && *abort_flag != 0) *p.status = *abort_flag;
}

__device__ __forceinline__ uint8_t* aligned_smem(uint8_t* raw) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
}

template <int RP, bool WMN>
__global__ void __launch_bounds__(kShrinkThreads)
lora_shrink_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const ShrinkParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ LoraShare share;
  shrink_rows<RP, WMN>(tmX, tmW, p, blockIdx.x / p.split, gridDim.x / p.split, aligned_smem(smem_raw), share);
}

// ------------------------------------------------------------------------------------------------ expand
// out[t, n] = base[t, n] + sum_r v[t, r] W_l[n, r]; WMN: W_l lies (R, N) (the backward's A).  Persistent CTAs take items of a row tile and 256 columns (128
// where there is one for an SM at most) from a counter: SMs do not get equal shares of the memory's rate, and a copy of 470 MB that deals tiles out in
// turns takes 82 us, one that takes them from a counter 75.  What is claimed ahead is kept short: four items; with eight the half of a small call is dealt
// out at its start (16384 x 2816, rank 64: 36 and 39).  The base's boxes land where the result leaves from: an epilogue warp fetches its own, a few columns
// ahead whatever the adapters' products wait for; tensor memory holds four (columns, adapter) products.
// us: 8192 x 14336, rank 32, nine stretches of rows with an adapter each or none 82 (92 in equal shares by weight, 90 in items of 128 columns), 72 at the
// rate of a plain copy; 16384 x 2816, rank 64, 37 (36 with v rounded to one number, which leaves room for one base more); 16384 x 2048 without a base 23, 10
// at that rate, but writing alone gets 3.85 TB/s here: 17.
constexpr int kExpEpi = 8, kExpThreads = 96 + 32 * kExpEpi;      // warps: loads, products, epilogue, items
constexpr int kExpOut = 128 * 128 * 2;
template <int RP> constexpr int kExpBase = RP > 32 ? 3 : 4;
template <int RP> constexpr int kExpW = (RP > 64 ? 2 : 1) * kLBox;               // one adapter's 128 columns
template <int RP> constexpr int kExpV = (RP > 32 ? RP / 32 : 1) * kLBox;         // both halves of v
template <int RP> constexpr int kExpVs = RP > 64 ? 1 : 2;
template <int RP> constexpr int kExpWStages = RP > 64 ? 2 : 4;
constexpr int kExpQueue = 4;                     // items known ahead: as many as bases are fetched ahead, of single columns each
template <int RP> constexpr int kExpBars = kExpEpi * kExpBase<RP> + 2 * kExpWStages<RP> + 2 * kExpQueue + 12;
template <int RP> constexpr int kExpSmem = kExpBase<RP> * kExpOut + kExpWStages<RP> * kExpW<RP> + kExpVs<RP> * kExpV<RP> + kExpBars<RP> * 8 + 16 + 1024;

struct ExpandParams {
  LoraTiles tiles;
  int N, chunk, items, has_base;      // an item: `chunk` times 128 columns of a row tile, or what is left of them
  int* counter;                       // items that have been handed out, besides each CTA's first
  int* status;
};
struct ExpandItem {
  int tile, ct0, ct1, n;              // row tile (-1: no more), columns from 128 ct0 to 128 ct1, adapters
};

template <int RP, bool WMN>
__global__ void __launch_bounds__(kExpThreads, 1)
lora_expand_kernel(const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmBase,
                   const __grid_constant__ CUtensorMap tmOut, const ExpandParams p) {
  constexpr int WS = kExpWStages<RP>, W = kExpW<RP>, BASES = kExpBase<RP>, V = kExpV<RP>, VS = kExpVs<RP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t *s_w = smem + BASES * kExpOut, *s_v = s_w + WS * W;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_v + VS * V);
  const uint32_t bar_base = smem_u32(bars);      // [stage][epilogue warp]
  const uint32_t bar_wfull = bar_base + 8 * kExpEpi * BASES, bar_wempty = bar_wfull + 8 * WS;
  const uint32_t bar_tfull = bar_wempty + 8 * WS, bar_tempty = bar_tfull + 32, bar_v = bar_tempty + 32, bar_vfree = bar_v + 16;
  const uint32_t bar_qfull = bar_vfree + 16, bar_qempty = bar_qfull + 8 * kExpQueue;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kExpBars<RP>);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ ExpandItem queue[kExpQueue];
  __shared__ __align__(4) signed char slots[kExpQueue][kLTile];      // of the item's rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kExpEpi * BASES; ++s) mbar_init(bar_base + 8 * s, 1);
    for (int s = 0; s < WS; ++s) {
      mbar_init(bar_wfull + 8 * s, 1);
      mbar_init(bar_wempty + 8 * s, 1);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(bar_tfull + 8 * b, 1);
      mbar_init(bar_tempty + 8 * b, kExpEpi);
    }
    for (int b = 0; b < VS; ++b) {
      mbar_init(bar_v + 8 * b, 1);
      mbar_init(bar_vfree + 8 * b, 1);
    }
    for (int s = 0; s < kExpQueue; ++s) {
      mbar_init(bar_qfull + 8 * s, 1);
      mbar_init(bar_qempty + 8 * s, 2 + kExpEpi);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmBase);
    tma_prefetch_desc(&tmOut);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  grid_dep_wait();
  const int nct = (p.N + 127) / 128;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int ws = 0, buf = 0;                               // places in the rings, their phases
  uint32_t wph = 0, tph = 0, vs = 0;
  bool ok = true;

  if (warp == kExpThreads / 32 - 1) {                // hands out the items, the one after the next asked for already
    const int per_tile = (nct + p.chunk - 1) / p.chunk;
    int at = blockIdx.x, next = 0;
    for (int e = 0;; ++e) {
      if (lane == 0) next = atomicAdd(p.counter, 1) + gridDim.x;
      ExpandItem it{-1, 0, 0, 0};
      uint32_t slot4 = 0;
      if (at < p.items) {
        it.tile = at / per_tile;
        it.ct0 = (at - it.tile * per_tile) * p.chunk;
        it.ct1 = min(nct, it.ct0 + p.chunk);
        it.n = tile_n(p.tiles, it.tile);
#pragma unroll
        for (int i = 0; i < 4; ++i) slot4 |= (static_cast<uint32_t>(tile_slot(p.tiles, it.tile, 4 * lane + i)) & 0xffu) << (8 * i);
      }
      const int s = e % kExpQueue;
      if (!__all_sync(0xffffffffu, mbar_wait(bar_qempty + 8 * s, (e / kExpQueue & 1) ^ 1, abort_flag, ST_WAIT_PRODUCER))) break;
      if (lane == 0) queue[s] = it;
      reinterpret_cast<uint32_t*>(slots[s])[lane] = slot4;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_qfull + 8 * s);
      if (it.tile < 0) break;
      at = __shfl_sync(0xffffffffu, next, 0);
    }
    __syncwarp();
  }
  const int q = warp & 3, part = (warp - 2) >> 2;    // epilogue: the quarter of the rows, the half of the columns
  const uint32_t my_box = smem_u32(smem) + (4 * part + q) * 4096;
  const bool epilogue = warp >= 2 && warp < 2 + kExpEpi;
  // lane 0 of an epilogue warp: the base of the columns after those it fetched last
  ExpandItem ahead{0, 0, 0, 0};
  int ahead_e = -1;
  auto fetch_base = [&](int stage) {
    if (ahead.tile < 0) return;
    if (ahead.ct0 == ahead.ct1) {
      ++ahead_e;
      const bool known = mbar_wait(bar_qfull + 8 * (ahead_e % kExpQueue), ahead_e / kExpQueue & 1, abort_flag, ST_WAIT_EPILOGUE);
      ahead.tile = -1;
      if (known) ahead = queue[ahead_e % kExpQueue];
      if (ahead.tile < 0) return;
    }
    const uint32_t bar = bar_base + 8 * (kExpEpi * stage + warp - 2);
    mbar_arrive_expect_tx(bar, 4096);
    tma_load_3d(my_box + stage * kExpOut, &tmBase, bar, ahead.ct0 * 128 + 64 * part, ahead.tile * kLTile + 32 * q, 0);
    ++ahead.ct0;
  };
  if (p.has_base && epilogue && lane == 0)
    for (int i = 0; i < BASES; ++i) fetch_base(i);
  __syncwarp();
  int bs = 0;
  uint32_t bph = 0;
  bool before = false;                               // epilogue: there is a result before this one
  for (int e = 0; warp < 2 + kExpEpi; ++e) {
    const int qs = e % kExpQueue;
    if (!__all_sync(0xffffffffu, mbar_wait(bar_qfull + 8 * qs, e / kExpQueue & 1, abort_flag, ST_WAIT_PRODUCER))) break;
    const ExpandItem it = queue[qs];
    if (it.tile < 0) break;
    const int tile = it.tile, ct0 = it.ct0, ct1 = it.ct1, n = it.n;
    __syncwarp();
    if (warp == 0) {
      if (elect_one()) {
        if (n > 0) {
          ok = ok && mbar_wait(bar_vfree + 8 * (vs % VS), (vs / VS & 1) ^ 1, abort_flag, ST_WAIT_PRODUCER);
          if (ok) {
            mbar_arrive_expect_tx(bar_v + 8 * (vs % VS), V);
            for (int h = 0; h < V / kLBox; ++h) tma_load_3d(smem_u32(s_v + vs % VS * V) + h * kLBox, &tmV, bar_v + 8 * (vs % VS), 64 * h, tile * kLTile, 0);
          }
        }
        for (int ct = ct0; ct < ct1 && ok; ++ct) {
          for (int j = 0; j < n; ++j) {
            ok = mbar_wait(bar_wempty + 8 * ws, wph ^ 1, abort_flag, ST_WAIT_PRODUCER);
            if (!ok) break;
            const uint32_t full = bar_wfull + 8 * ws, to = smem_u32(s_w + ws * W);
            const int l = tile_adapter(p.tiles, tile, j);
            if constexpr (WMN) {      // RP rows of 64 columns each
              mbar_arrive_expect_tx(full, 2 * RP * 128);
              tma_load_3d(to, &tmW, full, ct * 128, 0, l);
              tma_load_3d(to + RP * 128, &tmW, full, ct * 128 + 64, 0, l);
            } else {
              mbar_arrive_expect_tx(full, W);
              for (int h = 0; h < W / kLBox; ++h) tma_load_3d(to + h * kLBox, &tmW, full, 64 * h, ct * 128, l);
            }
            if (++ws == WS) {
              ws = 0;
              wph ^= 1;
            }
          }
        }
      }
    } else if (warp == 1) {
      if (elect_one()) {
        constexpr uint32_t idesc = umma_idesc_bf16(128, 0, WMN);
        if (n > 0) {
          ok = ok && mbar_wait(bar_v + 8 * (vs % VS), vs / VS & 1, abort_flag, ST_WAIT_MMA_FULL);
        }
        const uint32_t sv = smem_u32(s_v + vs % VS * V);
        for (int u = 0; u < (ct1 - ct0) * n && ok; ++u) {
          ok = mbar_wait(bar_tempty + 8 * buf, tph ^ 1, abort_flag, ST_WAIT_MMA_TMEM) &&
               mbar_wait(bar_wfull + 8 * ws, wph, abort_flag, ST_WAIT_MMA_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sw = smem_u32(s_w + ws * W);
#pragma unroll
          for (int i = 0; i < RP / 8; ++i) {      // the nearest, then the rests
            const int k = i % (RP / 16);
            umma_bf16(tmem + 128 * buf, umma_desc_sw128(sv + (i >> 2) * kLBox + 32 * (i & 3), 0, 1024),
                      WMN ? umma_desc_sw128(sw + 2048 * k, RP * 128, 1024) : umma_desc_sw128(sw + (k >> 2) * kLBox + 32 * (k & 3), 0, 1024), idesc,
                      i != 0);
          }
          umma_commit(bar_wempty + 8 * ws);
          umma_commit(bar_tfull + 8 * buf);
          if (++ws == WS) {
            ws = 0;
            wph ^= 1;
          }
          if (++buf == 4) {
            buf = 0;
            tph ^= 1;
          }
        }
        if (n > 0 && ok) umma_commit(bar_vfree + 8 * (vs % VS));
      }
    } else {
      const int mine = slots[qs][32 * q + lane];
      const uint32_t taddr = tmem + (static_cast<uint32_t>(32 * q) << 16) + 64 * part;
      for (int ct = ct0; ct < ct1; ++ct) {
        float acc[64];
        if (n != 1) {
#pragma unroll
          for (int i = 0; i < 64; ++i) acc[i] = 0.0f;
        }
        for (int j = 0; j < n; ++j) {
          ok = ok && mbar_wait(bar_tfull + 8 * buf, tph, abort_flag, ST_WAIT_EPILOGUE);
          __syncwarp();
          tc_fence_after();
          if (n == 1 || __any_sync(0xffffffffu, mine == j)) {
            uint32_t r[2][32];
            tmem_ld32(taddr + 128 * buf, r[0]);
            tmem_ld32(taddr + 128 * buf + 32, r[1]);
            tmem_ld_wait();
            if (n == 1) {
#pragma unroll
              for (int i = 0; i < 64; ++i) acc[i] = mine == 0 ? __uint_as_float(r[i >> 5][i & 31]) : 0.0f;
            } else {
#pragma unroll
              for (int i = 0; i < 64; ++i) acc[i] = mine == j ? __uint_as_float(r[i >> 5][i & 31]) : acc[i];
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_tempty + 8 * buf);
          if (++buf == 4) {
            buf = 0;
            tph ^= 1;
          }
        }
        uint8_t* box = smem + bs * kExpOut + (4 * part + q) * 4096;
        if (p.has_base) ok = ok && mbar_wait(bar_base + 8 * (kExpEpi * bs + warp - 2), bph, abort_flag, ST_WAIT_EPILOGUE);
        else if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(BASES - 1) : "memory");      // the box's result of a round ago has left
        ok = __all_sync(0xffffffffu, ok);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint4* at = reinterpret_cast<uint4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4));
          uint32_t w[4] = {0u, 0u, 0u, 0u};
          if (p.has_base) {
            const uint4 b = *at;
            w[0] = b.x; w[1] = b.y; w[2] = b.z; w[3] = b.w;
          }
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const float2 f = unpack_bf16x2(w[h]);
            w[h] = pack_bf16x2(f.x + acc[8 * j + 2 * h], f.y + acc[8 * j + 2 * h + 1]);
          }
          *at = make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (ok && ct * 128 + 64 * part < p.N && tile * kLTile + 32 * q < p.tiles.T) tma_store_3d(&tmOut, smem_u32(box), ct * 128 + 64 * part, tile * kLTile + 32 * q, 0);
          bulk_commit_group();
          if (p.has_base && before) {      // the result before has left its box, which takes the base of columns to come
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            fetch_base(bs == 0 ? BASES - 1 : bs - 1);
          }
        }
        before = true;
        if (++bs == BASES) {
          bs = 0;
          bph ^= 1;
        }
      }
    }
    if (n > 0) ++vs;
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_qempty + 8 * qs);
  }
  grid_dep_launch();
  if (epilogue && lane == 0) bulk_wait_all();
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag != 0) *p.status = *abort_flag;
}

// ------------------------------------------------------------------------------------------------ gradients of the factors
// P_l[d, r] = sum over the rows t of adapter l of Y[t, d] V[t, r].  A CTA: one adapter, 128 columns d, a share of the adapter's rows in blocks of 64.  A block of
// neighbouring rows is two boxes of Y and those of V; of others four warps copy the 64 rows of the adapter's list into the same places, 16 bytes a lane.
// 16384 x 2048, rank 64: 17 us, 10.3 at the copy rate, and 3 for the shares' sum.  V's rests are columns of their own, so its 16 KB a block are read for each 128
// columns (16 us with the nearest numbers alone; 256 columns a CTA would need twice the shares and their sums).  Shares added up in clusters of eight
// instead took 31: so many large CTAs of one cluster do not find room at once.  8192 x 2048, rank 16, rows of 32 adapters mixed: 18 (267 where each
// adapter's CTAs visited every block that has a row of it and set the others' rows to zero); 3001 rows of three adapters one after another 7.6 (11).
constexpr int kWgThreads = 192;
template <int RP> constexpr int kWgV = (RP > 32 ? RP / 32 : 1) * 8192;
template <int RP> constexpr int kWgStages = RP > 64 ? 2 : RP > 32 ? 3 : 4;
template <int RP> constexpr int kWgSmem = kWgStages<RP> * (kLBox + kWgV<RP>) + (2 * kWgStages<RP> + 1) * 8 + 16 + 1024;

struct WgradParams {
  int T, D, R, L, splits, transposed;      // transposed: P is (R, D), else (D, R)
  LoraLists lists;                         // order: nullptr: all rows are adapter 0's
  const __nv_bfloat16 *y, *v;              // (T, D) at ldy, (T, 2 RP)
  long long ldy;
  void* out;                               // (splits, L, ...) fp32; one split: the gradient itself
  int out_f32;
  int* status;
};
// 16 bytes of global memory, or zeros, into shared memory
__device__ __forceinline__ void copy_16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(reinterpret_cast<uint64_t>(from)), "r"(there ? 16 : 0) : "memory");
}

template <int RP>
__device__ __forceinline__ void wgrad_rows(const CUtensorMap& tmY, const CUtensorMap& tmV, const WgradParams& p, int part, uint8_t* smem) {
  constexpr int NB = RP < 32 ? 64 : 2 * RP, ST = kWgStages<RP>, STAGE = kLBox + kWgV<RP>;      // columns: of V its nearest, then its rests
  constexpr int AHEAD = ST - 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + ST * STAGE);
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * ST, bar_tfull = bar_empty + 8 * ST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * ST + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool listed = p.lists.order != nullptr;
  const int chunks = (p.D + 127) / 128;
  const int chunk = part % chunks, l = part / chunks % p.L, split = part / chunks / p.L;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar_full + 8 * s, listed ? 4 : 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_tfull, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmY);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), NB);
    tmem_relinquish();
  }
  grid_dep_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int start = listed ? p.lists.bounds[l] : 0, rows = listed ? p.lists.bounds[l + 1] - start : l == 0 ? p.T : 0, all = (rows + 63) / 64;
  const int b0 = static_cast<int>(static_cast<long long>(split) * all / p.splits), n = static_cast<int>(static_cast<long long>(split + 1) * all / p.splits) - b0;
  const bool any = n > 0;
  bool ok = true;
  // one thread: a block of neighbouring rows
  auto boxes = [&](int s, int row) {
    const uint32_t full = bar_full + 8 * s, sy = smem_u32(smem + s * STAGE);
    mbar_arrive_expect_tx(full, STAGE);
    tma_load_3d(sy, &tmY, full, chunk * 128, row, 0);
    tma_load_3d(sy + 8192, &tmY, full, chunk * 128 + 64, row, 0);
    for (int h = 0; h < NB / 64; ++h) tma_load_3d(sy + kLBox + 8192 * h, &tmV, full, 64 * h, row, 0);
  };
  if (warp == 0) {
    if (!listed && elect_one())
      for (int b = 0; b < n; ++b) {
        if (!mbar_wait(bar_empty + 8 * (b % ST), (b / ST & 1) ^ 1, abort_flag, ST_WAIT_PRODUCER)) break;
        boxes(b % ST, 64 * (b0 + b));
      }
    grid_dep_launch();
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_bf16(NB, 1, 1);
      for (int b = 0; b < n && ok; ++b) {
        const int s = b % ST;
        ok = mbar_wait(bar_full + 8 * s, b / ST & 1, abort_flag, ST_WAIT_MMA_FULL);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sy = smem_u32(smem + s * STAGE), sv = sy + kLBox;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_bf16(tmem, umma_desc_sw128(sy + 2048 * k, 8192, 1024), umma_desc_sw128(sv + 2048 * k, 8192, 1024), idesc, b > 0 || k > 0);
        umma_commit(bar_empty + 8 * s);
      }
      if (ok && any) umma_commit(bar_tfull);
    }
  } else {
    if (listed) {            // a warp 16 rows of a block
      const int w = warp - 2;
      const int* order = p.lists.order + start;
      // lanes below 16: a row; lanes 16 and 17: the block's first and last; -1: there is none
      auto look = [&](int b) {
        const int i = 64 * (b0 + b) + (lane < 16 ? 16 * w + lane : lane == 16 ? 0 : 63);
        return b < n && i < rows ? order[i] : -1;
      };
      int next = look(0), sent = 0, b = 0;
      unsigned whole = 0;    // which of the last blocks are boxes
      auto arrived = [&](int upto) {
        fence_proxy_async_smem();
        __syncwarp();
        for (; sent < upto; ++sent)
          if (lane == 0 && (whole >> (sent & 31) & 1) == 0) mbar_arrive(bar_full + 8 * (sent % ST));
      };
      for (; b < n; ++b) {
        const int s = b % ST, mine = next;
        next = look(b + 1);
        const int head = __shfl_sync(0xffffffffu, mine, 16), tail = __shfl_sync(0xffffffffu, mine, 17);
        ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, (b / ST & 1) ^ 1, abort_flag, ST_WAIT_PRODUCER));
        if (!ok) break;
        if (tail - head == 63 && tail >= 0) {
          whole |= 1u << (b & 31);
          if (lane == 0) {
            if (w == 0) boxes(s, head);
            else mbar_arrive(bar_full + 8 * s);
          }
        } else {
          whole &= ~(1u << (b & 31));
          const uint32_t sy = smem_u32(smem + s * STAGE), sv = sy + kLBox;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = (32 * k + lane) >> 4, c = lane & 15, at = __shfl_sync(0xffffffffu, mine, r);
            const bool there = at >= 0 && chunk * 128 + 8 * c < p.D;
            copy_16(sy + (c >> 3) * 8192 + (16 * w + r) * 128 + (((c ^ r) & 7) << 4), there ? p.y + at * p.ldy + chunk * 128 + 8 * c : p.y, there);
          }
#pragma unroll
          for (int k = 0; k < RP / 8; ++k) {
            const int r = (32 * k + lane) / (RP / 4), c = (32 * k + lane) % (RP / 4), at = __shfl_sync(0xffffffffu, mine, r);
            copy_16(sv + (c >> 3) * 8192 + (16 * w + r) * 128 + (((c ^ r) & 7) << 4), at >= 0 ? p.v + static_cast<long long>(at) * (2 * RP) + 8 * c : p.v, at >= 0);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (b >= AHEAD) {
          asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
          arrived(b - AHEAD + 1);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      arrived(b);
    }
    const int q = warp & 3;
    if (any) ok = ok && mbar_wait(bar_tfull, 0, abort_flag, ST_WAIT_EPILOGUE);
    __syncwarp();
    tc_fence_after();
    // this CTA's sums into shared memory, whose stages have all been used
    const uint32_t taddr = tmem + (static_cast<uint32_t>(32 * q) << 16);
    float4* to = reinterpret_cast<float4*>(smem + (32 * q + lane) * (RP + 4) * 4);
#pragma unroll
    for (int c = 0; c < RP; c += 16) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.0f;
      if (any) lora_fetch<16>(taddr + c, true, v);
      float rest[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) rest[i] = 0.0f;
      if (any) lora_fetch<16>(taddr + RP + c, true, rest);
#pragma unroll
      for (int i = 0; i < 16; i += 4) to[(c + i) / 4] = make_float4(v[i] + rest[i], v[i + 1] + rest[i + 1], v[i + 2] + rest[i + 2], v[i + 3] + rest[i + 3]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // ... and out of it, four r a thread
  const int d0 = chunk * 128;
  const long long at = (static_cast<long long>(split) * p.L + l) * p.D * p.R;
  for (int i = threadIdx.x; i < 128 * (p.R / 4); i += kWgThreads) {
    const int row = p.transposed ? i % 128 : i / (p.R / 4), r = 4 * (p.transposed ? i / 128 : i % (p.R / 4));
    const float4 v = *reinterpret_cast<const float4*>(smem + 4 * (row * (RP + 4) + r));
    if (d0 + row >= p.D) continue;
    if (p.transposed) {
      const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const long long o = at + static_cast<long long>(r + h) * p.D + d0 + row;
        if (p.out_f32) static_cast<float*>(p.out)[o] = f[h];
        else static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(f[h]);
      }
    } else {
      const long long o = at + static_cast<long long>(d0 + row) * p.R + r;
      if (p.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + o) = v;
      else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    }
  }
  if (warp == 1) tmem_dealloc(tmem, NB);
  if (threadIdx.x == 0 && *abort_flag != 0) *p.status = *abort_flag;
}

template <int RP>
__global__ void __launch_bounds__(kWgThreads)
lora_wgrad_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmV, const WgradParams p) {
  extern __shared__ uint8_t smem_raw[];
  wgrad_rows<RP>(tmY, tmV, p, blockIdx.x, aligned_smem(smem_raw));
}

// Both products of the gradient g in one launch, shrink (u = g B) and wgrad (of B): by turns a cluster of the one and of the other, so that an SM has a
// CTA of each, one waits for memory while the other computes, and what one has read the other finds in L2.  16384 x 2816, rank 64: 31 us, one after the
// other 21 and 20.
constexpr int kBackThreads = kShrinkThreads;
static_assert(kShrinkThreads == kWgThreads, "roles of one launch");
template <int RP> constexpr int kBackSmem = kShrinkSmem > kWgSmem<RP> ? kShrinkSmem : kWgSmem<RP>;
template <int RP>
__global__ void __launch_bounds__(kBackThreads, 2)
lora_back_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmY,
                 const __grid_constant__ CUtensorMap tmV, const ShrinkParams p, const WgradParams w, int shrinks, int wgrads) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ LoraShare share;
  const int c = blockIdx.x / p.split, both = 2 * min(shrinks, wgrads);      // clusters of the roles
  const bool shrink = c < both ? (c & 1) == 0 : shrinks > wgrads;
  const int part = c < both ? c >> 1 : c - both / 2;
  if (shrink) shrink_rows<RP, true>(tmX, tmW, p, part, shrinks, aligned_smem(smem_raw), share);
  else if (const int at = part * p.split + static_cast<int>(blockIdx.x) % p.split; at < (w.D + 127) / 128 * w.L * w.splits)      // the last cluster may have more CTAs
    wgrad_rows<RP>(tmY, tmV, w, at, aligned_smem(smem_raw));
}

// the sum of the splits' shares, n values (a multiple of 4), always in the same order; eight of them are on their way at a time
__global__ void __launch_bounds__(128) lora_wgrad_sum_kernel(const float* part, int splits, long long n, void* out, int out_f32) {
  grid_dep_begin();
  const long long i = 4 * (static_cast<long long>(blockIdx.x) * 128 + threadIdx.x);
  if (i >= n) return;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s = 0; s < splits; s += 8) {
    float4 o[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) o[u] = s + u < splits ? *reinterpret_cast<const float4*>(part + (s + u) * n + i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      v.x += o[u].x; v.y += o[u].y; v.z += o[u].z; v.w += o[u].w;
    }
  }
  if (out_f32) *reinterpret_cast<float4*>(static_cast<float*>(out) + i) = v;
  else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + i) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

// ------------------------------------------------------------------------------------------------ few rows
// A cluster of eight CTAs (four, where there are many groups) takes up to sixteen rows of one adapter, and a share of the columns, where such groups are fewer than
// SMs: each CTA multiplies an eighth of the rows with all of A_l, the sums meet in distributed shared memory, and each expands its columns.  Both products are m16n8k16
// instructions; the order of the reduction index within one is free as long as both operands have it, so a lane's share of x and A_l is 16 neighbouring
// bytes of global memory, of B_l 8 of shared memory.  v is never rounded: it is split into two bf16 numbers that hold 16 bits of it.
// Bound by latency: each warp's bulk copies of its first columns of B_l and of the base are on their way while x and A_l are multiplied, and its result
// leaves from where the base landed.  us, L2 warm: one row, 4096 x 4096, rank 16 4.9; 64 rows of 32 adapters, 4096 x 14336 12.9 (17.9 with columns handed out
// to the CTA's warps in turns, 30 with columns fetched into registers four tiles ahead).
constexpr int kFewThreads = 256, kFewSm = 3, kFewWarps = kFewThreads / 32, kFewRows = 16, kFewMost = 512, kFewInline = 128;
constexpr int kFewChunk = 7680;          // of a warp: columns of B_l, and of the base and the result of each row
static int few_smem(int64_t R) { return static_cast<int>(kFewWarps * kFewChunk + kFewRows * R * 4 + std::max<int64_t>(4096, (R + 15) / 16 * 1024)); }

// A cluster's rows.  The rows are ranked among those of their adapter (or of none); sixteen ranks make a group, in the order of their first rows.  Up to
// kFewInline rows every CTA finds its group by itself; of more a kernel before ranks them, which costs 3 us and in every CTA took up to 10.
struct FewRank { int adapter, rank; };
struct __align__(16) FewGroup {
  int adapter[kFewInline];
  int rank[kFewInline];
  unsigned first[kFewInline / 32];      // rows that begin a group
  int rows[kFewRows];
  int n, l;
};
// groups at most: one for each sixteen rows and one more for each adapter and for none
static int few_groups(const LoraIndex& ix) {
  const int more = ix.index == nullptr || ix.T == 1 ? 0 : ix.L + 1;
  return std::min(ix.T, (ix.T + kFewRows - 1) / kFewRows + more);
}
// a row's rank among those of its adapter, by a whole warp for its 32 rows
__device__ __forceinline__ int few_rank(const int* adapters, int t) {
  const int l = adapters[t];
  int rank = __popc(__match_any_sync(0xffffffffu, l) & ((1u << (t & 31)) - 1u));
#pragma unroll 4
  for (int j = 0; j < (t >> 5) * 8; ++j) {      // the warps' rows before
    const int4 o = reinterpret_cast<const int4*>(adapters)[j];
    rank += (o.x == l) + (o.y == l) + (o.z == l) + (o.w == l);
  }
  return rank;
}
// one CTA: ranks (T), and of each of `groups` groups the adapter and the first rank, -1 where there is no such group
__global__ void __launch_bounds__(kFewMost) lora_rank_kernel(const LoraIndex ix, FewRank* ranks, FewRank* leaders, int groups) {
  grid_dep_wait();
  __shared__ __align__(16) int adapters[kFewMost];
  __shared__ int before[kFewMost / 32];
  const int t = threadIdx.x;
  const int l = t < ix.T ? lora_adapter(ix, t) : -2;
  adapters[t] = l;
  __syncthreads();
  const int rank = few_rank(adapters, t);
  const bool first = t < ix.T && rank % kFewRows == 0;
  const unsigned m = __ballot_sync(0xffffffffu, first);
  if ((t & 31) == 0) before[t >> 5] = __popc(m);
  if (t < ix.T) ranks[t] = FewRank{l, rank};
  __syncthreads();
  int n = __popc(m & ((1u << (t & 31)) - 1u)), all = 0;
  for (int w = 0; w < kFewMost / 32; ++w) {
    if (w < (t >> 5)) n += before[w];
    all += before[w];
  }
  if (first) leaders[n] = FewRank{l, rank};
  if (t >= all && t < groups) leaders[t] = FewRank{-1, -1};
  grid_dep_launch();
}
// Returns the number of the group's rows, 0: there is no such group.  Barriers inside.
__device__ __forceinline__ int few_group(const LoraIndex& ix, const FewRank* ranks, const FewRank* leaders, int group, FewGroup& s) {
  const int t = threadIdx.x;
  if (ix.index == nullptr || ix.T == 1) {
    const int n = max(0, min(kFewRows, ix.T - kFewRows * group));
    if (t == 0) s.l = lora_adapter(ix, 0);
    if (t < n) s.rows[t] = kFewRows * group + t;
    __syncthreads();
    return n;
  }
  if (t == 0) s.n = 0;
  if (ranks != nullptr) {
    const FewRank lead = leaders[group];
    FewRank r[kFewMost / kFewThreads];
#pragma unroll
    for (int i = 0; i < kFewMost / kFewThreads; ++i) {
      r[i] = FewRank{-2, -2};
      if (t + i * kFewThreads < ix.T) r[i] = ranks[t + i * kFewThreads];
    }
    __syncthreads();
    if (lead.rank < 0) return 0;
#pragma unroll
    for (int i = 0; i < kFewMost / kFewThreads; ++i)
      if (r[i].adapter == lead.adapter && r[i].rank >= lead.rank && r[i].rank < lead.rank + kFewRows) {
        s.rows[r[i].rank - lead.rank] = t + i * kFewThreads;
        atomicAdd(&s.n, 1);
      }
    if (t == 0) s.l = lead.adapter;
    __syncthreads();
    return s.n;
  }
  int l = -2, rank = 0;
  if (t < kFewInline) s.adapter[t] = l = t < ix.T ? lora_adapter(ix, t) : -2;
  __syncthreads();
  if (t < kFewInline) {
    s.rank[t] = rank = few_rank(s.adapter, t);
    const unsigned m = __ballot_sync(0xffffffffu, t < ix.T && rank % kFewRows == 0);
    if ((t & 31) == 0) s.first[t >> 5] = m;
  }
  __syncthreads();
  int leader = -1, skip = group;      // the group-th of the bits
#pragma unroll
  for (int w = 0; w < kFewInline / 32; ++w) {
    unsigned m = s.first[w];
    const int c = __popc(m);
    if (leader < 0 && skip < c) {
      for (int i = 0; i < skip; ++i) m &= m - 1;
      leader = 32 * w + __ffs(m) - 1;
    }
    skip -= c;
  }
  if (leader < 0) return 0;
  const int from = s.rank[leader], of = s.adapter[leader];
  if (t < kFewInline && l == of && rank >= from && rank < from + kFewRows) {
    s.rows[rank - from] = t;
    atomicAdd(&s.n, 1);
  }
  if (t == 0) s.l = of;
  __syncthreads();
  return s.n;
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
struct FewLora {
  LoraIndex ix;
  const __nv_bfloat16 *x, *a, *b, *base;
  __nv_bfloat16* out;
  long long ldx, ldb;
  const FewRank *ranks, *leaders;      // of lora_rank_kernel, or nullptr
  int K, N, R, parts;
  const float* scales;
  float scale;
};

// KS: steps of 16 r, 0: any number of them; CTAS: of a cluster
template <int KS, int CTAS>
__global__ void __launch_bounds__(kFewThreads, kFewSm) lora_few_kernel(const FewLora p) {
  extern __shared__ __align__(128) uint8_t smem[];                 // a chunk a warp, sums, and (by turns) partial sums or v as fragments
  __shared__ FewGroup group;
  __shared__ __align__(8) uint64_t bars[kFewWarps];
  __shared__ int abort_word;
  float* sums = reinterpret_cast<float*>(smem + kFewWarps * kFewChunk);    // of this CTA, [row][r]
  float* part = sums + kFewRows * p.R;                             // [warp][row][8 r]
  uint32_t* frag = reinterpret_cast<uint32_t*>(part);              // [16 r][lane][4 upper, 4 lower halves]
  if (threadIdx.x == 0) {
    for (int i = 0; i < kFewWarps; ++i) mbar_init(smem_u32(bars + i), 1);
    abort_word = 0;
    fence_mbar_init();
  }
  grid_dep_begin();
  const int rank = static_cast<int>(cluster_ctarank()), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int c = static_cast<int>(cluster_id_x());
  const int n = few_group(p.ix, p.ranks, p.leaders, c / p.parts, group);
  if (n == 0) return;                                              // the whole cluster
  const int l = group.l;
  // this warp's columns, in chunks of `wide`
  const int share = (c % p.parts * CTAS + rank) * kFewWarps + warp, shares = p.parts * CTAS * kFewWarps;
  const int col0 = 8 * static_cast<int>(static_cast<long long>(share) * (p.N / 8) / shares);
  const int col1 = 8 * static_cast<int>(static_cast<long long>(share + 1) * (p.N / 8) / shares);
  const int wide = kFewChunk / (2 * p.R + 2 * n) & ~7, ksteps = KS > 0 ? KS : (p.R + 15) / 16;
  uint8_t *chunk = smem + warp * kFewChunk, *rows = chunk + wide * p.R * 2;      // rows: the base's, then the result's
  const uint32_t full = smem_u32(bars + warp);
  const bool copies = l >= 0 || p.base != nullptr;
  auto fetch = [&](int col) {                                      // a lane a row
    const int w = min(wide, col1 - col);
    if (lane == 0) {
      mbar_arrive_expect_tx(full, (l >= 0 ? w * p.R * 2 : 0) + (p.base != nullptr ? n * w * 2 : 0));
      if (l >= 0) bulk_load_1d(smem_u32(chunk), p.b + (static_cast<long long>(l) * p.N + col) * p.R, w * p.R * 2, full);
    }
    __syncwarp();
    if (p.base != nullptr && lane < n) bulk_load_1d(smem_u32(rows) + lane * wide * 2, p.base + group.rows[lane] * p.ldb + col, w * 2, full);
  };
  if (copies && col0 < col1) fetch(col0);

  if (l >= 0) {
    const bool low = g < n, high = g + 8 < n;
    const __nv_bfloat16 *x0 = p.x + (low ? group.rows[g] : 0) * p.ldx, *x1 = p.x + (high ? group.rows[g + 8] : 0) * p.ldx;
    // tiles of eight r, and where these are fewer than warps, several warps a tile that split the columns
    const int rt = p.R / 8, split = rt < kFewWarps ? kFewWarps / rt : 1;
    const int steps = (p.K + 31) / 32;
    const int s0 = rank * steps / CTAS, s1 = (rank + 1) * steps / CTAS;
    for (int tile = warp % (rt * split) / split; tile < rt && warp < rt * split; tile += kFewWarps / split) {
      const int w = split > 1 ? warp % split : 0;
      const int first = s0 + w * (s1 - s0) / split, last = s0 + (w + 1) * (s1 - s0) / split;
      const __nv_bfloat16* a = p.a + (static_cast<long long>(l) * p.R + 8 * tile + g) * p.K;
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int s = first; s < last; ++s) {
        const int k = 32 * s + 8 * q;
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        const uint4 av = k < p.K ? *reinterpret_cast<const uint4*>(a + k) : zero;
        const uint4 u0 = k < p.K && low ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
        const uint4 u1 = k < p.K && high ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
        mma_bf16(d, u0.x, u1.x, u0.y, u1.y, av.x, av.y);
        mma_bf16(d, u0.z, u1.z, u0.w, u1.w, av.z, av.w);
      }
      // one warp a tile: to its place, else to the warps that add up
      float* to = split > 1 ? part + warp * (kFewRows * 8) : sums + 8 * tile;
      const int pitch = split > 1 ? 8 : p.R;
      *reinterpret_cast<float2*>(to + g * pitch + 2 * q) = make_float2(d[0], d[1]);
      *reinterpret_cast<float2*>(to + (g + 8) * pitch + 2 * q) = make_float2(d[2], d[3]);
    }
    if (split > 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < rt * kFewRows * 8; i += kFewThreads) {
        const int tile = i >> 7, at = i & 127;
        float s = 0.0f;
        for (int w = 0; w < split; ++w) s += part[(tile * split + w) * (kFewRows * 8) + at];
        sums[(at >> 3) * p.R + 8 * tile + (at & 7)] = s;
      }
    }
    __syncwarp();
    cluster_sync_all();
    // v of the whole row as the fragments that the second product reads: of each 16 r lane (g, q) holds 4 q ... 4 q + 3 of rows g and g + 8
    const float scale = p.scales != nullptr ? p.scales[l] : p.scale;
    for (int i = threadIdx.x; i < ksteps * 128; i += kFewThreads) {
      const int h = i & 3, at = i >> 2 & 31, row = (at >> 2) + 8 * (h & 1), r = 16 * (i >> 7) + 4 * (at & 3) + 2 * (h >> 1);
      float2 s = make_float2(0.0f, 0.0f);
      if (row < n && r < p.R) {
#pragma unroll
        for (int k = 0; k < CTAS; ++k) {
          float2 o;
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                       : "=f"(o.x), "=f"(o.y)
                       : "r"(mapa_shared(smem_u32(sums + row * p.R + r), k))
                       : "memory");
          s.x += o.x;
          s.y += o.y;
        }
      }
      split_bf16x2(make_float2(s.x * scale, s.y * scale), frag[(i >> 7) * 256 + at * 8 + h], frag[(i >> 7) * 256 + at * 8 + 4 + h]);
    }
    __syncthreads();
  }

  uint4 hi[KS > 0 ? KS : 1], lo[KS > 0 ? KS : 1];
  if (KS > 0 && l >= 0) {
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      hi[k] = *reinterpret_cast<const uint4*>(frag + k * 256 + lane * 8);
      lo[k] = *reinterpret_cast<const uint4*>(frag + k * 256 + lane * 8 + 4);
    }
  }
  uint32_t phase = 0;
  for (int col = col0; col < col1; col += wide, phase ^= 1) {
    const int w = min(wide, col1 - col);
    if (copies) mbar_wait(full, phase, &abort_word, ST_WAIT_ROWS);
    __syncwarp();
    constexpr int TILES = 4;                                       // of a warp at a time, fewer at the end
    const bool half = (p.R & 8) != 0 && q >= 2;                    // the last 16 r have 8 that are not there
    auto group_of_tiles = [&](int tile0, int tiles, auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      float d[TILES][4] = {};
      if (l >= 0) {
        const uint8_t* b = chunk + (8 * tile0 + g) * p.R * 2 + 8 * q;
        const int pitch = 16 * p.R;
        auto step = [&](int k, const uint4& u, const uint4& v) {
          const bool in = !(half && k == ksteps - 1);
          uint2 bw[TILES];
#pragma unroll
          for (int j = 0; j < TILES; ++j) bw[j] = in && (WHOLE || j < tiles) ? *reinterpret_cast<const uint2*>(b + j * pitch + 32 * k) : make_uint2(0u, 0u);
#pragma unroll
          for (int j = 0; j < TILES; ++j) mma_bf16(d[j], v.x, v.y, v.z, v.w, bw[j].x, bw[j].y);
#pragma unroll
          for (int j = 0; j < TILES; ++j) mma_bf16(d[j], u.x, u.y, u.z, u.w, bw[j].x, bw[j].y);
        };
        if constexpr (KS > 0) {
#pragma unroll
          for (int k = 0; k < KS; ++k) step(k, hi[k], lo[k]);
        } else {
          for (int k = 0; k < ksteps; ++k)
            step(k, *reinterpret_cast<const uint4*>(frag + k * 256 + lane * 8), *reinterpret_cast<const uint4*>(frag + k * 256 + lane * 8 + 4));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (8 * h >= n) break;
        uint32_t* at = reinterpret_cast<uint32_t*>(rows + (g + 8 * h) * wide * 2 + (8 * tile0 + 2 * q) * 2);
        if (g + 8 * h < n) {
          uint32_t o[TILES] = {};
          if (p.base != nullptr)
#pragma unroll
            for (int j = 0; j < TILES; ++j)
              if (WHOLE || j < tiles) o[j] = at[4 * j];
#pragma unroll
          for (int j = 0; j < TILES; ++j) {
            const float2 f = unpack_bf16x2(o[j]);
            if (WHOLE || j < tiles) at[4 * j] = pack_bf16x2(f.x + d[j][2 * h], f.y + d[j][2 * h + 1]);
          }
        }
      }
    };
    for (int tile0 = 0; tile0 < w / 8; tile0 += TILES) {
      if (tile0 + TILES <= w / 8) group_of_tiles(tile0, TILES, std::true_type());
      else group_of_tiles(tile0, w / 8 - tile0, std::false_type());
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane < n) bulk_store_1d(p.out + static_cast<long long>(group.rows[lane]) * p.N + col, smem_u32(rows) + lane * wide * 2, w * 2);
    bulk_commit_group();
    if (col + wide < col1) {
      bulk_wait_read_all();
      __syncwarp();
      if (copies) fetch(col + wide);
    }
  }
  bulk_wait_all();
  __syncwarp();
  cluster_sync_all();      // nobody leaves while another reads its sums, and every warp's waits are over
  if (threadIdx.x == 0 && abort_word != 0) *p.ix.status = abort_word;
}

// ------------------------------------------------------------------------------------------------ host
static int padded_rank(int64_t R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }
template <class F>
static int by_rank(int rp, F f) {
  if (rp == 16) return f(std::integral_constant<int, 16>());
  if (rp == 32) return f(std::integral_constant<int, 32>());
  if (rp == 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}

// CTAs that share the columns of a unit, for so many CTAs at a time
static int shrink_split(int64_t T, int64_t D, int64_t ctas) {
  const int64_t tiles = ceil_div(T, kLTile), blocks = ceil_div(D, 64);
  int split = 1;
  while (split < 8 && tiles * split * 2 <= ctas && blocks >= 4 * split) split *= 2;
  return split;
}
// `sms`: those that a call's grids are made for, gemm_cta_budget() at its start: the row tiles' kernels are persistent, and SMs reserved for an exchange are not
// theirs.  Workspaces are sized for num_sms(), which never gives fewer shares.
// W: (L,R,D), or (wmn) (L,D,R); split: 0, or that of the gradients' launch
static int lora_shrink(const void* X, int64_t ldx, const void* W, bool wmn, int64_t L, ShrinkParams p, int sms, cudaStream_t st) {
  return by_rank(padded_rank(p.R), [&](auto rp) -> int {
    constexpr int RP = decltype(rp)::value;
    const int64_t T = p.tiles.T, tiles = p.tiles.tiles;
    CUtensorMap tmX, tmW;
    int rc = make_map(&tmX, X, p.D, T, 1, ldx, ldx * T, 64, kLTile);
    if (rc == 0) rc = wmn ? make_map(&tmW, W, p.R, p.D, L, p.R, static_cast<int64_t>(p.R) * p.D, 64, 64)
                          : make_map(&tmW, W, p.D, p.R, L, p.D, static_cast<int64_t>(p.R) * p.D, 64, RP);
    if (rc) return rc;
    const int columns = wmn && RP < 64 ? 64 : RP;      // of an adapter; as many adapters as make 128 share a unit
    const int64_t slots = std::min<int64_t>(128 / columns, L), units = tiles * ceil_div(std::min<int64_t>(L, kLTile), slots);      // at most
    if (p.split == 0) p.split = shrink_split(T, p.D, 2 * sms);
    const int64_t clusters = std::min<int64_t>(units, 2 * sms / p.split);
    p.stage = kLBox + static_cast<int>(slots) * columns * 128;
    p.stages = std::min(kShrinkMost, kShrinkRing / p.stage);
    auto run = [&](auto mn) -> int {
      constexpr bool MN = decltype(mn)::value;
      static PerDevice allowed;
      B200_CUDA(allow_smem(allowed, lora_shrink_kernel<RP, MN>, kShrinkSmem));
      B200_CUDA(launch_chained(lora_shrink_kernel<RP, MN>, static_cast<int>(clusters * p.split), kShrinkThreads, kShrinkSmem, st, p.split, tmX, tmW, p));
      return 0;
    };
    return wmn ? run(std::true_type()) : run(std::false_type());
  });
}

// W: (L,N,R), or (wmn) (L,R,N)
static int lora_expand(const void* V, const void* W, bool wmn, int64_t L, int64_t R, const void* base, int64_t ldb, void* out, ExpandParams p, int sms, cudaStream_t st) {
  return by_rank(padded_rank(R), [&](auto rp) -> int {
    constexpr int RP = decltype(rp)::value;
    CUtensorMap tmV, tmW, tmB, tmO;
    const int64_t T = p.tiles.T, N = p.N;
    int rc = make_map(&tmV, V, 2 * RP, T, 1, 2 * RP, T * (2 * RP), 64, kLTile);
    if (rc == 0) rc = wmn ? make_map(&tmW, W, N, R, L, N, N * R, 64, RP) : make_map(&tmW, W, R, N, L, R, N * R, 64, 128);
    if (rc == 0) rc = make_map(&tmO, out, N, T, 1, N, N * T, 64, 32);
    tmB = tmO;
    if (rc == 0 && base != nullptr) rc = make_map(&tmB, base, N, T, 1, ldb, ldb * T, 64, 32);
    if (rc) return rc;
    p.has_base = base != nullptr;
    p.chunk = p.tiles.tiles * ceil_div(N, 128) <= sms ? 1 : 2;
    p.items = static_cast<int>(p.tiles.tiles * ceil_div(ceil_div(N, 128), p.chunk));
    const int grid = static_cast<int>(std::min<int64_t>(sms, p.items));
    auto run = [&](auto mn) -> int {
      constexpr bool MN = decltype(mn)::value;
      static PerDevice allowed;
      B200_CUDA(allow_smem(allowed, lora_expand_kernel<RP, MN>, kExpSmem<RP>));
      B200_LAUNCH((lora_expand_kernel<RP, MN>), grid, kExpThreads, kExpSmem<RP>, st, tmV, tmW, tmB, tmO, p);
      return 0;
    };
    return wmn ? run(std::true_type()) : run(std::false_type());
  });
}

// Shares of the rows: as many as it takes for two CTAs an SM, each with eight blocks of rows at least
static int wgrad_splits(int64_t T, int64_t D, int64_t L, int sms) {
  const int64_t blocks = ceil_div(T, 64), ctas = ceil_div(D, 128) * L;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2 * sms / ctas, blocks / 8)));
}
// The same for the gradient of B, which shares its launch with u = g B where that is wanted: one CTA an SM of either role.  By itself it has as many shares,
// so that its bits do not depend on what else is asked for.
static int back_wgrad_splits(int64_t T, int64_t D, int64_t L, int sms) {
  const int64_t blocks = ceil_div(T, 64), ctas = ceil_div(D, 128) * L;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms / ctas, blocks / 8)));
}
static int lora_wgrad(const void* Y, int64_t ldy, const void* V, int splits, WgradParams p, float* ws, void* out, int out_f32, cudaStream_t st) {
  return by_rank(padded_rank(p.R), [&](auto rp) -> int {
    constexpr int RP = decltype(rp)::value;
    CUtensorMap tmY, tmV;
    int rc = make_map(&tmY, Y, p.D, p.T, 1, ldy, ldy * p.T, 64, 64);
    if (rc == 0) rc = make_map(&tmV, V, 2 * RP, p.T, 1, 2 * RP, static_cast<int64_t>(p.T) * (2 * RP), 64, 64);
    if (rc) return rc;
    p.splits = splits;
    p.y = static_cast<const __nv_bfloat16*>(Y);
    p.v = static_cast<const __nv_bfloat16*>(V);
    p.ldy = ldy;
    p.out = p.splits > 1 ? static_cast<void*>(ws) : out;
    p.out_f32 = p.splits > 1 || out_f32;
    static PerDevice allowed;
    B200_CUDA(allow_smem(allowed, lora_wgrad_kernel<RP>, kWgSmem<RP>));
    B200_LAUNCH(lora_wgrad_kernel<RP>, static_cast<int>(ceil_div(p.D, 128) * p.L * p.splits), kWgThreads, kWgSmem<RP>, st, tmY, tmV, p);
    if (p.splits > 1) {
      const long long n = static_cast<long long>(p.L) * p.D * p.R;
      B200_LAUNCH(lora_wgrad_sum_kernel, static_cast<int>(ceil_div(n, 512)), 128, 0, st, static_cast<const float*>(ws), p.splits, n, out, out_f32);
    }
    return 0;
  });
}

// The launch of both: an SM holds a CTA of each role
static int lora_back(const void* G, const void* B, const void* V, int64_t L, ShrinkParams p, WgradParams w, int splits, int sms, float* ws, void* out, int out_f32,
                     cudaStream_t st) {
  return by_rank(padded_rank(p.R), [&](auto rp) -> int {
    constexpr int RP = decltype(rp)::value;
    const int64_t T = p.tiles.T, D = p.D, tiles = p.tiles.tiles;
    CUtensorMap tmX, tmW, tmY, tmV;
    int rc = make_map(&tmX, G, D, T, 1, D, D * T, 64, kLTile);
    if (rc == 0) rc = make_map(&tmW, B, p.R, D, L, p.R, static_cast<int64_t>(p.R) * D, 64, 64);
    if (rc == 0) rc = make_map(&tmY, G, D, T, 1, D, D * T, 64, 64);
    if (rc == 0) rc = make_map(&tmV, V, 2 * RP, T, 1, 2 * RP, T * (2 * RP), 64, 64);
    if (rc) return rc;
    const int columns = RP < 64 ? 64 : RP;
    const int64_t slots = std::min<int64_t>(128 / columns, L), units = tiles * ceil_div(std::min<int64_t>(L, kLTile), slots);
    const int64_t shrinks = std::min<int64_t>(units, sms / p.split);
    p.stage = kLBox + static_cast<int>(slots) * columns * 128;
    p.stages = std::min(kShrinkMost, kShrinkRing / p.stage);
    w.splits = splits;
    w.y = static_cast<const __nv_bfloat16*>(G);
    w.v = static_cast<const __nv_bfloat16*>(V);
    w.ldy = D;
    w.out = w.splits > 1 ? static_cast<void*>(ws) : out;
    w.out_f32 = w.splits > 1 || out_f32;
    const int64_t wgrads = ceil_div(ceil_div(D, 128) * L * w.splits, p.split);
    static PerDevice allowed;
    B200_CUDA(allow_smem(allowed, lora_back_kernel<RP>, kBackSmem<RP>));
    B200_CUDA(launch_chained(lora_back_kernel<RP>, static_cast<int>((shrinks + wgrads) * p.split), kBackThreads, kBackSmem<RP>, st, p.split, tmX, tmW, tmY, tmV,
                             p, w, static_cast<int>(shrinks), static_cast<int>(wgrads)));
    if (w.splits > 1) {
      const long long n = static_cast<long long>(L) * D * p.R;
      B200_LAUNCH(lora_wgrad_sum_kernel, static_cast<int>(ceil_div(n, 512)), 128, 0, st, static_cast<const float*>(ws), w.splits, n, out, out_f32);
    }
    return 0;
  });
}

struct LoraCarver {
  char* base;
  size_t off = 0;
  template <class T>
  T* take(int64_t n) {
    off = (off + 255) & ~static_cast<size_t>(255);
    T* p = base != nullptr ? reinterpret_cast<T*>(base + off) : nullptr;
    off += static_cast<size_t>(n) * sizeof(T);
    return p;
  }
};
struct LoraKept {
  __nv_bfloat16* v;
  LoraTiles tiles;
  LoraLists lists;
  int* counter;
};
// index: the call has one
static LoraKept carve_lora(int64_t T, int64_t R, int64_t L, bool index, int keep, void* ws, size_t* bytes) {
  LoraCarver c{static_cast<char*>(ws)};
  LoraKept k{};
  const int64_t tiles = ceil_div(T, kLTile);
  k.v = c.take<__nv_bfloat16>(2 * T * padded_rank(R));
  k.counter = c.take<int>(1);
  k.tiles.T = static_cast<int>(T);
  k.tiles.tiles = static_cast<int>(tiles);
  if (index) {
    k.tiles.n = c.take<int>(tiles);
    k.tiles.adapter = c.take<int>(tiles * kLTile);
    k.tiles.slot = c.take<short>(tiles * kLTile);
    if (keep) {
      k.lists.order = c.take<int>(T);
      k.lists.bounds = c.take<int>(L + 1);
    }
  }
  *bytes = c.off;
  return k;
}
// Whether the kernel of few rows takes a call.  us, few rows / row tiles, L2 warm.  One adapter, 4096 x 14336, rank 16: 16 rows 8.4 / 10.0, 128 rows 9.8 /
// 10.5, 256 rows 14.4 / 11.8; 2048 x 2816, rank 64: 16 rows 9.3 / 9.5, 64 rows 11.4 / 9.4.  Several, 4096 x 4096, rank 16: rows of 32 adapters mixed 64 rows
// 8.7 / 22.5, 512 rows 15.9 / 28.7; of two packed 7.6 / 13.6 and 13.1 / 14.5.  The rule does not see that few adapters of a high rank are better in row tiles.  Up to 128
// rows it loses nothing up to rank 64 (4096 x 4096, rank 64, 128 rows of two packed 15.5 / 15.4) and a tenth at rank 128, but 2048 x 2816, two packed, 256 and 512 rows: rank 32 13.5 / 13.4 and 14.4 / 13.8, rank 64 17.8 / 14.3 and 18.8 / 14.9, rank 128
// 26.2 / 15.9 and 28.2 / 16.7; eight mixed, 512 rows: rank 64 20.1 / 18.1, rank 128 38.1 / 23.8.  With 32 mixed it is right at every rank: 24.0 / 40.0 and 47.7 / 73.1.
static bool lora_few(int64_t T, int64_t R, int64_t L, int keep) { return !keep && T <= (L > 1 ? kFewMost : R <= 32 ? 128 : 16); }

// CTAs of a cluster: eight, and four where the clusters of all groups there may be would not be on the SMs at once although a warp's columns fit one chunk, or
// would come round twice.  us, eight / four: 2048 x 2816, rank 16, 512 rows of 32 adapters 14.9 / 13.1, 128 rows of 128 16.8 / 9.5, 64 rows of 8 7.6 / 7.7; 4096 x
// 14336, 64 rows of 64 12.8 / 16.6, 512 rows of 32 26 / 29, 128 rows of 128 27 / 22; 4096 x 4096, 512 rows of 32 15.7 / 17.0, 256 rows of 128 27.5 / 24.0.
static int few_cluster(int64_t T, int64_t N, int64_t R, int64_t L, int64_t groups, int sms) {
  const int64_t room = static_cast<int64_t>(sms) * kFewSm, rows = std::min<int64_t>(kFewRows, ceil_div(T, L));
  const bool fits = N * 2 * (R + rows) <= 4 * kFewWarps * kFewChunk;
  return groups * 8 > (fits ? room : 2 * room) ? 4 : 8;
}

}  // namespace b200moe

using namespace b200moe;

static int check_lora(const char* who, int64_t T, int64_t K, int64_t N, int64_t R, int64_t L) {
  CHECK_DIM8(K);
  CHECK_DIM8(N);
  B200_CHECK_ARG(R >= 8 && R % 8 == 0 && R <= 128, B200MOE_E_UNSUPPORTED, "%s: rank %lld, supported are multiples of 8 up to 128", who, (long long)R);
  B200_CHECK_ARG(T >= 0 && T < (1LL << 31) - 256 && K < (1LL << 31) - 256 && N < (1LL << 31) - 256, B200MOE_E_BAD_SHAPE,
                 "%s: %lld rows, %lld -> %lld", who, (long long)T, (long long)K, (long long)N);
  B200_CHECK_ARG(L >= 1 && L <= 65536, B200MOE_E_BAD_SHAPE, "%s: %lld adapters, supported 1..65536", who, (long long)L);
  // Tiles of the second product, in an int; and stacks that a GPU can hold at all, 0.5 TB each, which leaves the gradients' CTAs (one for 128 columns of an
  // adapter) below 2^29.
  B200_CHECK_ARG(ceil_div(T, 128) * ceil_div(std::max(K, N), 128) < (1LL << 31) - 65536 && L * R * std::max(K, N) < (1LL << 38), B200MOE_E_BAD_SHAPE,
                 "%s: %lld rows, %lld adapters of %lld -> %lld are too many", who, (long long)T, (long long)L, (long long)K, (long long)N);
  return 0;
}

extern "C" {

size_t b200moe_lora_fwd_ws_bytes(int64_t T, int64_t R, int64_t L, int keep) {
  if (T <= 0 || R <= 0 || L <= 0) return 0;
  size_t bytes = 0;
  carve_lora(T, R, L, true, keep, nullptr, &bytes);
  return std::max(bytes, T <= kFewMost ? 2 * T * sizeof(FewRank) : 0);
}

int b200moe_lora_forward(const void* x, int64_t ldx, const void* a, const void* b, const void* index, int index_bytes, const float* scales, float scale,
                         const void* base, int64_t ldb, int64_t T, int64_t K, int64_t N, int64_t R, int64_t L, int keep, void* ws, void* out,
                         int32_t* status, b200moe_stream_t stream) {
  const int rc = check_lora("lora_forward", T, K, N, R, L);
  if (rc) return rc;
  B200_CHECK_ARG(ldx >= K && ldx % 8 == 0 && (base == nullptr || (ldb >= N && ldb % 8 == 0)), B200MOE_E_BAD_SHAPE,
                 "lora_forward: rows of x %lld apart, of base %lld (multiples of 8, at least K and N)", (long long)ldx, (long long)ldb);
  B200_CHECK_ARG(index == nullptr || index_bytes == 4 || index_bytes == 8, B200MOE_E_UNSUPPORTED, "lora_forward: an index of %d bytes", index_bytes);
  if (T == 0) return 0;
  B200_CHECK_ARG(x && a && b && ws && out && status, B200MOE_E_NULL, "lora_forward: null pointer");
  B200_CHECK_ARG(aligned16(x) && aligned16(a) && aligned16(b) && aligned16(base) && aligned16(ws) && aligned16(out) &&
                     (index == nullptr || reinterpret_cast<uintptr_t>(index) % index_bytes == 0),
                 B200MOE_E_ALIGN, "lora_forward: tensors must be 16-byte aligned, the index as its type");
  cudaStream_t st = (cudaStream_t)stream;
  const int sms = gemm_cta_budget();
  const LoraIndex ix{index, index_bytes, static_cast<int>(T), static_cast<int>(L), status};
  if (lora_few(T, R, L, keep)) {
    const int64_t groups = few_groups(ix);
    FewRank *ranks = index != nullptr && T > kFewInline ? static_cast<FewRank*>(ws) : nullptr, *leaders = ranks != nullptr ? ranks + T : nullptr;
    const int ctas = few_cluster(T, N, R, L, groups, sms);
    const int parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms / (groups * ctas), ceil_div(N, 8 * kFewWarps * ctas))));
    const FewLora p{ix, static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(a), static_cast<const __nv_bfloat16*>(b),
                    static_cast<const __nv_bfloat16*>(base), static_cast<__nv_bfloat16*>(out), ldx, ldb, ranks, leaders, static_cast<int>(K),
                    static_cast<int>(N), static_cast<int>(R), parts, scales, scale};
    OpScope scope("lora_few", ranks != nullptr ? 2 : 1);
    if (ranks != nullptr) B200_LAUNCH(lora_rank_kernel, 1, kFewMost, 0, st, ix, ranks, leaders, static_cast<int>(groups));
    auto run = [&](auto ks, auto of) -> int {
      constexpr int KS = decltype(ks)::value, CTAS = decltype(of)::value;
      static PerDevice allowed;
      B200_CUDA(allow_smem(allowed, lora_few_kernel<KS, CTAS>, few_smem(128)));
      B200_CUDA(launch_chained(lora_few_kernel<KS, CTAS>, static_cast<int>(groups * parts * CTAS), kFewThreads, few_smem(R), st, CTAS, p));
      return 0;
    };
    auto run_of = [&](auto of) -> int {
      return R <= 16 ? run(std::integral_constant<int, 1>(), of) : R <= 32 ? run(std::integral_constant<int, 2>(), of) : run(std::integral_constant<int, 0>(), of);
    };
    return ctas == 8 ? run_of(std::integral_constant<int, 8>()) : run_of(std::integral_constant<int, 4>());
  }
  size_t bytes;
  const LoraKept k = carve_lora(T, R, L, index != nullptr, keep, ws, &bytes);
  if (index != nullptr) {
    OpScope scope("lora_tiles", 1);
    B200_LAUNCH(lora_tiles_kernel, static_cast<int>(ceil_div(k.tiles.tiles, kTilesEach) + (keep ? L : 0)), kTilesThreads, 0, st, ix, k.tiles, k.lists);
  }
  {
    OpScope scope("lora_shrink", 1);
    const int rc2 = lora_shrink(x, ldx, a, false, L, ShrinkParams{k.tiles, static_cast<int>(K), static_cast<int>(R), 0, 0, 0, scales, scale, k.v, k.counter, status}, sms, st);
    if (rc2) return rc2;
  }
  OpScope scope("lora_expand", 1);
  return lora_expand(k.v, b, false, L, R, base, ldb, out, ExpandParams{k.tiles, static_cast<int>(N), 0, 0, 0, k.counter, status}, sms, st);
}

size_t b200moe_lora_bwd_ws_bytes(int64_t T, int64_t K, int64_t N, int64_t R, int64_t L) {
  if (T <= 0 || K <= 0 || N <= 0 || R <= 0 || L <= 0) return 0;
  LoraCarver c{nullptr};
  c.take<__nv_bfloat16>(2 * T * padded_rank(R));
  c.take<int>(1);
  const int sa = wgrad_splits(T, K, L, num_sms()), sb = back_wgrad_splits(T, N, L, num_sms());
  c.take<float>(std::max(sa > 1 ? sa * L * R * K : 0, sb > 1 ? sb * L * R * N : 0));
  return c.off;
}

int b200moe_lora_backward(const void* grad_out, const void* x, int64_t ldx, const void* a, const void* b, int has_index, const float* scales, float scale,
                          int64_t T, int64_t K, int64_t N, int64_t R, int64_t L, const void* fwd_ws, void* ws, void* grad_x, void* grad_a, void* grad_b,
                          int grad_f32, int32_t* status, b200moe_stream_t stream) {
  const int rc = check_lora("lora_backward", T, K, N, R, L);
  if (rc) return rc;
  B200_CHECK_ARG(T >= 1, B200MOE_E_BAD_SHAPE, "lora_backward: no rows");
  B200_CHECK_ARG(ldx >= K && ldx % 8 == 0, B200MOE_E_BAD_SHAPE, "lora_backward: rows of x %lld apart", (long long)ldx);
  B200_CHECK_ARG(grad_out && x && a && b && fwd_ws && ws && status && (grad_x || grad_a || grad_b), B200MOE_E_NULL, "lora_backward: null pointer");
  B200_CHECK_ARG(aligned16(grad_out) && aligned16(x) && aligned16(a) && aligned16(b) && aligned16(fwd_ws) && aligned16(ws) && aligned16(grad_x) &&
                     aligned16(grad_a) && aligned16(grad_b),
                 B200MOE_E_ALIGN, "lora_backward: tensors must be 16-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  const int sms = gemm_cta_budget();
  size_t bytes;
  const LoraKept k = carve_lora(T, R, L, has_index != 0, 1, const_cast<void*>(fwd_ws), &bytes);
  LoraCarver c{static_cast<char*>(ws)};
  __nv_bfloat16* u = c.take<__nv_bfloat16>(2 * T * padded_rank(R));
  int* counter = c.take<int>(1);
  float* part = c.take<float>(0);
  WgradParams w{static_cast<int>(T), 0, static_cast<int>(R), static_cast<int>(L), 1, 0, k.lists,
                nullptr, nullptr, 0, nullptr, 0, status};
#define RUN(name, launches, call)     \
  do {                                \
    OpScope scope__(name, launches);  \
    const int rc__ = (call);          \
    if (rc__) return rc__;            \
  } while (0)
  const ShrinkParams sp{k.tiles, static_cast<int>(N), static_cast<int>(R), shrink_split(T, N, sms), 0, 0, scales, scale, u, counter, status};
  const int sa = wgrad_splits(T, K, L, sms), sb = back_wgrad_splits(T, N, L, sms);
  if (grad_b && (grad_x || grad_a)) {
    w.D = static_cast<int>(N);
    RUN("lora_back", sb > 1 ? 2 : 1, lora_back(grad_out, b, k.v, L, sp, w, sb, sms, part, grad_b, grad_f32, st));
  } else if (grad_b) {
    w.D = static_cast<int>(N);
    RUN("lora_wgrad", sb > 1 ? 2 : 1, lora_wgrad(grad_out, N, k.v, sb, w, part, grad_b, grad_f32, st));
  } else {
    RUN("lora_shrink", 1, lora_shrink(grad_out, N, b, true, L, sp, sms, st));
  }
  if (grad_x)
    RUN("lora_expand", 1, lora_expand(u, a, true, L, R, nullptr, 0, grad_x, ExpandParams{k.tiles, static_cast<int>(K), 0, 0, 0, counter, status}, sms, st));
  if (grad_a) {
    w.D = static_cast<int>(K);
    w.transposed = 1;
    RUN("lora_wgrad", sa > 1 ? 2 : 1, lora_wgrad(x, ldx, u, sa, w, part, grad_a, grad_f32, st));
  }
#undef RUN
  return 0;
}

}  // extern "C"

// Products of e4m3 codes with fp32 scales per block of 128: rows of X carry a scale per row and 128 values of K, weights one per 128 x 128
// values.  tcgen05.mma.kind::f8f6f4, dense and grouped by experts, and the experts' SwiGLU with requantisation in the epilogue.
//
//   out[t, n] = sum_kb  sx[t, kb] * sw[n / 128, kb] * sum_{k in kb} X[t, k] W[n, k]
//
// The scales are arbitrary fp32 numbers, so the tensor cores cannot apply them: every k-block of 128 is a sum of its own in tensor
// memory, which the epilogue warps fetch and add to accumulators in registers, times its scales (one multiply-add a value).  Tensor memory
// is a ring, so that the MMAs of the next k-blocks run meanwhile.
#include <cuda.h>

#include <algorithm>

#include "few_tiles.cuh"
#include "fp8_block.cuh"
#include "gemm_common.cuh"

namespace b200moe {

constexpr int kBBK = 128;                 // k-block in elements = bytes: one swizzle row, four MMAs
constexpr int kBTile = 128 * kBBK;        // one operand box

struct BlockParams {
  GemmParams g;             // sched, M, N (SwiGLU: I), K, num_groups, tile_expert, poffs, counts, status
  const float* sx;          // scales of X, [k-block][row]
  long long sx_pitch;
  long long rows;           // rows of X that exist
  const float* sw;          // scales of the weights: group, column block, k-block
  long long sw_group;
  int sw_n, sw_k;           // elements between column blocks and between k-blocks
  int n_blocks;             // column blocks of one matrix (SwiGLU: of the gate half)
  uint8_t* q_out;           // SwiGLU: codes (rows, I) and their scales [column block][row]
  float* q_scale;
  long long q_pitch;
  __nv_bfloat16* out;       // few rows: (rows, N), or
  float* out_slots;         // ... (experts) the rows in fp32 at their slots of row_slot
  int split;                // few rows: CTAs of a cluster that share a tile's k-blocks
  int first_dense;          // few rows, dense: rows of X (no table)
  const __nv_bfloat16* x;   // few rows, quantised on the way: X in bf16, its rows those of the product or (row_slot) of the tokens, k slots each
  const int* row_slot;      // the slots, token and pick, of the rows
  int k;
};

__device__ __forceinline__ void umma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// e4m3 (format 0) operands, fp32 result; bit 16: B is MN-major
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n, int b_mn) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// two multiply-adds in one instruction
__device__ __forceinline__ void fma2(float2& d, uint32_t a0, uint32_t a1, float2 f) {
  asm("{\n\t.reg .b64 a, f, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 f, {%4, %5};\n\tmov.b64 d, {%0, %1};\n\t"
      "fma.rn.f32x2 d, a, f, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "+f"(d.x), "+f"(d.y)
      : "r"(a0), "r"(a1), "f"(f.x), "f"(f.y));
}
// Arrive on a barrier of another CTA of the cluster that guards tensor memory alone: nothing in memory is handed over, and
// tcgen05.fence orders the rest.  A release waits for the thread's own loads in flight (the scales ahead) twice a k-block: 8192 x 14336 x 4096
// took 984 us with it and takes 494 without.
__device__ __forceinline__ void mbar_arrive_tmem(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}
// N of the warp's 32 lanes' consecutive fp32 columns
template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 32) tmem_ld32(taddr, r);
  else if constexpr (N == 16) tmem_ld16(taddr, r);
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

// ------------------------------------------------------------------------------------------------ many rows: pairs of SMs
// A cluster of two CTAs computes 256 rows x 256 columns with cta_group::2 MMAs: each stages its own 128 rows of X and 128 rows of W (SwiGLU: one
// the gate, the other the up rows of the same 128 columns).  Two k-blocks' sums of 256 columns fill tensor memory.  An epilogue warp owns
// 32 rows and 128 columns (SwiGLU: 64 of gate and the same 64 of up), 128 accumulators a thread.
//
// Bound: the MMAs of a k-block take 512 cycles, the multiply-adds of the epilogue 386 after them, and between the two lie four signals of 130 to 220
// cycles each, so a slot of tensor memory comes round in some 1700 cycles and, with two of them, a k-block takes 870: the tensor cores are
// busy for 60 % of the time.  So what counts is how long the epilogue holds
// tensor memory.  8192 x 14336 x 4096, us: arrivals as releases 984 (mbar_arrive_tmem), scales from global memory by the epilogue's threads 488,
// by a warp that prepares them 455; 2112 TFLOP/s.  Slower: 16 epilogue warps 519; columns 32 at a time 485; plain multiply-adds in place of
// packed ones 466; the other CTA's arrivals passed on by one thread 500; tensor memory as four half k-blocks 535.  Each of the 128 + 16
// registers counts: twelve warps could have 168 each, at which every form spilled in the loop (500 to 900 us), so the four that issue
// loads and MMAs hand theirs over, 4 x 72 + 8 x 216 = 12 x 168.
constexpr int kBEpi = 8;                       // epilogue warps
constexpr int kBParts = kBEpi / 4;             // ... that share a tile's columns
constexpr int kBCols = 256 / kBParts;          // columns of one
constexpr int kBThreads = 32 * (4 + kBEpi);
template <int EPI> constexpr int kBStages = EPI == EPI_STORE ? 5 : 6;
constexpr int kBRing = 8;                      // k-blocks whose scales are in shared memory
constexpr int kBStage = 2 * kBTile;
template <int EPI> constexpr int kBEpiBytes = EPI == EPI_STORE ? kBEpi * 2048 : 0;     // SwiGLU stores its codes from registers
template <int EPI> constexpr int kBSmemBytes = kBStages<EPI> * kBStage + kBEpiBytes<EPI> + kBRing * 1024 + (2 * kBStages<EPI> + 4) * 8 + 16 + 1024;

template <int EPI, bool BMN>
__global__ void __launch_bounds__(kBThreads, 1)
block_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmD,
                  const BlockParams bp) {
  const GemmParams& p = bp.g;
  constexpr int kStages = kBStages<EPI>;
  constexpr int TM = 256, TN = EPI == EPI_SWIGLU ? 128 : 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* epi_smem = smem + kStages * kBStage;
  float* ring = reinterpret_cast<float*>(epi_smem + kBEpiBytes<EPI>);      // [k-block % kBRing][column block][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kBRing * 256);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = smem_u32(bars + kStages);
  const uint32_t bar_tfull = smem_u32(bars + 2 * kStages);
  const uint32_t bar_tempty = smem_u32(bars + 2 * kStages + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ uint32_t s_amax[2][kBParts][128];
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int cta_rank = static_cast<int>(cluster_ctarank());
  const int first_tile = static_cast<int>(cluster_id_x());
  const int tile_step = static_cast<int>(num_clusters_x());

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull + 8 * b, 2);      // the MMAs and the scales
      mbar_init(bar_tempty + 8 * b, 2 * kBEpi);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (EPI == EPI_STORE) tma_prefetch_desc(&tmD);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  grid_dep_wait();
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total = total_tiles(p, TN, TM);
  const int nkb = (p.K + kBBK - 1) / kBBK;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ------------------------------------------------------------------------------ producer (each CTA)
      if (elect_one()) {
        const uint32_t full0 = mapa_shared(bar_full, 0);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = first_tile; tile < total && ok; tile += tile_step) {
          const Tile t = get_tile(p, tile, TN, TM, kBBK);
          const int m0 = t.m0 + BM * cta_rank;
          const int n0 = EPI == EPI_SWIGLU ? t.n0 + p.I * cta_rank : t.n0 + 128 * cta_rank;
          for (int kb = 0; kb < nkb; ++kb) {
            if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, abort_flag, ST_WAIT_PRODUCER)) {
              ok = false;
              break;
            }
            if (cta_rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, 2 * kBStage);
            const uint32_t sa = smem_u32(smem + s * kBStage), full = full0 + 8 * s;
            tma_load_3d_pair(sa, &tmA, full, kb * kBBK, m0, 0);
            if (BMN) tma_load_3d_pair(sa + kBTile, &tmB, full, n0, kb * kBBK, t.g);
            else tma_load_3d_pair(sa + kBTile, &tmB, full, kb * kBBK, n0, t.g);
            if (++s == kStages) {
              s = 0;
              ph ^= 1;
            }
          }
        }
      }
      grid_dep_launch();   // the last loads are on their way
    } else if (warp == 1) {
      // ------------------------------------------------------------------------------ MMA issuer (leader)
      if (cta_rank == 0 && elect_one()) {
        constexpr uint32_t idesc = idesc_f8(256, 256, BMN);
        int s = 0;
        uint32_t ph = 0, it = 0;
        bool ok = true;
        for (int tile = first_tile; tile < total && ok; tile += tile_step) {
          for (int kb = 0; kb < nkb; ++kb, ++it) {
            const int buf = it & 1;
            if (!mbar_wait(bar_tempty + 8 * buf, ((it >> 1) & 1) ^ 1, abort_flag, ST_WAIT_MMA_TMEM) ||
                !mbar_wait(bar_full + 8 * s, ph, abort_flag, ST_WAIT_MMA_FULL)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = smem_u32(smem + s * kBStage), sb = sa + kBTile;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8_pair(tmem_base + 256 * buf, umma_desc_sw128(sa + 32 * k, 0, 1024),
                           umma_desc_sw128(sb + (BMN ? 4096 : 32) * k, 0, 1024), idesc, k != 0);
            umma_commit_pair(bar_empty + 8 * s);
            umma_commit_pair(bar_tfull + 8 * buf);
            if (++s == kStages) {
              s = 0;
              ph ^= 1;
            }
          }
        }
      }
    } else if (warp == 2) {
      // ------------------------------------------------------------------------------ scales
      // This warp multiplies the scales of 128 rows and of the tile's two column blocks, k-block by k-block, for the epilogue, whose warps have
      // neither the registers nor the time to wait for global memory.  The MMAs of k-block i are complete only after the epilogue gave back
      // the tensor memory of i - 2, having read its scales: once they are, the slot of i - 2 is free.  The arrival for k-block i has to follow
      // the phase of i - 2 of the same barrier.
      constexpr int kAhead = 4;
      uint32_t it = 0;
      bool ok = true;
      for (int tile = first_tile; tile < total; tile += tile_step) {
        const Tile t = get_tile(p, tile, TN, TM, kBBK);
        const int nb = t.n0 >> 7;
        const long long row = t.m0 + BM * cta_rank;
        const bool rows = row < bp.rows;         // else none of these 128 exists
        const float4* sx = reinterpret_cast<const float4*>(bp.sx + (rows ? row : 0)) + lane;
        const float* sw = bp.sw + t.g * bp.sw_group + static_cast<long long>(nb) * bp.sw_n;
        const float* sw2 = sw + static_cast<long long>(EPI == EPI_SWIGLU ? bp.n_blocks : nb + 1 < bp.n_blocks ? 1 : 0) * bp.sw_n;
        float4 x[kAhead];
        float w[kAhead], w2[kAhead];
        auto get = [&](int kb, int u) {
          if (kb < nkb) {
            x[u] = sx[static_cast<long long>(kb) * (bp.sx_pitch >> 2)];
            w[u] = sw[static_cast<long long>(kb) * bp.sw_k];
            w2[u] = sw2[static_cast<long long>(kb) * bp.sw_k];
          }
        };
#pragma unroll
        for (int u = 0; u < kAhead; ++u) get(u, u);
        for (int kb0 = 0; kb0 < nkb; kb0 += kAhead) {
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            if (kb0 + u >= nkb) break;
            if (it >= 2) ok = ok && mbar_wait(bar_tfull + 8 * (it & 1), ((it >> 1) & 1) ^ 1, abort_flag, ST_WAIT_EPILOGUE);
            float4* to = reinterpret_cast<float4*>(ring + (it & (kBRing - 1)) * 256) + lane;
            to[0] = make_float4(x[u].x * w[u], x[u].y * w[u], x[u].z * w[u], x[u].w * w[u]);
            to[32] = make_float4(x[u].x * w2[u], x[u].y * w2[u], x[u].z * w2[u], x[u].w * w2[u]);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_tfull + 8 * (it & 1));
            get(kb0 + u + kAhead, u);
            ++it;
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------------------ epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp & 3, part = (warp - 4) >> 2;
    constexpr int HC = kBCols / 2;     // SwiGLU: columns of gate, and of up
    const uint32_t tempty_leader = mapa_shared(bar_tempty, 0);
    uint8_t* sbuf = epi_smem + (warp - 4) * 2048;
    uint32_t it = 0;
    int flip = 0;
    bool ok = true;      // a warp that gave up goes on to the barriers of the others
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + (EPI == EPI_SWIGLU ? HC : kBCols) * part;
    for (int tile = first_tile; tile < total; tile += tile_step) {
      const Tile t = get_tile(p, tile, TN, TM, kBBK);
      const int row0 = t.m0 + BM * cta_rank + 32 * q;
      const bool live = p.sched != SCHED_GROUPED_M || row0 < p.poffs[t.g] + p.counts[t.g];   // else nothing but pad rows
      float2 acc[kBCols / 2];
#pragma unroll
      for (int i = 0; i < kBCols / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
      for (int kb = 0; kb < nkb; ++kb, ++it) {
        const int buf = it & 1;
        ok = ok && mbar_wait(bar_tfull + 8 * buf, (it >> 1) & 1, abort_flag, ST_WAIT_EPILOGUE);
        __syncwarp();
        tc_fence_after();
        const float* fs = ring + (it & (kBRing - 1)) * 256 + 32 * q + lane;
        const float f = EPI == EPI_SWIGLU ? fs[0] : fs[2 * part >= kBParts ? 128 : 0], f2 = EPI == EPI_SWIGLU ? fs[128] : f;
        if (live) {
          const uint32_t ta = taddr + 256 * buf;
          constexpr int NC = kBCols / 16;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            uint32_t r[16];
            tmem_ld16(ta + (EPI == EPI_SWIGLU && 2 * c >= NC ? 128 - HC : 0) + 16 * c, r);
            tmem_ld_wait();
            if (c == NC - 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_tmem(tempty_leader + 8 * buf);
            }
            const float s = EPI == EPI_SWIGLU && 2 * c >= NC ? f2 : f;
#pragma unroll
            for (int i = 0; i < 8; ++i) fma2(acc[8 * c + i], r[2 * i], r[2 * i + 1], make_float2(s, s));
          }
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_tmem(tempty_leader + 8 * buf);
        }
      }
      if constexpr (EPI == EPI_STORE) {
        ok = __all_sync(0xffffffffu, ok);      // the lanes meet in there
        if (live && ok) {
#pragma unroll
          for (int cc = 0; cc < kBCols / 32; ++cc) {
            const int c = t.n0 + kBCols * part + 32 * cc;
            if (c < p.N) {
              staging_free(lane);
#pragma unroll
              for (int j = 0; j < 4; ++j) {      // 32 columns of a row, 64-byte swizzle
                const float2* x = acc + 16 * cc + 4 * j;
                *reinterpret_cast<uint4*>(sbuf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                    make_uint4(pack_bf16x2(x[0].x, x[0].y), pack_bf16x2(x[1].x, x[1].y), pack_bf16x2(x[2].x, x[2].y), pack_bf16x2(x[3].x, x[3].y));
              }
              store_box(&tmD, sbuf, lane, c, row0, 0);
            }
          }
        }
      } else {
        // acc: gate, then up of the same HC columns
        uint32_t amax = 0u;
#pragma unroll
        for (int i = 0; i < HC / 2; ++i) {
          acc[i].x = silu_mul(acc[i].x, acc[HC / 2 + i].x);
          acc[i].y = silu_mul(acc[i].y, acc[HC / 2 + i].y);
          amax = max(amax, max(__float_as_uint(acc[i].x) & 0x7fffffffu, __float_as_uint(acc[i].y) & 0x7fffffffu));
        }
        // the other parts of the row's 128 columns: two buffers, since another warp may be a tile ahead
        s_amax[flip][part][32 * q + lane] = amax;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + q), "n"(32 * kBParts) : "memory");
#pragma unroll
        for (int o = 0; o < kBParts; ++o) amax = max(amax, s_amax[flip][o][32 * q + lane]);
        flip ^= 1;
        if (live && ok) {
          float scale, inv;
          block_scale_factor(amax, scale, inv);
          const long long orow = row0 + lane;
          uint4* dst = reinterpret_cast<uint4*>(bp.q_out + orow * p.I + t.n0 + HC * part);
#pragma unroll
          for (int v = 0; v < HC / 16; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 x = acc[8 * v + 2 * j], y = acc[8 * v + 2 * j + 1];
              w[j] = cvt4_e4m3(x.x * inv, x.y * inv, y.x * inv, y.y * inv);
            }
            dst[v] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (part == 0) bp.q_scale[scale_at(t.n0 >> 7, bp.q_pitch, orow)] = scale;
        }
      }
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();
  if (threadIdx.x == 0 && *abort_flag != 0 && p.status != nullptr) atomicCAS(p.status, 0, *abort_flag);
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// The weights are the M operand, 128 rows of them a tile, and up to NT rows of X the N operand, so that every weight is read once for
// the rows that want it.  A stage is 32 KB of weights: two k-blocks (store), or the gate and the up rows of one (SwiGLU).  Lanes of an
// epilogue warp are output columns, its registers NT / 2 rows of X; the rows' scales come with the operands, through shared memory.
// Bound: HBM, by the one read of the weights.  Where the tiles do not fill the SMs, the k-blocks of a tile are shared by the CTAs of a
// cluster, which send their sums to the first one (in the order of the ranks: the same bits every time).
//
// QUANT: X comes in bf16, and eight more warps write its codes and scales into the stages, the live rows alone, with the bits of the quantiser, which
// needs no launch then.  Every tile makes them again: see quant_inside.
constexpr int kQuantWarps = 8;
template <int EPI, int NT>
struct FewBlockCfg {
  static constexpr int XB = EPI == EPI_SWIGLU ? 1 : 2;                 // k-blocks of a stage
  static constexpr int X_BYTES = NT * kBBK;
  static constexpr int STAGE = 2 * kBTile + XB * X_BYTES;
  static constexpr int ACCS = EPI == EPI_SWIGLU ? NT : NT / 2;         // fp32 sums of a thread
  static constexpr int RANK_BYTES = 32 * kEpiWarps * ACCS * 4;
  static constexpr int MAX_SPLIT = ACCS <= 8 ? 8 : ACCS <= 16 ? 4 : ACCS <= 32 ? 2 : 1;
  static constexpr int RED_BYTES = (MAX_SPLIT - 1) * RANK_BYTES;
  static constexpr int SLOTS = 512 / (2 * NT) < 8 ? 512 / (2 * NT) : 8;   // tensor-memory ring, a stage each
  static constexpr int kFit = (232448 - 8192 - RED_BYTES) / STAGE;
  static constexpr int NSTAGE = kFit > 8 ? 8 : kFit;
  static constexpr int SF = NSTAGE + SLOTS;                            // ring of the rows' scales, see the producer
  static constexpr int SF_BYTES = XB * NT * 4;
  static constexpr int TMEM_COLS = SLOTS * 2 * NT;                     // 256 or 512
  static constexpr int BARS = 2 * NSTAGE + 2 * SLOTS + SF + 2;
  static constexpr int SMEM_BYTES = NSTAGE * STAGE + RED_BYTES + SF * SF_BYTES + BARS * 8 + 16 + 1024;
  static_assert(SMEM_BYTES <= 232448 - 4608, "shared memory");         // 4.5 KB are static
  static_assert(TMEM_COLS == 256 || TMEM_COLS == 512, "a power of two");
};

// as mbar_wait, for a barrier that other CTAs of the cluster arrive on: their writes before it are visible
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  const long long t0 = clock64();
  for (uint32_t it = 1;; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 0xff) == 0) {
      if (*abort_flag != 0) return false;
      if (clock64() - t0 > kWaitLimitCycles) {
        *abort_flag = code;
        return false;
      }
    }
  }
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <int EPI, int NT, bool QUANT>
__global__ void __launch_bounds__(kThreads + (QUANT ? 32 * kQuantWarps : 0), 1)
block_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const BlockParams bp) {
  using C = FewBlockCfg<EPI, NT>;
  const GemmParams& p = bp.g;
  constexpr int NSTAGE = C::NSTAGE, SLOTS = C::SLOTS, XB = C::XB, HC = NT / 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* red = reinterpret_cast<float*>(smem + NSTAGE * C::STAGE);
  float* sf = reinterpret_cast<float*>(smem + NSTAGE * C::STAGE + C::RED_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + NSTAGE * C::STAGE + C::RED_BYTES + C::SF * C::SF_BYTES);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = smem_u32(bars + NSTAGE);
  const uint32_t bar_tfull = smem_u32(bars + 2 * NSTAGE);
  const uint32_t bar_tempty = smem_u32(bars + 2 * NSTAGE + SLOTS);
  const uint32_t bar_sf = smem_u32(bars + 2 * NSTAGE + 2 * SLOTS);
  const uint32_t bar_sums = smem_u32(bars + 2 * NSTAGE + 2 * SLOTS + C::SF);       // rank 0: the others' sums are here
  const uint32_t bar_taken = bar_sums + 8;                                         // the others: rank 0 has read theirs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int pre[B200MOE_MAX_EXPERTS + 1];
  __shared__ uint32_t s_amax[2][4][NT];
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = bp.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int first_tile = static_cast<int>(blockIdx.x) / bp.split, tile_step = static_cast<int>(gridDim.x) / bp.split;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NSTAGE; ++s) {
      mbar_init(bar_full + 8 * s, QUANT ? 1 + kQuantWarps : 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < SLOTS; ++b) {
      mbar_init(bar_tfull + 8 * b, 1);
      mbar_init(bar_tempty + 8 * b, kEpiWarps);
    }
    for (int b = 0; b < C::SF; ++b) mbar_init(bar_sf + 8 * b, QUANT ? kQuantWarps : 1);
    mbar_init(bar_sums, bp.split > 1 ? (bp.split - 1) * kEpiWarps : 1);
    mbar_init(bar_taken, kEpiWarps);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmW);
    if (!QUANT) tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  grid_dep_wait();
  if (warp == 2) {
    if (p.counts != nullptr) few_prefix<NT>(p.counts, p.num_groups, lane, pre);
    else if (lane == 0) {
      pre[0] = 0;
      pre[1] = (bp.first_dense + NT - 1) / NT;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (bp.split > 1) {
    __syncwarp();
    cluster_sync_all();
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int mt = (p.N + 127) >> 7;
  const int total = pre[p.num_groups] * mt;
  const int nkb = (p.K + kBBK - 1) / kBBK;
  const int kb_lo = nkb * rank / bp.split, kb_hi = nkb * (rank + 1) / bp.split;
  const int steps = (kb_hi - kb_lo + XB - 1) / XB;       // stages of a tile
  auto tile_of = [&](int tile) {
    if (p.counts != nullptr) return few_tile<NT, 128>(p.counts, p.poffs, p.num_groups, p.N, pre, tile);
    FewTile t;
    const int c = tile / mt;
    t.e = 0;
    t.m0 = (tile - c * mt) * 128;
    t.row0 = c * NT;
    t.live = min(NT, bp.first_dense - c * NT);
    return t;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (elect_one()) {
      int s = 0, f = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = first_tile; tile < total && ok; tile += tile_step) {
        const FewTile t = tile_of(tile);
        for (int kb = kb_lo; kb < kb_hi; kb += XB) {
          const int n = min(XB, kb_hi - kb);
          if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, abort_flag, ST_WAIT_PRODUCER)) {
            ok = false;
            break;
          }
          const uint32_t full = bar_full + 8 * s, st = smem_u32(smem + s * C::STAGE), xs = st + 2 * kBTile;
          mbar_arrive_expect_tx(full, (EPI == EPI_SWIGLU ? 2 : n) * kBTile + (QUANT ? 0 : n * C::X_BYTES));
          if constexpr (EPI == EPI_SWIGLU) {
            tma_load_3d(st, &tmW, full, kb * kBBK, t.m0, t.e);
            tma_load_3d(st + kBTile, &tmW, full, kb * kBBK, p.I + t.m0, t.e);
            if (!QUANT) tma_load_3d(xs, &tmX, full, kb * kBBK, t.row0, 0);
          } else {
            for (int i = 0; i < n; ++i) {
              tma_load_3d(st + i * kBTile, &tmW, full, (kb + i) * kBBK, t.m0, t.e);
              if (!QUANT) tma_load_3d(xs + i * C::X_BYTES, &tmX, full, (kb + i) * kBBK, t.row0, 0);
            }
          }
          // The MMAs of the stage NSTAGE before are complete (bar_empty), so the epilogue has given back the tensor memory of the one SLOTS
          // before that: it has read those scales, and this slot of a ring of NSTAGE + SLOTS is free.
          if constexpr (!QUANT) {
            const uint32_t bf = bar_sf + 8 * f;
            mbar_arrive_expect_tx(bf, n * NT * 4);
            for (int i = 0; i < n; ++i)
              bulk_load_1d(smem_u32(sf + f * (XB * NT) + i * NT), bp.sx + scale_at(kb + i, bp.sx_pitch, t.row0), NT * 4, bf);
            if (++f == C::SF) f = 0;
          }
          if (++s == NSTAGE) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
    grid_dep_launch();   // the last loads are on their way
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_f8(128, NT, 0);
      int s = 0, slot = 0;
      uint32_t ph = 0, sph = 1;
      bool ok = true;
      for (int tile = first_tile; tile < total && ok; tile += tile_step) {
        for (int kb = kb_lo; kb < kb_hi; kb += XB) {
          const int n = EPI == EPI_SWIGLU ? 2 : min(XB, kb_hi - kb);
          if (!mbar_wait(bar_tempty + 8 * slot, sph, abort_flag, ST_WAIT_MMA_TMEM) ||
              !mbar_wait(bar_full + 8 * s, ph, abort_flag, ST_WAIT_MMA_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t st = smem_u32(smem + s * C::STAGE);
          for (int i = 0; i < n; ++i) {
            const uint32_t sw = st + i * kBTile, sx = st + 2 * kBTile + (EPI == EPI_SWIGLU ? 0 : i * C::X_BYTES);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8(tmem_base + (2 * slot + i) * NT, umma_desc_sw128(sw + 32 * k, 0, 1024), umma_desc_sw128(sx + 32 * k, 0, 1024), idesc,
                      k != 0);
          }
          umma_commit(bar_empty + 8 * s);
          umma_commit(bar_tfull + 8 * slot);
          if (++slot == SLOTS) {
            slot = 0;
            sph ^= 1;
          }
          if (++s == NSTAGE) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (QUANT && warp >= 2 + kEpiWarps) {
    // ------------------------------------------------------------------ codes and scales of X, kQAhead stages' values on their way
    // kQLanes lanes a row and k-block.  A slot of the scales is free when the stage's is, as for the producer.  Rows that are not live are left as
    // they are: what they make of a stage goes nowhere.
    if constexpr (QUANT) {
      constexpr int kQLanes = 32 * kQuantWarps / (XB * NT), kQVec = 16 / kQLanes, kQAhead = 8 / kQVec;
      static_assert(kQLanes * kQVec == 16 && kQVec <= 2, "a block of 128 is 16 vectors");
      const int at = threadIdx.x - kThreads, ql = at % kQLanes, box = at / kQLanes / NT, r = at / kQLanes % NT;
      int s = 0, f = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = first_tile; tile < total && ok; tile += tile_step) {
        const FewTile t = tile_of(tile);
        const bool live = r < t.live;
        long long row = t.row0 + r;
        if (live && bp.row_slot != nullptr) row = bp.row_slot[row] / bp.k;
        const __nv_bfloat16* x = bp.x + row * p.K;
        uint4 v[kQAhead][2];
        auto get = [&](int kb, uint4 (&to)[2]) {
#pragma unroll
          for (int h = 0; h < kQVec; ++h) {
            const int c = kb * kBBK + 64 * h + 8 * ql;
            to[h] = make_uint4(0u, 0u, 0u, 0u);
            if (live && kb < kb_hi && c < p.K) to[h] = *reinterpret_cast<const uint4*>(x + c);      // K is a multiple of 16
          }
        };
#pragma unroll
        for (int u = 0; u < kQAhead; ++u) get(kb_lo + u * XB + box, v[u]);
        for (int kb0 = kb_lo; kb0 < kb_hi && ok; kb0 += kQAhead * XB) {
#pragma unroll
          for (int u = 0; u < kQAhead; ++u) {
            const int kb = kb0 + u * XB;
            if (kb >= kb_hi || !ok) break;
            uint32_t m = absmax8(0u, v[u][0]);
            if (kQVec == 2) m = absmax8(m, v[u][1]);
#pragma unroll
            for (int off = kQLanes / 2; off > 0; off >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, off));
            m = max(m & 0xffffu, m >> 16) << 16;
            float scale, factor;
            block_scale_factor(m, scale, factor);
            uint2 o[kQVec];
#pragma unroll
            for (int h = 0; h < kQVec; ++h) o[h] = block_codes8(v[u][h], factor, m < 0x7f800000u);
            // all lanes give up or none does: those that went on would wait in the next shuffle for those that left
            ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph ^ 1, abort_flag, ST_WAIT_PRODUCER));
            if (live && ok && kb + box < kb_hi) {
              uint8_t* to = smem + s * C::STAGE + 2 * kBTile + box * C::X_BYTES + r * kBBK + 8 * (ql & 1);      // 128-byte swizzle
#pragma unroll
              for (int h = 0; h < kQVec; ++h) *reinterpret_cast<uint2*>(to + ((((ql >> 1) + 4 * h) ^ (r & 7)) << 4)) = o[h];
              if (ql == 0) sf[f * (XB * NT) + box * NT + r] = scale;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(bar_full + 8 * s);
              mbar_arrive(bar_sf + 8 * f);
            }
            get(kb + kQAhead * XB + box, v[u]);
            if (++f == C::SF) f = 0;
            if (++s == NSTAGE) {
              s = 0;
              ph ^= 1;
            }
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue: lane = output column, register = row of X
    const int q = warp & 3, half = (warp - 2) >> 2, tid = threadIdx.x - 64;
    constexpr int CH = HC < 32 ? HC : 32;      // columns fetched at a time
    int slot = 0, f = 0, flip = 0;
    uint32_t sph = 0, fph = 0, tph = 0;
    bool ok = true;                            // a warp that gave up goes on to the barriers of the others
    for (int tile = first_tile; tile < total; tile += tile_step) {
      const FewTile t = tile_of(tile);
      const float* sw = bp.sw + t.e * bp.sw_group + static_cast<long long>(t.m0 >> 7) * bp.sw_n;
      const float* sw2 = sw + static_cast<long long>(bp.n_blocks) * bp.sw_n;       // SwiGLU: up
      const int col = t.m0 + 32 * q + lane;
      int slot_of = 0;      // lane i: of this warp's row i
      if (EPI == EPI_STORE && bp.out_slots != nullptr && lane < min(HC, t.live - half * HC)) slot_of = bp.row_slot[t.row0 + half * HC + lane];
      float acc[EPI == EPI_SWIGLU ? 2 : 1][HC];
#pragma unroll
      for (int i = 0; i < HC; ++i) {
        acc[0][i] = 0.0f;
        if constexpr (EPI == EPI_SWIGLU) acc[1][i] = 0.0f;
      }
      // the weights' scales of the next stage: of its two k-blocks, or of gate and up
      float w0 = 0.0f, w1 = 0.0f;
      auto weights = [&](int kb) {
        if (kb >= kb_hi) return;
        w0 = sw[static_cast<long long>(kb) * bp.sw_k];
        if constexpr (EPI == EPI_SWIGLU) w1 = sw2[static_cast<long long>(kb) * bp.sw_k];
        else if (kb + 1 < kb_hi) w1 = sw[static_cast<long long>(kb + 1) * bp.sw_k];
      };
      weights(kb_lo);
      for (int i = 0, kb = kb_lo; i < steps; ++i, kb += XB) {
        ok = ok && mbar_wait(bar_sf + 8 * f, fph, abort_flag, ST_WAIT_EPILOGUE) &&
             mbar_wait(bar_tfull + 8 * slot, sph, abort_flag, ST_WAIT_EPILOGUE);
        __syncwarp();
        tc_fence_after();
        const float c0 = w0, c1 = w1;
        weights(kb + XB);
        const uint32_t ta = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + 2 * slot * NT + half * HC;
        const int boxes = EPI == EPI_SWIGLU ? 2 : min(XB, kb_hi - kb);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (b < boxes) {
            const float4* x4 = reinterpret_cast<const float4*>(sf + f * (XB * NT) + (EPI == EPI_SWIGLU ? 0 : b * NT) + half * HC);
            const float c = b ? c1 : c0;
            float(&a)[HC] = acc[EPI == EPI_SWIGLU ? b : 0];
#pragma unroll
            for (int j0 = 0; j0 < HC; j0 += CH) {
              uint32_t r[CH];
              tmem_ld_cols<CH>(ta + b * NT + j0, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < CH; j += 4) {
                const float4 x = x4[(j0 + j) >> 2];
                a[j0 + j] += __uint_as_float(r[j]) * (x.x * c);
                a[j0 + j + 1] += __uint_as_float(r[j + 1]) * (x.y * c);
                a[j0 + j + 2] += __uint_as_float(r[j + 2]) * (x.z * c);
                a[j0 + j + 3] += __uint_as_float(r[j + 3]) * (x.w * c);
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_tempty + 8 * slot);
        if (++slot == SLOTS) {
          slot = 0;
          sph ^= 1;
        }
        if (++f == C::SF) {
          f = 0;
          fph ^= 1;
        }
      }
      if constexpr (C::MAX_SPLIT > 1) {
        if (bp.split > 1) {
          if (rank != 0) {
            // wait until rank 0 has taken the last tile's, send, say so
            ok = ok && mbar_wait_cluster(bar_taken, tph ^ 1, abort_flag, ST_WAIT_EPILOGUE);
            const uint32_t to = mapa_shared(smem_u32(red), 0) + (rank - 1) * C::RANK_BYTES + 4 * tid;
            if (ok) {
#pragma unroll
              for (int i = 0; i < C::ACCS; ++i) st_cluster(to + i * (32 * kEpiWarps * 4), acc[i / HC][i % HC]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_shared(bar_sums, 0));
            tph ^= 1;
            continue;
          }
          ok = ok && mbar_wait_cluster(bar_sums, tph, abort_flag, ST_WAIT_EPILOGUE);
          tph ^= 1;
          __syncwarp();
          if (ok) {
            for (int o = 0; o < bp.split - 1; ++o)
#pragma unroll
              for (int i = 0; i < C::ACCS; ++i) acc[i / HC][i % HC] += red[o * (C::RANK_BYTES / 4) + i * (32 * kEpiWarps) + tid];
          }
          __syncwarp();
          if (lane == 0)
            for (int o = 1; o < bp.split; ++o) mbar_arrive_cluster(mapa_shared(bar_taken, o));
        }
      }
      const int mine = min(HC, t.live - half * HC);       // rows of this warp
      const long long row = t.row0 + half * HC;
      if constexpr (EPI == EPI_STORE) {
        if (bp.out_slots != nullptr) {
#pragma unroll
          for (int i = 0; i < HC; ++i) {
            const long long to = __shfl_sync(0xffffffffu, slot_of, i);
            if (i < mine && ok) bp.out_slots[to * p.N + col] = acc[0][i];      // N is a multiple of 128
          }
        } else if (ok && col < p.N) {
#pragma unroll
          for (int i = 0; i < HC; ++i)
            if (i < mine) bp.out[(row + i) * p.N + col] = __float2bfloat16_rn(acc[0][i]);
        }
      } else {
        // a row's largest value over the tile's 128 columns: 32 of this warp, the other three warps' through shared memory (two buffers,
        // since a warp may be a tile ahead)
#pragma unroll
        for (int i = 0; i < HC; ++i) {
          acc[0][i] = silu_mul(acc[0][i], acc[1][i]);
          const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(acc[0][i]) & 0x7fffffffu);
          if (lane == 0) s_amax[flip][q][half * HC + i] = m;
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
        if (ok) {
#pragma unroll
          for (int i = 0; i < HC; ++i) {
            const int j = half * HC + i;
            if (i < mine) {
              const uint32_t m = max(max(s_amax[flip][0][j], s_amax[flip][1][j]), max(s_amax[flip][2][j], s_amax[flip][3][j]));
              float scale, inv;
              block_scale_factor(m, scale, inv);
              bp.q_out[(row + i) * p.I + col] = static_cast<uint8_t>(__nv_cvt_float_to_fp8(acc[0][i] * inv, __NV_SATFINITE, __NV_E4M3));
              if (q == 0 && lane == 0) bp.q_scale[scale_at(t.m0 >> 7, bp.q_pitch, row + i)] = scale;
            }
          }
        }
        flip ^= 1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (bp.split > 1) {
    __syncwarp();
    cluster_sync_all();      // nobody's shared memory goes before the others have sent to it
  }
  if (threadIdx.x == 0 && *abort_flag != 0 && p.status != nullptr) atomicCAS(p.status, 0, *abort_flag);
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------------ host side
template <int EPI, bool BMN>
static int launch_pair(const void* X, int64_t x_rows, int64_t ldx, const void* W, int64_t w_inner, int64_t w_rows, int64_t groups,
                       const BlockParams& bp, int64_t max_tiles, cudaStream_t stream) {
  static PerDevice smem_allowed;
  B200_CUDA(allow_smem(smem_allowed, block_pair_kernel<EPI, BMN>, kBSmemBytes<EPI>));
  CUtensorMap tmA, tmB, tmD;
  int rc = make_map(&tmA, X, bp.g.K, x_rows, 1, ldx, x_rows * ldx, kBBK, 128, 1);
  if (rc == 0) rc = make_map(&tmB, W, w_inner, w_rows, groups, w_inner, w_rows * w_inner, 128, 128, 1);
  tmD = tmA;
  if (rc == 0 && EPI == EPI_STORE) rc = make_map(&tmD, bp.g.D, bp.g.N, x_rows, 1, bp.g.ldd, x_rows * bp.g.ldd, 32, 32, 2, 64);
  if (rc) return rc;
  const int pairs = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(gemm_cta_budget() / 2, max_tiles)));
  B200_CUDA(launch_chained(block_pair_kernel<EPI, BMN>, pairs * 2, kBThreads, kBSmemBytes<EPI>, stream, 2, tmA, tmB, tmD, bp));
  return 0;
}

// CTAs that share a tile's k-blocks: as many as the idle SMs allow, each with four k-blocks at least
static int few_split(int64_t tiles, int nkb, int most) {
  int s = 1;
  while (2 * s <= most && tiles * 2 * s <= gemm_cta_budget() && nkb >= 8 * s) s *= 2;
  return s;
}

template <int EPI, int NT, bool QUANT = false>
static int launch_few(const void* X, int64_t x_rows, int64_t ldx, const void* W, int64_t w_rows, BlockParams bp, int64_t tiles,
                      int64_t max_tiles, cudaStream_t stream) {
  using C = FewBlockCfg<EPI, NT>;
  static PerDevice smem_allowed;
  B200_CUDA(allow_smem(smem_allowed, block_few_kernel<EPI, NT, QUANT>, C::SMEM_BYTES));
  CUtensorMap tmW, tmX;
  int rc = make_map(&tmW, W, bp.g.K, w_rows, bp.g.num_groups, bp.g.K, w_rows * bp.g.K, kBBK, 128, 1);
  tmX = tmW;
  if (rc == 0 && !QUANT) rc = make_map(&tmX, X, bp.g.K, x_rows, 1, ldx, x_rows * ldx, kBBK, NT, 1);
  if (rc) return rc;
  bp.split = few_split(tiles, static_cast<int>(ceil_div(bp.g.K, kBBK)), C::MAX_SPLIT);
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(gemm_cta_budget() / bp.split, max_tiles)) * bp.split;
  B200_CUDA(launch_chained(block_few_kernel<EPI, NT, QUANT>, static_cast<int>(grid), kThreads + (QUANT ? 32 * kQuantWarps : 0), C::SMEM_BYTES,
                           stream, bp.split, tmW, tmX, bp));
  return 0;
}
template <int EPI>
static int launch_few_nt(int nt, const void* X, int64_t x_rows, int64_t ldx, const void* W, int64_t w_rows, const BlockParams& bp,
                         int64_t tiles, int64_t max_tiles, cudaStream_t st) {
  if (bp.x != nullptr) return launch_few<EPI, 16, true>(X, x_rows, ldx, W, w_rows, bp, tiles, max_tiles, st);
  if (nt <= 16) return launch_few<EPI, 16>(X, x_rows, ldx, W, w_rows, bp, tiles, max_tiles, st);
  if (nt <= 32) return launch_few<EPI, 32>(X, x_rows, ldx, W, w_rows, bp, tiles, max_tiles, st);
  return launch_few<EPI, 64>(X, x_rows, ldx, W, w_rows, bp, tiles, max_tiles, st);
}

// Rows of a chunk of the few-rows kernel for a dense product, 0 for row tiles: the fewest whose tiles are one wave of CTAs, since more CTAs
// that read the weights once more out of L2 beat fewer; or all rows in one chunk.  Weights of 32 MB and more want fewer reads.  us with
// chunks of 16, 32, 64 / row tiles, L2 flushed.  4096 x 4096, 64 rows 17.4, 19.5, 21.5 / 25.6; 128 rows 23.6, 19.5, 21.5 / 27.6; 256 rows 37.9,
// 27.6, 23.6 / 27.6; 384 rows 50.2, 35.8, 35.8 / 29.7.  1408 x 2048, 192 rows 13.3, 15.4, 17.4 / 19.5; 768 rows 25.6, 19.5, 17.4 / 21.5;
// 1024 rows 29.7, 25.6, 25.6 / 21.5.  4096 x 14336, 16 rows 25.6, 27.6, 33.8 / 58.4; 64 rows 37.9, 31.8, 35.8 / 58.4; 256 rows 101, 66.6, 50.2 /
// 62.5; 384 rows 144, 93.2, 85.0 / 66.4.  (Chunks of 128 rows, whose accumulators spill, were never the best.)
static int few_dense(int64_t M, int64_t N, int64_t K) {
  const int64_t columns = ceil_div(N, 128);
  const int least = N * K < (32LL << 20) || M <= 16 ? 16 : M <= 64 ? 32 : 64;
  for (int nt = least; nt <= 64; nt *= 2)
    if (M <= nt || columns * ceil_div(M, nt) <= gemm_cta_budget()) return nt;
  return 0;
}

// The same for experts, by their mean rows, as the host knows them.  us of a whole block with chunks of 16, 32, 64 / row tiles, L2 flushed, even
// and rank^-1.1 routing.  64 experts of 2048 x 1408: 12 rows each 133, 135, 150 / 170, 119, 115, 125 / 133; 24 rows 152, 137, 156 / 170 and 162,
// 145, 147 / 156; 32 rows 172, 150, 160 / 174 and 193, 164, 162 / 164; 48 rows 223, 182, 164 / 176 and 240, 199, 201 / 172.  8 of 4096 x 14336:
// 8 rows 242, 248, 272 / 340 and 236, 227, 256 / 309; 24 rows 356, 254, 287 / 342 and 352, 303, 279 / 344; 32 rows 424, 307, 291 / 344 and 383,
// 303, 283 / 342; 48 rows 537, 363, 293 / 348 and 514, 371, 361 / 346; 64 rows 635, 459, 381 / 346.  128 of 512 x 512: 8 rows 59, 64, 80 / 80; 32 rows
// 78, 70, 84 / 80 and 72, 68, 74 / 66; 48 rows 90, 82, 84 / 80.
static int few_experts(int64_t mean) { return mean <= 12 ? 16 : mean <= 28 ? 32 : mean <= 40 ? 64 : 0; }

struct BlockCarver {
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

// Whether the few-rows kernel quantises X itself: where its rows are few and its weights no long read, the launch saved is worth more than
// what the tiles do over again.  us with the quantiser / inside, L2 flushed.  A block of 64 experts of 2048 x 1408: 1 token 36.9 / 34.8, 4 rows an expert 125 /
// 123, 12 rows under rank^-1.1 routing 119 / 125; of 128 of 512 x 512, 4 rows 55.3 / 53.2; of 8 of 4096 x 14336, 1 row 194.6 / 196.6, 4 rows 239.6 / 241.7.
// Dense (one chunk is all rows): 4 x 4096 x 4096 16.4 / 14.3 and 2.4 less on the host, 16 x 4096 x 14336 24.6 / 22.5; 64 x 4096 x 4096 in four
// chunks 16.4 / 18.5.
static bool quant_inside(int64_t mean, int64_t weights) { return mean <= 4 && weights < (32LL << 20); }

// out (M, N) = x (M, K) * w (N, K)^T, or (b_mn) out (M, K') = x (M, N') * w (N', K'): N and K of the params are of the product.  x: bf16 rows that
// are quantised here, or (x_scale) their codes
static int block_dense(const void* x, const float* x_scale, int64_t x_pitch, const void* w, const float* sw, int64_t M, int64_t N, int64_t K, int b_mn, void* ws, void* out, int32_t* status,
                       cudaStream_t st) {
  BlockParams bp{};
  bp.g.sched = SCHED_DENSE; bp.g.M = (int)M; bp.g.N = (int)N; bp.g.K = (int)K; bp.g.num_groups = 1;
  bp.g.D = out; bp.g.ldd = N; bp.g.status = status;
  bp.rows = M; bp.sw = sw;
  bp.n_blocks = (int)ceil_div(N, 128);
  bp.sw_n = b_mn ? 1 : (int)ceil_div(K, 128);
  bp.sw_k = b_mn ? (int)ceil_div(N, 128) : 1;
  const int nt = b_mn ? 0 : few_dense(M, N, K);
  const int64_t ldq = code_pitch(K);
  BlockCarver c{static_cast<char*>(ws)};
  const void* q = x;
  if (x_scale != nullptr) {
    bp.sx = x_scale;
    bp.sx_pitch = x_pitch;
  } else if (nt == 16 && M <= 16) {
    bp.x = reinterpret_cast<const __nv_bfloat16*>(x);
  } else {
    uint8_t* codes = c.take<uint8_t>(M * ldq);
    float* sx = c.take<float>(scale_pitch(M) * ceil_div(K, 128));
    q = codes;
    bp.sx = sx;
    bp.sx_pitch = scale_pitch(M);
    const int rc = fp8_block_quant(x, M, K, M, nullptr, 1, codes, ldq, sx, bp.sx_pitch, st);
    if (rc) return rc;
  }
  OpScope scope("fp8_block_linear", 1);
  if (nt > 0) {
    bp.out = reinterpret_cast<__nv_bfloat16*>(out);
    bp.first_dense = (int)M;
    const int64_t tiles = ceil_div(N, 128) * ceil_div(M, nt);
    return launch_few_nt<EPI_STORE>(nt, q, M, ldq, w, N, bp, tiles, tiles, st);
  }
  const int64_t tiles = ceil_div(M, 256) * ceil_div(N, 256);
  return b_mn ? launch_pair<EPI_STORE, true>(q, M, ldq, w, N, K, 1, bp, tiles, st)
              : launch_pair<EPI_STORE, false>(q, M, ldq, w, K, N, 1, bp, tiles, st);
}

struct BlockExperts {
  int32_t *counts, *offs, *poffs, *slot_row, *row_slot, *tile_expert;
  void* scratch;
  size_t scratch_bytes;
  uint8_t *xq, *iq;
  float *xs, *is;
  void* eo;                 // the experts' results: bf16 rows as the products have them, or (few rows) fp32 at their slots
};
static BlockExperts carve_block(int64_t T, int64_t H, int64_t I, int E, int k, void* ws, size_t* bytes) {
  BlockCarver c{static_cast<char*>(ws)};
  BlockExperts f{};
  const int64_t M = T * k, cap = b200moe_padded_rows_cap(M, E);
  f.counts = c.take<int32_t>(E);
  f.offs = c.take<int32_t>(E + 1);
  f.poffs = c.take<int32_t>(E + 1);
  f.slot_row = c.take<int32_t>(M);
  f.row_slot = c.take<int32_t>(cap);
  f.tile_expert = c.take<int32_t>(cap / B200MOE_TILE_M);
  f.scratch_bytes = b200moe_permute_ws_bytes(M, E);
  f.scratch = c.take<char>(f.scratch_bytes);
  f.xq = c.take<uint8_t>(cap * H);
  f.xs = c.take<float>(cap * (H / 128));
  f.iq = c.take<uint8_t>(cap * I);
  f.is = c.take<float>(cap * (I / 128));
  if (few_experts(ceil_div(M, E)) > 0) f.eo = c.take<float>(M * H);
  else f.eo = c.take<uint16_t>(cap * H);
  *bytes = c.off;
  return f;
}

}  // namespace b200moe

using namespace b200moe;

static int check_linear(const char* who, int64_t M, int64_t N, int64_t K) {
  B200_CHECK_ARG(M >= 0 && M < (1LL << 31) - 256, B200MOE_E_BAD_SHAPE, "%s: %lld rows", who, (long long)M);
  B200_CHECK_ARG(N > 0 && N % 8 == 0 && N < (1LL << 31) - 256, B200MOE_E_BAD_SHAPE, "%s: N = %lld must be a positive multiple of 8", who, (long long)N);
  B200_CHECK_ARG(K > 0 && K % 16 == 0 && K < (1LL << 31) - 256, B200MOE_E_BAD_SHAPE, "%s: K = %lld must be a positive multiple of 16", who, (long long)K);
  return 0;
}

extern "C" {

size_t b200moe_fp8_block_linear_ws_bytes(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0) return 0;
  BlockCarver c{nullptr};
  c.take<uint8_t>(M * code_pitch(K));
  c.take<float>(scale_pitch(M) * ceil_div(K, 128));
  return c.off;
}

int b200moe_fp8_block_linear(const void* x, const void* w, const float* w_scale, int64_t M, int64_t N, int64_t K, int transposed, void* ws,
                             void* out, int32_t* status, b200moe_stream_t stream) {
  int rc = check_linear("fp8_block_linear", M, N, K);
  if (rc) return rc;
  if (M == 0) return 0;
  B200_CHECK_ARG(x && w && w_scale && ws && out, B200MOE_E_NULL, "fp8_block_linear: null pointer");
  B200_CHECK_ARG(aligned16(x) && aligned16(w) && aligned16(ws) && aligned16(out), B200MOE_E_ALIGN,
                 "fp8_block_linear: tensors must be 16-byte aligned");
  return block_dense(x, nullptr, 0, w, w_scale, M, transposed ? K : N, transposed ? N : K, transposed, ws, out, status, (cudaStream_t)stream);
}

int b200moe_fp8_block_linear_rows(const void* q, const float* q_scale, int64_t scale_pitch_, const void* w, const float* w_scale, int64_t M, int64_t N,
                                  int64_t K, void* out, int32_t* status, b200moe_stream_t stream) {
  int rc = check_linear("fp8_block_linear_rows", M, N, K);
  if (rc) return rc;
  if (M == 0) return 0;
  B200_CHECK_ARG(q && q_scale && w && w_scale && out, B200MOE_E_NULL, "fp8_block_linear_rows: null pointer");
  B200_CHECK_ARG(scale_pitch_ >= scale_pitch(M) && scale_pitch_ % 4 == 0, B200MOE_E_BAD_SHAPE,
                 "fp8_block_linear_rows: scales %lld apart, %lld rows rounded up to whole 128 are wanted", (long long)scale_pitch_, (long long)M);
  B200_CHECK_ARG(aligned16(q) && aligned16(q_scale) && aligned16(w) && aligned16(out), B200MOE_E_ALIGN,
                 "fp8_block_linear_rows: tensors must be 16-byte aligned");
  return block_dense(q, q_scale, scale_pitch_, w, w_scale, M, N, K, 0, nullptr, out, status, (cudaStream_t)stream);
}

size_t b200moe_moe_fp8_block_ws_bytes(int64_t T, int64_t H, int64_t I, int E, int k) {
  if (T <= 0 || H <= 0 || I <= 0 || E < 1 || k < 1) return 0;
  size_t bytes = 0;
  carve_block(T, H, I, E, k, nullptr, &bytes);
  return bytes;
}

int b200moe_moe_fp8_block_forward(const void* x, const int64_t* idx, const float* w, const void* gate_up, const float* gate_up_scale,
                                  const void* down, const float* down_scale, int64_t T, int64_t H, int64_t I, int E, int k, void* ws,
                                  void* out, int32_t* status, b200moe_stream_t stream) {
  B200_CHECK_ARG(T >= 0 && T < (1LL << 31) && H > 0 && I > 0 && H % 128 == 0 && I % 128 == 0, B200MOE_E_BAD_SHAPE,
                 "moe_fp8_block: T = %lld, H = %lld, I = %lld (positive multiples of 128)", (long long)T, (long long)H, (long long)I);
  B200_CHECK_ARG(E >= 1 && E <= B200MOE_MAX_EXPERTS, B200MOE_E_UNSUPPORTED, "moe_fp8_block: E = %d, supported 1..%d", E, B200MOE_MAX_EXPERTS);
  B200_CHECK_ARG(k >= 1 && k <= B200MOE_MAX_TOPK, B200MOE_E_BAD_SHAPE, "moe_fp8_block: k = %d", k);
  B200_CHECK_ARG(2 * I < (1LL << 31) && H < (1LL << 31) && b200moe_padded_rows_cap(T * k, E) < (1LL << 31) - 256, B200MOE_E_BAD_SHAPE,
                 "moe_fp8_block: %lld routed rows do not fit int32 tables", (long long)(T * k));
  if (T == 0) return 0;
  B200_CHECK_ARG(x && idx && w && gate_up && gate_up_scale && down && down_scale && ws && out && status, B200MOE_E_NULL,
                 "moe_fp8_block: null pointer");
  B200_CHECK_ARG(aligned16(x) && aligned16(gate_up) && aligned16(down) && aligned16(ws) && aligned16(out), B200MOE_E_ALIGN,
                 "moe_fp8_block: tensors must be 16-byte aligned");
  size_t bytes;
  const BlockExperts f = carve_block(T, H, I, E, k, ws, &bytes);
  const int64_t M = T * k, cap = b200moe_padded_rows_cap(M, E);
  cudaStream_t st = (cudaStream_t)stream;
#define RUN(name, launches, call)     \
  do {                                \
    OpScope scope__(name, launches);  \
    const int rc__ = (call);          \
    if (rc__) return rc__;            \
  } while (0)
  RUN("permute_build", M > 1024 ? 2 : 1,
      permute_build(idx, T, k, E, f.counts, f.offs, f.poffs, f.slot_row, f.row_slot, f.tile_expert, nullptr, nullptr, f.scratch, f.scratch_bytes,
                    nullptr, nullptr, status, stream));
  const int nt = few_experts(ceil_div(M, E));
  const bool inside = quant_inside(ceil_div(M, E), H * I);
  if (!inside) {
    const int rc = fp8_block_quant(x, T, H, cap, f.slot_row, k, f.xq, H, f.xs, cap, stream);
    if (rc) return rc;
  }
  // gate and up
  BlockParams up{};
  up.g.sched = SCHED_GROUPED_M; up.g.N = up.g.I = (int)I; up.g.K = (int)H; up.g.num_groups = E;
  up.g.tile_expert = f.tile_expert; up.g.poffs = f.poffs; up.g.counts = f.counts; up.g.status = status;
  up.sx = f.xs; up.sx_pitch = cap; up.rows = cap; up.sw = gate_up_scale;
  up.n_blocks = (int)(I / 128); up.sw_n = (int)(H / 128); up.sw_k = 1; up.sw_group = 2 * (I / 128) * (H / 128);
  if (inside) { up.x = reinterpret_cast<const __nv_bfloat16*>(x); up.row_slot = f.row_slot; up.k = k; }
  up.q_out = f.iq; up.q_scale = f.is; up.q_pitch = cap;
  // down
  BlockParams dn{};
  dn.g.sched = SCHED_GROUPED_M; dn.g.N = (int)H; dn.g.K = (int)I; dn.g.num_groups = E;
  dn.g.tile_expert = f.tile_expert; dn.g.poffs = f.poffs; dn.g.counts = f.counts; dn.g.status = status;
  if (nt > 0) { dn.out_slots = static_cast<float*>(f.eo); dn.row_slot = f.row_slot; }
  else { dn.g.D = f.eo; dn.g.ldd = H; }
  dn.sx = f.is; dn.sx_pitch = cap; dn.rows = cap; dn.sw = down_scale;
  dn.n_blocks = (int)(H / 128); dn.sw_n = (int)(I / 128); dn.sw_k = 1; dn.sw_group = (H / 128) * (I / 128);
  const int64_t hit = std::min<int64_t>(E, M);           // experts that can have a row
  if (nt > 0) {
    const int64_t chunks = E + M / nt;                   // at most
    RUN("fp8_block_gate_up", 1, launch_few_nt<EPI_SWIGLU>(nt, f.xq, cap, H, gate_up, 2 * I, up, hit * (I / 128), chunks * (I / 128), st));
    RUN("fp8_block_down", 1, launch_few_nt<EPI_STORE>(nt, f.iq, cap, I, down, H, dn, hit * (H / 128), chunks * (H / 128), st));
  } else {
    const int64_t tiles = cap / 256;
    RUN("fp8_block_gate_up", 1, (launch_pair<EPI_SWIGLU, false>(f.xq, cap, H, gate_up, H, 2 * I, E, up, tiles * (I / 128), st)));
    RUN("fp8_block_down", 1, (launch_pair<EPI_STORE, false>(f.iq, cap, I, down, I, H, E, dn, tiles * ceil_div(H, 256), st)));
  }
  // Of few rows the results stay in fp32 until the sum over a token's k is rounded, which costs nothing (us a block, bf16 rows / fp32: 1 token
  // of top-6 through 64 experts of 2048 x 1408 34.9 / 34.8, 256 tokens 137 / 139, 400 tokens 162 / 156; 64 tokens of top-2 through 8 of 4096 x 14336 258 / 258).
  // Row tiles store them in bf16, as the bf16 block does: in fp32 they would be 2 H bytes a row more, written and read (16 384 tokens of 2048, top-6: 120 us
  // beside 1210), for an error of 0.0017 instead of 0.0024.
  if (nt > 0) RUN("combine", 1, combine_f32(static_cast<const float*>(f.eo), w, f.slot_row, T, k, H, out, stream));
  else RUN("combine", 1, b200moe_combine(f.eo, w, f.slot_row, T, k, H, out, stream));
#undef RUN
  return 0;
}

}  // extern "C"

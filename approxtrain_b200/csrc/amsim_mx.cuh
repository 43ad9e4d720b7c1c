// Product of two matrices in 4-bit floats with a scale per 32 elements (layout: amsim_mx.cu):
//     out[t, n] = act(sum_k A[t, k] B[n, k] + bias[n]).
//
// The rows of B (output columns) go to the 128 lanes of tensor memory and the rows of A (tokens) to its columns, so a thread
// of the epilogue holds one output column for many tokens and the 32 lanes of a warp write 32 adjacent outputs: no staging,
// any alignment, one bias value a thread.
//
// Large products: two CTAs (tcgen05 cta_group::2) share a tile of 256 output columns x 256 tokens; each loads 128 rows of either
// operand, the tensor cores read both halves.  Small ones: one CTA and a tile of 128 columns x up to 128 tokens; where those
// leave multiprocessors idle, 2, 4 or 8 CTAs (a cluster) take a share of the reduction each, put their sums in shared memory and
// each finishes a share of the tokens, adding the others' sums in their order through distributed shared memory.  A warp issues bulk copies, one
// more the products, the rest take finished tiles out of tensor memory into registers and write them while the next
// tile's products run.
//
// Measured: 8192 cubed with bf16 outputs 175 us, 6.3 PFLOP/s, the tensor pipe 85 % active at 1.59 GHz (power); 4096 cubed 30 us;
// 16 tokens x 8192 x 8192 9 us (weights at 3.9 TB/s); 8192 x 2048 FP32 outputs over 512 elements 18 us (3.7 TB/s of outputs).
//
// The accumulators truncate at every instruction (64 elements), towards zero: for FP32 outputs a chunk of the reduction is
// taken out after 2048 elements and added in registers with rounding to nearest, for 16-bit outputs after 8192.
#pragma once
#include <stdint.h>

#include "amsim_elem.cuh"

namespace amsim {
namespace mx {

constexpr int CODE_BYTES = 128 * 128;         // codes of a tile: 128 rows x 256 elements
constexpr int TILE_BYTES = CODE_BYTES + 1024;  // and its scales

struct GemmParams {
  const uint8_t *a, *b;       // tokens; output columns
  const float* bias;
  void* out;
  long long m, n;             // tokens, output columns
  int a_tiles, b_tiles, kt;   // tiles of 128 rows; of 256 elements
  int last_steps;             // 64-element steps of the last tile along the reduction
  int chunk;                  // tiles summed in tensor memory at a time
  int relu, no_tries;
  int split;                  // CTAs of a cluster that share a tile's reduction (one CTA a tile otherwise)
  int tiles_n, tiles;         // output tiles along the columns, in all
  unsigned* stuck;
};

namespace ptx {
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{.reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// A word to the other CTA, counted on its barrier (a release in the cluster).
__device__ __forceinline__ void st_async(uint32_t addr, uint32_t v, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(addr), "r"(v), "r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_barrier() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Untiled copy of `bytes` (a multiple of 16) to this CTA's shared memory, counted on its barrier.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Shared-memory matrix: layout 2 = rows of 128 bytes, 128-byte swizzle, 8-row groups 1024 bytes apart; 0 = 8 x 16-byte core matrices.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo, int layout) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) | ((uint64_t)layout << 61);
}
// kind::mxf4: E2M1 codes on both sides, E8M0 scales, FP32 sums
__host__ __device__ constexpr uint32_t idesc(int m, int n) { return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27); }
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile("{.reg .pred p; setp.ne.b32 p, %6, 0;\ntcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else
    asm volatile("{.reg .pred p; setp.ne.b32 p, %6, 0;\ntcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
template <int CG>
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
  if constexpr (CG == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Arrives at this barrier (of both CTAs) when the products issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t holder) {
  if constexpr (CG == 2) asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\ntcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::"r"(holder) : "memory");
  else asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\ntcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::"r"(holder) : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool elect_lane() {
  uint32_t e;
  asm volatile("{.reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p;}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr) : "memory");
}
}  // namespace ptx

// Waits for a phase of an mbarrier, at most so many tries (each waits a while by itself).  A thread whose wait has run out is dead: it
// waits no more and issues nothing, and the host learns of it by the mark.
constexpr int MAX_TRIES = 1 << 20;
struct Waiter {
  unsigned* stuck;
  bool dead;
  __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity) {
    if (dead) return;
    for (int i = 0; i < MAX_TRIES; ++i)
      if (ptx::mbar_try(bar, parity)) return;
    dead = true;
    *(volatile unsigned*)stuck = 1u;
  }
  __device__ __forceinline__ void wait_warp(uint32_t bar, uint32_t parity) {
    wait(bar, parity);
    dead = __any_sync(0xffffffffu, dead);
  }
};

// CG CTAs (1 or 2) share a tile of CG * 128 output columns x BN tokens.
template <int CG, int BN>
struct Shape {
  static constexpr int ROWS_A = BN / CG;                        // tokens whose codes a CTA loads
  static constexpr int HALVES = CG;                             // groups of 128 tokens' scales
  static constexpr int OFF_A = TILE_BYTES;
  static constexpr int A_CODES = ROWS_A * 128;
  static constexpr int OFF_SFA = OFF_A + (A_CODES + 1023) / 1024 * 1024;
  static constexpr int STAGE = OFF_SFA + HALVES * 1024;
  static constexpr int BYTES = TILE_BYTES + A_CODES + HALVES * 1024;  // copied per stage
  static constexpr int STAGES = 216 * 1024 / STAGE < 10 ? 216 * 1024 / STAGE : 10;
  static constexpr int SMEM = STAGES * STAGE + 1024;
  static constexpr int NACC = CG == 2 ? 1 : 2;                  // accumulators: 256 columns once, or up to 128 twice
  static constexpr int EPI = CG == 2 ? 8 : 4;                   // warps that take tiles out
  static constexpr int COLS = BN * 4 / EPI;                     // tokens of a thread
  static constexpr int THREADS = 128 + 32 * EPI;                // a warp group for copies and products (two warps of it idle), the rest for results
  static constexpr int SF_COLS = (1 + HALVES) * 2 * 4;
  static constexpr int T_SF = NACC * BN;                        // two sets of scales behind the accumulators
  static_assert(T_SF + 2 * SF_COLS <= 512, "tensor memory");
  static_assert(SMEM > 114 * 1024, "one CTA a multiprocessor: each takes all of its tensor memory");
};

template <int CG, int BN, typename T>
__global__ void __launch_bounds__(Shape<CG, BN>::THREADS, 1) gemm(const __grid_constant__ GemmParams p) {
  using S = Shape<CG, BN>;
  using namespace ptx;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[3 * S::STAGES + 2 * S::NACC + 1];
  __shared__ uint32_t tmem_holder, signal;   // signal: where the other CTA's words go
  const uint32_t smem0 = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const int lane = threadIdx.x & 31, w = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const uint32_t rank = CG == 2 ? blockIdx.x & 1u : 0u;
  const int split = CG == 1 ? p.split : 1, share = split > 1 ? blockIdx.x % split : 0;
  const int team = blockIdx.x / (CG * split), teams = gridDim.x / (CG * split);
  const int k_begin = (int)((long long)p.kt * share / split), k_end = (int)((long long)p.kt * (share + 1) / split);
  const uint32_t bar_full = smem_addr(bars), bar_empty = bar_full + 8 * S::STAGES, bar_peer = bar_empty + 8 * S::STAGES;
  const uint32_t bar_done = bar_peer + 8 * S::STAGES, bar_free = bar_done + 8 * S::NACC, bar_exit = bar_free + 8 * S::NACC;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_empty + 8 * i, 1);
      mbar_init(bar_peer + 8 * i, 1);
    }
    for (int i = 0; i < S::NACC; ++i) {
      mbar_init(bar_done + 8 * i, 1);
      mbar_init(bar_free + 8 * i, S::EPI);
    }
    mbar_init(bar_exit, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (w == 1) tmem_alloc<CG>(smem_addr(&tmem_holder));
  fence_before();
  __syncthreads();
  if (CG == 2) cluster_barrier();
  fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_holder, 0);
  Waiter wt{p.stuck, p.no_tries != 0};
  if (p.no_tries && threadIdx.x == 0) *(volatile unsigned*)p.stuck = 1u;

  // Registers for the results of a tile of 256 tokens: 128 x 64 + 256 x 216 of the launch's 384 x 168.
  if (w < 4) {
  if constexpr (CG == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (w == 0) {
    // ---- copies: a stage is one tile of either operand along the reduction -------------------------
    uint32_t b = 0, phase = 1, full_of = 0;  // full_of: bit i, copies went to stage i
    for (int tile = team; tile < p.tiles; tile += teams) {
      const int tn = tile % p.tiles_n, tt = tile / p.tiles_n;
      const int bt = min(tn * CG + (int)rank, p.b_tiles - 1);              // (a half that does not exist: any tile, its outputs are not written)
      const uint8_t* const src_b = p.b + (long long)bt * p.kt * TILE_BYTES;
      const uint8_t* const src_a = p.a + (long long)min(tt * CG + (int)rank, p.a_tiles - 1) * p.kt * TILE_BYTES;
      const uint8_t* src_s[S::HALVES];
#pragma unroll
      for (int h = 0; h < S::HALVES; ++h) src_s[h] = p.a + (long long)min(tt * CG + h, p.a_tiles - 1) * p.kt * TILE_BYTES + CODE_BYTES;
      for (int k = k_begin; k < k_end; ++k) {
        wt.wait_warp(bar_empty + 8 * b, phase);
        if (lane == 0 && !wt.dead) {
          const uint32_t at = smem0 + b * S::STAGE, bar = bar_full + 8 * b;
          const long long off = (long long)k * TILE_BYTES;
          mbar_expect(bar, S::BYTES);
          bulk_copy(at, src_b + off, TILE_BYTES, bar);
          bulk_copy(at + S::OFF_A, src_a + off, S::A_CODES, bar);
#pragma unroll
          for (int h = 0; h < S::HALVES; ++h) bulk_copy(at + S::OFF_SFA + 1024 * h, src_s[h] + off, 1024, bar);
        }
        __syncwarp();
        if (!wt.dead) full_of |= 1u << b;
        if (++b == S::STAGES) b = 0, phase ^= 1;
      }
    }
    // Copies that nobody waited for (a wait ran out) end before the CTA does.  (Otherwise this passes at once: a stage behind b
    // has been filled in this turn of the ring, the others in the one before.)
    Waiter last{p.stuck, false};
    for (uint32_t i = 0; i < (uint32_t)S::STAGES; ++i)
      if ((full_of >> i) & 1u) last.wait_warp(bar_full + 8 * i, i < b ? phase ^ 1 : phase);
  } else if (w == 1 && rank != 0) {
    // ---- tells the issuing CTA that a stage of this one is full --------------------------------------
    const uint32_t lead = cluster_addr(bar_peer, 0), word = cluster_addr(smem_addr(&signal), 0);
    uint32_t b = 0, phase = 0;
    for (int tile = team; tile < p.tiles; tile += teams)
      for (int k = k_begin; k < k_end; ++k) {
        wt.wait_warp(bar_full + 8 * b, phase);
        if (lane == 0 && !wt.dead) st_async(word, 0, lead + 8 * b);
        if (++b == S::STAGES) b = 0, phase ^= 1;
      }
  } else if (w == 1) {
    // ---- products --------------------------------------------------------------------------------------
    const bool elected = elect_lane();
    uint32_t b = 0, phase = 0, set = 0, acc = 0, acc_phase = 1;
    const uint64_t desc = smem_desc(smem0, 16, 1024, 2), desc_sf = smem_desc(smem0, 128, 128, 0);
    constexpr uint32_t id0 = idesc(128 * CG, BN);
    for (int tile = team; tile < p.tiles; tile += teams) {
      int left = 0;
      for (int k = k_begin; k < k_end; ++k) {
        const bool first = left == 0;
        if (first) {
          left = min(p.chunk, k_end - k);
          wt.wait_warp(bar_free + 8 * acc, acc_phase);
        }
        if (CG == 2 && lane == 0 && !wt.dead) mbar_expect(bar_peer + 8 * b, 4);
        wt.wait_warp(bar_full + 8 * b, phase);
        if (CG == 2) wt.wait_warp(bar_peer + 8 * b, phase);
        fence_after();
        const uint64_t at = desc + b * (S::STAGE >> 4), sf = desc_sf + b * (S::STAGE >> 4);
        const uint32_t sfb_t = tmem + S::T_SF + set * S::SF_COLS, sfa_t = sfb_t + 8;  // columns: B [half of k], A [half of k][128 tokens]
        const int steps = k + 1 == p.kt ? p.last_steps : 4;
        if (elected && !wt.dead) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (2 * j >= steps) break;
            scales_to_tmem<CG>(sfb_t + 4 * j, sf + ((CODE_BYTES + 512 * j) >> 4));
#pragma unroll
            for (int h = 0; h < S::HALVES; ++h) scales_to_tmem<CG>(sfa_t + (j * S::HALVES + h) * 4, sf + ((S::OFF_SFA + 1024 * h + 512 * j) >> 4));
          }
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            if (s >= steps) break;
            const uint32_t half = (uint32_t)(s & 1) * 2;
            mma<CG>(tmem + acc * BN, at + 2 * s, at + (S::OFF_A >> 4) + 2 * s, id0 | (half << 4) | (half << 29), sfb_t + (s >> 1) * 4, sfa_t + (s >> 1) * S::HALVES * 4, !first || s > 0);
          }
          commit<CG>(bar_empty + 8 * b);
          if (left == 1) commit<CG>(bar_done + 8 * acc);
        }
        __syncwarp();
        set ^= 1;
        if (--left == 0 && ++acc == S::NACC) acc = 0, acc_phase ^= 1;
        if (++b == S::STAGES) b = 0, phase ^= 1;
      }
    }
    // no signal is on its way to this CTA when it ends: every accumulator has been handed back
    for (int i = 0; i < S::NACC; ++i) {
      wt.wait_warp(bar_free + 8 * acc, acc_phase);
      if (++acc == S::NACC) acc = 0, acc_phase ^= 1;
    }
  }
  } else {
    if constexpr (CG == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---- results: 32 output columns (lanes) x S::COLS tokens a warp ----------------------------------
    const int quarter = w & 3, part = (w - 4) >> 2;
    const uint32_t lead_free = CG == 2 ? cluster_addr(bar_free, 0) : bar_free, word = CG == 2 ? cluster_addr(smem_addr(&signal), 0) : 0;
    uint32_t acc = 0, acc_phase = 0;
    for (int tile = team; tile < p.tiles; tile += teams) {
      const int tn = tile % p.tiles_n, tt = tile / p.tiles_n;
      float v[S::COLS];
      uint32_t at = 0;
      auto begin_chunk = [&]() {
        wt.wait_warp(bar_done + 8 * acc, acc_phase);
        fence_after();
        at = tmem + ((uint32_t)quarter << 21) + acc * BN + part * S::COLS;
      };
      auto end_chunk = [&]() {  // the accumulator may be written again
        fence_before();
        __syncwarp();
        if (lane == 0 && !wt.dead) {
          if (rank != 0) st_async(word, 0, lead_free + 8 * acc);
          else if (CG == 2 && w == 4) mbar_expect(bar_free + 8 * acc, 4 * S::EPI);
          else mbar_arrive(bar_free + 8 * acc);
        }
        if (++acc == S::NACC) acc = 0, acc_phase ^= 1;
      };
      begin_chunk();
      if constexpr (S::COLS < 32) {
        tmem_load16(at, v);
      } else {
#pragma unroll
        for (int c = 0; c < S::COLS; c += 32) tmem_load32(at + c, *reinterpret_cast<float(*)[32]>(v + c));
      }
      end_chunk();
#pragma unroll 1
      for (int k = k_begin + p.chunk; k < k_end; k += p.chunk) {
        begin_chunk();
#pragma unroll
        for (int c = 0; c < S::COLS; c += 16) {
          float x[16];
          tmem_load16(at + c, x);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[c + i] = __fadd_rn(v[c + i], x[i]);
        }
        end_chunk();
      }
      const long long n = (long long)(tn * CG + (int)rank) * 128 + quarter * 32 + lane;
      const long long t0 = (long long)tt * BN + part * S::COLS;
      const float bias = p.bias && n < p.n ? __ldg(p.bias + n) : 0.f;
      const long long pitch = p.n;
      T* out = static_cast<T*>(p.out) + t0 * p.n + n;
      auto write = [&](float o) {
        if (p.bias) o += bias;
        *out = elem_from_float<T>(p.relu && o < 0.f ? 0.f : o);
        out += pitch;
        asm volatile("" : "+l"(out));  // (one running address: the compiler would keep one for every column, and spill)
      };
      const int count = (int)min((long long)S::COLS, p.m - t0);
      if (CG == 1 && split > 1) {  // (one tile a cluster, and its stages are all used up: their place takes the sums)
        const uint32_t mine = smem0 + (quarter * 32 + lane) * 16;  // four columns at a time, 2 KB apart
#pragma unroll
        for (int c = 0; c < S::COLS; c += 4)
          asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + c * 512), "f"(v[c]), "f"(v[c + 1]), "f"(v[c + 2]), "f"(v[c + 3]) : "memory");
        cluster_barrier();
        const int c0 = S::COLS / split * share, c1 = min(count, S::COLS / split * (share + 1));  // (S::COLS / split is a multiple of 4)
        out += c0 * pitch;
        constexpr int AT_ONCE = S::COLS < 64 ? 8 : 32;  // columns of two CTAs on their way before the first is added: each round waits for the other CTA's memory
#pragma unroll 1
        for (int c = c0; c < c1; c += AT_ONCE) {
          float sum[AT_ONCE];
#pragma unroll
          for (int j = 0; j < AT_ONCE; ++j) sum[j] = 0.f;
#pragma unroll 1
          for (int i = 0; i < split; i += 2) {  // (split is even)
            float x[2][AT_ONCE];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t from = cluster_addr(mine, i + h) + c * 512;
#pragma unroll
              for (int j = 0; j < AT_ONCE; j += 4)
                if (c + j < c1) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[h][j]), "=f"(x[h][j + 1]), "=f"(x[h][j + 2]), "=f"(x[h][j + 3]) : "r"(from + j * 512) : "memory");
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = 0; j < AT_ONCE; ++j)
                if (c + j < c1) sum[j] = __fadd_rn(sum[j], x[h][j]);
          }
          if (n < p.n) {
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
              if (c + j < c1) write(sum[j]);
          }
        }
      } else if (n < p.n) {
        if (count == S::COLS) {
#pragma unroll
          for (int c = 0; c < S::COLS; ++c) write(v[c]);
        } else {
#pragma unroll
          for (int c = 0; c < S::COLS; ++c)
            if (c < count) write(v[c]);
        }
      }
    }
  }
  if (w == 1) {
    // Products that a dead warp left in flight end before the tensor memory goes.  (Otherwise this passes at once.)
    if (rank == 0 && elect_lane()) commit<CG>(bar_exit);
    Waiter last{p.stuck, false};
    last.wait_warp(bar_exit, 0);
    if (wt.dead) __nanosleep(100000);
  }
  if (CG == 1 && split > 1 && w < 4) cluster_barrier();  // (the one that the sums wait at)
  fence_before();
  __syncthreads();
  if (CG == 2 || split > 1) cluster_barrier();  // neither leaves while another may still reach its memory
  if (w == 1) tmem_free<CG>(tmem);
}

}  // namespace mx
}  // namespace amsim

// Kernels and launches of the norms around a residual block, with the block's gate and residual scale:
//     u = N_post(block) or block,   r = x + scale * gate * u,   y = N_pre(r),
//     N(z) = (z - mean z) rstd w + b  (layer)   or   z rms(z)^-1 w  (rms),
// and the gradient
//     a = dy w_pre,  g = dr + rstd (a - [mean a] - hat mean(a hat)),  hat = (r - mean) rstd
//     dx = g,  du = scale gate g,  dgate = sum scale u g,  dblock = N_post'(du) in the same form,
//     dw = sum dy hat, db = sum dy (and the same of du for N_post).
// Both are bound by memory: the forward pass reads x and block and writes y (and r where it is wanted); the backward pass
// reads dy, dr, x and block, from which it makes r and hat again, unrounded (taken from a stored bf16 r, the gradients of the FP32 weights
// were 1.6e-3 off), and writes dx and dblock.  A row stays in registers from its one read to its one write: `tpr` threads
// (4, 8, 16 or a multiple of 32 up to 512) hold E elements each; rows wider than a CTA's share go to a cluster of 2, 4 or 8 CTAs
// that add their row sums through distributed shared memory.  What a thread will need of its next rows is already on
// its way to a place of its own in shared memory (cp.async, no barrier), since the chain of two or four row sums per row
// leaves the memory idle otherwise.  Means, variances and every sum are FP32 (a variance around the thread's own mean, joined in pairs);
// r is rounded once, and y is computed from the sum before that rounding.
//
// Column sums (weights, biases, gate) are kept in registers over the consecutive rows of a worker, then added over the
// workers in a fixed order by norm_reduce: the same bits on every run, no atomics.  A gate of one row per group of rows is
// handed over whenever a worker leaves a group: directly if the whole group was its own, else through one of its two slots.
#pragma once
#include "amsim_elem.cuh"
#include "amsim_host.h"

namespace amsim {
namespace normk {

constexpr int MAX_THREADS = 512;
constexpr int SHARED_CTA = 256;   // threads of a CTA that several rows share
constexpr int GROUPS = 4;         // rows of more than a warp each that may share a CTA

struct NormParams {
  const void *x, *block, *gate, *post_w, *post_b, *pre_w, *pre_b;
  void *sum, *y;
  float* stats;              // rows x 4: mean and 1 / deviation of N_post, then of N_pre
  const void *dsum, *dy;     // backward
  int n_in;                  // tensors fetched ahead, and the places of x, block, dy, dsum and a gate of one row per row among them
  int in_x, in_block, in_dy, in_dsum, in_gate;
  void *dx, *dblock, *dgate, *dpost_w, *dpost_b, *dpre_w, *dpre_b;
  float *part, *gate_part;   // column sums: [teams][4][width], [workers][2][width]
  long long rows, per_gate;  // rows that share a row of the gate
  long long per_worker;      // consecutive rows of a worker (the threads of one row)
  long long workers;
  int width, tpr, cluster;
  int w_type, gate_type;
  float scale, eps, inv_width;
  int pre;
};

// The CTAs of a cluster meet before one writes another's shared memory: only then is it known that all of them have begun.  The arrival
// comes before the first loads and the wait behind them, so that nobody waits for long.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// What a gate is to the kernels: none; rows shared by several rows, kept like the weights; or one row for each row, fetched ahead.
constexpr int GATE_NONE = 0, GATE_SHARED = 1, GATE_ROWS = 2;

// Sums over the threads of a row.  Two buffers per sum: a warp that runs ahead writes the other one, and cannot come back to
// the first before everybody has passed the barrier between.
struct RowSum {
  float* red;     // [2][2][16] partial results of the row's warps
  float* peers;   // [2][2][8] partial results of the cluster's CTAs
  int tpr, cluster, rank, group, first_warp, buf;

  // a and b of this warp to the row's others; lane i gets those of warp i (16 and more: as i - 16), zeros where there is none
  __device__ __forceinline__ void across_warps(float& a, float& b, bool both) const {
    if ((threadIdx.x & 31) == 0) {
      const int w = (threadIdx.x >> 5) - first_warp;
      red[buf * 32 + w] = a;
      if (both) red[buf * 32 + 16 + w] = b;
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(tpr) : "memory");  // (the row's threads)
    const int i = threadIdx.x & 15;
    const bool there = i < (tpr >> 5);
    a = there ? red[buf * 32 + i] : 0.f;
    if (both) b = there ? red[buf * 32 + 16 + i] : 0.f;
  }
  // a and b of this CTA to every CTA of the cluster, in the places of its rank
  __device__ __forceinline__ void across_cluster(float a, float b) const {
    if (threadIdx.x < cluster) {
      const uint32_t at = (uint32_t)__cvta_generic_to_shared(peers + buf * 16 + rank);
      asm volatile("{.reg .b32 r; mapa.shared::cluster.u32 r, %0, %1; st.shared::cluster.f32 [r], %2; st.shared::cluster.f32 [r + 32], %3;}" ::"r"(at),
                   "r"(threadIdx.x), "f"(a), "f"(b) : "memory");
    }
    cluster_arrive();
    cluster_wait();
  }
  __device__ __forceinline__ static void add_lanes(float& a, float& b, bool both, int lanes) {
    for (int o = lanes >> 1; o; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      if (both) b += __shfl_xor_sync(0xffffffffu, b, o);
    }
  }

  __device__ __forceinline__ void operator()(float& a, float& b, bool both) {
    add_lanes(a, b, both, tpr < 32 ? tpr : 32);
    if (tpr <= 32) return;
    across_warps(a, b, both);
    add_lanes(a, b, both, 16);
    if (cluster > 1) {
      across_cluster(a, b);
      a = b = 0.f;
      for (int i = 0; i < cluster; ++i) {
        a += peers[buf * 16 + i];
        b += peers[buf * 16 + 8 + i];
      }
    }
    buf ^= 1;
  }

  // Mean and sum of squares around it over threads of n elements each, from the threads' own: one exchange between warps where a
  // mean and then a variance take two, and as exact.  Pairs of lanes join their parts (T. Chan, G. Golub, R. LeVeque 1979),
  // warps and CTAs add theirs around the mean of the means.
  __device__ __forceinline__ void spread(float n, float& mean, float& m2) {
    for (int o = 1; o < (tpr < 32 ? tpr : 32); o <<= 1, n *= 2.f) {
      const float mean1 = __shfl_xor_sync(0xffffffffu, mean, o), m21 = __shfl_xor_sync(0xffffffffu, m2, o), d = mean1 - mean;
      mean = 0.5f * (mean + mean1);
      m2 = __fadd_rn(__fadd_rn(m2, m21), __fmul_rn(__fmul_rn(d, d), 0.5f * n));
    }
    if (tpr <= 32) return;
    across_warps(mean, m2, true);
    const int warps = tpr >> 5;
    float all = mean, none = 0.f;
    add_lanes(all, none, false, 16);
    all /= (float)warps;
    if ((threadIdx.x & 15) < warps) m2 += n * (mean - all) * (mean - all);
    add_lanes(m2, none, false, 16);
    mean = all;
    if (cluster > 1) {
      n *= (float)warps;
      across_cluster(mean, m2);
      mean = m2 = 0.f;
      for (int i = 0; i < cluster; ++i) mean += peers[buf * 16 + i];
      mean /= (float)cluster;
      for (int i = 0; i < cluster; ++i) m2 += peers[buf * 16 + 8 + i] + n * (peers[buf * 16 + i] - mean) * (peers[buf * 16 + i] - mean);
    }
    buf ^= 1;
  }
};

// Where a thread's elements are: chunk c holds columns at(c) .. at(c) + V - 1.  FULL: every chunk of every thread exists.
template <int V, bool FULL>
struct Cols {
  int first, step, width;
  __device__ __forceinline__ int at(int c) const { return first + c * step; }
  __device__ __forceinline__ bool ok(int c) const { return FULL || at(c) < width; }
};

// Rows fetched ahead of their use, each thread its own chunks of 16, 8 or 4 bytes: stage, tensor, chunk.  Single 16-bit elements (rows of
// odd length) are loaded when they are needed.
template <typename T, int V, int N, bool FULL>
struct Ahead {
  static constexpr int CHUNK = V * (int)sizeof(T);
  static constexpr bool ON = CHUNK >= 4;
  static constexpr int STAGES = sizeof(T) == 4 ? 2 : 3;
  uint32_t base;
  int n_in, stage;
  __device__ __forceinline__ Ahead(const NormParams& p, void* smem) : n_in(p.n_in), stage(0) {
    base = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * CHUNK;
  }
  // bytes that a CTA's stages take
  __host__ __device__ static __forceinline__ int bytes(int n_in, int threads) { return ON ? STAGES * n_in * N * CHUNK * threads : 0; }
  __device__ __forceinline__ uint32_t place(int st, int k, int c) const { return base + ((st * n_in + k) * N + c) * (blockDim.x * CHUNK); }
  // tensor number k of the row whose first element of this thread is number `at`, into stage `st`
  __device__ __forceinline__ void fetch(int st, int k, const void* src, long long at, const Cols<V, FULL>& cols) const {
    if (!ON || !src) return;
    const T* from = static_cast<const T*>(src) + at;
    uint32_t to = place(st, k, 0);
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (cols.ok(c)) {
        if constexpr (CHUNK == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
        else if constexpr (CHUNK == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
        else if constexpr (CHUNK == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
      }
      from += cols.step;
      to += blockDim.x * CHUNK;
    }
  }
  __device__ __forceinline__ void commit() const {
    if (ON) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void ready() const {
    if (ON) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
  }
  // the stage that is filled while `stage` is used: the one used before it
  __device__ __forceinline__ int free_stage() const { return stage == 0 ? STAGES - 1 : stage - 1; }
  __device__ __forceinline__ void next() { stage = stage + 1 == STAGES ? 0 : stage + 1; }
  __device__ __forceinline__ void read(int k, int c, const void* src, long long at, const Cols<V, FULL>& cols, float (&o)[V]) const {
    if constexpr (CHUNK == 16) {
      uint32_t w[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(place(stage, k, c)) : "memory");
      unpack16<T, V>(w, o);
    } else if constexpr (CHUNK == 8) {
      static_assert(sizeof(T) == 4, "two floats");
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(o[0]), "=f"(o[1]) : "r"(place(stage, k, c)) : "memory");
    } else if constexpr (CHUNK == 4) {
      uint32_t w;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(place(stage, k, c)) : "memory");
      T e[V];
      memcpy(e, &w, 4);
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = elem_to_float(e[i]);
    } else {
      load_vec<T, V>(src, at + cols.at(c), o);
    }
  }
};

// Weights, biases and the gate's row of a thread's columns, as FP32 in places of its own in shared memory: read for every row
// without a look at their type or at whether they exist.
template <int V, int N, bool FULL>
struct Kept {
  float* base;
  __device__ __forceinline__ Kept(void* smem) : base(static_cast<float*>(smem) + threadIdx.x * (V < 4 ? 1 : 4)) {}
  __device__ __forceinline__ float* place(int a, int c, int f) const {
    return V < 4 ? base + ((a * N + c) * V + f) * (int)blockDim.x : base + ((a * N + c) * (V / 4) + f) * (4 * (int)blockDim.x);
  }
  __device__ __forceinline__ void keep(int a, const void* src, long long at, bool f32, int t16, float absent, const Cols<V, FULL>& cols) const {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = absent;
      if (src && cols.ok(c)) load_param<V>(src, at + cols.at(c), f32, t16, v);
      if constexpr (V < 4) {
#pragma unroll
        for (int f = 0; f < V; ++f) *place(a, c, f) = v[f];
      } else {
#pragma unroll
        for (int f = 0; f < V / 4; ++f) *reinterpret_cast<float4*>(place(a, c, f)) = make_float4(v[4 * f], v[4 * f + 1], v[4 * f + 2], v[4 * f + 3]);
      }
    }
  }
  __device__ __forceinline__ void read(int a, int c, float (&o)[V]) const {
    if constexpr (V < 4) {
#pragma unroll
      for (int f = 0; f < V; ++f) o[f] = *place(a, c, f);
    } else {
#pragma unroll
      for (int f = 0; f < V / 4; ++f) {
        const float4 v = *reinterpret_cast<const float4*>(place(a, c, f));
        o[4 * f] = v.x; o[4 * f + 1] = v.y; o[4 * f + 2] = v.z; o[4 * f + 3] = v.w;
      }
    }
  }
};

// Places among the kept arrays: N_pre's weight and bias (forward), N_post's, the gate.
template <bool LAYER, bool POST, int GATE, bool BWD>
struct Places {
  static constexpr int PRE_W = 0, PRE_B = 1, POST_W = LAYER && !BWD ? 2 : 1, POST_B = POST_W + 1, GATE_V = POST_W + (POST ? LAYER ? 2 : 1 : 0);
  static constexpr int COUNT = GATE_V + (GATE == GATE_SHARED ? 1 : 0);
};

template <bool LAYER, int N, int V, bool FULL>
__device__ __forceinline__ void row_stats(const float (&z)[N][V], const Cols<V, FULL>& cols, const NormParams& p, RowSum& sum, float& mean, float& rstd) {
  float s = 0.f, m2 = 0.f, none = 0.f;
  mean = 0.f;
  if (LAYER) {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) s += z[c][e];  // (columns past the end hold zeros)
    if (FULL) {
      mean = s * (1.f / (N * V));  // (the thread's own)
    } else {
      sum(s, none, false);
      mean = s * p.inv_width;
    }
  }
#pragma unroll
  for (int c = 0; c < N; ++c)
    if (!LAYER || cols.ok(c)) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = LAYER ? z[c][e] - mean : z[c][e];
        m2 += d * d;
      }
    }
  if (LAYER && FULL) sum.spread((float)(N * V), mean, m2);
  else sum(m2, none, false);
  rstd = 1.f / sqrtf(m2 * p.inv_width + p.eps);
}

// The rows of a worker and the gate's row that they share, walked in order.
struct Walk {
  long long row, last, at, gate_row, gate_left;  // at: first element; gate_left: rows until the gate's next one
  __device__ __forceinline__ Walk(const NormParams& p, long long worker) {
    row = min(worker * p.per_worker, p.rows);
    last = min(row + p.per_worker, p.rows);
    at = row * p.width;
    gate_row = row / p.per_gate;
    gate_left = p.per_gate - (row - gate_row * p.per_gate);
  }
  __device__ __forceinline__ bool live() const { return row < last; }
  // true where the gate's next row begins
  __device__ __forceinline__ bool next(const NormParams& p) {
    ++row;
    at += p.width;
    if (--gate_left) return false;
    gate_left = p.per_gate;
    ++gate_row;
    return true;
  }
};

// Forward.  8192 x 512 FP32, x + block and a layer norm: 11.7 us (4.3 TB/s; 50 MB from and to memory).  16384 x 2048 bf16 with both
// rms norms, a gate per sequence and the sum written: 59 us (4.6 TB/s), 57 % of the issue slots and 44 % of DRAM: latency, as below.
template <typename T, int V, bool LAYER, bool POST, int GATE, int E, bool FULL>
__global__ void __launch_bounds__(MAX_THREADS) norm_fwd(const __grid_constant__ NormParams p) {
  constexpr int N = E / V;
  using A = Ahead<T, V, N, FULL>;
  using P = Places<LAYER, POST, GATE, false>;
  __shared__ float red[GROUPS][64], peers[32];
  extern __shared__ __align__(16) uint8_t smem[];
  const int group = threadIdx.x / p.tpr, t = threadIdx.x - group * p.tpr, groups = blockDim.x / p.tpr;
  const int rank = blockIdx.x % p.cluster;
  RowSum sum{red[p.tpr > 32 ? group : 0], peers, p.tpr, p.cluster, rank, group, group * p.tpr >> 5, 0};
  const Cols<V, FULL> cols{(rank * N * p.tpr + t) * V, p.tpr * V, p.width};
  Walk w(p, (long long)(blockIdx.x / p.cluster) * groups + group);
  if (p.cluster > 1) cluster_arrive();
  A in(p, smem);
  const Kept<V, N, FULL> kept(smem + A::bytes(p.n_in, blockDim.x));
  long long to_fetch = w.last - w.row, fetch_at = w.at + cols.first;
  auto fetch = [&](int st) {
    if (to_fetch > 0) {
      in.fetch(st, p.in_x, p.x, fetch_at, cols);
      in.fetch(st, p.in_block, p.block, fetch_at, cols);
      if (GATE == GATE_ROWS) in.fetch(st, p.in_gate, p.gate, fetch_at, cols);
      fetch_at += p.width;
      --to_fetch;
    }
    in.commit();
  };
  for (int i = 0; i < A::STAGES - 1; ++i) fetch(i);
  const bool w32 = p.w_type == 0, g32 = p.gate_type == 0;
  if (p.pre) {
    kept.keep(P::PRE_W, p.pre_w, 0, w32, type16<T>(), 1.f, cols);
    if (LAYER) kept.keep(P::PRE_B, p.pre_b, 0, w32, type16<T>(), 0.f, cols);
  }
  if (POST) {
    kept.keep(P::POST_W, p.post_w, 0, w32, type16<T>(), 1.f, cols);
    if (LAYER) kept.keep(P::POST_B, p.post_b, 0, w32, type16<T>(), 0.f, cols);
  }
  if (p.cluster > 1) cluster_wait();
  bool new_gate = true;
  for (long long i = 0; i < p.per_worker; ++i, in.next()) {  // (the same trips for all threads)
    const bool live = w.live();
    float r[N][V], u[N][V];
    fetch(in.free_stage());
    if (GATE == GATE_SHARED && live && new_gate) kept.keep(P::GATE_V, p.gate, w.gate_row * p.width, g32, type16<T>(), 0.f, cols);
    in.ready();
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (live && cols.ok(c)) {
        in.read(p.in_x, c, p.x, w.at, cols, r[c]);
        if (p.block) in.read(p.in_block, c, p.block, w.at, cols, u[c]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) r[c][e] = u[c][e] = 0.f;
      }
    }
    if (POST) {
      float mean, rstd;
      row_stats<LAYER>(u, cols, p, sum, mean, rstd);
#pragma unroll
      for (int c = 0; c < N; ++c) {
        float wv[V], bv[V];
        kept.read(P::POST_W, c, wv);
        if (LAYER) kept.read(P::POST_B, c, bv);
#pragma unroll
        for (int e = 0; e < V; ++e) u[c][e] = LAYER ? (u[c][e] - mean) * rstd * wv[e] + bv[e] : u[c][e] * rstd * wv[e];
      }
      if (p.stats && live && t == 0 && rank == 0) *reinterpret_cast<float2*>(p.stats + w.row * 4) = make_float2(mean, rstd);
    }
    if (p.block) {
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if (!cols.ok(c)) continue;  // (what N_post's bias left there stays out of the row's sums)
        if (GATE != GATE_NONE) {
          float gv[V];
          if (GATE == GATE_SHARED) {
            kept.read(P::GATE_V, c, gv);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) gv[e] = 0.f;
            if (live) in.read(p.in_gate, c, p.gate, w.at, cols, gv);
          }
#pragma unroll
          for (int e = 0; e < V; ++e) u[c][e] *= gv[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) r[c][e] += p.scale * u[c][e];
      }
    }
    if (p.sum && live) {
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (cols.ok(c)) store_vec<T, V>(p.sum, w.at + cols.at(c), r[c]);
    }
    if (p.pre) {
      float mean, rstd;
      row_stats<LAYER>(r, cols, p, sum, mean, rstd);
      if (live) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
          if (!cols.ok(c)) continue;
          float wv[V], bv[V];
          kept.read(P::PRE_W, c, wv);
          if (LAYER) kept.read(P::PRE_B, c, bv);
#pragma unroll
          for (int e = 0; e < V; ++e) r[c][e] = LAYER ? (r[c][e] - mean) * rstd * wv[e] + bv[e] : r[c][e] * rstd * wv[e];
          store_vec<T, V>(p.y, w.at + cols.at(c), r[c]);
        }
        if (p.stats && t == 0 && rank == 0) *reinterpret_cast<float2*>(p.stats + w.row * 4 + 2) = make_float2(mean, rstd);
      }
    }
    new_gate = w.next(p);
  }
}

// Adds one array of column sums over the row groups of a block and writes the block's line of partial sums.
template <int N, int V, bool FULL>
__device__ __forceinline__ void flush_block(float (&acc)[N][V], const Cols<V, FULL>& cols, float* line, float* buf, int t, int group, int groups, int tpr) {
  if (groups == 1) {
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (cols.ok(c)) {
#pragma unroll
        for (int e = 0; e < V; ++e) line[cols.at(c) + e] = acc[c][e];
      }
    return;
  }
#pragma unroll
  for (int c = 0; c < N; ++c) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      __syncthreads();
      buf[threadIdx.x] = acc[c][e];
      __syncthreads();
      if (group == 0 && cols.ok(c)) {
        float s = 0.f;
        for (int g = 0; g < groups; ++g) s += buf[g * tpr + t];
        line[cols.at(c) + e] = s;
      }
    }
  }
}

// Backward.  The same cases: 14.7 us (4.6 TB/s) and 5.1 us of norm_reduce; 120 us (3.3 TB/s) and 6 us.  The second is bound by latency: 54 % of
// the issue slots and 37 % of DRAM, with 16 warps a multiprocessor (118 registers), each in a chain of two row sums a row; about 70 instructions
// an element (conversions, 28 of arithmetic, and a row's fixed share over 8 elements) leave little to hide it behind.
template <typename T, int V, bool LAYER, bool POST, int GATE, int E, bool FULL>
__global__ void __launch_bounds__(MAX_THREADS) norm_bwd(const __grid_constant__ NormParams p) {
  constexpr int N = E / V;
  using A = Ahead<T, V, N, FULL>;
  using P = Places<LAYER, POST, GATE, true>;
  __shared__ float red[GROUPS][64], peers[32], buf[SHARED_CTA];
  extern __shared__ __align__(16) uint8_t smem[];
  const int group = threadIdx.x / p.tpr, t = threadIdx.x - group * p.tpr, groups = blockDim.x / p.tpr;
  const int rank = blockIdx.x % p.cluster;
  RowSum sum{red[p.tpr > 32 ? group : 0], peers, p.tpr, p.cluster, rank, group, group * p.tpr >> 5, 0};
  const Cols<V, FULL> cols{(rank * N * p.tpr + t) * V, p.tpr * V, p.width};
  const long long team = blockIdx.x / p.cluster, worker = team * groups + group;
  Walk w(p, worker);
  const long long first = w.row;
  float dw[N][V], db[N][V], dpw[N][V], dpb[N][V], dg[N][V];
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[c][e] = db[c][e] = dpw[c][e] = dpb[c][e] = dg[c][e] = 0.f;
  if (p.cluster > 1) cluster_arrive();
  A in(p, smem);
  const Kept<V, N, FULL> kept(smem + A::bytes(p.n_in, blockDim.x));
  long long to_fetch = w.last - w.row, fetch_at = w.at + cols.first;
  auto fetch = [&](int st) {
    if (to_fetch > 0) {
      in.fetch(st, p.in_dy, p.dy, fetch_at, cols);
      in.fetch(st, p.in_x, p.x, fetch_at, cols);
      in.fetch(st, p.in_block, p.block, fetch_at, cols);
      in.fetch(st, p.in_dsum, p.dsum, fetch_at, cols);
      if (GATE == GATE_ROWS) in.fetch(st, p.in_gate, p.gate, fetch_at, cols);
      fetch_at += p.width;
      --to_fetch;
    }
    in.commit();
  };
  for (int i = 0; i < A::STAGES - 1; ++i) fetch(i);
  const float4* stats_at = reinterpret_cast<const float4*>(p.stats) + w.row;
  float4 st_next = w.live() ? __ldg(stats_at) : make_float4(0.f, 0.f, 0.f, 0.f);
  const bool w32 = p.w_type == 0, g32 = p.gate_type == 0;
  if (p.dy) kept.keep(P::PRE_W, p.pre_w, 0, w32, type16<T>(), 1.f, cols);
  if (POST) {
    kept.keep(P::POST_W, p.post_w, 0, w32, type16<T>(), 1.f, cols);
    if (LAYER) kept.keep(P::POST_B, p.post_b, 0, w32, type16<T>(), 0.f, cols);
  }
  auto read_gate = [&](int c, float (&gv)[V]) {
    if (GATE == GATE_SHARED) kept.read(P::GATE_V, c, gv);
    else in.read(p.in_gate, c, p.gate, w.at, cols, gv);
  };
  if (p.cluster > 1) cluster_wait();
  bool new_gate = true;
  for (long long i = 0; i < p.per_worker; ++i, in.next()) {  // (the same trips for all threads)
    const bool live = w.live();
    float g[N][V], hat[N][V], u[N][V];
    const float4 st = st_next;
    if (w.row + 1 < w.last) st_next = __ldg(++stats_at);
    fetch(in.free_stage());
    if (GATE == GATE_SHARED && live && new_gate) kept.keep(P::GATE_V, p.gate, w.gate_row * p.width, g32, type16<T>(), 0.f, cols);
    in.ready();
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (!live || !cols.ok(c)) {
#pragma unroll
        for (int e = 0; e < V; ++e) g[c][e] = hat[c][e] = u[c][e] = 0.f;
        continue;
      }
      // the sum again, as the forward pass had it before rounding
      if (p.block) {
        in.read(p.in_block, c, p.block, w.at, cols, u[c]);
        if (POST) {
          float wv[V], bv[V];
          kept.read(P::POST_W, c, wv);
          if (LAYER) kept.read(P::POST_B, c, bv);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            u[c][e] = LAYER ? (u[c][e] - st.x) * st.y : u[c][e] * st.y;
            hat[c][e] = LAYER ? u[c][e] * wv[e] + bv[e] : u[c][e] * wv[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) hat[c][e] = u[c][e];
        }
        if (GATE != GATE_NONE) {
          float gv[V];
          read_gate(c, gv);
#pragma unroll
          for (int e = 0; e < V; ++e) hat[c][e] *= gv[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) hat[c][e] = u[c][e] = 0.f;
      }
      if (p.dy) {
        float xv[V], wv[V];
        in.read(p.in_x, c, p.x, w.at, cols, xv);
        in.read(p.in_dy, c, p.dy, w.at, cols, g[c]);
        kept.read(P::PRE_W, c, wv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float r = xv[e] + p.scale * hat[c][e];
          hat[c][e] = LAYER ? (r - st.z) * st.w : r * st.w;
          dw[c][e] += g[c][e] * hat[c][e];
          if (LAYER) db[c][e] += g[c][e];
          g[c][e] *= wv[e];
          if (LAYER) s1 += g[c][e];
          s2 += g[c][e] * hat[c][e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) g[c][e] = 0.f;
      }
    }
    if (p.dy) {
      sum(LAYER ? s1 : s2, LAYER ? s2 : s1, LAYER);
      s1 *= p.inv_width;
      s2 *= p.inv_width;
#pragma unroll
      for (int c = 0; c < N; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) g[c][e] = st.w * ((LAYER ? g[c][e] - s1 : g[c][e]) - hat[c][e] * s2);
    }
    if (live) {
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if (!cols.ok(c)) continue;
        if (p.dsum) {
          float dr[V];
          in.read(p.in_dsum, c, p.dsum, w.at, cols, dr);
#pragma unroll
          for (int e = 0; e < V; ++e) g[c][e] += dr[e];
        }
        store_vec<T, V>(p.dx, w.at + cols.at(c), g[c]);
      }
    }
    if (!POST && GATE == GATE_NONE) {
      if (p.dblock && live) {
#pragma unroll
        for (int c = 0; c < N; ++c)
          if (cols.ok(c)) {
            float d[V];
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = p.scale * g[c][e];
            store_vec<T, V>(p.dblock, w.at + cols.at(c), d);
          }
      }
      w.next(p);
      continue;
    }
    s1 = s2 = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (!live || !cols.ok(c)) continue;
      float wv[V], bv[V], gv[V];
      if (POST) kept.read(P::POST_W, c, wv);
      if (POST && GATE != GATE_NONE && LAYER) kept.read(P::POST_B, c, bv);
      if (GATE != GATE_NONE) read_gate(c, gv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = u[c][e], d = p.scale * g[c][e];
        if (GATE != GATE_NONE) dg[c][e] += (!POST ? h : LAYER ? h * wv[e] + bv[e] : h * wv[e]) * d;
        float du = GATE != GATE_NONE ? d * gv[e] : d;
        if (POST) {
          dpw[c][e] += du * h;
          if (LAYER) dpb[c][e] += du;
          du *= wv[e];
          if (LAYER) s1 += du;
          s2 += du * h;
        }
        g[c][e] = du;
      }
    }
    if (POST) {
      sum(LAYER ? s1 : s2, LAYER ? s2 : s1, LAYER);
      s1 *= p.inv_width;
      s2 *= p.inv_width;
#pragma unroll
      for (int c = 0; c < N; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) g[c][e] = st.y * ((LAYER ? g[c][e] - s1 : g[c][e]) - u[c][e] * s2);
    }
    if (p.dblock && live) {
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (cols.ok(c)) store_vec<T, V>(p.dblock, w.at + cols.at(c), g[c]);
    }
    if (GATE != GATE_NONE && live && p.dgate && (w.row + 1 == w.last || w.gate_left == 1)) {
      const long long begin = w.gate_row * p.per_gate;
      const bool whole = begin >= first && begin + p.per_gate <= w.last;
      float* slot = p.gate_part + (worker * 2 + (begin < first ? 0 : 1)) * p.width;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if (!cols.ok(c)) continue;
        if (whole) {
          store_param<V>(p.dgate, w.gate_row * p.width + cols.at(c), g32, type16<T>(), dg[c]);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) slot[cols.at(c) + e] = dg[c][e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) dg[c][e] = 0.f;
      }
    }
    new_gate = w.next(p);
  }
  float* line = p.part + team * 4 * p.width;
  if (p.dpre_w) flush_block(dw, cols, line, buf, t, group, groups, p.tpr);
  if (LAYER && p.dpre_b) flush_block(db, cols, line + p.width, buf, t, group, groups, p.tpr);
  if (POST && p.dpost_w) flush_block(dpw, cols, line + 2 * p.width, buf, t, group, groups, p.tpr);
  if (POST && LAYER && p.dpost_b) flush_block(dpb, cols, line + 3 * p.width, buf, t, group, groups, p.tpr);
}

// blockIdx.y < 4: sums a weight's or bias's lines over the teams.  Then the rows of the gate that several workers share, each the sum of
// its slots: one block for each row of the gate, or, where there are more of those than workers, for each worker that takes
// over a row from the one before it, where that row began.  32 columns x 16 consecutive shares.
constexpr int SHARES = 16;
template <typename T>
__global__ void __launch_bounds__(32 * SHARES) norm_reduce(const __grid_constant__ NormParams p, int teams, int by_worker) {
  __shared__ float part[SHARES][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), share = threadIdx.x >> 5;
  const bool ok = col < p.width;
  float s = 0.f;
  void* out = nullptr;
  long long out_at = col;
  bool f32 = p.w_type == 0;
  if (blockIdx.y < 4) {
    out = blockIdx.y == 0 ? p.dpre_w : blockIdx.y == 1 ? p.dpre_b : blockIdx.y == 2 ? p.dpost_w : p.dpost_b;
    if (!out) return;
    const int per = (teams + SHARES - 1) / SHARES, end = min(teams, (share + 1) * per);
    const float* at = p.part + (long long)blockIdx.y * p.width + col;
#pragma unroll 8
    for (int i = share * per; i < end; ++i) s += ok ? __ldcg(at + (long long)i * 4 * p.width) : 0.f;
  } else {
    const long long item = (long long)blockIdx.y - 4;
    long long g = item;
    if (by_worker) {
      const long long row = (item + 1) * p.per_worker;
      if (row >= p.rows || row % p.per_gate == 0) return;
      g = row / p.per_gate;
      if (g * p.per_gate / p.per_worker != item) return;
    }
    const long long begin = g * p.per_gate, w0 = begin / p.per_worker, w1 = (begin + p.per_gate - 1) / p.per_worker, n = w1 - w0 + 1;
    if (n == 1) return;
    const long long per = (n + SHARES - 1) / SHARES, end = min(n, (share + 1) * per);  // slots: the second of w0, the first of the others
#pragma unroll 4
    for (long long i = share * per; i < end; ++i) s += ok ? __ldcg(p.gate_part + ((w0 + i) * 2 + (i == 0 ? 1 : 0)) * p.width + col) : 0.f;
    out = p.dgate;
    out_at = g * p.width + col;
    f32 = p.gate_type == 0;
  }
  part[share][threadIdx.x & 31] = s;
  __syncthreads();
  if (share == 0 && ok) {
    float v[1] = {0.f};
    for (int i = 0; i < SHARES; ++i) v[0] += part[i][threadIdx.x & 31];
    store_param<1>(out, out_at, f32, type16<T>(), v);
  }
}

// Zeros for gradients of a call without rows.
template <typename T>
__global__ void norm_zero(const __grid_constant__ NormParams p) {
  const int col = blockIdx.x * blockDim.x + threadIdx.x;
  if (col >= p.width) return;
  void* out = blockIdx.y == 0 ? p.dpre_w : blockIdx.y == 1 ? p.dpre_b : blockIdx.y == 2 ? p.dpost_w : p.dpost_b;
  const float zero[1] = {0.f};
  if (out) store_param<1>(out, col, p.w_type == 0, type16<T>(), zero);
}

struct Shape {
  int e, tpr, cluster, threads;
};

// Threads per row: enough for E elements each: 4, 8, 16 or a multiple of 32; rows of up to 128 threads share CTAs of 256.
static bool shape_of(int width, int e, Shape* s) {
  s->e = e;
  s->cluster = 1;
  while ((long long)s->cluster * MAX_THREADS * e < width) s->cluster *= 2;
  if (s->cluster > 8) return false;
  const int share = (width + s->cluster - 1) / s->cluster, need = (share + e - 1) / e;
  s->tpr = need <= 4 ? 4 : need <= 8 ? 8 : need <= 16 ? 16 : (need + 31) / 32 * 32;
  const int groups = s->tpr < SHARED_CTA ? SHARED_CTA / s->tpr : 1;
  s->threads = groups * s->tpr;  // (a multiple of 32: 256 for rows of fewer threads)
  return true;
}

struct Plan {
  Shape s;
  int groups;
  long long teams, workers, per_worker;
  size_t part_bytes, gate_bytes;
};

// Consecutive rows for each worker: as many CTAs as stay resident (`resident` threads a multiprocessor), at least `least` rows a worker.
static bool make_plan(long long rows, int width, int elems, int resident, int least, bool gate, int device, Plan* pl) {
  if (!shape_of(width, elems, &pl->s)) return false;
  pl->groups = pl->s.threads / pl->s.tpr;
  long long teams = (long long)host_sm_count(device) * (resident / pl->s.threads) / pl->s.cluster;
  const long long most = (rows + (long long)least * pl->groups - 1) / ((long long)least * pl->groups);
  if (teams > most) teams = most;
  if (teams < 1) teams = 1;
  pl->per_worker = (rows + teams * pl->groups - 1) / (teams * pl->groups);
  if (pl->per_worker < 1) pl->per_worker = 1;
  pl->teams = (rows + pl->per_worker * pl->groups - 1) / (pl->per_worker * pl->groups);
  if (pl->teams < 1) pl->teams = 1;
  pl->workers = pl->teams * pl->groups;
  pl->part_bytes = ((size_t)pl->teams * 4 * width * sizeof(float) + 255) & ~(size_t)255;
  pl->gate_bytes = gate ? (size_t)pl->workers * 2 * width * sizeof(float) : 0;
  return true;
}
// Backward: each worker leaves a line of column sums, so at least four rows.  Passes through N_post or a gate keep up to five arrays of
// them: 8 elements a thread fit 128 registers.  FP32 without them: 8 as well (four tensors of 16, two stages, do not fit shared
// memory for 512 threads), but 16 for rows that 8 would split over a cluster, as long as those fit (36 bytes a column).
static bool bwd_plan(long long rows, int width, bool post, bool gate, int dtype, int device, Plan* pl) {
  const bool eight = post || gate || (dtype == 0 && (width <= MAX_THREADS * 8 || width > 6144));
  return make_plan(rows, width, eight ? 8 : 16, 512, 4, gate, device, pl);
}

static bool aligned(const void* p, unsigned bytes = 16) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// Whether every row of every tensor is whole chunks of `v` elements at multiples of `bytes`.
static bool chunks_ok(const NormParams& p, int v, unsigned bytes) {
  if (p.width % v) return false;
  for (const void* t : {p.x, p.block, p.gate, p.post_w, p.post_b, p.pre_w, p.pre_b, (const void*)p.sum, (const void*)p.y, p.dsum, p.dy, (const void*)p.dx, (const void*)p.dblock, (const void*)p.dgate})
    if (!aligned(t, bytes)) return false;
  return true;
}

constexpr int MOST_SMEM = 224 * 1024;  // dynamic; the static arrays have the rest of a CTA's 227 KB
template <auto kernel>
static cudaError_t launch(const Plan& pl, int smem, cudaStream_t st, const NormParams& p) {
  if (smem > 40 * 1024) {  // (48 KB with the static arrays)
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = host_allow_smem(kernel, MOST_SMEM, done);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pl.teams * pl.s.cluster));
  cfg.blockDim = dim3(pl.s.threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = pl.s.cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = pl.s.cluster > 1 ? 1 : 0;
  host_count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int V, bool LAYER, bool POST, int GATE, int E>
static cudaError_t launch_bwd(const NormParams& p, cudaStream_t st, const Plan& pl) {
  constexpr bool WIDE = V * sizeof(T) == 16;  // (the form without checks of the width only for these)
  const int smem = Ahead<T, V, E / V, false>::bytes(p.n_in, pl.s.threads) + Places<LAYER, POST, GATE, true>::COUNT * E * 4 * pl.s.threads;
  if (WIDE && p.width == pl.s.tpr * E * pl.s.cluster) return launch<norm_bwd<T, V, LAYER, POST, GATE, E, WIDE>>(pl, smem, st, p);
  return launch<norm_bwd<T, V, LAYER, POST, GATE, E, false>>(pl, smem, st, p);
}
// `fits`: whether this many elements a thread fit shared memory (nothing is launched otherwise).
template <typename T, int V, bool LAYER, bool POST, int GATE, int E>
static cudaError_t launch_fwd(NormParams& p, int device, cudaStream_t st, bool* fits) {
  constexpr bool WIDE = V * sizeof(T) == 16;
  Plan pl;
  if (!make_plan(p.rows, p.width, E, 512, 1, false, device, &pl)) return cudaErrorInvalidValue;
  const int smem = Ahead<T, V, E / V, false>::bytes(p.n_in, pl.s.threads) + Places<LAYER, POST, GATE, false>::COUNT * E * 4 * pl.s.threads;
  *fits = smem <= MOST_SMEM;
  if (!*fits) return cudaSuccess;
  p.tpr = pl.s.tpr; p.cluster = pl.s.cluster; p.per_worker = pl.per_worker; p.workers = pl.workers;
  if (WIDE && p.width == pl.s.tpr * E * pl.s.cluster) return launch<norm_fwd<T, V, LAYER, POST, GATE, E, WIDE>>(pl, smem, st, p);
  return launch<norm_fwd<T, V, LAYER, POST, GATE, E, false>>(pl, smem, st, p);
}

template <typename T, int V, bool LAYER, bool POST, int GATE>
static cudaError_t launch_t(NormParams& p, bool backward, int device, cudaStream_t st, const Plan* bwd) {
  if (backward) {
    if constexpr (!POST && GATE == GATE_NONE)
      if (bwd->s.e == 16) return launch_bwd<T, V, LAYER, POST, GATE, 16>(p, st, *bwd);
    if constexpr (POST || GATE != GATE_NONE || sizeof(T) == 4) return launch_bwd<T, V, LAYER, POST, GATE, 8>(p, st, *bwd);
    return cudaErrorInvalidValue;  // (no plan says so)
  }
  // 16 elements a thread where 512 threads a multiprocessor have room for them; where they have not, 8, unless that would split rows
  // over a cluster, whose two or four exchanges a row cost more than the threads that do not fit
  constexpr int ROOM = 512 * 16 * (4 * Places<LAYER, POST, GATE, false>::COUNT + (sizeof(T) == 4 ? 8 : 6) * (GATE == GATE_ROWS ? 3 : 2));
  bool fits = false;
  if (ROOM <= MOST_SMEM || p.width > MAX_THREADS * 8) {
    const cudaError_t e = launch_fwd<T, V, LAYER, POST, GATE, 16>(p, device, st, &fits);
    if (fits || e != cudaSuccess) return e;
  }
  return launch_fwd<T, V, LAYER, POST, GATE, 8>(p, device, st, &fits);
}

template <typename T, int V, bool LAYER>
static cudaError_t launch_l(NormParams& p, bool backward, bool post, int gate, int device, cudaStream_t st, const Plan* bwd) {
  if (gate == GATE_ROWS) return post ? launch_t<T, V, LAYER, true, GATE_ROWS>(p, backward, device, st, bwd) : launch_t<T, V, LAYER, false, GATE_ROWS>(p, backward, device, st, bwd);
  if (gate == GATE_SHARED) return post ? launch_t<T, V, LAYER, true, GATE_SHARED>(p, backward, device, st, bwd) : launch_t<T, V, LAYER, false, GATE_SHARED>(p, backward, device, st, bwd);
  return post ? launch_t<T, V, LAYER, true, GATE_NONE>(p, backward, device, st, bwd) : launch_t<T, V, LAYER, false, GATE_NONE>(p, backward, device, st, bwd);
}

template <typename T, int V>
static cudaError_t launch_v(NormParams& p, bool backward, bool layer, bool post, int gate, int device, cudaStream_t st, const Plan* bwd) {
  return layer ? launch_l<T, V, true>(p, backward, post, gate, device, st, bwd) : launch_l<T, V, false>(p, backward, post, gate, device, st, bwd);
}

// Chunks of 16 bytes where width and addresses allow them, else two elements, else single ones.  (Rows of 3950 FP32, N_post and a gate of
// every row, forward and backward: 1241 us with single elements loaded when needed, 618 us with them fetched ahead, 435 us in twos.)
template <typename T>
cudaError_t launch_type(NormParams& p, bool backward, bool layer, bool post, int gate, int device, cudaStream_t st, const Plan* bwd) {
  constexpr int V = 16 / sizeof(T);
  if (chunks_ok(p, V, 16)) return launch_v<T, V>(p, backward, layer, post, gate, device, st, bwd);
  if (chunks_ok(p, 2, 2 * sizeof(T))) return launch_v<T, 2>(p, backward, layer, post, gate, device, st, bwd);
  return launch_v<T, 1>(p, backward, layer, post, gate, device, st, bwd);
}

template <typename T>
cudaError_t launch_reduce(const NormParams& p, const Plan& pl, cudaStream_t st) {
  const bool weights = p.dpre_w || p.dpre_b || p.dpost_w || p.dpost_b;
  const bool gates = p.dgate != nullptr && pl.workers > 1;
  if (!weights && !gates) return cudaSuccess;
  const long long gate_rows = p.rows / p.per_gate;
  const int by_worker = gate_rows > pl.workers - 1;
  const long long items = !gates ? 0 : by_worker ? pl.workers - 1 : gate_rows;  // (at most 2 x 64 workers a multiprocessor: 18944 of 65531)
  host_count_launch();
  norm_reduce<T><<<dim3((p.width + 31) / 32, (unsigned)(4 + items)), 32 * SHARES, 0, st>>>(p, (int)pl.teams, by_worker);
  return cudaGetLastError();
}

}  // namespace normk
}  // namespace amsim

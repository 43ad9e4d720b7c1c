// The norms around a residual block, with the block's gate and residual scale:
//     u = N_post(block) or block,   r = x + scale * gate * u,   y = N_pre(r),
//     N(z) = (z - mean z) rstd w + b  (layer)   or   z rms(z)^-1 w  (rms),
// and the gradient
//     a = dy w_pre,  g = dr + rstd (a - [mean a] - hat mean(a hat)),  hat = (r - mean) rstd
//     dx = g,  du = scale gate g,  dgate = sum scale u g,  dblock = N_post'(du) in the same form,
//     dw = sum dy hat, db = sum dy (and the same of du for N_post).
// Both are bound by memory: the forward pass reads x and block and writes y (and r where it is wanted); the backward pass
// reads dy, dr, x and block, from which it makes r and hat again, unrounded (taken from a stored bf16 r, the gradients of the FP32 weights
// were 1.6e-3 off), and writes dx and dblock.  A row stays in registers from its one read to its one write: `tpr` threads
// (a power of two from 4 to 512) hold E elements each; rows wider than a CTA's share go to a cluster of 2, 4 or 8 CTAs
// that add their row sums through distributed shared memory.  What a thread will need of its next rows is already on
// its way to a place of its own in shared memory (cp.async, no barrier), since the chain of two or four row sums per row
// leaves the memory idle otherwise.  Means, variances and every sum are FP32; the variance is taken around the mean in a
// second pass over the registers; r is rounded once, and y is computed from the sum before that rounding.
//
// Column sums (weights, biases, gate) are kept in registers over the consecutive rows of a worker, then added over the
// workers in a fixed order by norm_reduce: the same bits on every run, no atomics.  A gate of one row per group of rows is
// handed over whenever a worker leaves a group: directly if the whole group was its own, else through one of its two slots.
#include "amsim_elem.cuh"
#include "amsim_host.h"

namespace amsim {
namespace normk {

constexpr int MAX_THREADS = 512;

struct NormParams {
  const void *x, *block, *gate, *post_w, *post_b, *pre_w, *pre_b;
  void *sum, *y;
  float* stats;              // rows x 4: mean and 1 / deviation of N_post, then of N_pre
  const void *dsum, *dy;     // backward
  int n_in;                  // tensors fetched ahead, and the places of x, block, dy, dsum among them
  int in_x, in_block, in_dy, in_dsum;
  void *dx, *dblock, *dgate, *dpost_w, *dpost_b, *dpre_w, *dpre_b;
  float *part, *gate_part;   // column sums: [workers][arrays][width], [workers][2][width]
  long long rows, per_gate;  // rows that share a row of the gate
  long long per_worker;      // rows of a worker (backward)
  long long workers;
  int width, tpr, tpr_log, cluster;
  int w_type, gate_type;
  float scale, eps, inv_width;
  int post, pre;
};

// Sums over the threads of a row.  Two buffers per sum: a warp that runs ahead writes the other one, and cannot come back to
// the first before everybody has passed the barrier between.
struct RowSum {
  float* red;     // [2][2][16] partial sums of the CTA's warps
  float* peers;   // [2][2][8] partial sums of the cluster's CTAs
  int tpr, cluster, rank, buf;

  __device__ __forceinline__ void operator()(float& a, float& b, bool both) {
    const int lanes = tpr < 32 ? tpr : 32;
    for (int o = lanes >> 1; o; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      if (both) b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (tpr <= 32) return;
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
      red[buf * 32 + w] = a;
      if (both) red[buf * 32 + 16 + w] = b;
    }
    __syncthreads();
    a = 0.f;
    b = 0.f;
    for (int i = 0; i < (tpr >> 5); ++i) {
      a += red[buf * 32 + i];
      if (both) b += red[buf * 32 + 16 + i];
    }
    if (cluster > 1) {
      if (threadIdx.x < cluster) {
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(peers + buf * 16 + rank);
        asm volatile("{.reg .b32 r; mapa.shared::cluster.u32 r, %0, %1; st.shared::cluster.f32 [r], %2; st.shared::cluster.f32 [r + 32], %3;}" ::"r"(at),
                     "r"(threadIdx.x), "f"(a), "f"(b) : "memory");
      }
      asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
      a = 0.f;
      b = 0.f;
      for (int i = 0; i < cluster; ++i) {
        a += peers[buf * 16 + i];
        b += peers[buf * 16 + 8 + i];
      }
    }
    buf ^= 1;
  }
};

// Where a thread's elements are: chunk c holds columns at(c) .. at(c) + V - 1.
template <int V>
struct Cols {
  int first, step, width;
  __device__ __forceinline__ int at(int c) const { return first + c * step; }
  __device__ __forceinline__ bool ok(int c) const { return at(c) < width; }
};

// Rows fetched ahead of their use, each thread its own 16-byte chunks: stage, tensor, chunk.  Without 16-byte chunks (V = 1) elements are
// loaded when they are needed.
template <typename T, int V, int N>
struct Ahead {
  static constexpr int STAGES = sizeof(T) == 4 ? 2 : 3;
  uint32_t base;
  int n_in, stage;
  __device__ __forceinline__ Ahead(const NormParams& p, void* smem) : n_in(p.n_in), stage(0) {
    base = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16;
  }
  __device__ __forceinline__ uint32_t place(int st, int k, int c) const { return base + ((st * n_in + k) * N + c) * (blockDim.x * 16); }
  // tensor number k of row `at` into the stage that is `ahead` uses away
  __device__ __forceinline__ void fetch(int ahead, int k, const void* src, long long at, bool live, const Cols<V>& cols) const {
    if (V == 1 || !src || !live) return;
    const int st = stage + ahead >= STAGES ? stage + ahead - STAGES : stage + ahead;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (cols.ok(c))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place(st, k, c)), "l"(static_cast<const T*>(src) + at + cols.at(c)) : "memory");
  }
  __device__ __forceinline__ void commit() const {
    if (V > 1) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void ready() const {
    if (V > 1) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
  }
  __device__ __forceinline__ void next() { stage = stage + 1 == STAGES ? 0 : stage + 1; }
  __device__ __forceinline__ void read(int k, int c, const void* src, long long at, const Cols<V>& cols, float (&o)[V]) const {
    if constexpr (V == 1) {
      load_vec<T, 1>(src, at + cols.at(c), o);
    } else {
      uint32_t w[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(place(stage, k, c)) : "memory");
      unpack16<T, V>(w, o);
    }
  }
};

template <bool LAYER, int N, int V>
__device__ __forceinline__ void row_stats(const float (&z)[N][V], const Cols<V>& cols, const NormParams& p, RowSum& sum, float& mean, float& rstd) {
  float s = 0.f, none = 0.f;
  mean = 0.f;
  if (LAYER) {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) s += z[c][e];  // (columns past the end hold zeros)
    sum(s, none, false);
    mean = s * p.inv_width;
  }
  s = 0.f;
#pragma unroll
  for (int c = 0; c < N; ++c)
    if (cols.ok(c)) {
#pragma unroll
      for (int e = 0; e < V; ++e) s += (z[c][e] - mean) * (z[c][e] - mean);
    }
  sum(s, none, false);
  rstd = 1.f / sqrtf(s * p.inv_width + p.eps);
}

template <bool LAYER, int N, int V>
__device__ __forceinline__ void affine(float (&z)[N][V], const Cols<V>& cols, const void* w, const void* b, int type16, bool f32, float mean, float rstd) {
#pragma unroll
  for (int c = 0; c < N; ++c) {
    if (!cols.ok(c)) continue;
    float wv[V], bv[V];
    if (w) load_param<V>(w, cols.at(c), f32, type16, wv);
    if (LAYER && b) load_param<V>(b, cols.at(c), f32, type16, bv);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float h = LAYER ? (z[c][e] - mean) * rstd : z[c][e] * rstd;
      if (w) h *= wv[e];
      if (LAYER && b) h += bv[e];
      z[c][e] = h;
    }
  }
}

template <typename T, int V, bool LAYER, int E>
__global__ void __launch_bounds__(MAX_THREADS) norm_fwd(const __grid_constant__ NormParams p) {
  constexpr int N = E / V;
  __shared__ float red[64], peers[32];
  extern __shared__ __align__(16) uint8_t smem[];
  const int t = threadIdx.x & (p.tpr - 1), group = threadIdx.x >> p.tpr_log, groups = blockDim.x >> p.tpr_log;
  const int rank = blockIdx.x % p.cluster;
  RowSum sum{red, peers, p.tpr, p.cluster, rank, 0};
  const Cols<V> cols{(rank * N * p.tpr + t) * V, p.tpr * V, p.width};
  const long long step = (long long)(gridDim.x / p.cluster) * groups;
  Ahead<T, V, N> in(p, smem);
  constexpr int STAGES = Ahead<T, V, N>::STAGES;
  auto fetch = [&](int ahead, long long row) {
    in.fetch(ahead, p.in_x, p.x, row * p.width, row < p.rows, cols);
    in.fetch(ahead, p.in_block, p.block, row * p.width, row < p.rows, cols);
    in.commit();
  };
  const long long begin = (long long)(blockIdx.x / p.cluster) * groups;
  for (int i = 0; i < STAGES - 1; ++i) fetch(i, begin + group + i * step);
  for (long long base = begin; base < p.rows; base += step, in.next()) {  // (the same trips for all threads)
    const long long row = base + group;
    const bool live = row < p.rows;
    const long long at = row * p.width;
    float r[N][V], u[N][V];
    fetch(STAGES - 1, row + (STAGES - 1) * step);
    in.ready();
#pragma unroll
    for (int c = 0; c < N; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e) r[c][e] = u[c][e] = 0.f;
      if (live && cols.ok(c)) {
        in.read(p.in_x, c, p.x, at, cols, r[c]);
        if (p.block) in.read(p.in_block, c, p.block, at, cols, u[c]);
      }
    }
    if (p.block) {
      if (p.post) {
        float mean, rstd;
        row_stats<LAYER>(u, cols, p, sum, mean, rstd);
        affine<LAYER>(u, cols, p.post_w, p.post_b, type16<T>(), p.w_type == 0, mean, rstd);
        if (p.stats && live && t == 0 && rank == 0) *reinterpret_cast<float2*>(p.stats + row * 4) = make_float2(mean, rstd);
      }
      const long long gate_at = p.gate && live ? row / p.per_gate * p.width : 0;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if (!live || !cols.ok(c)) continue;
        float gv[V];
        if (p.gate) load_param<V>(p.gate, gate_at + cols.at(c), p.gate_type == 0, type16<T>(), gv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float b = p.gate ? u[c][e] * gv[e] : u[c][e];
          r[c][e] += p.scale * b;
        }
      }
    }
    if (p.sum && live) {
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (cols.ok(c)) store_vec<T, V>(p.sum, at + cols.at(c), r[c]);
    }
    if (p.pre) {
      float mean, rstd;
      row_stats<LAYER>(r, cols, p, sum, mean, rstd);
      affine<LAYER>(r, cols, p.pre_w, p.pre_b, type16<T>(), p.w_type == 0, mean, rstd);
      if (live) {
#pragma unroll
        for (int c = 0; c < N; ++c)
          if (cols.ok(c)) store_vec<T, V>(p.y, at + cols.at(c), r[c]);
        if (p.stats && t == 0 && rank == 0) *reinterpret_cast<float2*>(p.stats + row * 4 + 2) = make_float2(mean, rstd);
      }
    }
  }
}

// Adds one array of column sums over the row groups of a block and writes the block's line of partial sums.
template <int N, int V>
__device__ __forceinline__ void flush_block(float (&acc)[N][V], const Cols<V>& cols, float* line, float* buf, int t, int group, int groups, int tpr) {
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

template <typename T, int V, bool LAYER, bool POST, bool GATE, int E>
__global__ void __launch_bounds__(MAX_THREADS) norm_bwd(const __grid_constant__ NormParams p) {
  constexpr int N = E / V;
  __shared__ float red[64], peers[32], buf[128];
  extern __shared__ __align__(16) uint8_t smem[];
  const int t = threadIdx.x & (p.tpr - 1), group = threadIdx.x >> p.tpr_log, groups = blockDim.x >> p.tpr_log;
  const int rank = blockIdx.x % p.cluster;
  RowSum sum{red, peers, p.tpr, p.cluster, rank, 0};
  const Cols<V> cols{(rank * N * p.tpr + t) * V, p.tpr * V, p.width};
  const long long team = blockIdx.x / p.cluster, worker = team * groups + group;
  const long long first = min(worker * p.per_worker, p.rows), last = min(first + p.per_worker, p.rows);
  float dw[N][V], db[N][V], dpw[N][V], dpb[N][V], dg[N][V];
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[c][e] = db[c][e] = dpw[c][e] = dpb[c][e] = dg[c][e] = 0.f;
  Ahead<T, V, N> in(p, smem);
  constexpr int STAGES = Ahead<T, V, N>::STAGES;
  auto fetch = [&](int ahead, long long row) {
    const bool live = row < last;
    in.fetch(ahead, p.in_dy, p.dy, row * p.width, live, cols);
    in.fetch(ahead, p.in_x, p.x, row * p.width, live, cols);
    in.fetch(ahead, p.in_block, p.block, row * p.width, live, cols);
    in.fetch(ahead, p.in_dsum, p.dsum, row * p.width, live, cols);
    in.commit();
  };
  for (int i = 0; i < STAGES - 1; ++i) fetch(i, first + i);

  for (long long i = 0; i < p.per_worker; ++i, in.next()) {  // (the same trips for all threads)
    const long long row = first + i;
    const bool live = row < last;
    const long long at = row * p.width;
    float g[N][V], hat[N][V], u[N][V];
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) st = __ldg(reinterpret_cast<const float4*>(p.stats + row * 4));
    fetch(STAGES - 1, row + STAGES - 1);
    const long long gate_row = GATE && live ? row / p.per_gate : 0;
    in.ready();
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e) g[c][e] = hat[c][e] = u[c][e] = 0.f;
      if (!live || !cols.ok(c)) continue;
      // the sum again, as the forward pass had it before rounding
      if (p.block) {
        in.read(p.in_block, c, p.block, at, cols, u[c]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (POST) u[c][e] = LAYER ? (u[c][e] - st.x) * st.y : u[c][e] * st.y;
          hat[c][e] = u[c][e];
        }
        if (POST && p.post_w) {
          float wv[V];
          load_param<V>(p.post_w, cols.at(c), p.w_type == 0, type16<T>(), wv);
#pragma unroll
          for (int e = 0; e < V; ++e) hat[c][e] *= wv[e];
        }
        if (POST && LAYER && p.post_b) {
          float bv[V];
          load_param<V>(p.post_b, cols.at(c), p.w_type == 0, type16<T>(), bv);
#pragma unroll
          for (int e = 0; e < V; ++e) hat[c][e] += bv[e];
        }
        if (GATE) {
          float gv[V];
          load_param<V>(p.gate, gate_row * p.width + cols.at(c), p.gate_type == 0, type16<T>(), gv);
#pragma unroll
          for (int e = 0; e < V; ++e) hat[c][e] *= gv[e];
        }
      }
      if (p.dy) {
        float xv[V], wv[V];
        in.read(p.in_x, c, p.x, at, cols, xv);
        in.read(p.in_dy, c, p.dy, at, cols, g[c]);
        if (p.pre_w) load_param<V>(p.pre_w, cols.at(c), p.w_type == 0, type16<T>(), wv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float r = xv[e] + p.scale * hat[c][e];
          hat[c][e] = LAYER ? (r - st.z) * st.w : r * st.w;
          dw[c][e] += g[c][e] * hat[c][e];
          if (LAYER) db[c][e] += g[c][e];
          if (p.pre_w) g[c][e] *= wv[e];
          if (LAYER) s1 += g[c][e];
          s2 += g[c][e] * hat[c][e];
        }
      }
    }
    if (p.dy) {
      sum(s1, s2, true);
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
          in.read(p.in_dsum, c, p.dsum, at, cols, dr);
#pragma unroll
          for (int e = 0; e < V; ++e) g[c][e] += dr[e];
        }
        store_vec<T, V>(p.dx, at + cols.at(c), g[c]);
      }
    }
    if (!POST && !GATE) {
      if (p.dblock && live) {
#pragma unroll
        for (int c = 0; c < N; ++c)
          if (cols.ok(c)) {
            float d[V];
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = p.scale * g[c][e];
            store_vec<T, V>(p.dblock, at + cols.at(c), d);
          }
      }
      continue;
    }
    s1 = s2 = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (!live || !cols.ok(c)) continue;
      float wv[V], bv[V], gv[V];
      if (POST && p.post_w) load_param<V>(p.post_w, cols.at(c), p.w_type == 0, type16<T>(), wv);
      if (POST && GATE && LAYER && p.post_b) load_param<V>(p.post_b, cols.at(c), p.w_type == 0, type16<T>(), bv);
      if (GATE) load_param<V>(p.gate, gate_row * p.width + cols.at(c), p.gate_type == 0, type16<T>(), gv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = u[c][e], d = p.scale * g[c][e];
        if (GATE) {
          float v = h;
          if (POST && p.post_w) v *= wv[e];
          if (POST && LAYER && p.post_b) v += bv[e];
          dg[c][e] += v * d;
        }
        float du = GATE ? d * gv[e] : d;
        if (POST) {
          dpw[c][e] += du * h;
          if (LAYER) dpb[c][e] += du;
          if (p.post_w) du *= wv[e];
          if (LAYER) s1 += du;
          s2 += du * h;
        }
        g[c][e] = du;
      }
    }
    if (POST) {
      sum(s1, s2, true);
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
        if (cols.ok(c)) store_vec<T, V>(p.dblock, at + cols.at(c), g[c]);
    }
    if (GATE && live && p.dgate && (row + 1 == last || (row + 1) / p.per_gate != gate_row)) {
      const long long begin = gate_row * p.per_gate;
      const bool whole = begin >= first && begin + p.per_gate <= last;
      float* slot = p.gate_part + (worker * 2 + (begin < first ? 0 : 1)) * p.width;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if (!cols.ok(c)) continue;
        if (whole) {
          store_param<V>(p.dgate, gate_row * p.width + cols.at(c), p.gate_type == 0, type16<T>(), dg[c]);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) slot[cols.at(c) + e] = dg[c][e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) dg[c][e] = 0.f;
      }
    }
  }
  float* line = p.part + team * 4 * p.width;
  if (p.dpre_w) flush_block(dw, cols, line, buf, t, group, groups, p.tpr);
  if (LAYER && p.dpre_b) flush_block(db, cols, line + p.width, buf, t, group, groups, p.tpr);
  if (POST && p.dpost_w) flush_block(dpw, cols, line + 2 * p.width, buf, t, group, groups, p.tpr);
  if (POST && LAYER && p.dpost_b) flush_block(dpb, cols, line + 3 * p.width, buf, t, group, groups, p.tpr);
}

// blockIdx.y < 4: sums a weight's or bias's lines over the teams; then one block for each worker that takes over a group of the
// gate from the worker before it, where that group began: sums the group's slots.  32 columns x 32 consecutive shares.
template <typename T>
__global__ void __launch_bounds__(1024) norm_reduce(const __grid_constant__ NormParams p, int teams) {
  __shared__ float part[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), share = threadIdx.x >> 5;
  const bool ok = col < p.width;
  float s = 0.f;
  void* out = nullptr;
  long long out_at = col;
  bool f32 = p.w_type == 0;
  if (blockIdx.y < 4) {
    out = blockIdx.y == 0 ? p.dpre_w : blockIdx.y == 1 ? p.dpre_b : blockIdx.y == 2 ? p.dpost_w : p.dpost_b;
    if (!out) return;
    const int per = (teams + 31) / 32, end = min(teams, (share + 1) * per);
    const float* at = p.part + (long long)blockIdx.y * p.width + col;
#pragma unroll 8
    for (int i = share * per; i < end; ++i) s += ok ? __ldcg(at + (long long)i * 4 * p.width) : 0.f;
  } else {
    const long long w = (long long)blockIdx.y - 4 + 1;
    if (w >= p.workers) return;
    const long long row = w * p.per_worker;
    if (row >= p.rows || row % p.per_gate == 0) return;
    const long long g = row / p.per_gate, begin = g * p.per_gate;
    if (begin / p.per_worker != w - 1) return;
    const long long w1 = (begin + p.per_gate - 1) / p.per_worker, n = w1 - w + 2;  // slots: the second of w - 1, the first of w .. w1
    const long long per = (n + 31) / 32, end = min(n, (share + 1) * per);
#pragma unroll 4
    for (long long i = share * per; i < end; ++i) s += ok ? __ldcg(p.gate_part + ((w - 1 + i) * 2 + (i == 0 ? 1 : 0)) * p.width + col) : 0.f;
    out = p.dgate;
    out_at = g * p.width + col;
    f32 = p.gate_type == 0;
  }
  part[share][threadIdx.x & 31] = s;
  __syncthreads();
  if (share == 0 && ok) {
    float v[1] = {0.f};
    for (int i = 0; i < 32; ++i) v[0] += part[i][threadIdx.x & 31];
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
  int e, tpr, tpr_log, cluster, threads;
};

// Threads per row: enough for E elements each, at least 4; rows of up to 32 threads share CTAs of 128.
static bool shape_of(int width, int e, Shape* s) {
  s->e = e;
  s->cluster = 1;
  while ((long long)s->cluster * MAX_THREADS * e < width) s->cluster *= 2;
  if (s->cluster > 8) return false;
  s->tpr = 4;
  s->tpr_log = 2;
  while ((long long)s->tpr * e * s->cluster < width) s->tpr *= 2, ++s->tpr_log;
  s->threads = s->tpr > 128 ? s->tpr : 128;
  if (s->tpr > 32) s->threads = s->tpr;
  return true;
}

// Elements per thread.  Backward passes through N_post or a gate keep five arrays of column sums: 8 elements fit 128 registers;
// four FP32 tensors of 16 elements for 512 threads, two stages, do not fit shared memory.
template <typename T>
constexpr int bwd_elems(bool post, bool gate) { return post || gate || sizeof(T) == 4 ? 8 : 16; }
constexpr int FWD_ELEMS = 16;

struct Plan {
  Shape s;
  int groups;
  long long teams, workers, per_worker;
  size_t part_bytes, gate_bytes;
};

static bool bwd_plan(long long rows, int width, bool post, bool gate, int dtype, int device, Plan* pl) {
  if (!shape_of(width, dtype == 0 ? bwd_elems<float>(post, gate) : bwd_elems<__half>(post, gate), &pl->s)) return false;
  pl->groups = pl->s.threads / pl->s.tpr;
  // as many CTAs as stay resident (128 registers a thread), and at least four rows for a worker: each leaves a line of sums
  long long teams = (long long)host_sm_count(device) * (512 / pl->s.threads) / pl->s.cluster;
  const long long most = (rows + 4LL * pl->groups - 1) / (4LL * pl->groups);
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

static bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

static bool vector_ok(const NormParams& p, int v) {
  return p.width % v == 0 && aligned(p.x) && aligned(p.block) && aligned(p.gate) && aligned(p.post_w) && aligned(p.post_b) && aligned(p.pre_w) &&
         aligned(p.pre_b) && aligned(p.sum) && aligned(p.y) && aligned(p.dsum) && aligned(p.dy) && aligned(p.dx) && aligned(p.dblock) && aligned(p.dgate);
}

// The bytes of a CTA's fetched-ahead rows: `elems` elements a thread of each tensor.
template <typename T, int V>
static int ahead_bytes(const NormParams& p, int elems, int threads) {
  return V == 1 ? 0 : Ahead<T, V, 1>::STAGES * p.n_in * elems * (int)sizeof(T) * threads;
}

template <typename K>
static cudaError_t launch(K kernel, unsigned grid, int threads, int cluster, int smem, cudaStream_t st, const NormParams& p) {
  if (smem > 40 * 1024) {  // (48 KB with the static arrays; per device and kernel; a call that raises it again costs under a microsecond)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  host_count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int V>
static cudaError_t fwd_launch(const NormParams& p, bool layer, unsigned grid, const Shape& s, cudaStream_t st) {
  const int smem = ahead_bytes<T, V>(p, FWD_ELEMS, s.threads);
  return layer ? launch(norm_fwd<T, V, true, FWD_ELEMS>, grid, s.threads, s.cluster, smem, st, p)
               : launch(norm_fwd<T, V, false, FWD_ELEMS>, grid, s.threads, s.cluster, smem, st, p);
}

template <typename T, int V, bool LAYER>
static cudaError_t bwd_launch(const NormParams& p, bool post, bool gate, const Plan& pl, cudaStream_t st) {
  const unsigned grid = (unsigned)(pl.teams * pl.s.cluster);
  const int smem = ahead_bytes<T, V>(p, pl.s.e, pl.s.threads);
  if (post && gate) return launch(norm_bwd<T, V, LAYER, true, true, 8>, grid, pl.s.threads, pl.s.cluster, smem, st, p);
  if (post) return launch(norm_bwd<T, V, LAYER, true, false, 8>, grid, pl.s.threads, pl.s.cluster, smem, st, p);
  if (gate) return launch(norm_bwd<T, V, LAYER, false, true, 8>, grid, pl.s.threads, pl.s.cluster, smem, st, p);
  return launch(norm_bwd<T, V, LAYER, false, false, bwd_elems<T>(false, false)>, grid, pl.s.threads, pl.s.cluster, smem, st, p);
}

template <typename T>
static cudaError_t reduce_launch(const NormParams& p, const Plan& pl, cudaStream_t st) {
  const bool weights = p.dpre_w || p.dpre_b || p.dpost_w || p.dpost_b;
  const bool gates = p.dgate != nullptr && pl.workers > 1;
  if (!weights && !gates) return cudaSuccess;
  const long long items = gates ? pl.workers - 1 : 0;
  const dim3 grid((p.width + 31) / 32, (unsigned)(4 + items));  // (items: at most 4 x 32 workers a multiprocessor: 18944 of 65531)
  host_count_launch();
  norm_reduce<T><<<grid, 1024, 0, st>>>(p, (int)pl.teams);
  return cudaGetLastError();
}

static int check(long long rows, int width, const void* gate, long long gate_rows, int dtype, int w_dtype, int gate_dtype, unsigned flags) {
  if (flags & ~(AMSIM_NORM_RMS | AMSIM_NORM_POST | AMSIM_NORM_PRE)) return host_fail(AMSIM_ERR_INVALID, "residual norm: unknown flag bits 0x%x", flags);
  if (rows < 0 || width <= 0) return host_fail(AMSIM_ERR_INVALID, "residual norm: rows >= 0 and width > 0 expected");
  if (width > AMSIM_NORM_MAX_WIDTH) return host_fail(AMSIM_ERR_UNSUPPORTED, "residual norm: rows of at most %d elements", AMSIM_NORM_MAX_WIDTH);
  if (rows > (1ll << 40) / width) return host_fail(AMSIM_ERR_UNSUPPORTED, "residual norm: more than 2^40 elements");
  if (dtype < 0 || dtype > 2) return host_fail(AMSIM_ERR_INVALID, "residual norm: unknown type %d", dtype);
  if ((w_dtype != 0 && w_dtype != dtype) || (gate_dtype != 0 && gate_dtype != dtype))
    return host_fail(AMSIM_ERR_INVALID, "residual norm: weights and gate are float32 or have the activations' type");
  if (gate && (gate_rows <= 0 || (rows > 0 && rows % gate_rows != 0)))
    return host_fail(AMSIM_ERR_INVALID, "residual norm: %lld rows cannot share %lld rows of the gate evenly", rows, gate_rows);
  return AMSIM_OK;
}

}  // namespace normk
}  // namespace amsim

using namespace amsim;

extern "C" {

int amsim_residual_norm(void* stream, const void* x, const void* block, const void* gate, const void* post_w, const void* post_b,
                        const void* pre_w, const void* pre_b, void* sum, void* y, float* stats, long long rows, int width,
                        long long gate_rows, float scale, float eps, int dtype, int w_dtype, int gate_dtype, unsigned flags) {
  using namespace amsim::normk;
  if (const int rc = check(rows, width, gate, gate_rows, dtype, w_dtype, gate_dtype, flags)) return rc;
  const bool post = flags & AMSIM_NORM_POST, pre = flags & AMSIM_NORM_PRE, layer = !(flags & AMSIM_NORM_RMS);
  if (rows == 0) return AMSIM_OK;  // (empty tensors may have no address)
  if (!block && (post || gate)) return host_fail(AMSIM_ERR_INVALID, "residual norm: a norm after the block or a gate needs a block");
  if (!layer && (post_b || pre_b)) return host_fail(AMSIM_ERR_INVALID, "residual norm: rms norms have no bias");
  if (!(eps >= 0.f)) return host_fail(AMSIM_ERR_INVALID, "residual norm: eps >= 0 expected");
  if (!sum && !pre) return host_fail(AMSIM_ERR_INVALID, "residual norm: nothing to compute");
  if (!x || (pre && !y)) return host_fail(AMSIM_ERR_INVALID, "NULL tensor pointer");
  if (stats && !aligned(stats)) return host_fail(AMSIM_ERR_INVALID, "residual norm: stats must be 16-byte aligned");
  NormParams p = {};
  p.x = x; p.block = block; p.gate = gate; p.post_w = post_w; p.post_b = post_b; p.pre_w = pre_w; p.pre_b = pre_b;
  p.sum = sum; p.y = y; p.stats = stats;
  p.rows = rows; p.per_gate = gate ? rows / gate_rows : 1; p.width = width;
  p.w_type = w_dtype; p.gate_type = gate_dtype; p.scale = scale; p.eps = eps; p.inv_width = 1.f / (float)width;
  p.post = post; p.pre = pre;
  p.in_x = p.n_in++;
  if (block) p.in_block = p.n_in++;
  Shape s;
  if (!shape_of(width, FWD_ELEMS, &s)) return host_fail(AMSIM_ERR_UNSUPPORTED, "residual norm: width");
  p.tpr = s.tpr; p.tpr_log = s.tpr_log; p.cluster = s.cluster;
  const int groups = s.threads / s.tpr;
  long long teams = (rows + groups - 1) / groups;
  const long long most = (long long)host_sm_count(host_device()) * 32 / s.cluster;  // (more CTAs than stay resident: they balance the last rows)
  if (teams > most) teams = most;
  const unsigned grid = (unsigned)(teams * s.cluster);
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = vector_ok(p, dtype == 0 ? 4 : 8);
  cudaError_t e;
  if (dtype == 0) e = vec ? fwd_launch<float, 4>(p, layer, grid, s, st) : fwd_launch<float, 1>(p, layer, grid, s, st);
  else if (dtype == 1) e = vec ? fwd_launch<__nv_bfloat16, 8>(p, layer, grid, s, st) : fwd_launch<__nv_bfloat16, 1>(p, layer, grid, s, st);
  else e = vec ? fwd_launch<__half, 8>(p, layer, grid, s, st) : fwd_launch<__half, 1>(p, layer, grid, s, st);
  AMSIM_HOST_TRY(e);
  return AMSIM_OK;
}

size_t amsim_residual_norm_grad_workspace(long long rows, int width, int has_gate, int dtype, unsigned flags) {
  using namespace amsim::normk;
  Plan pl;
  if (rows <= 0 || width <= 0 || width > AMSIM_NORM_MAX_WIDTH) return 0;
  if (!bwd_plan(rows, width, flags & AMSIM_NORM_POST, has_gate != 0, dtype, host_device(), &pl)) return 0;
  return pl.part_bytes + pl.gate_bytes;
}

int amsim_residual_norm_grad(void* stream, const void* dsum, const void* dy, const void* x, const void* block, const void* gate,
                             const void* post_w, const void* post_b, const void* pre_w, const float* stats, void* dx, void* dblock,
                             void* dgate, void* dpost_w, void* dpost_b, void* dpre_w, void* dpre_b, long long rows, int width,
                             long long gate_rows, float scale, int dtype, int w_dtype, int gate_dtype, void* workspace,
                             size_t workspace_bytes, unsigned flags) {
  using namespace amsim::normk;
  if (const int rc = check(rows, width, gate, gate_rows, dtype, w_dtype, gate_dtype, flags)) return rc;
  const bool post = flags & AMSIM_NORM_POST, pre = flags & AMSIM_NORM_PRE, layer = !(flags & AMSIM_NORM_RMS);
  if (!layer && (post_b || dpost_b || dpre_b)) return host_fail(AMSIM_ERR_INVALID, "residual norm: rms norms have no bias");
  if (dgate && !gate) return host_fail(AMSIM_ERR_INVALID, "residual norm: no gate");
  if (!pre && (dpre_w || dpre_b || dy)) return host_fail(AMSIM_ERR_INVALID, "residual norm: no norm before the next block");
  if (!post && (dpost_w || dpost_b)) return host_fail(AMSIM_ERR_INVALID, "residual norm: no norm after the block");
  NormParams p = {};
  p.block = block; p.gate = gate; p.post_w = post_w; p.post_b = post_b; p.pre_w = pre_w;
  p.x = x; p.stats = const_cast<float*>(stats); p.dsum = dsum; p.dy = dy;
  p.dx = dx; p.dblock = dblock; p.dgate = dgate; p.dpost_w = dpost_w; p.dpost_b = dpost_b; p.dpre_w = dpre_w; p.dpre_b = dpre_b;
  p.rows = rows; p.per_gate = gate ? rows / gate_rows : 1; p.width = width;
  p.w_type = w_dtype; p.gate_type = gate_dtype; p.scale = scale; p.inv_width = 1.f / (float)width;
  p.post = post; p.pre = pre;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    const dim3 grid((width + 255) / 256, 4);
    host_count_launch();
    if (dtype == 0) norm_zero<float><<<grid, 256, 0, st>>>(p);
    else if (dtype == 1) norm_zero<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
    else norm_zero<__half><<<grid, 256, 0, st>>>(p);
    AMSIM_HOST_TRY(cudaGetLastError());
    if (dgate) AMSIM_HOST_TRY(cudaMemsetAsync(dgate, 0, (size_t)gate_rows * width * (gate_dtype == 0 ? 4 : 2), st));
    return AMSIM_OK;
  }
  if (!dsum && !dy) return host_fail(AMSIM_ERR_INVALID, "residual norm: no output gradient");
  if (!dx || !stats || (dy && !x) || ((post || gate) && !block)) return host_fail(AMSIM_ERR_INVALID, "NULL tensor pointer");
  if (!aligned(stats)) return host_fail(AMSIM_ERR_INVALID, "residual norm: stats must be 16-byte aligned");
  Plan pl;
  if (!bwd_plan(rows, width, post, gate != nullptr, dtype, host_device(), &pl)) return host_fail(AMSIM_ERR_UNSUPPORTED, "residual norm: width");
  const size_t need = pl.part_bytes + pl.gate_bytes;
  if (!workspace || workspace_bytes < need)
    return host_fail(AMSIM_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned(workspace)) return host_fail(AMSIM_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  p.part = static_cast<float*>(workspace);
  p.gate_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.part_bytes);
  p.per_worker = pl.per_worker; p.workers = pl.workers;
  p.tpr = pl.s.tpr; p.tpr_log = pl.s.tpr_log; p.cluster = pl.s.cluster;
  if (dy) p.in_dy = p.n_in++, p.in_x = p.n_in++;
  else p.x = nullptr;  // (without a gradient through N_pre neither x nor the sum is needed)
  if (!dy && !post && !gate) p.block = nullptr;
  if (p.block) p.in_block = p.n_in++;
  if (dsum) p.in_dsum = p.n_in++;
  const bool vec = vector_ok(p, dtype == 0 ? 4 : 8);
  cudaError_t e;
#define AMSIM_BWD(T, V) (layer ? bwd_launch<T, V, true>(p, post, gate != nullptr, pl, st) : bwd_launch<T, V, false>(p, post, gate != nullptr, pl, st))
  if (dtype == 0) e = vec ? AMSIM_BWD(float, 4) : AMSIM_BWD(float, 1);
  else if (dtype == 1) e = vec ? AMSIM_BWD(__nv_bfloat16, 8) : AMSIM_BWD(__nv_bfloat16, 1);
  else e = vec ? AMSIM_BWD(__half, 8) : AMSIM_BWD(__half, 1);
#undef AMSIM_BWD
  AMSIM_HOST_TRY(e);
  e = dtype == 0 ? reduce_launch<float>(p, pl, st) : dtype == 1 ? reduce_launch<__nv_bfloat16>(p, pl, st) : reduce_launch<__half>(p, pl, st);
  AMSIM_HOST_TRY(e);
  return AMSIM_OK;
}

}  // extern "C"

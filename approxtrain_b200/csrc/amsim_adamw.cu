// One AdamW step over many tensors:
//     p <- p (1 - lr decay),   m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,
//     p <- p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps),
// with both moments in FP32, or in 8 bits: blocks of 256 elements in E4M3 codes with an FP32 scale (largest value at 448), v as its
// square root, which has half the exponent range.
//
// Rounding of the 8-bit moments.  v moves by (1 - b2) of itself a step, far below the 6 % between two codes: rounded to nearest, a
// moment would stay where it is.  So both are rounded up with the probability of the rest (the average over steps is exact),
// with 16 random bits each from a 32-bit hash of (seed, step, place): MurmurHash3's finaliser (A. Appleby, public domain),
// twice for the key.  A root that is not zero never becomes zero: m / (0 + eps) would throw the parameter away.
// Moments of a block whose largest is below 2^-100 are zero (the reciprocal of the scale has to be finite).
//
// Bound by memory: 28 bytes a parameter with FP32 moments, 16 with 8 bits.  The step reads its tensors from a table in the
// kernel's parameters, so nothing is kept between calls; the step number is on the device (a replayed graph counts on),
// read by every CTA and advanced by the last one to end.  1 - b^t is taken in 64 bits, by squaring.
#include <stdint.h>

#include "amsim_elem.cuh"
#include "amsim_host.h"

namespace amsim {
namespace adamwk {

constexpr int THREADS = 256;
constexpr int CHUNK = 4096;     // elements a CTA takes at a time: twice 8 a thread, or two blocks of 256 a warp
constexpr int BLOCK = 256;

struct Entry {
  void* p;
  const void* g;
  long long n, at;              // elements; first element in the moments
  float decay;
};

struct Common {
  void *m, *v;
  float *m_scale, *v_scale;
  long long* step;              // [0] steps taken, [1] CTAs that have ended (as unsigned)
  const float *lr_dev, *g_scale_dev;
  double lr, b1, b2, g_scale;
  float eps;
  uint32_t seed;
  int count, advance;
  long long units;              // chunks of 4096 elements, or blocks of 256 (8 bits)
};

template <int CAP>
struct Table {
  Common c;
  Entry e[CAP];
  int first[CAP];               // unit where a tensor begins
};

struct Rates {  // FP32 factors of a step
  float lr, b1, c1, b2, c2, inv_root2, step, g_scale, eps;
  uint32_t key;
};

__device__ __forceinline__ uint32_t mix(uint32_t h) {
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  return h ^ (h >> 16);
}

__device__ __forceinline__ double power(double b, unsigned long long t) {
  double r = 1.0;
  for (; t; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}

// The moments of gradient g.  Every product and sum is rounded (no fused ones), so that 8-bit codes do not depend on the
// compiler's choices: a moment next to the place where rounding turns is then the same in any FP32 program.
__device__ __forceinline__ void moments(float g, float& m, float& v, const Rates& r) {
  g = __fmul_rn(g, r.g_scale);
  m = __fadd_rn(__fmul_rn(r.b1, m), __fmul_rn(r.c1, g));
  v = __fadd_rn(__fmul_rn(r.b2, v), __fmul_rn(r.c2, __fmul_rn(g, g)));
}
// The parameter's update from the new moments; keep = 1 - lr decay.  (The approximate quotient is good to two steps of
// FP32 of an update that is itself about lr.)
__device__ __forceinline__ float update(float p, float m, float root, float keep, const Rates& r) {
  return p * keep - r.step * __fdividef(m, root * r.inv_root2 + r.eps);
}

template <typename T>
__device__ __forceinline__ float load1(const void* base, long long i) { return elem_to_float(static_cast<const T*>(base)[i]); }
template <typename T>
__device__ __forceinline__ void store1(void* base, long long i, float v) { static_cast<T*>(base)[i] = elem_from_float<T>(v); }

// FP32 moments: 8 elements of a thread at a time, twice four adjacent ones (VEC), or each beside its neighbour thread's.  (8 at
// 80 registers, 52 to 60 bytes of them spilled, keep 96 KB of a multiprocessor in flight.)
template <typename TP, typename TG, bool VEC>
__device__ __forceinline__ void half_chunk32(const Entry& e, const Common& c, long long base, const Rates& r) {
  float* const m_at = static_cast<float*>(c.m) + e.at;
  float* const v_at = static_cast<float*>(c.v) + e.at;
  const bool full = base + CHUNK / 2 <= e.n;
  const float keep = 1.f - r.lr * e.decay;
  if (VEC) {
    float p[2][4], g[2][4], m[2][4], v[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long long i = base + (k * THREADS + threadIdx.x) * 4;
      if (full || i + 4 <= e.n) {
        load_vec<TP, 4>(e.p, i, p[k]);
        load_vec<TG, 4>(e.g, i, g[k]);
        load_vec<float, 4>(m_at, i, m[k]);
        load_vec<float, 4>(v_at, i, v[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long long i = base + (k * THREADS + threadIdx.x) * 4;
      if (full || i + 4 <= e.n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          moments(g[k][j], m[k][j], v[k][j], r);
          p[k][j] = update(p[k][j], m[k][j], sqrtf(v[k][j]), keep, r);
        }
        store_vec<TP, 4>(e.p, i, p[k]);
        store_vec<float, 4>(m_at, i, m[k]);
        store_vec<float, 4>(v_at, i, v[k]);
      } else {
        for (long long j = i; j < e.n && j < i + 4; ++j) {
          float m1 = m_at[j], v1 = v_at[j];
          moments(load1<TG>(e.g, j), m1, v1, r);
          store1<TP>(e.p, j, update(load1<TP>(e.p, j), m1, sqrtf(v1), keep, r));
          m_at[j] = m1;
          v_at[j] = v1;
        }
      }
    }
  } else {
    float p[8], g[8], m[8], v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long i = base + k * THREADS + threadIdx.x;
      if (full || i < e.n) {
        p[k] = load1<TP>(e.p, i);
        g[k] = load1<TG>(e.g, i);
        m[k] = m_at[i];
        v[k] = v_at[i];
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long i = base + k * THREADS + threadIdx.x;
      if (full || i < e.n) {
        moments(g[k], m[k], v[k], r);
        store1<TP>(e.p, i, update(p[k], m[k], sqrtf(v[k]), keep, r));
        m_at[i] = m[k];
        v_at[i] = v[k];
      }
    }
  }
}

// The code of |a| / scale in the top byte (below it garbage), rounded up where the bits below the code's and 16 random ones carry.
// Times 2^-120 an E4M3 value's FP32 pattern begins with its code, values below 2^-6 (E4M3's subnormal ones) among FP32's: no cases.
// A value that the clamp holds at 448 has no bits to carry.  random16: the random bits times 16, plus 8.
__device__ __forceinline__ uint32_t round8(float a, float inv, uint32_t random16, bool at_least) {
  const float q = fminf(fabsf(a) * inv, 448.f) * 0x1p-120f;
  uint32_t code = __float_as_uint(q) + random16;
  if (at_least) code = max(code, q > 0.f ? 1u << 20 : 0u);
  return code << 4;
}
__device__ __forceinline__ float2 unpack8(uint16_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
  __half2 h2;
  memcpy(&h2, &h, 4);
  return __half22float2(h2);
}

// Two FP32 operations in one instruction (each rounded as if alone).
struct Two {
  uint64_t v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two t;
  asm("mov.b64 %0, {%1, %2};" : "=l"(t.v) : "f"(a), "f"(b));
  return t;
}
__device__ __forceinline__ void apart(Two t, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t.v)); }
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two t;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.v) : "l"(a.v), "l"(b.v));
  return t;
}
// (the sums apart: as one instruction they ended up fused with the products, and single codes differed)
__device__ __forceinline__ void sum_apart(Two a, Two b, float& x, float& y) {
  float a0, a1, b0, b1;
  apart(a, a0, a1);
  apart(b, b0, b1);
  x = __fadd_rn(a0, b0);
  y = __fadd_rn(a1, b1);
}

// Where a lane's elements of a block are: four adjacent ones twice, 128 apart (vec), or one every 32.  The addresses walk from
// block to block; computed anew for each they were a fifth of the instructions.
struct Cursor {
  char *p, *m, *v;
  const char* g;
  long long left;       // elements of the tensor from this block on
  uint32_t place;       // of the block among the moments, folded to 32 bits (a block does not straddle 2^32)
  uint32_t scale;       // number of its scales: places are below 2^40
  float keep;           // 1 - lr decay
  bool vec;
};
struct Block {
  float p[8], g[8], ms, vs;
  uint32_t mc[2], vc[2];
};

// The low and high words of a block's place, as one.
__device__ __forceinline__ uint32_t fold(uint32_t block) { return block * BLOCK + (block >> 24) * 0x9E3779B1u; }

template <typename TP, typename TG>
__device__ __forceinline__ void point(Cursor& at, const Entry& e, const Common& c, long long base, float lr) {
  const int lane = threadIdx.x & 31;
  at.vec = ((((uintptr_t)e.p) | ((uintptr_t)e.g)) & 15) == 0;
  const int mine = at.vec ? 4 * lane : lane;
  const unsigned long long place = (unsigned long long)(e.at + base);
  at.p = static_cast<char*>(e.p) + (base + mine) * sizeof(TP);
  at.g = static_cast<const char*>(e.g) + (base + mine) * sizeof(TG);
  at.m = static_cast<char*>(c.m) + place + mine;
  at.v = static_cast<char*>(c.v) + place + mine;
  at.left = e.n - base;
  at.scale = (uint32_t)(place / BLOCK);
  at.place = fold(at.scale);
  at.keep = 1.f - lr * e.decay;
}
template <typename TP, typename TG>
__device__ __forceinline__ void walk(Cursor& at, int blocks) {
  at.p += blocks * BLOCK * sizeof(TP);
  at.g += blocks * BLOCK * sizeof(TG);
  at.m += blocks * BLOCK;
  at.v += blocks * BLOCK;
  at.left -= blocks * BLOCK;
  at.scale += blocks;
  at.place = fold(at.scale);
}

// Element number j of a lane: its distance from the lane's first one.
template <bool VEC>
__device__ __forceinline__ constexpr int elem_of(int j) { return VEC ? (j >> 2) * 128 + (j & 3) : j * 32; }

template <typename TP, typename TG, bool VEC>
__device__ __forceinline__ void load8(Block& b, const Cursor& at, const Common& c) {
  const int lane = threadIdx.x & 31, n = at.left < BLOCK ? (int)at.left - (VEC ? 4 * lane : lane) : BLOCK;  // (elements from the lane's first on)
  b.ms = c.m_scale[at.scale];
  b.vs = c.v_scale[at.scale];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (VEC) {
      b.mc[h] = *reinterpret_cast<const uint32_t*>(at.m + elem_of<VEC>(4 * h));
      b.vc[h] = *reinterpret_cast<const uint32_t*>(at.v + elem_of<VEC>(4 * h));
    } else {
      b.mc[h] = b.vc[h] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b.mc[h] |= (uint32_t)(uint8_t)at.m[elem_of<VEC>(4 * h + i)] << (8 * i);
        b.vc[h] |= (uint32_t)(uint8_t)at.v[elem_of<VEC>(4 * h + i)] << (8 * i);
      }
    }
    if (VEC && n == BLOCK) {
      load_vec<TP, 4>(at.p, elem_of<VEC>(4 * h), *reinterpret_cast<float(*)[4]>(b.p + 4 * h));
      load_vec<TG, 4>(at.g, elem_of<VEC>(4 * h), *reinterpret_cast<float(*)[4]>(b.g + 4 * h));
    } else {
#pragma unroll
      for (int j = 4 * h; j < 4 * h + 4; ++j) {
        const bool ok = n == BLOCK || elem_of<VEC>(j) < n;
        b.p[j] = ok ? load1<TP>(at.p, elem_of<VEC>(j)) : 0.f;
        b.g[j] = ok ? load1<TG>(at.g, elem_of<VEC>(j)) : 0.f;
      }
    }
  }
}

template <typename TP, bool VEC>
__device__ __forceinline__ void step8(const Block& in, const Cursor& at, const Common& c, const Rates& r) {
  const int lane = threadIdx.x & 31, n = at.left < BLOCK ? (int)at.left - (VEC ? 4 * lane : lane) : BLOCK;
  const Two b1 = two(r.b1, r.b1), c1 = two(r.c1, r.c1), b2 = two(r.b2, r.b2), c2 = two(r.c2, r.c2), gs = two(r.g_scale, r.g_scale), ms = two(in.ms, in.ms), vs = two(in.vs, in.vs);
  float p[8], m[8], root[8];
  uint32_t m_top = 0, v_top = 0;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 mv = unpack8((uint16_t)(in.mc[j >> 2] >> (8 * (j & 3)))), vv = unpack8((uint16_t)(in.vc[j >> 2] >> (8 * (j & 3))));
    // (as in moments(), two at a time)
    const Two g = mul(two(in.g[j], in.g[j + 1]), gs), old = mul(two(vv.x, vv.y), vs);
    float v[2];
    sum_apart(mul(b1, mul(two(mv.x, mv.y), ms)), mul(c1, g), m[j], m[j + 1]);
    sum_apart(mul(b2, mul(old, old)), mul(c2, mul(g, g)), v[0], v[1]);
#pragma unroll
    for (int i = j; i < j + 2; ++i) {
      root[i] = sqrtf(v[i - j]);
      p[i] = update(in.p[i], m[i], root[i], at.keep, r);
      m_top = max(m_top, __float_as_uint(m[i]) & 0x7FFFFFFFu);
      v_top = max(v_top, __float_as_uint(root[i]));
    }
  }
  const float mt = __uint_as_float(__reduce_max_sync(0xffffffffu, m_top)), vt = __uint_as_float(__reduce_max_sync(0xffffffffu, v_top));
  // (the scale as a product with 1 / 448 and its inverse as 448 times a reciprocal, each rounded)
  const float m_inv = mt >= 0x1p-100f ? __fmul_rn(448.f, __frcp_rn(mt)) : 0.f, v_inv = vt >= 0x1p-100f ? __fmul_rn(448.f, __frcp_rn(vt)) : 0.f;
  const uint32_t place = at.place + (VEC ? 4 * lane : lane);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = 4 * h + i;
      const uint32_t rnd = mix((place + elem_of<VEC>(j)) ^ r.key);
      a[i] = (round8(m[j], m_inv, ((rnd << 4) & 0xFFFF0u) | 8u, false) & 0x7FFFFFFFu) | (__float_as_uint(m[j]) & 0x80000000u);
      b[i] = round8(root[j], v_inv, ((rnd >> 12) & 0xFFFF0u) | 8u, true);
    }
    if (VEC) {
      *reinterpret_cast<uint32_t*>(at.m + elem_of<VEC>(4 * h)) = __byte_perm(__byte_perm(a[0], a[1], 0x0073), __byte_perm(a[2], a[3], 0x0073), 0x5410);
      *reinterpret_cast<uint32_t*>(at.v + elem_of<VEC>(4 * h)) = __byte_perm(__byte_perm(b[0], b[1], 0x0073), __byte_perm(b[2], b[3], 0x0073), 0x5410);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at.m[elem_of<VEC>(4 * h + i)] = (char)(a[i] >> 24);
        at.v[elem_of<VEC>(4 * h + i)] = (char)(b[i] >> 24);
      }
    }
    if (VEC && n == BLOCK) {
      store_vec<TP, 4>(at.p, elem_of<VEC>(4 * h), *reinterpret_cast<float(*)[4]>(p + 4 * h));
    } else {
#pragma unroll
      for (int j = 4 * h; j < 4 * h + 4; ++j)
        if (n == BLOCK || elem_of<VEC>(j) < n) store1<TP>(at.p, elem_of<VEC>(j), p[j]);
    }
  }
  if (lane == 0) {
    c.m_scale[at.scale] = mt < 0x1p-100f ? 0.f : __fmul_rn(mt, 1.f / 448.f);  // (not a number: neither are the block's moments)
    c.v_scale[at.scale] = vt < 0x1p-100f ? 0.f : __fmul_rn(vt, 1.f / 448.f);
  }
}

// The last tensor of the table that begins at or before `unit`.
template <int CAP>
__device__ __forceinline__ int find(const Table<CAP>& tab, long long unit) {
  int lo = 0, hi = tab.c.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid] <= unit) lo = mid;
    else hi = mid;
  }
  return lo;
}

// 56 million parameters in 244 tensors: FP32 moments 260 us (6.1 TB/s), 8 bits 207 us (4.4 TB/s), bound by the issue of
// instructions: 84 a parameter, 65 % of the issue slots, which 16 warps a multiprocessor (114 to 120 registers) do not fill.
template <typename TP, typename TG, int BITS, int CAP>
__global__ void __launch_bounds__(THREADS, BITS == 32 ? 3 : 2) adamw(const __grid_constant__ Table<CAP> tab) {
  __shared__ Rates rates;
  const Common& c = tab.c;
  if (threadIdx.x == 0) {
    const unsigned long long t = (unsigned long long)c.step[0] + 1;
    const double lr = c.lr_dev ? (double)*c.lr_dev : c.lr;
    Rates r;
    r.lr = (float)lr;
    r.b1 = (float)c.b1;
    r.c1 = (float)(1.0 - c.b1);
    r.b2 = (float)c.b2;
    r.c2 = (float)(1.0 - c.b2);
    r.step = (float)(lr / (1.0 - power(c.b1, t)));
    r.inv_root2 = (float)(1.0 / sqrt(1.0 - power(c.b2, t)));
    r.g_scale = (float)(c.g_scale_dev ? c.g_scale * *c.g_scale_dev : c.g_scale);
    r.eps = c.eps;
    r.key = mix(c.seed ^ mix((uint32_t)t));
    rates = r;
  }
  if constexpr (BITS == 32) {
    __syncthreads();
    const Rates r = rates;
    for (long long chunk = blockIdx.x; chunk < c.units; chunk += gridDim.x) {
      const int k = find(tab, chunk);
      const Entry& e = tab.e[k];
      const long long base = (chunk - tab.first[k]) * CHUNK;
      const bool vec = ((((uintptr_t)e.p) | ((uintptr_t)e.g) | (uintptr_t)(e.at * 4)) & 15) == 0;
#pragma unroll 1
      for (int h = 0; h < 2 && base + h * (CHUNK / 2) < e.n; ++h) {
        if (vec) half_chunk32<TP, TG, true>(e, c, base + h * (CHUNK / 2), r);
        else half_chunk32<TP, TG, false>(e, c, base + h * (CHUNK / 2), r);
      }
    }
  } else {
    // a CTA's blocks are consecutive, its warps take them in turn, and the next one is on its way while a warp works on one
    // (without that, 56 million parameters took 258 us instead of 226; what bounds it then is the issue of instructions)
    constexpr int WARPS = THREADS / 32;
    __syncthreads();
    const Rates r = rates;
    const long long begin = c.units * blockIdx.x / gridDim.x, end = c.units * (blockIdx.x + 1) / gridDim.x;
    long long unit = begin + (threadIdx.x >> 5);
    int k = find(tab, unit);
    long long next_first = k + 1 < c.count ? tab.first[k + 1] : c.units;  // where the next tensor begins
    Cursor at;
    point<TP, TG>(at, tab.e[k], c, (unit - tab.first[k]) * BLOCK, r.lr);
    Block next;
    auto load = [&]() {
      if (at.vec) load8<TP, TG, true>(next, at, c);
      else load8<TP, TG, false>(next, at, c);
    };
    if (unit < end) load();
    while (unit < end) {
      const Block now = next;
      const Cursor here = at;
      unit += WARPS;
      if (unit < end) {
        if (unit < next_first) {
          walk<TP, TG>(at, WARPS);
        } else {
          do ++k; while (k + 1 < c.count && tab.first[k + 1] <= unit);
          next_first = k + 1 < c.count ? tab.first[k + 1] : c.units;
          point<TP, TG>(at, tab.e[k], c, (unit - tab.first[k]) * BLOCK, r.lr);
        }
        load();
      }
      if (here.vec) step8<TP, true>(now, here, c, r);
      else step8<TP, false>(now, here, c, r);
    }
  }
  if (c.advance && threadIdx.x == 0) {
    __threadfence();
    if (atomicInc(reinterpret_cast<unsigned*>(c.step + 1), gridDim.x - 1) == gridDim.x - 1) c.step[0] += 1;  // (the counter is at zero again)
  }
}

struct Call {
  const void* const* params;
  const void* const* grads;
  const long long* sizes;
  const float* decay;
  int tensors;
  Common c;
};

// Launches over as many tensors as a table holds; the last one advances the step.
template <typename TP, typename TG, int BITS, int CAP>
static cudaError_t run(const Call& call, int device, cudaStream_t st) {
  Table<CAP> tab;
  tab.c = call.c;
  long long at = 0;
  int i = 0;
  do {
    tab.c.count = 0;
    constexpr int UNIT = BITS == 32 ? CHUNK : BLOCK;
    long long units = 0;
    while (i < call.tensors && tab.c.count < CAP) {
      const long long n = call.sizes[i];
      const long long more = (n + UNIT - 1) / UNIT;
      if (units + more >= (1ll << 31)) break;  // (a tensor has fewer than 2^31 units: see the size check)
      if (n > 0) {
        const int k = tab.c.count++;
        tab.e[k] = {const_cast<void*>(call.params[i]), call.grads[i], n, at, call.decay[i]};
        tab.first[k] = (int)units;
        units += more;
        at += BITS == 32 ? n : more * BLOCK;
      }
      ++i;
    }
    tab.c.units = units;
    tab.c.advance = i == call.tensors;
    const long long work = BITS == 32 ? units : (units + THREADS / 32 - 1) / (THREADS / 32);
    const long long most = (BITS == 32 ? 3LL : 2LL) * host_sm_count(device);  // (what stays resident)
    const unsigned grid = (unsigned)(work < 1 ? 1 : work < most ? work : most);
    host_count_launch();
    adamw<TP, TG, BITS, CAP><<<grid, THREADS, 0, st>>>(tab);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  } while (i < call.tensors);
  return cudaSuccess;
}

template <typename TP, typename TG>
static cudaError_t run_types(const Call& call, int bits, int device, cudaStream_t st) {
  const bool few = call.tensors <= 32;  // (a small table is copied to the device sooner)
  if (bits == 32) return few ? run<TP, TG, 32, 32>(call, device, st) : run<TP, TG, 32, 640>(call, device, st);
  return few ? run<TP, TG, 8, 32>(call, device, st) : run<TP, TG, 8, 640>(call, device, st);
}

}  // namespace adamwk
}  // namespace amsim

extern "C" int amsim_adamw(void* stream, int tensors, const void* const* params, const void* const* grads, const long long* sizes, const float* decay,
                           void* exp_avg, float* exp_avg_scale, void* exp_avg_sq, float* exp_avg_sq_scale, long long* step, double lr,
                           const float* lr_dev, double beta1, double beta2, double eps, double grad_scale, const float* grad_scale_dev,
                           unsigned seed, int dtype, int grad_dtype, int bits) {
  using namespace amsim;
  using namespace amsim::adamwk;
  if (tensors < 0) return host_fail(AMSIM_ERR_INVALID, "adamw: tensors >= 0 expected");
  if (bits != 32 && bits != 8) return host_fail(AMSIM_ERR_INVALID, "adamw: moments of 32 or 8 bits, got %d", bits);
  if (dtype < 0 || dtype > 2 || (grad_dtype != 0 && grad_dtype != dtype)) return host_fail(AMSIM_ERR_INVALID, "adamw: gradients are float32 or have the parameters' type");
  if (!(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0)) return host_fail(AMSIM_ERR_INVALID, "adamw: betas in [0, 1) and eps >= 0 expected");
  if (!step || (tensors && (!params || !grads || !sizes || !decay))) return host_fail(AMSIM_ERR_INVALID, "NULL argument");
  bool any = false;
  long long all = 0;
  for (int i = 0; i < tensors; ++i) {
    if (sizes[i] < 0 || sizes[i] >= (1ll << 38)) return host_fail(AMSIM_ERR_INVALID, "adamw: tensor %d has %lld elements", i, sizes[i]);
    if (sizes[i] && (!params[i] || !grads[i])) return host_fail(AMSIM_ERR_INVALID, "adamw: NULL tensor %d", i);
    any = any || sizes[i] > 0;
    all += (sizes[i] + BLOCK - 1) / BLOCK;
    if (all >= (1ll << 32)) return host_fail(AMSIM_ERR_UNSUPPORTED, "adamw: more than 2^40 elements");
  }
  if (any && (!exp_avg || !exp_avg_sq || (bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)))) return host_fail(AMSIM_ERR_INVALID, "NULL moment pointer");
  if ((((uintptr_t)exp_avg) | ((uintptr_t)exp_avg_sq)) & 15) return host_fail(AMSIM_ERR_INVALID, "adamw: moments must be 16-byte aligned");
  Call call = {params, grads, sizes, decay, tensors, {}};
  call.c.m = exp_avg; call.c.v = exp_avg_sq; call.c.m_scale = exp_avg_scale; call.c.v_scale = exp_avg_sq_scale; call.c.step = step;
  call.c.lr = lr; call.c.lr_dev = lr_dev; call.c.b1 = beta1; call.c.b2 = beta2; call.c.eps = (float)eps;
  call.c.g_scale = grad_scale; call.c.g_scale_dev = grad_scale_dev; call.c.seed = seed;
  cudaStream_t st = (cudaStream_t)stream;
  const int device = host_device();
  cudaError_t e;
  if (dtype == 0) e = run_types<float, float>(call, bits, device, st);
  else if (dtype == 1) e = grad_dtype ? run_types<__nv_bfloat16, __nv_bfloat16>(call, bits, device, st) : run_types<__nv_bfloat16, float>(call, bits, device, st);
  else e = grad_dtype ? run_types<__half, __half>(call, bits, device, st) : run_types<__half, float>(call, bits, device, st);
  AMSIM_HOST_TRY(e);
  return AMSIM_OK;
}

// Rotary positions: the pair (a, b) number i of a head at position p becomes
//     s (a cos t - b sin t,  b cos t + a sin t),   t = p f_i,
// with the pairs adjacent (interleaved) or half of the rotated part apart, the elements behind the rotated part as they are, and
// t negated for the gradient.  Queries and keys go through one launch: they share positions and angles.
//
// Bound by memory: one read and one write of each element.  Far positions need the angle to more than FP32 holds (at 10^6 an
// FP32 angle is off by 0.06): p f_i / 2 pi is taken in 64 bits, its whole turns dropped, and the rest of a turn goes through
// sincospif, whose argument is then exact to 2^-25 turns.  A CTA does that once per token and pair, for all heads of both
// tensors, into shared memory; its first elements are already on their way meanwhile.
#include "amsim_elem.cuh"
#include "amsim_host.h"

namespace amsim {
namespace rotary {

constexpr int THREADS = 256;
constexpr int UNROLL = 4;             // units of a thread in flight
constexpr int MAX_PAIRS = 4096;       // angles of a CTA: 32 KB

struct Div {  // n / d for n < 2^31 by a multiplication
  uint32_t mul, shift, d;
};
static Div make_div(uint32_t d) {
  uint32_t s = 0;
  while ((1u << s) < d) ++s;
  return {(uint32_t)((((1ull << 32) * ((1ull << s) - d)) / d) + 1), s, d};
}
__device__ __forceinline__ uint32_t quot(uint32_t n, const Div& v) { return (__umulhi(n, v.mul) + n) >> v.shift; }

struct Side {           // one tensor: its heads at x + b xb + s xs + h xh (elements), the last axis dense
  const void* x;
  void* out;
  long long xb, xs, xh, ob, os, oh;
};

struct Params {
  Side side[2];
  const void* positions;
  const double* freqs;
  long long pos_b, pos_s, tokens;
  Div seq, units, heads;               // units of a head; heads of both tensors
  int heads0, half, rot, n_rot;        // n_rot: units that are rotated, the rest are copied
  int tokens_per_cta, pos32, interleaved;
  float scale, sign;
};

template <typename T, int V>
struct Unit {
  float a[V], b[V];
};

template <typename T, int V>
__global__ void __launch_bounds__(THREADS) rotate(const __grid_constant__ Params p) {
  __shared__ float2 turn[MAX_PAIRS];
  const long long token0 = (long long)blockIdx.x * p.tokens_per_cta;
  const int tokens = (int)min((long long)p.tokens_per_cta, p.tokens - token0);
  const uint32_t all = (uint32_t)tokens * p.heads.d * p.units.d;

  struct Place {
    const T* x;
    T* out;
    int tok, unit;
  };
  // unit number i of the CTA: its head's first element in both tensors
  auto place = [&](uint32_t i) {
    const uint32_t head_all = quot(i, p.units), unit = i - head_all * p.units.d;
    const uint32_t tok = quot(head_all, p.heads);
    uint32_t head = head_all - tok * p.heads.d;
    const long long t = token0 + tok;
    const long long b = p.tokens < (1ll << 31) ? quot((uint32_t)t, p.seq) : t / p.seq.d;
    const long long s = t - b * p.seq.d;
    const int which = head >= (uint32_t)p.heads0;
    if (which) head -= p.heads0;
    const Side& d = p.side[which];
    return Place{static_cast<const T*>(d.x) + (b * d.xb + s * d.xs + head * d.xh), static_cast<T*>(d.out) + (b * d.ob + s * d.os + head * d.oh), (int)tok, (int)unit};
  };
  auto load = [&](const Place& at, Unit<T, V>& u) {
    if (at.unit < p.n_rot) {
      const int first = p.interleaved ? 2 * V * at.unit : V * at.unit;
      load_vec<T, V>(at.x, first, u.a);
      load_vec<T, V>(at.x, first + (p.interleaved ? V : p.half), u.b);
    } else {
      load_vec<T, V>(at.x, p.rot + V * (at.unit - p.n_rot), u.a);
    }
  };
  auto finish = [&](const Place& at, Unit<T, V>& u) {
    if (at.unit >= p.n_rot) {
      store_vec<T, V>(at.out, p.rot + V * (at.unit - p.n_rot), u.a);
      return;
    }
    const float2* cs = turn + at.tok * p.half + V * at.unit;
    if (p.interleaved) {  // a, b: 2 V adjacent elements, V pairs
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float& x = 2 * e < V ? u.a[(2 * e) % V] : u.b[(2 * e) % V];
        float& y = 2 * e + 1 < V ? u.a[(2 * e + 1) % V] : u.b[(2 * e + 1) % V];
        const float2 c = cs[e];
        const float r = x * c.x - y * c.y;
        y = y * c.x + x * c.y;
        x = r;
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 c = cs[e];
        const float r = u.a[e] * c.x - u.b[e] * c.y;
        u.b[e] = u.b[e] * c.x + u.a[e] * c.y;
        u.a[e] = r;
      }
    }
    const int first = p.interleaved ? 2 * V * at.unit : V * at.unit;
    store_vec<T, V>(at.out, first, u.a);
    store_vec<T, V>(at.out, first + (p.interleaved ? V : p.half), u.b);
  };

  Place at[UNROLL];
  Unit<T, V> u[UNROLL];
  uint32_t i0 = threadIdx.x;
  auto load_all = [&]() {
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      if (i0 + k * THREADS < all) {
        at[k] = place(i0 + k * THREADS);
        load(at[k], u[k]);
      }
  };
  load_all();
  for (int i = threadIdx.x; i < tokens * p.half; i += THREADS) {
    const int tok = i / p.half, pair = i - tok * p.half;
    const long long t = token0 + tok, b = t / p.seq.d, s = t - b * p.seq.d, where = b * p.pos_b + s * p.pos_s;
    const double pos = p.pos32 ? (double)static_cast<const int*>(p.positions)[where] : (double)static_cast<const long long*>(p.positions)[where];
    double turns = pos * (p.freqs[pair] * 0.15915494309189533577);  // 1 / 2 pi
    turns -= rint(turns);
    float sn, cs;
    sincospif((float)(2.0 * turns), &sn, &cs);
    turn[i] = make_float2(p.scale * cs, p.sign * (p.scale * sn));
  }
  __syncthreads();
  while (i0 < all) {
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      if (i0 + k * THREADS < all) finish(at[k], u[k]);
    i0 += UNROLL * THREADS;
    load_all();
  }
}

template <typename T>
static cudaError_t launch(const Params& p, bool vec, unsigned grid, cudaStream_t st) {
  host_count_launch();
  if (vec) rotate<T, 16 / sizeof(T)><<<grid, THREADS, 0, st>>>(p);
  else rotate<T, 1><<<grid, THREADS, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace rotary
}  // namespace amsim

extern "C" int amsim_rotary(void* stream, const void* x, void* out, int heads, const void* x2, void* out2, int heads2, const void* positions,
                            const double* freqs, long long batch, long long seq, int dim, int rotary_dim, const long long* strides,
                            float scale, int dtype, unsigned flags) {
  using namespace amsim;
  using namespace amsim::rotary;
  if (flags & ~(AMSIM_ROTARY_INTERLEAVED | AMSIM_ROTARY_INVERSE | AMSIM_ROTARY_POS32)) return host_fail(AMSIM_ERR_INVALID, "rotary: unknown flag bits 0x%x", flags);
  if (dtype < 0 || dtype > 2) return host_fail(AMSIM_ERR_INVALID, "rotary: unknown type %d", dtype);
  if (batch < 0 || seq < 0 || heads < 0 || heads2 < 0 || dim <= 0) return host_fail(AMSIM_ERR_INVALID, "rotary: sizes must not be negative");
  if (rotary_dim <= 0 || rotary_dim > dim || rotary_dim % 2) return host_fail(AMSIM_ERR_INVALID, "rotary: an even number of rotated elements in 2 .. %d expected, got %d", dim, rotary_dim);
  if (rotary_dim / 2 > MAX_PAIRS || heads > 65536 || heads2 > 65536 || dim > 65536) return host_fail(AMSIM_ERR_UNSUPPORTED, "rotary: more than %d rotated elements, or 65536 heads or elements", 2 * MAX_PAIRS);
  if (batch >= (1ll << 31) || seq >= (1ll << 31) || (batch && seq > (1ll << 40) / batch)) return host_fail(AMSIM_ERR_UNSUPPORTED, "rotary: more than 2^31 sequences or positions");
  if (batch * seq == 0 || heads + heads2 == 0) return AMSIM_OK;
  if (!positions || !freqs || !strides || (heads && (!x || !out)) || (heads2 && (!x2 || !out2))) return host_fail(AMSIM_ERR_INVALID, "NULL tensor pointer");
  Params p = {};
  const int per = dtype == 0 ? 4 : 8;
  const bool in_place = (!heads || x == out) && (!heads2 || x2 == out2);
  bool vec = rotary_dim / 2 % per == 0 && (in_place || (dim - rotary_dim) % per == 0);
  p.side[0] = {x, out, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5]};
  p.side[1] = {x2, out2, strides[6], strides[7], strides[8], strides[9], strides[10], strides[11]};
  for (int i = 0; i < 2; ++i) {
    if (!(i ? heads2 : heads)) continue;
    const Side& s = p.side[i];
    vec = vec && ((uintptr_t)s.x & 15) == 0 && ((uintptr_t)s.out & 15) == 0;
    for (const long long v : {s.xb, s.xs, s.xh, s.ob, s.os, s.oh}) vec = vec && v % per == 0;
    // an output over its own input is the same elements in the same places, or the rows of one thread would be read by another
    // after they are written
    if (s.x == s.out && (s.xb != s.ob || s.xs != s.os || s.xh != s.oh)) return host_fail(AMSIM_ERR_INVALID, "rotary: in place needs equal strides");
  }
  const int v = vec ? per : 1;
  p.positions = positions; p.freqs = freqs;
  p.pos_b = strides[12]; p.pos_s = strides[13];
  p.tokens = batch * seq;
  p.half = rotary_dim / 2; p.rot = rotary_dim; p.n_rot = p.half / v;
  const uint32_t units = p.n_rot + (in_place ? 0 : (dim - rotary_dim) / v);
  p.seq = make_div((uint32_t)seq); p.units = make_div(units); p.heads = make_div((uint32_t)(heads + heads2));
  p.heads0 = heads;
  p.interleaved = (flags & AMSIM_ROTARY_INTERLEAVED) != 0; p.pos32 = (flags & AMSIM_ROTARY_POS32) != 0;
  p.scale = scale; p.sign = flags & AMSIM_ROTARY_INVERSE ? -1.f : 1.f;
  // Tokens of a CTA: two rounds of units for every thread, as long as that leaves four CTAs a multiprocessor; their angles fit the table.
  const long long per_token = (long long)units * (heads + heads2);
  long long n = 2 * UNROLL * THREADS / per_token;
  n = n < MAX_PAIRS / p.half ? n : MAX_PAIRS / p.half;
  const long long spread = p.tokens / (4LL * host_sm_count(host_device()));
  n = n < spread ? n : spread;
  p.tokens_per_cta = (int)(n < 1 ? 1 : n);
  if (per_token >= (1ll << 31)) return host_fail(AMSIM_ERR_UNSUPPORTED, "rotary: more than 2^31 pieces in a token");
  const long long ctas = (p.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  if (ctas >= (1ll << 31)) return host_fail(AMSIM_ERR_UNSUPPORTED, "rotary: more than 2^31 tokens");
  cudaStream_t st = (cudaStream_t)stream;
  AMSIM_HOST_TRY(dtype == 0 ? launch<float>(p, vec, (unsigned)ctas, st) : dtype == 1 ? launch<__nv_bfloat16>(p, vec, (unsigned)ctas, st) : launch<__half>(p, vec, (unsigned)ctas, st));
  return AMSIM_OK;
}

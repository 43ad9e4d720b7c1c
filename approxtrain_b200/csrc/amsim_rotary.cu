// Rotary positions: the pair (a, b) number i of a head at position p becomes
//     s (a cos t - b sin t,  b cos t + a sin t),   t = p f_i,
// with the pairs adjacent (interleaved) or half of the rotated part apart, the elements behind the rotated part as they are, and
// t negated for the gradient.  Queries and keys go through one launch: they share positions and angles.
//
// Bound by memory: one read and one write of each element.  Far positions need the angle to more than FP32 holds (at 10^6 an
// FP32 angle is off by 0.06): p f_i / 2 pi is taken in 64 bits, its whole turns dropped, and the rest of a turn goes through
// sincospif, whose argument is then exact to 2^-25 turns.  A CTA does that once per token and pair, for all heads of both
// tensors, into shared memory.  A thread keeps its place within the head (a 16-byte chunk, or two that turn together)
// and walks over the heads of the CTA's tokens, so nothing is divided on the way and neighbours touch neighbouring chunks.
#include "amsim_elem.cuh"
#include "amsim_host.h"

namespace amsim {
namespace rotary {

constexpr int THREADS = 256;
constexpr int MAX_PAIRS = 4096;       // angles of a CTA: 32 KB
constexpr int MAX_TOKENS = 64;        // tokens of a CTA

struct Side {           // one tensor: its heads at x + b xb + s xs + h xh (elements), the last axis dense
  const void* x;
  void* out;
  long long xb, xs, xh, ob, os, oh;
};

struct Params {
  Side side[2];
  const void* positions;
  const double* freqs;
  long long pos_b, pos_s, tokens, seq;
  int heads, heads0;                   // of both tensors, of the first
  int half, rot, n_rot, units;         // chunks of a head that turn, and all of them
  int tokens_per_cta, pos32;
  float scale, sign;
};

// A chunk as it is loaded: 16 bytes, two elements, or one.
template <typename T, int V>
struct Chunk {
  using type = uint4;
  __device__ static __forceinline__ void unpack(const uint4& c, float (&o)[V]) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    unpack16<T, V>(w, o);
  }
};
template <>
struct Chunk<float, 2> {
  using type = float2;
  __device__ static __forceinline__ void unpack(const float2& c, float (&o)[2]) { o[0] = c.x; o[1] = c.y; }
};
template <typename T>
struct Chunk<T, 2> {
  using type = uint32_t;
  __device__ static __forceinline__ void unpack(const uint32_t& c, float (&o)[2]) {
    T pair[2];
    memcpy(pair, &c, 4);
    o[0] = elem_to_float(pair[0]);
    o[1] = elem_to_float(pair[1]);
  }
};
template <typename T>
struct Chunk<T, 1> {
  using type = T;
  __device__ static __forceinline__ void unpack(const T& c, float (&o)[1]) { o[0] = elem_to_float(c); }
};

// 32768 positions of 40 heads of 128 in bf16, half of each head turned: 122 us (5.5 TB/s); three CTAs of 80 registers a multiprocessor (two of
// 89: 141 us).  V elements a chunk.  HALF: a chunk of the first half turns with the one half behind it; else a chunk holds V / 2 pairs (V = 1: two
// adjacent elements).
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(THREADS, 3) rotate(const __grid_constant__ Params p) {
  constexpr bool TWO = HALF || V == 1;           // a turning chunk is two loads
  constexpr int PAIRS = TWO ? V : V / 2;         // pairs of a turning chunk
  constexpr int UNROLL = TWO ? 4 : 8;            // heads of a thread in flight
  using Raw = typename Chunk<T, V>::type;
  __shared__ __align__(16) float2 turn[MAX_PAIRS];
  __shared__ long long in_at[2][MAX_TOKENS], out_at[2][MAX_TOKENS];
  __shared__ double pos[MAX_TOKENS];
  const long long token0 = (long long)blockIdx.x * p.tokens_per_cta;
  const int tokens = (int)min((long long)p.tokens_per_cta, p.tokens - token0);
  for (int i = threadIdx.x; i < tokens; i += THREADS) {
    const long long t = token0 + i, b = t / p.seq, s = t - b * p.seq, where = b * p.pos_b + s * p.pos_s;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      in_at[k][i] = b * p.side[k].xb + s * p.side[k].xs;
      out_at[k][i] = b * p.side[k].ob + s * p.side[k].os;
    }
    pos[i] = p.pos32 ? (double)static_cast<const int*>(p.positions)[where] : (double)static_cast<const long long*>(p.positions)[where];
  }
  __syncthreads();

  const int wide = min(p.units, THREADS), lanes = THREADS / wide, lane = threadIdx.x / wide, rows = lane < lanes ? tokens * p.heads : 0;
  int unit = threadIdx.x - lane * wide, row = lane, tok = lane / p.heads, head = lane - tok * p.heads;
  bool turns = false;
  int first = 0, second = 0;
  auto begin_unit = [&]() {
    turns = unit < p.n_rot;
    first = !turns ? p.rot + V * (unit - p.n_rot) : HALF ? V * unit : 2 * PAIRS * unit;
    second = first + (HALF ? p.half : V);
  };
  begin_unit();
  Raw a[UNROLL], b[TWO ? UNROLL : 1];
  T* out[UNROLL];
  int of[UNROLL];
  auto load = [&]() {  // the next heads of this thread, as many as there are
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      if (row + k * lanes >= rows) break;
      const int which = head >= p.heads0, h = which ? head - p.heads0 : head;
      const Side& d = p.side[which];
      const T* const x = static_cast<const T*>(d.x) + (in_at[which][tok] + h * d.xh);
      out[k] = static_cast<T*>(d.out) + (out_at[which][tok] + h * d.oh);
      of[k] = tok;
      a[k] = *reinterpret_cast<const Raw*>(x + first);
      if (TWO && turns) b[TWO ? k : 0] = *reinterpret_cast<const Raw*>(x + second);
      for (head += lanes; head >= p.heads; head -= p.heads) ++tok;
    }
  };
  load();  // (on their way while the angles are made)
  for (int i = threadIdx.x; i < tokens * p.half; i += THREADS) {
    const int t = i / p.half, pair = i - t * p.half;
    double whole = pos[t] * (p.freqs[pair] * 0.15915494309189533577);  // turns: 1 / 2 pi
    whole -= rint(whole);
    float sn, cs;
    sincospif((float)(2.0 * whole), &sn, &cs);
    turn[i] = make_float2(p.scale * cs, p.sign * (p.scale * sn));
  }
  __syncthreads();
  while (row < rows) {
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      if (row + k * lanes >= rows) break;
      if (!turns) {
        *reinterpret_cast<Raw*>(out[k] + first) = a[k];
        continue;
      }
      float x[V], y[V];
      Chunk<T, V>::unpack(a[k], x);
      if (TWO) Chunk<T, V>::unpack(b[TWO ? k : 0], y);
      const float2* cs = turn + of[k] * p.half + PAIRS * unit;
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        const float2 c = cs[e];
        float& u = TWO ? x[e % V] : x[(2 * e) % V];
        float& v = TWO ? y[e % V] : x[(2 * e + 1) % V];
        const float r = u * c.x - v * c.y;
        v = v * c.x + u * c.y;
        u = r;
      }
      store_vec<T, V>(out[k], first, x);
      if (TWO) store_vec<T, V>(out[k], second, y);
    }
    row += UNROLL * lanes;
    if (row >= rows && unit + wide < p.units) {  // (heads of more chunks than the CTA has threads)
      unit += wide;
      row = lane;
      tok = lane / p.heads;
      head = lane - tok * p.heads;
      begin_unit();
    }
    load();
  }
}

template <typename T>
static cudaError_t launch(const Params& p, int v, bool half, unsigned grid, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  host_count_launch();
  if (v == V) half ? rotate<T, V, true><<<grid, THREADS, 0, st>>>(p) : rotate<T, V, false><<<grid, THREADS, 0, st>>>(p);
  else if (v == 2) half ? rotate<T, 2, true><<<grid, THREADS, 0, st>>>(p) : rotate<T, 2, false><<<grid, THREADS, 0, st>>>(p);
  else half ? rotate<T, 1, true><<<grid, THREADS, 0, st>>>(p) : rotate<T, 1, false><<<grid, THREADS, 0, st>>>(p);
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
  if (heads && heads2 && out == out2) return host_fail(AMSIM_ERR_INVALID, "rotary: both tensors have the same output");
  rotary::Params p = {};
  const bool in_place = (!heads || x == out) && (!heads2 || x2 == out2);
  const bool half = !(flags & AMSIM_ROTARY_INTERLEAVED);
  p.side[0] = {x, out, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5]};
  p.side[1] = {x2, out2, strides[6], strides[7], strides[8], strides[9], strides[10], strides[11]};
  for (int i = 0; i < 2; ++i) {
    const Side& s = p.side[i];
    // an output over its own input is the same elements in the same places, or the rows of one thread would be read by another
    // after they are written
    if ((i ? heads2 : heads) && s.x == s.out && (s.xb != s.ob || s.xs != s.os || s.xh != s.oh)) return host_fail(AMSIM_ERR_INVALID, "rotary: in place needs equal strides");
  }
  // Elements a chunk: 16 bytes, else two, else one: the largest that divides the turning part (HALF: its half), the rest, the strides
  // and the addresses.  (Heads of 128 with 6 turning, bf16, 31196 positions of 42 heads: 984 us one by one, forward and backward, 675 us in twos.)
  auto whole = [&](int v) {
    bool ok = (half ? rotary_dim / 2 : rotary_dim) % v == 0 && (in_place || (dim - rotary_dim) % v == 0);
    for (int i = 0; i < 2; ++i) {
      if (!(i ? heads2 : heads)) continue;
      const Side& s = p.side[i];
      ok = ok && ((uintptr_t)s.x | (uintptr_t)s.out) % (v * (dtype == 0 ? 4 : 2)) == 0;
      for (const long long st : {s.xb, s.xs, s.xh, s.ob, s.os, s.oh}) ok = ok && st % v == 0;
    }
    return ok;
  };
  const int wide = dtype == 0 ? 4 : 8, v = whole(wide) ? wide : whole(2) ? 2 : 1;
  p.positions = positions; p.freqs = freqs;
  p.pos_b = strides[12]; p.pos_s = strides[13];
  p.tokens = batch * seq; p.seq = seq;
  p.heads = heads + heads2; p.heads0 = heads;
  p.half = rotary_dim / 2; p.rot = rotary_dim;
  p.n_rot = half || v == 1 ? p.half / v : rotary_dim / v;
  p.units = p.n_rot + (in_place ? 0 : (dim - rotary_dim) / v);
  p.pos32 = (flags & AMSIM_ROTARY_POS32) != 0;
  p.scale = scale; p.sign = flags & AMSIM_ROTARY_INVERSE ? -1.f : 1.f;
  // Tokens of a CTA: 16 heads for every thread, as long as that leaves four CTAs a multiprocessor; their angles fit the table.
  const long long per_token = (long long)p.units * p.heads;
  long long n = 16 * THREADS / per_token;
  n = n < MAX_PAIRS / p.half ? n : MAX_PAIRS / p.half;
  n = n < MAX_TOKENS ? n : MAX_TOKENS;
  const long long spread = p.tokens / (4LL * host_sm_count(host_device()));
  n = n < spread ? n : spread;
  p.tokens_per_cta = (int)(n < 1 ? 1 : n);
  const long long ctas = (p.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  if (ctas >= (1ll << 31)) return host_fail(AMSIM_ERR_UNSUPPORTED, "rotary: more than 2^31 tokens");
  cudaStream_t st = (cudaStream_t)stream;
  AMSIM_HOST_TRY(dtype == 0 ? launch<float>(p, v, half, (unsigned)ctas, st) : dtype == 1 ? launch<__nv_bfloat16>(p, v, half, (unsigned)ctas, st) : launch<__half>(p, v, half, (unsigned)ctas, st));
  return AMSIM_OK;
}

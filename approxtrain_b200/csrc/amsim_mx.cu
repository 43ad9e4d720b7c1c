// Matrices in 4-bit floats with a scale per 32 elements along the reduction (the OCP microscaling format MXFP4: E2M1 elements, E8M0
// scales), and their products on the tensor cores.
//
// Quantisation of a block: the scale is 2^(floor(log2 max|x|) - 2), so the largest element lands in [4, 8) and elements beyond 6
// become 6; x / scale is exact and is rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even code.  A block
// with an infinity or a NaN has the NaN scale: all of it reads as NaN.
//
// Layout.  A product contracts the quantised axes of both operands, so a matrix is stored as `rows` x `k` with k the quantised axis,
// in tiles of 128 rows x 256 elements, 17 KB each: 128 bytes of codes a row, 16-byte chunk (= block) c of row r at chunk
// c ^ (r & 7), then two 512-byte groups of scales (128 elements each: row r's four at (r % 32) * 16 + (r / 32) * 4).  That is what
// the tensor core reads from shared memory, so a stage of the product is a few untiled bulk copies of whole tiles: no tensor
// maps, no bounds (k is padded with zero codes; rows beyond the last are whatever was there, and only make outputs that
// nobody writes).  A matrix can be quantised along either axis, or along both with one read: the backward products of a
// layer contract the other axis.
#include <stdint.h>

#include "amsim_elem.cuh"
#include "amsim_host.h"
#include "amsim_mx.cuh"

namespace amsim {
namespace mx {

// ---- quantisation ------------------------------------------------------------------------------
// A CTA takes 128 x 128 elements through shared memory as they are, all of them on their way at once (cp.async): with four
// 16-byte loads of a thread in flight 8192 x 2048 FP32 both ways took 31 us.  Blocks of 32 have 16 bytes to spare behind them, so that
// eight lanes reading 16 bytes of 2 rows x 4 blocks, and 32 lanes reading an element of 32 columns, touch every bank once.
constexpr int Q_THREADS = 256;
template <typename T>
struct Stage {
  static constexpr int BLOCK = 32 * sizeof(T) + 16, ROW = 4 * BLOCK, BYTES = 128 * ROW;
  __device__ static __forceinline__ int at(int r, int c) { return r * ROW + (c >> 5) * BLOCK + (c & 31) * (int)sizeof(T); }
};
// (back to floats: FP32 in rows of four blocks of 36 words)
constexpr int Q_BLOCK = 36, Q_ROW = 4 * Q_BLOCK, Q_ROW_T = Q_ROW + 4;
constexpr int Q_SMEM_T = 128 * Q_ROW_T * 4;

struct QuantParams {
  const void* x;
  uint8_t *along, *across;    // codes of the rows (blocks along the columns), of the columns; either may be null
  long long rows, cols;
  long long along_kt, across_kt;  // tiles along the reduction
  long long gx;                   // CTAs along the columns
  float* sums;                    // [row tile][cols]: sums of the columns' elements, or null
  int vec;
};

// The codes of 32 elements in order, element 0 in the low half of the first byte; returns the scale byte.
__device__ __forceinline__ uint32_t quantise_block(const float (&v)[32], uint4& codes) {
  float top = 0.f;  // (NaN if one of them is)
#pragma unroll
  for (int i = 0; i < 32; i += 2) asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(top), "f"(v[i]), "f"(v[i + 1]));
  const int e = (int)((__float_as_uint(top) >> 23) & 255u);
  if (e == 255) {
    codes = make_uint4(0, 0, 0, 0);
    return 255;
  }
  const int byte = max(e - 2, 0);
  const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = v[8 * i + j] * inv;
    asm("{.reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};}"
        : "=r"(w[i]) : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  }
  codes = make_uint4(w[0], w[1], w[2], w[3]);
  return (uint32_t)byte;
}

__device__ __forceinline__ uint8_t* tile_of(uint8_t* base, long long row_tile, long long kts, long long kt) { return base + (row_tile * kts + kt) * TILE_BYTES; }

// 8192 x 2048 FP32 both ways 20.7 us (85 MB, 4.1 TB/s), 8192 x 8192 bf16 along its rows 33.5 us (170 MB, 5.1 TB/s).
template <typename T>
__global__ void __launch_bounds__(Q_THREADS) quantise(const __grid_constant__ QuantParams p) {
  extern __shared__ __align__(16) uint8_t elems[];
  __shared__ __align__(16) uint8_t scales[2][512];
  constexpr int V = 16 / sizeof(T);
  using St = Stage<T>;
  const int t = threadIdx.x;
  const long long by = blockIdx.x / p.gx, bx = blockIdx.x - by * p.gx, r0 = by * 128, c0 = bx * 128;
  if (p.vec) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(elems);
    const T* const x = static_cast<const T*>(p.x);
#pragma unroll
    for (int i = t; i < 128 * 128 / V; i += Q_THREADS) {
      const int r = i / (128 / V), c = i % (128 / V) * V;
      const bool ok = r0 + r < p.rows && c0 + c < p.cols;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + St::at(r, c)), "l"(ok ? x + (r0 + r) * p.cols + c0 + c : x), "r"(ok ? 16 : 0) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
#pragma unroll 8
    for (int i = t; i < 128 * 128; i += Q_THREADS) {
      const int r = i >> 7, c = i & 127;
      *reinterpret_cast<T*>(elems + St::at(r, c)) = r0 + r < p.rows && c0 + c < p.cols ? static_cast<const T*>(p.x)[(r0 + r) * p.cols + c0 + c] : elem_from_float<T>(0.f);
    }
  }
  __syncthreads();
  if (p.along && r0 < p.rows) {
    uint8_t* const tile = tile_of(p.along, by, p.along_kt, bx >> 1);
#pragma unroll 1
    for (int i = t; i < 512; i += Q_THREADS) {
      const int r = i >> 2, b = i & 3;
      float v[32];
#pragma unroll
      for (int j = 0; j < 32 / V; ++j) {
        const uint4 f = *reinterpret_cast<const uint4*>(elems + St::at(r, 32 * b) + 16 * j);
        const uint32_t w[4] = {f.x, f.y, f.z, f.w};
        unpack16<T, V>(w, *reinterpret_cast<float(*)[V]>(v + V * j));
      }
      uint4 codes;
      scales[0][(r & 31) * 16 + (r >> 5) * 4 + b] = (uint8_t)quantise_block(v, codes);
      const int chunk = (int)(bx & 1) * 4 + b;
      *reinterpret_cast<uint4*>(tile + r * 128 + ((chunk ^ (r & 7)) << 4)) = codes;
    }
  }
  if (p.across && c0 < p.cols) {
    uint4 codes[2];
    float sum[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = t & 127, b = (t >> 7) + 2 * i;
      float v[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = elem_to_float(*reinterpret_cast<const T*>(elems + St::at(32 * b + j, c)));
      scales[1][(c & 31) * 16 + (c >> 5) * 4 + b] = (uint8_t)quantise_block(v, codes[i]);
      if (p.sums) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j & 3] += v[j];
        sum[i] = (s[0] + s[1]) + (s[2] + s[3]);
      }
    }
    __syncthreads();  // (all have read the elements: their place takes the codes, which leave in whole sectors)
    uint4* const out = reinterpret_cast<uint4*>(elems);
#pragma unroll
    for (int i = 0; i < 2; ++i) out[(t & 127) * 5 + (t >> 7) + 2 * i] = codes[i];
    float* const half_sum = reinterpret_cast<float*>(out + 128 * 5);
    if (p.sums && t >= 128) half_sum[t - 128] = sum[0] + sum[1];
    __syncthreads();
    if (p.sums && t < 128 && c0 + t < p.cols && r0 < p.rows) p.sums[by * p.cols + c0 + t] = (sum[0] + sum[1]) + half_sum[t];
    uint8_t* const tile = tile_of(p.across, bx, p.across_kt, by >> 1);
#pragma unroll
    for (int i = t; i < 512; i += Q_THREADS) {
      const int c = i >> 2, b = i & 3, chunk = (int)(by & 1) * 4 + b;
      *reinterpret_cast<uint4*>(tile + c * 128 + ((chunk ^ (c & 7)) << 4)) = out[c * 5 + b];
    }
  }
  __syncthreads();
  if (t < 64) {
    const int which = t >> 5;
    if (which == 0 ? p.along && r0 < p.rows : p.across && c0 < p.cols) {
      uint8_t* const tile = which == 0 ? tile_of(p.along, by, p.along_kt, bx >> 1) : tile_of(p.across, bx, p.across_kt, by >> 1);
      const int half = (int)(which == 0 ? bx & 1 : by & 1);
      reinterpret_cast<uint4*>(tile + CODE_BYTES + half * 512)[t & 31] = reinterpret_cast<const uint4*>(scales[which])[t & 31];
    }
  }
}

// Adds the row tiles' column sums: 32 columns x 16 consecutive shares of the tiles.
__global__ void __launch_bounds__(512) add_sums(const float* __restrict__ sums, float* __restrict__ out, long long cols, int tiles) {
  __shared__ float part[16][33];
  const long long col = (long long)blockIdx.x * 32 + (threadIdx.x & 31);
  const int share = threadIdx.x >> 5, per = (tiles + 15) / 16, end = min(tiles, (share + 1) * per);
  float s = 0.f;
  if (col < cols) {
#pragma unroll 8
    for (int i = share * per; i < end; ++i) s += __ldcg(sums + (long long)i * cols + col);
  }
  part[share][threadIdx.x & 31] = s;
  __syncthreads();
  if (share == 0 && col < cols) {
    float all = 0.f;
    for (int i = 0; i < 16; ++i) all += part[i][threadIdx.x & 31];
    out[col] = all;
  }
}

// ---- back to floats ----------------------------------------------------------------------------
struct DequantParams {
  const uint8_t* data;
  void* out;
  long long rows, k, kt, gx;
  int transposed, vec, pitch;
};

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == 255 ? __uint_as_float(0x7FFFFFFFu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// 8192 x 2048 to FP32, either way round: 15.6 us (76 MB, 4.9 TB/s).
template <typename T>
__global__ void __launch_bounds__(Q_THREADS) dequantise(const __grid_constant__ DequantParams p) {
  extern __shared__ __align__(16) float stage[];
  const int t = threadIdx.x;
  const long long by = blockIdx.x / p.gx, bx = blockIdx.x - by * p.gx;
  const uint8_t* const tile = p.data + (by * p.kt + (bx >> 1)) * TILE_BYTES;
  const int half = (int)(bx & 1);
#pragma unroll
  for (int i = t; i < 512; i += Q_THREADS) {
    const int r = i >> 2, b = i & 3, chunk = half * 4 + b;
    const uint4 codes = *reinterpret_cast<const uint4*>(tile + r * 128 + ((chunk ^ (r & 7)) << 4));
    const float s = scale_value(tile[CODE_BYTES + half * 512 + (r & 31) * 16 + (r >> 5) * 4 + b]);
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v[8];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint32_t pair;
        asm("{.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %1;\ncvt.rn.f16x2.e2m1x2 %0, a;}" : "=r"(pair) : "r"(w[j] >> (8 * h)));
        __half2 h2;
        memcpy(&h2, &pair, 4);
        const float2 f = __half22float2(h2);
        v[2 * h] = f.x * s;
        v[2 * h + 1] = f.y * s;
      }
      float* const at = stage + r * p.pitch + b * Q_BLOCK + 8 * j;
      *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(at + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
  __syncthreads();
  const long long r0 = by * 128, k0 = bx * 128;
  constexpr int V = 16 / sizeof(T);
  if (!p.transposed && p.vec) {
#pragma unroll 4
    for (int i = t; i < 128 * 128 / V; i += Q_THREADS) {
      const int r = i / (128 / V), c = i % (128 / V) * V;
      if (r0 + r >= p.rows || k0 + c >= p.k) continue;
      float v[V];
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(stage + r * Q_ROW + (c >> 5) * Q_BLOCK + (c & 31) + j);
        v[j] = f.x; v[j + 1] = f.y; v[j + 2] = f.z; v[j + 3] = f.w;
      }
      store_vec<T, V>(p.out, (r0 + r) * p.k + k0 + c, v);
    }
  } else if (!p.transposed) {
#pragma unroll 8
    for (int i = t; i < 128 * 128; i += Q_THREADS) {
      const int r = i >> 7, c = i & 127;
      if (r0 + r < p.rows && k0 + c < p.k) static_cast<T*>(p.out)[(r0 + r) * p.k + k0 + c] = elem_from_float<T>(stage[r * Q_ROW + (c >> 5) * Q_BLOCK + (c & 31)]);
    }
  } else {
    // out is [k][rows]: 32 stored rows beside each other, four elements of k from each (a row is 148 words here: eight lanes reading
    // 16 bytes of eight rows touch every bank once)
#pragma unroll 4
    for (int i = t; i < 128 * 32; i += Q_THREADS) {
      const int r = i & 127, c = (i >> 7) * 4;
      const float4 f = *reinterpret_cast<const float4*>(stage + r * Q_ROW_T + (c >> 5) * Q_BLOCK + (c & 31));
      const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r0 + r < p.rows && k0 + c + j < p.k) static_cast<T*>(p.out)[(k0 + c + j) * p.rows + r0 + r] = elem_from_float<T>(v[j]);
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------
static long long tiles128(long long n) { return (n + 127) / 128; }
static long long tiles256(long long k) { return k <= 0 ? 1 : (k + 255) / 256; }
static bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int check_size(long long rows, long long k, const char* what) {
  if (rows < 0 || k < 0) return host_fail(AMSIM_ERR_INVALID, "%s: sizes must not be negative", what);
  if (rows >= (1ll << 31) || k >= (1ll << 31) || (k && rows > (1ll << 40) / k)) return host_fail(AMSIM_ERR_UNSUPPORTED, "%s: more than 2^31 rows or columns, or 2^40 elements", what);
  return AMSIM_OK;
}

template <auto kernel, int SMEM, typename P>
static cudaError_t launch(long long grid, int threads, int cluster, cudaStream_t st, const P& p) {
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = host_allow_smem(kernel, SMEM, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = SMEM;
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

template <int CG, int BN>
static cudaError_t gemm_launch(GemmParams& p, int dtype, int device, cudaStream_t st) {
  using S = Shape<CG, BN>;
  p.tiles_n = (p.b_tiles + CG - 1) / CG;
  const long long tiles_t = (p.m + BN - 1) / BN;
  p.tiles = (int)(p.tiles_n * tiles_t);
  const int teams = host_sm_count(device) / CG;
  long long grid = (long long)(p.tiles < teams ? p.tiles : teams) * CG;
  // Tiles that leave half of the multiprocessors idle share their reductions, as long as each CTA has 2048 elements of it: putting
  // the shares together costs 2 us (16 x 8000 outputs over 512 elements 4.1 us, shared by two 6.1).
  p.split = 1;
  while (CG == 1 && p.split < 8 && p.tiles * p.split * 2 <= teams && p.kt >= 16 * p.split && S::COLS / p.split >= 8) p.split *= 2;
  if (p.split > 1) grid = (long long)p.tiles * p.split;
  if (dtype == 0) return launch<gemm<CG, BN, float>, S::SMEM>(grid, S::THREADS, CG * p.split, st, p);
  if (dtype == 1) return launch<gemm<CG, BN, __nv_bfloat16>, S::SMEM>(grid, S::THREADS, CG * p.split, st, p);
  return launch<gemm<CG, BN, __half>, S::SMEM>(grid, S::THREADS, CG * p.split, st, p);
}

}  // namespace mx
}  // namespace amsim

extern "C" {

size_t amsim_mx_bytes(long long rows, long long k) {
  using namespace amsim::mx;
  if (rows <= 0 || k < 0 || rows >= (1ll << 31) || k >= (1ll << 31)) return 0;
  return (size_t)tiles128(rows) * (size_t)tiles256(k) * TILE_BYTES;
}

size_t amsim_mx_quantize_workspace(long long rows, long long cols) {
  using namespace amsim::mx;
  return rows <= 0 || cols <= 0 ? 0 : (size_t)tiles128(rows) * (size_t)cols * sizeof(float);
}

int amsim_mx_quantize(void* stream, const void* x, long long rows, long long cols, int dtype, void* along, void* across, float* sums, void* workspace,
                      size_t workspace_bytes) {
  using namespace amsim;
  using namespace amsim::mx;
  if (const int rc = check_size(rows, cols, "mx_quantize")) return rc;
  if (dtype < 0 || dtype > 2) return host_fail(AMSIM_ERR_INVALID, "mx_quantize: unknown type %d", dtype);
  if (sums && !across) return host_fail(AMSIM_ERR_INVALID, "mx_quantize: column sums come with the columns' codes");
  if (rows == 0) along = nullptr;   // (no rows to store)
  if (cols == 0) across = nullptr, sums = nullptr;
  if (sums && rows == 0) {
    AMSIM_HOST_TRY(cudaMemsetAsync(sums, 0, (size_t)cols * sizeof(float), (cudaStream_t)stream));
    sums = nullptr;
  }
  const size_t need = sums ? amsim_mx_quantize_workspace(rows, cols) : 0;
  if (need && (!workspace || workspace_bytes < need)) return host_fail(AMSIM_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
  if (need && ((uintptr_t)workspace & 3)) return host_fail(AMSIM_ERR_WORKSPACE, "workspace must be 4-byte aligned");
  if (!along && !across) return rows == 0 || cols == 0 ? AMSIM_OK : host_fail(AMSIM_ERR_INVALID, "mx_quantize: no output");
  if (rows && cols && !x) return host_fail(AMSIM_ERR_INVALID, "NULL tensor pointer");
  if (!aligned(along) || !aligned(across)) return host_fail(AMSIM_ERR_INVALID, "mx_quantize: outputs must be 16-byte aligned");
  QuantParams p = {};
  p.x = x; p.along = static_cast<uint8_t*>(along); p.across = static_cast<uint8_t*>(across);
  p.rows = rows; p.cols = cols; p.along_kt = tiles256(cols); p.across_kt = tiles256(rows);
  p.vec = aligned(x) && cols % (dtype == 0 ? 4 : 8) == 0;
  p.sums = sums ? static_cast<float*>(workspace) : nullptr;
  p.gx = along ? 2 * p.along_kt : tiles128(cols);
  const long long grid = p.gx * (across ? 2 * p.across_kt : tiles128(rows));
  if (grid >= (1ll << 31)) return host_fail(AMSIM_ERR_UNSUPPORTED, "mx_quantize: more than 2^31 tiles");
  cudaStream_t st = (cudaStream_t)stream;
  AMSIM_HOST_TRY(dtype == 0 ? launch<quantise<float>, Stage<float>::BYTES>(grid, Q_THREADS, 1, st, p)
                            : dtype == 1 ? launch<quantise<__nv_bfloat16>, Stage<__half>::BYTES>(grid, Q_THREADS, 1, st, p) : launch<quantise<__half>, Stage<__half>::BYTES>(grid, Q_THREADS, 1, st, p));
  if (sums) {
    host_count_launch();
    add_sums<<<(unsigned)((cols + 31) / 32), 512, 0, st>>>(p.sums, sums, cols, (int)tiles128(rows));
    AMSIM_HOST_TRY(cudaGetLastError());
  }
  return AMSIM_OK;
}

int amsim_mx_dequantize(void* stream, const void* data, long long rows, long long k, int transposed, void* out, int dtype) {
  using namespace amsim;
  using namespace amsim::mx;
  if (const int rc = check_size(rows, k, "mx_dequantize")) return rc;
  if (dtype < 0 || dtype > 2) return host_fail(AMSIM_ERR_INVALID, "mx_dequantize: unknown type %d", dtype);
  if (rows == 0 || k == 0) return AMSIM_OK;
  if (!data || !out) return host_fail(AMSIM_ERR_INVALID, "NULL tensor pointer");
  if (!aligned(data)) return host_fail(AMSIM_ERR_INVALID, "mx_dequantize: the matrix must be 16-byte aligned");
  DequantParams p = {};
  p.data = static_cast<const uint8_t*>(data); p.out = out; p.rows = rows; p.k = k; p.kt = tiles256(k);
  p.transposed = transposed != 0; p.pitch = transposed ? Q_ROW_T : Q_ROW;
  p.vec = aligned(out) && k % (dtype == 0 ? 4 : 8) == 0;
  p.gx = tiles128(k);
  const long long grid = p.gx * tiles128(rows);
  if (grid >= (1ll << 31)) return host_fail(AMSIM_ERR_UNSUPPORTED, "mx_dequantize: more than 2^31 tiles");
  cudaStream_t st = (cudaStream_t)stream;
  AMSIM_HOST_TRY(dtype == 0 ? launch<dequantise<float>, Q_SMEM_T>(grid, Q_THREADS, 1, st, p)
                            : dtype == 1 ? launch<dequantise<__nv_bfloat16>, Q_SMEM_T>(grid, Q_THREADS, 1, st, p) : launch<dequantise<__half>, Q_SMEM_T>(grid, Q_THREADS, 1, st, p));
  return AMSIM_OK;
}

int amsim_mx_matmul(void* stream, const void* a, const void* b, long long m, long long n, long long k, const float* bias, int act, void* out, int dtype) {
  using namespace amsim;
  using namespace amsim::mx;
  if (const int rc = check_size(m, k, "mx_matmul")) return rc;
  if (const int rc = check_size(n, k, "mx_matmul")) return rc;
  if (m && n > (1ll << 40) / m) return host_fail(AMSIM_ERR_UNSUPPORTED, "mx_matmul: more than 2^40 outputs");
  if (dtype < 0 || dtype > 2) return host_fail(AMSIM_ERR_INVALID, "mx_matmul: unknown type %d", dtype);
  if (act != AMSIM_ACT_NONE && act != AMSIM_ACT_RELU) return host_fail(AMSIM_ERR_INVALID, "unknown activation %d", act);
  if (m == 0 || n == 0) return AMSIM_OK;
  if (!a || !b || !out) return host_fail(AMSIM_ERR_INVALID, "NULL tensor pointer");
  if (!aligned(a) || !aligned(b)) return host_fail(AMSIM_ERR_INVALID, "mx_matmul: operands must be 16-byte aligned");
  const int device = host_device();
  GemmParams p = {};
  if (const int rc = host_stuck_word(device, &p.stuck)) return rc;
  if (const int rc = host_report_stuck(device)) return rc;
  p.a = static_cast<const uint8_t*>(a); p.b = static_cast<const uint8_t*>(b); p.bias = bias; p.out = out;
  p.m = m; p.n = n; p.a_tiles = (int)tiles128(m); p.b_tiles = (int)tiles128(n); p.kt = (int)tiles256(k);
  p.last_steps = k == 0 ? 1 : (int)((k - (long long)(p.kt - 1) * 256 + 63) / 64);
  p.chunk = dtype == 0 ? 8 : 32;
  p.relu = act == AMSIM_ACT_RELU;
  p.no_tries = host_no_tries();
  if ((long long)((p.a_tiles + 1) / 2 + 1) * p.b_tiles >= (1ll << 30)) return host_fail(AMSIM_ERR_UNSUPPORTED, "mx_matmul: more than 2^30 tiles");
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  // Up to 64 tokens: tiles of 128 columns x 16, 32 or 64, so that little of the tokens' operand is copied in vain.  Else pairs of CTAs with
  // tiles of 256 x 256, unless those fill less than a quarter of the multiprocessors, where tiles of 128 x 128 are four times as many
  // (512 x 2048 outputs over 8192 elements: 16 pairs' tiles or 64).
  if (m <= 16) e = gemm_launch<1, 16>(p, dtype, device, st);
  else if (m <= 32) e = gemm_launch<1, 32>(p, dtype, device, st);
  else if (m <= 64) e = gemm_launch<1, 64>(p, dtype, device, st);
  else if (((m + 255) / 256) * ((n + 255) / 256) * 4 < host_sm_count(device)) e = gemm_launch<1, 128>(p, dtype, device, st);
  else e = gemm_launch<2, 256>(p, dtype, device, st);
  AMSIM_HOST_TRY(e);
  return AMSIM_OK;
}

}  // extern "C"

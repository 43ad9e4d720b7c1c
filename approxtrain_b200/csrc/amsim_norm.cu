// The C entry points of the norms around a residual block, and its FP32 kernels (amsim_norm.cuh).
#include "amsim_norm.cuh"

namespace amsim {
namespace normk {

extern template cudaError_t launch_type<__nv_bfloat16>(NormParams&, bool, bool, bool, int, int, cudaStream_t, const Plan*);
extern template cudaError_t launch_type<__half>(NormParams&, bool, bool, bool, int, int, cudaStream_t, const Plan*);
extern template cudaError_t launch_reduce<__nv_bfloat16>(const NormParams&, const Plan&, cudaStream_t);
extern template cudaError_t launch_reduce<__half>(const NormParams&, const Plan&, cudaStream_t);

static cudaError_t dispatch(NormParams& p, bool backward, bool layer, bool post, int dtype, int device, cudaStream_t st, const Plan* bwd) {
  // a gate of one row per row, of the activations' type, is fetched ahead like them
  const int gate = !p.gate ? GATE_NONE : p.per_gate == 1 && p.gate_type == dtype ? GATE_ROWS : GATE_SHARED;
  if (gate == GATE_ROWS) p.in_gate = p.n_in++;
  if (dtype == 0) return launch_type<float>(p, backward, layer, post, gate, device, st, bwd);
  if (dtype == 1) return launch_type<__nv_bfloat16>(p, backward, layer, post, gate, device, st, bwd);
  return launch_type<__half>(p, backward, layer, post, gate, device, st, bwd);
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
  p.pre = pre;
  p.in_x = p.n_in++;
  if (block) p.in_block = p.n_in++;
  AMSIM_HOST_TRY(dispatch(p, false, layer, post, dtype, host_device(), (cudaStream_t)stream, nullptr));
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
  p.pre = pre;
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
  p.tpr = pl.s.tpr; p.cluster = pl.s.cluster;
  if (dy) p.in_dy = p.n_in++, p.in_x = p.n_in++;
  else p.x = nullptr;  // (without a gradient through N_pre neither x nor the sum is needed)
  if (!dy && !post && !gate) p.block = nullptr;
  if (p.block) p.in_block = p.n_in++;
  if (dsum) p.in_dsum = p.n_in++;
  AMSIM_HOST_TRY(dispatch(p, true, layer, post, dtype, host_device(), st, &pl));
  AMSIM_HOST_TRY(dtype == 0 ? launch_reduce<float>(p, pl, st) : dtype == 1 ? launch_reduce<__nv_bfloat16>(p, pl, st) : launch_reduce<__half>(p, pl, st));
  return AMSIM_OK;
}

}  // extern "C"

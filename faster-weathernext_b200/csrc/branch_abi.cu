// C ABI of the residual branches (include/fwn_attn.h): argument checks and launches.
#include <algorithm>

#include "abi.cuh"
#include "branch.cuh"

using namespace fwn;

namespace {

fwn_status check_drop(const fwn_dropout_desc& d) {
  if (d.threshold > 65536u) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "dropout threshold %u exceeds 65536", d.threshold);
  if (!abi_aligned(d.seed_at, 8)) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "seed_at must be 8-byte aligned");
  return FWN_OK;
}
DropParams drop_of(const fwn_dropout_desc& d) { return drop_params(d.seed, d.seed_at, d.site, d.threshold); }

fwn_status check_branch(const fwn_branch_desc* d, bool bwd) {
  if (!d) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "desc is null");
  if (d->rows < 0 || d->d <= 0) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bad rows=%lld or d=%d", static_cast<long long>(d->rows), d->d);
  if (d->d > kBranchMaxWidth) return abi_fail(FWN_ERR_UNSUPPORTED, "d=%d exceeds %d", d->d, kBranchMaxWidth);
  if (d->rows > INT32_MAX) return abi_fail(FWN_ERR_UNSUPPORTED, "rows=%lld exceeds 2^31 - 1", static_cast<long long>(d->rows));
  if (!abi_float(d->x_dtype) || !abi_float(d->y_dtype) || !abi_float(d->post_dtype) || !abi_float(d->weight_dtype) ||
      !abi_float(d->gate_dtype))
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "x, y, the weights and the gate are bf16 or float32");
  if (!abi_float(d->out_dtype) && (bwd || d->out_dtype != FWN_DTYPE_E4M3))
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "unknown out dtype %d", d->out_dtype);
  if (!(d->eps >= 0.f)) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "eps must not be negative");
  if (d->rows > 1 && (d->x_stride < d->d || d->y_stride < d->d))
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "row strides must be at least d");
  if (d->rows > 0 && (d->gate_span < 1 || d->gate_span > d->rows || d->rows % d->gate_span != 0))
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "gate_span=%lld does not divide rows=%lld", static_cast<long long>(d->gate_span),
                    static_cast<long long>(d->rows));
  return check_drop(d->drop);
}

// Whether a tensor starts where 8 values are one access: 32 bytes of float32, 16 of bf16, 8 of e4m3.
bool starts_wide(const void* p, int32_t dtype) { return abi_aligned(p, 8 * abi_size(dtype)); }

// 1: rows of whole wide accesses, 0: contiguous rows of any width, -1: neither.
int branch_wide(const fwn_branch_desc& d, bool starts) {
  if (!starts) return -1;
  if (d.d % 8 == 0 && (d.rows <= 1 || (d.x_stride % 8 == 0 && d.y_stride % 8 == 0))) return 1;
  return d.d + 7 <= kBranchMaxWidth && (d.rows <= 1 || (d.x_stride == d.d && d.y_stride == d.d)) ? 0 : -1;
}
bool gate_values(const fwn_branch_desc& d, const void* gate) { return gate && d.gate_span == 1 && d.rows > 1; }
// Gates with rows of their own to sum over.
int gates_of(const fwn_branch_desc& d, bool gate, bool values) { return gate && !values ? static_cast<int>(d.rows / d.gate_span) : 1; }

fwn_status no_access() {
  return abi_fail(FWN_ERR_UNSUPPORTED, "rows off 8 values (or 16 bytes of bf16, 32 of float32) must be contiguous, start there and be at most %d wide",
                  kBranchMaxWidth - 7);
}

struct BwdPlan {
  int gates, slices, blocks;
  size_t u, bytes;  // bytes of the partials of u, of all
};
BwdPlan plan_bwd(const fwn_branch_desc& d, bool gate, bool values, bool wide) {
  BwdPlan pl{};
  pl.gates = gates_of(d, gate, values);
  branch_bwd_shape(d.rows, d.d, pl.gates, abi_sms(), wide, &pl.slices, &pl.blocks);
  const size_t row = static_cast<size_t>(d.d) * sizeof(float);
  pl.u = static_cast<size_t>(pl.gates) * pl.slices * row;
  pl.bytes = pl.u + static_cast<size_t>(pl.blocks) * row;
  return pl;
}

}  // namespace

extern "C" {

fwn_status fwn_dropout(const fwn_dropout_desc* drop, const void* x, void* out, int64_t n, int32_t dtype, void* stream) {
  if (!drop) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "drop is null");
  if (fwn_status s = check_drop(*drop); s != FWN_OK) return s;
  if (n < 0) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bad n=%lld", static_cast<long long>(n));
  if (!abi_float(dtype)) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "values are bf16 or float32 (got dtype %d)", dtype);
  if (n > (1ll << 42)) return abi_fail(FWN_ERR_UNSUPPORTED, "n=%lld too large", static_cast<long long>(n));
  if (n == 0) return abi_ok();
  if (!x || !out) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  if (fwn_status s = abi_elements({{x, abi_size(dtype)}, {out, abi_size(dtype)}}); s != FWN_OK) return s;
  cudaError_t e = launch_dropout(x, out, n, dtype == FWN_DTYPE_BF16, starts_wide(x, dtype) && starts_wide(out, dtype),
                                 drop_of(*drop), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return abi_cuda_fail(e, "dropout");
  return abi_ok();
}

fwn_status fwn_branch_norm(const fwn_branch_desc* desc, const void* x, const void* y, const void* post_weight,
                           const void* weight, const void* gate, void* s, void* h, float* scale, float* rstd, void* stream) {
  if (fwn_status st = check_branch(desc, false); st != FWN_OK) return st;
  const fwn_branch_desc& d = *desc;
  if (d.rows == 0) return abi_ok();
  if (!x || !y || !s || !h) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  if ((d.out_dtype == FWN_DTYPE_E4M3) != (scale != nullptr))
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "scale goes with an E4M3 output, and with that alone");
  const int64_t xs = abi_size(d.x_dtype), ys = abi_size(d.y_dtype);
  if (fwn_status st = abi_elements({{x, xs}, {s, xs}, {y, ys}, {h, abi_size(d.out_dtype)}, {post_weight, abi_size(d.post_dtype)},
                                    {weight, abi_size(d.weight_dtype)}, {gate, abi_size(d.gate_dtype)}, {scale, 4}, {rstd, 8}});
      st != FWN_OK)
    return st;
  // The weights and a gate of few rows are read in 16-byte accesses where rows are wide, by single values elsewhere.
  const bool values = gate_values(d, gate);
  bool starts = starts_wide(x, d.x_dtype) && starts_wide(s, d.x_dtype) && starts_wide(y, d.y_dtype) && starts_wide(h, d.out_dtype);
  if (values) starts = starts && starts_wide(gate, d.gate_dtype);
  const bool columns = abi_aligned(post_weight, 16) && abi_aligned(weight, 16) && abi_aligned(gate, 16);
  int wide = branch_wide(d, starts);
  if (wide == 1 && !columns)
    wide = d.d + 7 <= kBranchMaxWidth && (d.rows <= 1 || (d.x_stride == d.d && d.y_stride == d.d)) ? 0 : -1;
  if (wide < 0) return no_access();
  BranchParams p{};
  p.x = x;
  p.y = y;
  p.post_weight = post_weight;
  p.weight = weight;
  p.gate = gate;
  p.s = s;
  p.h = h;
  p.scale = scale;
  p.rstd = rstd;
  p.rows = d.rows;
  p.x_stride = d.x_stride;
  p.y_stride = d.y_stride;
  p.gate_span = d.gate_span;
  p.d = d.d;
  p.eps = d.eps;
  p.alpha = d.residual_scale;
  p.out_type = d.out_dtype == FWN_DTYPE_BF16 ? kRmsBf16 : d.out_dtype == FWN_DTYPE_F32 ? kRmsF32 : kRmsE4m3;
  p.x_bf16 = d.x_dtype == FWN_DTYPE_BF16;
  p.y_bf16 = d.y_dtype == FWN_DTYPE_BF16;
  p.post_bf16 = d.post_dtype == FWN_DTYPE_BF16;
  p.weight_bf16 = d.weight_dtype == FWN_DTYPE_BF16;
  p.gate_bf16 = d.gate_dtype == FWN_DTYPE_BF16;
  p.wide = wide == 1;
  p.sms = abi_sms();
  p.drop = drop_of(d.drop);
  cudaError_t e = launch_branch(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return abi_cuda_fail(e, "branch_norm");
  return abi_ok();
}

fwn_status fwn_branch_norm_bwd_workspace_size(const fwn_branch_desc* desc, size_t* bytes) {
  if (!bytes) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bytes is null");
  if (fwn_status s = check_branch(desc, true); s != FWN_OK) return s;
  *bytes = 0;
  if (desc->rows == 0) return abi_ok();
  // The launch goes by the operands' addresses and by which there are: the most that any of them needs.
  for (bool gate : {false, true})
    for (bool wide : {false, true})
      *bytes = std::max(*bytes, plan_bwd(*desc, gate, gate && desc->gate_span == 1 && desc->rows > 1, wide).bytes);
  return abi_ok();
}

fwn_status fwn_branch_norm_bwd(const fwn_branch_desc* desc, const void* x, const void* y, const void* post_weight,
                               const void* weight, const void* gate, const float* rstd, const void* dh, const void* ds, void* dx,
                               void* dy, void* d_post_weight, void* d_weight, void* d_gate, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (fwn_status st = check_branch(desc, true); st != FWN_OK) return st;
  const fwn_branch_desc& d = *desc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((d_post_weight && !post_weight) || (d_weight && !weight) || (d_gate && !gate))
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "a gradient needs what it belongs to");
  const int64_t xs = abi_size(d.x_dtype), ys = abi_size(d.y_dtype), ps = abi_size(d.post_dtype), ws = abi_size(d.weight_dtype),
                gs = abi_size(d.gate_dtype);
  if (fwn_status s = abi_elements({{x, xs}, {ds, xs}, {dx, xs}, {y, ys}, {dy, ys}, {dh, abi_size(d.out_dtype)}, {post_weight, ps},
                                   {d_post_weight, ps}, {weight, ws}, {d_weight, ws}, {gate, gs}, {d_gate, gs}, {rstd, 8}});
      s != FWN_OK)
    return s;
  if (d.rows == 0) {
    cudaError_t e = cudaSuccess;
    if (d_post_weight) e = cudaMemsetAsync(d_post_weight, 0, d.d * ps, st);
    if (e == cudaSuccess && d_weight) e = cudaMemsetAsync(d_weight, 0, d.d * ws, st);
    if (e != cudaSuccess) return abi_cuda_fail(e, "clear the weights' gradients");
    return abi_ok();  // a gate of no rows has no gradient to write
  }
  if (!x || !y || !rstd) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  const bool values = gate_values(d, gate);
  bool starts = true;
  for (const void* t : {x, ds, static_cast<const void*>(dx)}) starts = starts && starts_wide(t, d.x_dtype);
  for (const void* t : {y, static_cast<const void*>(dy)}) starts = starts && starts_wide(t, d.y_dtype);
  starts = starts && starts_wide(dh, d.out_dtype);
  if (values) starts = starts && starts_wide(gate, d.gate_dtype) && starts_wide(d_gate, d.gate_dtype);
  const bool columns = abi_aligned(post_weight, 16) && abi_aligned(weight, 16) && abi_aligned(gate, 16);
  int wide = branch_wide(d, starts);
  if (wide == 1 && !columns)
    wide = d.d + 7 <= kBranchMaxWidth && (d.rows <= 1 || (d.x_stride == d.d && d.y_stride == d.d)) ? 0 : -1;
  if (wide < 0) return no_access();
  const BwdPlan pl = plan_bwd(d, gate != nullptr, values, wide == 1);
  size_t need = 0;
  if (fwn_status s = fwn_branch_norm_bwd_workspace_size(desc, &need); s != FWN_OK) return s;
  if (need > 0 && (!workspace || workspace_bytes < need || !abi_aligned(workspace, 16)))
    return abi_fail(FWN_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed", need);
  BranchBwdParams p{};
  p.x = x;
  p.y = y;
  p.post_weight = post_weight;
  p.weight = weight;
  p.gate = gate;
  p.rstd = rstd;
  p.dh = dh;
  p.ds = ds;
  p.dx = dx;
  p.dy = dy;
  p.d_post = d_post_weight;
  p.d_weight = d_weight;
  p.d_gate = d_gate;
  p.part_u = d_post_weight || (d_gate && !values) ? static_cast<float*>(workspace) : nullptr;
  p.part_w = d_weight ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + pl.u) : nullptr;
  p.rows = d.rows;
  p.x_stride = d.x_stride;
  p.y_stride = d.y_stride;
  p.gate_span = d.gate_span;
  p.d = d.d;
  p.alpha = d.residual_scale;
  p.x_bf16 = d.x_dtype == FWN_DTYPE_BF16;
  p.y_bf16 = d.y_dtype == FWN_DTYPE_BF16;
  p.post_bf16 = d.post_dtype == FWN_DTYPE_BF16;
  p.weight_bf16 = d.weight_dtype == FWN_DTYPE_BF16;
  p.gate_bf16 = d.gate_dtype == FWN_DTYPE_BF16;
  p.dh_bf16 = d.out_dtype == FWN_DTYPE_BF16;
  p.wide = wide == 1;
  p.gate_values = values;
  p.gates = pl.gates;
  p.slices = pl.slices;
  p.blocks = pl.blocks;
  p.drop = drop_of(d.drop);
  cudaError_t e = p.x_bf16 ? launch_branch_bwd_bf16(p, st) : launch_branch_bwd_f32(p, st);
  if (e == cudaSuccess) e = launch_branch_bwd_finish(p, st);
  if (e != cudaSuccess) return abi_cuda_fail(e, "branch_norm_bwd");
  return abi_ok();
}

}  // extern "C"

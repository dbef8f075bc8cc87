// PyTorch operator layer: defines the rbln_custom_ops schemas (identical to
// the ones the reference's torch.library.custom_op definitions generate,
// test/rbln/test_custom_kernel.py:31-486, 576-645) and registers CUDA kernels that
// validate the tensors, allocate the output and scratch from the PyTorch
// caching allocator, and call the C-ABI entry points of librbln_attn.
//
// Argument checks follow the reference frontends
// (torch_rbln/_internal/register_custom_ops.py:175-450): the cache's last
// dimension must be a multiple of 64, inputs are made contiguous. Departures,
// on purpose: the output dtype is q.dtype (not forced fp16), the caller's
// scale is honoured, batch > 1 prefill is allowed.
#include <ATen/ATen.h>
#include <ATen/Context.h>
#include <ATen/SDPBackend.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/_fused_sdp_choice_native.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <string>
#include <vector>

#include "rbln_attn.h"

namespace {

int to_rbln_dtype(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return RBLN_DT_F32;
    case at::kHalf: return RBLN_DT_F16;
    case at::kBFloat16: return RBLN_DT_BF16;
    case at::kFloat8_e4m3fn: return RBLN_DT_FP8_E4M3;
    case at::kShort: return RBLN_DT_I16;
    case at::kInt: return RBLN_DT_I32;
    case at::kLong: return RBLN_DT_I64;
    case at::kBool: return RBLN_DT_BOOL;
    case at::kByte: return RBLN_DT_BOOL;
    default: return -1;
  }
}

const char* status_name(int rc) {
  switch (rc) {
    case RBLN_ERR_INVALID_ARGUMENT: return "invalid argument";
    case RBLN_ERR_UNSUPPORTED: return "unsupported configuration";
    case RBLN_ERR_WORKSPACE: return "workspace too small";
    case RBLN_ERR_LAUNCH: return "kernel launch failed";
    case RBLN_ERR_NO_DEVICE: return "no sm_100 device";
    default: return "unknown error";
  }
}

bool debug_checks() {
  static const bool on = [] {
    const char* e = std::getenv("RBLN_ATTN_CHECK");
    return e && std::string(e) != "0";
  }();
  return on;
}

// Moves an index/mask tensor to q's device (callers may keep small tensors on
// the host, as the reference's tests do for `scale`).
at::Tensor on_device(const at::Tensor& t, const at::Tensor& like) {
  return t.device() == like.device() ? t : t.to(like.device());
}

struct Common {
  at::Tensor q, k, v, seq, bt, mask, scale_dev, out, err, sinks;
  rbln_paged_attn_params_t p{};
};

// Shared validation and parameter fill for the paged ops. k and v undefined:
// their rows are in the cache already.
void fill_paged(Common& c, const char* op, const at::Tensor& q_in, const at::Tensor& k_in,
                const at::Tensor& v_in, at::Tensor& kcache, at::Tensor& vcache, const at::Tensor& seq_in,
                const at::Tensor& scale, const at::Tensor& block_table_in, int64_t block_size,
                const std::optional<at::Tensor>& mask_in, bool decode) {
  TORCH_CHECK(q_in.is_cuda(), op, ": expected CUDA tensors, q is on ", q_in.device());
  const bool rows = k_in.defined();
  TORCH_CHECK(q_in.dim() == 5 && (!rows || (k_in.dim() == 5 && v_in.dim() == 5)), op,
              ": q/k/v must be 5-D [B, Hkv, G, S, D] / [B, Hkv, 1, S, D]");
  TORCH_CHECK(kcache.dim() == 5 && vcache.dim() == 5, op,
              ": kcache/vcache must be 5-D [num_blocks, Hkv, 1, block_size, D]");
  TORCH_CHECK(kcache.size(-1) % 64 == 0, op,
              ": the last dimension of K-cache must be a multiple of 64, but got shape ", kcache.sizes());
  TORCH_CHECK(vcache.size(-1) % 64 == 0, op,
              ": the last dimension of V-cache must be a multiple of 64, but got shape ", vcache.sizes());
  TORCH_CHECK(kcache.sizes() == vcache.sizes() && kcache.strides() == vcache.strides() &&
                  kcache.scalar_type() == vcache.scalar_type(),
              op, ": kcache and vcache must match in shape, strides and dtype");
  // k, v or a cache of another device would be read through a pointer that q's GPU does not have
  TORCH_CHECK(kcache.device() == q_in.device() && vcache.device() == q_in.device(), op,
              ": caches must be on q's device");
  TORCH_CHECK(!rows || (k_in.device() == q_in.device() && v_in.device() == q_in.device()), op,
              ": k and v must be on q's device");
  TORCH_CHECK(kcache.stride(-1) == 1 && kcache.size(2) == 1, op,
              ": caches must be [num_blocks, Hkv, 1, block_size, D] with a contiguous last dim");
  const auto dt = q_in.scalar_type();
  TORCH_CHECK(dt == at::kBFloat16 || dt == at::kHalf, op, ": q must be bfloat16 or float16, got ", dt);
  TORCH_CHECK(!rows || (k_in.scalar_type() == dt && v_in.scalar_type() == dt), op, ": q, k, v must share a dtype");

  c.q = q_in.contiguous();
  const int64_t B = c.q.size(0), Hkv = c.q.size(1), G = c.q.size(2), S = c.q.size(3), D = c.q.size(4);
  if (rows) {
    c.k = k_in.contiguous();
    c.v = v_in.contiguous();
    TORCH_CHECK(c.k.size(0) == B && c.k.size(1) == Hkv && c.k.size(2) == 1 && c.k.size(3) == S &&
                    c.k.size(4) == D && c.v.sizes() == c.k.sizes(),
                op, ": k/v must be [B, Hkv, 1, S, D] matching q ", c.q.sizes(), ", got ", c.k.sizes());
  }
  TORCH_CHECK(kcache.size(1) == Hkv, op, ": caches hold ", kcache.size(1), " KV heads, q has ", Hkv);
  TORCH_CHECK(D <= kcache.size(-1), op, ": head_dim ", D, " exceeds the cache's last dim ", kcache.size(-1));
  TORCH_CHECK(kcache.size(3) == block_size, op, ": block_size ", block_size,
              " does not match the cache's block dimension ", kcache.size(3));
  if (decode) TORCH_CHECK(S == 1, op, ": decode takes one query token per sequence, got S = ", S);

  c.seq = on_device(seq_in, c.q);
  TORCH_CHECK(c.seq.numel() == B, op, ": seq must hold one entry per sequence, got ", c.seq.sizes());
  if (c.seq.scalar_type() != at::kInt) c.seq = c.seq.to(at::kInt);
  c.seq = c.seq.contiguous();

  c.bt = on_device(block_table_in, c.q);
  if (c.bt.dim() == 1) c.bt = c.bt.unsqueeze(0).expand({B, c.bt.size(0)});
  TORCH_CHECK(c.bt.dim() == 2 && (c.bt.size(0) == B || c.bt.size(0) == 1), op,
              ": block_table must be [B, max_blocks], got ", c.bt.sizes());
  const auto btt = c.bt.scalar_type();
  TORCH_CHECK(btt == at::kShort || btt == at::kInt || btt == at::kLong, op,
              ": block_table must be int16/int32/int64");
  if (c.bt.stride(1) != 1) c.bt = c.bt.contiguous();

  auto& p = c.p;
  p.batch = (int32_t)B;
  p.num_kv_heads = (int32_t)Hkv;
  p.group = (int32_t)G;
  p.q_len = (int32_t)S;
  p.head_dim = (int32_t)D;
  p.num_blocks = (int32_t)kcache.size(0);
  p.block_size = (int32_t)block_size;
  p.max_blocks = (int32_t)c.bt.size(1);
  p.q = c.q.data_ptr();
  for (int i = 0; i < 4; ++i) p.q_stride[i] = c.q.stride(i);
  p.q_dtype = to_rbln_dtype(dt);
  c.out = at::empty_like(c.q, at::MemoryFormat::Contiguous);
  p.out = c.out.data_ptr();
  for (int i = 0; i < 4; ++i) p.out_stride[i] = c.out.stride(i);
  if (rows) {
    p.k_new = c.k.data_ptr();
    p.v_new = c.v.data_ptr();
    p.k_new_stride[0] = c.k.stride(0); p.k_new_stride[1] = c.k.stride(1); p.k_new_stride[2] = c.k.stride(3);
    p.v_new_stride[0] = c.v.stride(0); p.v_new_stride[1] = c.v.stride(1); p.v_new_stride[2] = c.v.stride(3);
  }
  p.kcache = kcache.data_ptr();
  p.vcache = vcache.data_ptr();
  p.kv_dtype = to_rbln_dtype(kcache.scalar_type());
  p.cache_stride[0] = kcache.stride(0);
  p.cache_stride[1] = kcache.stride(1);
  p.cache_stride[2] = kcache.stride(3);
  p.seq = c.seq.data_ptr<int32_t>();
  p.seq_stride = 1;
  p.block_table = c.bt.data_ptr();
  p.block_table_dtype = to_rbln_dtype(btt);
  p.block_table_stride = c.bt.size(0) == 1 ? 0 : c.bt.stride(0);

  if (mask_in.has_value() && mask_in->defined()) {
    c.mask = on_device(*mask_in, c.q);
    TORCH_CHECK(c.mask.scalar_type() == at::kFloat || c.mask.scalar_type() == at::kHalf ||
                    c.mask.scalar_type() == at::kBFloat16 || c.mask.scalar_type() == at::kBool,
                op, ": mask must be floating point or bool");
    // an empty one has no pointer, which would read as no mask
    TORCH_CHECK(c.mask.dim() > 0 && c.mask.size(-1) > 0, op, ": mask covers no position, got ", c.mask.sizes());
    if (c.mask.stride(-1) != 1) c.mask = c.mask.contiguous();
    p.mask = c.mask.data_ptr();
    p.mask_dtype = to_rbln_dtype(c.mask.scalar_type());
    p.mask_len = (int32_t)std::min<int64_t>(c.mask.size(-1), (int64_t)p.max_blocks * block_size);
    // batch stride: the mask's leading dim is the batch (or broadcast 1)
    p.mask_stride[0] = c.mask.size(0) == 1 ? 0 : c.mask.stride(0);
    // query-row stride for prefill keep-masks [B, 1, 1, S_q, L]
    p.mask_stride[1] = (c.mask.dim() >= 2 && c.mask.size(-2) == S) ? c.mask.stride(-2) : 0;
  }

  if (scale.is_cuda()) {
    c.scale_dev = on_device(scale, c.q).to(at::kFloat);
    p.scale_dev = c.scale_dev.data_ptr<float>();
  } else {
    p.scale = scale.item<float>();
  }
  if (debug_checks()) {
    c.err = at::zeros({1}, c.q.options().dtype(at::kInt));
    p.error_flags = reinterpret_cast<uint32_t*>(c.err.data_ptr<int32_t>());
  }
}

// The scales of an fp8 cache: float32 [num_blocks, Hkv], alike, beside it.
void check_scales(const char* op, const at::Tensor& kcache, const at::Tensor& k_scale, const at::Tensor& v_scale) {
  TORCH_CHECK(k_scale.scalar_type() == at::kFloat && v_scale.scalar_type() == at::kFloat && k_scale.dim() == 2 &&
                  k_scale.size(0) == kcache.size(0) && k_scale.size(1) == kcache.size(1) &&
                  v_scale.sizes() == k_scale.sizes() && v_scale.strides() == k_scale.strides(),
              op, ": k_scale/v_scale must be float32 [num_blocks, Hkv], alike");
  TORCH_CHECK(k_scale.device() == kcache.device() && v_scale.device() == kcache.device(), op,
              ": scales must be on the caches' device");
}

void check_rc(int rc, const char* op) {
  TORCH_CHECK(rc == RBLN_OK, op, ": ", status_name(rc), " (status ", rc, ")");
}

void check_device_flags(const Common& c, const char* op) {
  if (!c.err.defined()) return;
  const int flags = c.err.item<int>();
  TORCH_CHECK(flags == 0, op, ": device-side input check failed (flags 0x", std::hex, flags,
              "): block_table entry out of range or seq out of range");
}

at::Tensor run_decode(Common& c, at::Tensor& kcache, const char* op, bool require_mask) {
  c10::cuda::CUDAGuard guard(c.q.device());
  size_t ws = 0;
  check_rc(rbln_paged_decode_workspace_size(&c.p, &ws), op);
  at::Tensor wst;
  if (ws > 0) {
    wst = at::empty({(int64_t)ws}, c.q.options().dtype(at::kByte));
    c.p.workspace = wst.data_ptr();
    c.p.workspace_bytes = ws;
  }
  auto stream = at::cuda::getCurrentCUDAStream(c.q.device().index());
  const int rc = require_mask ? rbln_paged_attn_decode(&c.p, stream.stream())
                              : rbln_paged_causal_attn_decode(&c.p, stream.stream());
  check_rc(rc, op);
  check_device_flags(c, op);
  return c.out;
}

// rbln_custom_ops::paged_attn_decode (register_custom_ops.py:253-293)
at::Tensor paged_attn_decode_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                  const at::Tensor& mask, at::Tensor& kcache, at::Tensor& vcache,
                                  const at::Tensor& seq, const at::Tensor& scale,
                                  const at::Tensor& block_table, int64_t block_size) {
  Common c;
  TORCH_CHECK(kcache.scalar_type() == q.scalar_type(), "paged_attn_decode: cache dtype must equal q dtype");
  fill_paged(c, "paged_attn_decode", q, k, v, kcache, vcache, seq, scale, block_table, block_size, mask, true);
  return run_decode(c, kcache, "paged_attn_decode", true);
}

// rbln_custom_ops::paged_causal_attn_decode (register_custom_ops.py:409-450)
at::Tensor paged_causal_attn_decode_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                         at::Tensor& kcache, at::Tensor& vcache, const at::Tensor& seq,
                                         const at::Tensor& scale, const at::Tensor& block_table,
                                         int64_t block_size, const std::optional<at::Tensor>& mask) {
  Common c;
  TORCH_CHECK(kcache.scalar_type() == q.scalar_type(),
              "paged_causal_attn_decode: cache dtype must equal q dtype (use the _kvfp8 op for fp8 caches)");
  fill_paged(c, "paged_causal_attn_decode", q, k, v, kcache, vcache, seq, scale, block_table, block_size,
             mask, true);
  return run_decode(c, kcache, "paged_causal_attn_decode", false);
}

// fp8-e4m3 KV cache with one fp32 dequant scale per (block, KV head). No
// counterpart in the reference's op set; same contract as
// paged_causal_attn_decode plus the two scale tensors [num_blocks, Hkv].
at::Tensor paged_causal_attn_decode_kvfp8_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                               at::Tensor& kcache, at::Tensor& vcache,
                                               const at::Tensor& k_scale, const at::Tensor& v_scale,
                                               const at::Tensor& seq, const at::Tensor& scale,
                                               const at::Tensor& block_table, int64_t block_size,
                                               const std::optional<at::Tensor>& mask) {
  const char* op = "paged_causal_attn_decode_kvfp8";
  TORCH_CHECK(kcache.scalar_type() == at::kFloat8_e4m3fn, op, ": caches must be float8_e4m3fn");
  TORCH_CHECK(k_scale.scalar_type() == at::kFloat && v_scale.scalar_type() == at::kFloat, op,
              ": k_scale/v_scale must be float32 [num_blocks, Hkv]");
  TORCH_CHECK(k_scale.dim() == 2 && k_scale.size(0) == kcache.size(0) && k_scale.size(1) == kcache.size(1) &&
                  v_scale.sizes() == k_scale.sizes() && v_scale.strides() == k_scale.strides(),
              op, ": k_scale/v_scale must be [num_blocks, Hkv]");
  TORCH_CHECK(k_scale.device() == q.device() && v_scale.device() == q.device(), op,
              ": scales must be on q's device");
  Common c;
  fill_paged(c, op, q, k, v, kcache, vcache, seq, scale, block_table, block_size, mask, true);
  c.p.k_scale = k_scale.data_ptr<float>();
  c.p.v_scale = v_scale.data_ptr<float>();
  c.p.scale_stride[0] = k_scale.stride(0);
  c.p.scale_stride[1] = k_scale.stride(1);
  return run_decode(c, kcache, op, false);
}

// rbln_custom_ops::paged_causal_attn_decode_shared: paged_causal_attn_decode
// for a batch in which group g, the sequences [group_starts[g],
// group_starts[g + 1]), shares its first shared_lens[g] positions. No
// counterpart in the reference's op set.
at::Tensor paged_causal_attn_decode_shared_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                at::Tensor& kcache, at::Tensor& vcache, const at::Tensor& seq,
                                                const at::Tensor& scale, const at::Tensor& block_table,
                                                int64_t block_size, const at::Tensor& group_starts,
                                                const at::Tensor& shared_lens) {
  const char* op = "paged_causal_attn_decode_shared";
  TORCH_CHECK(kcache.scalar_type() == q.scalar_type(), op, ": cache dtype must equal q dtype");
  auto whole = [&](const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.dim() == 1 && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong), op, ": ", name,
                " must be 1-D of int32/int64, got ", t.sizes(), " of ", t.scalar_type());
    const at::Tensor x = on_device(t, q);
    // values that 32 bits do not hold are cut as all others are
    return (x.scalar_type() == at::kLong ? x.clamp(-1, INT32_MAX).to(at::kInt) : x).contiguous();
  };
  TORCH_CHECK(q.is_cuda(), op, ": expected CUDA tensors, q is on ", q.device());
  c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor starts = whole(group_starts, "group_starts"), lens = whole(shared_lens, "shared_lens");
  TORCH_CHECK(starts.numel() == lens.numel() + 1, op, ": group_starts must hold one entry more than shared_lens, got ",
              starts.numel(), " and ", lens.numel());
  Common c;
  fill_paged(c, op, q, k, v, kcache, vcache, seq, scale, block_table, block_size, std::nullopt, true);
  rbln_shared_prefix_t s{};
  s.num_groups = (int32_t)lens.numel();
  s.group_starts = starts.data_ptr<int32_t>();
  s.shared_lens = lens.data_ptr<int32_t>();
  size_t ws = 0;
  check_rc(rbln_paged_decode_shared_workspace_size(&c.p, &s, &ws), op);
  const at::Tensor workspace = at::empty({(int64_t)ws}, c.q.options().dtype(at::kByte));
  c.p.workspace = workspace.data_ptr();
  c.p.workspace_bytes = ws;
  check_rc(rbln_paged_causal_attn_decode_shared(&c.p, &s, at::cuda::getCurrentCUDAStream(c.q.device().index()).stream()),
           op);
  check_device_flags(c, op);
  return c.out;
}

at::Tensor run_prefill(Common& c, const char* op, bool keep_mask) {
  c10::cuda::CUDAGuard guard(c.q.device());
  size_t ws = 0;
  check_rc(rbln_paged_prefill_workspace_size(&c.p, &ws), op);
  at::Tensor wst;
  if (ws > 0) {
    wst = at::empty({(int64_t)ws}, c.q.options().dtype(at::kByte));
    c.p.workspace = wst.data_ptr();
    c.p.workspace_bytes = ws;
  }
  auto stream = at::cuda::getCurrentCUDAStream(c.q.device().index());
  const int rc = keep_mask ? rbln_paged_attn_prefill(&c.p, stream.stream())
                           : rbln_paged_causal_attn_prefill(&c.p, stream.stream());
  check_rc(rc, op);
  check_device_flags(c, op);
  return c.out;
}

// rbln_custom_ops::paged_attn_prefill (register_custom_ops.py:175-229)
at::Tensor paged_attn_prefill_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                   const at::Tensor& mask, at::Tensor& kcache, at::Tensor& vcache,
                                   const at::Tensor& seq, const at::Tensor& scale, const at::Tensor& block_table,
                                   int64_t block_size) {
  const char* op = "paged_attn_prefill";
  TORCH_CHECK(kcache.scalar_type() == q.scalar_type(), op, ": cache dtype must equal q dtype");
  Common c;
  fill_paged(c, op, q, k, v, kcache, vcache, seq, scale, block_table, block_size, mask, false);
  return run_prefill(c, op, true);
}

// rbln_custom_ops::paged_causal_attn_prefill (register_custom_ops.py:324-379)
at::Tensor paged_causal_attn_prefill_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                          at::Tensor& kcache, at::Tensor& vcache, const at::Tensor& seq,
                                          const at::Tensor& scale, const at::Tensor& block_table, int64_t block_size,
                                          bool is_bidirectional, const std::optional<at::Tensor>& mask) {
  const char* op = "paged_causal_attn_prefill";
  TORCH_CHECK(kcache.scalar_type() == q.scalar_type(), op, ": cache dtype must equal q dtype");
  Common c;
  fill_paged(c, op, q, k, v, kcache, vcache, seq, scale, block_table, block_size, mask, false);
  c.p.causal = is_bidirectional ? 0 : 1;
  return run_prefill(c, op, false);
}

// rbln_custom_ops::paged_causal_attn_prefill_kvfp8: paged_causal_attn_prefill
// over an fp8-e4m3 cache with one fp32 dequant scale per (block, KV head). No
// counterpart in the reference's op set; k and v absent: their rows are in the
// cache already (rotary_paged_kv_write).
at::Tensor paged_causal_attn_prefill_kvfp8_cuda(const at::Tensor& q, const std::optional<at::Tensor>& k,
                                                const std::optional<at::Tensor>& v, at::Tensor& kcache,
                                                at::Tensor& vcache, at::Tensor& k_scale, at::Tensor& v_scale,
                                                const at::Tensor& seq, const at::Tensor& scale,
                                                const at::Tensor& block_table, int64_t block_size,
                                                bool is_bidirectional, const std::optional<at::Tensor>& mask) {
  const char* op = "paged_causal_attn_prefill_kvfp8";
  TORCH_CHECK(kcache.scalar_type() == at::kFloat8_e4m3fn, op, ": caches must be float8_e4m3fn");
  const bool rows = k.has_value() && k->defined();
  TORCH_CHECK(rows == (v.has_value() && v->defined()), op, ": k and v go together");
  TORCH_CHECK(q.dim() == 5, op, ": q must be 5-D [B, Hkv, G, S, D]");
  check_scales(op, kcache, k_scale, v_scale);
  Common c;
  fill_paged(c, op, q, rows ? *k : at::Tensor(), rows ? *v : at::Tensor(), kcache, vcache, seq, scale, block_table,
             block_size, mask, false);
  if (c.mask.defined())
    TORCH_CHECK(c.mask.dim() == 2 && (c.mask.size(0) == 1 || c.mask.size(0) == q.size(0)), op,
                ": mask must be a position mask [B, L], got ", c.mask.sizes());
  c.p.k_scale = k_scale.data_ptr<float>();
  c.p.v_scale = v_scale.data_ptr<float>();
  c.p.scale_stride[0] = k_scale.stride(0);
  c.p.scale_stride[1] = k_scale.stride(1);
  c.p.causal = is_bidirectional ? 0 : 1;
  return run_prefill(c, op, false);
}

// ---------------------------------------------------------------------------
// Rotary positions (rotary.cu)
// ---------------------------------------------------------------------------
bool is_float16or32(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

at::Tensor check_inv_freq(const char* op, const at::Tensor& inv_freq, const at::Tensor& like) {
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kFloat && inv_freq.numel() > 0, op,
              ": inv_freq must be float32 [rotary_dim / 2], got ", inv_freq.sizes(), " of ", inv_freq.scalar_type());
  TORCH_CHECK(2 * inv_freq.numel() <= like.size(-1), op, ": rotary_dim ", 2 * inv_freq.numel(),
              " exceeds the head dimension ", like.size(-1));
  return on_device(inv_freq, like).contiguous();
}

// rbln_attn::rotary: q [B, Hq, S, D] and k [B, Hk, S, D] turned by their
// positions [B, S] (or [S]); the outputs keep the inputs' layout.
std::tuple<at::Tensor, at::Tensor> rotary_cuda(const at::Tensor& q_in, const at::Tensor& k_in,
                                               const at::Tensor& positions, const at::Tensor& inv_freq_in,
                                               bool interleaved, double mscale, bool inverse) {
  const char* op = "rotary";
  TORCH_CHECK(q_in.is_cuda() && k_in.device() == q_in.device(), op, ": q and k must be on one CUDA device");
  TORCH_CHECK(q_in.dim() == 4 && k_in.dim() == 4 && k_in.size(0) == q_in.size(0) && k_in.size(2) == q_in.size(2) &&
                  k_in.size(3) == q_in.size(3),
              op, ": q and k must be [B, H, S, D] alike but for H, got ", q_in.sizes(), " and ", k_in.sizes());
  const auto dt = q_in.scalar_type();
  TORCH_CHECK(is_float16or32(dt) && k_in.scalar_type() == dt, op,
              ": q and k must share one of bfloat16, float16 and float32, got ", dt, " and ", k_in.scalar_type());
  const int64_t B = q_in.size(0), S = q_in.size(2), D = q_in.size(3);
  at::Tensor inv_freq = check_inv_freq(op, inv_freq_in, q_in);
  at::Tensor pos = on_device(positions, q_in);
  TORCH_CHECK(pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong, op,
              ": positions must be int32 or int64, got ", pos.scalar_type());
  if (pos.dim() == 1) pos = pos.unsqueeze(0);
  TORCH_CHECK(pos.dim() == 2 && (pos.size(0) == B || pos.size(0) == 1) && pos.size(1) == S, op,
              ": positions must be [B, S] or [S], got ", positions.sizes(), " for ", q_in.sizes());
  c10::cuda::CUDAGuard guard(q_in.device());
  auto inner = [](const at::Tensor& t) { return t.stride(-1) == 1 || t.numel() == 0 ? t : t.contiguous(); };
  at::Tensor q = inner(q_in), k = inner(k_in);
  at::Tensor qo = at::empty_like(q_in), ko = at::empty_like(k_in);
  if (qo.stride(-1) != 1) qo = at::empty_like(q_in, at::MemoryFormat::Contiguous);
  if (ko.stride(-1) != 1) ko = at::empty_like(k_in, at::MemoryFormat::Contiguous);
  rbln_rotary_params_t p{};
  p.batch = (int32_t)B;
  p.q_heads = (int32_t)q.size(1);
  p.k_heads = (int32_t)k.size(1);
  p.seq_len = (int32_t)S;
  p.head_dim = (int32_t)D;
  p.rotary_dim = (int32_t)(2 * inv_freq.numel());
  p.dtype = to_rbln_dtype(dt);
  p.q = q.data_ptr();
  p.q_out = qo.data_ptr();
  p.k = k.data_ptr();
  p.k_out = ko.data_ptr();
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = q.stride(i);
    p.q_out_stride[i] = qo.stride(i);
    p.k_stride[i] = k.stride(i);
    p.k_out_stride[i] = ko.stride(i);
  }
  p.positions = pos.data_ptr();
  p.positions_dtype = to_rbln_dtype(pos.scalar_type());
  p.positions_stride[0] = pos.size(0) == 1 ? 0 : pos.stride(0);
  p.positions_stride[1] = pos.stride(1);
  p.inv_freq = inv_freq.data_ptr<float>();
  p.interleaved = interleaved;
  p.inverse = inverse;
  p.mscale = (float)mscale;
  check_rc(rbln_rotary(&p, at::cuda::getCurrentCUDAStream(q.device().index()).stream()), op);
  return {qo, ko};
}

using RotaryOp = std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                    const at::Tensor&, bool, double, bool);
std::tuple<at::Tensor, at::Tensor> call_rotary(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                                               const at::Tensor& inv_freq, bool interleaved, double mscale,
                                               bool inverse) {
  static auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("rbln_attn::rotary", "").typed<RotaryOp>();
  return op.call(q, k, positions, inv_freq, interleaved, mscale, inverse);
}

// The map is linear: the gradient is the transposed map of the outputs'
// gradients, the same op (so it can be differentiated again).
struct RotaryBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable positions, inv_freq;
  at::TensorOptions options;
  std::vector<c10::SymInt> q_size, k_size;  // symbols in a trace
  bool interleaved, inverse;
  double mscale;

  std::string name() const override { return "RotaryBackward"; }
  void release_variables() override {
    positions.reset_data();
    inv_freq.reset_data();
  }
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grad) override {
    // an output that nothing used has no gradient: zeros stand for it
    const at::Tensor gq = grad[0].defined() ? grad[0] : at::zeros_symint(q_size, options);
    const at::Tensor gk = grad[1].defined() ? grad[1] : at::zeros_symint(k_size, options);
    auto [dq, dk] = call_rotary(gq, gk, positions.unpack(), inv_freq.unpack(), interleaved, mscale, !inverse);
    return {task_should_compute_output(0) ? dq : at::Tensor(), task_should_compute_output(1) ? dk : at::Tensor()};
  }
};

// A leaf of a graph that still lives has its gradient node on the stream of
// that graph; a backward pass captured on another stream would make the
// engine wait for it, which breaks the capture. Refused before that. Only a
// leaf that has such a node makes the CUDA runtime be asked, and a traced one
// on a machine without a GPU does not.
void check_capture(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors) {
    if (!t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto at = node ? node->stream() : std::nullopt;
    if (!at.has_value() || c10::cuda::device_count() == 0) continue;
    const auto now = at::cuda::getCurrentCUDAStream(t->device().index());
    if (*at == now.unwrap()) continue;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    C10_CUDA_CHECK(cudaStreamIsCapturing(now.stream(), &status));
    TORCH_CHECK(status == cudaStreamCaptureStatusNone, "rotary: an input belongs to a graph that lives on another "
                "stream; free that graph before capturing, or capture with inputs of their own");
  }
}

std::tuple<at::Tensor, at::Tensor> rotary_autograd(const at::Tensor& q, const at::Tensor& k,
                                                   const at::Tensor& positions, const at::Tensor& inv_freq,
                                                   bool interleaved, double mscale, bool inverse) {
  const bool grads = c10::GradMode::is_enabled();
  TORCH_CHECK(!(grads && inv_freq.requires_grad()) && !inv_freq._fw_grad(0).defined(),
              "rotary: inv_freq has no gradient (detach it)");
  const bool graph = grads && (q.requires_grad() || k.requires_grad());
  if (graph) check_capture({&q, &k});
  std::shared_ptr<RotaryBackward> node;
  if (graph) {
    node = std::shared_ptr<RotaryBackward>(new RotaryBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k));
    node->positions = torch::autograd::SavedVariable(positions, false);
    node->inv_freq = torch::autograd::SavedVariable(inv_freq, false);
    node->options = q.options();
    node->q_size = q.sym_sizes().vec();
    node->k_size = k.sym_sizes().vec();
    node->interleaved = interleaved;
    node->inverse = inverse;
    node->mscale = mscale;
  }
  at::Tensor qo, ko;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    std::tie(qo, ko) = call_rotary(q, k, positions, inv_freq, interleaved, mscale, inverse);
  }
  if (node) torch::autograd::set_history(torch::autograd::variable_list{qo, ko}, node);
  // Forward mode: the map is linear, so it takes the tangents as it takes the tensors.
  const at::Tensor qt = q._fw_grad(0), kt = k._fw_grad(0);
  if (qt.defined() || kt.defined()) {
    auto zeros = [](const at::Tensor& t) { return at::zeros_symint(t.sym_sizes(), t.options()); };
    auto [dq, dk] = call_rotary(qt.defined() ? qt : zeros(q), kt.defined() ? kt : zeros(k), positions, inv_freq,
                                interleaved, mscale, inverse);
    if (qt.defined()) qo._set_fw_grad(dq, 0, false);
    if (kt.defined()) ko._set_fw_grad(dk, 0, false);
  }
  return {qo, ko};
}

// rbln_attn::rotary_paged_kv_write: q [B, Hkv, G, S, D] rotated and returned,
// k rotated and v as it is written into the paged cache, as paged_kv_write
// writes them; positions seq[b] + s.
at::Tensor rotary_paged_kv_write_cuda(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                      at::Tensor& kcache, at::Tensor& vcache, const at::Tensor& seq_in,
                                      const at::Tensor& block_table_in, int64_t block_size,
                                      const at::Tensor& inv_freq_in, bool interleaved, double mscale,
                                      const std::optional<at::Tensor>& k_scale,
                                      const std::optional<at::Tensor>& v_scale) {
  const char* op = "rotary_paged_kv_write";
  TORCH_CHECK(q_in.is_cuda() && q_in.dim() == 5, op, ": q must be CUDA [B, Hkv, G, S, D]");
  const bool fp8 = kcache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || kcache.scalar_type() == q_in.scalar_type(), op, ": cache dtype must be q's or float8_e4m3fn");
  TORCH_CHECK(kcache.size(-1) == q_in.size(-1), op, ": cache head_dim differs from q's");
  Common c;
  fill_paged(c, op, q_in, k_in, v_in, kcache, vcache, seq_in, at::scalar_tensor(1.0, at::kFloat), block_table_in,
             block_size, std::nullopt, false);
  at::Tensor inv_freq = check_inv_freq(op, inv_freq_in, q_in);
  if (fp8) {
    TORCH_CHECK(k_scale.has_value() && v_scale.has_value(), op, ": fp8 caches need k_scale and v_scale");
    check_scales(op, kcache, *k_scale, *v_scale);
    c.p.k_scale = k_scale->data_ptr<float>();
    c.p.v_scale = v_scale->data_ptr<float>();
    c.p.scale_stride[0] = k_scale->stride(0);
    c.p.scale_stride[1] = k_scale->stride(1);
  }
  rbln_rotary_params_t r{};
  r.rotary_dim = (int32_t)(2 * inv_freq.numel());
  r.inv_freq = inv_freq.data_ptr<float>();
  r.interleaved = interleaved;
  r.mscale = (float)mscale;
  c10::cuda::CUDAGuard guard(c.q.device());
  check_rc(rbln_rotary_paged_kv_write(&c.p, &r, at::cuda::getCurrentCUDAStream(c.q.device().index()).stream()), op);
  check_device_flags(c, op);
  return c.out;
}

// rbln_attn::paged_kv_read: rows [0, lengths[b]) of every sequence as dense
// k, v [B, Hkv, 1, max_len, D], zeros behind them.
std::tuple<at::Tensor, at::Tensor> paged_kv_read_cuda(const at::Tensor& kcache, const at::Tensor& vcache,
                                                      const at::Tensor& lengths_in, const at::Tensor& block_table_in,
                                                      int64_t block_size, int64_t max_len,
                                                      const std::optional<at::Tensor>& k_scale,
                                                      const std::optional<at::Tensor>& v_scale,
                                                      std::optional<at::ScalarType> dtype) {
  const char* op = "paged_kv_read";
  TORCH_CHECK(kcache.is_cuda() && kcache.dim() == 5 && kcache.sizes() == vcache.sizes() &&
                  kcache.strides() == vcache.strides() && kcache.scalar_type() == vcache.scalar_type() &&
                  vcache.device() == kcache.device() && kcache.stride(-1) == 1 && kcache.size(2) == 1,
              op, ": caches must be CUDA [num_blocks, Hkv, 1, block_size, D], alike, with a contiguous last dim");
  TORCH_CHECK(kcache.size(3) == block_size, op, ": block_size ", block_size,
              " does not match the cache's block dimension ", kcache.size(3));
  const auto ct = kcache.scalar_type();
  const bool fp8 = ct == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || ct == at::kBFloat16 || ct == at::kHalf, op,
              ": caches must be bfloat16, float16 or float8_e4m3fn, got ", ct);
  const auto dt = dtype.has_value() ? *dtype : fp8 ? at::kBFloat16 : ct;
  TORCH_CHECK(is_float16or32(dt), op, ": dtype must be bfloat16, float16 or float32, got ", dt);
  TORCH_CHECK(max_len >= 0 && max_len <= INT32_MAX, op, ": max_len must be in [0, 2^31)");
  at::Tensor len = on_device(lengths_in, kcache).reshape({-1}).to(at::kInt).contiguous();
  const int64_t B = len.numel(), Hkv = kcache.size(1), D = kcache.size(-1);
  at::Tensor bt = on_device(block_table_in, kcache);
  if (bt.dim() == 1) bt = bt.unsqueeze(0);
  TORCH_CHECK(bt.dim() == 2 && (bt.size(0) == B || bt.size(0) == 1), op, ": block_table must be [B, max_blocks]");
  TORCH_CHECK(bt.scalar_type() == at::kShort || bt.scalar_type() == at::kInt || bt.scalar_type() == at::kLong, op,
              ": block_table must be int16/int32/int64");
  if (bt.stride(1) != 1) bt = bt.contiguous();
  rbln_paged_attn_params_t p{};
  p.batch = (int32_t)B;
  p.num_kv_heads = (int32_t)Hkv;
  p.group = 1;
  p.q_len = (int32_t)max_len;
  p.head_dim = (int32_t)D;
  p.num_blocks = (int32_t)kcache.size(0);
  p.block_size = (int32_t)block_size;
  p.max_blocks = (int32_t)bt.size(1);
  p.q_dtype = to_rbln_dtype(dt);
  p.kcache = kcache.data_ptr();
  p.vcache = vcache.data_ptr();
  p.kv_dtype = to_rbln_dtype(ct);
  p.cache_stride[0] = kcache.stride(0); p.cache_stride[1] = kcache.stride(1); p.cache_stride[2] = kcache.stride(3);
  if (fp8) {
    TORCH_CHECK(k_scale.has_value() && v_scale.has_value(), op, ": fp8 caches need k_scale and v_scale");
    check_scales(op, kcache, *k_scale, *v_scale);
    p.k_scale = k_scale->data_ptr<float>();
    p.v_scale = v_scale->data_ptr<float>();
    p.scale_stride[0] = k_scale->stride(0);
    p.scale_stride[1] = k_scale->stride(1);
  }
  p.seq = len.data_ptr<int32_t>();
  p.seq_stride = 1;
  p.block_table = bt.data_ptr();
  p.block_table_dtype = to_rbln_dtype(bt.scalar_type());
  p.block_table_stride = bt.size(0) == 1 ? 0 : bt.stride(0);
  c10::cuda::CUDAGuard guard(kcache.device());
  at::Tensor err;
  if (debug_checks()) {
    err = at::zeros({1}, kcache.options().dtype(at::kInt));
    p.error_flags = reinterpret_cast<uint32_t*>(err.data_ptr<int32_t>());
  }
  at::Tensor k = at::empty({B, Hkv, 1, max_len, D}, kcache.options().dtype(dt));
  at::Tensor v = at::empty({B, Hkv, 1, max_len, D}, kcache.options().dtype(dt));
  const int64_t os[3] = {k.stride(0), k.stride(1), k.stride(3)};
  check_rc(rbln_paged_kv_read(&p, k.data_ptr(), v.data_ptr(), os,
                              at::cuda::getCurrentCUDAStream(kcache.device().index()).stream()),
           op);
  if (err.defined()) {
    const int flags = err.item<int>();
    TORCH_CHECK(flags == 0, op, ": device-side input check failed (flags 0x", std::hex, flags, ")");
  }
  return {k, v};
}

// rbln_attn::paged_kv_write: the paged ops' append step on its own (k, v
// [B, Hkv, 1, S, D] at positions [seq[b], seq[b] + S)); fp8 caches take
// k_scale / v_scale [num_blocks, Hkv] and get per-(block, head) scales
// recomputed (rbln_paged_kv_write, kv_write.cu).
void paged_kv_write_cuda(const at::Tensor& k_in, const at::Tensor& v_in, at::Tensor& kcache, at::Tensor& vcache,
                         const at::Tensor& seq_in, const at::Tensor& block_table_in, int64_t block_size,
                         const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale) {
  const char* op = "paged_kv_write";
  TORCH_CHECK(k_in.is_cuda() && k_in.dim() == 5 && v_in.sizes() == k_in.sizes() && k_in.size(2) == 1, op,
              ": k/v must be CUDA [B, Hkv, 1, S, D]");
  TORCH_CHECK(kcache.dim() == 5 && kcache.sizes() == vcache.sizes() && kcache.strides() == vcache.strides() &&
                  kcache.stride(-1) == 1 && kcache.size(3) == block_size && kcache.device() == k_in.device() &&
                  vcache.device() == k_in.device() && v_in.device() == k_in.device(),
              op, ": caches must be [num_blocks, Hkv, 1, block_size, D] on k's and v's device, alike");
  const auto dt = k_in.scalar_type();
  TORCH_CHECK((dt == at::kBFloat16 || dt == at::kHalf) && v_in.scalar_type() == dt, op, ": k/v bf16 or f16");
  const bool fp8 = kcache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || kcache.scalar_type() == dt, op, ": cache dtype must be k's or float8_e4m3fn");
  TORCH_CHECK(vcache.scalar_type() == kcache.scalar_type(), op, ": kcache and vcache dtypes differ");
  at::Tensor k = k_in.contiguous(), v = v_in.contiguous();
  const int64_t B = k.size(0), Hkv = k.size(1), S = k.size(3), D = k.size(4);
  TORCH_CHECK(kcache.size(1) == Hkv && kcache.size(-1) == D, op, ": cache heads / head_dim differ from k's");
  at::Tensor seq = on_device(seq_in, k).reshape({-1}).to(at::kInt).contiguous();
  TORCH_CHECK(seq.numel() == B, op, ": seq must hold one entry per sequence");
  at::Tensor bt = on_device(block_table_in, k);
  if (bt.dim() == 1) bt = bt.unsqueeze(0);
  TORCH_CHECK(bt.dim() == 2 && (bt.size(0) == B || bt.size(0) == 1), op, ": block_table must be [B, max_blocks]");
  if (bt.stride(1) != 1) bt = bt.contiguous();
  rbln_paged_attn_params_t p{};
  p.batch = (int32_t)B;
  p.num_kv_heads = (int32_t)Hkv;
  p.group = 1;
  p.q_len = (int32_t)S;
  p.head_dim = (int32_t)D;
  p.num_blocks = (int32_t)kcache.size(0);
  p.block_size = (int32_t)block_size;
  p.max_blocks = (int32_t)bt.size(1);
  p.q_dtype = to_rbln_dtype(dt);
  p.k_new = k.data_ptr();
  p.v_new = v.data_ptr();
  p.k_new_stride[0] = k.stride(0); p.k_new_stride[1] = k.stride(1); p.k_new_stride[2] = k.stride(3);
  p.v_new_stride[0] = v.stride(0); p.v_new_stride[1] = v.stride(1); p.v_new_stride[2] = v.stride(3);
  p.kcache = kcache.data_ptr();
  p.vcache = vcache.data_ptr();
  p.kv_dtype = to_rbln_dtype(kcache.scalar_type());
  p.cache_stride[0] = kcache.stride(0); p.cache_stride[1] = kcache.stride(1); p.cache_stride[2] = kcache.stride(3);
  if (fp8) {
    TORCH_CHECK(k_scale.has_value() && v_scale.has_value() && k_scale->scalar_type() == at::kFloat &&
                    v_scale->scalar_type() == at::kFloat && k_scale->dim() == 2 &&
                    k_scale->size(0) == kcache.size(0) && k_scale->size(1) == Hkv &&
                    v_scale->sizes() == k_scale->sizes() && v_scale->strides() == k_scale->strides() &&
                    k_scale->device() == k.device() && v_scale->device() == k.device(),
                op, ": fp8 caches need float32 k_scale / v_scale [num_blocks, Hkv] on the caches' device");
    p.k_scale = k_scale->data_ptr<float>();
    p.v_scale = v_scale->data_ptr<float>();
    p.scale_stride[0] = k_scale->stride(0);
    p.scale_stride[1] = k_scale->stride(1);
  }
  p.seq = seq.data_ptr<int32_t>();
  p.seq_stride = 1;
  p.block_table = bt.data_ptr();
  p.block_table_dtype = to_rbln_dtype(bt.scalar_type());
  p.block_table_stride = bt.size(0) == 1 ? 0 : bt.stride(0);
  at::Tensor err;
  if (debug_checks()) {
    err = at::zeros({1}, k.options().dtype(at::kInt));
    p.error_flags = reinterpret_cast<uint32_t*>(err.data_ptr<int32_t>());
  }
  c10::cuda::CUDAGuard guard(k.device());
  check_rc(rbln_paged_kv_write(&p, at::cuda::getCurrentCUDAStream(k.device().index()).stream()), op);
  if (err.defined()) {
    const int flags = err.item<int>();
    TORCH_CHECK(flags == 0, op, ": device-side input check failed (flags 0x", std::hex, flags, ")");
  }
}

// ---------------------------------------------------------------------------
// Pages that several sequences share (pages.cu): the caller's state is one
// block table for all layers and refs, how many of its entries hold each page.
// ---------------------------------------------------------------------------
bool is_index(at::ScalarType t) { return t == at::kShort || t == at::kInt || t == at::kLong; }

// A table that the call writes must hold every entry at a place of its own.
rbln_pages_params_t check_pages(const char* op, const at::Tensor& block_table, const at::Tensor& refs,
                                int64_t block_size, bool written) {
  TORCH_CHECK(block_table.is_cuda(), op, ": expected CUDA tensors, block_table is on ", block_table.device());
  TORCH_CHECK(block_table.dim() == 2 && is_index(block_table.scalar_type()), op,
              ": block_table must be [B, max_blocks] of int16/int32/int64, got ", block_table.sizes(), " of ",
              block_table.scalar_type());
  TORCH_CHECK(!written || at::has_internal_overlap(block_table) != at::MemOverlap::Yes, op,
              ": block_table is written and must not be expanded");
  TORCH_CHECK(refs.dim() == 1 && refs.scalar_type() == at::kInt && refs.is_contiguous(), op,
              ": refs must be contiguous int32 [num_blocks], got ", refs.sizes(), " of ", refs.scalar_type());
  TORCH_CHECK(refs.device() == block_table.device(), op, ": refs must be on block_table's device");
  TORCH_CHECK(block_size > 0 && block_size <= INT32_MAX, op, ": block_size must be positive, got ", block_size);
  TORCH_CHECK(block_table.size(0) <= INT32_MAX && refs.numel() <= INT32_MAX &&
                  block_table.size(1) <= INT32_MAX / block_size,
              op, ": block_table spans 2^31 positions or more");
  TORCH_CHECK(block_table.scalar_type() != at::kShort || refs.numel() <= 32768, op,
              ": an int16 block_table cannot name ", refs.numel(), " blocks");
  rbln_pages_params_t p{};
  p.batch = (int32_t)block_table.size(0);
  p.max_blocks = (int32_t)block_table.size(1);
  p.num_blocks = (int32_t)refs.numel();
  p.block_size = (int32_t)block_size;
  p.block_table = block_table.data_ptr();
  p.block_table_dtype = to_rbln_dtype(block_table.scalar_type());
  p.block_table_stride[0] = block_table.stride(0);
  p.block_table_stride[1] = block_table.stride(1);
  p.refs = refs.data_ptr<int32_t>();
  p.lengths_dtype = RBLN_DT_I32;
  return p;
}

// One whole number a row of the table, kept alive by the caller.
at::Tensor check_lengths(const char* op, const char* name, const at::Tensor& lengths_in, const at::Tensor& block_table,
                         rbln_pages_params_t& p) {
  at::Tensor n = on_device(lengths_in, block_table);
  if (n.dim() != 1) n = n.reshape({-1});
  TORCH_CHECK(is_index(n.scalar_type()), op, ": ", name, " must be int16/int32/int64, got ", n.scalar_type());
  TORCH_CHECK(n.numel() == block_table.size(0), op, ": ", name, " must hold one entry per row, got ",
              lengths_in.sizes(), " for ", block_table.sizes());
  p.lengths = n.data_ptr();
  p.lengths_dtype = to_rbln_dtype(n.scalar_type());
  p.lengths_stride = n.stride(0);
  return n;
}

struct LayerPointers {
  std::vector<void*> k, v;
  std::vector<float*> ks, vs;
};
using TensorLists = std::optional<std::vector<at::Tensor>>;

// The caches of all layers, alike, [num_blocks, Hkv, 1, block_size, D]; their
// number of blocks is refs'. Scales go with float8_e4m3fn caches only.
void check_layers(const char* op, at::TensorList kcaches, at::TensorList vcaches, const TensorLists& k_scales,
                  const TensorLists& v_scales, const at::Tensor& block_table, rbln_pages_params_t& p,
                  LayerPointers& ptrs) {
  TORCH_CHECK(!kcaches.empty() && kcaches.size() == vcaches.size(), op,
              ": kcaches and vcaches must hold one cache for each layer, got ", kcaches.size(), " and ",
              vcaches.size());
  const at::Tensor& c = kcaches[0];
  const auto ct = c.scalar_type();
  const bool fp8 = ct == at::kFloat8_e4m3fn;
  TORCH_CHECK(c.dim() == 5 && c.size(2) == 1 && c.stride(-1) == 1, op,
              ": caches must be [num_blocks, Hkv, 1, block_size, D] with a contiguous last dim, got ", c.sizes());
  TORCH_CHECK(fp8 || ct == at::kBFloat16 || ct == at::kHalf, op,
              ": caches must be bfloat16, float16 or float8_e4m3fn, got ", ct);
  TORCH_CHECK(c.size(0) == p.num_blocks, op, ": caches hold ", c.size(0), " blocks, refs ", p.num_blocks);
  TORCH_CHECK(c.size(1) > 0 && c.size(-1) > 0 && c.size(-1) % 64 == 0, op,
              ": the last dimension of a cache must be a multiple of 64, but got shape ", c.sizes());
  TORCH_CHECK(at::has_internal_overlap(c) != at::MemOverlap::Yes, op, ": caches are written and must not be expanded");
  for (const at::TensorList list : {kcaches, vcaches})
    for (const at::Tensor& t : list) {
      TORCH_CHECK(t.device() == block_table.device(), op, ": caches must be on block_table's device");
      TORCH_CHECK(t.sizes() == c.sizes() && t.strides() == c.strides() && t.scalar_type() == ct, op,
                  ": all caches must match in shape, strides and dtype");
    }
  TORCH_CHECK(k_scales.has_value() == fp8 && v_scales.has_value() == fp8, op,
              ": k_scales and v_scales go with float8_e4m3fn caches, and only with them");
  p.num_layers = (int32_t)kcaches.size();
  p.num_kv_heads = (int32_t)c.size(1);
  p.head_dim = (int32_t)c.size(-1);
  p.kv_dtype = to_rbln_dtype(ct);
  p.block_size = (int32_t)c.size(3);
  p.cache_stride[0] = c.stride(0);
  p.cache_stride[1] = c.stride(1);
  p.cache_stride[2] = c.stride(3);
  ptrs.k.reserve(kcaches.size());
  ptrs.v.reserve(kcaches.size());
  for (size_t i = 0; i < kcaches.size(); ++i) {
    ptrs.k.push_back(kcaches[i].data_ptr());
    ptrs.v.push_back(vcaches[i].data_ptr());
  }
  p.kcaches = ptrs.k.data();
  p.vcaches = ptrs.v.data();
  if (!fp8) return;
  TORCH_CHECK(k_scales->size() == kcaches.size() && v_scales->size() == kcaches.size(), op,
              ": k_scales and v_scales must hold one tensor for each layer");
  for (size_t i = 0; i < kcaches.size(); ++i) {
    check_scales(op, c, (*k_scales)[i], (*v_scales)[i]);
    TORCH_CHECK((*k_scales)[i].strides() == (*k_scales)[0].strides(), op, ": all scales must match in strides");
    ptrs.ks.push_back((*k_scales)[i].data_ptr<float>());
    ptrs.vs.push_back((*v_scales)[i].data_ptr<float>());
  }
  p.k_scales = ptrs.ks.data();
  p.v_scales = ptrs.vs.data();
  p.scale_stride[0] = (*k_scales)[0].stride(0);
  p.scale_stride[1] = (*k_scales)[0].stride(1);
}

at::Tensor pages_workspace(const char* op, rbln_pages_params_t& p, int64_t new_tokens, const at::Tensor& like) {
  size_t bytes = 0;
  check_rc(rbln_paged_kv_pages_workspace_size(&p, (int32_t)new_tokens, &bytes), op);
  at::Tensor w = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
  p.workspace = w.data_ptr();
  p.workspace_bytes = bytes;
  return w;
}

cudaStream_t stream_of(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// rbln_attn::paged_kv_fork: rows parents[i] of the table as rows of a new one,
// their pages shared and counted.
std::tuple<at::Tensor, at::Tensor> paged_kv_fork_cuda(const at::Tensor& block_table, const at::Tensor& lengths_in,
                                                      const at::Tensor& parents_in, at::Tensor& refs,
                                                      int64_t block_size) {
  const char* op = "paged_kv_fork";
  rbln_pages_params_t p = check_pages(op, block_table, refs, block_size, false);
  c10::cuda::CUDAGuard guard(block_table.device());
  const at::Tensor lengths = check_lengths(op, "lengths", lengths_in, block_table, p);
  const at::Tensor parents = on_device(parents_in, block_table);
  TORCH_CHECK(parents.dim() == 1 && is_index(parents.scalar_type()), op,
              ": parents must be 1-D of int16/int32/int64, got ", parents.sizes(), " of ", parents.scalar_type());
  const int64_t N = parents.numel();
  TORCH_CHECK(N + p.batch <= INT32_MAX, op, ": too many forks");
  at::Tensor table = at::empty({N, block_table.size(1)}, block_table.options());
  at::Tensor out_lengths = at::empty({N}, lengths.options());
  check_rc(rbln_paged_kv_fork(&p, parents.data_ptr(), to_rbln_dtype(parents.scalar_type()),
                              N > 0 ? parents.stride(0) : 1, (int32_t)N, table.data_ptr(), table.stride(0),
                              out_lengths.data_ptr(), stream_of(block_table)),
           op);
  return {table, out_lengths};
}

// rbln_attn::paged_kv_free: the pages behind the first keep[b] positions of
// every row go back.
void paged_kv_free_cuda(at::Tensor& block_table, const at::Tensor& keep_in, at::Tensor& refs, int64_t block_size) {
  const char* op = "paged_kv_free";
  rbln_pages_params_t p = check_pages(op, block_table, refs, block_size, true);
  c10::cuda::CUDAGuard guard(block_table.device());
  const at::Tensor keep = check_lengths(op, "keep", keep_in, block_table, p);
  check_rc(rbln_paged_kv_free(&p, stream_of(block_table)), op);
}

// rbln_attn::paged_kv_reserve: pages of their own for every row's next
// new_tokens positions; returns how many of them may be written.
at::Tensor paged_kv_reserve_cuda(at::TensorList kcaches, at::TensorList vcaches, at::Tensor& block_table,
                                 const at::Tensor& seq_in, at::Tensor& refs, int64_t block_size, int64_t new_tokens,
                                 const TensorLists& k_scales, const TensorLists& v_scales) {
  const char* op = "paged_kv_reserve";
  rbln_pages_params_t p = check_pages(op, block_table, refs, block_size, true);
  LayerPointers ptrs;
  check_layers(op, kcaches, vcaches, k_scales, v_scales, block_table, p, ptrs);
  TORCH_CHECK(p.block_size == block_size, op, ": block_size ", block_size,
              " does not match the cache's block dimension ", p.block_size);
  TORCH_CHECK(new_tokens >= 0 && new_tokens <= INT32_MAX, op, ": new_tokens must be in [0, 2^31), got ", new_tokens);
  c10::cuda::CUDAGuard guard(block_table.device());
  const at::Tensor seq = check_lengths(op, "seq", seq_in, block_table, p);
  at::Tensor granted = at::empty({block_table.size(0)}, block_table.options().dtype(at::kInt));
  const at::Tensor workspace = pages_workspace(op, p, new_tokens, block_table);
  check_rc(rbln_paged_kv_reserve(&p, (int32_t)new_tokens, granted.data_ptr<int32_t>(), stream_of(block_table)), op);
  return granted;
}

// rbln_attn::paged_kv_compact: pages in use moved to the front of the pool;
// returns where each went and how many there are.
std::tuple<at::Tensor, at::Tensor> paged_kv_compact_cuda(at::TensorList kcaches, at::TensorList vcaches,
                                                         at::Tensor& block_table, at::Tensor& refs,
                                                         const TensorLists& k_scales, const TensorLists& v_scales) {
  const char* op = "paged_kv_compact";
  TORCH_CHECK(!kcaches.empty() && kcaches[0].dim() == 5, op, ": kcaches must hold [num_blocks, Hkv, 1, block_size, D]");
  rbln_pages_params_t p = check_pages(op, block_table, refs, kcaches[0].size(3), true);
  LayerPointers ptrs;
  check_layers(op, kcaches, vcaches, k_scales, v_scales, block_table, p, ptrs);
  c10::cuda::CUDAGuard guard(block_table.device());
  at::Tensor moved = at::empty_like(refs);
  at::Tensor live = at::empty({1}, refs.options());
  const at::Tensor workspace = pages_workspace(op, p, -1, block_table);
  check_rc(rbln_paged_kv_compact(&p, moved.data_ptr<int32_t>(), live.data_ptr<int32_t>(), stream_of(block_table)), op);
  return {moved, live};
}

// ---------------------------------------------------------------------------
// flash_attention_naive_{prefill,decode}: the unified-cache form of the paged
// ops (torch_rbln/_internal/register_custom_ops.py:453-560; CPU semantics in
// test/rbln/test_custom_kernel.py:546-573). kv_cache [2, num_blocks, Hkv, 1,
// P, D] stacks the K pool (index 0) and the V pool (index 1), each block one
// partition of P tokens; block_tables lists a sequence's partitions (1-D for
// prefill, [B, NP] for decode); seq_idx [B, 1] is the position of the first
// new token; mask is a keep-mask over partition positions. The new rows are
// written at seq_idx through the block table and attention runs over the
// mask's positions: the keep-mask paged path on kv_cache[0] / kv_cache[1].
// slot_mapping is accepted for the schema and not read (the positions follow
// from seq_idx and block_tables, as in the reference's CPU semantics).
// sinks [Hkv * G] (any float dtype) are per-query-head sink logits.
// ---------------------------------------------------------------------------
at::Tensor flash_attention_naive(const char* op, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                 at::Tensor& kv_cache, const at::Tensor& mask, const at::Tensor& scale,
                                 const at::Tensor& seq_idx, const at::Tensor& block_tables,
                                 const at::Tensor& slot_mapping, const std::optional<at::Tensor>& sinks,
                                 bool decode) {
  TORCH_CHECK(kv_cache.dim() == 6 && kv_cache.size(0) == 2, op,
              ": kv_cache must be [2, num_blocks, Hkv, 1, partition, D], got ", kv_cache.sizes());
  TORCH_CHECK(kv_cache.size(-1) % 64 == 0, op,
              ": The last dimension of kv_cache must be a multiple of 64, but got shape ", kv_cache.sizes());
  TORCH_CHECK(kv_cache.scalar_type() == q.scalar_type(), op, ": kv_cache dtype must equal q dtype");
  if (!decode)
    for (const at::Tensor* t : {&q, &k, &v})
      TORCH_CHECK(t->dim() >= 1 && t->size(0) == 1, op, " batch size of q/k/v must be 1, but got shape ",
                  t->sizes());
  TORCH_CHECK(slot_mapping.defined(), op, ": slot_mapping is required");
  at::Tensor kcache = kv_cache.select(0, 0);
  at::Tensor vcache = kv_cache.select(0, 1);
  // seq_idx [B, 1] (or [B]): one start position per sequence
  const at::Tensor seq = seq_idx.dim() == 2 ? seq_idx.select(1, 0) : seq_idx;
  Common c;
  fill_paged(c, op, q, k, v, kcache, vcache, seq, scale, block_tables, kv_cache.size(-2), mask, decode);
  if (sinks.has_value() && sinks->defined()) {
    TORCH_CHECK(at::isFloatingType(sinks->scalar_type()), op, ": sinks must be floating point");
    TORCH_CHECK(sinks->numel() == (int64_t)c.p.num_kv_heads * c.p.group, op, ": sinks must hold one logit per ",
                "query head (", c.p.num_kv_heads * c.p.group, "), got ", sinks->sizes());
    c.sinks = on_device(*sinks, c.q).to(at::kFloat).contiguous();
    c.p.sinks = c.sinks.data_ptr<float>();
  }
  return decode ? run_decode(c, kcache, op, true) : run_prefill(c, op, true);
}

at::Tensor flash_attention_naive_prefill_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                              at::Tensor& kv_cache, const at::Tensor& mask, const at::Tensor& scale,
                                              const at::Tensor& seq_idx, const at::Tensor& block_tables,
                                              const at::Tensor& slot_mapping,
                                              const std::optional<at::Tensor>& sinks) {
  return flash_attention_naive("flash_attention_naive_prefill", q, k, v, kv_cache, mask, scale, seq_idx,
                               block_tables, slot_mapping, sinks, false);
}

at::Tensor flash_attention_naive_decode_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                             at::Tensor& kv_cache, const at::Tensor& mask, const at::Tensor& scale,
                                             const at::Tensor& seq_idx, const at::Tensor& block_tables,
                                             const at::Tensor& slot_mapping,
                                             const std::optional<at::Tensor>& sinks) {
  return flash_attention_naive("flash_attention_naive_decode", q, k, v, kv_cache, mask, scale, seq_idx,
                               block_tables, slot_mapping, sinks, true);
}

// ---------------------------------------------------------------------------
// SDPA: aten::_scaled_dot_product_fused_attention_overrideable on CUDA, and
// the backend choice that routes F.scaled_dot_product_attention to it
// (mirrors _fused_sdp_choice_privateuse1, aten/src/ATen/native/
// RBLNRegisterOps.cpp:89-102, which picks "overrideable" for 4-D inputs).
// ---------------------------------------------------------------------------
std::atomic<bool> g_sdpa_route{[] {
  const char* e = std::getenv("RBLN_ATTN_SDPA");
  return !(e && std::string(e) == "0");
}()};

bool sm100_device(const at::Tensor& t) {
  if (!t.is_cuda()) return false;
  const auto* prop = at::cuda::getDeviceProperties(t.device().index());
  return prop->major == 10;
}

// The inputs the CUDA kernels here take; anything else goes to torch's own
// CUDA backends.
bool sdpa_supported(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                    const std::optional<at::Tensor>& mask, double dropout_p) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4) return false;
  if (q.is_nested() || k.is_nested() || v.is_nested()) return false;
  const auto dt = q.scalar_type();
  if (dt != at::kBFloat16 && dt != at::kHalf && dt != at::kFloat) return false;
  if (k.scalar_type() != dt || v.scalar_type() != dt) return false;
  if (k.device() != q.device() || v.device() != q.device() || !sm100_device(q)) return false;
  const int64_t D = q.size(3);
  if ((D != 64 && D != 128) || k.size(3) != D || v.size(3) != D) return false;
  if (k.size(0) != q.size(0) || v.size(0) != q.size(0) || k.size(1) != v.size(1) || k.size(2) != v.size(2))
    return false;
  if (k.size(1) == 0 || q.size(1) % k.size(1) != 0) return false;
  if (q.numel() == 0 || k.numel() == 0) return false;
  if (dropout_p > 0.0) return false;
  // the backward (sdpa_bwd.cu) runs on the tensor cores: bf16 / f16 only
  const bool grad = c10::GradMode::is_enabled() &&
                    (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                     (mask.has_value() && mask->defined() && mask->requires_grad()));
  if (grad && dt == at::kFloat) return false;
  if (mask.has_value() && mask->defined()) {
    const auto& m = *mask;
    if (m.dim() < 2 || m.dim() > 4 || m.device() != q.device()) return false;
    if (m.scalar_type() != at::kBool && !at::isFloatingType(m.scalar_type())) return false;
  }
  return true;
}

int64_t fused_sdp_choice_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                              const std::optional<at::Tensor>& mask, double dropout_p, bool is_causal,
                              std::optional<double> scale, bool enable_gqa) {
  if (g_sdpa_route.load() && at::globalContext().userEnabledOverrideableSDP() &&
      sdpa_supported(q, k, v, mask, dropout_p))
    return static_cast<int64_t>(at::SDPBackend::overrideable);
  return at::native::_fused_sdp_choice_cuda(q, k, v, mask, dropout_p, is_causal, scale, enable_gqa);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, c10::SymInt, c10::SymInt, at::Tensor, at::Tensor,
           at::Tensor>
sdpa_overrideable_cuda(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
                       const std::optional<at::Tensor>& attn_bias, double dropout_p, bool is_causal,
                       bool return_debug_mask, std::optional<double> scale) {
  // input validation as in the reference (sdpa.py:85-119): ValueError
  TORCH_CHECK_VALUE(query.scalar_type() == key.scalar_type() && query.scalar_type() == value.scalar_type(),
                    "Expected query, key, and value to have the same dtype, but got query.dtype: ",
                    query.scalar_type(), ", key.dtype: ", key.scalar_type(), ", and value.dtype: ",
                    value.scalar_type(), " instead.");
  TORCH_CHECK_VALUE(query.device() == key.device() && query.device() == value.device(),
                    "Expected query, key, and value to have the same device type, but got query.device: ",
                    query.device(), ", key.device: ", key.device(), ", and value.device: ", value.device(),
                    " instead.");
  if (attn_bias.has_value() && attn_bias->defined()) {
    TORCH_CHECK_VALUE(attn_bias->scalar_type() == at::kBool || at::isFloatingType(attn_bias->scalar_type()),
                      "Expected attn_mask to have dtype bool or floating point, but got attn_mask.dtype: ",
                      attn_bias->scalar_type(), " instead.");
    TORCH_CHECK_VALUE(attn_bias->device() == query.device(),
                      "Expected attn_mask to have the same device as query, but got attn_mask.device: ",
                      attn_bias->device(), " and query.device: ", query.device(), " instead.");
  }
  TORCH_CHECK(sdpa_supported(query, key, value, attn_bias, dropout_p),
              "_scaled_dot_product_fused_attention_overrideable (CUDA, sm_100a): unsupported inputs "
              "(need 4-D bf16/f16/f32 q/k/v with head_dim 64 or 128, Hq % Hkv == 0, no dropout; "
              "bf16/f16 when a gradient is needed)");
  c10::cuda::CUDAGuard guard(query.device());
  auto inner = [](const at::Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); };
  at::Tensor q = inner(query), k = inner(key), v = inner(value);
  const int64_t B = q.size(0), H = q.size(1), L = q.size(2), D = q.size(3);
  const int64_t Hkv = k.size(1), S = k.size(2);
  at::Tensor out = at::empty({B, H, L, D}, q.options());
  at::Tensor lse = at::empty({B, H, L}, q.options().dtype(at::kFloat));
  rbln_sdpa_params_t p{};
  p.batch = (int32_t)B;
  p.num_heads = (int32_t)H;
  p.num_kv_heads = (int32_t)Hkv;
  p.q_len = (int32_t)L;
  p.kv_len = (int32_t)S;
  p.head_dim = (int32_t)D;
  p.dtype = to_rbln_dtype(q.scalar_type());
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.out = out.data_ptr();
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = q.stride(i);
    p.k_stride[i] = k.stride(i);
    p.v_stride[i] = v.stride(i);
    p.out_stride[i] = out.stride(i);
    p.lse_stride[i] = lse.stride(i);
  }
  p.lse = lse.data_ptr<float>();
  at::Tensor m;
  if (attn_bias.has_value() && attn_bias->defined()) {
    m = *attn_bias;
    if (m.scalar_type() != at::kBool && m.scalar_type() != at::kFloat && m.scalar_type() != at::kHalf &&
        m.scalar_type() != at::kBFloat16)
      m = m.to(at::kFloat);
    while (m.dim() < 4) m = m.unsqueeze(0);
    m = m.expand({B, H, L, S});
    if (m.stride(3) != 1 && q.scalar_type() != at::kFloat) m = m.contiguous();
    p.mask = m.data_ptr();
    p.mask_dtype = to_rbln_dtype(m.scalar_type());
    p.mask_additive = m.scalar_type() == at::kBool ? 0 : 1;
    for (int i = 0; i < 4; ++i) p.mask_stride[i] = m.stride(i);
  }
  p.causal = is_causal ? 1 : 0;
  p.scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)D));
  at::Tensor err;
  if (debug_checks()) {
    err = at::zeros({1}, q.options().dtype(at::kInt));
    p.error_flags = reinterpret_cast<uint32_t*>(err.data_ptr<int32_t>());
  }
  auto stream = at::cuda::getCurrentCUDAStream(q.device().index());
  check_rc(rbln_sdpa_fwd(&p, stream.stream()), "_scaled_dot_product_fused_attention_overrideable");
  if (err.defined()) {
    const int flags = err.item<int>();
    TORCH_CHECK(flags == 0, "_scaled_dot_product_fused_attention_overrideable: device error flags 0x", std::hex,
                flags);
  }
  at::Tensor debug = return_debug_mask ? at::empty({B, H, L, S}, q.options().dtype(at::kFloat))
                                       : at::empty({0}, q.options().dtype(at::kFloat));
  at::Tensor cum_q = at::empty({0}, q.options().dtype(at::kLong));
  at::Tensor cum_k = at::empty({0}, q.options().dtype(at::kLong));
  at::Tensor seed = at::empty({}, at::TensorOptions().dtype(at::kLong).device(at::kCPU));
  at::Tensor offset = at::empty({}, at::TensorOptions().dtype(at::kLong).device(at::kCPU));
  return {out, lse, cum_q, cum_k, c10::SymInt(L), c10::SymInt(S), seed, offset, debug};
}

// aten::_scaled_dot_product_fused_attention_overrideable_backward on CUDA
// (reference sdpa.py:754-821): dq, dk, dv as grad_input_mask asks, and
// grad_attn_bias for a floating-point mask (full [B, H, L, S], in the mask's
// dtype; autograd sums it down to the mask's broadcast shape). P is
// recomputed from q, k and the forward's logsumexp.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> sdpa_overrideable_backward_cuda(
    const at::Tensor& grad_out, const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
    const at::Tensor& attn_bias, std::array<bool, 4> grad_input_mask, const at::Tensor& out,
    const at::Tensor& logsumexp, const at::Tensor& cum_seq_q, const at::Tensor& cum_seq_k, c10::SymInt max_q,
    c10::SymInt max_k, double dropout_p, bool is_causal, const at::Tensor& philox_seed,
    const at::Tensor& philox_offset, std::optional<double> scale) {
  const char* op = "_scaled_dot_product_fused_attention_overrideable_backward";
  TORCH_CHECK(dropout_p == 0.0, op, ": dropout is not supported");
  TORCH_CHECK(query.dim() == 4 && key.dim() == 4 && value.dim() == 4 && grad_out.dim() == 4 && out.dim() == 4, op,
              ": expected 4-D tensors");
  const auto dt = query.scalar_type();
  TORCH_CHECK(dt == at::kBFloat16 || dt == at::kHalf, op, ": bf16 / f16 only, got ", dt);
  TORCH_CHECK(key.scalar_type() == dt && value.scalar_type() == dt && grad_out.scalar_type() == dt &&
                  out.scalar_type() == dt,
              op, ": q, k, v, out and grad_out must share a dtype");
  for (const at::Tensor* t : {&key, &value, &grad_out, &out, &logsumexp, &attn_bias})
    TORCH_CHECK(!t->defined() || t->numel() == 0 || t->device() == query.device(), op,
                ": all tensors must be on query's device, got ", t->device(), " beside ", query.device());
  c10::cuda::CUDAGuard guard(query.device());
  // last dim contiguous and 16-byte aligned rows
  auto rows16 = [](const at::Tensor& t) {
    const bool ok = t.stride(-1) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0 &&
                    (t.stride(0) * 2) % 16 == 0 && (t.stride(1) * 2) % 16 == 0 && (t.stride(2) * 2) % 16 == 0;
    return ok ? t : t.contiguous();
  };
  at::Tensor q = rows16(query), k = rows16(key), v = rows16(value), o = rows16(out), dout = rows16(grad_out);
  const int64_t B = q.size(0), H = q.size(1), L = q.size(2), D = q.size(3);
  const int64_t Hkv = k.size(1), S = k.size(2);
  TORCH_CHECK(logsumexp.defined() && logsumexp.dim() == 3 && logsumexp.size(0) == B && logsumexp.size(1) == H &&
                  logsumexp.size(2) == L && logsumexp.scalar_type() == at::kFloat,
              op, ": logsumexp must be the forward's fp32 [B, H, L]");
  at::Tensor lse = logsumexp;
  at::Tensor dq = grad_input_mask[0] ? at::empty_like(q, at::MemoryFormat::Contiguous) : at::Tensor();
  at::Tensor dk = grad_input_mask[1] ? at::empty_like(k, at::MemoryFormat::Contiguous) : at::Tensor();
  at::Tensor dv = grad_input_mask[2] ? at::empty_like(v, at::MemoryFormat::Contiguous) : at::Tensor();
  rbln_sdpa_bwd_params_t p{};
  p.batch = (int32_t)B;
  p.num_heads = (int32_t)H;
  p.num_kv_heads = (int32_t)Hkv;
  p.q_len = (int32_t)L;
  p.kv_len = (int32_t)S;
  p.head_dim = (int32_t)D;
  p.dtype = to_rbln_dtype(dt);
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.out = o.data_ptr();
  p.dout = dout.data_ptr();
  p.lse = lse.data_ptr<float>();
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = q.stride(i);
    p.k_stride[i] = k.stride(i);
    p.v_stride[i] = v.stride(i);
    p.out_stride[i] = o.stride(i);
    p.dout_stride[i] = dout.stride(i);
    p.lse_stride[i] = lse.stride(i);
    if (dq.defined()) p.dq_stride[i] = dq.stride(i);
    if (dk.defined()) p.dk_stride[i] = dk.stride(i);
    if (dv.defined()) p.dv_stride[i] = dv.stride(i);
  }
  p.dq = dq.defined() ? dq.data_ptr() : nullptr;
  p.dk = dk.defined() ? dk.data_ptr() : nullptr;
  p.dv = dv.defined() ? dv.data_ptr() : nullptr;
  at::Tensor m, dbias;
  if (attn_bias.defined() && attn_bias.numel() > 0) {  // an empty tensor means no mask (sdpa.py:800)
    m = attn_bias;
    TORCH_CHECK(m.scalar_type() == at::kBool || at::isFloatingType(m.scalar_type()), op,
                ": attn_bias must be bool or floating point");
    if (m.scalar_type() != at::kBool && m.scalar_type() != at::kFloat && m.scalar_type() != at::kHalf &&
        m.scalar_type() != at::kBFloat16)
      m = m.to(at::kFloat);
    while (m.dim() < 4) m = m.unsqueeze(0);
    m = m.expand({B, H, L, S});
    if (m.stride(3) != 1) m = m.contiguous();
    p.mask = m.data_ptr();
    p.mask_dtype = to_rbln_dtype(m.scalar_type());
    p.mask_additive = m.scalar_type() == at::kBool ? 0 : 1;
    for (int i = 0; i < 4; ++i) p.mask_stride[i] = m.stride(i);
    if (grad_input_mask[3] && m.scalar_type() != at::kBool) {
      dbias = at::empty({B, H, L, S}, q.options().dtype(at::kFloat));
      p.dbias = dbias.data_ptr<float>();
    }
  }
  p.causal = is_causal ? 1 : 0;
  p.scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)D));
  size_t ws = 0;
  check_rc(rbln_sdpa_bwd_workspace_size(&p, &ws), op);
  at::Tensor wst = at::empty({(int64_t)std::max<size_t>(ws, 16)}, q.options().dtype(at::kByte));
  p.workspace = wst.data_ptr();
  p.workspace_bytes = ws;
  at::Tensor err;
  if (debug_checks()) {
    err = at::zeros({1}, q.options().dtype(at::kInt));
    p.error_flags = reinterpret_cast<uint32_t*>(err.data_ptr<int32_t>());
  }
  auto stream = at::cuda::getCurrentCUDAStream(q.device().index());
  check_rc(rbln_sdpa_bwd(&p, stream.stream()), op);
  if (err.defined()) {
    const int flags = err.item<int>();
    TORCH_CHECK(flags == 0, op, ": device error flags 0x", std::hex, flags);
  }
  at::Tensor gbias;
  if (dbias.defined()) gbias = dbias.to(attn_bias.scalar_type());
  return {dq, dk, dv, gbias};
}

void set_sdpa_route(bool enabled) { g_sdpa_route.store(enabled); }
bool sdpa_route_enabled() { return g_sdpa_route.load(); }

}  // namespace

TORCH_LIBRARY(rbln_attn, m) {
  m.def("set_sdpa_route(bool enabled) -> ()");
  m.def("sdpa_route_enabled() -> bool");
  m.def(
      "paged_kv_write(Tensor k, Tensor v, Tensor(a!) kcache, Tensor(b!) vcache, Tensor seq, Tensor block_table, "
      "SymInt block_size, Tensor(c!)? k_scale=None, Tensor(d!)? v_scale=None) -> ()");
  m.def(
      "rotary(Tensor q, Tensor k, Tensor positions, Tensor inv_freq, bool interleaved=False, float mscale=1.0, "
      "bool inverse=False) -> (Tensor, Tensor)");
  m.def(
      "rotary_paged_kv_write(Tensor q, Tensor k, Tensor v, Tensor(a!) kcache, Tensor(b!) vcache, Tensor seq, "
      "Tensor block_table, SymInt block_size, Tensor inv_freq, bool interleaved=False, float mscale=1.0, "
      "Tensor(c!)? k_scale=None, Tensor(d!)? v_scale=None) -> Tensor");
  m.def(
      "paged_kv_read(Tensor kcache, Tensor vcache, Tensor lengths, Tensor block_table, SymInt block_size, "
      "SymInt max_len, Tensor? k_scale=None, Tensor? v_scale=None, ScalarType? dtype=None) -> (Tensor, Tensor)");
  m.def(
      "paged_kv_fork(Tensor block_table, Tensor lengths, Tensor parents, Tensor(a!) refs, SymInt block_size) -> "
      "(Tensor, Tensor)");
  m.def("paged_kv_free(Tensor(a!) block_table, Tensor keep, Tensor(b!) refs, SymInt block_size) -> ()");
  m.def(
      "paged_kv_reserve(Tensor(a!)[] kcaches, Tensor(b!)[] vcaches, Tensor(c!) block_table, Tensor seq, "
      "Tensor(d!) refs, SymInt block_size, SymInt new_tokens, Tensor(e!)[]? k_scales=None, "
      "Tensor(f!)[]? v_scales=None) -> Tensor");
  m.def(
      "paged_kv_compact(Tensor(a!)[] kcaches, Tensor(b!)[] vcaches, Tensor(c!) block_table, Tensor(d!) refs, "
      "Tensor(e!)[]? k_scales=None, Tensor(f!)[]? v_scales=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(rbln_attn, CUDA, m) {
  m.impl("paged_kv_write", &paged_kv_write_cuda);
  m.impl("rotary", &rotary_cuda);
  m.impl("rotary_paged_kv_write", &rotary_paged_kv_write_cuda);
  m.impl("paged_kv_read", &paged_kv_read_cuda);
  m.impl("paged_kv_fork", &paged_kv_fork_cuda);
  m.impl("paged_kv_free", &paged_kv_free_cuda);
  m.impl("paged_kv_reserve", &paged_kv_reserve_cuda);
  m.impl("paged_kv_compact", &paged_kv_compact_cuda);
}

TORCH_LIBRARY_IMPL(rbln_attn, AutogradCUDA, m) { m.impl("rotary", &rotary_autograd); }

TORCH_LIBRARY_IMPL(rbln_attn, CompositeExplicitAutograd, m) {
  m.impl("set_sdpa_route", &set_sdpa_route);
  m.impl("sdpa_route_enabled", &sdpa_route_enabled);
}

TORCH_LIBRARY_IMPL(aten, CUDA, m) {
  m.impl("_fused_sdp_choice", &fused_sdp_choice_cuda);
  m.impl("_scaled_dot_product_fused_attention_overrideable", &sdpa_overrideable_cuda);
  m.impl("_scaled_dot_product_fused_attention_overrideable_backward", &sdpa_overrideable_backward_cuda);
}

TORCH_LIBRARY(rbln_custom_ops, m) {
  m.def(
      "paged_attn_prefill(Tensor q, Tensor k, Tensor v, Tensor mask, Tensor(a4!) kcache, Tensor(a5!) vcache, "
      "Tensor seq, Tensor scale, Tensor block_table, SymInt block_size) -> Tensor");
  m.def(
      "paged_attn_decode(Tensor q, Tensor k, Tensor v, Tensor mask, Tensor(a4!) kcache, Tensor(a5!) vcache, "
      "Tensor seq, Tensor scale, Tensor block_table, SymInt block_size) -> Tensor");
  m.def(
      "paged_causal_attn_prefill(Tensor q, Tensor k, Tensor v, Tensor(a3!) kcache, Tensor(a4!) vcache, "
      "Tensor seq, Tensor scale, Tensor block_table, SymInt block_size, bool is_bidirectional, "
      "Tensor? mask=None) -> Tensor");
  m.def(
      "paged_causal_attn_prefill_kvfp8(Tensor q, Tensor? k, Tensor? v, Tensor(a3!) kcache, Tensor(a4!) vcache, "
      "Tensor(a5!) k_scale, Tensor(a6!) v_scale, Tensor seq, Tensor scale, Tensor block_table, SymInt block_size, "
      "bool is_bidirectional, Tensor? mask=None) -> Tensor");
  m.def(
      "paged_causal_attn_decode(Tensor q, Tensor k, Tensor v, Tensor(a3!) kcache, Tensor(a4!) vcache, "
      "Tensor seq, Tensor scale, Tensor block_table, SymInt block_size, Tensor? mask=None) -> Tensor");
  m.def(
      "paged_causal_attn_decode_shared(Tensor q, Tensor k, Tensor v, Tensor(a3!) kcache, Tensor(a4!) vcache, "
      "Tensor seq, Tensor scale, Tensor block_table, SymInt block_size, Tensor group_starts, Tensor shared_lens) -> "
      "Tensor");
  m.def(
      "paged_causal_attn_decode_kvfp8(Tensor q, Tensor k, Tensor v, Tensor(a3!) kcache, Tensor(a4!) vcache, "
      "Tensor k_scale, Tensor v_scale, Tensor seq, Tensor scale, Tensor block_table, SymInt block_size, "
      "Tensor? mask=None) -> Tensor");
  m.def(
      "flash_attention_naive_prefill(Tensor q, Tensor k, Tensor v, Tensor(a3!) kv_cache, Tensor mask, "
      "Tensor scale, Tensor seq_idx, Tensor block_tables, Tensor slot_mapping, Tensor? sinks=None) -> Tensor");
  m.def(
      "flash_attention_naive_decode(Tensor q, Tensor k, Tensor v, Tensor(a3!) kv_cache, Tensor mask, "
      "Tensor scale, Tensor seq_idx, Tensor block_tables, Tensor slot_mapping, Tensor? sinks=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(rbln_custom_ops, CUDA, m) {
  m.impl("paged_attn_prefill", &paged_attn_prefill_cuda);
  m.impl("paged_causal_attn_prefill", &paged_causal_attn_prefill_cuda);
  m.impl("paged_causal_attn_prefill_kvfp8", &paged_causal_attn_prefill_kvfp8_cuda);
  m.impl("paged_attn_decode", &paged_attn_decode_cuda);
  m.impl("paged_causal_attn_decode", &paged_causal_attn_decode_cuda);
  m.impl("paged_causal_attn_decode_shared", &paged_causal_attn_decode_shared_cuda);
  m.impl("paged_causal_attn_decode_kvfp8", &paged_causal_attn_decode_kvfp8_cuda);
  m.impl("flash_attention_naive_prefill", &flash_attention_naive_prefill_cuda);
  m.impl("flash_attention_naive_decode", &flash_attention_naive_decode_cuda);
}

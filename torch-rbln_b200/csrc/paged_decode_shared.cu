// Paged decode for a batch whose sequences share their first positions in
// groups (rbln_paged_causal_attn_decode_shared):
//   out[b] = softmax(scale q[b] K^T) V over positions [0, min(seq[b] + 1, span)),
// positions below the group's shared length read through the table of its
// first sequence, the others through the sequence's own.

#include <algorithm>

#include "decode_segment.cuh"

namespace rbln {
namespace {

constexpr int kMaxBatch = 4096, kMaxGroups = 1024;
constexpr int kPlanThreads = 1024;

struct SharedArgs {
  int groups;
  const int32_t* starts;
  const int32_t* lens;
  int* row_shared;  // [B] positions that are read through row_lead's table
  int* row_lead;    // [B]
};

// One CTA: every row's group and the positions that it shares.
__global__ void __launch_bounds__(kPlanThreads, 1) shared_plan_kernel(const DecodeArgs a, const SharedArgs s) {
  __shared__ int start[kMaxGroups + 1];
  for (int g = threadIdx.x; g <= s.groups; g += kPlanThreads) start[g] = min(max(s.starts[g], 0), a.B);
  __syncthreads();
  if (threadIdx.x == 0)
    for (int g = 1; g <= s.groups; ++g) start[g] = max(start[g], start[g - 1]);
  __syncthreads();
  for (int b = threadIdx.x; b < a.B; b += kPlanThreads) {
    int lo = -1, hi = s.groups;  // the last group that starts at or before b
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= b) lo = mid; else hi = mid - 1;
    }
    int n = 0;
    if (lo >= 0 && lo < s.groups) {
      n = min(max(s.lens[lo], 0), a.span);
      if (a.seq[b * a.seq_stride] < n) n = 0;
    }
    s.row_shared[b] = n;
    s.row_lead[b] = n > 0 ? start[lo] : b;
  }
}

// CTA (h, b): the whole context of one (sequence, KV head).
template <int D, int KV, bool Q_BF16, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 2) shared_decode_kernel(const DecodeArgs a, const SharedArgs s) {
  extern __shared__ __align__(16) unsigned char dsm[];
  const int h = blockIdx.x, b = blockIdx.y;
  int pos;
  const int L = seq_len(a, b, pos);
  if (pos < 0 && h == 0 && threadIdx.x == 0) flag_error(a.err, RBLN_DEVERR_SEQ_RANGE);
  decode_segment<D, KV, Q_BF16, NT, false, true>(a, dsm, b, h, 0, L, pos >= 0 && pos < a.span, true, 0, s.row_lead[b],
                                                 s.row_shared[b]);
}

template <int D, int KV, bool QB, int NT>
int launch(const DecodeArgs& a, const SharedArgs& s, cudaStream_t st) {
  shared_plan_kernel<<<1, kPlanThreads, 0, st>>>(a, s);
  static SmemOptIn done;
  if (!allow_smem(reinterpret_cast<const void*>(shared_decode_kernel<D, KV, QB, NT>), segment_smem<D, NT>(), done))
    return RBLN_ERR_LAUNCH;
  shared_decode_kernel<D, KV, QB, NT><<<dim3(a.Hkv, a.B), kThreads, segment_smem<D, NT>(), st>>>(a, s);
  return cudaGetLastError() == cudaSuccess ? RBLN_OK : RBLN_ERR_LAUNCH;
}

template <int D>
int launch_any(const DecodeArgs& a, const SharedArgs& s, bool bf16, cudaStream_t st) {
  if (bf16) return a.G > 8 ? launch<D, KV_BF16, true, 2>(a, s, st) : launch<D, KV_BF16, true, 1>(a, s, st);
  return a.G > 8 ? launch<D, KV_F16, false, 2>(a, s, st) : launch<D, KV_F16, false, 1>(a, s, st);
}

struct Plan {
  size_t row_shared, row_lead, total;
};

int plan_shared(const rbln_paged_attn_params_t* p, const rbln_shared_prefix_t* s, Plan* pl) {
  if (!p || !s || p->batch < 0 || p->num_kv_heads <= 0 || p->group <= 0 || p->block_size <= 0 || p->max_blocks <= 0 ||
      p->num_blocks <= 0 || s->num_groups < 0)
    return RBLN_ERR_INVALID_ARGUMENT;
  if (p->head_dim != 64 && p->head_dim != 128) return RBLN_ERR_UNSUPPORTED;
  if (p->group > 16 || p->batch > kMaxBatch || s->num_groups > kMaxGroups || p->num_kv_heads > 65535)
    return RBLN_ERR_UNSUPPORTED;
  if ((int64_t)p->max_blocks * p->block_size > (1 << 30)) return RBLN_ERR_UNSUPPORTED;
  const bool tiles = p->block_size % 128 == 0 || (p->block_size >= 8 && 128 % p->block_size == 0);
  if (!tiles) return RBLN_ERR_UNSUPPORTED;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t start = at;
    at += (n + 255) / 256 * 256;
    return start;
  };
  pl->row_shared = take(p->batch * sizeof(int));
  pl->row_lead = take(p->batch * sizeof(int));
  pl->total = at + 256;
  return RBLN_OK;
}

int run_shared(const rbln_paged_attn_params_t* p, const rbln_shared_prefix_t* s, cudaStream_t st) {
  Plan pl;
  const int rc = plan_shared(p, s, &pl);
  if (rc != RBLN_OK) return rc;
  if (p->q_len != 1) return RBLN_ERR_INVALID_ARGUMENT;
  if (p->mask || p->sinks || p->num_splits || p->prof_events[0] || p->prof_events[1]) return RBLN_ERR_UNSUPPORTED;
  if ((p->q_dtype != RBLN_DT_BF16 && p->q_dtype != RBLN_DT_F16) || p->kv_dtype != p->q_dtype)
    return RBLN_ERR_UNSUPPORTED;
  if (p->block_table_dtype != RBLN_DT_I16 && p->block_table_dtype != RBLN_DT_I32 &&
      p->block_table_dtype != RBLN_DT_I64)
    return RBLN_ERR_UNSUPPORTED;
  if (s->num_groups > 0 && (!s->group_starts || !s->shared_lens)) return RBLN_ERR_INVALID_ARGUMENT;
  if (p->batch == 0) return RBLN_OK;
  if (!p->q || !p->out || !p->kcache || !p->vcache || !p->seq || !p->block_table || (!p->k_new != !p->v_new))
    return RBLN_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (p->cache_stride[i] * 2 % 16 != 0 || p->q_stride[i] * 2 % 16 != 0 || p->out_stride[i] * 2 % 8 != 0)
      return RBLN_ERR_INVALID_ARGUMENT;
  if (!aligned16(p->q) || !aligned16(p->kcache) || !aligned16(p->vcache) ||
      (reinterpret_cast<uintptr_t>(p->out) & 7u) != 0)
    return RBLN_ERR_INVALID_ARGUMENT;
  if (p->k_new) {
    if (!aligned16(p->k_new) || !aligned16(p->v_new)) return RBLN_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < 2; ++i)
      if (p->k_new_stride[i] * 2 % 16 != 0 || p->v_new_stride[i] * 2 % 16 != 0) return RBLN_ERR_INVALID_ARGUMENT;
  }
  // rows are addressed as 32-bit counts of 16 bytes
  const int64_t reach = ((int64_t)(p->num_blocks - 1) * p->cache_stride[0] + (int64_t)(p->num_kv_heads - 1) * p->cache_stride[1] +
                         (int64_t)(p->block_size - 1) * p->cache_stride[2] + p->head_dim) * 2;
  if (reach / 16 > (int64_t)UINT32_MAX) return RBLN_ERR_UNSUPPORTED;
  if (!p->workspace || p->workspace_bytes < pl.total) return RBLN_ERR_WORKSPACE;
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p->workspace) + 255) & ~uintptr_t(255));

  DecodeArgs a{};
  a.q = static_cast<const char*>(p->q);
  a.qs_b = p->q_stride[0] * 2; a.qs_h = p->q_stride[1] * 2; a.qs_g = p->q_stride[2] * 2;
  a.out = static_cast<char*>(p->out);
  a.os_b = p->out_stride[0] * 2; a.os_h = p->out_stride[1] * 2; a.os_g = p->out_stride[2] * 2;
  a.k_new = static_cast<const char*>(p->k_new);
  a.v_new = static_cast<const char*>(p->v_new);
  a.kn_b = p->k_new_stride[0] * 2; a.kn_h = p->k_new_stride[1] * 2;
  a.vn_b = p->v_new_stride[0] * 2; a.vn_h = p->v_new_stride[1] * 2;
  a.kcache = static_cast<char*>(p->kcache);
  a.vcache = static_cast<char*>(p->vcache);
  a.cs_block = p->cache_stride[0]; a.cs_head = p->cache_stride[1]; a.cs_tok = p->cache_stride[2];
  a.seq = p->seq; a.seq_stride = p->seq_stride;
  a.bt = p->block_table; a.bt_dtype = p->block_table_dtype; a.bt_stride = p->block_table_stride;
  a.scale = p->scale; a.scale_dev = p->scale_dev;
  a.B = p->batch; a.Hkv = p->num_kv_heads; a.G = p->group; a.num_blocks = p->num_blocks;
  a.bs = p->block_size; a.span = p->max_blocks * p->block_size;
  a.err = p->error_flags;
  SharedArgs x{};
  x.groups = s->num_groups;
  x.starts = s->group_starts;
  x.lens = s->shared_lens;
  x.row_shared = reinterpret_cast<int*>(ws + pl.row_shared);
  x.row_lead = reinterpret_cast<int*>(ws + pl.row_lead);
  const bool bf16 = p->q_dtype == RBLN_DT_BF16;
  return p->head_dim == 128 ? launch_any<128>(a, x, bf16, st) : launch_any<64>(a, x, bf16, st);
}

}  // namespace
}  // namespace rbln

extern "C" {

size_t rbln_shared_prefix_sizeof(void) { return sizeof(rbln_shared_prefix_t); }

int rbln_paged_decode_shared_workspace_size(const rbln_paged_attn_params_t* p, const rbln_shared_prefix_t* s,
                                            size_t* bytes) {
  if (!bytes) return RBLN_ERR_INVALID_ARGUMENT;
  rbln::Plan pl;
  const int rc = rbln::plan_shared(p, s, &pl);
  if (rc != RBLN_OK) return rc;
  *bytes = pl.total;
  return RBLN_OK;
}

int rbln_paged_causal_attn_decode_shared(const rbln_paged_attn_params_t* p, const rbln_shared_prefix_t* s,
                                         cudaStream_t stream) {
  return rbln::run_shared(p, s, stream);
}

}  // extern "C"

// A step's queries and keys rotated and its keys and values written into the
// paged cache, in one launch (rbln_rotary_paged_kv_write): what a rotary
// layer, and then rbln_paged_kv_write on its result, would do in three, with
// one read of q, k and v and the rotated keys quantised from float32, not
// from a rounded copy.
//
// Token s of sequence b sits at position seq[b] + s. An fp8 cache follows the
// rule of rbln_paged_kv_write (kv_write.cu): scale = max(amax, 1e-6) / 448
// over the rows the sequence holds in a touched (block, head) and the new
// ones, held rows re-quantised when the scale changes, codes
// e4m3(x * (1 / scale)) in float32.
//
// Bound by HBM (2 bytes in and 1 to 2 out an element) where a step has many
// tokens, by latency where it has few. A CTA takes one (sequence, touched
// block) and a group of KV heads with their query heads: the angles depend on
// the token alone, so their sines and cosines are found once for the block,
// in shared memory. q (and the rows of a 16-bit cache) stream through all
// threads; a warp takes one (head, K or V) of an fp8 cache, 16 rows at a
// time, in registers from the amax to the codes: a block of 16 rows is read
// once, a larger one twice (its last 16 rows once).

#include "rotary.cuh"

namespace rbln {
namespace {

constexpr int kRwThreads = 256;
constexpr int kRwWarps = kRwThreads / 32;
constexpr int kTileRows = 16;
constexpr int kTableRows = 128;  // rows whose angles a CTA keeps; rows past them find theirs again (blocks > 128)

struct RotWriteArgs {
  const char* q;
  char* out;
  int64_t qs_b, qs_h, qs_g, qs_s, os_b, os_h, os_g, os_s;  // bytes
  const char* k_new;
  const char* v_new;
  int64_t kn_b, kn_h, kn_s, vn_b, vn_h, vn_s;  // bytes
  char* kcache;
  char* vcache;
  int64_t cs_block, cs_head, cs_tok;  // elements
  float* k_scale;
  float* v_scale;
  int64_t ss_block, ss_head;
  const int32_t* seq;
  int64_t seq_stride;
  const void* bt;
  int bt_dtype;
  int64_t bt_stride;
  const float* inv_freq;
  int B, Hkv, G, S, R, bs, max_blocks, num_blocks, slots, hg;  // hg: KV heads a CTA
  bool interleaved;
  float mscale;
  uint32_t* err;
};

// One item's 16 values (two vectors) from 32 bytes of bf16 / f16.
template <bool BF16>
__device__ __forceinline__ void widen16(uint4 w0, uint4 w1, float (&x)[16]) {
  const uint32_t u[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = unpack2<BF16>(u[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 narrow8(const float* x) {
  return make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7]));
}
// Eight values times inv as e4m3, saturated to +-448, round to nearest even.
__device__ __forceinline__ uint2 codes8(const float* x, float inv) {
  uint32_t u[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo =
        __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] * inv, x[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi =
        __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    u[i] = (lo & 0xffffu) | (hi << 16);
  }
  return make_uint2(u[0], u[1]);
}
// Eight codes times `s`.
__device__ __forceinline__ void decode8(uint2 w, float s, float (&x)[8]) {
  uint32_t h[4];
  e4m3x4_to_f16x2x2(w.x, h[0], h[1]);
  e4m3x4_to_f16x2x2(w.y, h[2], h[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<false>(h[i]);
    x[2 * i] = f.x * s;
    x[2 * i + 1] = f.y * s;
  }
}

template <int D, bool BF16, bool FP8>
__global__ void __launch_bounds__(kRwThreads, FP8 && D == 128 ? 2 : 3) rotary_write_kernel(const RotWriteArgs a) {
  constexpr int V = 8, NI = D / 16;           // items a row
  constexpr int PER = kTileRows * NI / 32;    // items a lane of a 16-row tile
  extern __shared__ float2 table[];           // [min(rows, kTableRows)][R/2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = blockIdx.x % a.slots, b = blockIdx.x / a.slots;
  const int h0 = blockIdx.y * a.hg, h1 = min(h0 + a.hg, a.Hkv);
  const int s0 = a.seq[b * a.seq_stride];
  // row of the first token in its block (s0 may be negative: refused below)
  const int p0 = ((s0 % a.bs) + a.bs) % a.bs;
  const int lo = max(j * a.bs - p0, 0), hi = (int)min((int64_t)(j + 1) * a.bs - p0, (int64_t)a.S);
  if (lo >= hi) return;  // tokens [lo, hi) fall in this block
  const int rows = hi - lo;

  // write target: the block's pool index, or none
  bool write = true;
  if (s0 < 0 || (int64_t)s0 + a.S > (int64_t)a.max_blocks * a.bs) {
    write = false;
    if (threadIdx.x == 0 && a.err) atomicOr(a.err, RBLN_DEVERR_SEQ_RANGE);
  }
  int64_t phys = 0;
  if (write) {
    phys = load_index(a.bt, a.bt_dtype, b * a.bt_stride + s0 / a.bs + j);
    if (phys < 0 || phys >= a.num_blocks) {
      write = false;
      if (threadIdx.x == 0 && a.err) atomicOr(a.err, RBLN_DEVERR_BLOCK_ID_RANGE);
    }
  }
  const int row0 = j == 0 ? p0 : 0;        // block row of token lo
  const int held = j == 0 && s0 > 0 ? p0 : 0;  // block rows the sequence holds already

  const int half = a.R / 2;
  for (int i = threadIdx.x; i < min(rows, kTableRows) * half; i += kRwThreads) {
    const int r = i / half, p = i - r * half;
    table[i] = rotary_cos_sin((double)((int64_t)s0 + lo + r), a.inv_freq[p], a.mscale);
  }
  __syncthreads();
  // x: the two vectors of item c of token lo + r
  auto turn = [&](int r, int c, float (&x)[16]) {
    float2 cs[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
      cs[i] = r < kTableRows ? table[r * half + c * V + i]
                             : rotary_cos_sin((double)((int64_t)s0 + lo + r), a.inv_freq[c * V + i], a.mscale);
    rotary_turn<V>(x, cs, a.interleaved);
  };

  if constexpr (FP8) {
    // one warp per (head, K or V): amax, scale, held rows, codes
    for (int u = warp; write && u < 2 * (h1 - h0); u += kRwWarps) {
      const int h = h0 + (u >> 1), part = u & 1;
      const char* src = part == 0 ? a.k_new + b * a.kn_b + h * a.kn_h : a.v_new + b * a.vn_b + h * a.vn_h;
      const int64_t src_s = part == 0 ? a.kn_s : a.vn_s;
      float* sp = (part == 0 ? a.k_scale : a.v_scale) + phys * a.ss_block + (int64_t)h * a.ss_head;
      uint8_t* c8 = reinterpret_cast<uint8_t*>(part == 0 ? a.kcache : a.vcache) + phys * a.cs_block +
                    (int64_t)h * a.cs_head;
      const float old = *sp;
      const int ntile = (rows + kTileRows - 1) / kTileRows;
      float x[PER][16];
      auto load_tile = [&](int t) {
        uint4 w0[PER], w1[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int i = lane + 32 * k, r = t * kTileRows + i / NI;
          const RotaryItem it = rotary_item(i % NI, V, part == 0 ? a.R : 0, a.interleaved);
          if (r < rows) {
            const char* p = src + (int64_t)(lo + r) * src_s;
            w0[k] = *reinterpret_cast<const uint4*>(p + it.e0 * 2);
            w1[k] = *reinterpret_cast<const uint4*>(p + it.e1 * 2);
          } else {
            w0[k] = w1[k] = make_uint4(0, 0, 0, 0);
          }
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int i = lane + 32 * k, r = t * kTileRows + i / NI;
          widen16<BF16>(w0[k], w1[k], x[k]);
          if (r < rows && rotary_item(i % NI, V, part == 0 ? a.R : 0, a.interleaved).turned) turn(r, i % NI, x[k]);
        }
      };
      float m = 0.f;
      for (int i = lane; i < held * (D / 8); i += 32) {
        const int r = i / (D / 8), c = i % (D / 8);
        float y[8];
        decode8(*reinterpret_cast<const uint2*>(c8 + (int64_t)r * a.cs_tok + c * 8), old, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(y[e]));
      }
      for (int t = 0; t < ntile; ++t) {
        load_tile(t);
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(x[k][e]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float scale = __fdiv_rn(fmaxf(m, 1e-6f), 448.f);
      const float inv = __frcp_rn(scale);
      if (held > 0 && scale != old) {
        for (int i = lane; i < held * (D / 8); i += 32) {
          const int r = i / (D / 8), c = i % (D / 8);
          uint2* w = reinterpret_cast<uint2*>(c8 + (int64_t)r * a.cs_tok + c * 8);
          float y[8];
          decode8(*w, old, y);
          *w = codes8(y, inv);
        }
      }
      for (int t = ntile - 1; t >= 0; --t) {  // the last tile is still in registers
        if (t != ntile - 1) load_tile(t);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int i = lane + 32 * k, r = t * kTileRows + i / NI;
          const RotaryItem it = rotary_item(i % NI, V, part == 0 ? a.R : 0, a.interleaved);
          if (r < rows) {
            uint8_t* w = c8 + (int64_t)(row0 + r) * a.cs_tok;
            *reinterpret_cast<uint2*>(w + it.e0) = codes8(x[k], inv);
            *reinterpret_cast<uint2*>(w + it.e1) = codes8(x[k] + 8, inv);
          }
        }
      }
      __syncwarp();  // every lane has read `old` before it is replaced
      if (lane == 0) *sp = scale;
    }
  }

  // the query heads, and the rows of a 16-bit cache: items one by one
  const int nq = (h1 - h0) * a.G, heads = nq + (FP8 ? 0 : 2 * (h1 - h0));
  const int total = heads * rows * NI;  // rows <= S, bounded on the host
  constexpr int U = 4;
  for (int i0 = threadIdx.x; i0 < total; i0 += U * kRwThreads) {
    uint4 w0[U], w1[U];
    char* to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kRwThreads;
      to[u] = nullptr;
      if (i >= total) continue;
      const int c = i % NI, r = (i / NI) % rows, hh = i / (NI * rows);
      const char* src;
      int turned = a.R;
      if (hh < nq) {
        const int h = h0 + hh / a.G, g = hh % a.G;
        src = a.q + b * a.qs_b + h * a.qs_h + g * a.qs_g + (int64_t)(lo + r) * a.qs_s;
        to[u] = a.out + b * a.os_b + h * a.os_h + g * a.os_g + (int64_t)(lo + r) * a.os_s;
      } else {
        const int part = (hh - nq) & 1, h = h0 + ((hh - nq) >> 1);
        if (!write) continue;
        src = part == 0 ? a.k_new + b * a.kn_b + h * a.kn_h + (int64_t)(lo + r) * a.kn_s
                        : a.v_new + b * a.vn_b + h * a.vn_h + (int64_t)(lo + r) * a.vn_s;
        to[u] = (part == 0 ? a.kcache : a.vcache) +
                (phys * a.cs_block + (int64_t)h * a.cs_head + (int64_t)(row0 + r) * a.cs_tok) * 2;
        if (part == 1) turned = 0;
      }
      const RotaryItem it = rotary_item(c, V, turned, a.interleaved);
      w0[u] = *reinterpret_cast<const uint4*>(src + it.e0 * 2);
      w1[u] = *reinterpret_cast<const uint4*>(src + it.e1 * 2);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (to[u] == nullptr) continue;
      const int i = i0 + u * kRwThreads;
      const int c = i % NI, r = (i / NI) % rows, hh = i / (NI * rows);
      const RotaryItem it = rotary_item(c, V, hh >= nq && ((hh - nq) & 1) ? 0 : a.R, a.interleaved);
      if (it.turned) {
        float x[16];
        widen16<BF16>(w0[u], w1[u], x);
        turn(r, c, x);
        w0[u] = narrow8<BF16>(x);
        w1[u] = narrow8<BF16>(x + 8);
      }
      *reinterpret_cast<uint4*>(to[u] + it.e0 * 2) = w0[u];
      *reinterpret_cast<uint4*>(to[u] + it.e1 * 2) = w1[u];
    }
  }
}

template <int D, bool BF16>
int launch_rotary_write(const RotWriteArgs& a, bool fp8, dim3 grid, size_t smem, cudaStream_t st) {
  const void* fn = fp8 ? (const void*)rotary_write_kernel<D, BF16, true> : (const void*)rotary_write_kernel<D, BF16, false>;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return RBLN_ERR_LAUNCH;
  if (fp8) rotary_write_kernel<D, BF16, true><<<grid, kRwThreads, smem, st>>>(a);
  else rotary_write_kernel<D, BF16, false><<<grid, kRwThreads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? RBLN_OK : RBLN_ERR_LAUNCH;
}

}  // namespace
}  // namespace rbln

extern "C" int rbln_rotary_paged_kv_write(const rbln_paged_attn_params_t* p, const rbln_rotary_params_t* r,
                                          cudaStream_t stream) {
  using namespace rbln;
  if (!p || !r || p->batch < 0 || p->num_kv_heads <= 0 || p->group <= 0 || p->q_len < 0 || p->block_size <= 0 ||
      p->max_blocks <= 0 || p->num_blocks <= 0 || r->rotary_dim <= 0 || r->rotary_dim > p->head_dim)
    return RBLN_ERR_INVALID_ARGUMENT;
  if (p->batch == 0 || p->q_len == 0) return RBLN_OK;
  if (p->head_dim != 64 && p->head_dim != 128) return RBLN_ERR_UNSUPPORTED;
  if (r->rotary_dim % 16) return RBLN_ERR_UNSUPPORTED;  // whole 16-byte vectors of both halves
  if (p->q_dtype != RBLN_DT_BF16 && p->q_dtype != RBLN_DT_F16) return RBLN_ERR_UNSUPPORTED;
  const bool fp8 = p->kv_dtype == RBLN_DT_FP8_E4M3;
  if (!fp8 && p->kv_dtype != p->q_dtype) return RBLN_ERR_UNSUPPORTED;
  if (p->block_table_dtype != RBLN_DT_I16 && p->block_table_dtype != RBLN_DT_I32 &&
      p->block_table_dtype != RBLN_DT_I64)
    return RBLN_ERR_UNSUPPORTED;
  if (!p->q || !p->out || !p->k_new || !p->v_new || !p->kcache || !p->vcache || !p->seq || !p->block_table ||
      !r->inv_freq || (fp8 && (!p->k_scale || !p->v_scale)))
    return RBLN_ERR_INVALID_ARGUMENT;
  {
    auto al = [](const void* q, unsigned m) { return (reinterpret_cast<uintptr_t>(q) & m) == 0; };
    const unsigned cm = fp8 ? 7u : 15u;
    if (!al(p->q, 15u) || !al(p->out, 15u) || !al(p->k_new, 15u) || !al(p->v_new, 15u) || !al(p->kcache, cm) ||
        !al(p->vcache, cm))
      return RBLN_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < 4; ++i)
      if (p->q_stride[i] % 8 || p->out_stride[i] % 8) return RBLN_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < 3; ++i)
      if (p->k_new_stride[i] % 8 || p->v_new_stride[i] % 8 || p->cache_stride[i] % 8) return RBLN_ERR_INVALID_ARGUMENT;
  }
  if ((int64_t)p->max_blocks * p->block_size > (1 << 30) || p->q_len > (1 << 30)) return RBLN_ERR_UNSUPPORTED;
  RotWriteArgs a{};
  a.q = static_cast<const char*>(p->q);
  a.qs_b = p->q_stride[0] * 2; a.qs_h = p->q_stride[1] * 2; a.qs_g = p->q_stride[2] * 2; a.qs_s = p->q_stride[3] * 2;
  a.out = static_cast<char*>(p->out);
  a.os_b = p->out_stride[0] * 2; a.os_h = p->out_stride[1] * 2; a.os_g = p->out_stride[2] * 2; a.os_s = p->out_stride[3] * 2;
  a.k_new = static_cast<const char*>(p->k_new);
  a.v_new = static_cast<const char*>(p->v_new);
  a.kn_b = p->k_new_stride[0] * 2; a.kn_h = p->k_new_stride[1] * 2; a.kn_s = p->k_new_stride[2] * 2;
  a.vn_b = p->v_new_stride[0] * 2; a.vn_h = p->v_new_stride[1] * 2; a.vn_s = p->v_new_stride[2] * 2;
  a.kcache = static_cast<char*>(p->kcache);
  a.vcache = static_cast<char*>(p->vcache);
  a.cs_block = p->cache_stride[0]; a.cs_head = p->cache_stride[1]; a.cs_tok = p->cache_stride[2];
  a.k_scale = const_cast<float*>(p->k_scale);
  a.v_scale = const_cast<float*>(p->v_scale);
  a.ss_block = p->scale_stride[0]; a.ss_head = p->scale_stride[1];
  a.seq = p->seq; a.seq_stride = p->seq_stride;
  a.bt = p->block_table; a.bt_dtype = p->block_table_dtype; a.bt_stride = p->block_table_stride;
  a.inv_freq = r->inv_freq;
  a.B = p->batch; a.Hkv = p->num_kv_heads; a.G = p->group; a.S = p->q_len; a.R = r->rotary_dim; a.bs = p->block_size;
  a.max_blocks = p->max_blocks; a.num_blocks = p->num_blocks;
  a.interleaved = r->interleaved != 0;
  a.mscale = r->mscale;
  a.err = p->error_flags;
  // blocks a sequence's tokens can touch: S rows from anywhere in a block
  const int64_t slots = ((int64_t)a.S + a.bs - 1) / a.bs + 1;
  if (slots * a.B > INT32_MAX) return RBLN_ERR_UNSUPPORTED;
  const int block_rows = a.S < a.bs ? a.S : a.bs;
  // a CTA's items are counted in 32 bits
  if ((int64_t)a.Hkv * (a.G + 2) * block_rows * (p->head_dim / 16) > (1 << 30)) return RBLN_ERR_UNSUPPORTED;
  a.slots = (int)slots;
  // All heads of a block in one CTA, unless that leaves the GPU short of CTAs
  // (about four an SM): then groups of KV heads, each finding the angles anew.
  a.hg = a.Hkv;
  while (a.hg > 1 && slots * a.B * ((a.Hkv + a.hg - 1) / a.hg) < 4 * 148) a.hg = (a.hg + 1) / 2;
  const int gy = (a.Hkv + a.hg - 1) / a.hg;
  if (gy > 65535) return RBLN_ERR_UNSUPPORTED;
  const size_t smem = (size_t)(block_rows < kTableRows ? block_rows : kTableRows) * (a.R / 2) * sizeof(float2);
  const dim3 grid((unsigned)(slots * a.B), (unsigned)gy);
  const bool bf = p->q_dtype == RBLN_DT_BF16;
  if (p->head_dim == 128)
    return bf ? launch_rotary_write<128, true>(a, fp8, grid, smem, stream)
              : launch_rotary_write<128, false>(a, fp8, grid, smem, stream);
  return bf ? launch_rotary_write<64, true>(a, fp8, grid, smem, stream)
            : launch_rotary_write<64, false>(a, fp8, grid, smem, stream);
}

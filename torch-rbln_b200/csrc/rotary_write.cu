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
constexpr int kTableRows = 128;  // rows whose angles are kept at once

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

// MULTI: blocks of more than 16 rows. Their rows are taken 128 at a time (the
// angles kept in shared memory), an fp8 cache's twice: for the amax, then for
// the codes. Blocks of up to 16 rows stay in registers in between.
template <int D, bool BF16, bool FP8, bool MULTI>
__global__ void __launch_bounds__(kRwThreads, FP8 && D == 128 ? 2 : 3) rotary_write_kernel(const RotWriteArgs a) {
  constexpr int V = 8, NI = D / 16;           // items a row
  constexpr int PER = kTileRows * NI / 32;    // items a lane of a 16-row tile
  // [rows][V][R / 16] pairs, a row padded so that the lanes of neighbouring
  // rows meet other banks: pair c V + i of a row at i R/16 + c
  extern __shared__ float2 table[];
  __shared__ float unit_max[MULTI ? 64 : 1];  // an fp8 block's amax so far, of each (head, K or V)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = blockIdx.x % a.slots, b = blockIdx.x / a.slots;
  const int h0 = blockIdx.y * a.hg, h1 = min(h0 + a.hg, a.Hkv);
  const int s0 = a.seq[b * a.seq_stride];
  // row of the first token in its block (s0 may be negative: refused below)
  const int p0 = ((s0 % a.bs) + a.bs) % a.bs;
  const int lo = max(j * a.bs - p0, 0), hi = (int)min((int64_t)(j + 1) * a.bs - p0, (int64_t)a.S);
  if (lo >= hi) return;  // tokens [lo, hi) fall in this block

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
  const int row0 = j == 0 ? p0 : 0;            // block row of token lo
  const int held = j == 0 && s0 > 0 ? p0 : 0;  // block rows the sequence holds already
  const int units = FP8 && write ? 2 * (h1 - h0) : 0;  // (head, K or V) of an fp8 cache, one a warp

  const int half = a.R / 2, groups = a.R / 16, stride = half + groups;
  auto fill_table = [&](int from, int rows) {  // angles of tokens [from, from + rows)
    for (int i = threadIdx.x; i < rows * half; i += kRwThreads) {
      const int r = i / half, p = i - r * half;
      table[r * stride + (p % V) * groups + p / V] =
          rotary_cos_sin((double)((int64_t)s0 + from + r), a.inv_freq[p], a.mscale);
    }
    __syncthreads();
  };
  // x: the two vectors of item c of the table's row r
  auto turn = [&](int r, int c, float (&x)[16]) {
    float2 cs[V];
#pragma unroll
    for (int i = 0; i < V; ++i) cs[i] = table[r * stride + i * groups + c];
    rotary_turn<V>(x, cs, a.interleaved);
  };
  // where unit u's rows come from and go to
  struct Unit {
    const char* src;
    int64_t src_s;
    float* scale;
    uint8_t* codes;
    int R;  // rotated dimensions (values: none)
  };
  auto unit_of = [&](int u) {
    const int h = h0 + (u >> 1), part = u & 1;
    Unit t;
    t.src = part == 0 ? a.k_new + b * a.kn_b + h * a.kn_h : a.v_new + b * a.vn_b + h * a.vn_h;
    t.src_s = part == 0 ? a.kn_s : a.vn_s;
    t.scale = (part == 0 ? a.k_scale : a.v_scale) + phys * a.ss_block + (int64_t)h * a.ss_head;
    t.codes = reinterpret_cast<uint8_t*>(part == 0 ? a.kcache : a.vcache) + phys * a.cs_block + (int64_t)h * a.cs_head;
    t.R = part == 0 ? a.R : 0;
    return t;
  };
  // tokens [from, from + n) of the unit, n <= 16, the first at the table's row `at`
  auto load_tile = [&](const Unit& t, int from, int n, int at, float (&x)[PER][16]) {
    uint4 w0[PER], w1[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = lane + 32 * k, r = i / NI;
      const RotaryItem it = rotary_item(i % NI, V, t.R, a.interleaved);
      w0[k] = w1[k] = make_uint4(0, 0, 0, 0);
      if (r < n) {
        const char* p = t.src + (int64_t)(from + r) * t.src_s;
        w0[k] = *reinterpret_cast<const uint4*>(p + it.e0 * 2);
        w1[k] = *reinterpret_cast<const uint4*>(p + it.e1 * 2);
      }
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = lane + 32 * k, r = i / NI;
      widen16<BF16>(w0[k], w1[k], x[k]);
      if (r < n && rotary_item(i % NI, V, t.R, a.interleaved).turned) turn(at + r, i % NI, x[k]);
    }
  };
  auto tile_max = [&](const float (&x)[PER][16], float m) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(x[k][e]));
    return m;
  };
  auto held_max = [&](const Unit& t, float old) {
    float m = 0.f;
#pragma unroll 1
    for (int i = lane; i < held * (D / 8); i += 32) {
      float y[8];
      decode8(*reinterpret_cast<const uint2*>(t.codes + (int64_t)(i / (D / 8)) * a.cs_tok + (i % (D / 8)) * 8), old, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(y[e]));
    }
    return m;
  };
  auto recode_held = [&](const Unit& t, float old, float inv) {
#pragma unroll 1
    for (int i = lane; i < held * (D / 8); i += 32) {
      uint2* w = reinterpret_cast<uint2*>(t.codes + (int64_t)(i / (D / 8)) * a.cs_tok + (i % (D / 8)) * 8);
      float y[8];
      decode8(*w, old, y);
      *w = codes8(y, inv);
    }
  };
  auto store_tile = [&](const Unit& t, int row, int n, const float (&x)[PER][16], float inv) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = lane + 32 * k, r = i / NI;
      const RotaryItem it = rotary_item(i % NI, V, t.R, a.interleaved);
      if (r < n) {
        uint8_t* w = t.codes + (int64_t)(row + r) * a.cs_tok;
        *reinterpret_cast<uint2*>(w + it.e0) = codes8(x[k], inv);
        *reinterpret_cast<uint2*>(w + it.e1) = codes8(x[k] + 8, inv);
      }
    }
  };
  auto warp_max = [](float m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  };
  // the query heads, and the rows of a 16-bit cache, tokens [from, from + rows): items one by one
  auto stream_rows = [&](int from, int rows) {
    const int nq = (h1 - h0) * a.G, heads = nq + (FP8 || !write ? 0 : 2 * (h1 - h0));
    const int total = heads * rows * NI;
    constexpr int U = 2;
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < total; i0 += U * kRwThreads) {
      uint4 w0[U], w1[U];
      char* to[U];
      RotaryItem it[U];
      int rc[U];  // table row x NI + item
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kRwThreads;
        to[u] = nullptr;
        if (i >= total) continue;
        const int q = i / NI, c = i % NI, hh = q / rows, r = q - hh * rows;
        rc[u] = r * NI + c;
        const char* src;
        int turned = a.R;
        if (FP8 || hh < nq) {
          const int hk = hh / a.G, h = h0 + hk, g = hh - hk * a.G;
          src = a.q + b * a.qs_b + h * a.qs_h + g * a.qs_g + (int64_t)(from + r) * a.qs_s;
          to[u] = a.out + b * a.os_b + h * a.os_h + g * a.os_g + (int64_t)(from + r) * a.os_s;
        } else {
          const int part = (hh - nq) & 1, h = h0 + ((hh - nq) >> 1);
          src = part == 0 ? a.k_new + b * a.kn_b + h * a.kn_h + (int64_t)(from + r) * a.kn_s
                          : a.v_new + b * a.vn_b + h * a.vn_h + (int64_t)(from + r) * a.vn_s;
          to[u] = (part == 0 ? a.kcache : a.vcache) +
                  (phys * a.cs_block + (int64_t)h * a.cs_head + (int64_t)(row0 + from - lo + r) * a.cs_tok) * 2;
          if (part == 1) turned = 0;
        }
        it[u] = rotary_item(c, V, turned, a.interleaved);
        w0[u] = *reinterpret_cast<const uint4*>(src + it[u].e0 * 2);
        w1[u] = *reinterpret_cast<const uint4*>(src + it[u].e1 * 2);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (to[u] == nullptr) continue;
        if (it[u].turned) {
          float x[16];
          widen16<BF16>(w0[u], w1[u], x);
          turn(rc[u] / NI, rc[u] % NI, x);
          w0[u] = narrow8<BF16>(x);
          w1[u] = narrow8<BF16>(x + 8);
        }
        *reinterpret_cast<uint4*>(to[u] + it[u].e0 * 2) = w0[u];
        *reinterpret_cast<uint4*>(to[u] + it[u].e1 * 2) = w1[u];
      }
    }
  };

  if constexpr (!MULTI) {
    fill_table(lo, hi - lo);
#pragma unroll 1
    for (int u = warp; u < units; u += kRwWarps) {
      const Unit t = unit_of(u);
      const float old = *t.scale;
      float x[PER][16];
      load_tile(t, lo, hi - lo, 0, x);
      const float m = warp_max(tile_max(x, held_max(t, old)));
      const float scale = __fdiv_rn(fmaxf(m, 1e-6f), 448.f);
      const float inv = __frcp_rn(scale);
      if (scale != old) recode_held(t, old, inv);
      store_tile(t, row0, hi - lo, x, inv);
      __syncwarp();  // every lane has read `old` before it is replaced
      if (lane == 0) *t.scale = scale;
    }
    stream_rows(lo, hi - lo);
  } else {
    const bool again = hi - lo > kTableRows;  // the angles do not fit at once
    if (!again || units == 0) fill_table(lo, min(hi - lo, kTableRows));
    if (units > 0) {
#pragma unroll 1
      for (int from = lo; from < hi; from += kTableRows) {
        const int rows = min(hi - from, kTableRows);
        if (again) {
          __syncthreads();
          fill_table(from, rows);
        }
#pragma unroll 1
        for (int u = warp; u < units; u += kRwWarps) {
          const Unit t = unit_of(u);
          float m = from == lo ? held_max(t, *t.scale) : unit_max[u];
#pragma unroll 1
          for (int r = 0; r < rows; r += kTileRows) {
            float x[PER][16];
            load_tile(t, from + r, min(rows - r, kTileRows), r, x);
            m = tile_max(x, m);
          }
          m = warp_max(m);
          __syncwarp();
          if (lane == 0) unit_max[u] = m;
          __syncwarp();
        }
      }
    }
#pragma unroll 1
    for (int from = lo; from < hi; from += kTableRows) {
      const int rows = min(hi - from, kTableRows);
      if (again && (units > 0 || from > lo)) {
        __syncthreads();
        fill_table(from, rows);
      }
#pragma unroll 1
      for (int u = warp; u < units; u += kRwWarps) {
        const Unit t = unit_of(u);
        const float old = *t.scale;
        const float scale = __fdiv_rn(fmaxf(unit_max[u], 1e-6f), 448.f);
        const float inv = __frcp_rn(scale);
        if (from == lo && scale != old) recode_held(t, old, inv);
#pragma unroll 1
        for (int r = 0; r < rows; r += kTileRows) {
          float x[PER][16];
          load_tile(t, from + r, min(rows - r, kTileRows), r, x);
          store_tile(t, row0 + from - lo + r, min(rows - r, kTileRows), x, inv);
        }
        __syncwarp();  // every lane has read `old` before it is replaced
        if (lane == 0) *t.scale = scale;
        __syncwarp();
      }
      stream_rows(from, rows);
    }
  }
}

template <int D, bool BF16, bool FP8, bool MULTI>
int launch_rotary_write(const RotWriteArgs& a, dim3 grid, size_t smem, cudaStream_t st) {
  auto kernel = rotary_write_kernel<D, BF16, FP8, MULTI>;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return RBLN_ERR_LAUNCH;
  kernel<<<grid, kRwThreads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? RBLN_OK : RBLN_ERR_LAUNCH;
}
template <int D, bool BF16>
int launch_rotary_write(const RotWriteArgs& a, bool fp8, dim3 grid, size_t smem, cudaStream_t st) {
  if (a.bs > kTileRows)
    return fp8 ? launch_rotary_write<D, BF16, true, true>(a, grid, smem, st)
               : launch_rotary_write<D, BF16, false, true>(a, grid, smem, st);
  return fp8 ? launch_rotary_write<D, BF16, true, false>(a, grid, smem, st)
             : launch_rotary_write<D, BF16, false, false>(a, grid, smem, st);
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
  a.hg = a.Hkv < 32 ? a.Hkv : 32;  // unit_max holds 64
  while (a.hg > 1 && slots * a.B * ((a.Hkv + a.hg - 1) / a.hg) < 4 * 148) a.hg = (a.hg + 1) / 2;
  const int gy = (a.Hkv + a.hg - 1) / a.hg;
  if (gy > 65535) return RBLN_ERR_UNSUPPORTED;
  const size_t smem = (size_t)(block_rows < kTableRows ? block_rows : kTableRows) * (a.R / 2 + a.R / 16) * sizeof(float2);
  const dim3 grid((unsigned)(slots * a.B), (unsigned)gy);
  const bool bf = p->q_dtype == RBLN_DT_BF16;
  if (p->head_dim == 128)
    return bf ? launch_rotary_write<128, true>(a, fp8, grid, smem, stream)
              : launch_rotary_write<128, false>(a, fp8, grid, smem, stream);
  return bf ? launch_rotary_write<64, true>(a, fp8, grid, smem, stream)
            : launch_rotary_write<64, false>(a, fp8, grid, smem, stream);
}

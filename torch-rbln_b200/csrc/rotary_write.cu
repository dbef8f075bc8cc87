// A step's queries and keys rotated and its keys and values written into the
// paged cache, in one launch (rbln_rotary_paged_kv_write): what a rotary
// layer, and then rbln_paged_kv_write on its result, would do in three, with
// one read of q, k and v and the rotated keys quantised from float32, not
// from a rounded copy. (The torch op copies inputs that are not contiguous
// before that.)
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
// threads, two 16-byte loads and stores an item; the rows that are quantised
// wait in shared memory between their amax and their codes (held in registers
// by an unrolled tile: 65.7 us against 26.6 for 8 sequences of 512 tokens, and
// 16.4 against 10.3 for 256 of one; instruction fetch bounded that). The 512
// tokens run at 3.5 TB/s, 53 % of the copy rate.

#include "rotary.cuh"

namespace rbln {
namespace {

constexpr int kRwThreads = 256;
constexpr int kRwWarps = kRwThreads / 32;
constexpr int kTableRows = 128;  // rows whose angles a streaming CTA keeps at once
constexpr int kStageRows = 16;   // rows a quantising CTA holds in shared memory

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
  int B, Hkv, G, S, R, bs, max_blocks, num_blocks, slots;
  int hg, kv_groups, sg;  // KV heads a quantising CTA, its groups; KV heads a streaming CTA
  uint32_t g_mul, g_shift;  // n / G = (mulhi(n, g_mul) + n) >> g_shift, n < 2^30
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

// 16 bytes global -> shared in the background.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// grid (blocks touched x sequences, kv_groups + stream_groups): the first
// kv_groups CTAs of a block quantise groups of KV heads of an fp8 cache, the
// others stream groups of query heads (and a 16-bit cache's rows).
//
// A quantising CTA copies 16 rows of its heads' keys and values into shared
// memory, all of them on their way at once, finds the angles meanwhile, and
// then works out of shared memory, one warp a (head, K or V): the amax, held
// rows among it, then the codes. A block of more than 16 rows passes twice.
// The loops are rolled: most launches are a few microseconds long, and a
// 16-row tile unrolled in registers spent them fetching instructions.
template <int D, bool BF16, bool FP8>
__global__ void __launch_bounds__(kRwThreads, 4) rotary_write_kernel(const RotWriteArgs a) {
  constexpr int V = 8, NI = D / 16;  // items a row
  extern __shared__ __align__(16) unsigned char dsm[];
  // (cos, sin) of two pairs a float4: pairs c V + 2 i and c V + 2 i + 1 of a
  // row at i R/16 + c, so that the eight items of a row meet all banks once
  float4* table = reinterpret_cast<float4*>(dsm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = blockIdx.x % a.slots, b = blockIdx.x / a.slots;
  const int s0 = a.seq[b * a.seq_stride];
  // row of the first token in its block (s0 may be negative: refused below)
  const int p0 = ((s0 % a.bs) + a.bs) % a.bs;
  const int lo = max(j * a.bs - p0, 0), hi = (int)min((int64_t)(j + 1) * a.bs - p0, (int64_t)a.S);
  if (lo >= hi) return;  // tokens [lo, hi) fall in this block
  const bool quantise = FP8 && (int)blockIdx.y < a.kv_groups;

  // write target: the block's pool index, or none
  bool write = quantise || !FP8;
  if (write && (s0 < 0 || (int64_t)s0 + a.S > (int64_t)a.max_blocks * a.bs)) {
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
  const int row0 = j == 0 ? p0 : 0;  // block row of token lo

  const int half = a.R / 2, groups = a.R / 16, stride = a.R / 4;
  auto fill_table = [&](int from, int rows) {  // angles of tokens [from, from + rows)
#pragma unroll 1
    for (int i = threadIdx.x; i < rows * half; i += kRwThreads) {
      const int r = i / half, p = i - r * half;
      float4* to = table + r * stride + (p % V) / 2 * groups + p / V;
      reinterpret_cast<float2*>(to)[p & 1] =
          rotary_cos_sin((double)((int64_t)s0 + from + r), a.inv_freq[p], a.mscale);
    }
  };
  // x: the two vectors of item c of the table's row r
  auto turn = [&](int r, int c, float (&x)[16]) {
    float2 cs[V];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float4 w = table[r * stride + i * groups + c];
      cs[2 * i] = make_float2(w.x, w.y);
      cs[2 * i + 1] = make_float2(w.z, w.w);
    }
    rotary_turn<V>(x, cs, a.interleaved);
  };

  if (quantise) {
    if (!write) return;
    const int h0 = blockIdx.y * a.hg, h1 = min(h0 + a.hg, a.Hkv), units = 2 * (h1 - h0);
    const int held = j == 0 && s0 > 0 ? p0 : 0;  // block rows the sequence holds already
    // rows [unit][16][D] after the angles of 16 rows; each unit's amax
    unsigned char* stage = dsm + kStageRows * stride * sizeof(float4);
    float* unit_max = reinterpret_cast<float*>(stage + a.hg * 2 * kStageRows * D * 2);
    auto fetch = [&](int from, int rows) {
      constexpr int C = D / 8;  // 16-byte pieces a row
      for (int i = threadIdx.x; i < units * rows * C; i += kRwThreads) {
        const int c = i % C, z = i / C, u = z / rows, r = z - u * rows, h = h0 + (u >> 1);
        const char* src = u & 1 ? a.v_new + b * a.vn_b + h * a.vn_h + (int64_t)(from + r) * a.vn_s
                                : a.k_new + b * a.kn_b + h * a.kn_h + (int64_t)(from + r) * a.kn_s;
        copy16(stage + ((u * kStageRows + r) * C + c) * 16, src + c * 16);
      }
      fill_table(from, rows);
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();
    };
    // item i of unit u's rows in shared memory: its 16 values, turned
    auto item = [&](int u, int i, RotaryItem& it, float (&x)[16]) {
      const int r = i / NI, c = i % NI;
      it = rotary_item(c, V, u & 1 ? 0 : a.R, a.interleaved);
      const unsigned char* p = stage + (u * kStageRows + r) * D * 2;
      widen16<BF16>(*reinterpret_cast<const uint4*>(p + it.e0 * 2), *reinterpret_cast<const uint4*>(p + it.e1 * 2), x);
      if (it.turned) turn(r, c, x);
    };
    auto scale_of = [&](int u) {
      return (u & 1 ? a.v_scale : a.k_scale) + phys * a.ss_block + (int64_t)(h0 + (u >> 1)) * a.ss_head;
    };
    auto codes_of = [&](int u) {
      return reinterpret_cast<uint8_t*>(u & 1 ? a.vcache : a.kcache) + phys * a.cs_block +
             (int64_t)(h0 + (u >> 1)) * a.cs_head;
    };
    auto held_piece = [&](uint8_t* codes, int i) {
      return reinterpret_cast<uint2*>(codes + (int64_t)(i / (D / 8)) * a.cs_tok + (i % (D / 8)) * 8);
    };
    auto amax = [&](int from, int rows) {
#pragma unroll 1
      for (int u = warp; u < units; u += kRwWarps) {
        float m = from == lo ? 0.f : unit_max[u];
        if (from == lo) {
          const float old = *scale_of(u);
          uint8_t* codes = codes_of(u);
#pragma unroll 4
          for (int i = lane; i < held * (D / 8); i += 32) {
            float y[8];
            decode8(*held_piece(codes, i), old, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(y[e]));
          }
        }
#pragma unroll 1
        for (int i = lane; i < rows * NI; i += 32) {
          RotaryItem it;
          float x[16];
          item(u, i, it, x);
#pragma unroll
          for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        __syncwarp();
        if (lane == 0) unit_max[u] = m;
        __syncwarp();
      }
    };
    auto encode = [&](int from, int rows) {
#pragma unroll 1
      for (int u = warp; u < units; u += kRwWarps) {
        uint8_t* codes = codes_of(u);
        const float old = *scale_of(u);
        const float scale = __fdiv_rn(fmaxf(unit_max[u], 1e-6f), 448.f);
        const float inv = __frcp_rn(scale);
        if (from == lo && scale != old) {
#pragma unroll 4
          for (int i = lane; i < held * (D / 8); i += 32) {
            float y[8];
            decode8(*held_piece(codes, i), old, y);
            *held_piece(codes, i) = codes8(y, inv);
          }
        }
#pragma unroll 1
        for (int i = lane; i < rows * NI; i += 32) {
          RotaryItem it;
          float x[16];
          item(u, i, it, x);
          uint8_t* w = codes + (int64_t)(row0 + from - lo + i / NI) * a.cs_tok;
          *reinterpret_cast<uint2*>(w + it.e0) = codes8(x, inv);
          *reinterpret_cast<uint2*>(w + it.e1) = codes8(x + 8, inv);
        }
        __syncwarp();  // every lane has read `old` before it is replaced
        if (lane == 0) *scale_of(u) = scale;
        __syncwarp();
      }
    };
#pragma unroll 1
    for (int from = lo; from < hi; from += kStageRows) {
      if (from > lo) __syncthreads();  // the rows before have been read
      fetch(from, min(hi - from, kStageRows));
      amax(from, min(hi - from, kStageRows));
    }
#pragma unroll 1
    for (int from = lo; from < hi; from += kStageRows) {
      if (hi - lo > kStageRows) {
        __syncthreads();
        fetch(from, min(hi - from, kStageRows));
      }
      encode(from, min(hi - from, kStageRows));
    }
    return;
  }

  // The query heads, and the rows of a 16-bit cache: a thread keeps its item
  // of a row and walks (head, row), row fastest.
  const int h0 = (blockIdx.y - a.kv_groups) * a.sg, h1 = min(h0 + a.sg, a.Hkv);
  const int nq = (h1 - h0) * a.G, heads = nq + (write ? 2 * (h1 - h0) : 0);
  constexpr int STEP = kRwThreads / NI, U = 2;  // rows a step; steps whose loads are in flight
  const int c = threadIdx.x % NI, z = threadIdx.x / NI;
  const RotaryItem turned = rotary_item(c, V, a.R, a.interleaved), passed = rotary_item(c, V, 0, false);
#pragma unroll 1
  for (int from = lo; from < hi; from += kTableRows) {
    const int rows = min(hi - from, kTableRows);
    if (from > lo) __syncthreads();
    fill_table(from, rows);
    __syncthreads();
    const int dh = STEP / rows, dr = STEP - dh * rows;
    const char* qb = a.q + b * a.qs_b + h0 * a.qs_h + (int64_t)from * a.qs_s;
    char* ob = a.out + b * a.os_b + h0 * a.os_h + (int64_t)from * a.os_s;
    int hh = z / rows, r = z - hh * rows;
#pragma unroll 1
    while (hh < heads) {
      uint4 w0[U], w1[U];
      char* to[U];
      RotaryItem it[U];
      int row[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        to[u] = nullptr;
        row[u] = r;
        it[u] = turned;
        if (hh < heads) {
          const char* src;
          if (FP8 || hh < nq) {
            const int hk = (int)((__umulhi((uint32_t)hh, a.g_mul) + (uint32_t)hh) >> a.g_shift), g = hh - hk * a.G;
            src = qb + hk * a.qs_h + g * a.qs_g + r * a.qs_s;
            to[u] = ob + hk * a.os_h + g * a.os_g + r * a.os_s;
          } else {
            const int part = (hh - nq) & 1, h = h0 + ((hh - nq) >> 1);
            src = part == 0 ? a.k_new + b * a.kn_b + h * a.kn_h + (int64_t)(from + r) * a.kn_s
                            : a.v_new + b * a.vn_b + h * a.vn_h + (int64_t)(from + r) * a.vn_s;
            to[u] = (part == 0 ? a.kcache : a.vcache) +
                    (phys * a.cs_block + (int64_t)h * a.cs_head + (int64_t)(row0 + from - lo + r) * a.cs_tok) * 2;
            if (part == 1) it[u] = passed;
          }
          w0[u] = *reinterpret_cast<const uint4*>(src + it[u].e0 * 2);
          w1[u] = *reinterpret_cast<const uint4*>(src + it[u].e1 * 2);
          hh += dh;
          r += dr;
          if (r >= rows) {
            r -= rows;
            ++hh;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (to[u] == nullptr) continue;
        if (it[u].turned) {
          float x[16];
          widen16<BF16>(w0[u], w1[u], x);
          turn(row[u], c, x);
          w0[u] = narrow8<BF16>(x);
          w1[u] = narrow8<BF16>(x + 8);
        }
        *reinterpret_cast<uint4*>(to[u] + it[u].e0 * 2) = w0[u];
        *reinterpret_cast<uint4*>(to[u] + it[u].e1 * 2) = w1[u];
      }
    }
  }
}

template <int D, bool BF16>
int launch_rotary_write(const RotWriteArgs& a, bool fp8, dim3 grid, size_t smem, cudaStream_t st) {
  auto kernel = fp8 ? rotary_write_kernel<D, BF16, true> : rotary_write_kernel<D, BF16, false>;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return RBLN_ERR_LAUNCH;
  kernel<<<grid, kRwThreads, smem, st>>>(a);
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
  for (a.g_shift = 0; (1u << a.g_shift) < (uint32_t)a.G; ++a.g_shift) {
  }
  a.g_mul = (uint32_t)(((uint64_t)((1u << a.g_shift) - (uint32_t)a.G) << 32) / (uint32_t)a.G + 1);
  a.mscale = r->mscale;
  a.err = p->error_flags;
  // blocks a sequence's tokens can touch: S rows from anywhere in a block
  const int64_t slots = ((int64_t)a.S + a.bs - 1) / a.bs + 1;
  if (slots * a.B > INT32_MAX) return RBLN_ERR_UNSUPPORTED;
  const int block_rows = a.S < a.bs ? a.S : a.bs;
  // a CTA's items are counted in 32 bits
  if ((int64_t)a.Hkv * (a.G + 2) * block_rows * (p->head_dim / 16) > (1 << 30)) return RBLN_ERR_UNSUPPORTED;
  a.slots = (int)slots;
  const int64_t work = ((int64_t)a.S + a.bs - 1) / a.bs * a.B;  // blocks that are touched, about
  // Four KV heads a quantising CTA: one (head, K or V) a warp, 32 KB of rows
  // (one, two, four heads: 128, 100, 90 us for 32 sequences of 512 tokens, 32
  // query heads over 8 KV heads of 128; 24.6, 18.4, 16.3 for 256 of one).
  // A streaming CTA takes all heads of a block, or a group of them where that
  // leaves the GPU short of CTAs (three an SM), down to one KV head. Same
  // heads, all against this rule against one head: 17.2, 12.3, 13.2 us for 1
  // sequence of 512 tokens, 34.8, 31.6, 36.8 for 8 of them, 88.8, 90.0, 117
  // for 32, and 14.3, 16.3, 22.5 for 256 of one token.
  a.hg = a.Hkv < 4 ? a.Hkv : 4;
  a.kv_groups = fp8 ? (a.Hkv + a.hg - 1) / a.hg : 0;
  a.sg = a.Hkv;
  while (a.sg > 1 && work * ((a.Hkv + a.sg - 1) / a.sg) < 3 * 148) a.sg = (a.sg + 1) / 2;
  const int64_t gy = a.kv_groups + (a.Hkv + a.sg - 1) / a.sg;
  if (gy > 65535) return RBLN_ERR_UNSUPPORTED;
  const size_t angles = (size_t)(a.R / 4) * sizeof(float4);
  const size_t stream_smem = angles * (block_rows < kTableRows ? block_rows : kTableRows);
  const size_t quant_smem = fp8 ? angles * kStageRows + (size_t)a.hg * 2 * (kStageRows * p->head_dim * 2 + sizeof(float)) : 0;
  const size_t smem = stream_smem > quant_smem ? stream_smem : quant_smem;
  const dim3 grid((unsigned)(slots * a.B), (unsigned)gy);
  const bool bf = p->q_dtype == RBLN_DT_BF16;
  if (p->head_dim == 128)
    return bf ? launch_rotary_write<128, true>(a, fp8, grid, smem, stream)
              : launch_rotary_write<128, false>(a, fp8, grid, smem, stream);
  return bf ? launch_rotary_write<64, true>(a, fp8, grid, smem, stream)
            : launch_rotary_write<64, false>(a, fp8, grid, smem, stream);
}

// Attention of S_q new tokens a sequence over an fp8-e4m3 paged KV cache with
// one fp32 scale for each (block, KV head): the kv_dtype FP8_E4M3 form of
// rbln_paged_causal_attn_prefill. The new rows are written first, by the rule
// of rbln_paged_kv_write (scales of touched blocks found anew), and read back
// with the rest.
//
//   out[s] = sum_t p_st v_t / sum_t p_st,  p_st = exp(scale q_s . k_t)
// over the keys t <= seq[b] + s (causal) or t < seq[b] + S_q (both ways) that
// the position mask, where there is one, keeps. With k_t = ks c_t and
// v_t = vs d_t, c and d the e4m3 codes of a block and ks, vs its scales, the
// products run on the codes: every code is exact in f16, ks multiplies the
// score in float32 and vs the probability, which is rounded to f16 once.
// A bf16 query goes to f16 with a power of two of its row, so that its largest
// magnitude lies in [2^14, 2^15): exact down to 2^-28 of the row's largest.
// The probabilities' vs is taken relative to a running power of two (vref) at
// or above the largest scale seen, so a cache of small values keeps all of
// f16's bits and one of large values cannot overflow; the accumulator is
// rescaled when vref grows. A block whose scale is far below vref keeps its
// probabilities to 2^-25 of vref, an error of 2^-25 of the largest value.
// The running maximum, the sums and the accumulators are float32.

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace rbln {
namespace {

constexpr int kMqWarps = 4;
constexpr int kMqThreads = kMqWarps * 32;
constexpr int kMqTile = 16;     // keys a warp's tile
constexpr int kSegCost = 128;   // virtual keys charged to each unit's start
constexpr int kMinW = 256;      // smallest share of a CTA, in keys
constexpr int kMaxItems = 4096; // (sequence, row tile) items whose prefix a CTA holds in shared memory

struct Fp8Args {
  const char* q;
  char* out;
  int64_t qs_b, qs_h, qs_g, qs_s, os_b, os_h, os_g, os_s;  // bytes
  const char* kcache;
  const char* vcache;
  int64_t cs_block, cs_head, cs_tok;  // elements = bytes
  const float* k_scale;
  const float* v_scale;
  int64_t ss_block, ss_head;
  const int32_t* seq;
  int64_t seq_stride;
  const void* bt;
  int bt_dtype;
  int64_t bt_stride;
  const void* mask;  // optional position keep-mask [B, L]
  int mask_dtype, mask_len;
  int64_t mask_stride;
  float scale;
  const float* scale_dev;
  int B, Hkv, G, S, num_blocks, bs, max_blocks, span;
  int causal;
  int tiles, items;  // row tiles a sequence; items = B * tiles
  int balanced;      // 1: the keys of all units cut into equal shares; 0: whole units, grid-strided
  // balanced: desc[2c], desc[2c + 1] = the unit that CTA c continues / starts
  // without finishing (-1: none), with its partial result in the same slot
  int* desc;
  float* part_o;   // [2 nCTA][rows][D], relative to 2^m, times the V scales
  float2* part_ml; // [2 nCTA][rows]: (m, l)
  uint32_t* err;
};

__device__ __forceinline__ void dependents_enter() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Smallest power of two above x / 2^1 that is >= x (x clamped to a sane range).
__device__ __forceinline__ float pow2_above(float x) {
  x = fminf(fmaxf(x, 1e-30f), 1e30f);
  return __uint_as_float((__float_as_uint(x) + 0x007fffffu) & 0x7f800000u);
}

// Keys [0, L) that some row of item's row tile may see; `last` is the tile's last token.
__device__ __forceinline__ int item_keys(const Fp8Args& a, int b, int last) {
  const int pos = a.seq[b * a.seq_stride];
  if (pos < 0) return 0;
  const int64_t end = (int64_t)pos + (a.causal ? min(last, a.S - 1) + 1 : a.S);
  return (int)min(end, (int64_t)a.span);
}

// Exclusive prefix P[0..items] of the items' costs (keys rounded up to 16
// plus kSegCost), by the whole CTA. rows: rows of a row tile.
template <int THREADS>
__device__ __forceinline__ void cost_prefix(const Fp8Args& a, int rows, int* P) {
  __shared__ int wsum[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.items + THREADS - 1) / THREADS;
  const int first = tid * per;
  auto cost = [&](int i) {
    const int b = i / a.tiles, t = i - b * a.tiles;
    return ((item_keys(a, b, (int)(((int64_t)(t + 1) * rows - 1) / a.G)) + 15) & ~15) + kSegCost;
  };
  int sum = 0;
  for (int i = 0; i < per; ++i)
    if (first + i < a.items) sum += cost(first + i);
  int x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) wsum[warp] = x;
  __syncthreads();
  int off = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) off += w < warp ? wsum[w] : 0;
  int run = off + x - sum;
  for (int i = 0; i < per; ++i)
    if (first + i < a.items) {
      P[first + i] = run;
      run += cost(first + i);
    }
  if (tid == THREADS - 1) P[a.items] = off + x;
  __syncthreads();
}

// ---------------------------------------------------------------------------
// Few rows (S_q G up to 16 of a KV head a tile): bound by HBM, one read of
// the cached bytes. As in the one-token decode, tokens are the M side of
// mma.m16n8k16 and the rows (token s, head g), s G + g, the N side, so that a
// tile's codes go from 16-byte loads to f16 fragments in registers; four warps
// take 16-key tiles round-robin and are joined in shared memory. The keys of
// all (head, sequence) units are cut into equal shares, one CTA each.
// ---------------------------------------------------------------------------
template <int D, bool BF16, int NT>
__device__ __forceinline__ void mq_segment(const Fp8Args& a, unsigned char* dsm, int b, int h, int tile, int t0,
                                           int t1, bool whole, int slot) {
  constexpr int KCH = D / 64, KR = D / 8, VSEG = D == 128 ? 16 : 8, NVW = D / 32, MT = D / 16, NC = 8 * NT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int c0 = tile * NC, cols = min(NC, a.S * a.G - c0);
  const int pos = a.seq[b * a.seq_stride];

  struct Entry {
    int blk;
    bool keep;
  };
  auto entry = [&](int ts, Entry& e) {
    const int t = ts + (lane & 15);
    const bool in = t < t1;
    e.keep = in && (a.mask == nullptr ||
                    (t < a.mask_len && load_keep(a.mask, a.mask_dtype, b * a.mask_stride + t)));
    const int64_t blk = in ? load_index(a.bt, a.bt_dtype, b * a.bt_stride + t / a.bs) : -1;
    e.blk = (blk >= 0 && blk < a.num_blocks) ? (int)blk : -1;
  };
  Entry ent;
  entry(t0 + warp * kMqTile, ent);

  // query fragments (B operand: k = head_dim, n = column gid + 8 nt) in f16
  uint32_t qf[NT][KR];
  float colmul[NT][2];
  int lim[NT][2];
  {
    const float mult = (a.scale_dev ? *a.scale_dev : a.scale) * kLog2e;
    float undo[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = c0 + gid + 8 * nt;
      const bool live = gid + 8 * nt < cols;
      const int s = live ? c / a.G : 0, g = live ? c - s * a.G : 0;
      const char* row = a.q + b * a.qs_b + h * a.qs_h + g * a.qs_g + s * a.qs_s;
      float qmax = 0.f;
#pragma unroll
      for (int i = 0; i < KCH; ++i) {
        const char* src = row + (4 * i + tig) * 32;
        const uint4 x0 = live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
        const uint4 x1 = live ? *reinterpret_cast<const uint4*>(src + 16) : make_uint4(0, 0, 0, 0);
        const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          qf[nt][8 * i + k] = w[k];
          const float2 f = unpack2<BF16>(w[k]);
          qmax = fmaxf(qmax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      undo[nt] = 1.f;
      if constexpr (BF16) {
        qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, 1));
        qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, 2));
        float up = 1.f;
        if (qmax > 0.f && qmax < 3e38f) {
          const int e = (int)(__float_as_uint(qmax) >> 23) - 127;  // qmax in [2^e, 2^(e+1))
          const int k = min(max(14 - e, -120), 120);
          up = __uint_as_float((uint32_t)(127 + k) << 23);
          undo[nt] = __uint_as_float((uint32_t)(127 - k) << 23);
        }
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          const float2 f = unpack2<true>(qf[nt][k]);
          qf[nt][k] = pack2<false>(f.x * up, f.y * up);
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // this lane's score columns 2 tig + k
        const int c = 2 * tig + k;
        colmul[nt][k] = mult * __shfl_sync(0xffffffffu, undo[nt], c * 4);
        lim[nt][k] = c + 8 * nt >= cols ? 0
                     : a.causal         ? min((int64_t)pos + (c0 + c + 8 * nt) / a.G + 1, (int64_t)t1)
                                        : t1;
      }
  }

  float o_acc[NT][MT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) o_acc[nt][mt][k] = 0.f;
  float m_run[NT][2], l_run[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_run[nt][0] = m_run[nt][1] = neg_inf();
    l_run[nt][0] = l_run[nt][1] = 0.f;
  }
  float vref = 0.f, inv_vref = 0.f;  // power of two at or above every V scale met, and its reciprocal
  const int tv[4] = {2 * tig, 2 * tig + 1, 2 * tig + 8, 2 * tig + 9};

  struct Tile {
    uint4 kraw[2][KCH];
    uint32_t vraw[4][NVW];
    uint32_t vmask;
    float ksc, vsc;
  };
  auto fetch = [&](int ts, Tile& T, const Entry& e) {
    const int t = ts + (lane & 15);
    bool valid = e.keep;
    int64_t off = 0;
    T.ksc = 1.f;
    T.vsc = 0.f;
    if (valid) {
      if (e.blk < 0) {
        valid = false;
        if (a.err) atomicOr(a.err, RBLN_DEVERR_BLOCK_ID_RANGE);
      } else {
        off = e.blk * a.cs_block + h * a.cs_head + (t % a.bs) * a.cs_tok;
        T.ksc = a.k_scale[e.blk * a.ss_block + h * a.ss_head];
        T.vsc = a.v_scale[e.blk * a.ss_block + h * a.ss_head];
      }
    }
    T.vmask = __ballot_sync(0xffffffffu, valid) & 0xffffu;
    if (T.vmask == 0) return;
    const int64_t ok0 = __shfl_sync(0xffffffffu, off, gid);
    const int64_t ok1 = __shfl_sync(0xffffffffu, off, gid + 8);
    const bool vk0 = (T.vmask >> gid) & 1, vk1 = (T.vmask >> (gid + 8)) & 1;
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      T.kraw[0][i] = vk0 ? ld_stream_v4(a.kcache + ok0 + (4 * i + tig) * 16) : make_uint4(0, 0, 0, 0);
      T.kraw[1][i] = vk1 ? ld_stream_v4(a.kcache + ok1 + (4 * i + tig) * 16) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t ov = __shfl_sync(0xffffffffu, off, tv[j]);
      const bool vv = (T.vmask >> tv[j]) & 1;
      const char* row = a.vcache + ov + gid * VSEG;
      if constexpr (NVW == 4) {
        const uint4 x = vv ? ld_stream_v4(row) : make_uint4(0, 0, 0, 0);
        T.vraw[j][0] = x.x; T.vraw[j][1] = x.y; T.vraw[j][2] = x.z; T.vraw[j][3] = x.w;
      } else {
        const uint2 x = vv ? ld_stream_v2(row) : make_uint2(0, 0);
        T.vraw[j][0] = x.x; T.vraw[j][1] = x.y;
      }
    }
  };

  auto consume = [&](int ts, const Tile& T) {
    if (T.vmask == 0) return;  // warp-uniform (ballot)
    const bool vk0 = (T.vmask >> gid) & 1, vk1 = (T.vmask >> (gid + 8)) & 1;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const uint32_t* r0 = reinterpret_cast<const uint32_t*>(&T.kraw[0][i]);
      const uint32_t* r1 = reinterpret_cast<const uint32_t*>(&T.kraw[1][i]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a0, a1, a2, a3;
        e4m3x4_to_f16x2x2(r0[w], a0, a2);
        e4m3x4_to_f16x2x2(r1[w], a1, a3);
        const int kk = 4 * i + w;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816<false>(s[nt], a0, a1, a2, a3, qf[nt][2 * kk], qf[nt][2 * kk + 1]);
      }
    }
    // V scales relative to vref; positive floats order as their bits
    const uint32_t vmaxb = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(T.vsc, 0.f)));
    if (__uint_as_float(vmaxb) > vref) {
      const float now = pow2_above(__uint_as_float(vmaxb));
      const float inv = 1.f / now;  // a power of two: exact
      const float f = vref * inv;
      if (f > 0.f) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int k = 0; k < 4; ++k) o_acc[nt][mt][k] *= f;
      }
      vref = now;
      inv_vref = inv;
    }
    const float ks0 = __shfl_sync(0xffffffffu, T.ksc, gid), ks1 = __shfl_sync(0xffffffffu, T.ksc, gid + 8);
    const float vs0 = __shfl_sync(0xffffffffu, T.vsc, gid) * inv_vref;
    const float vs1 = __shfl_sync(0xffffffffu, T.vsc, gid + 8) * inv_vref;
    uint32_t pb0[NT], pb1[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r0 = ts + gid, r1 = r0 + 8;
      const float x0 = vk0 && r0 < lim[nt][0] ? s[nt][0] * (colmul[nt][0] * ks0) : neg_inf();
      const float x1 = vk0 && r0 < lim[nt][1] ? s[nt][1] * (colmul[nt][1] * ks0) : neg_inf();
      const float x2 = vk1 && r1 < lim[nt][0] ? s[nt][2] * (colmul[nt][0] * ks1) : neg_inf();
      const float x3 = vk1 && r1 < lim[nt][1] ? s[nt][3] * (colmul[nt][1] * ks1) : neg_inf();
      const float mn0 = fmaxf(m_run[nt][0], warp_max_xor_rows(fmaxf(x0, x2)));
      const float mn1 = fmaxf(m_run[nt][1], warp_max_xor_rows(fmaxf(x1, x3)));
      const float ms0 = (mn0 == neg_inf()) ? 0.f : mn0;
      const float ms1 = (mn1 == neg_inf()) ? 0.f : mn1;
      const float al0 = exp2_approx(m_run[nt][0] - ms0), al1 = exp2_approx(m_run[nt][1] - ms1);
      const float p0 = exp2_approx(x0 - ms0), p2 = exp2_approx(x2 - ms0);
      const float p1 = exp2_approx(x1 - ms1), p3 = exp2_approx(x3 - ms1);
      l_run[nt][0] = l_run[nt][0] * al0 + p0 + p2;
      l_run[nt][1] = l_run[nt][1] * al1 + p1 + p3;
      m_run[nt][0] = mn0;
      m_run[nt][1] = mn1;
      // the factors are exactly 1 once the maxima settle
      if (__any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          o_acc[nt][mt][0] *= al0; o_acc[nt][mt][2] *= al0;
          o_acc[nt][mt][1] *= al1; o_acc[nt][mt][3] *= al1;
        }
      }
      pb0[nt] = movmatrix_trans(pack2<false>(p0 * vs0, p1 * vs0));
      pb1[nt] = movmatrix_trans(pack2<false>(p2 * vs1, p3 * vs1));
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int w = mt >> 1;
      const uint32_t sel = (mt & 1) ? 0x7362u : 0x5140u;
      uint32_t a0, a1, a2, a3;
      e4m3x4_to_f16x2x2(prmt(T.vraw[0][w], T.vraw[1][w], sel), a0, a1);
      e4m3x4_to_f16x2x2(prmt(T.vraw[2][w], T.vraw[3][w], sel), a2, a3);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma16816<false>(o_acc[nt][mt], a0, a1, a2, a3, pb0[nt], pb1[nt]);
    }
  };

  for (int ts = t0 + warp * kMqTile; ts < t1; ts += kMqWarps * kMqTile) {
    Tile T;
    fetch(ts, T, ent);
    entry(ts + kMqWarps * kMqTile, ent);  // the next tile's look-up overlaps this tile's loads and math
    consume(ts, T);
  }

  // ---- join the four warps ------------------------------------------------
  auto sO = reinterpret_cast<float(*)[NC][D]>(dsm);
  auto sM = reinterpret_cast<float(*)[NC]>(dsm + kMqWarps * NC * D * 4);
  auto sL = reinterpret_cast<float(*)[NC]>(dsm + kMqWarps * NC * D * 4 + kMqWarps * NC * 4);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float l0 = warp_sum_xor_rows(l_run[nt][0]), l1 = warp_sum_xor_rows(l_run[nt][1]);
    const int c = 2 * tig + 8 * nt;
    if (gid == 0) {
      sM[warp][c] = m_run[nt][0]; sM[warp][c + 1] = m_run[nt][1];
      sL[warp][c] = l0; sL[warp][c + 1] = l1;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int d0 = gid * VSEG + 2 * mt, d1 = d0 + 1;
      sO[warp][c][d0] = o_acc[nt][mt][0] * vref;
      sO[warp][c + 1][d0] = o_acc[nt][mt][1] * vref;
      sO[warp][c][d1] = o_acc[nt][mt][2] * vref;
      sO[warp][c + 1][d1] = o_acc[nt][mt][3] * vref;
    }
  }
  __syncthreads();
  for (int idx = tid; idx < cols * (D / 4); idx += kMqThreads) {
    const int c = idx / (D / 4), d4 = (idx % (D / 4)) * 4;
    float M = neg_inf();
#pragma unroll
    for (int w = 0; w < kMqWarps; ++w) M = fmaxf(M, sM[w][c]);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kMqWarps; ++w) {
      const float f = (sM[w][c] == neg_inf()) ? 0.f : exp2_approx(sM[w][c] - M);
      L += f * sL[w][c];
      const float4 o = *reinterpret_cast<const float4*>(&sO[w][c][d4]);
      acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w;
    }
    if (whole) {
      const float inv = 1.f / L;  // no visible key: 0 / 0, as the softmax over nothing
      const int cg = c0 + c, s = cg / a.G, g = cg - s * a.G;
      *reinterpret_cast<uint2*>(a.out + b * a.os_b + h * a.os_h + g * a.os_g + s * a.os_s + d4 * 2) =
          make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
    } else {
      *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * NC + c) * D + d4) = acc;
      if (d4 == 0) a.part_ml[(int64_t)slot * NC + c] = make_float2(M, L);
    }
  }
  __syncthreads();  // the area is reused by the CTA's next segment
}

// Walks the share [lo, hi) of the list of all units (head-major, items in
// order; unit (h, i) covers [h T + P[i], h T + P[i + 1])), calling
// seg(h, item, L, t0, t1, whole, slot) for each segment with keys, or with an
// empty unit's start, and leaves the CTA's descriptors in a.desc.
template <typename Keys, typename Seg>
__device__ __forceinline__ void walk_share(const Fp8Args& a, const int* P, int64_t lo, int64_t hi, Keys keys, Seg seg) {
  const int64_t T = P[a.items];
  int cont = -1, start = -1;
  const int64_t first = lo;
  while (lo < hi) {
    const int h = (int)(lo / T);
    const int x = (int)(lo - h * T);
    int i = 0, j = a.items - 1;  // last item that starts at or before x
    while (i < j) {
      const int mid = (i + j + 1) >> 1;
      if (P[mid] <= x) i = mid; else j = mid - 1;
    }
    const int64_t u0 = h * T + P[i] + kSegCost, u1 = h * T + P[i + 1];
    const int64_t seg_lo = lo > u0 ? lo : u0, seg_hi = hi < u1 ? hi : u1;
    const bool starts = lo == u0 - kSegCost;
    const int L = keys(i);
    const int unit = h * a.items + i;
    lo = seg_hi > lo ? seg_hi : (hi < u1 ? hi : u1);
    if (L == 0) {
      if (starts) seg(h, i, 0, 0, 0, true, 0);
      continue;
    }
    if (seg_lo >= seg_hi) continue;  // only virtual keys of the unit are in this share
    const int t0 = (int)(seg_lo - u0), t1 = (int)min(seg_hi - u0, (int64_t)L);
    const bool head = t0 == 0, whole = head && t1 == L;
    if (!whole) {
      if (head) start = unit; else cont = unit;
    }
    seg(h, i, L, t0, t1, whole, 2 * (int)blockIdx.x + (head ? 1 : 0));
  }
  (void)first;
  if (threadIdx.x == 0) {
    a.desc[2 * blockIdx.x] = cont;
    a.desc[2 * blockIdx.x + 1] = start;
  }
}

template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(kMqThreads, NT == 1 ? 4 : 2) paged_attn_fp8_rows_kernel(const Fp8Args a) {
  extern __shared__ __align__(16) unsigned char dsm[];
  constexpr int NC = 8 * NT;
  dependents_enter();
  auto keys = [&](int i) {
    const int b = i / a.tiles, t = i - b * a.tiles;
    return item_keys(a, b, (int)(((int64_t)(t + 1) * NC - 1) / a.G));
  };
  auto seg = [&](int h, int i, int L, int t0, int t1, bool whole, int slot) {
    const int b = i / a.tiles;
    mq_segment<D, BF16, NT>(a, dsm, b, h, i - b * a.tiles, t0, t1, whole, slot);
  };
  if (blockIdx.x == 0 && a.err)
    for (int b = threadIdx.x; b < a.B; b += kMqThreads)
      if (a.seq[b * a.seq_stride] < 0) atomicOr(a.err, RBLN_DEVERR_SEQ_RANGE);
  if (!a.balanced) {
    const int64_t units = (int64_t)a.items * a.Hkv;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
      const int i = (int)(u / a.Hkv), h = (int)(u - (int64_t)i * a.Hkv);
      const int L = keys(i);
      seg(h, i, L, 0, L, true, 0);
    }
    return;
  }
  int* P = reinterpret_cast<int*>(dsm + kMqWarps * NC * (D * 4 + 8));
  cost_prefix<kMqThreads>(a, NC, P);
  const int64_t total = (int64_t)P[a.items] * a.Hkv;
  int64_t W = ((total + gridDim.x - 1) / gridDim.x + 15) & ~(int64_t)15;
  if (W < kMinW) W = kMinW;
  const int64_t lo = min(W * blockIdx.x, total);
  walk_share(a, P, lo, min(lo + W, total), keys, seg);
}

// Joins the partial results of the units that several CTAs share. CTA (c, y):
// the chain that CTA c of the attention kernel starts, in parts c, c + 1, ...
// while those continue the same unit; 8 warps = RPC rows x KS slices of the
// chain, a lane holding 4 (D = 128) or 2 dimensions of its row.
template <int D, bool BF16, int ROWS, int RPC>
__global__ void __launch_bounds__(256) paged_attn_fp8_merge_kernel(const Fp8Args a, int n_cta, int qt) {
  constexpr int KS = 8 / RPC, E = D / 32;
  __shared__ float so[8][D];
  __shared__ float2 sml[8];
  __shared__ int s_len;
  dependents_enter();
  const int c = blockIdx.x;
  const int unit = a.desc[2 * c + 1];
  if (unit < 0) return;
  if (threadIdx.x == 0) s_len = n_cta - c - 1;
  __syncthreads();
  for (int i = threadIdx.x; c + 1 + i < n_cta; i += 256)
    if (a.desc[2 * (c + 1 + i)] != unit) {
      atomicMin(&s_len, i);
      break;
    }
  __syncthreads();
  const int parts = s_len + 1;  // the chain's start and the parts that follow
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.y * RPC + warp % RPC, slice = warp / RPC;
  float M = neg_inf(), L = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  constexpr int U = 4;
  for (int i0 = slice; i0 < parts; i0 += U * KS) {
    float2 ml[U];
    float o[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * KS;
      ml[u] = make_float2(neg_inf(), 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) o[u][e] = 0.f;
      if (i < parts) {
        const int64_t at = ((int64_t)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * ROWS + row);
        ml[u] = a.part_ml[at];
        if constexpr (E == 4) {
          const float4 v = *reinterpret_cast<const float4*>(a.part_o + at * D + lane * 4);
          o[u][0] = v.x; o[u][1] = v.y; o[u][2] = v.z; o[u][3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(a.part_o + at * D + lane * 2);
          o[u][0] = v.x; o[u][1] = v.y;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ml[u].x == neg_inf()) continue;
      const float mn = fmaxf(M, ml[u].x);
      const float f0 = exp2_approx(M - mn), f1 = exp2_approx(ml[u].x - mn);
      M = mn;
      L = L * f0 + ml[u].y * f1;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * f0 + o[u][e] * f1;
    }
  }
  if (KS > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = acc[e];
    if (lane == 0) sml[warp] = make_float2(M, L);
    __syncthreads();
    if (slice != 0) return;
    for (int k = 1; k < KS; ++k) {
      const float2 ml = sml[warp + k * RPC];
      if (ml.x == neg_inf()) continue;
      const float mn = fmaxf(M, ml.x);
      const float f0 = exp2_approx(M - mn), f1 = exp2_approx(ml.x - mn);
      M = mn;
      L = L * f0 + ml.y * f1;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * f0 + so[warp + k * RPC][lane * E + e] * f1;
    }
  }
  const int h = unit / a.items, i = unit - h * a.items;
  const int b = i / a.tiles, tile = i - b * a.tiles;
  int s, g;
  if (qt == 0) {  // rows in the order s G + g
    const int cg = tile * ROWS + row;
    s = cg / a.G;
    g = cg - s * a.G;
  } else {  // 128-row tiles of G heads x qt tokens
    const int r = row & 127;
    g = r / qt;
    s = (tile * (ROWS / 128) + (row >> 7)) * qt + r - g * qt;
  }
  if (g >= a.G || s >= a.S) return;
  const float inv = 1.f / L;
  char* to = a.out + b * a.os_b + h * a.os_h + g * a.os_g + s * a.os_s + lane * E * 2;
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(to) =
        make_uint2(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(to) = pack2<BF16>(acc[0] * inv, acc[1] * inv);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct Fp8Plan {
  int nt;       // 8-column groups of the row kernel
  int rows;     // rows of a row tile
  int tiles, items;
  bool balanced;
  int ctas;
  size_t desc, ml, o, total;  // workspace regions
};

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

int plan_fp8(const rbln_paged_attn_params_t* p, Fp8Plan* pl) {
  const int64_t span = (int64_t)p->max_blocks * p->block_size;
  const int64_t rows = (int64_t)p->q_len * p->group;
  pl->nt = rows <= 8 ? 1 : 2;
  pl->rows = 8 * pl->nt;
  const int64_t tiles = (rows + pl->rows - 1) / pl->rows;
  if (tiles * p->batch * p->num_kv_heads > INT32_MAX) return RBLN_ERR_UNSUPPORTED;
  pl->tiles = (int)tiles;
  pl->items = (int)(tiles * p->batch);
  const int64_t slots = 148LL * (pl->nt == 1 ? 4 : 2);
  // the prefix fits shared memory and counts in 32 bits; with more items than
  // that there are enough whole units for every CTA
  pl->balanced = pl->items <= kMaxItems && (int64_t)pl->items * (span + 16 + kSegCost) < INT32_MAX;
  const int64_t units = (int64_t)pl->items * p->num_kv_heads;
  pl->ctas = (int)(pl->balanced ? slots : std::min<int64_t>(units, slots * 8));
  size_t off = 0;
  if (pl->balanced) {
    pl->desc = off;
    off += round256((size_t)2 * pl->ctas * sizeof(int));
    pl->ml = off;
    off += round256((size_t)2 * pl->ctas * pl->rows * sizeof(float2));
    pl->o = off;
    off += round256((size_t)2 * pl->ctas * pl->rows * p->head_dim * sizeof(float));
  }
  pl->total = off ? off + 256 : 0;
  return RBLN_OK;
}

template <typename... A>
int launch_after(void (*kernel)(A...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? RBLN_OK : RBLN_ERR_LAUNCH;
}

template <int D, bool BF16, int NT>
int launch_rows(const Fp8Args& a, const Fp8Plan& pl, cudaStream_t st) {
  const size_t smem = (size_t)kMqWarps * pl.rows * (D * 4 + 8) + (pl.balanced ? (pl.items + 1) * sizeof(int) : 0);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(paged_attn_fp8_rows_kernel<D, BF16, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)smem) != cudaSuccess)
    return RBLN_ERR_LAUNCH;
  int rc = launch_after(paged_attn_fp8_rows_kernel<D, BF16, NT>, dim3(pl.ctas), kMqThreads, smem, st, a);
  if (rc != RBLN_OK || !pl.balanced) return rc;
  return launch_after(paged_attn_fp8_merge_kernel<D, BF16, 8 * NT, 4>, dim3(pl.ctas, 2 * NT), 256, 0, st, a, pl.ctas, 0);
}

template <int D, bool BF16>
int launch_fp8(const Fp8Args& a, const Fp8Plan& pl, cudaStream_t st) {
  return pl.nt == 1 ? launch_rows<D, BF16, 1>(a, pl, st) : launch_rows<D, BF16, 2>(a, pl, st);
}

int check_shapes(const rbln_paged_attn_params_t* p) {
  if (!p || p->batch < 0 || p->num_kv_heads <= 0 || p->group <= 0 || p->block_size <= 0 || p->max_blocks <= 0 ||
      p->num_blocks <= 0 || p->q_len < 0)
    return RBLN_ERR_INVALID_ARGUMENT;
  if (p->head_dim != 64 && p->head_dim != 128) return RBLN_ERR_UNSUPPORTED;
  if (p->group > 128) return RBLN_ERR_UNSUPPORTED;
  const int bs = p->block_size;
  if (!((bs >= 8 && bs <= 128 && 128 % bs == 0) || bs % 128 == 0)) return RBLN_ERR_UNSUPPORTED;
  if ((int64_t)p->max_blocks * bs > (1 << 30) || p->q_len > (1 << 30)) return RBLN_ERR_UNSUPPORTED;
  return RBLN_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

// Scratch of the fp8 form (called by rbln_paged_prefill_workspace_size).
size_t fp8_prefill_ws_bytes(const rbln_paged_attn_params_t* p) {
  Fp8Plan pl{};
  if (check_shapes(p) != RBLN_OK || p->batch == 0 || p->q_len == 0 || plan_fp8(p, &pl) != RBLN_OK) return 0;
  return pl.total;
}

// The kv_dtype FP8_E4M3 form of rbln_paged_causal_attn_prefill.
int run_prefill_fp8(const rbln_paged_attn_params_t* p, cudaStream_t st) {
  int rc = check_shapes(p);
  if (rc != RBLN_OK) return rc;
  if (p->q_dtype != RBLN_DT_BF16 && p->q_dtype != RBLN_DT_F16) return RBLN_ERR_UNSUPPORTED;
  if (p->sinks) return RBLN_ERR_UNSUPPORTED;
  if (p->block_table_dtype != RBLN_DT_I16 && p->block_table_dtype != RBLN_DT_I32 &&
      p->block_table_dtype != RBLN_DT_I64)
    return RBLN_ERR_UNSUPPORTED;
  if (p->batch == 0 || p->q_len == 0) return RBLN_OK;
  if (!p->q || !p->out || !p->kcache || !p->vcache || !p->seq || !p->block_table || !p->k_scale || !p->v_scale ||
      (p->k_new == nullptr) != (p->v_new == nullptr))
    return RBLN_ERR_INVALID_ARGUMENT;
  if (!aligned16(p->q) || !aligned16(p->out) || !aligned16(p->kcache) || !aligned16(p->vcache))
    return RBLN_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 4; ++i)
    if (p->q_stride[i] % 8 || p->out_stride[i] % 8) return RBLN_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (p->cache_stride[i] % 16) return RBLN_ERR_INVALID_ARGUMENT;
  Fp8Plan pl{};
  rc = plan_fp8(p, &pl);
  if (rc != RBLN_OK) return rc;
  if (pl.total > 0 && (!p->workspace || p->workspace_bytes < pl.total)) return RBLN_ERR_WORKSPACE;
  if (p->k_new) {
    rc = rbln_paged_kv_write(p, st);
    if (rc != RBLN_OK) return rc;
  }
  Fp8Args a{};
  a.q = static_cast<const char*>(p->q);
  a.qs_b = p->q_stride[0] * 2; a.qs_h = p->q_stride[1] * 2; a.qs_g = p->q_stride[2] * 2; a.qs_s = p->q_stride[3] * 2;
  a.out = static_cast<char*>(p->out);
  a.os_b = p->out_stride[0] * 2; a.os_h = p->out_stride[1] * 2; a.os_g = p->out_stride[2] * 2; a.os_s = p->out_stride[3] * 2;
  a.kcache = static_cast<const char*>(p->kcache);
  a.vcache = static_cast<const char*>(p->vcache);
  a.cs_block = p->cache_stride[0]; a.cs_head = p->cache_stride[1]; a.cs_tok = p->cache_stride[2];
  a.k_scale = p->k_scale; a.v_scale = p->v_scale;
  a.ss_block = p->scale_stride[0]; a.ss_head = p->scale_stride[1];
  a.seq = p->seq; a.seq_stride = p->seq_stride;
  a.bt = p->block_table; a.bt_dtype = p->block_table_dtype; a.bt_stride = p->block_table_stride;
  a.mask = p->mask; a.mask_dtype = p->mask_dtype; a.mask_len = p->mask_len; a.mask_stride = p->mask_stride[0];
  a.scale = p->scale; a.scale_dev = p->scale_dev;
  a.B = p->batch; a.Hkv = p->num_kv_heads; a.G = p->group; a.S = p->q_len;
  a.num_blocks = p->num_blocks; a.bs = p->block_size; a.max_blocks = p->max_blocks;
  a.span = p->max_blocks * p->block_size;
  a.causal = p->causal;
  a.tiles = pl.tiles; a.items = pl.items;
  a.balanced = pl.balanced;
  if (pl.balanced) {
    char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p->workspace) + 255) & ~uintptr_t(255));
    a.desc = reinterpret_cast<int*>(base + pl.desc);
    a.part_ml = reinterpret_cast<float2*>(base + pl.ml);
    a.part_o = reinterpret_cast<float*>(base + pl.o);
  }
  a.err = p->error_flags;
  if (p->prof_events[0]) cudaEventRecord(static_cast<cudaEvent_t>(p->prof_events[0]), st);
  const bool bf = p->q_dtype == RBLN_DT_BF16;
  if (p->head_dim == 128) rc = bf ? launch_fp8<128, true>(a, pl, st) : launch_fp8<128, false>(a, pl, st);
  else rc = bf ? launch_fp8<64, true>(a, pl, st) : launch_fp8<64, false>(a, pl, st);
  if (p->prof_events[1]) cudaEventRecord(static_cast<cudaEvent_t>(p->prof_events[1]), st);
  return rc;
}

}  // namespace rbln

// Attention of S_q new tokens a sequence over an fp8-e4m3 paged KV cache with
// one fp32 scale for each (block, KV head): the kv_dtype FP8_E4M3 form of
// rbln_paged_causal_attn_prefill. The new rows are written first, as
// rbln_paged_kv_write writes them (scales of touched blocks found anew, but as
// amax * (1 / 448)), and read back with the rest.
//
//   out[s] = sum_t p_st v_t / sum_t p_st,  p_st = exp(scale q_s . k_t)
// over the keys t <= seq[b] + s (causal) or t < seq[b] + S_q (both ways) that
// the position mask, where there is one, keeps. With k_t = ks c_t and
// v_t = vs d_t, c and d the e4m3 codes of a block and ks, vs its scales, the
// products run on the codes: every code is exact in f16, ks multiplies the
// score in float32 and vs the probability, which is rounded to f16 once.
// Few rows: a bf16 query goes to f16 with a power of two of its row, so that
// its largest magnitude lies in [2^14, 2^15): exact down to 2^-28 of the row's
// largest. Many rows: the keys go to bf16 instead, exact too.
// The probabilities' vs is taken relative to a running power of two (vref) at
// or above the largest scale that the row has seen, so a cache of small values
// keeps all of f16's bits and one of large values cannot overflow; the row's
// accumulator is rescaled when vref grows. It is each row's own: what a row may
// not see costs it nothing (but see kFarBelow). A block whose scale is far
// below vref keeps its probabilities to 2^-25 of vref each, so T keys err by T
// 2^-25 of the largest value that the row sees at most.
// The running maximum, the sums and the accumulators are float32, and the
// accumulators stay relative to vref until their mean is taken: sums of values
// near float32's largest would pass it.

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "sm100.cuh"
#include "tma_map.cuh"

namespace rbln {

int kv_write(const rbln_paged_attn_params_t* p, cudaStream_t stream, bool reciprocal);  // kv_write.cu

namespace {

constexpr int kMqWarps = 4;
constexpr int kMqThreads = kMqWarps * 32;
constexpr int kMqTile = 32;     // keys a warp's tile
// Virtual keys charged to each unit's start: 64, 128, 256, 384, 512 took 111,
// 108, 103, 103, 103 us for 64 sequences of 4 tokens behind 128 to 4096 keys.
constexpr int kSegCost = 256;
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
  uint32_t bs_mul, bs_shift;  // n / bs = (mulhi(n, bs_mul) + n) >> bs_shift
  int causal;
  int tiles, items;  // row tiles a sequence; items = B * tiles
  int balanced;      // 1: the keys of all units cut into equal shares; 0: whole units, grid-strided
  // balanced: desc[2c], desc[2c + 1] = the unit that CTA c continues / starts
  // without finishing (-1: none), with its partial result in the same slot
  int* desc;
  float* part_o;   // [2 nCTA][rows][D], relative to 2^m and vref
  float4* part_ml; // [2 nCTA][rows]: (m, l, vref, 0)
  uint32_t* err;
};

__device__ __forceinline__ int div_bs(const Fp8Args& a, int n) {
  return (int)((__umulhi((uint32_t)n, a.bs_mul) + (uint32_t)n) >> a.bs_shift);  // n < 2^30: no carry
}

__device__ __forceinline__ void dependents_enter() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// The smallest power of two at or above x, within [2^-126, 2^126]: those have a
// normal reciprocal, and no float is over four times the largest.
__device__ __forceinline__ float pow2_above(float x) {
  x = fminf(fmaxf(x, 1.1754944e-38f), 8.5070592e37f);
  return __uint_as_float((__float_as_uint(x) + 0x007fffffu) & 0x7f800000u);
}

// Reciprocal of a power of two that pow2_above gave; 2^127 for zero, which
// stands for no scale yet.
__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

// vref is held above this times the largest scale behind the row's limit, so
// that the ratio of the two stays finite (and zero times it is zero). That
// costs the row bits only where what it may not see is 2^112 times larger.
constexpr float kFarBelow = 1.1754944e-38f;  // 2^-126

// Power of two that brings a row's largest magnitude m to [2^14, 2^15), and
// its inverse; 1 for rows of zeros, infinities or NaN.
__device__ __forceinline__ float f16_factor(float m, float& undo) {
  undo = 1.f;
  if (!(m > 0.f && m <= 3.4028235e38f)) return 1.f;
  const int e = (int)(__float_as_uint(m) >> 23) - 127;  // m in [2^e, 2^(e+1)), or subnormal
  const int k = min(max(14 - e, -120), 120);
  undo = __uint_as_float((uint32_t)(127 - k) << 23);
  return __uint_as_float((uint32_t)(127 + k) << 23);
}

// Keys [0, L) that some row of item's row tile may see; `last` is the tile's last token.
__device__ __forceinline__ int item_keys(const Fp8Args& a, int b, int last) {
  const int pos = a.seq[b * a.seq_stride];
  if (pos < 0) return 0;
  const int64_t end = (int64_t)pos + (a.causal ? min(last, a.S - 1) + 1 : a.S);
  return (int)min(end, (int64_t)a.span);
}

// Exclusive prefix P[0..items] of the items' costs, by the whole CTA: keys
// rounded up to a multiple of `unit`, in units of it, plus `seg` for the
// unit's start. keys(i): keys of item i.
template <int THREADS, typename Keys>
__device__ __forceinline__ void cost_prefix(const Fp8Args& a, int unit, int scale, int seg, Keys keys, int* wsum,
                                            int* P) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.items + THREADS - 1) / THREADS;
  const int first = tid * per;
  auto cost = [&](int i) { return (keys(i) + unit - 1) / unit * scale + seg; };
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
// Few rows (S_q G up to 16 of a KV head): one read of the cached bytes. As in
// the one-token decode, tokens are the M side of mma.m16n8k16 and the rows
// (token s, head g), s G + g, the N side, so that a tile's codes go from
// shared memory to f16 fragments in registers; four warps take 32-key tiles
// round-robin, each with a ring of two filled by cp.async, and are joined in
// shared memory. The keys of all (head, sequence) units are cut into equal
// shares, one CTA each, three CTAs an SM (two: 110 us against 102 for 64
// sequences of 4 tokens, G = 4, 8 KV heads, behind 128 to 4096 keys). There it
// takes 107 us with its merge and reads 2.7 TB/s, 41 % of the copy rate:
// latency of 12 warps an SM and the segments' starts bound it (copies alone 82
// us, products alone 77). Issue slots are busy 37 % of the time; of the 7.7
// cycles from one instruction of a warp to its next 1.7 are for the one before,
// 1.4 for long loads, 1.2 for the next to be fetched, 0.9 for shared memory.
// ---------------------------------------------------------------------------
// A warp's ring of tiles in shared memory, filled by cp.async. Rows are
// swizzled by 16-byte chunks so that the fragments' loads meet no bank twice:
// K fragments take rows gid and gid + 8, four neighbouring chunks at once, V
// fragments rows 2 tig (+ 1, + 8, + 9), one piece of each.
template <int D>
struct MqRing {
  static constexpr int STAGES = 2;
  static constexpr int K = 0, V = kMqTile * D, KS = 2 * kMqTile * D, VS = KS + 4 * kMqTile, MASK = VS + 4 * kMqTile;
  static constexpr int STAGE = MASK + 32;
  static constexpr int WARP = STAGES * STAGE;
  static __device__ __forceinline__ int k_at(int row, int chunk) {
    return row * D + ((D == 128 ? chunk ^ ((row & 1) << 2) : chunk) << 4);
  }
  static __device__ __forceinline__ int v_at(int row, int chunk) {
    if (D == 128) return row * D + ((chunk ^ (((row >> 1) & 3) << 1)) << 4);
    const int slot = (row & 16) + (row & 1) * 8 + ((row & 15) >> 1);
    return slot * D + ((chunk ^ (((slot >> 1) & 1) << 1)) << 4);
  }
};
// 16 (or 4) bytes global -> shared in the background; zeros when not `valid`.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int D, bool BF16, int NT>
__device__ __forceinline__ void mq_segment(const Fp8Args& a, unsigned char* dsm, int b, int h, int tile, int t0,
                                           int t1, bool whole, int slot) {
  constexpr int KCH = D / 64, KR = D / 8, VSEG = D == 128 ? 16 : 8, NVW = D / 32, MT = D / 16, NC = 8 * NT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int c0 = tile * NC, cols = min(NC, a.S * a.G - c0);
  const int pos = a.seq[b * a.seq_stride];

  // Row offset, in 16-byte units, of this lane's key ts + lane and its place
  // in the scales; at = -1 for a key that is not seen.
  struct Entry {
    uint32_t off;
    int at;
  };
  auto entry = [&](int ts, Entry& e) {
    const int t = ts + lane;
    e.at = -1;
    if (t < t1) {
      const int bi = div_bs(a, t);
      const int64_t blk = load_index(a.bt, a.bt_dtype, b * a.bt_stride + bi);
      const bool keep =
          a.mask == nullptr || (t < a.mask_len && load_keep(a.mask, a.mask_dtype, b * a.mask_stride + t));
      if (blk >= 0 && blk < a.num_blocks) {
        if (keep) e.at = (int)blk;
        e.off = (uint32_t)((blk * a.cs_block + h * a.cs_head + (t - bi * a.bs) * a.cs_tok) >> 4);
      } else if (a.err) {
        atomicOr(a.err, RBLN_DEVERR_BLOCK_ID_RANGE);
      }
    }
  };
  using R = MqRing<D>;
  unsigned char* ring = dsm + warp * R::WARP;
  const uint32_t ring_s = smem_u32(ring);
  // issues the copies of the tile of entry e into stage st
  auto issue = [&](int st, const Entry& e) {
    const uint32_t to = ring_s + st * R::STAGE;
    const bool valid = e.at >= 0;
    const uint32_t vmask = __ballot_sync(0xffffffffu, valid);
    if (lane == 0) *reinterpret_cast<uint32_t*>(ring + st * R::STAGE + R::MASK) = vmask;
    if (vmask != 0) {
      const int64_t so = valid ? e.at * a.ss_block + h * a.ss_head : 0;
      copy4(to + R::KS + lane * 4, a.k_scale + so, valid);
      copy4(to + R::VS + lane * 4, a.v_scale + so, valid);
      constexpr int CPR = D / 16, RPI = 32 / CPR;  // chunks a row, rows a step
      const int c = lane % CPR;
#pragma unroll
      for (int k = 0; k < kMqTile / RPI; ++k) {
        const int row = k * RPI + lane / CPR;
        const uint32_t ro = __shfl_sync(0xffffffffu, e.off, row);
        const bool ok = (vmask >> row) & 1;
        const size_t at = ok ? (size_t)ro * 16 + c * 16 : 0;
        copy16(to + R::K + R::k_at(row, c), a.kcache + at, ok);
        copy16(to + R::V + R::v_at(row, c), a.vcache + at, ok);
      }
    }
    copy_commit();
  };
  // the first tiles on their way before the queries are looked at
  const int step = kMqWarps * kMqTile, first = t0 + warp * kMqTile;
  static_assert(R::STAGES == 2, "one tile ahead");
  Entry e0, ent;
  entry(first, e0);
  entry(first + step, ent);  // both look-ups at once
  if (first < t1) issue(0, e0);
  else copy_commit();

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
        const float up = f16_factor(qmax, undo[nt]);
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
  // keys below this are every live row's (their columns' limits)
  const int all_lim = a.causal ? (int)min((int64_t)pos + c0 / a.G + 1, (int64_t)t1) : t1;
  // Each column's power of two at or above every V scale that it has seen, as
  // its exponent in a byte (0: none yet).
  uint32_t vexp = 0;
  auto vref = [&](int nt, int k) { return __uint_as_float((vexp >> (16 * nt + 8 * k) & 0xffu) << 23); };

  auto consume = [&](int ts, int st) {
    const unsigned char* stage = ring + st * R::STAGE;
    const uint32_t vmask = *reinterpret_cast<const uint32_t*>(stage + R::MASK);
    if (vmask == 0) return;  // the same for the whole warp
    const float* ks = reinterpret_cast<const float*>(stage + R::KS);
    const float* vs = reinterpret_cast<const float*>(stage + R::VS);
    // scores of keys gid + 8 r (r = 0..3): s[nt][2 r + k], column 2 tig + k
    float s[NT][8];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[nt][k] = 0.f;
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      uint4 kr[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        kr[r] = *reinterpret_cast<const uint4*>(stage + R::K + R::k_at(8 * r + gid, 4 * i + tig));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int kk = 4 * i + w;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          uint32_t a0, a1, a2, a3;
          e4m3x4_to_f16x2x2(reinterpret_cast<const uint32_t*>(&kr[2 * sub])[w], a0, a2);
          e4m3x4_to_f16x2x2(reinterpret_cast<const uint32_t*>(&kr[2 * sub + 1])[w], a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<false>(reinterpret_cast<float(&)[4]>(s[nt][4 * sub]), a0, a1, a2, a3, qf[nt][2 * kk],
                            qf[nt][2 * kk + 1]);
        }
      }
    }
    const bool inside = ts + kMqTile <= all_lim;  // no key behind a live column's limit
    float ksc[4], vsc[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      ksc[r] = ks[gid + 8 * r];
      vsc[r] = vs[gid + 8 * r];
    }
    // the tile's largest V scale; positive floats order as their bits
    const float vmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(vs[lane], 0.f))));
    // A lane's first column is of its earliest token and sees no more than the
    // others; while all tiles are inside, they are all alike.
    if (__any_sync(0xffffffffu, vmax > vref(0, 0))) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float m = vmax;
          if (!inside) {  // the largest that this column sees
            m *= kFarBelow;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (ts + gid + 8 * r < lim[nt][k]) m = fmaxf(m, vsc[r]);
            m = warp_max_xor_rows(m);
          }
          const float was = vref(nt, k), now = m > was ? pow2_above(m) : was;
          const float f = was * pow2_inverse(now);  // zero where what is held is too small to count
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            o_acc[nt][mt][k] *= f;
            o_acc[nt][mt][2 + k] *= f;
          }
          const int at = 16 * nt + 8 * k;
          vexp = (vexp & ~(0xffu << at)) | (__float_as_uint(now) >> 23 << at);
        }
    }
    {
      const float inv = pow2_inverse(vref(0, 0));
#pragma unroll
      for (int r = 0; r < 4; ++r) vsc[r] = inside ? vsc[r] * inv : 1.f;  // 1: by each column's own, below
    }
    const bool whole_tile = vmask == 0xffffffffu && inside;
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k) s[nt][2 * r + k] *= colmul[nt][k] * ksc[r];
      if (!whole_tile) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (!((vmask >> (gid + 8 * r)) & 1u) || ts + gid + 8 * r >= lim[nt][k]) s[nt][2 * r + k] = neg_inf();
      }
      float al[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float mx = fmaxf(fmaxf(s[nt][k], s[nt][2 + k]), fmaxf(s[nt][4 + k], s[nt][6 + k]));
        const float mn = fmaxf(m_run[nt][k], warp_max_xor_rows(mx));
        const float ms = (mn == neg_inf()) ? 0.f : mn;
        al[k] = exp2_approx(m_run[nt][k] - ms);
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[nt][2 * r + k] = exp2_approx(s[nt][2 * r + k] - ms);
          sum += s[nt][2 * r + k];
        }
        l_run[nt][k] = l_run[nt][k] * al[k] + sum;
        m_run[nt][k] = mn;
      }
      // the factors are exactly 1 once the maxima settle
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          o_acc[nt][mt][0] *= al[0]; o_acc[nt][mt][2] *= al[0];
          o_acc[nt][mt][1] *= al[1]; o_acc[nt][mt][3] *= al[1];
        }
      }
      if (!inside) {
        const float inv[2] = {pow2_inverse(vref(nt, 0)), pow2_inverse(vref(nt, 1))};
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int k = 0; k < 2; ++k) s[nt][2 * r + k] *= vs[gid + 8 * r] * inv[k];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        pb[r >> 1][nt][r & 1] =
            movmatrix_trans(pack2<false>(s[nt][2 * r] * vsc[r], s[nt][2 * r + 1] * vsc[r]));
    }
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      uint32_t vraw[4][NVW];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 16 * sub + 2 * tig + (j & 1) + (j >> 1) * 8;
        if constexpr (NVW == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(stage + R::V + R::v_at(row, gid));
          vraw[j][0] = x.x; vraw[j][1] = x.y; vraw[j][2] = x.z; vraw[j][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(stage + R::V + R::v_at(row, gid >> 1) + (gid & 1) * 8);
          vraw[j][0] = x.x; vraw[j][1] = x.y;
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int w = mt >> 1;
        const uint32_t sel = (mt & 1) ? 0x7362u : 0x5140u;
        uint32_t a0, a1, a2, a3;
        e4m3x4_to_f16x2x2(prmt(vraw[0][w], vraw[1][w], sel), a0, a1);
        e4m3x4_to_f16x2x2(prmt(vraw[2][w], vraw[3][w], sel), a2, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816<false>(o_acc[nt][mt], a0, a1, a2, a3, pb[sub][nt][0], pb[sub][nt][1]);
      }
    }
  };

  int st = 0;
  for (int ts = first; ts < t1; ts += step) {
    if (ts + step < t1) issue(st ^ 1, ent);
    else copy_commit();
    entry(ts + 2 * step, ent);  // the look-up of the tile after it
    copy_wait<1>();
    __syncwarp();
    consume(ts, st);
    __syncwarp();
    st ^= 1;
  }
  copy_wait<0>();
  __syncwarp();

  // ---- join the four warps ------------------------------------------------
  // a warp's O and its vrefs lie over its own ring; the maxima and sums behind all rings
  static_assert(NC * (D + 1) * 4 <= R::WARP, "O over the ring");
  auto sO = [&](int w) { return reinterpret_cast<float(*)[D]>(dsm + w * R::WARP); };
  auto sV = [&](int w) { return reinterpret_cast<float*>(dsm + w * R::WARP + NC * D * 4); };
  auto sM = reinterpret_cast<float(*)[NC]>(dsm + kMqWarps * R::WARP);
  auto sL = reinterpret_cast<float(*)[NC]>(dsm + kMqWarps * R::WARP + kMqWarps * NC * 4);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float l0 = warp_sum_xor_rows(l_run[nt][0]), l1 = warp_sum_xor_rows(l_run[nt][1]);
    const int c = 2 * tig + 8 * nt;
    if (gid == 0) {
      sM[warp][c] = m_run[nt][0]; sM[warp][c + 1] = m_run[nt][1];
      sL[warp][c] = l0; sL[warp][c + 1] = l1;
      sV(warp)[c] = vref(nt, 0); sV(warp)[c + 1] = vref(nt, 1);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int d0 = gid * VSEG + 2 * mt, d1 = d0 + 1;
      sO(warp)[c][d0] = o_acc[nt][mt][0];
      sO(warp)[c + 1][d0] = o_acc[nt][mt][1];
      sO(warp)[c][d1] = o_acc[nt][mt][2];
      sO(warp)[c + 1][d1] = o_acc[nt][mt][3];
    }
  }
  __syncthreads();
  for (int idx = tid; idx < cols * (D / 4); idx += kMqThreads) {
    const int c = idx / (D / 4), d4 = (idx % (D / 4)) * 4;
    float M = neg_inf(), up = 0.f;
#pragma unroll
    for (int w = 0; w < kMqWarps; ++w) {
      M = fmaxf(M, sM[w][c]);
      up = fmaxf(up, sV(w)[c]);
    }
    const float down = pow2_inverse(up);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kMqWarps; ++w) {
      float f = (sM[w][c] == neg_inf()) ? 0.f : exp2_approx(sM[w][c] - M);
      L += f * sL[w][c];
      f *= sV(w)[c] * down;
      const float4 o = *reinterpret_cast<const float4*>(&sO(w)[c][d4]);
      acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w;
    }
    if (whole) {
      const float inv = 1.f / L;  // no visible key: 0 / 0, as the softmax over nothing
      const int cg = c0 + c, s = cg / a.G, g = cg - s * a.G;
      *reinterpret_cast<uint2*>(a.out + b * a.os_b + h * a.os_h + g * a.os_g + s * a.os_s + d4 * 2) =
          make_uint2(pack2<BF16>(acc.x * inv * up, acc.y * inv * up), pack2<BF16>(acc.z * inv * up, acc.w * inv * up));
    } else {
      *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * NC + c) * D + d4) = acc;
      if (d4 == 0) a.part_ml[(int64_t)slot * NC + c] = make_float4(M, L, up, 0.f);
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
    lo = seg_hi;  // hi or u1: past lo either way
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
  if (threadIdx.x == 0) {
    a.desc[2 * blockIdx.x] = cont;
    a.desc[2 * blockIdx.x + 1] = start;
  }
}

constexpr int kMqCtas = 3;  // CTAs an SM: their rings fill its shared memory
template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(kMqThreads, kMqCtas) paged_attn_fp8_rows_kernel(const Fp8Args a) {
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
  int* P = reinterpret_cast<int*>(dsm + kMqWarps * (MqRing<D>::WARP + NC * 8));
  __shared__ int wsum[kMqWarps];
  cost_prefix<kMqThreads>(a, kMqTile, kMqTile, kSegCost, keys, wsum, P);  // counted in keys
  const int64_t total = (int64_t)P[a.items] * a.Hkv;
  int64_t W = (total + gridDim.x - 1) / gridDim.x;
  W = (W + kMqTile - 1) / kMqTile * kMqTile;
  if (W < kMinW) W = kMinW;
  const int64_t lo = min(W * blockIdx.x, total);
  walk_share(a, P, lo, min(lo + W, total), keys, seg);
}

// ---------------------------------------------------------------------------
// Many rows: bound by the tensor cores, or by HBM behind a long context.
// One persistent CTA an SM on tcgen05; a unit is one KV head's G query heads x
// NX row tiles of 128 rows (rows = G heads x QT = 128 / G tokens), key tiles
// are 128 keys. Roles:
//   softmax     NX warpgroups, thread = row: scores from TMEM, times the
//               block's K scale, online softmax, probabilities times the
//               block's relative V scale, as f16 over the scores in TMEM;
//   producer    one warp: the codes' tiles by TMA through the block table into
//               a ring of raw tiles (16 KB at D = 128), and Q;
//   scales      one warp: each tile's 16 K and V scales (one for 8 keys, the
//               smallest block) and 128 keep bits, into a ring of four;
//   convert     four warps: codes to f16 in the 128-byte-swizzled operand
//               layout, V rows that no query may see as zeros;
//   MMA         one thread: S = Q K^T, O += P V, accumulators in TMEM.
// Both 16-bit types take every code exactly, so no scale enters the operands;
// V and the keys of f16 queries are f16 (one instruction for two codes), the
// keys of bf16 queries bf16. Reading codes instead of 16-bit rows halves HBM
// and L2 traffic. Shared memory (D = 128, NX = 2): Q 64 KB, K and V 2 x 32 KB
// each, raw 2 x 16 KB. Loops are rolled: unrolled, with the roles' code in one
// instruction cache, the chunk below took 633 us. It measures 387 us, 754
// TFLOP/s, for 8 sequences of 512 queries behind 512 to 7680 keys. The chain
// from a row tile's scores through its softmax to its product bounds it: the
// tensor pipe is busy 40 % of the time, the exponentials' 40 %, issue slots 51
// %; of the 7.8 cycles from one instruction of a warp to its next 2.2 are for
// long loads, 1.8 for the one before, 0.5 for the next to be fetched.
//
// The key tiles of all units, head-major, are cut into equal shares, one a
// CTA, so that there is one wave without a tail however unequal the
// sequences; the units that shares cut are joined by the merge kernel.
// NX = 2: one score buffer a row tile, PV(j - 1) before QK(j), so that one
// tile's softmax runs under the other's products. NX = 1: two score buffers,
// QK(j) before PV(j - 1), so that they run under the only softmax.
// Every wait is bounded; on expiry the CTA raises RBLN_DEVERR_TIMEOUT, lets
// its copies and products finish, frees TMEM and returns.
// ---------------------------------------------------------------------------
using namespace sm100;

// sm100's bounded wait with a time for the hardware to suspend the warp in:
// two dozen warps that poll take issue slots from those at work.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort) {
  const long long t0 = clock64();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(100000u)  // nanoseconds
        : "memory");
    if (ok) return true;
    if (*abort) return false;
    if (clock64() - t0 > kWaitLimitCycles) {
      *abort = 1;
      return false;
    }
  }
}

constexpr int kPanel = 128 * 128;  // 128 rows of 64 f16
constexpr int kTcSegCost = 2;      // key tiles charged to a unit's start (1, 2, 3: 395, 390, 391 us for that chunk)
constexpr int kMetaRing = 4;

struct TileMeta {
  float ks[16], vs[16];  // of keys [8 g, 8 g + 8): key_factor, V scale
  uint32_t keep[4];
  float vmax;
  float pad[3];
};

template <int D, int NX>
struct TcSmem {
  static constexpr int NP = D / 64;
  static constexpr int TILE = NP * kPanel;  // 128 rows x D of f16
  static constexpr int RAW = 128 * D;       // 128 rows x D codes
  static constexpr int NRAW = (D == 128 && NX == 2) ? 2 : 4;
  static constexpr int Q = 0;
  static constexpr int K0 = Q + NX * TILE;
  static constexpr int V0 = K0 + 2 * TILE;
  static constexpr int R0 = V0 + 2 * TILE;
  static constexpr int META = R0 + NRAW * RAW;
  static constexpr int BAR = META + kMetaRing * (int)sizeof(TileMeta);
  static constexpr int MISC = BAR + 40 * 8;  // TMEM slot, abort, share start (5 ints), prefix sums (16 ints)
  static constexpr int TOTAL = MISC + 32 * 4;
  static constexpr int ALLOC = TOTAL + 1024;
  static_assert(ALLOC <= 232448, "shared memory");
};

template <int NX>
struct TcCfg {
  static constexpr int THREADS = 128 * NX + 256;
  // registers a thread after the split: softmax, control, convert. The
  // launch has 128 (512 threads) or 168 (384 threads) each.
  static constexpr uint32_t RS = NX == 2 ? 152 : 216, RC = NX == 2 ? 96 : 64, RV = NX == 2 ? 112 : 104;
  static constexpr uint32_t LAUNCH = NX == 2 ? 128 : 168;
  static_assert(128 * (NX * RS + RC + RV) <= THREADS * LAUNCH, "register split exceeds the launch");
};

enum TcBar {
  T_RF = 0, T_RE = 4,    // raw ring
  T_KF = 8, T_KE = 10,   // f16 K stages
  T_VF = 12, T_VE = 14,  // f16 V stages
  T_MF = 16, T_ME = 20,  // scales and keep bits
  T_QF = 24, T_QE = 25,
  T_SF = 26,   // scores (NX = 2: of row tile x; NX = 1: of buffer T & 1)
  T_PF = 28,   // probabilities written (NX = 2: of row tile x; NX = 1: one)
  T_PV = 30,   // NX = 1: a PV complete
  T_O = 31,    // last PV of a segment complete, row tile x
  T_OE = 33,   // O read
  T_DONE = 35, T_COUNT = 36
};

// Keys of bf16 queries are multiplied by 2^-17: then no sum of D <= 256
// products of a code (at most 448) and a finite bf16 reaches 2^128.
constexpr float kKeyUp = 131072.f;

// What raw scores are multiplied by besides their key's scale. The sign of a
// negative softmax scale is in the converted keys. NaN stays NaN.
template <bool BF16>
__device__ __forceinline__ float score_mult(const Fp8Args& a) {
  return fabsf(a.scale_dev ? *a.scale_dev : a.scale) * (BF16 ? kKeyUp * kLog2e : kLog2e);
}

// That times a key's scale, which is what the softmax warps get: above zero,
// whatever the two are, so that -inf stays -inf (the smallest float makes no
// finite score more than 5e-7 in size), and finite where both are.
__device__ __forceinline__ float key_factor(float ks, float mult) {
  constexpr float kMost = 3.4028235e38f;
  const float f = ks * mult;
  const float g = f > kMost && fmaxf(ks, mult) <= kMost ? kMost : f;
  return g < 1.4e-45f ? 1.4e-45f : g;
}

// Eight f16 that stand for codes as bf16 times 2^-17, exact: a code has four
// bits. One packed product: f32 products before the rounding take the same
// time (389 us against 387 for 8 sequences of 512 queries behind 512 to 7680
// keys, 32 heads of 128 over 8 KV heads).
__device__ __forceinline__ uint4 f16_to_bf16(uint4 w) {
  uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<false>(u[i]);
    u[i] = pack2<true>(f.x, f.y);
    asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(u[i]) : "r"(0x37003700u));
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// A CTA's share as every role walks it: `left` positions from position `off`
// of unit (h, i) on; each unit has kTcSegCost positions and then one a key tile.
struct Share {
  int h, i, off, left;
};
struct Segment {
  int h, i, b, tile, keys, j0, j1;
  bool head, whole;
};
template <int NX>
__device__ __forceinline__ int tc_keys(const Fp8Args& a, int qt, int i) {
  const int b = i / a.tiles, t = i - b * a.tiles;
  return item_keys(a, b, (int)min((int64_t)(t + 1) * NX * qt - 1, (int64_t)a.S));
}
template <int NX>
__device__ __forceinline__ bool next_segment(const Fp8Args& a, int qt, Share& sh, Segment& g) {
  while (sh.left > 0) {
    if (!a.balanced && sh.i >= a.items) return false;
    const int keys = tc_keys<NX>(a, qt, sh.i);
    const int nt = (keys + 127) / 128, cost = nt + kTcSegCost;
    g.h = sh.h;
    g.i = sh.i;
    const int from = sh.off, to = a.balanced ? min(from + sh.left, cost) : cost;
    if (a.balanced) {
      sh.left -= to - from;
      sh.off = to;
      if (to == cost) {
        sh.off = 0;
        if (++sh.i == a.items) {
          sh.i = 0;
          ++sh.h;
        }
      }
    } else {  // whole units, every gridDim.x-th of item-major order
      const int64_t u = (int64_t)sh.i * a.Hkv + sh.h + gridDim.x;
      sh.i = (int)(u / a.Hkv);
      sh.h = (int)(u - (int64_t)sh.i * a.Hkv);
    }
    g.b = g.i / a.tiles;
    g.tile = g.i - g.b * a.tiles;
    g.keys = keys;
    g.j0 = max(from - kTcSegCost, 0);
    g.j1 = max(to - kTcSegCost, 0);
    g.head = g.j0 == 0;
    g.whole = g.head && g.j1 == nt;
    if (nt == 0 ? from == 0 : g.j1 > g.j0) return true;
  }
  return false;
}

// Block (-1: none) of the key that starts group `key` of sequence b.
__device__ __forceinline__ int block_of(const Fp8Args& a, int b, int key, int keys) {
  if (key >= keys) return -1;
  const int64_t v = load_index(a.bt, a.bt_dtype, b * a.bt_stride + key / a.bs);
  if (v >= 0 && v < a.num_blocks) return (int)v;
  if (a.err) atomicOr(a.err, RBLN_DEVERR_BLOCK_ID_RANGE);
  return -1;
}

template <int D, bool BF16, int NX>
__global__ void __launch_bounds__(TcCfg<NX>::THREADS, 1)
    paged_attn_fp8_tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                const __grid_constant__ CUtensorMap tm_v, const Fp8Args a, const int qt) {
  using L = TcSmem<D, NX>;
  using C = TcCfg<NX>;
  constexpr int NP = L::NP, NRAW = L::NRAW;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  int* misc = reinterpret_cast<int*>(sgen + L::MISC);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
  volatile int* abort = misc + 1;
  TileMeta* meta = reinterpret_cast<TileMeta*>(sgen + L::META);
  auto bar = [&](int i) { return sbase + L::BAR + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int W0 = 4 * NX;  // first control warp: producer, MMA, scales, -; then four converters

  if (threadIdx.x == 0) {
    *abort = 0;
    for (int i = 0; i < T_COUNT; ++i) {
      uint32_t n = 1;
      if (i >= T_RE && i < T_KF) n = 4;                                          // converters
      if ((i >= T_KF && i < T_KE) || (i >= T_VF && i < T_VE)) n = 4;             // converters
      if (i >= T_ME && i < T_QF) n = 4 + 4 * NX;                                 // converters and softmax warps
      if ((i >= T_PF && i < T_PV) || i == T_OE || i == T_OE + 1) n = 4;          // a row tile's softmax warps
      mbar_init(bar(i), n);
    }
    fence_mbar_init();
  }
  if (warp == W0 + 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  dependents_enter();
  // this CTA's share
  if (a.balanced) {
    int* P = reinterpret_cast<int*>(sgen + L::K0);  // before any copy or conversion uses it
    auto keys = [&](int i) { return tc_keys<NX>(a, qt, i); };
    cost_prefix<C::THREADS>(a, 128, 1, kTcSegCost, keys, misc + 8, P);
    if (threadIdx.x == 0) {
      const int64_t T = P[a.items], total = T * a.Hkv;
      // at least a tile a CTA; fewer CTAs work then
      const int64_t W = max((total + gridDim.x - 1) / gridDim.x, (int64_t)(1 + kTcSegCost));
      const int64_t lo = min(W * blockIdx.x, total), hi = min(lo + W, total);
      int i = 0;
      int64_t h = 0;
      if (lo < hi) {
        h = lo / T;
        const int x = (int)(lo - h * T);
        int j = a.items - 1;
        while (i < j) {
          const int mid = (i + j + 1) >> 1;
          if (P[mid] <= x) i = mid; else j = mid - 1;
        }
        misc[4] = x - P[i];
      }
      misc[2] = (int)h;
      misc[3] = i;
      misc[5] = (int)(hi - lo);
    }
    fence_proxy_async_smem();  // the prefix lay where the keys go, which the MMA reads
  } else if (threadIdx.x == 0) {
    misc[2] = (int)(blockIdx.x % a.Hkv);
    misc[3] = (int)(blockIdx.x / a.Hkv);
    misc[4] = 0;
    misc[5] = 1;
  }
  if (blockIdx.x == 0 && a.err)
    for (int b = threadIdx.x; b < a.B; b += C::THREADS)
      if (a.seq[b * a.seq_stride] < 0) atomicOr(a.err, RBLN_DEVERR_SEQ_RANGE);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Share sh{misc[2], misc[3], misc[4], misc[5]};
  Segment g;
  auto t_o = [&](int x) { return tmem + 256 + x * 128; };
  // score buffer of row tile x at running tile T
  auto t_s = [&](int x, int T) { return tmem + (NX == 2 ? x : (T & 1)) * 128; };
  // row tiles of a segment with tokens in the chunk
  auto active = [&](const Segment& s) { return NX == 1 || (s.tile * NX + 1) * qt >= a.S ? 1 : 2; };

  if (warp >= W0 + 4) {
    // ---------------------------------------------------------- convert
    setmaxnreg_dec<C::RV>();
    const int cw = warp - W0 - 4;
    constexpr int LPR = D / 16;          // lanes a row
    constexpr int RPI = 32 / LPR;        // rows a warp and step
    constexpr int STEPS = 128 / (4 * RPI);
    const int c16 = lane % LPR;
    const uint32_t dst_panel = (uint32_t)(c16 >> 2) * kPanel;
    const int row0 = cw * RPI + lane / LPR;  // first row; then every 4 RPI-th, of the same swizzle
    // The upper panel's lanes take their two chunks in the other order, so
    // that eight lanes of one row cover all banks.
    const int swap = (D == 128 && c16 >= 4) ? 8 : 0;
    const int chunk = 2 * (c16 & 3) + swap / 8;
    const int x0 = (chunk ^ (row0 & 7)) * 16, x1 = ((chunk ^ 1) ^ (row0 & 7)) * 16;
    // a negative softmax scale turns the order of the scores round: its sign goes into the keys
    const uint32_t flip = (a.scale_dev ? *a.scale_dev : a.scale) < 0.f ? 0x80808080u : 0u;
    int T = 0;
    bool ok = true;
    while (ok && next_segment<NX>(a, qt, sh, g)) {
      for (int j = g.j0; ok && j < g.j1; ++j, ++T) {
        const int ms = T % kMetaRing;
        uint32_t kw[4];
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
          const int n = 2 * T + part, rs = n % NRAW, st = T & 1;
          const int full = (part ? T_VF : T_KF) + st, empty = (part ? T_VE : T_KE) + st;
          ok = wait_for(bar(T_RF + rs), (n / NRAW) & 1, abort);
          if (ok && T >= 2) ok = wait_for(bar(empty), ((T >> 1) - 1) & 1, abort);
          bool all = true;
          if (part == 1 && ok) {
            ok = wait_for(bar(T_MF + ms), (T / kMetaRing) & 1, abort);
            const uint4 k = *reinterpret_cast<const uint4*>(meta[ms].keep);
            kw[0] = k.x; kw[1] = k.y; kw[2] = k.z; kw[3] = k.w;
            all = (k.x & k.y & k.z & k.w) == 0xffffffffu;
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t turn = part == 0 ? flip : 0u;
          const uint8_t* src = sgen + L::R0 + rs * L::RAW + row0 * D + c16 * 16;
          uint8_t* dst = sgen + (part ? L::V0 : L::K0) + st * L::TILE + row0 * 128 + dst_panel;
          // two steps a turn, for the instruction cache that the roles share (one, two, four steps:
          // 386, 387, 404 us for 8 sequences of 512 queries behind 512 to 7680 keys, 251, 250,
          // 257 for 4 of 48 queries behind some 18000 to 31000; eight: a third slower than two)
#pragma unroll 2
          for (int k = 0; k < STEPS; ++k) {
            uint2 w0 = *reinterpret_cast<const uint2*>(src + k * 4 * RPI * D + swap);
            uint2 w1 = *reinterpret_cast<const uint2*>(src + k * 4 * RPI * D + 8 - swap);
            if (turn) {
              w0.x ^= turn; w0.y ^= turn; w1.x ^= turn; w1.y ^= turn;
            }
            if (!all) {
              const int r = row0 + k * 4 * RPI;
              const uint32_t word = r < 64 ? (r < 32 ? kw[0] : kw[1]) : (r < 96 ? kw[2] : kw[3]);
              if (!((word >> (r & 31)) & 1u)) w0 = w1 = make_uint2(0, 0);
            }
            uint4 o0, o1;
            e4m3x4_to_f16x2x2(w0.x, o0.x, o0.y);
            e4m3x4_to_f16x2x2(w0.y, o0.z, o0.w);
            e4m3x4_to_f16x2x2(w1.x, o1.x, o1.y);
            e4m3x4_to_f16x2x2(w1.y, o1.z, o1.w);
            if (BF16 && part == 0) {
              o0 = f16_to_bf16(o0);
              o1 = f16_to_bf16(o1);
            }
            *reinterpret_cast<uint4*>(dst + k * 4 * RPI * 128 + x0) = o0;
            *reinterpret_cast<uint4*>(dst + k * 4 * RPI * 128 + x1) = o1;
          }
          fence_proxy_async_smem();  // read by the MMA; and the raw slot is rewritten by TMA
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bar(full));
            mbar_arrive(bar(T_RE + rs));
            if (part == 1) mbar_arrive(bar(T_ME + ms));
          }
        }
      }
    }
  } else if (warp >= W0) {
    setmaxnreg_dec<C::RC>();
    if (warp == W0) {
      // -------------------------------------------------------- producer
      if (lane == 0) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
      }
      const int rpb = min(a.bs, 128), nbox = 128 / rpb;  // nbox <= 16
      int T = 0, act = 0, issued = 0;
      bool ok = true;
      while (ok && next_segment<NX>(a, qt, sh, g)) {
        if (g.j1 == g.j0) continue;  // an empty unit
        const int nx = active(g);
        int blk = lane < nbox ? block_of(a, g.b, g.j0 * 128 + lane * rpb, g.keys) : -1;
        for (int j = g.j0; ok && j < g.j1; ++j, ++T) {
          const int row = (j * 128 + lane * rpb) % a.bs;
          const int now = blk < 0 ? a.num_blocks : blk;  // out of range: zeros
          if (j + 1 < g.j1 && lane < nbox) blk = block_of(a, g.b, (j + 1) * 128 + lane * rpb, g.keys);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const int n = 2 * T + part, rs = n % NRAW;
            if (n >= NRAW && !__all_sync(0xffffffffu, wait_for(bar(T_RE + rs), ((n / NRAW) - 1) & 1, abort))) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive_expect_tx(bar(T_RF + rs), L::RAW);
            __syncwarp();
            if (lane < nbox)
              tma_load_4d(sbase + L::R0 + rs * L::RAW + lane * rpb * D, part ? &tm_v : &tm_k, bar(T_RF + rs), 0, row,
                          g.h, now);
            issued = n + 1;
          }
          if (ok && j == g.j0) {
            // Q behind the first codes: the previous segment's QKs must be done
            if (act >= 1 && !__all_sync(0xffffffffu, wait_for(bar(T_QE), (act - 1) & 1, abort))) {
              ok = false;
              break;
            }
            if (lane == 0) {
              mbar_arrive_expect_tx(bar(T_QF), nx * NP * qt * a.G * 128);
              for (int x = 0; x < nx; ++x)
                for (int p = 0; p < NP; ++p)
                  tma_load_5d(sbase + L::Q + x * L::TILE + p * kPanel, &tm_q, bar(T_QF), p * 64,
                              (g.tile * NX + x) * qt, 0, g.h, g.b);
            }
            __syncwarp();
          }
        }
        ++act;
      }
      if (*abort) {  // let the copies in flight land before the CTA exits
        const long long t0 = clock64();
        for (int n = max(0, issued - NRAW); n < issued; ++n)
          while (!mbar_try_wait(bar(T_RF + n % NRAW), (n / NRAW) & 1) && clock64() - t0 < 4000000) {
          }
        if (act >= 0)
          while (!mbar_try_wait(bar(T_QF), (act > 0 ? act - 1 : 0) & 1) && clock64() - t0 < 8000000) {
          }
      }
    } else if (warp == W0 + 1) {
      // ------------------------------------------------------------- MMA
      if (lane == 0) {
        const uint32_t id_qk = idesc_f16(BF16, 128, 128, false);
        const uint32_t id_pv = idesc_f16(false, 128, D, true);
        int T = 0, act = 0, actx[2] = {0, 0}, segx[2] = {0, 0};  // tiles, segments; of each row tile
        bool ok = true;
        // A descriptor's address field counts 16-byte units and no operand
        // passes its 14 bits, so an offset within shared memory is one add.
        const uint32_t hi = (uint32_t)(sw128_desc(0, 16, 1024) >> 32);
        const uint32_t lo_k = (uint32_t)sw128_desc(sbase, 16, 1024), lo_v = (uint32_t)sw128_desc(sbase, kPanel, 1024);
        auto desc = [&](uint32_t lo) { return ((uint64_t)hi << 32) | lo; };
        auto qk = [&](int x, int Tj) {
          const uint32_t qb = lo_k + (L::Q + x * L::TILE) / 16, kb = lo_k + (L::K0 + (Tj & 1) * L::TILE) / 16;
          const uint32_t to = t_s(x, Tj);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kPanel + (kk & 3) * 32) / 16;
            umma_f16_ss(to, desc(qb + off), desc(kb + off), id_qk, kk > 0 ? 1u : 0u);
          }
          umma_commit(bar(T_SF + (NX == 2 ? x : (Tj & 1))));
        };
        auto pv = [&](int x, int Tj, bool first) {
          const uint32_t vb = lo_v + (L::V0 + (Tj & 1) * L::TILE) / 16;
          const uint32_t to = t_o(x), from = t_s(x, Tj);
          umma_f16_ts(to, from, desc(vb), id_pv, first ? 0u : 1u);
#pragma unroll
          for (int kk = 1; kk < 8; ++kk) umma_f16_ts(to, from + kk * 8, desc(vb + kk * 16 * 128 / 16), id_pv, 1u);
        };
        while (ok && next_segment<NX>(a, qt, sh, g)) {
          const int nt = g.j1 - g.j0;
          if (nt == 0) continue;
          const int nx = active(g);
          ok = wait_for(bar(T_QF), act & 1, abort);
          for (int j = 0; ok && j <= nt; ++j) {
            const int Tj = T + j;
            if (j < nt && !wait_for(bar(T_KF + (Tj & 1)), (Tj >> 1) & 1, abort)) {
              ok = false;
              break;
            }
            if constexpr (NX == 1) {
              if (j < nt) {
                tc_fence_after();
                qk(0, Tj);
                umma_commit(bar(T_KE + (Tj & 1)));
                if (j == nt - 1) umma_commit(bar(T_QE));
              }
            }
            if (j >= 1 && !wait_for(bar(T_VF + ((Tj - 1) & 1)), ((Tj - 1) >> 1) & 1, abort)) {
              ok = false;
              break;
            }
            for (int x = 0; x < nx; ++x) {
              if (j >= 1) {
                // the row tile's P; its first PV overwrites O once the last segment's is read
                const int ph = NX == 2 ? actx[x] + j - 1 : Tj - 1;
                if (!wait_for(bar(T_PF + x), ph & 1, abort) ||
                    (j == 1 && segx[x] >= 1 && !wait_for(bar(T_OE + x), (segx[x] - 1) & 1, abort))) {
                  ok = false;
                  break;
                }
                tc_fence_after();
                pv(x, Tj - 1, j == 1);
                if (NX == 1) umma_commit(bar(T_PV));
                if (j == nt) umma_commit(bar(T_O + x));
              }
              if (NX == 2 && j < nt) {
                tc_fence_after();
                qk(x, Tj);
              }
            }
            if (!ok) break;
            if (NX == 2 && j < nt) {
              umma_commit(bar(T_KE + (Tj & 1)));
              if (j == nt - 1) umma_commit(bar(T_QE));
            }
            if (j >= 1) umma_commit(bar(T_VE + ((Tj - 1) & 1)));
          }
          T += nt;
          ++act;
          for (int x = 0; x < nx; ++x) {
            actx[x] += nt;
            ++segx[x];
          }
        }
        if (!ok) {
          umma_commit(bar(T_DONE));
          const long long t0 = clock64();
          while (!mbar_try_wait(bar(T_DONE), 0) && clock64() - t0 < 4000000) {
          }
        }
      }
    } else if (warp == W0 + 2) {
      // ---------------------------------------------------------- scales
      const float mult = score_mult<BF16>(a);
      int T = 0;
      bool ok = true;
      while (ok && next_segment<NX>(a, qt, sh, g)) {
        if (g.j1 == g.j0) continue;
        const int grp = lane & 15;
        int blk = block_of(a, g.b, g.j0 * 128 + grp * 8, g.keys);
        for (int j = g.j0; j < g.j1; ++j, ++T) {
          const int ms = T % kMetaRing, t0 = j * 128;
          const int now = blk;
          float ks = 1.f, vs = 0.f;
          if (now >= 0) {
            ks = a.k_scale[now * a.ss_block + g.h * a.ss_head];
            vs = a.v_scale[now * a.ss_block + g.h * a.ss_head];
          }
          if (j + 1 < g.j1) blk = block_of(a, g.b, t0 + 128 + grp * 8, g.keys);
          uint32_t kw[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int key = t0 + 32 * w + lane;
            bool keep = __shfl_sync(0xffffffffu, now, 4 * w + (lane >> 3)) >= 0 && key < g.keys;
            if (keep && a.mask)
              keep = key < a.mask_len && load_keep(a.mask, a.mask_dtype, g.b * a.mask_stride + key);
            kw[w] = __ballot_sync(0xffffffffu, keep);
          }
          // a group none of whose keys is kept: its scales may be anything
          const uint32_t word = grp < 8 ? (grp < 4 ? kw[0] : kw[1]) : (grp < 12 ? kw[2] : kw[3]);
          if (((word >> (8 * (grp & 3))) & 0xffu) == 0) {
            ks = 1.f;
            vs = 0.f;
          }
          ks = key_factor(ks, mult);
          const uint32_t vmax = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(vs, 0.f)));
          if (T >= kMetaRing &&
              !__all_sync(0xffffffffu, wait_for(bar(T_ME + ms), ((T / kMetaRing) - 1) & 1, abort))) {
            ok = false;
            break;
          }
          if (lane < 16) {
            meta[ms].ks[lane] = ks;
            meta[ms].vs[lane] = vs;
          }
          if (lane == 0) {
#pragma unroll
            for (int w = 0; w < 4; ++w) meta[ms].keep[w] = kw[w];
            meta[ms].vmax = __uint_as_float(vmax);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(T_MF + ms));
        }
      }
    }
  } else {
    setmaxnreg_inc<C::RS>();
    // ----------------------------------------------------------- softmax
    const int x = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const int gq = r / qt, i = r - gq * qt;
    int T = 0, act = 0, TX = 0;  // tiles of the CTA; segments and tiles of this row tile
    int cont = -1, start = -1;
    bool ok = true;
    while (ok && next_segment<NX>(a, qt, sh, g)) {
      const int unit = g.h * a.items + g.i;
      const int nt = g.j1 - g.j0;
      if (!g.whole) {
        if (g.head) start = unit; else cont = unit;
      }
      if (x >= active(g)) {  // no tokens in this row tile: only pass the ring on
        for (int j = 0; j < nt; ++j, ++T) {
          if (!__all_sync(0xffffffffu, wait_for(bar(T_MF + T % kMetaRing), (T / kMetaRing) & 1, abort))) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive(bar(T_ME + T % kMetaRing));
        }
        continue;
      }
      const int s = (g.tile * NX + x) * qt + i;
      const bool row_ok = gq < a.G && s < a.S;
      const int pos = a.seq[g.b * a.seq_stride];
      const int lim = a.causal ? (int)min((int64_t)pos + s + 1, (int64_t)g.keys) : g.keys;
      // of the tile's first token
      const int first_lim = a.causal ? (int)min((int64_t)pos + (g.tile * NX + x) * qt + 1, (int64_t)g.keys) : g.keys;
      float m_run = neg_inf(), l_run = 0.f, vref = 0.f;
      for (int j = 0; j < nt; ++j, ++T, ++TX) {
        const int ms = T % kMetaRing, t0 = (g.j0 + j) * 128;
        const int sfb = NX == 2 ? x : (T & 1), sfp = NX == 2 ? TX & 1 : (T >> 1) & 1;
        ok = wait_for(bar(T_MF + ms), (T / kMetaRing) & 1, abort) && wait_for(bar(T_SF + sfb), sfp, abort);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        __syncwarp();
        // Two passes over the row's 128 scores, 32 at a time in rolled loops:
        // the roles share one instruction cache, and the code of a whole row
        // unrolled, masks in it, took three times as long, waiting for
        // instructions.
        const uint32_t ts = t_s(x, T) + lane_off;
        uint32_t v[32];
        float* const p = reinterpret_cast<float*>(v);
        const uint4 kwv = *reinterpret_cast<const uint4*>(meta[ms].keep);
        float vm = meta[ms].vmax;
        if ((kwv.x & kwv.y & kwv.z & kwv.w) != 0xffffffffu || t0 + 128 > first_lim) {
          // some key is not for some row: -inf over those scores first, and
          // the largest V scale of the groups of which the row sees a key
          vm *= kFarBelow;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const int n = lim - (t0 + 32 * c);  // keys of the chunk before the row's limit
            const uint32_t kw = meta[ms].keep[c] & (n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u);
            tmem_ld32(ts + c * 32, v);
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if ((kw >> (8 * u)) & 0xffu) vm = fmaxf(vm, meta[ms].vs[4 * c + u]);
            tmem_wait_ld32(v);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((kw >> e) & 1u)) v[e] = 0xff800000u;
            tmem_st32(ts + c * 32, v);
          }
          tmem_wait_st();
        }
        // maximum of the scaled scores: each group's raw maximum times its scale
        float mt = neg_inf();
        uint32_t v2[32];
        auto max_of = [&](int c, const uint32_t (&r)[32]) {
          const float* q = reinterpret_cast<const float*>(r);
          const float4 ks = *reinterpret_cast<const float4*>(meta[ms].ks + 4 * c);
          const float k4[4] = {ks.x, ks.y, ks.z, ks.w};
          float mg[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float* w = q + u * 8;
            mg[u] = fmaxf(max3(max3(w[0], w[1], w[2]), w[3], w[4]), max3(w[5], w[6], w[7])) * k4[u];
          }
          mt = fmaxf(mt, max3(mg[0], mg[1], fmaxf(mg[2], mg[3])));
        };
        tmem_ld32(ts, v);
#pragma unroll 1
        for (int c = 0; c < 4; c += 2) {
          tmem_wait_ld32(v);
          tmem_ld32(ts + c * 32 + 32, v2);
          max_of(c, v);
          tmem_wait_ld32(v2);
          if (c == 0) tmem_ld32(ts + 64, v);
          max_of(c + 1, v2);
        }
        const float m_new = fmaxf(m_run, mt);
        const bool grow = m_new > m_run + 8.f;
        float factor = 1.f;
        if (grow) {
          factor = exp2_approx(m_run - m_new);
          l_run *= factor;
          m_run = m_new;
        }
        if (vm > vref) {
          const float now = pow2_above(vm);
          factor *= vref * pow2_inverse(now);
          vref = now;
        }
        if (j >= 1 && __any_sync(0xffffffffu, factor != 1.f)) {
          // NX = 2: the scores come after PV(j - 1) in issue order; NX = 1: wait for it
          if (NX == 1 && !__all_sync(0xffffffffu, wait_for(bar(T_PV), (T - 1) & 1, abort))) {
            ok = false;
            break;
          }
          tc_fence_after();
          __syncwarp();
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o(x) + lane_off + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st32(t_o(x) + lane_off + c * 32, o);
          }
          tmem_wait_st();
        }
        const float nmu = (m_run == neg_inf()) ? 0.f : -m_run, inv_vref = pow2_inverse(vref);
        float sa0 = 0.f, sa1 = 0.f, sb0 = 0.f, sb1 = 0.f;
        // P of a chunk is 16 columns of f16 pairs over scores that are done with
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          tmem_ld32(ts + c * 32, v);
          const float4 ks = *reinterpret_cast<const float4*>(meta[ms].ks + 4 * c);
          const float4 vs = *reinterpret_cast<const float4*>(meta[ms].vs + 4 * c);
          const float k4[4] = {ks.x, ks.y, ks.z, ks.w}, v4[4] = {vs.x, vs.y, vs.z, vs.w};
          uint32_t pk[16];
          tmem_wait_ld32(v);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float km = k4[u], vr = v4[u] * inv_vref;
#pragma unroll
            for (int e = 8 * u; e < 8 * u + 8; e += 2) {
              fma2(p[e], p[e + 1], km, km, nmu, nmu);
              p[e] = exp2_approx(p[e]);
              p[e + 1] = exp2_approx(p[e + 1]);
            }
            add2(sa0, sa1, p[8 * u], p[8 * u + 1]);
            add2(sb0, sb1, p[8 * u + 2], p[8 * u + 3]);
            add2(sa0, sa1, p[8 * u + 4], p[8 * u + 5]);
            add2(sb0, sb1, p[8 * u + 6], p[8 * u + 7]);
#pragma unroll
            for (int e = 8 * u; e < 8 * u + 8; e += 2) {
              mul2(p[e], p[e + 1], vr, vr);
              pk[e / 2] = pack2<false>(p[e], p[e + 1]);
            }
          }
          tmem_st16(ts + c * 16, pk);
        }
        l_run += (sa0 + sa1) + (sb0 + sb1);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(T_PF + x));
          mbar_arrive(bar(T_ME + ms));
        }
      }
      if (!ok) break;
      if (nt > 0 && !__all_sync(0xffffffffu, wait_for(bar(T_O + x), act & 1, abort))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const float inv_l = 1.f / l_run;  // a row that sees no key: 0 times infinity
      const int64_t slot = ((int64_t)(2 * blockIdx.x + (g.head ? 1 : 0)) * NX + x) * 128 + r;
      char* orow = a.out + g.b * a.os_b + g.h * a.os_h + gq * a.os_g + (int64_t)s * a.os_s;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (nt > 0) {
          __syncwarp();
          tmem_ld32(t_o(x) + lane_off + c * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (!row_ok) continue;
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(o[e]);
        if (g.whole) {
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = f[e] * inv_l * vref;
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<uint4*>(orow + (c * 32 + q4 * 8) * 2) =
                make_uint4(pack2<BF16>(f[q4 * 8], f[q4 * 8 + 1]), pack2<BF16>(f[q4 * 8 + 2], f[q4 * 8 + 3]),
                           pack2<BF16>(f[q4 * 8 + 4], f[q4 * 8 + 5]), pack2<BF16>(f[q4 * 8 + 6], f[q4 * 8 + 7]));
        } else {
#pragma unroll
          for (int q4 = 0; q4 < 8; ++q4)
            *reinterpret_cast<float4*>(a.part_o + slot * D + c * 32 + q4 * 4) =
                make_float4(f[q4 * 4], f[q4 * 4 + 1], f[q4 * 4 + 2], f[q4 * 4 + 3]);
        }
      }
      if (!g.whole && row_ok) a.part_ml[slot] = make_float4(m_run, l_run, vref, 0.f);
      if (nt > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(T_OE + x));
        ++act;
      }
    }
    if (a.balanced && threadIdx.x == 0) {
      a.desc[2 * blockIdx.x] = cont;
      a.desc[2 * blockIdx.x + 1] = start;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort && threadIdx.x == 0 && a.err) atomicOr(a.err, RBLN_DEVERR_TIMEOUT);
  if (warp == W0 + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Takes a part (maximum, sum, vref) of a row into the row's so far; w0 and w1
// are what their accumulators count with. False: the part saw no key. Scores
// that are all NaN leave a maximum of -inf too (it passes over NaN), but a sum
// of NaN, which is taken on.
__device__ __forceinline__ bool join(float4& row, const float4& part, float& w0, float& w1) {
  if (part.x == neg_inf() && part.y == 0.f) return false;
  const float m = fmaxf(row.x, part.x), v = fmaxf(row.z, part.z), down = pow2_inverse(v);
  w0 = exp2_approx(row.x - m);
  w1 = exp2_approx(part.x - m);
  row.y = row.y * w0 + part.y * w1;
  w0 *= row.z * down;
  w1 *= part.z * down;
  row.x = m;
  row.z = v;
  return true;
}

// Joins the partial results of the units that several CTAs share. CTA (c, y):
// the chain that CTA c of the attention kernel starts, in parts c, c + 1, ...
// while those continue the same unit. 8 warps = RPC rows x KS slices of the
// chain, PASSES times over, a lane holding 4 (D = 128) or 2 dimensions of its
// row; the next four parts' loads (of each slice two; four: 109 us for 64
// sequences of 4 tokens, against 106) are issued before any is used. Bound by
// the parts' bytes in L2, and by its launch where there are few.
template <int D, bool BF16, int ROWS, int RPC, int PASSES>
__global__ void __launch_bounds__(256) paged_attn_fp8_merge_kernel(const Fp8Args a, int n_cta, int qt) {
  constexpr int KS = 8 / RPC, E = D / 32, U = KS == 1 ? 4 : 2;
  static_assert(KS == 1 || PASSES == 1, "slices meet once");
  __shared__ float so[8][D];
  __shared__ float4 sml[8];
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slice = warp / RPC;
  const int h = unit / a.items, item = unit - h * a.items;
  const int b = item / a.tiles, tile = item - b * a.tiles;
#pragma unroll 1
  for (int pass = 0; pass < PASSES; ++pass) {
    const int row = (blockIdx.y * PASSES + pass) * RPC + warp % RPC;
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
    const bool live = g < a.G && s < a.S;
    float4 all = make_float4(neg_inf(), 0.f, 0.f, 0.f);
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int i0 = slice; live && i0 < parts; i0 += U * KS) {
      float4 ml[U];
      float o[U][E];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * KS;
        ml[u] = make_float4(neg_inf(), 0.f, 0.f, 0.f);
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
        float w0, w1;
        if (!join(all, ml[u], w0, w1)) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * w0 + o[u][e] * w1;
      }
    }
    if (KS > 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) so[warp][lane * E + e] = acc[e];
      if (lane == 0) sml[warp] = all;
      __syncthreads();
      for (int k = 1; slice == 0 && k < KS; ++k) {
        float w0, w1;
        if (!join(all, sml[warp + k * RPC], w0, w1)) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * w0 + so[warp + k * RPC][lane * E + e] * w1;
      }
    }
    if (!live || slice != 0) continue;
    const float inv = 1.f / all.y;  // a row that sees no key: 0 times infinity
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * inv * all.z;
    char* to = a.out + b * a.os_b + h * a.os_h + g * a.os_g + (int64_t)s * a.os_s + lane * E * 2;
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(to) = make_uint2(pack2<BF16>(acc[0], acc[1]), pack2<BF16>(acc[2], acc[3]));
    else
      *reinterpret_cast<uint32_t*>(to) = pack2<BF16>(acc[0], acc[1]);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct Fp8Plan {
  int nx;       // row tiles of 128 of the tile kernel; 0: the row kernel
  int nt;       // 8-column groups of the row kernel
  int qt;       // tokens of a 128-row tile
  int rows;     // rows of a unit
  int tiles, items;
  bool balanced;
  int ctas;
  size_t desc, ml, o, total;  // workspace regions
};

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// Dynamic shared memory of the row kernel: rings, maxima and sums, prefix.
size_t rows_smem(int D, int rows, int items) {
  const int ring = D == 128 ? MqRing<128>::WARP : MqRing<64>::WARP;
  return (size_t)kMqWarps * (ring + rows * 8) + (items + 1) * sizeof(int);
}

int plan_fp8(const rbln_paged_attn_params_t* p, Fp8Plan* pl) {
  const int64_t span = (int64_t)p->max_blocks * p->block_size;
  const int64_t rows = (int64_t)p->q_len * p->group;
  // Up to 16 rows of a KV head the row kernel reads the codes once; more rows
  // would read them again for each 16, so they go to 128-row tiles. 16
  // sequences behind 4096 keys, row kernel against tiles: 62 to 99 us at 8
  // rows, 74 to 99 at 16, 101 to 99 at 20, 134 to 101 at 48.
  // (Pools of over 64 GB take the tiles too: the row kernel's offsets are 32 bits of 16 bytes.)
  // Two row tiles share a key tile's conversion where there are over 128 rows:
  // one tile against two, same sequences: 105 to 111 us at 128 rows, 169 to
  // 124 at 160, 310 to 216 at 512.
  const int64_t last = (p->num_blocks - 1) * p->cache_stride[0] + (p->num_kv_heads - 1) * p->cache_stride[1] +
                       (p->block_size - 1) * p->cache_stride[2];  // where the pool's last row starts
  pl->nx = rows <= 16 && last >> 4 <= (int64_t)UINT32_MAX ? 0 : rows <= 128 ? 1 : 2;
  pl->nt = rows <= 8 ? 1 : 2;
  pl->qt = 128 / p->group;
  pl->rows = pl->nx ? 128 * pl->nx : 8 * pl->nt;
  const int64_t tiles = pl->nx ? (p->q_len + (int64_t)pl->nx * pl->qt - 1) / (pl->nx * pl->qt)
                               : (rows + pl->rows - 1) / pl->rows;
  if (tiles * p->batch * p->num_kv_heads > INT32_MAX) return RBLN_ERR_UNSUPPORTED;
  pl->tiles = (int)tiles;
  pl->items = (int)(tiles * p->batch);
  // CTAs that run at once: a long prefix leaves room for fewer
  const int64_t fit = 232448 / (int64_t)(rows_smem(p->head_dim, pl->rows, std::min(pl->items, kMaxItems)) + 1024);
  const int64_t slots = 148LL * (pl->nx ? 1 : std::min<int64_t>(kMqCtas, fit));
  // the prefix fits shared memory and counts in 32 bits; with more items than
  // that there are enough whole units for every CTA
  pl->balanced = pl->items <= kMaxItems && (int64_t)pl->items * (span + kMqTile + kSegCost) < INT32_MAX;
  const int64_t units = (int64_t)pl->items * p->num_kv_heads;
  pl->ctas = (int)(pl->balanced ? slots : std::min<int64_t>(units, pl->nx ? slots : slots * 8));
  size_t off = 0;
  if (pl->balanced) {
    pl->desc = off;
    off += round256((size_t)2 * pl->ctas * sizeof(int));
    pl->ml = off;
    off += round256((size_t)2 * pl->ctas * pl->rows * sizeof(float4));
    pl->o = off;
    off += round256((size_t)2 * pl->ctas * pl->rows * p->head_dim * sizeof(float));
  }
  pl->total = off ? off + 256 : 0;
  return RBLN_OK;
}

template <typename... A, typename... B>
int launch_after(void (*kernel)(A...), dim3 grid, int threads, size_t smem, cudaStream_t st, const B&... args) {
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
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<A>(args)...) == cudaSuccess ? RBLN_OK : RBLN_ERR_LAUNCH;
}

template <int D, bool BF16, int NT>
int launch_rows(const Fp8Args& a, const Fp8Plan& pl, cudaStream_t st) {
  const size_t smem = rows_smem(D, pl.rows, pl.balanced ? pl.items : -1);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(paged_attn_fp8_rows_kernel<D, BF16, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)smem) != cudaSuccess)
    return RBLN_ERR_LAUNCH;
  int rc = launch_after(paged_attn_fp8_rows_kernel<D, BF16, NT>, dim3(pl.ctas), kMqThreads, smem, st, a);
  if (rc != RBLN_OK || !pl.balanced) return rc;
  return launch_after(paged_attn_fp8_merge_kernel<D, BF16, 8 * NT, 4, 1>, dim3(pl.ctas, 2 * NT), 256, 0, st, a, pl.ctas, 0);
}

// cache [NB, Hkv, bs, D] of codes -> 4-D map of bytes, box {D, rpb, 1, 1}, not swizzled
bool map_codes(CUtensorMap* m, const rbln_paged_attn_params_t* p, const void* cache) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)p->head_dim, (cuuint64_t)p->block_size, (cuuint64_t)p->num_kv_heads,
                              (cuuint64_t)p->num_blocks};
  const cuuint64_t str[3] = {(cuuint64_t)p->cache_stride[2], (cuuint64_t)p->cache_stride[1],
                             (cuuint64_t)p->cache_stride[0]};
  const cuuint32_t box[4] = {(cuuint32_t)p->head_dim, (cuuint32_t)std::min(p->block_size, 128), 1, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(cache), dims, str, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16, int NX>
int launch_tiles(const rbln_paged_attn_params_t* p, const Fp8Args& a, const Fp8Plan& pl, cudaStream_t st) {
  using L = TcSmem<D, NX>;
  using C = TcCfg<NX>;
  auto kernel = paged_attn_fp8_tiles_kernel<D, BF16, NX>;
  // the register split assumes the launch's count; with fewer a warpgroup
  // that raises its own would never be served
  static const bool regs_ok = [kernel] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, kernel) == cudaSuccess &&
           128 * (NX * C::RS + C::RC + C::RV) <= (uint32_t)fa.numRegs * C::THREADS;
  }();
  if (!regs_ok) return RBLN_ERR_LAUNCH;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::ALLOC) != cudaSuccess)
    return RBLN_ERR_LAUNCH;
  CUtensorMap tq, tk, tv;
  if (!map_codes(&tk, p, p->kcache) || !map_codes(&tv, p, p->vcache)) return RBLN_ERR_LAUNCH;
  {  // [B, Hkv, G, S, D] -> 5-D map, box {64, QT, G, 1, 1}
    const uint64_t dims[5] = {(uint64_t)D, (uint64_t)a.S, (uint64_t)a.G, (uint64_t)a.Hkv, (uint64_t)a.B};
    const uint64_t str[4] = {(uint64_t)a.qs_s, (uint64_t)a.qs_g, (uint64_t)a.qs_h, (uint64_t)a.qs_b};
    const uint32_t box[5] = {64, (uint32_t)pl.qt, (uint32_t)a.G, 1, 1};
    if (!make_map(&tq, tmap_dtype(p->q_dtype), 5, const_cast<void*>(p->q), dims, str, box)) return RBLN_ERR_LAUNCH;
  }
  int rc = launch_after(kernel, dim3(pl.ctas), C::THREADS, L::ALLOC, st, tq, tk, tv, a, pl.qt);
  if (rc != RBLN_OK || !pl.balanced) return rc;
  return launch_after(paged_attn_fp8_merge_kernel<D, BF16, 128 * NX, 8, 4>, dim3(pl.ctas, 4 * NX), 256, 0, st, a, pl.ctas,
                      pl.qt);
}

template <int D, bool BF16>
int launch_fp8(const rbln_paged_attn_params_t* p, const Fp8Args& a, const Fp8Plan& pl, cudaStream_t st) {
  if (pl.nx == 2) return launch_tiles<D, BF16, 2>(p, a, pl, st);
  if (pl.nx == 1) return launch_tiles<D, BF16, 1>(p, a, pl, st);
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
    rc = kv_write(p, st, /*reciprocal=*/true);
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
  for (a.bs_shift = 0; (1u << a.bs_shift) < (uint32_t)a.bs; ++a.bs_shift) {
  }
  a.bs_mul = (uint32_t)(((uint64_t)((1u << a.bs_shift) - (uint32_t)a.bs) << 32) / (uint32_t)a.bs + 1);
  a.causal = p->causal;
  a.tiles = pl.tiles; a.items = pl.items;
  a.balanced = pl.balanced;
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p->workspace) + 255) & ~uintptr_t(255));
  if (pl.balanced) {
    a.desc = reinterpret_cast<int*>(base + pl.desc);
    a.part_ml = reinterpret_cast<float4*>(base + pl.ml);
    a.part_o = reinterpret_cast<float*>(base + pl.o);
  }
  a.err = p->error_flags;
  if (p->prof_events[0]) cudaEventRecord(static_cast<cudaEvent_t>(p->prof_events[0]), st);
  const bool bf = p->q_dtype == RBLN_DT_BF16;
  if (p->head_dim == 128)
    rc = bf ? launch_fp8<128, true>(p, a, pl, st) : launch_fp8<128, false>(p, a, pl, st);
  else
    rc = bf ? launch_fp8<64, true>(p, a, pl, st) : launch_fp8<64, false>(p, a, pl, st);
  if (p->prof_events[1]) cudaEventRecord(static_cast<cudaEvent_t>(p->prof_events[1]), st);
  return rc;
}

}  // namespace rbln

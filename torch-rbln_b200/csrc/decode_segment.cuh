// What the paged decode kernels share: their arguments, and the attention of
// the query heads of one (sequence, KV head) over a range of its context,
// with the new token's append. paged_decode.cu says how it is built.
#pragma once

#include <atomic>

#include "common.cuh"
#include "ranges.cuh"

namespace rbln {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxDevices = 64;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16;

enum KvKind { KV_BF16 = 0, KV_F16 = 1, KV_FP8 = 2 };

struct DecodeArgs {
  const char* q;
  int64_t qs_b, qs_h, qs_g;  // bytes
  char* out;
  int64_t os_b, os_h, os_g;  // bytes
  const char* k_new;
  const char* v_new;
  int64_t kn_b, kn_h, vn_b, vn_h;  // bytes
  char* kcache;
  char* vcache;
  int64_t cs_block, cs_head, cs_tok;  // elements
  const float* k_scale;
  const float* v_scale;
  int64_t ss_block, ss_head;
  const int32_t* seq;
  int64_t seq_stride;
  const void* bt;
  int bt_dtype;
  int64_t bt_stride;
  const void* mask;
  int mask_dtype;
  int mask_len;
  int64_t mask_stride;
  float scale;
  const float* scale_dev;
  int B, Hkv, G, num_blocks, bs, span;
  int chunk;
  int max_splits;
  int nchunk;       // balanced split: chunks per KV head (grid.x)
  int min_w;        // balanced split: smallest chunk, in tokens
  int seg_cost;     // balanced split: virtual tokens charged to each sequence's start (multiple of 16)
  int* prefix;      // balanced split: [B + 1] padded-length prefix, then W
  // per-sequence split: [B][Hkv][max_splits][G]; balanced: [Hkv][nchunk + B][G]
  float* part_o;    // (.., D) floats per slot
  float* part_lse;  // log2-sum-exp per slot
  uint32_t* err;
  // head-sharded multi-GPU decode: final outputs go to every rank's buffer
  char* const* out_peers;  // nullptr: write `out` only
  int n_peers;
  int head0;  // first head of this rank in the full output
  const float* sinks;  // optional [Hkv * G] sink logits (natural-log units), index h * G + g
  // epoch exchange in the last CTA of the balanced merge kernel (nullptr: none)
  uint32_t* const* peer_flags;
  int peer_rank;
  uint32_t epoch;
  uint64_t wait_ns;
  int* merge_ctr;  // balanced workspace: merge CTAs done (zeroed by the decode kernel)
};

// Sink logit of local query head (h, g) in the log2 domain of the scores,
// or -inf when there are no sinks.
__device__ __forceinline__ float sink_log2(const DecodeArgs& a, int h, int g) {
  return a.sinks ? a.sinks[h * a.G + g] * kLog2e : neg_inf();
}

__device__ __forceinline__ void flag_error(uint32_t* err, uint32_t bit) {
  if (err) atomicOr(err, bit);
}

// Every kernel of the decode chain is launched as a programmatic dependent
// of the previous launch on its stream. It first waits until that grid has
// completed and its writes are visible (a no-op when the previous launch
// was not made that way), then lets the next grid on the stream be
// scheduled onto the SMs as this grid's CTAs retire; that grid waits here in
// the same way, so nothing it reads or writes is touched early.
__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Stores 4 output elements (one 8-byte pair of pairs) of (b, local head h,
// query head g, column d4): to `out`, or to every rank's buffer when the
// heads are sharded over GPUs.
__device__ __forceinline__ void store_out(const DecodeArgs& a, int b, int h, int g, int d4, uint2 v) {
  const int64_t off = b * a.os_b + (int64_t)(a.head0 + h) * a.os_h + (int64_t)g * a.os_g + d4 * 2;
  if (a.out_peers == nullptr) {
    *reinterpret_cast<uint2*>(a.out + off) = v;
  } else {
    for (int r = 0; r < a.n_peers; ++r) *reinterpret_cast<uint2*>(a.out_peers[r] + off) = v;
  }
}

// Context length seen by sequence b, and the number of splits covering it.
__device__ __forceinline__ void decode_extent(const DecodeArgs& a, int b, int& pos, int& L,
                                              int& nsplit) {
  pos = a.seq[b * a.seq_stride];
  if (a.mask) {
    L = min(a.span, a.mask_len);
  } else {
    L = positions_seen(pos, a.span);
  }
  nsplit = max(1, (L + a.chunk - 1) / a.chunk);
}

template <int D, int KV>
struct Cfg {
  static constexpr int SZ = (KV == KV_FP8) ? 1 : 2;  // bytes per cache element
  static constexpr int ROW = D * SZ;                  // bytes per token row
  static constexpr int KCH = ROW / 64;                // 16-B K chunks per lane per row
  static constexpr int KR = D / 8;                    // u32 MMA registers per K row
  static constexpr int VSEG = (KV == KV_FP8) ? ((D == 128) ? 16 : 8) : 8;  // contiguous d per seg
  static constexpr int NVE = D / 8;                   // d values per lane per V row
  static constexpr int NSEG = NVE / VSEG;             // 2 for 16-bit D=128, else 1
  static constexpr int NVW = NVE * SZ / 4;            // raw u32 per lane per V row
  static constexpr int MT = D / 16;                   // PV m-tiles
  static constexpr bool MMA_BF16 = (KV == KV_BF16);
};

// d index of a lane's e-th V value (gid = lane/4).
template <int D, int KV>
__device__ __forceinline__ int v_dim(int gid, int e) {
  using C = Cfg<D, KV>;
  return gid * C::VSEG + (e / C::VSEG) * 64 + (e % C::VSEG);
}

// Writes the new token's k/v (bf16/f16 copy, or fp8 quantised with the
// block's scale) at position `pos` of sequence b, KV head h. Threads 0..63
// take K and 64..127 take V, 8 elements each. No barrier inside.
template <int D, int KV, bool Q_BF16>
__device__ __forceinline__ void append_token(const DecodeArgs& a, int b, int h, int pos) {
  using C = Cfg<D, KV>;
  const int tid = threadIdx.x;
  const int64_t blk = load_index(a.bt, a.bt_dtype, b * a.bt_stride + pos / a.bs);
  if (blk < 0 || blk >= a.num_blocks) {
    if (tid == 0) flag_error(a.err, RBLN_DEVERR_BLOCK_ID_RANGE);
  } else {
    const int64_t row = (blk * a.cs_block + h * a.cs_head + (pos % a.bs) * a.cs_tok) * C::SZ;
    const int part = tid >> 6;  // 0: K, 1: V
    const int j = tid & 63;     // 8 elements per thread
    if (j < D / 8) {
      const char* src = (part == 0 ? a.k_new + b * a.kn_b + h * a.kn_h
                                   : a.v_new + b * a.vn_b + h * a.vn_h) + j * 16;
      char* dst = (part == 0 ? a.kcache : a.vcache) + row;
      const uint4 x = *reinterpret_cast<const uint4*>(src);
      if constexpr (KV != KV_FP8) {
        *reinterpret_cast<uint4*>(dst + j * 16) = x;
      } else {
        const float sc = (part == 0 ? a.k_scale : a.v_scale)[blk * a.ss_block + h * a.ss_head];
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint32_t o[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float f[4];
          float2 lo = unpack2<Q_BF16>(w[2 * k]), hi = unpack2<Q_BF16>(w[2 * k + 1]);
          f[0] = lo.x / sc; f[1] = lo.y / sc; f[2] = hi.x / sc; f[3] = hi.y / sc;
          __nv_fp8x2_storage_t p01 = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
          __nv_fp8x2_storage_t p23 = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
          o[k] = uint32_t(p01) | (uint32_t(p23) << 16);
        }
        *reinterpret_cast<uint2*>(dst + j * 8) = make_uint2(o[0], o[1]);
      }
    }
  }
}

// Attention of the G query heads of KV head h of sequence b over the
// context tokens [t0, t1): the CTA's 4 warps take 16-token tiles round-robin;
// their (max, sum, O) are combined in shared memory and written as the final
// output (whole = the CTA saw every token of the sequence) or as the
// (O/l, log2-sum-exp) partial at part_o/part_lse index slot + g.
// Bytes of the CTA combine area: per-warp O [kWarps][8*NT][D] and max/sum.
template <int D, int NT>
__host__ __device__ constexpr int combine_bytes() {
  return (kWarps * 8 * NT * D + 2 * kWarps * 8 * NT) * 4;
}
// Dynamic shared memory of a split CTA (the balanced kernel adds B + 1 ints).
template <int D, int NT>
__host__ __device__ constexpr int segment_smem() {
  return combine_bytes<D, NT>();
}

// LA (block-table lookahead): false = look up each tile's block where it is
// fetched; true = load the next tile's entry into registers one tile early,
// so that the lookup is off the tile's critical path.
template <int D, int KV, bool Q_BF16, int NT, bool LA>
__device__ __forceinline__ void decode_segment(const DecodeArgs& a, unsigned char* dsm, int b, int h, int t0,
                                               int t1, bool append, bool whole, int64_t slot) {
  using C = Cfg<D, KV>;
  constexpr bool MB = C::MMA_BF16;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gid = lane >> 2, tig = lane & 3;

  // ---- append the new token (write-then-read, like the reference) --------
  if (append && a.k_new != nullptr) {
    append_token<D, KV, Q_BF16>(a, b, h, a.seq[b * a.seq_stride]);
    __syncthreads();
  }

  // Block id (-1 when outside [0, num_blocks)) and keep bit of token
  // ts + (lane & 15) (lanes 16..31 repeat it).
  struct TileEntry {
    int blk;
    bool keep;
  };
  auto bt_entry = [&](int ts, TileEntry& e) {
    const int tpos = ts + (lane & 15);
    const bool in = tpos < t1;
    e.keep = in && (a.mask == nullptr || load_keep(a.mask, a.mask_dtype, b * a.mask_stride + tpos));
    const int64_t blk = in ? load_index(a.bt, a.bt_dtype, b * a.bt_stride + tpos / a.bs) : -1;
    e.blk = (blk >= 0 && blk < a.num_blocks) ? (int)blk : -1;
  };
  TileEntry ent;
  if constexpr (LA) bt_entry(t0 + warp * kTile, ent);  // before the query loads: independent of them

  // ---- query fragments: B operand (k = head_dim, n = head) ---------------
  float scale = a.scale_dev ? *a.scale_dev : a.scale;
  uint32_t qf[NT][C::KR];
  float qmax = 0.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int g = gid + 8 * nt;
    const bool live = g < a.G;
    const char* qrow = a.q + b * a.qs_b + h * a.qs_h + (int64_t)g * a.qs_g;
#pragma unroll
    for (int i = 0; i < C::KCH; ++i) {
      if constexpr (KV != KV_FP8) {
        uint4 x = live ? *reinterpret_cast<const uint4*>(qrow + (4 * i + tig) * 16) : make_uint4(0, 0, 0, 0);
        qf[nt][4 * i + 0] = x.x; qf[nt][4 * i + 1] = x.y; qf[nt][4 * i + 2] = x.z; qf[nt][4 * i + 3] = x.w;
      } else {
        // 16 fp8 K elements <-> 16 q elements (32 bytes) at d = 16*(4i+tig)
        const char* src = qrow + (4 * i + tig) * 32;
        uint4 x0 = live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
        uint4 x1 = live ? *reinterpret_cast<const uint4*>(src + 16) : make_uint4(0, 0, 0, 0);
        const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          qf[nt][8 * i + k] = w[k];
          float2 f = unpack2<Q_BF16>(w[k]);
          qmax = fmaxf(qmax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
    }
  }
  float qk_mult = scale * kLog2e;
  if constexpr (KV == KV_FP8) {
    // q goes to f16 for the f16 MMA. A bf16 q is rescaled by a power of two
    // so its largest magnitude sits in [2^14, 2^15): exact, no overflow.
    float qs = 1.f;
    if constexpr (Q_BF16) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, o));
      if (qmax > 0.f) {
        int ex;
        frexpf(qmax, &ex);
        ex = min(max(15 - ex, -120), 120);
        qs = ldexpf(1.f, ex);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < C::KR; ++k) {
          float2 f = unpack2<true>(qf[nt][k]);
          qf[nt][k] = pack2<false>(f.x * qs, f.y * qs);
        }
    }
    qk_mult = qk_mult / qs;
  }

  // ---- main loop over this warp's tiles -----------------------------------
  float o_acc[NT][C::MT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) o_acc[nt][mt][k] = 0.f;
  float m_run[NT][2], l_run[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_run[nt][0] = m_run[nt][1] = neg_inf();
    l_run[nt][0] = l_run[nt][1] = 0.f;
  }

  const char* kc = a.kcache;
  const char* vc = a.vcache;
  const int tv[4] = {2 * tig, 2 * tig + 1, 2 * tig + 8, 2 * tig + 9};

  // One 16-token tile in flight: lane l (mod 16) resolves token ts + l
  // through the block table; the row offsets reach the lanes that load them
  // by shuffles; then the K rows gid / gid+8 and the V rows tv[] are loaded.
  struct Tile {
    uint4 kraw[2][C::KCH];
    uint32_t vraw[4][C::NVW];
    uint32_t vmask;
    float ksc, vsc;
  };
  // The tile's block-table entry and mask byte come from `ent`, loaded one
  // tile earlier (bt_entry) so that the table lookup is off the critical path.
  auto fetch = [&](int ts, Tile& T, const TileEntry& ent) {
    const int tpos = ts + (lane & 15);
    bool valid = ent.keep;
    uint32_t off16 = 0;  // row byte offset / 16
    T.ksc = 1.f;
    T.vsc = 1.f;
    if (valid) {
      const int64_t blk = ent.blk;
      if (blk < 0) {
        valid = false;
        flag_error(a.err, RBLN_DEVERR_BLOCK_ID_RANGE);
      } else {
        off16 = (uint32_t)(((blk * a.cs_block + h * a.cs_head + (tpos % a.bs) * a.cs_tok) * C::SZ) >> 4);
        if constexpr (KV == KV_FP8) {
          T.ksc = a.k_scale[blk * a.ss_block + h * a.ss_head];
          T.vsc = a.v_scale[blk * a.ss_block + h * a.ss_head];
        }
      }
    }
    T.vmask = __ballot_sync(0xffffffffu, valid) & 0xffffu;
    if (T.vmask == 0) return;
    const uint32_t ok0 = __shfl_sync(0xffffffffu, off16, gid);
    const uint32_t ok1 = __shfl_sync(0xffffffffu, off16, gid + 8);
    const bool vk0 = (T.vmask >> gid) & 1, vk1 = (T.vmask >> (gid + 8)) & 1;
#pragma unroll
    for (int i = 0; i < C::KCH; ++i) {
      T.kraw[0][i] = vk0 ? ld_stream_v4(kc + (size_t)ok0 * 16 + (4 * i + tig) * 16) : make_uint4(0, 0, 0, 0);
      T.kraw[1][i] = vk1 ? ld_stream_v4(kc + (size_t)ok1 * 16 + (4 * i + tig) * 16) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t ov = __shfl_sync(0xffffffffu, off16, tv[j]);
      const bool vv = (T.vmask >> tv[j]) & 1;
      const char* rowp = vc + (size_t)ov * 16;
      if constexpr (C::NVW >= 4) {
#pragma unroll
        for (int sg = 0; sg < C::NVW / 4; ++sg) {
          uint4 x = vv ? ld_stream_v4(rowp + (gid * C::VSEG + sg * 64) * C::SZ) : make_uint4(0, 0, 0, 0);
          T.vraw[j][4 * sg + 0] = x.x; T.vraw[j][4 * sg + 1] = x.y;
          T.vraw[j][4 * sg + 2] = x.z; T.vraw[j][4 * sg + 3] = x.w;
        }
      } else {
        uint2 x = vv ? ld_stream_v2(rowp + gid * C::VSEG * C::SZ) : make_uint2(0, 0);
        T.vraw[j][0] = x.x; T.vraw[j][1] = x.y;
      }
    }
  };

  auto consume = [&](const Tile& T) {
    if (T.vmask == 0) return;  // warp-uniform (ballot)
    const bool vk0 = (T.vmask >> gid) & 1, vk1 = (T.vmask >> (gid + 8)) & 1;
    // S^T = K . Q^T
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
    if constexpr (KV != KV_FP8) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int i = kk >> 1, sgl = (kk & 1) * 2;
        const uint32_t* r0 = reinterpret_cast<const uint32_t*>(&T.kraw[0][i]);
        const uint32_t* r1 = reinterpret_cast<const uint32_t*>(&T.kraw[1][i]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816<MB>(s[nt], r0[sgl], r1[sgl], r0[sgl + 1], r1[sgl + 1], qf[nt][2 * kk], qf[nt][2 * kk + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < C::KCH; ++i) {
        const uint32_t* r0 = reinterpret_cast<const uint32_t*>(&T.kraw[0][i]);
        const uint32_t* r1 = reinterpret_cast<const uint32_t*>(&T.kraw[1][i]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {  // kk = 4i + w uses chunk word w (4 fp8)
          uint32_t a0, a1, a2, a3;
          e4m3x4_to_f16x2x2(r0[w], a0, a2);
          e4m3x4_to_f16x2x2(r1[w], a1, a3);
          const int kk = 4 * i + w;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<false>(s[nt], a0, a1, a2, a3, qf[nt][2 * kk], qf[nt][2 * kk + 1]);
        }
      }
    }

    // online softmax (log2 domain); rows gid / gid+8 are tokens
    float k0m = qk_mult, k1m = qk_mult;
    float vs0 = 1.f, vs1 = 1.f;
    if constexpr (KV == KV_FP8) {
      k0m *= __shfl_sync(0xffffffffu, T.ksc, gid);
      k1m *= __shfl_sync(0xffffffffu, T.ksc, gid + 8);
      vs0 = __shfl_sync(0xffffffffu, T.vsc, gid);
      vs1 = __shfl_sync(0xffffffffu, T.vsc, gid + 8);
    }
    uint32_t pb0[NT], pb1[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float x0 = vk0 ? s[nt][0] * k0m : neg_inf();
      const float x1 = vk0 ? s[nt][1] * k0m : neg_inf();
      const float x2 = vk1 ? s[nt][2] * k1m : neg_inf();
      const float x3 = vk1 ? s[nt][3] * k1m : neg_inf();
      const float mx0 = warp_max_xor_rows(fmaxf(x0, x2));
      const float mx1 = warp_max_xor_rows(fmaxf(x1, x3));
      const float mn0 = fmaxf(m_run[nt][0], mx0), mn1 = fmaxf(m_run[nt][1], mx1);
      const float ms0 = (mn0 == neg_inf()) ? 0.f : mn0;
      const float ms1 = (mn1 == neg_inf()) ? 0.f : mn1;
      const float al0 = exp2_approx(m_run[nt][0] - ms0), al1 = exp2_approx(m_run[nt][1] - ms1);
      const float p0 = exp2_approx(x0 - ms0), p2 = exp2_approx(x2 - ms0);
      const float p1 = exp2_approx(x1 - ms1), p3 = exp2_approx(x3 - ms1);
      l_run[nt][0] = l_run[nt][0] * al0 + p0 + p2;
      l_run[nt][1] = l_run[nt][1] * al1 + p1 + p3;
      m_run[nt][0] = mn0;
      m_run[nt][1] = mn1;
      // once the running maxima settle the factors are exactly 1 (their
      // exponent is exactly 0): the fp8 variant, which spends more issue
      // slots per tile on conversions, skips the rescale for the warp then
      // (measured +0.4 %); for 16-bit caches the vote cost as much as it saved
      if (KV != KV_FP8 || __any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
          o_acc[nt][mt][0] *= al0; o_acc[nt][mt][2] *= al0;
          o_acc[nt][mt][1] *= al1; o_acc[nt][mt][3] *= al1;
        }
      }
      pb0[nt] = movmatrix_trans(pack2<MB>(p0 * vs0, p1 * vs0));
      pb1[nt] = movmatrix_trans(pack2<MB>(p2 * vs1, p3 * vs1));
    }

    // O^T += V^T . P^T
#pragma unroll
    for (int mt = 0; mt < C::MT; ++mt) {
      uint32_t a0, a1, a2, a3;
      if constexpr (KV != KV_FP8) {
        a0 = prmt(T.vraw[0][mt], T.vraw[1][mt], 0x5410);
        a1 = prmt(T.vraw[0][mt], T.vraw[1][mt], 0x7632);
        a2 = prmt(T.vraw[2][mt], T.vraw[3][mt], 0x5410);
        a3 = prmt(T.vraw[2][mt], T.vraw[3][mt], 0x7632);
      } else {
        const int w = mt >> 1;
        const uint32_t sel = (mt & 1) ? 0x7362u : 0x5140u;
        const uint32_t x = prmt(T.vraw[0][w], T.vraw[1][w], sel);
        const uint32_t y = prmt(T.vraw[2][w], T.vraw[3][w], sel);
        e4m3x4_to_f16x2x2(x, a0, a1);
        e4m3x4_to_f16x2x2(y, a2, a3);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma16816<MB>(o_acc[nt][mt], a0, a1, a2, a3, pb0[nt], pb1[nt]);
    }
  };

  for (int ts = t0 + warp * kTile; ts < t1; ts += kWarps * kTile) {
    Tile T;
    if constexpr (!LA) bt_entry(ts, ent);
    fetch(ts, T, ent);
    // next tile's lookup overlaps this tile's loads and math
    if constexpr (LA) bt_entry(ts + kWarps * kTile, ent);
    consume(T);
  }

  // ---- combine the 4 warps of this CTA ------------------------------------
  constexpr int GP = 8 * NT;
  auto sO = reinterpret_cast<float(*)[GP][D]>(dsm);
  auto sM = reinterpret_cast<float(*)[GP]>(dsm + kWarps * GP * D * 4);
  auto sL = reinterpret_cast<float(*)[GP]>(dsm + kWarps * GP * D * 4 + kWarps * GP * 4);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float l0 = warp_sum_xor_rows(l_run[nt][0]);
    const float l1 = warp_sum_xor_rows(l_run[nt][1]);
    const int h0 = 2 * tig + 8 * nt;
    if (gid == 0) {
      sM[warp][h0] = m_run[nt][0]; sM[warp][h0 + 1] = m_run[nt][1];
      sL[warp][h0] = l0; sL[warp][h0 + 1] = l1;
    }
#pragma unroll
    for (int mt = 0; mt < C::MT; ++mt) {
      const int d0 = v_dim<D, KV>(gid, 2 * mt), d1 = v_dim<D, KV>(gid, 2 * mt + 1);
      sO[warp][h0][d0] = o_acc[nt][mt][0];
      sO[warp][h0 + 1][d0] = o_acc[nt][mt][1];
      sO[warp][h0][d1] = o_acc[nt][mt][2];
      sO[warp][h0 + 1][d1] = o_acc[nt][mt][3];
    }
  }
  __syncthreads();

  const bool final_out = whole;
  for (int idx = tid; idx < a.G * (D / 4); idx += kThreads) {
    const int g = idx / (D / 4), d4 = (idx % (D / 4)) * 4;
    float M = neg_inf();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sM[w][g]);
    float Lsum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = (sM[w][g] == neg_inf()) ? 0.f : exp2_approx(sM[w][g] - M);
      Lsum += f * sL[w][g];
      const float4 o = *reinterpret_cast<const float4*>(&sO[w][g][d4]);
      acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w;
    }
    if (final_out) {
      // the sink adds e^{sink - M} to the denominator only; all positions
      // masked (M = -inf) then gives 0, and NaN without a sink
      const float inv = 1.f / (a.sinks ? Lsum + exp2f(sink_log2(a, h, g) - M) : Lsum);
      acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
      store_out(a, b, h, g, d4, make_uint2(pack2<Q_BF16>(acc.x, acc.y), pack2<Q_BF16>(acc.z, acc.w)));
    } else {
      const float inv = 1.f / Lsum;
      acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
      const int64_t ps = slot + g;
      *reinterpret_cast<float4*>(a.part_o + ps * D + d4) = acc;
      // -inf for a part that saw nothing; one whose scores are all NaN has no maximum either, and stays NaN
      if (d4 == 0) a.part_lse[ps] = Lsum == 0.f ? neg_inf() : M + __log2f(Lsum);
    }
  }
  if (a.out_peers && final_out) __threadfence_system();  // peer stores before the epoch exchange
  __syncthreads();  // the combine area is reused by the CTA's next segment
}

// Context length seen by sequence b (see decode_extent).
__device__ __forceinline__ int seq_len(const DecodeArgs& a, int b, int& pos) {
  pos = a.seq[b * a.seq_stride];
  return a.mask ? min(a.span, a.mask_len) : positions_seen(pos, a.span);
}

// host side
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int dtype_bytes(int dt) {
  switch (dt) {
    case RBLN_DT_F32: case RBLN_DT_I32: return 4;
    case RBLN_DT_F16: case RBLN_DT_BF16: case RBLN_DT_I16: return 2;
    case RBLN_DT_I64: return 8;
    default: return 1;
  }
}

// Largest dynamic shared-memory size one kernel has been opted into, per
// device (one instance per kernel instantiation).
struct SmemOptIn {
  std::atomic<int> bytes[kMaxDevices] = {};
};

// Opts `kernel` into `bytes` of dynamic shared memory when that is above
// 48 KB and above what it was opted into before on this device.
bool allow_smem(const void* kernel, int bytes, SmemOptIn& opt) {
  if (bytes <= 48 * 1024) return true;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
  if (opt.bytes[dev].load(std::memory_order_relaxed) >= bytes) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return false;
  int cur = opt.bytes[dev].load(std::memory_order_relaxed);
  while (cur < bytes && !opt.bytes[dev].compare_exchange_weak(cur, bytes)) {
  }
  return true;
}

// Slices of the query heads per merge CTA: (KV head, sequence) pairs are
// split over heads (halving while G allows) until the merge grid has about
// two CTAs per SM. At 32 sequences x 1 KV head (a long-context decode
// sharded over 8 GPUs) that is 8 CTAs per pair; at 64 x 8 pairs, none.
int merge_head_split(int Hkv, int B, int G) {
  int gz = 1;
  while (G % (2 * gz) == 0 && (int64_t)Hkv * B * gz < 2 * 148) gz *= 2;
  return gz;
}

}  // namespace
}  // namespace rbln

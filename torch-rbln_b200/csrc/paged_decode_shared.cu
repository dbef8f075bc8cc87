// Paged decode for a batch whose sequences share their first positions in
// groups (rbln_paged_causal_attn_decode_shared):
//   out[b] = softmax(scale q[b] K^T) V over positions [0, min(seq[b] + 1, span)),
// positions below the group's shared length read through the table of its
// first sequence, the others through the sequence's own.
//
// The softmax over a union of positions is joined from its parts: part i
// gives O_i = sum_t e^{s_t - m_i} v_t / l_i and lse_i = m_i + log l_i, and
// O = sum_i e^{lse_i} O_i / sum_i e^{lse_i}. Three launches, each a
// programmatic dependent of the one before:
//  * shared_prefix_kernel (tcgen05, one CTA an SM): first the plan, made by
//    every CTA for itself: the rows' groups, the units of work, where each CTA
//    starts in them, how many SMs this kernel takes. Then the query heads of a
//    KV head of up to 2 x 128 rows of a group against the shared keys, so that
//    the tensor cores work on rows that a batch without a shared prefix would
//    bring one by one, and a key is read once for them;
//  * shared_own_kernel, beside it on the other SMs: each sequence's own
//    positions with the decode kernels' segments (mma.sync, one sequence and
//    KV head at a time), and the append of the new token (of one below the
//    shared length after the first kernel has written it, see append_below);
//  * shared_merge_kernel: the parts of every row.
// GPU time, heads of 128, pages of 16, bf16: 4 sequences x 4 query heads x 8
// KV heads behind 500 positions 14 us; 64 behind 4096, with 264 of their own
// on average, 32; 256 x 8 query heads behind 32768, with 512 of their own,
// 365. paged_causal_attn_decode, which reads the prefix once for each sequence,
// is the faster op behind short prefixes: with 8 KV heads of 4 query heads and
// 64 own positions on average, 4 sequences behind 512 positions 13.8 us here
// and 13.0 there, behind 8192 21.8 and 24.9; 64 behind 128 18.8 and 17.6,
// behind 512 20.2 and 27.9, behind 8192 34.9 and 226; 256 behind 128 68 and 46,
// behind 512 55 and 86.

#include <algorithm>

#include "decode_segment.cuh"
#include "sm100.cuh"
#include "tma_map.cuh"

namespace rbln {
namespace {

using namespace sm100;

constexpr int kMaxBatch = 4096, kMaxGroups = 1024;  // what the plan's CTA takes
constexpr int kKeys = 128;            // keys a tile
constexpr int kRows = 128;            // query rows a tile
constexpr int kPanel = 128 * 128;     // bytes: 128 rows of 64 elements
constexpr int kPrefixThreads = 384;   // softmax warpgroups 0-3 and 4-7, producers 8 and 10, MMA 9
// Own positions are counted in sixteens: what the start of a sequence's own
// part is charged, and the smallest share of a CTA (16 of them: 16.3 us for
// four sequences behind 500 positions, now 14.4).
constexpr int kSegCost = 8, kMinOwn = kSegCost + 1;
constexpr int kSms = 148;
// What a key tile costs a CTA with two row tiles and with one (whose two
// warpgroups take the tiles in turn), and a unit's start.
constexpr int kWideCost = 4, kTurnCost = 3, kUnitCost = 2;
// Registers a thread after the split (launch: 168 each): a softmax thread
// holds its whole row of 128 scores.
constexpr uint32_t kRegsSoftmax = 216, kRegsOther = 64;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsOther <= kPrefixThreads * 168, "register split exceeds the launch");

// What the plan leaves for the other kernels.
struct Totals {
  int cost;       // of all units of a KV head
  int share;      // of a CTA of the prefix kernel
  int rows;       // rows that a KV head's units store for each CTA that works on them
  int own;        // sixteens of own positions of a KV head, with what the sequences' starts are charged
  int own_share;  // of a CTA
};

// A CTA's key tiles of a unit of the prefix kernel.
struct Unit {
  int h, b0, n;   // KV head, sequences [b0, b0 + n)
  int lead, len;  // row of the block table, shared positions
  int wide;       // two row tiles, each against all keys; else one, its key tiles in turn by two warpgroups
  int t0, t1;     // this CTA's key tiles
  int row0;       // first stored row
  int group, next;  // the group, and where on the line the CTA goes on
};

// A CTA's segment of a sequence's own positions.
struct OwnPart {
  int h, b;
  int t0, t1;      // positions
  int append;      // the new token's position is among them
  int whole;       // they are all that the sequence sees
  long long next;  // where on the line the CTA goes on
};

struct SharedArgs {
  int groups;
  const int32_t* starts;
  const int32_t* lens;
  int seqs;            // sequences a row tile holds: 128 / G
  int ctas;            // of the prefix kernel, one an SM
  int own_ctas;        // of the own kernel on an SM
  float tile_us;       // time of a key tile of cost 1, and of an own position, on an SM
  float own_us;
  float late_us;       // what the prefix kernel has to do besides its tiles
  Totals* totals;
  int* row_shared;     // [B] positions that are read through the group's table
  int4* row_parts;     // [B] the row's unit: its first key tile on KV head 0's line, the last one less that (-1: no
                       // shared part), its stored row, the stored rows of x = 0 where tiles are taken in turn
  int* own;            // [B + 1] prefix of the rows' own positions in sixteens, their starts' charge included
  float* part_o;       // parts of the shared positions, see unit_at
  float* part_lse;
};

__host__ __device__ __forceinline__ int tiles_of(int positions) { return (positions + kKeys - 1) / kKeys; }

// A group's units: `full` of 2 x seqs sequences and one of the rest, which
// takes its tiles in turn where those fit in one row tile.
struct GroupUnits {
  int full, rest, tiles, full_cost, rest_cost;
  __device__ __forceinline__ GroupUnits(int n, int len, int seqs) {
    full = n / (2 * seqs);
    rest = n - full * 2 * seqs;
    tiles = tiles_of(len);
    full_cost = kWideCost * tiles + kUnitCost;
    rest_cost = rest == 0 ? 0 : (rest > seqs ? kWideCost : kTurnCost) * tiles + kUnitCost;
  }
};

// The units of all KV heads, head by head, group by group, stand end to end
// on a line, each unit's start charged kUnitCost, each key tile its cost; CTA
// c takes [c share, (c + 1) share), a tile by where it starts. A unit's rows
// as CTA c sees them are stored from row 256 c + R on, with R the rows that
// the units before it store: no two of them overlap, since a unit stores 256
// rows at most, and neither does one unit's with another's in one CTA.
//
// The unit at `lo` of the line, in group g of head h, as a CTA sees it that
// ends at `hi`; gr: the group, before: its start on the head's line.
__device__ __forceinline__ Unit unit_at(int lo, int hi, int cta, int h, int g, int4 gr, int before, int head_cost,
                                        int head_rows, int seqs, int G) {
  const GroupUnits gu(gr.y, gr.z, seqs);
  const int y = lo - h * head_cost - before, k = min(y / gu.full_cost, gu.full);
  const bool whole = k < gu.full;
  const int base = lo - y + k * gu.full_cost, end = base + (whole ? gu.full_cost : gu.rest_cost);
  Unit u;
  u.wide = whole || gu.rest > seqs;
  const int w = u.wide ? kWideCost : kTurnCost;
  const int first = base + kUnitCost;
  u.next = min(hi, end);
  u.t0 = (max(lo, first) - first + w - 1) / w;
  u.t1 = (max(u.next, first) - first + w - 1) / w;
  u.h = h;
  u.b0 = gr.x + k * 2 * seqs;
  u.n = whole ? 2 * seqs : gu.rest;
  u.lead = gr.x;
  u.len = gr.z;
  u.row0 = cta * 2 * kRows + h * head_rows + gr.w + k * 2 * seqs * G;
  u.group = g;
  return u;
}

// The own positions of all KV heads and sequences, each sequence's rounded up
// to sixteens and its start charged kSegCost, stand on another line, cut
// likewise: the segment at `lo` of a CTA that ends at `hi`, in sequence b,
// whose range of a KV head's line is [from, to).
__device__ __forceinline__ OwnPart own_at(long long lo, long long hi, int h, int b, int all, int from, int to, int shared,
                                          int seq, int span) {
  const long long pb = (long long)h * all + from + kSegCost, pe = (long long)h * all + to;
  const long long seg_lo = max(lo, pb), seg_hi = min(hi, pe);
  OwnPart p;
  p.h = h;
  p.b = b;
  p.next = seg_hi;
  const int L = positions_seen(seq, span);
  p.t0 = shared + 16 * (int)(seg_lo - pb);
  p.t1 = seg_lo < seg_hi ? min(shared + 16 * (int)(seg_hi - pb), L) : p.t0;
  p.append = seq < span && seq >= p.t0 && seq < p.t1;
  p.whole = seg_lo == pb && seg_hi == pe && shared == 0;
  return p;
}

// ------------------------------------------------------------------- plan
// Exclusive scan over the CTA's threads of N values (sum or maximum) at once;
// all[i]: of all threads.
template <int THREADS, bool MAX, int N>
__device__ __forceinline__ void scan_before(int (&v)[N], int (&all)[N]) {
  constexpr int W = THREADS / 32;
  __shared__ int warps[N][32];
  auto join = [](int a, int b) { return MAX ? max(a, b) : a + b; };  // of values from 0 up
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = v[i];
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x[i], o);
      if (lane >= o) x[i] = join(x[i], y);
    }
    if (lane == 31) warps[i][warp] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int w = lane < W ? warps[i][lane] : 0;
    for (int o = 1; o < W; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w = join(w, y);
    }
    all[i] = __shfl_sync(0xffffffffu, w, W - 1);
    const int wb = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    const int up = __shfl_up_sync(0xffffffffu, x[i], 1);
    v[i] = join(warp > 0 ? wb : 0, lane > 0 ? up : 0);
  }
}

// The last i of [-1, n] (0 <= i where `at` starts at 0) with at[i] <= x.
__device__ __forceinline__ int last_at_most(const int* at, int lo, int hi, int x) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// What a CTA of the prefix kernel knows of the plan.
struct PlanSmem {
  int start[kMaxGroups + 1], before[kMaxGroups + 1];  // first sequence; cost of the groups before it, in one KV head
  int len[kMaxGroups], stored[kMaxGroups];            // shared positions; rows that the groups before it store
  Totals totals;
  int below;  // whether group[b] is kBelow for any row
  Unit first, at[kPrefixThreads / 32];  // of this CTA; where each warp is
  __device__ __forceinline__ int4 group(int g) const {
    return make_int4(start[g], len[g] > 0 ? start[g + 1] - start[g] : 0, len[g], stored[g]);
  }
};

constexpr short kBelow = -2;

// The plan, made by every CTA of the prefix kernel for itself: that takes less
// time than a launch of its own. What the other kernels read is stored by all
// of them, a row by one; it is not read in this grid, whose CTAs do not wait
// for one another. own, group: scratch for all rows; group[b] is kBelow for a
// row whose new position lies below its group's shared length.
__device__ __forceinline__ void make_plan(const DecodeArgs& a, const SharedArgs& s, PlanSmem& P, int* own, short* group) {
  constexpr int T = kPrefixThreads, PG = (kMaxGroups + T) / T;  // starts a thread
  const int tid = threadIdx.x, cta = blockIdx.x;
  // the groups' starts, none before the one before it
  int cut[PG], top[1] = {0}, most[1];
#pragma unroll
  for (int k = 0; k < PG; ++k) {
    const int g = PG * tid + k;
    // (without groups there need not be any starts: P.start[0] = 0 then)
    if (s.groups > 0 && g <= s.groups) top[0] = max(top[0], min(max(s.starts[g], 0), a.B));
    cut[k] = top[0];
    if (g < s.groups) {
      P.len[g] = min(max(s.lens[g], 0), a.span);
      P.stored[g] = 0;
    }
  }
  if (tid == 0) P.below = 0;
  scan_before<T, true>(top, most);
#pragma unroll
  for (int k = 0; k < PG; ++k)
    if (PG * tid + k <= s.groups) P.start[PG * tid + k] = max(cut[k], top[0]);
  __syncthreads();
  // rows: group, shared positions, own positions
  for (int b = tid; b < a.B; b += T) {
    const int seq = a.seq[b * a.seq_stride], g = last_at_most(P.start, -1, s.groups, b);
    const int len = g >= 0 && g < s.groups ? P.len[g] : 0, shared = seq >= len ? len : 0;
    const bool early = seq >= 0 && seq < len;
    if (early) P.below = 1;
    if (shared > 0) P.stored[g] = 1;  // some row of the group has a shared part
    const int L = positions_seen(seq, a.span);
    own[b] = (L - shared + 15) / 16 + kSegCost;
    group[b] = (short)(shared > 0 ? g : early ? kBelow : -1);
  }
  __syncthreads();
  // own positions before this thread's rows; cost and stored rows of the groups before this thread's
  const int per = (a.B + T - 1) / T, b0 = min(per * tid, a.B), b1 = min(b0 + per, a.B);
  int v[3] = {0, 0, 0}, all[3], cost[PG], rows[PG];
  for (int b = b0; b < b1; ++b) v[0] += own[b];
#pragma unroll
  for (int k = 0; k < PG; ++k) {
    const int g = PG * tid + k;
    cost[k] = rows[k] = 0;
    if (g < s.groups && P.stored[g]) {
      const GroupUnits u(P.start[g + 1] - P.start[g], P.len[g], s.seqs);
      cost[k] = u.full * u.full_cost + u.rest_cost;
      rows[k] = (2 * s.seqs * u.full + (u.rest > s.seqs ? u.rest : 2 * u.rest)) * a.G;
    }
    v[1] += cost[k];
    v[2] += rows[k];
  }
  scan_before<T, false>(v, all);
  for (int b = b0, run = v[0]; b < b1; ++b) {
    const int n = own[b];
    own[b] = run;
    run += n;
  }
#pragma unroll
  for (int k = 0; k < PG; ++k) {
    const int g = PG * tid + k;
    if (g >= s.groups) break;
    if (cost[k] == 0) P.len[g] = 0;
    P.before[g] = v[1];
    P.stored[g] = v[2];
    v[1] += cost[k];
    v[2] += rows[k];
  }
  // The SMs are divided so that both kernels end together: with m of N SMs,
  //   line / m + late = own / (N - m),
  // all in microseconds.
  const int total = all[1], line = total * a.Hkv;
  const float N = (float)s.ctas, late = s.late_us, p = line * s.tile_us, o = 16.f * (float)all[0] * a.Hkv * s.own_us;
  const float half = 0.5f * (late * N - p - o);
  const int sms = min(s.ctas - 2, max(1, (int)((half + sqrtf(half * half + late * p * N)) / late + 0.5f)));
  // The line is below 2^30 long. A share of a wide tile at least: so every
  // CTA between a unit's first and last has a tile of it.
  const int share = max(kWideCost, (line + sms - 1) / sms);
  const int own_ctas = (s.ctas - (line + share - 1) / share) * s.own_ctas;
  const long long own_line = (long long)all[0] * a.Hkv;
  const int W = max(kMinOwn, (int)((own_line + own_ctas - 1) / own_ctas));
  if (tid == 0) {
    P.before[s.groups] = total;
    P.totals = Totals{total, share, all[2], all[0], W};
    if (cta == 0) {
      *s.totals = P.totals;
      s.own[a.B] = all[0];
    }
  }
  __syncthreads();
  for (int b = cta + tid * s.ctas; b < a.B; b += T * s.ctas) {
    const int g = group[b];
    int4 parts = make_int4(0, -1, 0, 0);
    if (g >= 0) {
      const int i = b - P.start[g], unit = i / (2 * s.seqs);
      const GroupUnits u(P.start[g + 1] - P.start[g], P.len[g], s.seqs);
      const bool wide = unit < u.full || u.rest > s.seqs;
      parts.x = P.before[g] + unit * u.full_cost + kUnitCost;
      parts.y = (u.tiles - 1) * (wide ? kWideCost : kTurnCost);
      parts.z = P.stored[g] + i * a.G;
      parts.w = wide ? 0 : u.rest * a.G;
    }
    s.own[b] = own[b];
    s.row_shared[b] = g >= 0 ? P.len[g] : 0;
    s.row_parts[b] = parts;
  }
  if (tid == T - 1) {
    const int lo = share_start(cta, share, line), hi = share_start(cta + 1, share, line);
    Unit u{};
    u.next = hi;
    if (lo < hi) {
      const int h = lo / total, g = last_at_most(P.before, 0, s.groups - 1, lo - h * total);
      u = unit_at(lo, hi, cta, h, g, P.group(g), P.before[g], total, all[2], s.seqs, a.G);
    }
    P.first = u;
  }
}

// The new tokens of rows that lie below their group's shared length: they may
// go to a page that the group's shared positions are read from (its first
// row's own, above all), so every CTA writes them, for the KV heads that it
// reads, before its first copy. The others write the same bytes, at any time,
// as the own kernel does, which reports pages outside the pool. Where no row
// has a shared part, the CTAs divide the heads: the own kernel, which starts
// behind this, reads those tokens through any row's table. Kept small:
// the code alone, which hardly any call runs, costs 0.2 us of a call (two
// nested loops around append_token 0.3 to 2).
template <int D>
__device__ __forceinline__ void append_below(const DecodeArgs& a, const PlanSmem& P, const short* group) {
  const int total = P.totals.cost, share = P.totals.share, line = total * a.Hkv;
  const int lo = share_start(blockIdx.x, share, line), hi = share_start(blockIdx.x + 1, share, line);
  const int ctas = gridDim.x, cta = blockIdx.x;
  const int h0 = line > 0 ? lo / total : cta * a.Hkv / ctas;
  const int h1 = line > 0 ? (lo < hi ? (hi - 1) / total + 1 : h0) : (cta + 1) * a.Hkv / ctas;
  if (h0 < h1 && a.k_new != nullptr) {
    // a warp a row; of a KV head's D / 4 pieces, K's half comes first
    const int pieces = (h1 - h0) * (D / 4);
#pragma unroll 1
    for (int b = threadIdx.x / 32; b < a.B; b += kPrefixThreads / 32) {
      if (group[b] != kBelow) continue;
      const int pos = a.seq[b * a.seq_stride], bi = pos / a.bs;
      const int64_t blk = load_index(a.bt, a.bt_dtype, b * a.bt_stride + bi);
      if (blk < 0 || blk >= a.num_blocks) continue;
#pragma unroll 1
      for (int i = threadIdx.x % 32; i < pieces; i += 32) {
        const int h = h0 + i / (D / 4), d = i % (D / 8) * 8;
        const bool key = i % (D / 4) < D / 8;
        const int64_t at = blk * a.cs_block + h * a.cs_head + (pos - bi * a.bs) * a.cs_tok + d;
        const char* from = (key ? a.k_new + b * a.kn_b + h * a.kn_h : a.v_new + b * a.vn_b + h * a.vn_h) + d * 2;
        *reinterpret_cast<uint4*>((key ? a.kcache : a.vcache) + at * 2) = *reinterpret_cast<const uint4*>(from);
      }
    }
  }
  fence_proxy_async_global();
}

// ----------------------------------------------------------------- prefix
// Goes on to the CTA's next unit with key tiles: u, which is P.first at first
// (begun false). One thread of a role does this for all of it, in shared
// memory, so that the unit takes no registers of the softmax's.
__device__ __forceinline__ bool next_unit(const PlanSmem& P, const SharedArgs& s, const DecodeArgs& a, Unit& u,
                                          bool begun) {
  if (!begun) {
    u = P.first;
    if (u.t0 < u.t1) return true;
  }
  const int cost = P.totals.cost, hi = share_start(blockIdx.x + 1, P.totals.share, cost * a.Hkv);
  while (u.next < hi) {
    const int lo = u.next, h = lo / cost, x = lo - h * cost;
    int g = u.group;
    if (x < P.before[g] || x >= P.before[g + 1]) g = last_at_most(P.before, 0, s.groups - 1, x);
    u = unit_at(lo, hi, blockIdx.x, h, g, P.group(g), P.before[g], cost, P.totals.rows, s.seqs, a.G);
    if (u.t0 < u.t1) return true;
  }
  return false;
}
// The same for all lanes of a warp.
__device__ __forceinline__ bool warp_next_unit(const PlanSmem& P, const SharedArgs& s, const DecodeArgs& a, Unit& u,
                                               bool begun) {
  __syncwarp();
  bool more = false;
  if ((threadIdx.x & 31) == 0) more = next_unit(P, s, a, u, begun);
  __syncwarp();
  return __shfl_sync(0xffffffffu, (int)more, 0) != 0;
}

template <int D>
struct PrefixSmem {
  static constexpr int NP = D / 64;
  static constexpr int STAGES = D == 128 ? 2 : 3;  // of K and of V
  static constexpr int TILE = NP * kPanel;
  static constexpr int Q = 0;  // two row tiles
  static constexpr int K = Q + 2 * TILE;
  static constexpr int V = K + STAGES * TILE;
  static constexpr int BAR = V + STAGES * TILE;
  static constexpr int TMEM = BAR + 32 * 8;
  static constexpr int ABORT = TMEM + 8;
  static constexpr int PLAN = ABORT + 8;
  static constexpr int TOTAL = PLAN + (int)sizeof(PlanSmem) + 1024;
  // the plan's scratch lies where the queries come later
  static_assert(2 * TILE >= kMaxBatch * 6, "scratch of the plan");
  // above half an SM's shared memory: one CTA an SM, which takes all of its TMEM
  static constexpr int ALLOC = TOTAL > 120 * 1024 ? TOTAL : 120 * 1024;
};

enum PrefixBar {
  B_QF, B_QE,                    // a unit's queries are there; their last product is done
  B_KF, B_KE = B_KF + 3,         // a stage of K is filled, free
  B_VF = B_KE + 3, B_VE = B_VF + 3,
  B_SF = B_VE + 3,               // scores of x computed, and every product before them
  B_PF = B_SF + 2,               // probabilities of x written (4 warps)
  B_OF = B_PF + 2,               // a unit's last product of x is done
  B_OE = B_OF + 2,               // its result is read (4 warps)
  B_DONE = B_OE + 2, B_COUNT
};

// Eight floats times f, one whole sector of memory: a thread holds a row, so
// that narrower stores of a warp would each touch 32 sectors in part.
__device__ __forceinline__ void store_sector(float* to, const uint32_t* o, float f) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(o[i]) * f;
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// Roles as in the chunked prefill's 128-key kernel: two softmax warpgroups x
// = 0, 1, each with a score buffer (128 columns of TMEM, the probabilities
// written over its first half) and an accumulator (D columns). In a wide
// unit they hold a row tile each and both work on every key tile; in the
// others they share the one row tile and take the key tiles in turn, so that
// up to 128 rows keep both of them and the copies busy too.
//
// A wide tile takes a CTA 2.3 us, with the tensor pipe 65 % busy: the softmax
// warps bound it (scores computed a step ahead, where TMEM has room for them,
// change nothing). With few rows it is bound by HBM: 8 rows behind 65536
// positions of 8 KV heads, 268 MB in 45 us, 91 % of the copy rate.
template <int D, bool BF16>
__global__ void __launch_bounds__(kPrefixThreads, 1)
    shared_prefix_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const DecodeArgs a, const SharedArgs s) {
  using L = PrefixSmem<D>;
  constexpr int NP = L::NP, ST = L::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  volatile int* abort = reinterpret_cast<volatile int*>(sgen + L::ABORT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sgen + L::TMEM);
  auto bar = [&](int i) { return sbase + L::BAR + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *abort = 0;
    for (int i = 0; i < B_COUNT; ++i)
      mbar_init(bar(i), (i >= B_PF && i < B_PF + 2) || (i >= B_OE && i < B_OE + 2) ? 4u : 1u);
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // The set-up above overlaps what ran before. Behind the plan the own kernel
  // may start on the SMs that are left: it needs the plan and what ran before,
  // and not the rest of this grid.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  PlanSmem& P = *reinterpret_cast<PlanSmem*>(sgen + L::PLAN);
  short* group = reinterpret_cast<short*>(sgen + L::Q + kMaxBatch * 4);
  make_plan(a, s, P, reinterpret_cast<int*>(sgen + L::Q), group);
  if (P.below) append_below<D>(a, P, group);
  __threadfence();
  fence_proxy_async_smem();  // the scratch is written by copies next
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Unit& u = P.at[warp];
  const uint32_t tmem = *tmem_slot;
  auto t_s = [&](int x) { return tmem + x * 128; };
  auto t_o = [&](int x) { return tmem + 256 + x * 128; };
  const int rpb = min(a.bs, kKeys), boxes = kKeys / rpb;  // <= 16 boxes a tile
  // lane's box of key tile t: its block (num_blocks: none), first row there
  auto block_of = [&](int lead, int len, int t, int& row) {
    int blk = a.num_blocks;
    row = 0;
    const int key = t * kKeys + lane * rpb;
    if (lane < boxes && key < len) {
      const int bi = key / a.bs;
      row = key - bi * a.bs;
      const int64_t v = load_index(a.bt, a.bt_dtype, lead * a.bt_stride + bi);
      if (v >= 0 && v < a.num_blocks) blk = (int)v;
    }
    return blk;
  };

  if (warp >= 8) {
   setmaxnreg_dec<kRegsOther>();
   if (warp == 8 || warp == 10) {
    // ----------------------------------------------------------- producers
    // warp 8: queries and K, warp 10: V. A stage of V is freed by a product
    // that waits for the softmax, one of K long before: in one queue the next
    // K tiles would stand behind it.
    const bool keys = warp == 8;
    const CUtensorMap* tm = keys ? &tm_k : &tm_v;
    const int full = keys ? B_KF : B_VF, empty = keys ? B_KE : B_VE;
    const uint32_t ring = sbase + (keys ? L::K : L::V);
    if (lane == 0) {
      if (keys) prefetch_tmap(&tm_q);
      prefetch_tmap(tm);
    }
    int T = 0, act = 0;
    bool ok = true;
    for (; ok && warp_next_unit(P, s, a, u, act > 0); ++act) {
      if (keys) {
        if (act >= 1 && !__all_sync(0xffffffffu, mbar_wait(bar(B_QE), (act - 1) & 1, abort))) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar(B_QF), (u.wide ? 2 : 1) * NP * s.seqs * a.G * 128);
          for (int x = 0; x < (u.wide ? 2 : 1); ++x)
            for (int p = 0; p < NP; ++p)
              tma_load_4d(sbase + L::Q + x * L::TILE + p * kPanel, &tm_q, bar(B_QF), p * 64, 0, u.h, u.b0 + x * s.seqs);
        }
      }
      const int t1 = u.t1, lead = u.lead, len = u.len, h = u.h;
      for (int t = u.t0; t < t1; ++t, ++T) {
        int row;
        const int blk = block_of(lead, len, t, row);
        if (keys && blk == a.num_blocks && lane < boxes && t * kKeys + lane * rpb < len)
          flag_error(a.err, RBLN_DEVERR_BLOCK_ID_RANGE);
        const int st = T % ST;
        if (T >= ST && !__all_sync(0xffffffffu, mbar_wait(bar(empty + st), (T / ST - 1) & 1, abort))) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(bar(full + st), NP * kPanel);
        __syncwarp();
        if (lane < boxes)
          for (int p = 0; p < NP; ++p)
            tma_load_4d(ring + st * L::TILE + p * kPanel + lane * rpb * 128, tm, bar(full + st), p * 64, row, h, blk);
      }
    }
    if (*abort) {
      // let the copies in flight land before the CTA exits
      const long long t0 = clock64();
      for (int j = max(0, T - ST); j < T; ++j)
        while (!mbar_try_wait(bar(full + j % ST), (j / ST) & 1) && clock64() - t0 < 4000000) {
        }
    }
   } else if (warp == 9 && lane == 0) {
    // ----------------------------------------------------------------- MMA
    // Step j of a unit, for x = 0, 1: the product with V of x's tile of step
    // j - 1, then the scores of its tile of step j. x's tile of step j is
    // t0 + j in a wide unit, t0 + 2 j + x in another.
    const uint32_t id_qk = idesc_f16(BF16, kRows, kKeys, false), id_pv = idesc_f16(BF16, kRows, D, true);
    int T = 0, act = 0, n_s[2] = {0, 0}, n_o[2] = {0, 0};
    bool ok = true;
    for (; ok && next_unit(P, s, a, u, act > 0);) {
      const bool wide = u.wide;
      const int nt = u.t1 - u.t0, steps = wide ? nt : (nt + 1) / 2;
      if (!mbar_wait(bar(B_QF), act & 1, abort)) break;
      for (int j = 0; ok && j <= steps; ++j) {
        for (int x = 0; x < 2; ++x) {
          const int i1 = wide ? j : 2 * j + x, i0 = wide ? j - 1 : i1 - 2;
          if (j >= 1 && i0 < nt) {
            const int Ti = T + i0, st = Ti % ST;
            if (!mbar_wait(bar(B_VF + st), (Ti / ST) & 1, abort) ||
                !mbar_wait(bar(B_PF + x), (n_s[x] - 1) & 1, abort) ||
                (j == 1 && n_o[x] >= 1 && !mbar_wait(bar(B_OE + x), (n_o[x] - 1) & 1, abort))) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t vb = sbase + L::V + st * L::TILE;
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk)
              umma_f16_ts(t_o(x), t_s(x) + kk * 8, sw128_desc(vb + kk * 16 * 128, kPanel, 1024), id_pv,
                          (j > 1 || kk > 0) ? 1u : 0u);
            if (i1 >= nt) {  // x's last tile of the unit
              umma_commit(bar(B_OF + x));
              ++n_o[x];
            }
            if (!wide || x == 1) umma_commit(bar(B_VE + st));
          }
          if (i1 < nt) {
            const int Ti = T + i1, st = Ti % ST;
            if (!mbar_wait(bar(B_KF + st), (Ti / ST) & 1, abort)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t qb = sbase + L::Q + (wide ? x * L::TILE : 0), kb = sbase + L::K + st * L::TILE;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_f16_ss(t_s(x), sw128_desc(qb + (kk >> 2) * kPanel + (kk & 3) * 32, 16, 1024),
                          sw128_desc(kb + (kk >> 2) * kPanel + (kk & 3) * 32, 16, 1024), id_qk, kk > 0 ? 1u : 0u);
            umma_commit(bar(B_SF + x));
            ++n_s[x];
            if (!wide || x == 1) umma_commit(bar(B_KE + st));
            if (i1 == nt - 1 && (!wide || x == 1)) umma_commit(bar(B_QE));
          }
        }
      }
      T += nt;
      ++act;
    }
    if (*abort) {
      umma_commit(bar(B_DONE));
      const long long t0 = clock64();
      while (!mbar_try_wait(bar(B_DONE), 0) && clock64() - t0 < 4000000) {
      }
    }
   }
  } else {
    setmaxnreg_inc<kRegsSoftmax>();
    // ------------------------------------------------------------- softmax
    const int x = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const int bl = r / a.G, g = r - bl * a.G;  // the row's sequence in its tile, and query head
    const float scale = a.scale_dev ? *a.scale_dev : a.scale;
    const float qk_mult = scale * kLog2e;
    const float mult = qk_mult > 0.f ? qk_mult : 1.f;
    int T = 0, n_s = 0, n_o = 0;
    bool ok = true;
    for (bool begun = false; ok && warp_next_unit(P, s, a, u, begun); begun = true, T += u.t1 - u.t0) {
      const bool wide = u.wide;
      const int t1 = u.t1, len = u.len, lead = u.lead;
      const int i = (wide ? x * s.seqs : 0) + bl;
      const bool row_ok = bl < s.seqs && i < u.n;
      // rows that are none are not masked: nothing reads what they give
      // (a row whose new position is below the shared ones sees none of them)
      const int lim = !row_ok ? len + kKeys : a.seq[(u.b0 + i) * a.seq_stride] >= len ? len : 0;
      const bool rows = __any_sync(0xffffffffu, row_ok);  // a warp without any only keeps the barriers' count
      float m_run = neg_inf(), l_run = 0.f;
      int done = 0;
      const int step = wide ? 1 : 2;
      // keys in blocks outside the pool: looked up a tile ahead
      auto none_of = [&](int t) {
        int row;
        return t < t1 && block_of(lead, len, t, row) == a.num_blocks && lane < boxes && t * kKeys + lane * rpb < len;
      };
      int t = u.t0 + (wide ? 0 : x);
      bool none = none_of(t);
      for (; t < t1; t += step, ++done) {
        const uint32_t bad = __ballot_sync(0xffffffffu, none);
        none = none_of(t + step);
        if (!__all_sync(0xffffffffu, mbar_wait(bar(B_SF + x), n_s & 1, abort))) {
          ok = false;
          break;
        }
        ++n_s;
        tc_fence_after();
        __syncwarp();
       if (rows) {
        float xv[kKeys];
        {
          uint32_t r0[32], r1[32], r2[32], r3[32];
          tmem_ld32(t_s(x) + lane_off + 0, r0);
          tmem_ld32(t_s(x) + lane_off + 32, r1);
          tmem_ld32(t_s(x) + lane_off + 64, r2);
          tmem_ld32(t_s(x) + lane_off + 96, r3);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            xv[e] = __uint_as_float(r0[e]);
            xv[32 + e] = __uint_as_float(r1[e]);
            xv[64 + e] = __uint_as_float(r2[e]);
            xv[96 + e] = __uint_as_float(r3[e]);
          }
        }
        // The maximum is taken on raw scores (a positive factor keeps the
        // order), the scale folded into the exponent's multiply-add.
        if (!(qk_mult > 0.f)) {
#pragma unroll
          for (int e = 0; e < kKeys; e += 2) mul2(xv[e], xv[e + 1], qk_mult, qk_mult);
        }
        const int seen = lim - t * kKeys;  // of this tile's keys
        if (seen < kKeys || bad) {
          const int per = __ffs(rpb) - 4;  // a box has 8 << per keys
#pragma unroll
          for (int z = 0; z < kKeys / 8; ++z) {
            const int n = (bad >> (z >> per)) & 1u ? 0 : seen - 8 * z;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e >= n) xv[8 * z + e] = neg_inf();
          }
        }
        float mx0 = neg_inf(), mx1 = neg_inf(), mx2 = neg_inf(), mx3 = neg_inf();
#pragma unroll
        for (int e = 0; e < kKeys; e += 8) {
          mx0 = max3(mx0, xv[e], xv[e + 1]);
          mx1 = max3(mx1, xv[e + 2], xv[e + 3]);
          mx2 = max3(mx2, xv[e + 4], xv[e + 5]);
          mx3 = max3(mx3, xv[e + 6], xv[e + 7]);
        }
        const float m_new = fmaxf(m_run, max3(mx0, mx1, fmaxf(mx2, mx3)) * mult);
        // O is rescaled only when the maximum grows by more than 2^8
        const bool grow = m_new > m_run + 8.f;
        float factor = 1.f;
        if (grow) {
          factor = exp2_approx(m_run - m_new);
          l_run *= factor;
          m_run = m_new;
        }
        // x's last product with V is done (its scores' barrier says so)
        if (done > 0 && __any_sync(0xffffffffu, grow && factor != 1.f)) {
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
        const float nmu = (m_run == neg_inf()) ? 0.f : -m_run;
        // A probability is rounded once to the inputs' type, as the product's
        // operands have to be of one type; its sum is of the unrounded ones.
        // Exponents, sums and stores 32 keys at a time, so that the stores of
        // one part overlap the exponentials of the next. All exponentials on
        // the SFU: some of them on the FMA pipe, by a polynomial, measured no
        // faster (every 4th pair 374 us for the largest case, every 8th and
        // none 364; 430 with every 8th under the power cap, 422 with none).
        float sa0 = 0.f, sa1 = 0.f, sb0 = 0.f, sb1 = 0.f;
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 32 * c; e < 32 * c + 32; e += 2) {
            fma2(xv[e], xv[e + 1], mult, mult, nmu, nmu);
            xv[e] = exp2_approx(xv[e]);
            xv[e + 1] = exp2_approx(xv[e + 1]);
            if ((e / 2) & 1) {
              add2(sb0, sb1, xv[e], xv[e + 1]);
            } else {
              add2(sa0, sa1, xv[e], xv[e + 1]);
            }
            pk[(e - 32 * c) / 2] = pack2<BF16>(xv[e], xv[e + 1]);
          }
          tmem_st16(t_s(x) + lane_off + c * 16, pk);
        }
        l_run += (sa0 + sa1) + (sb0 + sb1);
        tmem_wait_st();
       }
        // rows of V behind the shared positions may hold anything: zeros
        // before the probabilities are released (in a wide unit by x = 0,
        // whose product comes first)
        if (t * kKeys + kKeys > len && (x == 0 || !wide)) {
          const int Ti = T + t - u.t0, st = Ti % ST;
          if (!__all_sync(0xffffffffu, mbar_wait(bar(B_VF + st), (Ti / ST) & 1, abort))) {
            ok = false;
            break;
          }
          if (t * kKeys + r >= len) {
            uint8_t* vrow = sgen + L::V + st * L::TILE + r * 128;
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(vrow + p * kPanel + c * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_PF + x));
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // x = 1 stores behind x = 0: other rows in a wide unit, the same ones of other keys else
      const int64_t at = u.row0 + (x == 0 ? 0 : (wide ? s.seqs : u.n) * a.G) + bl * a.G + g;
      if (done == 0) {
        if (row_ok) s.part_lse[at] = neg_inf();
        continue;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(bar(B_OF + x), n_o & 1, abort))) {
        ok = false;
        break;
      }
      ++n_o;
      tc_fence_after();
      const float inv = 1.f / l_run;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        __syncwarp();
        tmem_ld32(t_o(x) + lane_off + c * 32, o);
        tmem_wait_ld();
        if (row_ok) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) store_sector(s.part_o + at * D + c * 32 + e, o + e, inv);
        }
      }
      // (a row that saw nothing has l = 0; one whose scores are all NaN stays NaN)
      if (row_ok) s.part_lse[at] = l_run == 0.f ? neg_inf() : m_run + __log2f(l_run);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_OE + x));
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort && threadIdx.x == 0) flag_error(a.err, RBLN_DEVERR_TIMEOUT);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -------------------------------------------------------------------- own
// As paged_decode_balanced_kernel, over the positions that a sequence does
// not share; segments of CTA c in sequence b of KV head h are stored in slot
// c + h B + b.
template <int D, int KV, bool Q_BF16, int NT>
__device__ __forceinline__ void own_chunk(const DecodeArgs& a, const SharedArgs& s, unsigned char* dsm) {
  __shared__ int before[kWarps];
  const int c = blockIdx.x;
  // (the plan is read past L1: it was made while this grid could already be on its way)
  const int W = __ldcg(&s.totals->own_share), all = __ldcg(&s.totals->own);
  const long long lo = (long long)c * W, hi = min(lo + W, (long long)all * a.Hkv);
  if (lo >= hi) return;
  // the sequence at `lo`: all threads count those that start at or before it
  const int h = (int)(lo / all), x = (int)(lo - (long long)h * all);
  int n = 0;
  for (int i = threadIdx.x; i < a.B; i += kThreads) n += __ldcg(s.own + i) <= x;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) before[threadIdx.x >> 5] = n;
  __syncthreads();
  OwnPart p;
  p.h = h;
  p.b = before[0] + before[1] + before[2] + before[3] - 1;
  p.next = lo;
  while (true) {
    p = own_at(p.next, hi, p.h, p.b, all, __ldcg(s.own + p.b), __ldcg(s.own + p.b + 1), __ldcg(s.row_shared + p.b),
               a.seq[p.b * a.seq_stride], a.span);
    if (p.t0 < p.t1)
      decode_segment<D, KV, Q_BF16, NT, false>(a, dsm, p.b, p.h, p.t0, p.t1, p.append, p.whole,
                                               ((int64_t)c + (int64_t)p.h * a.B + p.b) * a.G);
    if (p.next >= hi) return;
    if (++p.b == a.B) {
      p.b = 0;
      ++p.h;
    }
  }
}

// Runs beside the prefix kernel, whose CTAs have all begun, so that the plan
// and everything before it is complete. It ends only when that kernel has, by
// its first CTA (the others leave their SMs to those that wait to start): the
// merge waits for this grid, and so for both.
//
// Bound by latency: a segment costs its CTA about 4.5 us besides its tiles
// (place, query, table, first rows; combine and store at the end). 48 GB/s an
// SM beside the prefix kernel, 39 where all SMs share HBM.
template <int D, int KV, bool Q_BF16, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 2) shared_own_kernel(const DecodeArgs a, const SharedArgs s) {
  extern __shared__ __align__(16) unsigned char dsm[];
  __threadfence();  // nothing is read from a cache line older than the plan
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  own_chunk<D, KV, Q_BF16, NT>(a, s, dsm);
  if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------------ merge
// CTA (h, b, z): the parts of one (KV head, sequence), a slice of its query
// heads; parts of the shared positions first, then of the sequence's own.
// Thread = (query head, 4 dims), eight parts at once; where the heads leave
// threads over, `ways` of them share a row's parts and are joined in shared
// memory. Where the parts are is known from the plan, before the wait.
template <int D, bool Q_BF16>
__global__ void __launch_bounds__(kThreads) shared_merge_kernel(const DecodeArgs a, const SharedArgs s) {
  constexpr int kBatch = 8, kLanes = D / 4, kSlots = kThreads / kLanes;
  __shared__ float4 s_acc[kSlots][kLanes];
  __shared__ float2 s_ml[kSlots];
  __threadfence();  // as in the own kernel
  const int h = blockIdx.x, b = blockIdx.y;
  const int gn = a.G / (int)gridDim.z, g0 = (int)blockIdx.z * gn;
  int pos;
  const int L = seq_len(a, b, pos);
  Totals tot;
  tot.cost = __ldcg(&s.totals->cost);
  tot.share = __ldcg(&s.totals->share);
  tot.rows = __ldcg(&s.totals->rows);
  tot.own = __ldcg(&s.totals->own);
  tot.own_share = __ldcg(&s.totals->own_share);
  const int4 rp = __ldcg(s.row_parts + b);
  const int pb = __ldcg(s.own + b) + kSegCost, pe = __ldcg(s.own + b + 1);
  const long long own0 = (long long)h * tot.own + pb;
  const int cf = (int)(own0 / tot.own_share), own = pe > pb ? (int)((own0 + pe - pb - 1) / tot.own_share) - cf + 1 : 0;
  const int64_t own_slot = ((int64_t)cf + (int64_t)h * a.B + b) * a.G;
  // of every CTA that has tiles of the row's unit, two where x = 0, 1 took the tiles in turn
  int parts = 0;
  const int turn = rp.w > 0 ? 1 : 0;
  int64_t row = 0;
  if (rp.y >= 0) {
    const int first = h * tot.cost + rp.x, c0 = first / tot.share, c1 = (first + rp.y) / tot.share;
    parts = (c1 - c0 + 1) << turn;
    row = (int64_t)c0 * 2 * kRows + h * tot.rows + rp.z;
  }
  const int slot = threadIdx.x / kLanes, d4 = (threadIdx.x % kLanes) * 4;
  const int ways = max(1, kSlots / gn), way = slot % ways;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (pos < 0 && h == 0 && blockIdx.z == 0 && threadIdx.x == 0) flag_error(a.err, RBLN_DEVERR_SEQ_RANGE);
  if (L > 0 && rp.y < 0 && own == 1) return;  // one chunk held the whole sequence and wrote the output
  for (int r0 = 0; r0 < gn; r0 += kSlots / ways) {
    const int r = r0 + slot / ways, g = g0 + r;
    const bool live = r < gn;
    float M = neg_inf(), S = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = way; live && s0 < parts + own; s0 += kBatch * ways) {
      float l[kBatch];
      float4 o[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = s0 + u * ways;
        l[u] = neg_inf();
        o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i >= parts + own) continue;
        const bool mine = i >= parts;
        const int64_t at = mine ? own_slot + (int64_t)(i - parts) * a.G + g
                                : row + (int64_t)(i >> turn) * 2 * kRows + (i & turn) * rp.w + g;
        l[u] = (mine ? a.part_lse : s.part_lse)[at];
        o[u] = *reinterpret_cast<const float4*>((mine ? a.part_o : s.part_o) + at * D + d4);
      }
      float mb = M;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) mb = fmaxf(mb, l[u]);
      if (mb != M) {  // M == -inf: S and acc are still 0
        const float c = (M == neg_inf()) ? 0.f : exp2_approx(M - mb);
        S *= c;
        acc.x *= c; acc.y *= c; acc.z *= c; acc.w *= c;
        M = mb;
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (l[u] != neg_inf()) {  // a part with nothing visible carries no weight
          const float w = exp2_approx(l[u] - M);
          S += w;
          acc.x += w * o[u].x; acc.y += w * o[u].y; acc.z += w * o[u].z; acc.w += w * o[u].w;
        }
    }
    if (ways > 1) {  // the same for all threads; then one pass takes all rows
      s_acc[slot][d4 / 4] = acc;
      if (d4 == 0) s_ml[slot] = make_float2(M, S);
      __syncthreads();
      if (way != 0) return;
      float top = neg_inf();
      for (int w = 0; w < ways; ++w) top = fmaxf(top, s_ml[slot + w].x);
      S = 0.f;
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < ways; ++w) {
        const float2 ml = s_ml[slot + w];
        if (ml.y == 0.f) continue;  // saw nothing (where all parts are NaN, S is, and the maximum is -inf too)
        const float f = exp2_approx(ml.x - top);
        const float4 o = s_acc[slot + w][d4 / 4];
        S += f * ml.y;
        acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w;
      }
      M = top;
    }
    if (!live) continue;
    // no position visible: NaN, as softmax of all -inf
    const float inv = (M == neg_inf()) ? pos_nan() : 1.f / S;
    acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    store_out(a, b, h, g, d4, make_uint2(pack2<Q_BF16>(acc.x, acc.y), pack2<Q_BF16>(acc.z, acc.w)));
  }
}

// -------------------------------------------------------------- host side
struct Maps {
  CUtensorMap q, k, v;
};

template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, const A&... args) {
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

template <int D, int KV, bool QB, int NT>
int launch(const DecodeArgs& a, const SharedArgs& s, const Maps& m, cudaStream_t st) {
  // the register split assumes 168 registers a thread at launch: with fewer
  // it would never be granted
  static const bool regs_ok = [] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, shared_prefix_kernel<D, QB>) == cudaSuccess &&
           2 * 128 * kRegsSoftmax + 128 * kRegsOther <= (uint32_t)fa.numRegs * kPrefixThreads;
  }();
  if (!regs_ok) return RBLN_ERR_LAUNCH;
  // The own kernel starts on SMs that the prefix kernel has just left, with
  // nearly all of their memory given to shared memory. Its loads in flight
  // need L1: it asks for the shared memory that its CTAs take and no more
  // (317 us against 443 beside 32768 shared positions).
  static SmemOptIn carved;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return RBLN_ERR_LAUNCH;
  if (carved.bytes[dev].load(std::memory_order_relaxed) == 0) {
    if (cudaFuncSetAttribute(shared_own_kernel<D, KV, QB, NT>, cudaFuncAttributePreferredSharedMemoryCarveout, 40) !=
        cudaSuccess)
      return RBLN_ERR_LAUNCH;
    carved.bytes[dev].store(1, std::memory_order_relaxed);
  }
  static SmemOptIn prefix_smem, own_smem;
  if (!allow_smem(reinterpret_cast<const void*>(shared_prefix_kernel<D, QB>), PrefixSmem<D>::ALLOC, prefix_smem) ||
      !allow_smem(reinterpret_cast<const void*>(shared_own_kernel<D, KV, QB, NT>), segment_smem<D, NT>(), own_smem))
    return RBLN_ERR_LAUNCH;
  int rc = launch_after(shared_prefix_kernel<D, QB>, dim3(s.ctas), kPrefixThreads, PrefixSmem<D>::ALLOC, st, m.q,
                        m.k, m.v, a, s);
  if (rc == RBLN_OK)
    rc = launch_after(shared_own_kernel<D, KV, QB, NT>, dim3(s.ctas * s.own_ctas), kThreads, segment_smem<D, NT>(), st,
                      a, s);
  if (rc == RBLN_OK)
    rc = launch_after(shared_merge_kernel<D, QB>, dim3(a.Hkv, a.B, merge_head_split(a.Hkv, a.B, a.G)), kThreads, 0, st, a,
                      s);
  return rc;
}

template <int D>
int launch_any(const DecodeArgs& a, const SharedArgs& s, const Maps& m, bool bf16, cudaStream_t st) {
  if (bf16) return a.G > 8 ? launch<D, KV_BF16, true, 2>(a, s, m, st) : launch<D, KV_BF16, true, 1>(a, s, m, st);
  return a.G > 8 ? launch<D, KV_F16, false, 2>(a, s, m, st) : launch<D, KV_F16, false, 1>(a, s, m, st);
}

struct Plan {
  int own_ctas;
  size_t totals, row_shared, row_parts, own, own_o, own_lse, part_o, part_lse, total;
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
  // a KV head's own positions are counted in 32 bits, in sixteens
  if ((int64_t)p->batch * ((int64_t)p->max_blocks * p->block_size / 16 + 1 + kSegCost) >= (int64_t)1 << 30)
    return RBLN_ERR_UNSUPPORTED;
  // the units' line, and a place up to a share past its end, are counted in 32 bits; the bound also keeps a share of
  // the own positions' line below 2^31
  const int64_t units = (int64_t)p->batch / (2 * (kRows / p->group)) + s->num_groups + 1;
  if (p->num_kv_heads * units * (kWideCost * tiles_of(p->max_blocks * p->block_size) + kUnitCost) >= (int64_t)1 << 30)
    return RBLN_ERR_UNSUPPORTED;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t start = at;
    at += (n + 255) / 256 * 256;
    return start;
  };
  pl->own_ctas = p->group <= 8 ? 4 : 2;  // an SM holds
  const size_t B = p->batch, N = s->num_groups, D = p->head_dim;
  const size_t own = (size_t)(kSms * pl->own_ctas + p->num_kv_heads * B) * p->group;
  // a row of the shared parts is stored once for each CTA that has keys of it: 256 rows a CTA at most, and a unit's
  // rows (twice them where its key tiles are taken in turn) for its first one
  const size_t part = N == 0 ? 0 : (size_t)kSms * 2 * kRows + 2 * B * p->group * p->num_kv_heads;
  pl->totals = take(sizeof(Totals));
  pl->row_shared = take(B * sizeof(int));
  pl->row_parts = take(B * sizeof(int4));
  pl->own = take((B + 1) * sizeof(int));
  pl->own_o = take(own * D * sizeof(float));
  pl->own_lse = take(own * sizeof(float));
  pl->part_o = take(part * D * sizeof(float));
  pl->part_lse = take(part * sizeof(float));
  pl->total = at + 256;
  return RBLN_OK;
}

int run_shared(const rbln_paged_attn_params_t* p_in, const rbln_shared_prefix_t* s, cudaStream_t st) {
  Plan pl;
  const int rc = plan_shared(p_in, s, &pl);
  if (rc != RBLN_OK) return rc;
  // a dimension of one entry has any stride: one that the tensor maps take
  rbln_paged_attn_params_t q = *p_in;
  const rbln_paged_attn_params_t* p = &q;
  if (q.batch == 1) q.q_stride[0] = q.out_stride[0] = q.k_new_stride[0] = q.v_new_stride[0] = q.head_dim;
  if (q.num_kv_heads == 1) {
    q.q_stride[1] = q.out_stride[1] = q.k_new_stride[1] = q.v_new_stride[1] = q.head_dim;
    q.cache_stride[1] = q.head_dim;
  }
  if (q.group == 1) q.q_stride[2] = q.out_stride[2] = q.head_dim;
  if (q.num_blocks == 1) q.cache_stride[0] = q.head_dim;
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
  const int64_t reach = ((int64_t)(p->num_blocks - 1) * p->cache_stride[0] +
                         (int64_t)(p->num_kv_heads - 1) * p->cache_stride[1] +
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
  a.part_o = reinterpret_cast<float*>(ws + pl.own_o);
  a.part_lse = reinterpret_cast<float*>(ws + pl.own_lse);
  SharedArgs x{};
  x.groups = s->num_groups;
  x.starts = s->group_starts;
  x.lens = s->shared_lens;
  x.seqs = kRows / p->group;
  x.ctas = kSms;
  x.own_ctas = pl.own_ctas;
  // Measured with both kernels at work: a wide tile 2.3 us, an own position (of up to four CTAs) 9 and 7 ns. From 7.8
  // to 12 ns the largest case took 409, 385, 385, 366, 371, 379, 392 us, smaller ones the same within a tenth. All of
  // it with up to 8 query heads a KV head: with more, two CTAs of the own kernel share an SM, for which none of these
  // times was measured.
  x.tile_us = 0.58f;
  x.own_us = p->head_dim == 128 ? 0.0092f : 0.0073f;
  // the merge is released sooner where the prefix kernel ends first: 2, 4, 6, 8, 10 us here gave 35.1, 33.4, 31.8, 32.2,
  // 33.0 us for 64 sequences behind 4096 positions
  x.late_us = p->head_dim == 128 ? 6.f : 4.f;
  x.totals = reinterpret_cast<Totals*>(ws + pl.totals);
  x.row_shared = reinterpret_cast<int*>(ws + pl.row_shared);
  x.row_parts = reinterpret_cast<int4*>(ws + pl.row_parts);
  x.own = reinterpret_cast<int*>(ws + pl.own);
  x.part_o = reinterpret_cast<float*>(ws + pl.part_o);
  x.part_lse = reinterpret_cast<float*>(ws + pl.part_lse);
  Maps m;
  {
    // queries [B, Hkv, G, D] in boxes of `seqs` sequences of one KV head, rows in order (sequence, query head)
    const uint64_t dims[4] = {(uint64_t)p->head_dim, (uint64_t)p->group, (uint64_t)p->num_kv_heads, (uint64_t)p->batch};
    const uint64_t strides[3] = {(uint64_t)q.q_stride[2] * 2, (uint64_t)q.q_stride[1] * 2, (uint64_t)q.q_stride[0] * 2};
    const uint32_t box[4] = {64, (uint32_t)p->group, 1, (uint32_t)x.seqs};
    const int rpb = std::min(p->block_size, kKeys);
    if (!make_map(&m.q, tmap_dtype(p->q_dtype), 4, const_cast<void*>(p->q), dims, strides, box) ||
        !map_kv(&m.k, p->kcache, p->kv_dtype, p->num_blocks, p->num_kv_heads, p->block_size, p->head_dim,
                q.cache_stride[0], q.cache_stride[1], q.cache_stride[2], rpb) ||
        !map_kv(&m.v, p->vcache, p->kv_dtype, p->num_blocks, p->num_kv_heads, p->block_size, p->head_dim,
                q.cache_stride[0], q.cache_stride[1], q.cache_stride[2], rpb))
      return RBLN_ERR_INVALID_ARGUMENT;
  }
  const bool bf16 = p->q_dtype == RBLN_DT_BF16;
  return p->head_dim == 128 ? launch_any<128>(a, x, m, bf16, st) : launch_any<64>(a, x, m, bf16, st);
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

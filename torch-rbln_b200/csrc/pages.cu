// Pages of a paged KV cache that several sequences share: forking sequences,
// giving them pages of their own before they write, taking pages back, and
// moving the pages in use to the front of the pool.
//
// refs[p] counts the table entries that hold page p; p is free when it is at
// most 0. One table serves the caches of all layers. The results do not
// depend on the order in which threads run: counts are sums, and pages are
// given by rank (the k-th entry in need, rows in order, gets the k-th free
// page in ascending order).
//
// The tables and counts are small, so those kernels are bound by the latency
// of their dependent look-ups: free, fork, reserve and the copies of 64 forks
// of 16 prompts through 24 layers take 14 us of GPU time, for 256 forks of one
// prompt of 2048 pages 18. A reservation alone takes 6 us for 128 entries among
// 4096 pages and 42 among 65536, all of which one CTA searches for free ones;
// the cluster that takes larger calls 18 among 65537, 22 for 2048 entries among
// 20000 and 53 for 12000 among 400000. What is copied is bound by HBM: 980
// pages of 16 layers, 2.05 GB read and written, 336 us with the ranking before
// it, 93 % of the copy rate.

#include <algorithm>

#include "common.cuh"

namespace rbln {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;  // CTAs of a planning cluster (the portable size)
constexpr int kCopyThreads = 256;
constexpr int kCopyLoads = 8;   // 16-byte loads in flight a lane
constexpr int kMaxLayers = 64;  // a launch's layers: their pointers are kernel parameters

__device__ __forceinline__ void store_index(void* base, int dtype, int64_t i, int64_t v) {
  switch (dtype) {
    case RBLN_DT_I16: static_cast<int16_t*>(base)[i] = (int16_t)v; break;
    case RBLN_DT_I64: static_cast<int64_t*>(base)[i] = v; break;
    default: static_cast<int32_t*>(base)[i] = (int32_t)v;
  }
}

struct Table {
  void* ids;
  int dtype;
  int64_t s_row, s_col;
  int rows, cols, num_blocks, bs;
  int* refs;
};

__device__ __forceinline__ int64_t entry(const Table& t, int64_t row, int64_t col) {
  return load_index(t.ids, t.dtype, row * t.s_row + col * t.s_col);
}
__device__ __forceinline__ bool is_page(const Table& t, int64_t id) { return id >= 0 && id < t.num_blocks; }

struct Lengths {
  const void* at;
  int dtype;
  int64_t stride;
};
// A row's number of positions, cut to [-1, span] (span below 2^31).
__device__ __forceinline__ int length_of(const Lengths& l, int64_t row, int span) {
  const int64_t n = load_index(l.at, l.dtype, row * l.stride);
  return n < 0 ? -1 : (int)min(n, (int64_t)span);
}

// ------------------------------------------------------------------- fork
struct ForkArgs {
  Table t;
  Lengths len;
  const void* parents;
  int parents_dtype;
  int64_t parents_stride;
  int forks, span;
  void* out;
  int64_t os_row;
  void* len_out;  // the lengths' type
};

// CTA (x, y): row x, column part y of 256. Rows [0, B) are the parents: their
// pages' counts go up by the number of forks that they have, one atomic an
// entry however many forks share it. Rows from B on are the forks.
__global__ void __launch_bounds__(256) paged_kv_fork_kernel(const ForkArgs a) {
  const int col = blockIdx.y * 256 + threadIdx.x;
  if ((int)blockIdx.x < a.t.rows) {
    const int b = blockIdx.x;
    int n = 0;
    for (int i = threadIdx.x; i < a.forks; i += 256)
      n += load_index(a.parents, a.parents_dtype, i * a.parents_stride) == b;
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    __shared__ int sum[8];
    if ((threadIdx.x & 31) == 0) sum[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < 8; ++w) n += sum[w];
    if (n == 0 || col >= a.t.cols || (int64_t)col * a.t.bs >= length_of(a.len, b, a.span)) return;
    const int64_t id = entry(a.t, b, col);
    if (is_page(a.t, id)) atomicAdd(a.t.refs + id, n);
    return;
  }
  const int i = blockIdx.x - a.t.rows;
  const int64_t parent = load_index(a.parents, a.parents_dtype, i * a.parents_stride);
  const bool known = parent >= 0 && parent < a.t.rows;
  const int len = known ? max(0, length_of(a.len, parent, a.span)) : 0;
  if (blockIdx.y == 0 && threadIdx.x == 0) store_index(a.len_out, a.len.dtype, i, len);
  if (col >= a.t.cols) return;
  int64_t id = -1;
  if ((int64_t)col * a.t.bs < len) {
    id = entry(a.t, parent, col);
    if (!is_page(a.t, id)) id = -1;
  }
  store_index(a.out, a.t.dtype, i * a.os_row + col, id);
}

// ------------------------------------------------------------------- free
constexpr int kFreeRows = 16;

// CTA (x, y): 16 rows of 256 columns, a thread a column, all its loads at
// once. Forks of one parent hold the same page in a column: a run of equal
// entries is one atomic. A count goes down by n, never below 0: what a
// decrement takes too much it puts back, and none sees a count above the true
// one.
__global__ void __launch_bounds__(256) paged_kv_free_kernel(const Table t, const Lengths keep, int span) {
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= t.cols) return;
  const int r0 = blockIdx.x * kFreeRows;
  int64_t id[kFreeRows];
#pragma unroll
  for (int i = 0; i < kFreeRows; ++i) id[i] = r0 + i < t.rows ? entry(t, r0 + i, col) : -1;
  bool gone[kFreeRows];
#pragma unroll
  for (int i = 0; i < kFreeRows; ++i)
    gone[i] = r0 + i < t.rows && (int64_t)col * t.bs >= length_of(keep, r0 + i, span);
  int page[kFreeRows], n[kFreeRows];  // runs: the page, how many entries end here
  int last = -1, run = 0;
#pragma unroll
  for (int i = 0; i < kFreeRows; ++i) {
    if (gone[i] && id[i] != -1) store_index(t.ids, t.dtype, (int64_t)(r0 + i) * t.s_row + col * t.s_col, -1);
    const int p = gone[i] && is_page(t, id[i]) ? (int)id[i] : -1;
    const bool same = p == last;
    page[i] = last;
    n[i] = p < 0 || same ? 0 : run;  // a page behind another one ends that one's run
    if (p >= 0) {
      run = same ? run + 1 : 1;
      last = p;
    }
  }
  int old[kFreeRows + 1];
#pragma unroll
  for (int i = 0; i < kFreeRows; ++i) old[i] = n[i] > 0 ? atomicSub(t.refs + page[i], n[i]) : 0;
  old[kFreeRows] = run > 0 ? atomicSub(t.refs + last, run) : 0;
#pragma unroll
  for (int i = 0; i < kFreeRows; ++i)
    if (old[i] < n[i]) atomicAdd(t.refs + page[i], n[i] - max(old[i], 0));
  if (old[kFreeRows] < run) atomicAdd(t.refs + last, run - max(old[kFreeRows], 0));
}

// --------------------------------------------------------------- planning
// A cluster's barrier, with what its CTAs wrote to global memory visible
// behind it (readers use __ldcg: L1 is not coherent).
__device__ __forceinline__ void cluster_sync() {
  __threadfence();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Sum of v over the threads of the CTA before this one; all of them in total.
__device__ __forceinline__ int block_before(int v, int* total) {
  __shared__ int warps[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last call's sums have been read
  if (lane == 31) warps[warp] = x;
  __syncthreads();
  int s = warps[lane];
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  const int before = __shfl_sync(0xffffffffu, s, warp > 0 ? warp - 1 : 0);
  return (warp > 0 ? before : 0) + x - v;
}

// Sums over the CTAs of the grid before this one and over all of them, of
// what each left at ctas[2 * i + which].
__device__ __forceinline__ int ctas_before(const int* ctas, int which, int* total) {
  int before = 0, all = 0;
  for (int i = 0; i < (int)gridDim.x; ++i) {
    const int n = __ldcg(ctas + 2 * i + which);
    before += i < (int)blockIdx.x ? n : 0;
    all += n;
  }
  *total = all;
  return before;
}

// A page copy: rows [0, rows) of page src to page dst.
struct Move {
  int src, dst, rows;
};

struct ReserveArgs {
  Table t;
  Lengths seq;
  int span, fresh_tokens, slots;  // slots: entries a row may need
  int64_t entries;                // rows x slots, or 0
  int* granted;
  int* ctas;   // [2 * kPlanCtas]: entries in need, free pages
  int* here;   // [num_blocks] this call's entries that hold the page
  int* last;   // [num_blocks] the last of them
  int* given;  // [rows * slots] pages by rank
  int* take;   // [rows * slots] the page that an entry gets
  Move* moves;
  int* count;  // of moves
};

struct Want {
  int64_t id;  // the entry as it is
  int row, col, seq;
  bool want, page;
};
__device__ __forceinline__ Want want_of(const ReserveArgs& a, int64_t i) {
  Want w{};
  w.row = (int)((uint32_t)i / (uint32_t)a.slots);  // entries stay below 2^31
  w.seq = length_of(a.seq, w.row, a.span);
  if (w.seq < 0) return w;
  w.col = w.seq / a.t.bs + (int)i - w.row * a.slots;
  // 64 bits: seq + new tokens and the columns behind the table may pass 2^31
  w.want = (int64_t)w.col * a.t.bs < min((int64_t)w.seq + a.fresh_tokens, (int64_t)a.span);
  if (!w.want) return w;
  w.id = entry(a.t, w.row, w.col);
  w.page = is_page(a.t, w.id);
  return w;
}

// Whether entry i needs a page: it has none, or one that others hold too. Of
// a page that only entries of this call hold, the last of them keeps it: by
// then all others have moved.
__device__ __forceinline__ bool needs(const ReserveArgs& a, const Want& w, int64_t i) {
  if (!w.want) return false;
  if (!w.page) return true;
  const int n = __ldcg(a.t.refs + w.id);
  return n > 1 && !(__ldcg(a.here + w.id) >= n && __ldcg(a.last + w.id) == (int)i);
}

// One cluster. Thread g of it (in order) takes entries [g e, (g + 1) e) and
// pages [g p, (g + 1) p), so that a scan over threads ranks both.
__global__ void __launch_bounds__(kPlanThreads, 1) paged_kv_reserve_kernel(const ReserveArgs a) {
  const int threads = gridDim.x * kPlanThreads, g = blockIdx.x * kPlanThreads + threadIdx.x;
  const int64_t n = a.entries;
  const int64_t e_per = (n + threads - 1) / threads, p_per = ((int64_t)a.t.num_blocks + threads - 1) / threads;
  const int64_t e0 = min(g * e_per, n), e1 = min(e0 + e_per, n);
  const int64_t p0 = min(g * p_per, (int64_t)a.t.num_blocks), p1 = min(p0 + p_per, (int64_t)a.t.num_blocks);

  for (int b = g; b < a.t.rows; b += threads) {
    const int seq = length_of(a.seq, b, a.span);
    a.granted[b] = seq < 0 ? 0 : (int)min((int64_t)a.fresh_tokens, (int64_t)a.span - seq);
  }
  if (g == 0) *a.count = 0;
  for (int64_t i = e0; i < e1; ++i) {
    const Want w = want_of(a, i);
    if (w.page && a.t.refs[w.id] > 1) {
      a.here[w.id] = 0;
      a.last[w.id] = -1;
    }
  }
  int unused = 0;
  for (int64_t p = p0; p < p1; ++p) unused += a.t.refs[p] <= 0;
  cluster_sync();
  for (int64_t i = e0; i < e1; ++i) {
    const Want w = want_of(a, i);
    if (w.page && a.t.refs[w.id] > 1) {
      atomicAdd(a.here + w.id, 1);
      atomicMax(a.last + w.id, (int)i);
    }
  }
  cluster_sync();
  int need = 0;
  for (int64_t i = e0; i < e1; ++i) need += needs(a, want_of(a, i), i);
  int cta_need, cta_unused;
  int rank = block_before(need, &cta_need);
  int page_rank = block_before(unused, &cta_unused);
  if (threadIdx.x == 0) {
    a.ctas[2 * blockIdx.x] = cta_need;
    a.ctas[2 * blockIdx.x + 1] = cta_unused;
  }
  cluster_sync();
  int all_need, all_unused;
  rank += ctas_before(a.ctas, 0, &all_need);
  page_rank += ctas_before(a.ctas, 1, &all_unused);
  if (unused)
    for (int64_t p = p0; p < p1 && page_rank < all_need; ++p)
      if (a.t.refs[p] <= 0) a.given[page_rank++] = (int)p;
  cluster_sync();
  for (int64_t i = e0; i < e1; ++i) {
    int page = -1;
    if (needs(a, want_of(a, i), i)) {
      if (rank < all_unused) page = __ldcg(a.given + rank);
      ++rank;
    }
    a.take[i] = page;
  }
  cluster_sync();  // every need is settled before a count changes
  for (int64_t i = e0; i < e1; ++i) {
    const int page = a.take[i];
    if (page < 0) continue;
    const Want w = want_of(a, i);
    store_index(a.t.ids, a.t.dtype, w.row * a.t.s_row + w.col * a.t.s_col, page);
    a.t.refs[page] = 1;
    if (!w.page) continue;
    atomicSub(a.t.refs + w.id, 1);
    const int rows = w.seq - w.col * a.t.bs;  // of the first entry's page, those that the sequence holds
    if (rows > 0) a.moves[atomicAdd(a.count, 1)] = Move{(int)w.id, page, rows};
  }
  cluster_sync();
  // an entry may be written when nothing else holds its page
  for (int64_t i = e0; i < e1; ++i) {
    const Want w = want_of(a, i);
    if (w.want && !(w.page && __ldcg(a.t.refs + w.id) <= 1))
      atomicMin(a.granted + w.row, max(w.col * a.t.bs - w.seq, 0));
  }
}

constexpr int kSmallEntries = kPlanThreads;  // one a thread
constexpr int kSmallPages = 64 * kPlanThreads;
constexpr int kSlots = 2 * kSmallEntries;    // of the table of shared pages, a power of two

// The same for one entry a thread: one CTA, in which an entry is looked up
// once, and what the entries share is in shared memory. Three dependent
// reads (length, entry, count) beside the search for free pages.
__global__ void __launch_bounds__(kPlanThreads, 1) paged_kv_reserve_small_kernel(const ReserveArgs a) {
  __shared__ int key[kSlots], here[kSlots], last[kSlots];  // shared pages of this call's entries
  __shared__ int given[kSmallEntries];
  const int i = threadIdx.x, n = (int)a.entries;
  Want w{};
  if (i < n) w = want_of(a, i);
  for (int k = i; k < kSlots; k += kPlanThreads) {
    key[k] = here[k] = last[k] = -1;
  }
  for (int b = i; b < a.t.rows; b += kPlanThreads) {
    const int seq = length_of(a.seq, b, a.span);
    a.granted[b] = seq < 0 ? 0 : (int)min((int64_t)a.fresh_tokens, (int64_t)a.span - seq);
  }
  const int p_per = (a.t.num_blocks + kPlanThreads - 1) / kPlanThreads;
  const int p0 = min(i * p_per, a.t.num_blocks), p1 = min(p0 + p_per, a.t.num_blocks);
  uint64_t free_mask = 0;  // p_per <= 64
#pragma unroll 8
  for (int p = p0; p < p1; ++p) free_mask |= (uint64_t)(a.t.refs[p] <= 0) << (p - p0);
  const int count = w.page ? a.t.refs[w.id] : 0;
  const bool held = count > 1;
  __syncthreads();
  int slot = 0;
  if (held) {
    slot = (int)(((uint32_t)w.id * 2654435761u) >> 16) & (kSlots - 1);
    while (true) {  // at most as many pages as threads: half of the slots
      const int was = atomicCAS(key + slot, -1, (int)w.id);
      if (was == -1 || was == (int)w.id) break;
      slot = (slot + 1) & (kSlots - 1);
    }
    atomicAdd(here + slot, 1);  // from -1
    atomicMax(last + slot, i);
  }
  __syncthreads();
  const bool keeps = held && here[slot] + 1 >= count && last[slot] == i;
  const bool need = w.want && (!w.page || (held && !keeps));
  int all_need, all_unused;
  const int rank = block_before(need, &all_need);
  int page_rank = block_before(__popcll(free_mask), &all_unused);
  for (uint64_t m = free_mask; m && page_rank < all_need; m &= m - 1) given[page_rank++] = p0 + __ffsll((long long)m) - 1;
  here[i] = here[i + kSmallEntries] = 0;  // from here on: entries that moved
  __syncthreads();
  const bool got = need && rank < all_unused;
  if (got) {
    const int page = given[rank];
    store_index(a.t.ids, a.t.dtype, w.row * a.t.s_row + w.col * a.t.s_col, page);
    a.t.refs[page] = 1;
    if (held) {
      atomicSub(a.t.refs + w.id, 1);
      atomicAdd(here + slot, 1);
    }
  }
  const bool copies = got && held && w.seq > w.col * a.t.bs;
  int all_copies;
  const int move = block_before(copies, &all_copies);  // its barriers order the counts in `here`, too
  if (copies) a.moves[move] = Move{(int)w.id, given[rank], w.seq - w.col * a.t.bs};
  if (i == 0) *a.count = all_copies;
  if (w.want && !got && !(w.page && count - (held ? here[slot] : 0) <= 1))
    atomicMin(a.granted + w.row, max(w.col * a.t.bs - w.seq, 0));
}

struct CompactArgs {
  int* refs;
  int num_blocks, bs;
  int* moved;
  int* live;
  int* ctas;
  int* src;  // [num_blocks] pages that move, ascending
  int* dst;  // [num_blocks] where to
  Move* moves;
  int* count;
};

// One cluster, pages in threads' order as above. With `live` pages in use,
// the i-th free page below `live` takes the i-th page in use from there on:
// as many as there are of the other, and no page is both read and written.
__global__ void __launch_bounds__(kPlanThreads, 1) paged_kv_compact_kernel(const CompactArgs a) {
  const int threads = gridDim.x * kPlanThreads, g = blockIdx.x * kPlanThreads + threadIdx.x;
  const int64_t p_per = ((int64_t)a.num_blocks + threads - 1) / threads;
  const int p0 = (int)min(g * p_per, (int64_t)a.num_blocks), p1 = (int)min(p0 + p_per, (int64_t)a.num_blocks);
  // this thread's pages in use, kept as bits where 64 hold them
  uint64_t mask = 0;
  const bool bits = p_per <= 64;
  int used = 0, cta_used, live;
#pragma unroll 8
  for (int p = p0; p < p1; ++p) {
    const bool in = a.refs[p] > 0;
    used += in;
    if (bits) mask |= (uint64_t)in << (p - p0);
  }
  auto in_use = [&](int p) { return bits ? (mask >> (p - p0)) & 1 : a.refs[p] > 0; };
  block_before(used, &cta_used);
  if (threadIdx.x == 0) a.ctas[2 * blockIdx.x] = cta_used;
  cluster_sync();
  ctas_before(a.ctas, 0, &live);
  int holes = 0, movers = 0, n;
  for (int p = p0; p < p1; ++p) {
    const bool in = in_use(p);
    holes += p < live && !in;
    movers += p >= live && in;
  }
  int hole = block_before(holes, &n), *ctas = a.ctas + 2 * kPlanCtas;
  if (threadIdx.x == 0) ctas[2 * blockIdx.x] = n;
  int mover = block_before(movers, &n);
  if (threadIdx.x == 0) ctas[2 * blockIdx.x + 1] = n;
  cluster_sync();
  int all;
  hole += ctas_before(ctas, 0, &all);
  mover += ctas_before(ctas, 1, &all);
  for (int p = p0; p < p1; ++p) {
    const bool in = in_use(p);
    if (p < live && !in) a.dst[hole++] = p;
    if (p >= live && in) a.src[mover++] = p;
    a.moved[p] = in ? p : -1;
  }
  if (g == 0) {
    *a.live = live;
    *a.count = all;
  }
  cluster_sync();
  for (int i = g; i < all; i += threads) {
    const int s = __ldcg(a.src + i), d = __ldcg(a.dst + i);
    a.moves[i] = Move{s, d, a.bs};
    a.moved[s] = d;
    a.refs[d] = __ldcg(a.refs + s);
    a.refs[s] = 0;
  }
}

// ------------------------------------------------------------------- copy
struct CopyArgs {
  const Move* moves;
  const int* count;
  int layers, Hkv, row_vec;            // 16-byte pieces a row
  int64_t cs_block, cs_head, cs_tok;   // bytes
  int64_t ss_block, ss_head;           // elements; scales when ks[0] is set
  Table t;                             // entries follow `moved` when that is set
  const int* moved;
  char* k[kMaxLayers];
  char* v[kMaxLayers];
  float* ks[kMaxLayers];
  float* vs[kMaxLayers];
};

// A warp copies the rows of one (move, layer, K or V, head) at a time, eight
// 16-byte loads a lane in flight. Launched as a programmatic dependent of the
// kernel that plans the moves.
__global__ void __launch_bounds__(kCopyThreads) paged_kv_pages_copy_kernel(const __grid_constant__ CopyArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  if (a.moved != nullptr) {
    const int64_t n = (int64_t)a.t.rows * a.t.cols;
    for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kCopyThreads) {
      const int64_t row = i / a.t.cols, col = i - row * a.t.cols, id = entry(a.t, row, col);
      if (!is_page(a.t, id)) continue;
      const int now = a.moved[id];
      if (now >= 0 && now != id) store_index(a.t.ids, a.t.dtype, row * a.t.s_row + col * a.t.s_col, now);
    }
  }
  const int64_t tasks = (int64_t)*a.count * a.layers * 2 * a.Hkv;
  const int64_t warps = (int64_t)gridDim.x * (kCopyThreads / 32);
  for (int64_t x = (int64_t)blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); x < tasks; x += warps) {
    int64_t y = x / a.Hkv;
    const int h = (int)(x - y * a.Hkv), part = (int)(y & 1);
    y >>= 1;
    const int64_t item = y / a.layers;
    const int layer = (int)(y - item * a.layers);
    const Move m = a.moves[item];
    float* scale = nullptr;
    float old = 0.f;
    if (lane == 0 && a.ks[0] != nullptr) {
      scale = (part ? a.vs : a.ks)[layer] + h * a.ss_head;
      old = scale[m.src * a.ss_block];  // on its way while the rows are copied
    }
    char* base = (part ? a.v : a.k)[layer] + h * a.cs_head;
    const char* from = base + m.src * a.cs_block;
    char* to = base + m.dst * a.cs_block;
    const int vecs = m.rows * a.row_vec;
    const bool dense = a.cs_tok == a.row_vec * 16;
    for (int i0 = lane; i0 < vecs; i0 += 32 * kCopyLoads) {
      uint4 w[kCopyLoads];
      int64_t at[kCopyLoads];
#pragma unroll
      for (int u = 0; u < kCopyLoads; ++u) {
        const int i = i0 + 32 * u;
        if (i >= vecs) break;
        const int row = dense ? 0 : i / a.row_vec;
        at[u] = dense ? (int64_t)i * 16 : row * a.cs_tok + (i - row * a.row_vec) * 16;
        w[u] = ld_stream_v4(from + at[u]);
      }
#pragma unroll
      for (int u = 0; u < kCopyLoads; ++u)
        if (i0 + 32 * u < vecs) *reinterpret_cast<uint4*>(to + at[u]) = w[u];
    }
    if (scale != nullptr) scale[m.dst * a.ss_block] = old;
  }
}

// -------------------------------------------------------------- host side
bool index_type(int dt) { return dt == RBLN_DT_I16 || dt == RBLN_DT_I32 || dt == RBLN_DT_I64; }
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

int check_table(const rbln_pages_params_t* p, bool lengths = true) {
  if (!p || p->batch < 0 || p->max_blocks < 0 || p->num_blocks < 0 || p->block_size <= 0)
    return RBLN_ERR_INVALID_ARGUMENT;
  if (!index_type(p->block_table_dtype) || (lengths && !index_type(p->lengths_dtype))) return RBLN_ERR_UNSUPPORTED;
  if (p->block_table_dtype == RBLN_DT_I16 && p->num_blocks > 32768) return RBLN_ERR_UNSUPPORTED;
  if ((int64_t)p->max_blocks * p->block_size > INT32_MAX) return RBLN_ERR_UNSUPPORTED;
  if ((p->batch > 0 && p->max_blocks > 0 && !p->block_table) || (lengths && p->batch > 0 && !p->lengths) ||
      (p->num_blocks > 0 && !p->refs))
    return RBLN_ERR_INVALID_ARGUMENT;
  return RBLN_OK;
}

int check_caches(const rbln_pages_params_t* p) {
  if (p->num_layers < 1 || p->num_kv_heads < 1 || p->head_dim < 1 || !p->kcaches || !p->vcaches)
    return RBLN_ERR_INVALID_ARGUMENT;
  const bool half = p->kv_dtype == RBLN_DT_F16 || p->kv_dtype == RBLN_DT_BF16;
  const int size = p->kv_dtype == RBLN_DT_FP8_E4M3 ? 1 : half ? 2 : 0;
  if (size == 0) return RBLN_ERR_UNSUPPORTED;
  if ((p->k_scales == nullptr) != (p->v_scales == nullptr) || (size == 1) != (p->k_scales != nullptr))
    return RBLN_ERR_INVALID_ARGUMENT;
  if (p->head_dim * size % 16 != 0) return RBLN_ERR_INVALID_ARGUMENT;
  // a page's rows are counted in 16-byte pieces, in 32 bits, with room for a step of the copy past their end
  if (p->block_size * ((int64_t)p->head_dim * size / 16) > INT32_MAX - 32 * kCopyLoads) return RBLN_ERR_UNSUPPORTED;
  for (int i = 0; i < 3; ++i)
    if (p->cache_stride[i] * size % 16 != 0) return RBLN_ERR_INVALID_ARGUMENT;
  if (p->num_blocks == 0) return RBLN_OK;
  for (int l = 0; l < p->num_layers; ++l) {
    const uintptr_t k = reinterpret_cast<uintptr_t>(p->kcaches[l]), v = reinterpret_cast<uintptr_t>(p->vcaches[l]);
    if (!k || !v || ((k | v) & 15u)) return RBLN_ERR_INVALID_ARGUMENT;
    if (size == 1 && (!p->k_scales[l] || !p->v_scales[l])) return RBLN_ERR_INVALID_ARGUMENT;
  }
  return RBLN_OK;
}

Table table_of(const rbln_pages_params_t* p) {
  Table t{};
  t.ids = p->block_table;
  t.dtype = p->block_table_dtype;
  t.s_row = p->block_table_stride[0];
  t.s_col = p->block_table_stride[1];
  t.rows = p->batch;
  t.cols = p->max_blocks;
  t.num_blocks = p->num_blocks;
  t.bs = p->block_size;
  t.refs = p->refs;
  return t;
}
Lengths lengths_of(const rbln_pages_params_t* p) { return Lengths{p->lengths, p->lengths_dtype, p->lengths_stride}; }
int span_of(const rbln_pages_params_t* p) { return p->max_blocks * p->block_size; }

// Entries that a row's next `tokens` positions may touch.
int64_t slots_of(const rbln_pages_params_t* p, int tokens) {
  if (tokens <= 0) return 0;
  return std::min<int64_t>((int64_t)(tokens - 1) / p->block_size + 2, p->max_blocks);
}

struct Workspace {
  size_t ctas, here, last, given, take, moves, total;
};
// Reserve: entries = rows x slots, moves <= rows. Compact (entries < 0): here
// and last hold the pages that move and where to, moves <= num_blocks.
Workspace workspace_of(const rbln_pages_params_t* p, int64_t entries) {
  Workspace w{};
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t start = at;
    at += round256(n);
    return start;
  };
  const size_t e = entries < 0 ? 0 : (size_t)entries;
  w.ctas = take((4 * kPlanCtas + 1) * sizeof(int));
  w.here = take((size_t)p->num_blocks * sizeof(int));
  w.last = take((size_t)p->num_blocks * sizeof(int));
  w.given = take(e * sizeof(int));
  w.take = take(e * sizeof(int));
  w.moves = take((entries < 0 ? (size_t)p->num_blocks : (size_t)p->batch) * sizeof(Move));
  w.total = at + 256;
  return w;
}

template <typename A>
int launch_plan(void (*kernel)(A), int ctas, cudaStream_t st, const A& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? RBLN_OK : RBLN_ERR_LAUNCH;
}

// Launches the copies of `most` moves at most, and of the table's entries
// after `moved` when that is given, 64 layers a launch.
int launch_copies(const rbln_pages_params_t* p, const Move* moves, const int* count, int64_t most, const int* moved,
                  cudaStream_t st) {
  const int size = p->kv_dtype == RBLN_DT_FP8_E4M3 ? 1 : 2;
  for (int l0 = 0; l0 < p->num_layers; l0 += kMaxLayers) {
    CopyArgs a{};
    a.moves = moves;
    a.count = count;
    a.layers = std::min(kMaxLayers, p->num_layers - l0);
    a.Hkv = p->num_kv_heads;
    a.row_vec = p->head_dim * size / 16;
    a.cs_block = p->cache_stride[0] * size;
    a.cs_head = p->cache_stride[1] * size;
    a.cs_tok = p->cache_stride[2] * size;
    a.ss_block = p->scale_stride[0];
    a.ss_head = p->scale_stride[1];
    a.t = table_of(p);
    a.moved = l0 == 0 ? moved : nullptr;
    for (int l = 0; l < a.layers; ++l) {
      a.k[l] = static_cast<char*>(p->kcaches[l0 + l]);
      a.v[l] = static_cast<char*>(p->vcaches[l0 + l]);
      if (size == 1) {
        a.ks[l] = p->k_scales[l0 + l];
        a.vs[l] = p->v_scales[l0 + l];
      }
    }
    const int64_t tasks = most * a.layers * 2 * a.Hkv, entries = moved ? (int64_t)p->batch * p->max_blocks : 0;
    const int64_t want = std::max((tasks + 7) / 8, (entries + kCopyThreads - 1) / kCopyThreads);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(std::max<int64_t>(want, 1), 148 * 8));
    cfg.blockDim = dim3(kCopyThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, paged_kv_pages_copy_kernel, a) != cudaSuccess) return RBLN_ERR_LAUNCH;
  }
  return RBLN_OK;
}

char* workspace_base(const rbln_pages_params_t* p) {
  return reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p->workspace) + 255) & ~uintptr_t(255));
}

int launched() { return cudaGetLastError() == cudaSuccess ? RBLN_OK : RBLN_ERR_LAUNCH; }

}  // namespace
}  // namespace rbln

using namespace rbln;

extern "C" {

size_t rbln_pages_params_sizeof(void) { return sizeof(rbln_pages_params_t); }

int rbln_paged_kv_fork(const rbln_pages_params_t* p, const void* parents, int32_t parents_dtype,
                       int64_t parents_stride, int32_t forks, void* table_out, int64_t table_out_stride,
                       void* lengths_out, cudaStream_t stream) {
  const int rc = check_table(p);
  if (rc != RBLN_OK) return rc;
  if (forks < 0 || !index_type(parents_dtype)) return RBLN_ERR_INVALID_ARGUMENT;
  if (forks == 0) return RBLN_OK;
  if (!parents || !lengths_out || (p->max_blocks > 0 && !table_out)) return RBLN_ERR_INVALID_ARGUMENT;
  const int64_t rows = (int64_t)p->batch + forks, parts = std::max(1, (p->max_blocks + 255) / 256);
  if (rows > INT32_MAX || parts > 65535) return RBLN_ERR_UNSUPPORTED;
  ForkArgs a{};
  a.t = table_of(p);
  a.len = lengths_of(p);
  a.parents = parents;
  a.parents_dtype = parents_dtype;
  a.parents_stride = parents_stride;
  a.forks = forks;
  a.span = span_of(p);
  a.out = table_out;
  a.os_row = table_out_stride;
  a.len_out = lengths_out;
  paged_kv_fork_kernel<<<dim3((unsigned)rows, (unsigned)parts), 256, 0, stream>>>(a);
  return launched();
}

int rbln_paged_kv_free(const rbln_pages_params_t* p, cudaStream_t stream) {
  const int rc = check_table(p);
  if (rc != RBLN_OK) return rc;
  if (p->batch == 0 || p->max_blocks == 0) return RBLN_OK;
  const int parts = (p->max_blocks + 255) / 256;
  if (parts > 65535) return RBLN_ERR_UNSUPPORTED;
  paged_kv_free_kernel<<<dim3((p->batch + kFreeRows - 1) / kFreeRows, parts), 256, 0, stream>>>(
      table_of(p), lengths_of(p), span_of(p));
  return launched();
}

int rbln_paged_kv_pages_workspace_size(const rbln_pages_params_t* p, int32_t new_tokens, size_t* bytes) {
  if (!p || !bytes || p->batch < 0 || p->num_blocks < 0 || p->max_blocks < 0 || p->block_size <= 0)
    return RBLN_ERR_INVALID_ARGUMENT;
  const int64_t entries = new_tokens < 0 ? -1 : p->batch * slots_of(p, new_tokens);
  if (entries > INT32_MAX) return RBLN_ERR_UNSUPPORTED;
  *bytes = workspace_of(p, entries).total;
  return RBLN_OK;
}

int rbln_paged_kv_reserve(const rbln_pages_params_t* p, int32_t new_tokens, int32_t* granted, cudaStream_t stream) {
  int rc = check_table(p);
  if (rc == RBLN_OK) rc = check_caches(p);
  if (rc != RBLN_OK) return rc;
  if (new_tokens < 0 || (p->batch > 0 && !granted)) return RBLN_ERR_INVALID_ARGUMENT;
  if (p->batch == 0) return RBLN_OK;
  const int64_t slots = slots_of(p, new_tokens), entries = p->batch * slots;
  if (entries > INT32_MAX) return RBLN_ERR_UNSUPPORTED;
  const Workspace w = workspace_of(p, entries);
  if (!p->workspace || p->workspace_bytes < w.total) return RBLN_ERR_WORKSPACE;
  char* ws = workspace_base(p);
  ReserveArgs a{};
  a.t = table_of(p);
  a.seq = lengths_of(p);
  a.span = span_of(p);
  a.fresh_tokens = new_tokens;
  a.slots = (int)std::max<int64_t>(slots, 1);
  a.t.rows = p->batch;
  a.granted = granted;
  a.ctas = reinterpret_cast<int*>(ws + w.ctas);
  a.count = a.ctas + 4 * kPlanCtas;
  a.here = reinterpret_cast<int*>(ws + w.here);
  a.last = reinterpret_cast<int*>(ws + w.last);
  a.given = reinterpret_cast<int*>(ws + w.given);
  a.take = reinterpret_cast<int*>(ws + w.take);
  a.moves = reinterpret_cast<Move*>(ws + w.moves);
  a.entries = entries;
  if (entries <= kSmallEntries && p->num_blocks <= kSmallPages) {
    paged_kv_reserve_small_kernel<<<1, kPlanThreads, 0, stream>>>(a);
    rc = launched();
  } else {
    rc = launch_plan(paged_kv_reserve_kernel, kPlanCtas, stream, a);
  }
  if (rc != RBLN_OK || entries == 0) return rc;
  return launch_copies(p, a.moves, a.count, p->batch, nullptr, stream);
}

int rbln_paged_kv_compact(const rbln_pages_params_t* p, int32_t* moved, int32_t* live, cudaStream_t stream) {
  int rc = check_table(p, false);
  if (rc == RBLN_OK) rc = check_caches(p);
  if (rc != RBLN_OK) return rc;
  if (!live || (p->num_blocks > 0 && !moved)) return RBLN_ERR_INVALID_ARGUMENT;
  const Workspace w = workspace_of(p, -1);
  if (!p->workspace || p->workspace_bytes < w.total) return RBLN_ERR_WORKSPACE;
  char* ws = workspace_base(p);
  CompactArgs a{};
  a.refs = p->refs;
  a.num_blocks = p->num_blocks;
  a.bs = p->block_size;
  a.moved = moved;
  a.live = live;
  a.ctas = reinterpret_cast<int*>(ws + w.ctas);
  a.count = a.ctas + 4 * kPlanCtas;
  a.src = reinterpret_cast<int*>(ws + w.here);
  a.dst = reinterpret_cast<int*>(ws + w.last);
  a.moves = reinterpret_cast<Move*>(ws + w.moves);
  // one CTA where a thread has few pages, else a cluster of eight
  rc = launch_plan(paged_kv_compact_kernel, p->num_blocks <= 4 * kPlanThreads ? 1 : kPlanCtas, stream, a);
  if (rc != RBLN_OK || p->num_blocks == 0) return rc;
  return launch_copies(p, a.moves, a.count, p->num_blocks / 2, moved, stream);
}

}  // extern "C"

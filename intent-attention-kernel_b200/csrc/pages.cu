// Page operations of a paged cache: grow (allocate, copy-on-write), shrink, fork, free, compact.
//
// A page is free when no table entry holds it (refs 0), so freeing only counts down and needs no order, and the pages
// to hand out are the lowest free ones: the k-th free page goes to the k-th page wanted, whatever order blocks run in.
// Finding them reads refs once, 4 bytes a page; one cluster of 8 blocks does it, each with an eighth of the pages,
// the eighths' counts exchanged through distributed shared memory.  What follows (page copies, table entries) is a
// second kernel over all SMs; copies move 2 * page bytes at 16 bytes a lane, which bounds a compaction.  Small calls
// are bound by their launches.
// 98304 of 262144 pages of 8 KB moved: 17 us to plan, 255 us to copy (6.3 TB/s).
#include <cooperative_groups.h>

#include <algorithm>

#include "iak_internal.cuh"

namespace cg = cooperative_groups;

namespace iak {
namespace {

constexpr int kCluster = 8;
constexpr int kPlanThreads = 1024;
constexpr int kActThreads = 256;
constexpr int kListThreads = 512;
// Of a page that a warp copies.  (One page of 4.4 MB copied: 18 us, by a single warp 273.)
constexpr int64_t kPiece = 16384;

struct Seq {
  int32_t* refs; int num_pages;
  int32_t* table; int64_t sb, sh; int W;
  int32_t* lengths;
  int S, Ht, PS;
};
struct Planes {
  char* base[IAK_MAX_PLANES]; int64_t bytes[IAK_MAX_PLANES]; uint32_t formats[IAK_MAX_PLANES];
  int num, pieces;    // pieces: of the largest plane's pages
  void* tags; int tag_bytes; uint8_t tag_map[16]; uint8_t tag_default;
};

__device__ __forceinline__ int pages_of(int tokens, int PS) {
  return tokens <= 0 ? 0 : (tokens - 1) / PS + 1;      // no sum that could pass 2^31
}
// pages a slot holds: never more than its table has entries
__device__ __forceinline__ int held_pages(const Seq& q, int s) { return min(pages_of(q.lengths[s], q.PS), q.W); }
__device__ __forceinline__ bool in_pool(const Seq& q, int id) { return id >= 0 && id < q.num_pages; }

// sum over the block's threads before this one; *all = the block's sum
__device__ __forceinline__ int block_before(int v, int* all) {
  __shared__ int warp_sum[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();                                     // an earlier call's readers are done
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int x = lane < warps ? warp_sum[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, x, o);
      if (lane >= o) x += y;
    }
    if (lane < warps) warp_sum[lane] = x;
  }
  __syncthreads();
  *all = warp_sum[warps - 1];
  return inc - v + (warp ? warp_sum[warp - 1] : 0);
}

// copy piece `piece` of page `from` to page `to` by one warp: kPiece bytes of each plane of the page's format, and with
// the first the tag
__device__ __forceinline__ void copy_piece(const Planes& pl, int64_t from, int64_t to, int piece) {
  const int lane = threadIdx.x & 31;
  uint32_t mask = ~0u;
  if (pl.tags) {
    const int tag = pl.tag_bytes == 1 ? static_cast<int>(static_cast<const uint8_t*>(pl.tags)[from])
                                      : static_cast<const int32_t*>(pl.tags)[from];
    mask = 1u << ((tag >= 0 && tag < 16) ? pl.tag_map[tag] : pl.tag_default);
    __syncwarp();
    if (lane == 0 && piece == 0) {
      if (pl.tag_bytes == 1) static_cast<uint8_t*>(pl.tags)[to] = static_cast<uint8_t>(tag);
      else static_cast<int32_t*>(pl.tags)[to] = tag;
    }
  }
  for (int i = 0; i < pl.num; ++i) {
    if (pl.tags && !(pl.formats[i] & mask)) continue;
    const int64_t skip = piece * kPiece, n = min(pl.bytes[i] - skip, kPiece);
    if (n <= 0) continue;
    const char* src = pl.base[i] + from * pl.bytes[i] + skip;
    char* dst = pl.base[i] + to * pl.bytes[i] + skip;
    const uintptr_t low = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | static_cast<uintptr_t>(n);
    if ((low & 15) == 0) {
      const uint4* s = reinterpret_cast<const uint4*>(src);
      uint4* d = reinterpret_cast<uint4*>(dst);
      const int64_t m = n / 16;
      int64_t at = lane;
      for (; at + 7 * 32 < m; at += 8 * 32) {
        uint4 r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = __ldcs(s + at + j * 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) __stcs(d + at + j * 32, r[j]);
      }
      for (; at < m; at += 32) d[at] = s[at];
    } else if ((low & 3) == 0) {
      for (int64_t at = lane; at < n / 4; at += 32)
        reinterpret_cast<uint32_t*>(dst)[at] = reinterpret_cast<const uint32_t*>(src)[at];
    } else {
      for (int64_t at = lane; at < n; at += 32) dst[at] = src[at];
    }
  }
}

// The pages that block `rank` of the cluster scans: an eighth of them in whole runs of 32.  A thread takes 32 at a time,
// the block kRun.
constexpr int kRun = 32 * kPlanThreads;
__device__ __forceinline__ void slice_of(int pages, int rank, int* begin, int* end) {
  const int64_t per = ((static_cast<int64_t>(pages) + kCluster * 32 - 1) / (kCluster * 32)) * 32;
  *begin = static_cast<int>(min(static_cast<int64_t>(pages), per * rank));
  *end = static_cast<int>(min(static_cast<int64_t>(pages), per * (rank + 1)));
}

// bit i: page p + i is in use (p + i < end)
__device__ __forceinline__ unsigned live_mask(const int32_t* refs, int p, int end) {
  unsigned m = 0;
  if (p >= end) return 0;
  if (end - p >= 32 && (reinterpret_cast<uintptr_t>(refs + p) & 15) == 0) {
    int4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = reinterpret_cast<const int4*>(refs + p)[k];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      m |= ((v[k].x > 0 ? 1u : 0u) | (v[k].y > 0 ? 2u : 0u) | (v[k].z > 0 ? 4u : 0u) | (v[k].w > 0 ? 8u : 0u)) << (4 * k);
  } else {
    for (int k = 0; k < min(32, end - p); ++k) m |= (refs[p + k] > 0 ? 1u : 0u) << k;
  }
  return m;
}
// the low bits of a 32-page run at p that stand for pages below n
__device__ __forceinline__ unsigned below_mask(int p, int n) {
  return n <= p ? 0u : (n - p >= 32 ? ~0u : (1u << (n - p)) - 1u);
}

// A thread's 32 pages of the run at p0; those of the first run (all of them, up to 2^18 pages) stay in a register.
struct Masks {
  const int32_t* refs;
  int begin, end;
  unsigned first;
  __device__ __forceinline__ Masks(const int32_t* r, int b, int e) : refs(r), begin(b), end(e) {
    first = live_mask(refs, begin + 32 * static_cast<int>(threadIdx.x), end);
  }
  __device__ __forceinline__ unsigned at(int p0) const {
    return p0 == begin ? first : live_mask(refs, p0 + 32 * static_cast<int>(threadIdx.x), end);
  }
  // the block's pages in use below n
  __device__ __forceinline__ int count(int n) const {
    int live = 0, all;
    for (int p0 = begin; p0 < min(end, n); p0 += kRun)
      live += __popc(at(p0) & below_mask(p0 + 32 * static_cast<int>(threadIdx.x), n));
    block_before(live, &all);
    return all;
  }
};

// ------------------------------------------------------------------------ grow
// Scratch: first[S * Ht] = rank of the (slot, head)'s first new page, < 0 = gets none; open[S * Ht] = the page to copy,
// < 0 = none; bad[S] (an open page lies outside the pool); old_pages[S], fresh[S]; new_ids[rank].
struct GrowScratch { int32_t* first; int32_t* open; int32_t* bad; int32_t* old_pages; int32_t* fresh; int32_t* new_ids; };

// Each block of the cluster plans an eighth of the slots, too.  (All in one block, every (slot, head) reading all of the
// slot's open pages: 466 us for 256 slots of 128 heads, now 57.)
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kPlanThreads)
grow_plan_kernel(const Seq q, const int32_t* more, int32_t* rejected, const GrowScratch w) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  __shared__ int live_here, cut_here;                  // cut: first slot that the free pages do not reach
  __shared__ long long wanted_here;                    // pages that the block's slots want
  const int per_block = (q.S + kCluster - 1) / kCluster;
  const int s_begin = min(q.S, per_block * rank), s_end = min(q.S, s_begin + per_block);
  const int i_begin = s_begin * q.Ht, i_end = s_end * q.Ht;        // (the host keeps S * Ht within 31 bits)
  // the slot's tokens, those to come, and whether they fit its table
  auto read_slot = [&](int s, int* len, int* add) {
    *len = max(q.lengths[s], 0);
    *add = more[s];
    const int64_t total = static_cast<int64_t>(*len) + *add;
    return *add > 0 && total <= static_cast<int64_t>(q.W) * q.PS && total <= 0x7fffffff;
  };
  if (threadIdx.x == 0) cut_here = q.S;
  for (int s = s_begin + threadIdx.x; s < s_end; s += kPlanThreads) w.bad[s] = 0;
  __syncthreads();
  // open pages; one outside the pool refuses its slot, for all heads
  for (int i = i_begin + threadIdx.x; i < i_end; i += kPlanThreads) {
    const int s = i / q.Ht, h = i - s * q.Ht;
    int len, add, open = -1;
    if (read_slot(s, &len, &add) && len % q.PS != 0) {
      const int id = q.table[s * q.sb + h * q.sh + pages_of(len, q.PS) - 1];
      if (!in_pool(q, id)) w.bad[s] = 1;
      else if (q.refs[id] > 1) open = id;
    }
    w.open[i] = open;
  }
  __syncthreads();
  // ranks of the pages wanted, in order of (slot, head), from the block's first on
  int refused = 0;
  int64_t base = 0;
  for (int i0 = i_begin; i0 < i_end; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    bool ok = false;
    if (i < i_end) {
      const int s = i / q.Ht, h = i - s * q.Ht;
      int len, add;
      ok = read_slot(s, &len, &add) && !w.bad[s];
      const int old = ok ? pages_of(len, q.PS) : 0, fresh = ok ? pages_of(len + add, q.PS) - old : 0;
      need = fresh + (ok && w.open[i] >= 0 ? 1 : 0);
      if (h == 0) {
        w.old_pages[s] = old;
        w.fresh[s] = fresh;
        if (add != 0 && !ok) ++refused;
      }
    }
    int all;
    const int before = block_before(need, &all);       // (the host keeps 1024 rows' pages within 31 bits)
    if (i < i_end) w.first[i] = ok ? static_cast<int32_t>(min(base + before, static_cast<int64_t>(0x7fffffff))) : -1;
    base += all;
  }
  int begin, end;
  slice_of(q.num_pages, rank, &begin, &end);
  const Masks masks(q.refs, begin, end);
  const int live = masks.count(end);
  if (threadIdx.x == 0) {
    live_here = live;
    wanted_here = base;
  }
  cluster.sync();
  int free_before = 0, free_all = 0;                   // free pages below this slice, in all
  int64_t wanted_before = 0, wanted_all = 0;
  for (int r = 0; r < kCluster; ++r) {
    int bb, be;
    slice_of(q.num_pages, r, &bb, &be);
    const int f = be - bb - *cluster.map_shared_rank(&live_here, r);
    const int64_t n = *cluster.map_shared_rank(&wanted_here, r);
    if (r < rank) {
      free_before += f;
      wanted_before += n;
    }
    free_all += f;
    wanted_all += n;
  }
  // a slot that does not fit, and every later one that gets tokens, stays as it is
  for (int i = i_begin + threadIdx.x; i < i_end; i += kPlanThreads) {
    if (w.first[i] < 0) continue;
    const int s = i / q.Ht;
    const int64_t first = wanted_before + w.first[i];
    w.first[i] = static_cast<int32_t>(min(first, static_cast<int64_t>(0x7fffffff)));
    if (first + w.fresh[s] + (w.open[i] >= 0 ? 1 : 0) > free_all) atomicMin(&cut_here, s);
  }
  // the free pages of this slice, in ascending order
  const int want = static_cast<int>(min(wanted_all, static_cast<int64_t>(free_all)));
  int at = free_before;
  for (int p0 = begin; p0 < end && at < want; p0 += kRun) {
    const int p = p0 + 32 * static_cast<int>(threadIdx.x);
    unsigned free_bits = ~masks.at(p0) & below_mask(p, end);
    int all;
    int k = at + block_before(__popc(free_bits), &all);
    for (; free_bits && k < want; free_bits &= free_bits - 1, ++k) w.new_ids[k] = p + __ffs(free_bits) - 1;
    at += all;
  }
  cluster.sync();
  int last = q.S;
  for (int r = 0; r < kCluster; ++r) last = min(last, *cluster.map_shared_rank(&cut_here, r));
  for (int i = i_begin + threadIdx.x; i < i_end; i += kPlanThreads) {
    if (w.first[i] < 0) continue;
    const int s = i / q.Ht;
    const bool slot = i - s * q.Ht == 0;
    if (s >= last) {
      w.first[i] = -1;
      if (slot) ++refused;
    } else if (slot) {
      q.lengths[s] = max(q.lengths[s], 0) + more[s];
    }
  }
  if (rejected && refused) atomicAdd(rejected, refused);
  cluster.sync();                                      // no block leaves while another may read its counts
}

__global__ void __launch_bounds__(kActThreads) grow_act_kernel(const Seq q, const Planes pl, const GrowScratch w) {
  const int warps = kActThreads / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t jobs = static_cast<int64_t>(q.S) * q.Ht * pl.pieces;
  for (int64_t job = blockIdx.x * warps + warp; job < jobs; job += gridDim.x * warps) {
    const int i = static_cast<int>(job / pl.pieces), piece = static_cast<int>(job - static_cast<int64_t>(i) * pl.pieces);
    const int first = w.first[i];
    if (first < 0) continue;
    const int s = i / q.Ht, h = i - s * q.Ht;
    int32_t* row = q.table + s * q.sb + h * q.sh;
    const int old = w.old_pages[s], fresh = w.fresh[s], from = w.open[i], copy = from >= 0 ? 1 : 0;
    if (copy) {
      const int to = w.new_ids[first];
      copy_piece(pl, from, to, piece);
      if (lane == 0 && piece == 0) {
        row[old - 1] = to;
        q.refs[to] = 1;
        atomicSub(&q.refs[from], 1);
      }
    }
    if (piece) continue;
    for (int k = lane; k < fresh; k += 32) {
      const int id = w.new_ids[first + copy + k];
      row[old + k] = id;
      q.refs[id] = 1;
    }
  }
}

// ------------------------------------------------------------------ fork, free
// A cluster per listed item: all its blocks read the slot's length before one of them writes it.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kListThreads)
fork_kernel(const Seq q, const int32_t* src, const int32_t* dst, int n, int32_t* rejected) {
  cg::cluster_group cluster = cg::this_cluster();
  const int i = blockIdx.x / kCluster, rank = static_cast<int>(cluster.block_rank());
  const int from = src[i], to = dst[i];
  bool bad = from < 0 || from >= q.S || to < 0 || to >= q.S;
  if (!bad) bad = q.lengths[to] > 0;
  for (int j = threadIdx.x; j < n; j += kListThreads) bad = bad || dst[j] == from || (j < i && dst[j] == to);
  bad = __syncthreads_or(bad);
  const int held = bad ? 0 : held_pages(q, from);
  const int len = bad ? 0 : q.lengths[from];
  cluster.sync();
  if (bad) {
    if (rejected && rank == 0 && threadIdx.x == 0) atomicAdd(rejected, 1);
    return;
  }
  const int64_t entries = static_cast<int64_t>(q.Ht) * held;
  for (int64_t e = rank * kListThreads + threadIdx.x; e < entries; e += kCluster * kListThreads) {
    const int h = static_cast<int>(e / held), w = static_cast<int>(e - static_cast<int64_t>(h) * held);
    const int id = q.table[from * q.sb + h * q.sh + w];
    q.table[to * q.sb + h * q.sh + w] = id;
    if (in_pool(q, id)) atomicAdd(&q.refs[id], 1);
  }
  if (rank == 0 && threadIdx.x == 0) q.lengths[to] = len;
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kListThreads)
free_kernel(const Seq q, const int32_t* slots, int n, int32_t* rejected) {
  cg::cluster_group cluster = cg::this_cluster();
  const int i = blockIdx.x / kCluster, rank = static_cast<int>(cluster.block_rank());
  const int s = slots[i];
  const bool bad = s < 0 || s >= q.S;
  bool again = false;
  for (int j = threadIdx.x; j < i; j += kListThreads) again = again || slots[j] == s;
  again = __syncthreads_or(again);
  const int held = bad || again ? 0 : held_pages(q, s);
  cluster.sync();
  if (bad) {
    if (rejected && rank == 0 && threadIdx.x == 0) atomicAdd(rejected, 1);
    return;
  }
  if (again) return;
  const int64_t entries = static_cast<int64_t>(q.Ht) * held;
  for (int64_t e = rank * kListThreads + threadIdx.x; e < entries; e += kCluster * kListThreads) {
    const int h = static_cast<int>(e / held), w = static_cast<int>(e - static_cast<int64_t>(h) * held);
    int32_t* at = q.table + s * q.sb + h * q.sh + w;
    const int id = *at;
    *at = -1;
    if (in_pool(q, id)) atomicSub(&q.refs[id], 1);
  }
  if (rank == 0 && threadIdx.x == 0) q.lengths[s] = 0;
}

// A block per slot: its threads read the length before one of them writes it.
__global__ void __launch_bounds__(kActThreads) shrink_kernel(const Seq q, const int32_t* tokens, int32_t* rejected) {
  const int s = blockIdx.x, off = tokens[s], len = max(q.lengths[s], 0);
  if (off == 0) return;
  __syncthreads();
  if (off < 0 || off > len) {
    if (rejected && threadIdx.x == 0) atomicAdd(rejected, 1);
    return;
  }
  const int from = min(pages_of(len - off, q.PS), q.W), n = min(pages_of(len, q.PS), q.W) - from;
  for (int64_t e = threadIdx.x; e < static_cast<int64_t>(q.Ht) * n; e += kActThreads) {
    const int h = static_cast<int>(e / n), w = from + static_cast<int>(e - static_cast<int64_t>(h) * n);
    int32_t* at = q.table + s * q.sb + h * q.sh + w;
    const int id = *at;
    *at = -1;
    if (in_pool(q, id)) atomicSub(&q.refs[id], 1);
  }
  if (threadIdx.x == 0) q.lengths[s] = len - off;
}

// --------------------------------------------------------------------- compact
// Scratch: head[0] = pages in use n, head[1] = pages to move; from[k] and to[k] of move k; rank_of[page] of the pages
// that move.
struct CompactScratch { int32_t* head; int32_t* from; int32_t* to; int32_t* rank_of; };

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kPlanThreads)
compact_plan_kernel(const Seq q, int32_t* num_live, const CompactScratch w) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  __shared__ int live_here, live_below_n;              // live pages of the slice; of the slice and below n
  int begin, end;
  slice_of(q.num_pages, rank, &begin, &end);
  const Masks masks(q.refs, begin, end);
  const int live = masks.count(end);
  if (threadIdx.x == 0) live_here = live;
  cluster.sync();
  int live_before = 0, n = 0;
  for (int r = 0; r < kCluster; ++r) {
    const int x = *cluster.map_shared_rank(&live_here, r);
    if (r < rank) live_before += x;
    n += x;
  }
  const int below = masks.count(n);
  if (threadIdx.x == 0) live_below_n = below;
  cluster.sync();
  int stay = 0;                                        // live pages below n: they keep their place
  for (int r = 0; r < kCluster; ++r) stay += *cluster.map_shared_rank(&live_below_n, r);
  if (rank == 0 && threadIdx.x == 0) {
    w.head[0] = n;
    w.head[1] = n - stay;
    if (num_live) *num_live = n;
  }
  int at = live_before;                                // live pages before the run
  for (int p0 = begin; p0 < end; p0 += kRun) {
    const int p = p0 + 32 * static_cast<int>(threadIdx.x);
    const unsigned live_bits = masks.at(p0), low = below_mask(p, n);
    int all;
    const int before = at + block_before(__popc(live_bits), &all);
    // The k-th free page below n takes the k-th live page from n on.  A lane's 32 pages are written by the warp, a page
    // per lane, so that neighbours in rank are neighbours in memory.
    const int lane = threadIdx.x & 31;
    const unsigned any = __ballot_sync(~0u, ((~live_bits & low) | (live_bits & ~low)) & below_mask(p, end));
    for (unsigned todo = any; todo; todo &= todo - 1) {
      const int l = __ffs(todo) - 1, page = __shfl_sync(~0u, p, l) + lane;
      const unsigned bits = __shfl_sync(~0u, live_bits, l);
      const int rank = __shfl_sync(~0u, before, l) + __popc(bits & ((1u << lane) - 1u));
      if (page >= end) continue;
      const bool is_live = bits >> lane & 1;
      if (page < n && !is_live) w.to[page - rank] = page;
      if (page >= n && is_live) {
        w.from[rank - stay] = page;
        w.rank_of[page] = rank - stay;
      }
    }
    at += all;
  }
  cluster.sync();
}

__global__ void __launch_bounds__(kActThreads) compact_act_kernel(const Seq q, const Planes pl, const CompactScratch w) {
  const int n = w.head[0], moves = w.head[1];
  if (moves == 0) return;
  const int warps = kActThreads / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t jobs = static_cast<int64_t>(moves) * pl.pieces;
  for (int64_t job = blockIdx.x * warps + warp; job < jobs; job += gridDim.x * warps) {
    const int k = static_cast<int>(job / pl.pieces), piece = static_cast<int>(job - static_cast<int64_t>(k) * pl.pieces);
    const int from = w.from[k], to = w.to[k];
    copy_piece(pl, from, to, piece);
    if (lane == 0 && piece == 0) {
      q.refs[to] = q.refs[from];
      q.refs[from] = 0;
    }
  }
  // table entries of moved pages; rank_of holds anything for other pages, so the move has to agree
  const int rows = q.S * q.Ht;
  for (int r = blockIdx.x * warps + warp; r < rows; r += gridDim.x * warps) {
    const int s = r / q.Ht, h = r - s * q.Ht;
    int32_t* row = q.table + s * q.sb + h * q.sh;
    const int held = held_pages(q, s);
    for (int e = lane; e < held; e += 32) {
      const int id = row[e];
      if (!in_pool(q, id) || id < n) continue;
      const int k = w.rank_of[id];
      if (k >= 0 && k < moves && w.from[k] == id) row[e] = w.to[k];
    }
  }
}

// ------------------------------------------------------------------------ host
int check_seq(const iak_seq_pages* a, const char* what, Seq* q) {
  if (!a) return fail(IAK_ERR_INVALID_ARG, "%s: null arguments", what);
  if (a->num_pages < 0 || a->num_pages > 0x7fff0000LL || a->num_slots < 0 || a->num_table_heads < 0 || a->table_width < 0)
    return fail(IAK_ERR_INVALID_ARG, "%s: bad size", what);
  if (static_cast<int64_t>(a->num_slots) * a->num_table_heads > 0x7fff0000LL)
    return fail(IAK_ERR_UNSUPPORTED, "%s: more than 2^31 (slot, head) pairs", what);
  if (a->page_size <= 0) return fail(IAK_ERR_INVALID_ARG, "%s: page_size must be positive", what);
  const bool entries = a->num_slots > 0 && a->num_table_heads > 0 && a->table_width > 0;
  if ((a->num_slots > 0 && !a->lengths) || (a->num_pages > 0 && !a->refs) || (entries && !a->page_table))
    return fail(IAK_ERR_INVALID_ARG, "%s: null refs, page_table or lengths", what);
  *q = {a->refs, static_cast<int>(a->num_pages), a->page_table, a->pt_stride_s, a->pt_stride_h, a->table_width,
        a->lengths, a->num_slots, a->num_table_heads, a->page_size};
  return IAK_OK;
}

int check_planes(const iak_page_planes* a, const char* what, Planes* p) {
  *p = {};
  if (!a) return fail(IAK_ERR_INVALID_ARG, "%s: null planes", what);
  if (a->num_planes < 0 || a->num_planes > IAK_MAX_PLANES) return fail(IAK_ERR_INVALID_ARG, "%s: bad num_planes", what);
  for (int i = 0; i < a->num_planes; ++i) {
    if (!a->base[i] || a->bytes[i] <= 0) return fail(IAK_ERR_INVALID_ARG, "%s: empty plane %d", what, i);
    p->base[i] = static_cast<char*>(a->base[i]);
    p->bytes[i] = a->bytes[i];
    p->formats[i] = a->formats[i];
    const int64_t pieces = (a->bytes[i] + kPiece - 1) / kPiece;
    if (pieces > 0x7fffffffLL) return fail(IAK_ERR_UNSUPPORTED, "%s: pages too large", what);
    p->pieces = std::max(p->pieces, static_cast<int>(pieces));
  }
  p->num = a->num_planes;
  p->pieces = std::max(p->pieces, 1);                  // (tables and counts follow without planes too)
  p->tags = a->page_tags;
  if (a->page_tags && a->tag_bytes != 1 && a->tag_bytes != 4)
    return fail(IAK_ERR_INVALID_ARG, "%s: tag_bytes must be 1 or 4", what);
  p->tag_bytes = a->tag_bytes;
  for (int i = 0; i < 16; ++i) {
    if (a->page_tags && a->tag_map[i] >= 32) return fail(IAK_ERR_INVALID_ARG, "%s: bad tag_map", what);
    p->tag_map[i] = a->tag_map[i];
  }
  if (a->page_tags && a->tag_default >= 32) return fail(IAK_ERR_INVALID_ARG, "%s: bad tag_default", what);
  p->tag_default = a->tag_default;
  return IAK_OK;
}

// int32 words of scratch: the larger of what grow and compact use
size_t scratch_words(const iak_seq_pages* a) {
  const size_t rows = static_cast<size_t>(a->num_slots) * a->num_table_heads;
  const size_t grow = 2 * rows + 3 * static_cast<size_t>(a->num_slots) + static_cast<size_t>(a->num_pages);
  const size_t compact = 2 + 3 * static_cast<size_t>(a->num_pages);
  return std::max(grow, compact);
}

int check_ws(const iak_seq_pages* a, void* ws, size_t bytes, const char* what) {
  const size_t need = scratch_words(a) * 4;
  if (bytes < need || !ws) return fail(IAK_ERR_WORKSPACE, "%s needs %zu workspace bytes, got %zu", what, need, bytes);
  if (reinterpret_cast<uintptr_t>(ws) % 4) return fail(IAK_ERR_INVALID_ARG, "%s: workspace not aligned", what);
  return IAK_OK;
}

int launch_list_ok(int32_t count, const char* what) {
  if (count < 0) return fail(IAK_ERR_INVALID_ARG, "%s: negative count", what);
  if (count > 0x7fffffff / kCluster) return fail(IAK_ERR_UNSUPPORTED, "%s: too many slots", what);
  return IAK_OK;
}

}  // namespace
}  // namespace iak

using namespace iak;

extern "C" int iak_pages_workspace_size(const iak_seq_pages* pages, size_t* bytes) {
  Seq q;
  if (!bytes) return fail(IAK_ERR_INVALID_ARG, "iak_pages_workspace_size: null arguments");
  *bytes = 0;
  if (int st = check_seq(pages, "iak_pages_workspace_size", &q)) return st;
  *bytes = scratch_words(pages) * 4;
  return IAK_OK;
}

extern "C" int iak_pages_grow(const iak_seq_pages* pages, const iak_page_planes* planes, const int32_t* new_tokens,
                              int32_t* rejected, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "iak_pages_grow";
  Seq q;
  Planes pl;
  if (int st = check_seq(pages, what, &q)) return st;
  if (int st = check_planes(planes, what, &pl)) return st;
  if (q.S == 0 || q.Ht == 0) return IAK_OK;
  if (!new_tokens) return fail(IAK_ERR_INVALID_ARG, "%s: null new_tokens", what);
  if (int st = check_ws(pages, workspace, workspace_bytes, what)) return st;
  const int64_t rows = static_cast<int64_t>(q.S) * q.Ht;
  if (std::min<int64_t>(rows, kPlanThreads) * (static_cast<int64_t>(q.W) + 1) > 0x7fffffffLL)
    return fail(IAK_ERR_UNSUPPORTED, "%s: tables of %d pages a row", what, q.W);
  GrowScratch w;
  w.first = static_cast<int32_t*>(workspace);
  w.open = w.first + rows;
  w.bad = w.open + rows;
  w.old_pages = w.bad + q.S;
  w.fresh = w.old_pages + q.S;
  w.new_ids = w.fresh + q.S;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  grow_plan_kernel<<<kCluster, kPlanThreads, 0, s>>>(q, new_tokens, rejected, w);
  if (int st = check_cuda(cudaGetLastError(), "grow plan launch")) return st;
  const int64_t blocks = std::min<int64_t>((rows * pl.pieces + kActThreads / 32 - 1) / (kActThreads / 32), 8 * device_sm_count());
  grow_act_kernel<<<static_cast<unsigned>(blocks), kActThreads, 0, s>>>(q, pl, w);
  return check_cuda(cudaGetLastError(), "grow launch");
}

extern "C" int iak_pages_fork(const iak_seq_pages* pages, const int32_t* src, const int32_t* dst, int32_t count,
                              int32_t* rejected, void* stream) {
  const char* what = "iak_pages_fork";
  Seq q;
  if (int st = check_seq(pages, what, &q)) return st;
  if (int st = launch_list_ok(count, what)) return st;
  if (count == 0) return IAK_OK;
  if (!src || !dst) return fail(IAK_ERR_INVALID_ARG, "%s: null src or dst", what);
  fork_kernel<<<count * kCluster, kListThreads, 0, static_cast<cudaStream_t>(stream)>>>(q, src, dst, count, rejected);
  return check_cuda(cudaGetLastError(), "fork launch");
}

extern "C" int iak_pages_free(const iak_seq_pages* pages, const int32_t* slots, int32_t count, int32_t* rejected,
                              void* stream) {
  const char* what = "iak_pages_free";
  Seq q;
  if (int st = check_seq(pages, what, &q)) return st;
  if (int st = launch_list_ok(count, what)) return st;
  if (count == 0) return IAK_OK;
  if (!slots) return fail(IAK_ERR_INVALID_ARG, "%s: null slots", what);
  free_kernel<<<count * kCluster, kListThreads, 0, static_cast<cudaStream_t>(stream)>>>(q, slots, count, rejected);
  return check_cuda(cudaGetLastError(), "free launch");
}

extern "C" int iak_pages_shrink(const iak_seq_pages* pages, const int32_t* tokens, int32_t* rejected, void* stream) {
  const char* what = "iak_pages_shrink";
  Seq q;
  if (int st = check_seq(pages, what, &q)) return st;
  if (q.S == 0) return IAK_OK;
  if (!tokens) return fail(IAK_ERR_INVALID_ARG, "%s: null tokens", what);
  shrink_kernel<<<q.S, kActThreads, 0, static_cast<cudaStream_t>(stream)>>>(q, tokens, rejected);
  return check_cuda(cudaGetLastError(), "shrink launch");
}

extern "C" int iak_pages_compact(const iak_seq_pages* pages, const iak_page_planes* planes, int32_t* num_live,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "iak_pages_compact";
  Seq q;
  Planes pl;
  if (int st = check_seq(pages, what, &q)) return st;
  if (int st = check_planes(planes, what, &pl)) return st;
  if (int st = check_ws(pages, workspace, workspace_bytes, what)) return st;
  CompactScratch w;
  w.head = static_cast<int32_t*>(workspace);
  w.from = w.head + 2;
  w.to = w.from + q.num_pages;
  w.rank_of = w.to + q.num_pages;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  compact_plan_kernel<<<kCluster, kPlanThreads, 0, s>>>(q, num_live, w);
  if (int st = check_cuda(cudaGetLastError(), "compact plan launch")) return st;
  compact_act_kernel<<<8 * device_sm_count(), kActThreads, 0, s>>>(q, pl, w);
  return check_cuda(cudaGetLastError(), "compact launch");
}

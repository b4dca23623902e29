// Pages of a cache: copy, extend, fork, free, compact (dfcclPages* in ofccl.h).
//
// A cache is `npools` pools (keys and values of every layer, say) of the same number of pages that share one
// numbering, and its bookkeeping in three arrays of 32-bit integers on the GPU: a reference count per page (0 = free),
// a table row of page numbers per sequence, a length per sequence. Nothing else is kept, so there is no list of free
// pages to go stale: whoever needs pages takes the lowest free ones, found by a scan of the counts.
//
// The contents are moved by the same code in copy, fork and compact, bound by HBM (each byte read once and written
// once); the bookkeeping is a few integers per request, bound by the latency of its launches and scans.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/ofccl.h"
#include "indexed_common.h"

namespace dfccl {

constexpr int kMoveThreads = 256;
constexpr int kMoveWaves = kMoveThreads / 64;
constexpr int kMaxPools = 64;  // per launch; more pools take several
#ifndef DFCCL_SCAN_THREADS
#define DFCCL_SCAN_THREADS 1024
#endif
constexpr int kScanThreads = DFCCL_SCAN_THREADS;
constexpr int kScanWaves = kScanThreads / 64;
constexpr int kScanPer = 4;  // counts a thread reads at once
constexpr int kScanTile = kScanThreads * kScanPer;
// Up to so many tiles one workgroup scans all pages (5 us for 2048, 6 for 8192); above, a workgroup per tile counts and
// another launch lists (7 + 5 us for 262144 pages, where one workgroup took 54).
constexpr int kOneScan = 4;
constexpr int kFewRequests = 64;  // of an extend, carried out by the workgroup that scans: four for each of its waves, one
                                  // launch less (15 us for a turn of 16 sequences instead of 19)
// A workgroup per request, up to so many workgroups (a launch may not have 2^32 threads); more requests are walked. (A
// host build sets a lower limit, to get there with few requests.)
#ifndef DFCCL_REQUEST_GRID
#define DFCCL_REQUEST_GRID (1 << 20)
#endif
constexpr uint32_t kMaxRequestGrid = DFCCL_REQUEST_GRID;
// Counter of a walk over a list, the sequences or a table row: its last step goes beyond the last of up to 2^31 - 1 entries.
using ListIndex = uint32_t;

// The bookkeeping as the kernels see it.
struct Books {
  int32_t* refcounts;
  int32_t* tables;
  int32_t* lengths;
  int32_t* report;  // may be null
  int32_t pages, pageTokens, seqs, perSeq;
};
// Workspace: what one launch of a call hands to the next.
struct PageScratch {
  int32_t* owner;    // [seqs] first request that names the sequence
  int32_t* request;  // [seqs] per request: number of its first new page among those found, or -1 if it is refused
  int32_t* before;   // [seqs] per request: the sequence's (fork: the parent's) length before the call
  int32_t* found;    // [pages] the lowest free pages (compact: the holes to fill), in order
  int32_t* movers;   // [pages] compact: the pages that move, in order
  int32_t* rank;     // [pages] compact: place among the movers
  int32_t* tiles;    // [tiles of pages] free (compact: live) pages of each
  int32_t* counts;   // {pages found, pages that move, pages needed}
};

__device__ __forceinline__ int32_t pagesOf(int32_t tokens, int32_t pageTokens) {
  return tokens / pageTokens + (tokens % pageTokens != 0);
}

// ---- scan over the workgroup: exclusive prefix sum of v, and the total
struct ScanShared {
  int32_t wave[2][kScanWaves];
};
__device__ __forceinline__ int32_t blockScan(ScanShared& sh, int which, int32_t v, int32_t& total) {
  const int lane = (int)(threadIdx.x & 63), wave = waveInBlock();
  int32_t sum = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t from = __shfl(sum, (lane - d) & 63);
    if (lane >= d) sum += from;
  }
  if (lane == 63) sh.wave[which][wave] = sum;
  __syncthreads();
  int32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kScanWaves; w++) {
    const int32_t c = sh.wave[which][w];
    if (w < wave) before += c;
    total += c;
  }
  return before + sum - v;
}

// The numbers of a tile's pages that a thread looks at: kScanPer in a row.
__device__ __forceinline__ void loadCounts(const Books& b, int64_t first, int32_t (&c)[kScanPer]) {
#pragma unroll
  for (int i = 0; i < kScanPer; i++) c[i] = first + i < b.pages ? b.refcounts[first + i] : 1;
}

// One tile's free pages, in order, into found from place `have` on (as far as `most`); returns the tile's number.
__device__ __forceinline__ int32_t listFree(ScanShared& sh, int which, const Books& b, int64_t tileAt, int64_t have, int64_t most,
                                            int32_t* found) {
  const int64_t first = tileAt + (int64_t)threadIdx.x * kScanPer;
  int32_t c[kScanPer], mine = 0, total;
  loadCounts(b, first, c);
#pragma unroll
  for (int i = 0; i < kScanPer; i++) mine += c[i] == 0;
  int64_t to = have + blockScan(sh, which, mine, total);
#pragma unroll
  for (int i = 0; i < kScanPer; i++)
    if (c[i] == 0) {
      if (to < most) found[to] = (int32_t)(first + i);
      to++;
    }
  return total;
}

// ---- requests: which are valid, and which of the new pages each gets
struct Requests {
  const int32_t* a;  // extend: sequences; fork: parents
  const int32_t* b;  // extend: lengths;   fork: children
  int32_t n;
};
// extend: need = pages of the new length - pages of the old; fork: one page if the parent's last page is not full.
// One workgroup; returns the pages that all of them need.
template <bool FORK>
__device__ __forceinline__ int32_t readRequests(ScanShared& sh, const Books& b, const PageScratch& s, const Requests& q) {
  const ListIndex tid = threadIdx.x, n = (ListIndex)q.n;
  const int64_t most = (int64_t)b.perSeq * b.pageTokens;
  // the first request that names a sequence (a fork: a child) has it; the others are refused
  for (ListIndex i = tid; i < n; i += kScanThreads) {
    const int32_t seq = FORK ? q.b[i] : q.a[i];
    if (seq >= 0 && seq < b.seqs) s.owner[seq] = 0x7fffffff;
  }
  __syncthreads();
  for (ListIndex i = tid; i < n; i += kScanThreads) {
    const int32_t seq = FORK ? q.b[i] : q.a[i];
    if (seq >= 0 && seq < b.seqs)
      __hip_atomic_fetch_min(&s.owner[seq], (int32_t)i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  int32_t needed = 0;  // (at most seqs * perSeq, which the host keeps below 2^31)
  int which = 0;
  for (ListIndex at = 0; at < n; at += kScanThreads, which ^= 1) {
    const ListIndex i = at + tid;
    int32_t need = -1, before = 0;
    if (i < n) {
      const int32_t x = q.a[i], y = q.b[i];
      const int32_t seq = FORK ? y : x;
      if (seq >= 0 && seq < b.seqs && x >= 0 && x < b.seqs &&
          __hip_atomic_load(&s.owner[seq], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)i) {
        before = b.lengths[x];
        const bool sound = before >= 0 && before <= most;
        if constexpr (FORK) {
          if (sound && b.lengths[y] == 0) need = before % b.pageTokens != 0;
        } else {
          if (sound && y >= before && y <= most) need = pagesOf(y, b.pageTokens) - pagesOf(before, b.pageTokens);
        }
      }
      s.before[i] = before;
    }
    int32_t total;
    const int32_t first = blockScan(sh, which, need > 0 ? need : 0, total);
    if (i < n) s.request[i] = need < 0 ? -1 : needed + first;
    needed += total;
  }
  __syncthreads();
  if (tid == 0 && b.report != nullptr) b.report[0] = 0;  // the launch that carries the requests out counts the refusals
  return needed;
}

__device__ __forceinline__ void refuse(const Books& b) {
  if (b.report != nullptr) __hip_atomic_fetch_add(&b.report[0], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// One request of an extend, by `threads` threads: the new entries, their counts, the length.
__device__ __forceinline__ void extendOne(const Books& b, const PageScratch& s, const Requests& q, ListIndex i, int32_t foundPages,
                                          uint32_t thread, uint32_t threads) {
  const int32_t first = s.request[i];
  int32_t have = 0, want = 0, seq = 0, length = 0;
  bool met = false;
  if (first >= 0) {
    seq = q.a[i];
    length = q.b[i];
    have = pagesOf(s.before[i], b.pageTokens);
    want = pagesOf(length, b.pageTokens);
    met = want == have || first + (want - have) <= foundPages;
  }
  if (!met) {
    if (thread == 0) refuse(b);
    return;
  }
  int32_t* row = b.tables + (size_t)seq * b.perSeq;
  for (ListIndex k = (ListIndex)have + thread; k < (ListIndex)want; k += threads) {
    const int32_t page = s.found[(ListIndex)first + (k - (ListIndex)have)];
    row[k] = page;
    b.refcounts[page] = 1;
  }
  if (thread == 0) b.lengths[seq] = length;
}
__global__ __launch_bounds__(kMoveThreads) void extendKernel(Books b, PageScratch s, Requests q) {
  for (ListIndex i = blockIdx.x; i < (ListIndex)q.n; i += gridDim.x)
    extendOne(b, s, q, i, s.counts[0], threadIdx.x, kMoveThreads);
}

// A few tiles of pages: requests and free pages in one launch, and an extend of a few sequences as a whole.
template <bool FORK>
__global__ __launch_bounds__(kScanThreads) void assignKernel(Books b, PageScratch s, Requests q, bool carryOut) {
  struct Shared {
    ScanShared scan;
  };
  DFCCL_WG_SHARED(Shared, sh);
  const int32_t needed = readRequests<FORK>(sh.scan, b, s, q);
  int64_t have = 0;
  int which = 0;
  for (int64_t at = 0; at < b.pages && have < needed; at += kScanTile, which ^= 1)
    have += listFree(sh.scan, which, b, at, have, needed, s.found);
  const int32_t foundPages = (int32_t)(have < needed ? have : needed);
  if (threadIdx.x == 0) s.counts[0] = foundPages;
  if constexpr (!FORK) {
    if (!carryOut) return;
    __syncthreads();
    for (ListIndex i = (ListIndex)waveInBlock(); i < (ListIndex)q.n; i += kScanWaves)
      extendOne(b, s, q, i, foundPages, threadIdx.x & 63, 64);
  }
}

// Many tiles, first launch: workgroup 0 reads the requests (a compaction has none), the others count a tile each.
enum : int { kForExtend = 0, kForFork = 1, kForCompact = 2 };
template <int FOR>
__global__ __launch_bounds__(kScanThreads) void countTilesKernel(Books b, PageScratch s, Requests q) {
  struct Shared {
    ScanShared scan;
  };
  DFCCL_WG_SHARED(Shared, sh);
  if (blockIdx.x == 0) {
    if constexpr (FOR != kForCompact) {
      const int32_t needed = readRequests<FOR == kForFork>(sh.scan, b, s, q);
      if (threadIdx.x == 0) s.counts[2] = needed;
    }
    return;
  }
  const int32_t tile = (int32_t)blockIdx.x - 1;
  const int64_t first = (int64_t)tile * kScanTile + (int64_t)threadIdx.x * kScanPer;
  int32_t c[kScanPer], mine = 0, total;
  loadCounts(b, first, c);
#pragma unroll
  for (int i = 0; i < kScanPer; i++)
    mine += FOR == kForCompact ? c[i] > 0 && first + i < b.pages : c[i] == 0;
  (void)blockScan(sh.scan, 0, mine, total);
  if (threadIdx.x == 0) s.tiles[tile] = total;
}
// The sum of the first n tiles' counts, by the workgroup.
__device__ __forceinline__ int32_t sumTiles(ScanShared& sh, int which, const int32_t* tiles, int32_t n) {
  int32_t mine = 0, total;
  for (uint32_t t = threadIdx.x; t < (uint32_t)n; t += kScanThreads) mine += tiles[t];
  (void)blockScan(sh, which, mine, total);
  return total;
}
// Second launch: a workgroup per tile lists the tile's free pages behind those of the tiles before.
__global__ __launch_bounds__(kScanThreads) void listFreeKernel(Books b, PageScratch s, int32_t tiles) {
  struct Shared {
    ScanShared scan;
  };
  DFCCL_WG_SHARED(Shared, sh);
  const int32_t tile = (int32_t)blockIdx.x, needed = s.counts[2];
  const int32_t have = sumTiles(sh.scan, 0, s.tiles, tile);
  if (tile + 1 == tiles && threadIdx.x == 0) {
    const int32_t all = have + s.tiles[tile];
    s.counts[0] = all < needed ? all : needed;
  }
  if (have < needed) (void)listFree(sh.scan, 1, b, (int64_t)tile * kScanTile, have, needed, s.found);
}

// ---- contents

struct PoolSet {
  char* to[kMaxPools];
  const char* from[kMaxPools];
  int32_t npools;
  uint32_t parts;      // per page
  uint32_t lastBytes;  // of a page's last part
  size_t pageBytes;
};
// What one wave moves at a time, in 16-byte loads a lane has in flight: the sweeps behind each figure in the kernels.
constexpr int kCopyLoads = 1, kForkLoads = 2, kCompactLoads = 4;
constexpr uint32_t partBytes(int loads) { return 64 * 16 * (uint32_t)loads; }

// one part of a page, by one wave; stores (and with NT loads, too) do not stay in the caches
template <int LOADS, bool NT>
__device__ __forceinline__ void movePart(const char* from, char* to, uint32_t bytes, uint32_t lane) {
  if (bytes == partBytes(LOADS)) {
    u32x4 v[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; u++) v[u] = load16<1, NT>(from + (u * 64 + lane) * 16);
#pragma unroll
    for (int u = 0; u < LOADS; u++) store16<1, true>(to + (u * 64 + lane) * 16, v[u]);
    return;
  }
  const uint32_t packs = bytes / 16;
  for (uint32_t p = lane; p < packs; p += 64) store16<1>(to + p * 16, load16<1>(from + p * 16));
  for (uint32_t i = packs * 16 + lane; i < bytes; i += 64)
    ((DFCCL_GLOBAL char*)to)[i] = ((const DFCCL_GLOBAL char*)from)[i];
}
// The items of n moves: (pool, move, part), numbered so that neighbours touch neighbouring memory of one pool.
struct MoveItem {
  uint32_t pool, move, part;
};
__device__ __forceinline__ MoveItem itemOf(const PoolSet& p, uint64_t item, uint32_t n) {
  const uint64_t perPool = (uint64_t)n * p.parts;
  MoveItem m;
  m.pool = (uint32_t)(item / perPool);
  const uint64_t in = item - m.pool * perPool;
  m.move = (uint32_t)(in / p.parts);
  m.part = (uint32_t)(in - (uint64_t)m.move * p.parts);
  return m;
}
template <int LOADS, bool NT>
__device__ __forceinline__ void moveItem(const PoolSet& p, int32_t src, int32_t dst, const MoveItem& m, int lane) {
  const size_t at = (size_t)m.part * partBytes(LOADS);
  // (the last part's size comes from the host: the minimum of two 64-bit sizes that are the same in every lane is
  // compiled into a vector compare whose result the scalar select that follows does not read)
  const uint32_t bytes = m.part + 1 == p.parts ? p.lastBytes : partBytes(LOADS);
  movePart<LOADS, NT>(p.from[m.pool] + (size_t)src * p.pageBytes + at, p.to[m.pool] + (size_t)dst * p.pageBytes + at, bytes,
                      (uint32_t)lane);
}

// 300 pages of 32 KiB in 64 pools, 1.26 GB of traffic: 208 us = 6.0 TB/s, as much as the library's dense copy reaches
// (6.1). What that took: workgroups that move 4 KiB and end (16 KiB: 228 us; a fixed number of workgroups that walk the
// pages: 255), pool by pool (pair by pair 14 us more), stores that do not stay in the caches (18 us).
__global__ __launch_bounds__(kMoveThreads) void copyKernel(PoolSet p, const int32_t* srcPages, const int32_t* dstPages,
                                                           int32_t n, int32_t srcTotal, int32_t dstTotal) {
  const int lane = (int)(threadIdx.x & 63);
  const uint64_t items = (uint64_t)n * p.npools * p.parts;
  for (uint64_t item = (uint64_t)blockIdx.x * kMoveWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kMoveWaves) {
    const MoveItem m = itemOf(p, item, (uint32_t)n);
    const int32_t src = uniform(srcPages[m.move]), dst = uniform(dstPages[m.move]);
    if (src < 0 || src >= srcTotal || dst < 0 || dst >= dstTotal) continue;
    moveItem<kCopyLoads, false>(p, src, dst, m, lane);
  }
}

// One request of a fork, by a workgroup: the child's whole pages are the parent's, a last page that is not full is its own.
__device__ __forceinline__ void forkOne(const Books& b, const PageScratch& s, const Requests& q, ListIndex i) {
  const int32_t first = s.request[i], before = s.before[i];
  const int32_t whole = before / b.pageTokens, need = before % b.pageTokens != 0;
  if (first < 0 || (need != 0 && first >= s.counts[0])) {
    if (threadIdx.x == 0) refuse(b);
    return;
  }
  const int32_t parent = q.a[i], child = q.b[i];
  const int32_t* from = b.tables + (size_t)parent * b.perSeq;
  int32_t* to = b.tables + (size_t)child * b.perSeq;
  for (ListIndex k = threadIdx.x; k < (ListIndex)whole; k += kMoveThreads) {
    const int32_t page = from[k];
    to[k] = page;
    if (page >= 0 && page < b.pages) __hip_atomic_fetch_add(&b.refcounts[page], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (threadIdx.x == 0) {
    if (need != 0) {
      const int32_t page = s.found[first];
      to[whole] = page;
      b.refcounts[page] = 1;
    }
    b.lengths[child] = before;
  }
}
// 512 forks of 8 pools' 16 KiB pages: 16 children read the same page, so loads stay in the caches (25 us for the call; 39
// if they do not). Two loads a lane: 25 us, four 27, one 33 (every wave looks its request up).
// The first tableBlocks workgroups (of the first launch, if the pools take several) write the tables, the others copy the
// contents of the last pages. Neither reads what the other writes: children were empty, and parents stay as they are.
__global__ __launch_bounds__(kMoveThreads) void forkKernel(Books b, PageScratch s, Requests q, PoolSet p, uint32_t tableBlocks) {
  if (blockIdx.x < tableBlocks) {
    for (ListIndex i = blockIdx.x; i < (ListIndex)q.n; i += tableBlocks) forkOne(b, s, q, i);
    return;
  }
  const int lane = (int)(threadIdx.x & 63);
  const uint64_t items = (uint64_t)q.n * p.npools * p.parts;
  for (uint64_t item = (uint64_t)(blockIdx.x - tableBlocks) * kMoveWaves + waveInBlock(); item < items;
       item += (uint64_t)(gridDim.x - tableBlocks) * kMoveWaves) {
    const MoveItem m = itemOf(p, item, (uint32_t)q.n);
    const int32_t first = uniform(s.request[m.move]), before = uniform(s.before[m.move]);
    if (first < 0 || before % b.pageTokens == 0 || first >= uniform(s.counts[0])) continue;
    const int32_t src = uniform(b.tables[(size_t)uniform(q.a[m.move]) * b.perSeq + before / b.pageTokens]);
    if (src < 0 || src >= b.pages) continue;
    moveItem<kForkLoads, false>(p, src, uniform(s.found[first]), m, lane);
  }
}

// Free: one workgroup per sequence. Whoever takes the length out frees the pages, so a sequence that is listed
// twice is freed once.
__global__ __launch_bounds__(kMoveThreads) void freeKernel(Books b, const int32_t* seqs, int32_t n) {
  struct Shared {
    int32_t length;
  };
  DFCCL_WG_SHARED(Shared, sh);
  for (ListIndex i = blockIdx.x; i < (ListIndex)n; i += gridDim.x) {
    const int32_t seq = seqs[i];
    if (threadIdx.x == 0)
      sh.length = seq >= 0 && seq < b.seqs
                      ? __hip_atomic_exchange(&b.lengths[seq], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                      : 0;
    __syncthreads();
    const int32_t length = sh.length;
    if (length > 0) {
      int32_t used = pagesOf(length, b.pageTokens);
      if (used > b.perSeq) used = b.perSeq;
      int32_t* row = b.tables + (size_t)seq * b.perSeq;
      for (ListIndex k = threadIdx.x; k < (ListIndex)used; k += kMoveThreads) {
        const int32_t page = row[k];
        row[k] = -1;
        if (page >= 0 && page < b.pages)
          __hip_atomic_fetch_add(&b.refcounts[page], -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    __syncthreads();
  }
}

// Compact, the plan: with L pages live, the k-th live page at or above L goes to the k-th free page below L. Sources
// and destinations are disjoint, so all of them can move at once, and no plan moves fewer pages. One workgroup.
__global__ __launch_bounds__(kScanThreads) void compactPlanKernel(Books b, PageScratch s) {
  struct Shared {
    ScanShared scan;
  };
  DFCCL_WG_SHARED(Shared, sh);
  int32_t live = 0;
  int which = 0;
  for (int64_t at = 0; at < b.pages; at += kScanTile, which ^= 1) {
    int32_t c[kScanPer], mine = 0, total;
    loadCounts(b, at + (int64_t)threadIdx.x * kScanPer, c);
#pragma unroll
    for (int i = 0; i < kScanPer; i++) mine += c[i] > 0 && at + (int64_t)threadIdx.x * kScanPer + i < b.pages;
    (void)blockScan(sh.scan, which, mine, total);
    live += total;
  }
  int32_t holes = 0, movers = 0;
  for (int64_t at = 0; at < b.pages; at += kScanTile) {
    const int64_t first = at + (int64_t)threadIdx.x * kScanPer;
    int32_t c[kScanPer], hole = 0, mover = 0, totalHoles, totalMovers;
    loadCounts(b, first, c);
#pragma unroll
    for (int i = 0; i < kScanPer; i++) {
      hole += first + i < live && c[i] <= 0;
      mover += first + i >= live && first + i < b.pages && c[i] > 0;
    }
    __syncthreads();  // (the totals of the round before have been read)
    int32_t h = holes + blockScan(sh.scan, 0, hole, totalHoles);
    int32_t m = movers + blockScan(sh.scan, 1, mover, totalMovers);
#pragma unroll
    for (int i = 0; i < kScanPer; i++) {
      if (first + i < live && c[i] <= 0) s.found[h++] = (int32_t)(first + i);
      if (first + i >= live && first + i < b.pages && c[i] > 0) {
        s.rank[first + i] = m;
        s.movers[m++] = (int32_t)(first + i);
      }
    }
    holes += totalHoles;
    movers += totalMovers;
  }
  if (threadIdx.x == 0) {
    s.counts[0] = holes;
    s.counts[1] = movers;  // (as many as holes)
    if (b.report != nullptr) {
      b.report[1] = movers;
      b.report[2] = live;
    }
  }
}
// The plan over many tiles, second launch: a workgroup per tile. With the live pages before a page known, a hole's
// place is the number of free pages before it, and a mover's the number of live pages between L and it.
__global__ __launch_bounds__(kScanThreads) void listMovesKernel(Books b, PageScratch s, int32_t tiles) {
  struct Shared {
    ScanShared scan;
  };
  DFCCL_WG_SHARED(Shared, sh);
  const int32_t tile = (int32_t)blockIdx.x;
  const int32_t live = sumTiles(sh.scan, 0, s.tiles, tiles), before = sumTiles(sh.scan, 1, s.tiles, tile);
  __syncthreads();
  const int32_t edge = live / kScanTile;  // the tile that L lies in, or the one behind the last
  int32_t below = sumTiles(sh.scan, 0, s.tiles, edge);
  const int64_t edgeAt = (int64_t)edge * kScanTile + (int64_t)threadIdx.x * kScanPer, first =
      (int64_t)tile * kScanTile + (int64_t)threadIdx.x * kScanPer;
  int32_t c[kScanPer], mine = 0, total;
  loadCounts(b, edgeAt, c);
#pragma unroll
  for (int i = 0; i < kScanPer; i++) mine += edgeAt + i < live && c[i] > 0;
  (void)blockScan(sh.scan, 1, mine, total);
  below += total;  // live pages below L
  __syncthreads();
  mine = 0;
  loadCounts(b, first, c);
#pragma unroll
  for (int i = 0; i < kScanPer; i++) mine += first + i < b.pages && c[i] > 0;
  int32_t liveBefore = before + blockScan(sh.scan, 0, mine, total);
#pragma unroll
  for (int i = 0; i < kScanPer; i++)
    if (first + i < b.pages) {
      const int32_t page = (int32_t)(first + i);
      if (c[i] <= 0) {
        if (page < live) s.found[page - liveBefore] = page;
      } else {
        if (page >= live) {
          s.rank[page] = liveBefore - below;
          s.movers[liveBefore - below] = page;
        }
        liveBefore++;
      }
    }
  if (tile == 0 && threadIdx.x == 0) {
    s.counts[1] = live - below;
    if (b.report != nullptr) {
      b.report[1] = live - below;
      b.report[2] = live;
    }
  }
}

// 1000 moves of 16 pools' 16 KiB pages, 96 us for the call: the pages are read and written at 5.6 TB/s. How many move is
// known on the GPU only, so a grid of at most kMaxCompactGrid walks them: 96 us; 2048 workgroups 105. Four loads a lane
// that do not stay in the caches: 98 us in that sweep, two 103, one 105; loads that stay 104.
// Compact, the moves: the first bookBlocks workgroups (of the first launch) let table entries and counts follow, the
// others move the contents.
__global__ __launch_bounds__(kMoveThreads) void compactKernel(Books b, PageScratch s, PoolSet p, uint32_t bookBlocks) {
  const int32_t moves = uniform(s.counts[1]);
  if (blockIdx.x < bookBlocks) {
    for (ListIndex i = blockIdx.x * kMoveThreads + threadIdx.x; i < (ListIndex)moves; i += bookBlocks * kMoveThreads) {
      const int32_t from = s.movers[i], to = s.found[i];
      b.refcounts[to] = b.refcounts[from];
      b.refcounts[from] = 0;
    }
    for (ListIndex seq = blockIdx.x; seq < (ListIndex)b.seqs; seq += bookBlocks) {
      const int32_t length = b.lengths[seq];
      if (length <= 0) continue;
      int32_t used = pagesOf(length, b.pageTokens);
      if (used > b.perSeq) used = b.perSeq;
      int32_t* row = b.tables + (size_t)seq * b.perSeq;
      for (ListIndex k = threadIdx.x; k < (ListIndex)used; k += kMoveThreads) {
        const int32_t page = row[k];
        if (page < 0 || page >= b.pages) continue;
        const int32_t r = s.rank[page];  // (left over from anywhere for a page that does not move)
        if (r >= 0 && r < moves && s.movers[r] == page) row[k] = s.found[r];
      }
    }
    return;
  }
  const int lane = (int)(threadIdx.x & 63);
  const uint64_t items = (uint64_t)moves * p.npools * p.parts;
  for (uint64_t item = (uint64_t)(blockIdx.x - bookBlocks) * kMoveWaves + waveInBlock(); item < items;
       item += (uint64_t)(gridDim.x - bookBlocks) * kMoveWaves) {
    const MoveItem m = itemOf(p, item, (uint32_t)moves);
    moveItem<kCompactLoads, true>(p, uniform(s.movers[m.move]), uniform(s.found[m.move]), m, lane);
  }
}

// ---- host

struct PagePlan {
  size_t owner, request, before, found, movers, rank, tiles, counts, bytes;
};
static int64_t tilesOf(int64_t pages) { return (pages + kScanTile - 1) / kScanTile; }
static PagePlan planPages(int64_t pages, int64_t seqs) {
  PagePlan p{};
  size_t at = 0;
  auto take = [&at](int64_t ints) {
    const size_t here = at;
    at += ((size_t)ints * 4 + 255) & ~(size_t)255;
    return here;
  };
  p.owner = take(seqs);
  p.request = take(seqs);
  p.before = take(seqs);
  p.found = take(pages);
  p.movers = take(pages);
  p.rank = take(pages);
  p.tiles = take(tilesOf(pages));
  p.counts = take(4);
  p.bytes = at;
  return p;
}

static bool soundPools(const dfcclPageCache* c) {
  if (c == nullptr || c->structBytes < sizeof(dfcclPageCache)) return false;
  if (c->pages < 1 || c->npools < 1 || c->pageBytes == 0 || c->pools == nullptr) return false;
  for (int i = 0; i < c->npools; i++)
    if (c->pools[i] == nullptr) return false;
  return true;
}
static bool soundCache(const dfcclPageCache* c) {
  if (!soundPools(c)) return false;
  if (c->pageTokens < 1 || c->sequences < 1 || c->pagesPerSequence < 1) return false;
  // entries and lengths are 32-bit integers
  if ((int64_t)c->sequences * c->pagesPerSequence > 0x7fffffffll) return false;
  if ((int64_t)c->pagesPerSequence * c->pageTokens > 0x7fffffffll) return false;
  if (c->refcounts == nullptr || c->tables == nullptr || c->lengths == nullptr || c->workspace == nullptr) return false;
  return c->workspaceBytes >= planPages(c->pages, c->sequences).bytes && ((uintptr_t)c->workspace & 3u) == 0;
}
static Books booksOf(const dfcclPageCache* c) {
  Books b{};
  b.refcounts = c->refcounts;
  b.tables = c->tables;
  b.lengths = c->lengths;
  b.report = c->report;
  b.pages = c->pages;
  b.pageTokens = c->pageTokens;
  b.seqs = c->sequences;
  b.perSeq = c->pagesPerSequence;
  return b;
}
static PageScratch scratchOf(const dfcclPageCache* c) {
  const PagePlan p = planPages(c->pages, c->sequences);
  char* ws = (char*)c->workspace;
  PageScratch s{};
  s.owner = (int32_t*)(ws + p.owner);
  s.request = (int32_t*)(ws + p.request);
  s.before = (int32_t*)(ws + p.before);
  s.found = (int32_t*)(ws + p.found);
  s.movers = (int32_t*)(ws + p.movers);
  s.rank = (int32_t*)(ws + p.rank);
  s.tiles = (int32_t*)(ws + p.tiles);
  s.counts = (int32_t*)(ws + p.counts);
  return s;
}
static PoolSet poolSet(const dfcclPageCache* to, const dfcclPageCache* from, int first, int loads) {
  PoolSet p{};
  p.npools = std::min(kMaxPools, to->npools - first);
  for (int i = 0; i < p.npools; i++) {
    p.to[i] = (char*)to->pools[first + i];
    p.from[i] = (const char*)from->pools[first + i];
  }
  p.pageBytes = to->pageBytes;
  p.parts = (uint32_t)((to->pageBytes + partBytes(loads) - 1) / partBytes(loads));
  p.lastBytes = (uint32_t)(to->pageBytes - (size_t)(p.parts - 1) * partBytes(loads));
  return p;
}
static_assert(0x7fffffffull + kMaxRequestGrid <= (ListIndex)~0u, "a walk's last step");
constexpr uint64_t kMaxMoveGrid = 1u << 22;
constexpr unsigned kMaxCompactGrid = 1u << 16;
static unsigned moveGrid(uint64_t items) {
  return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>((items + kMoveWaves - 1) / kMoveWaves, kMaxMoveGrid));
}
static unsigned requestGrid(int n) { return std::min((uint32_t)n, kMaxRequestGrid); }
// Returns whether that has carried the requests out, too.
template <int FOR>
static bool launchAssign(const Books& b, const PageScratch& s, const Requests& q, hipStream_t st) {
  const int32_t tiles = (int32_t)tilesOf(b.pages);
  const bool few = FOR == kForExtend && q.n <= kFewRequests;
  if (tiles <= kOneScan) {
    DFCCL_LAUNCH_BLOCKS(assignKernel<FOR == kForFork>, 1, kScanThreads, st, b, s, q, few);
    return few;
  } else {
    DFCCL_LAUNCH_BLOCKS(countTilesKernel<FOR>, (unsigned)tiles + 1, kScanThreads, st, b, s, q);
    DFCCL_LAUNCH_BLOCKS(listFreeKernel, (unsigned)tiles, kScanThreads, st, b, s, tiles);
    return false;
  }
}
static ncclResult_t launched() { return hipGetLastError() == hipSuccess ? ncclSuccess : ncclUnhandledCudaError; }
// a page's parts over a launch's pools are counted in 32 bits
static bool soundPage(const dfcclPageCache* c) { return c->pageBytes <= ((size_t)1 << 36); }  // (2^26 parts, 64 pools)

}  // namespace dfccl

using namespace dfccl;

#define DFCCL_API extern "C" __attribute__((visibility("default")))

DFCCL_API ncclResult_t dfcclPageCacheWorkspace(int pages, int sequences, size_t* bytes) {
  if (pages < 1 || sequences < 1 || bytes == nullptr) return ncclInvalidArgument;
  *bytes = planPages(pages, sequences).bytes;
  return ncclSuccess;
}

DFCCL_API ncclResult_t dfcclPagesCopy(const dfcclPageCache* to, const dfcclPageCache* from, const int32_t* srcPages,
                                      const int32_t* dstPages, int n, void* stream) {
  if (!soundPools(to) || !soundPools(from) || !soundPage(to)) return ncclInvalidArgument;
  if (to->npools != from->npools || to->pageBytes != from->pageBytes || n < 0) return ncclInvalidArgument;
  if (n == 0) return ncclSuccess;
  if (srcPages == nullptr || dstPages == nullptr) return ncclInvalidArgument;
  for (int first = 0; first < to->npools; first += kMaxPools) {
    const PoolSet p = poolSet(to, from, first, kCopyLoads);
    DFCCL_LAUNCH_BLOCKS(copyKernel, moveGrid((uint64_t)n * p.npools * p.parts), kMoveThreads, (hipStream_t)stream, p, srcPages,
                        dstPages, n, from->pages, to->pages);
  }
  return launched();
}

DFCCL_API ncclResult_t dfcclPagesExtend(const dfcclPageCache* c, const int32_t* sequences, const int32_t* lengths, int n,
                                        void* stream) {
  if (!soundCache(c) || n < 0 || n > c->sequences) return ncclInvalidArgument;
  if (n > 0 && (sequences == nullptr || lengths == nullptr)) return ncclInvalidArgument;
  const Books b = booksOf(c);
  const hipStream_t st = (hipStream_t)stream;
  const PageScratch s = scratchOf(c);
  const Requests q{sequences, lengths, n};
  const bool done = launchAssign<kForExtend>(b, s, q, st);
  if (n > 0 && !done) DFCCL_LAUNCH_BLOCKS(extendKernel, requestGrid(n), kMoveThreads, st, b, s, q);
  return launched();
}

DFCCL_API ncclResult_t dfcclPagesFork(const dfcclPageCache* c, const int32_t* parents, const int32_t* children, int n,
                                      void* stream) {
  if (!soundCache(c) || !soundPage(c) || n < 0 || n > c->sequences) return ncclInvalidArgument;
  if (n > 0 && (parents == nullptr || children == nullptr)) return ncclInvalidArgument;
  const Books b = booksOf(c);
  const hipStream_t st = (hipStream_t)stream;
  const PageScratch s = scratchOf(c);
  const Requests q{parents, children, n};
  (void)launchAssign<kForFork>(b, s, q, st);
  for (int first = 0; n > 0 && first < c->npools; first += kMaxPools) {
    const PoolSet p = poolSet(c, c, first, kForkLoads);
    const unsigned tableBlocks = first == 0 ? requestGrid(n) : 0u;
    DFCCL_LAUNCH_BLOCKS(forkKernel, tableBlocks + moveGrid((uint64_t)n * p.npools * p.parts), kMoveThreads, st, b, s, q, p,
                        tableBlocks);
  }
  return launched();
}

DFCCL_API ncclResult_t dfcclPagesFree(const dfcclPageCache* c, const int32_t* sequences, int n, void* stream) {
  if (!soundCache(c) || n < 0 || (n > 0 && sequences == nullptr)) return ncclInvalidArgument;
  if (n == 0) return ncclSuccess;
  DFCCL_LAUNCH_BLOCKS(freeKernel, requestGrid(n), kMoveThreads, (hipStream_t)stream, booksOf(c), sequences, n);
  return launched();
}

DFCCL_API ncclResult_t dfcclPagesCompact(const dfcclPageCache* c, void* stream) {
  if (!soundCache(c) || !soundPage(c)) return ncclInvalidArgument;
  const Books b = booksOf(c);
  const PageScratch s = scratchOf(c);
  const hipStream_t st = (hipStream_t)stream;
  const int32_t tiles = (int32_t)tilesOf(b.pages);
  if (tiles <= kOneScan) {
    DFCCL_LAUNCH_BLOCKS(compactPlanKernel, 1, kScanThreads, st, b, s);
  } else {
    DFCCL_LAUNCH_BLOCKS(countTilesKernel<kForCompact>, (unsigned)tiles + 1, kScanThreads, st, b, s, Requests{});
    DFCCL_LAUNCH_BLOCKS(listMovesKernel, (unsigned)tiles, kScanThreads, st, b, s, tiles);
  }
  for (int first = 0; first < c->npools; first += kMaxPools) {
    const PoolSet p = poolSet(c, c, first, kCompactLoads);
    // how many pages move is known on the GPU only: at most half of them
    const uint64_t most = (uint64_t)(c->pages / 2) * p.npools * p.parts;
    const unsigned bookBlocks = first == 0 ? (unsigned)std::min(c->sequences, 2048) : 0u;
    DFCCL_LAUNCH_BLOCKS(compactKernel, bookBlocks + std::min(moveGrid(most), kMaxCompactGrid), kMoveThreads, st, b, s, p, bookBlocks);
  }
  return launched();
}

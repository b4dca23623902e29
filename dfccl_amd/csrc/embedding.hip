// Embedding lookup with scaling, and its gradient by sorted tokens (dfcclEmbeddingLookup, dfcclEmbeddingGrad in
// ofccl.h): a copy of rows and a sum of rows that are named by an index.
//
// Lookup:    out[t,:] = round(scale * table[id_t - first,:]), zeros for an id outside the piece.
// Gradient:  G[v,:] = round([G[v,:] +] scale * sum over the tokens t of all sources with id_t - first = v of
//            grad[t,:]), summed in fp32 in the order source, token.
// Both are bound by HBM: every row of the output is written once, every row of the input read once.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/ofccl.h"
#include "indexed_common.h"

namespace dfccl {

constexpr int kRowThreads = 256;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kPieceElems = 64 * kVec;  // what one wave covers of a row: eight elements a lane
constexpr int kMaxSrcs = 8;
// grids are capped here and walked with a stride (a launch may not have 2^32 threads)
constexpr uint64_t kMaxGrid = 1u << 22;

static bool rowType(int dt) { return dt == kF16 || dt == kBF16 || dt == kF32; }
static unsigned gridFor(uint64_t waves) {
  return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>((waves + kRowWaves - 1) / kRowWaves, kMaxGrid));
}

__device__ __forceinline__ int64_t loadId(const char* ids, int idBytes, size_t i) {
  if (idBytes == 8) return ((const DFCCL_GLOBAL int64_t*)ids)[i];
  return ((const DFCCL_GLOBAL int32_t*)ids)[i];
}

// the row of the piece that an id names, -1 for an id outside it
__device__ __forceinline__ int64_t rowOf(int64_t id, int64_t firstRow, int64_t rows) {
  const uint64_t row = (uint64_t)id - (uint64_t)firstRow;
  return id >= firstRow && row < (uint64_t)rows ? (int64_t)row : -1;
}

// ------------------------------------------------------------------------------------------------- lookup

struct LookupArgs {
  const char* table;
  const char* ids;
  char* out;
  int64_t firstRow, rows;
  size_t tableStride, outStride;  // bytes
  uint64_t tokens;
  uint32_t width, pieces;
  int idBytes;
  float scale;
};

// One wave takes one piece (512 elements) of U tokens' rows: the U ids, then the U loads are in flight together. Bound by
// HBM: 16385 rows of 4096, fp32 in, bfloat16 out, 46 us = 5.4 TB/s on each different row once (a dense copy of as much
// takes 41 us). Two rows a wave: 46 us, four 48, one 53; stores that stay in the caches: 55 (they push the table's
// frequent rows out). fp32 outputs are stored in two halves of a line each, which have to meet in a cache.
template <int IN, int OUT, int U>
__global__ __launch_bounds__(kRowThreads) void lookupKernel(LookupArgs a) {
  const int lane = (int)(threadIdx.x & 63);
  const uint64_t groups = (a.tokens + U - 1) / U, items = groups * a.pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * kRowWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kRowWaves) {
    const uint64_t t0 = item / a.pieces * U;
    const uint32_t col = (uint32_t)(item % a.pieces) * kPieceElems + (uint32_t)lane * kVec;
    const bool full = col + kVec <= a.width;
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      row[u] = t0 + u < a.tokens ? uniform(rowOf(loadId(a.ids, a.idBytes, t0 + u), a.firstRow, a.rows)) : -1;
    if (full) {
      Raw8<IN> raw[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const bool inside = row[u] >= 0;
        if (inside) raw[u] = loadRaw8<IN>(a.table + (size_t)row[u] * a.tableStride + (size_t)col * typeSize(IN));
        else raw[u] = Raw8<IN>{};
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (t0 + u >= a.tokens) break;
        const bool inside = row[u] >= 0;
        float f[kVec];
        widen8<IN>(raw[u], f);
#pragma unroll
        for (int i = 0; i < kVec; i++) f[i] = inside ? f[i] * a.scale : 0.0f;
        store8<OUT, OUT != kF32>(a.out + (t0 + u) * a.outStride + (size_t)col * typeSize(OUT), f);
      }
    } else if (col < a.width) {
      const int left = (int)(a.width - col);
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (t0 + u >= a.tokens) break;
        const bool inside = row[u] >= 0;
        float f[kVec] = {};
        if (inside) loadTail<IN>(a.table + (size_t)row[u] * a.tableStride + (size_t)col * typeSize(IN), left, f);
#pragma unroll
        for (int i = 0; i < kVec; i++) f[i] = inside ? f[i] * a.scale : 0.0f;
        storeTail<OUT>(a.out + (t0 + u) * a.outStride + (size_t)col * typeSize(OUT), left, f);
      }
    }
  }
}

typedef void (*LookupKernel)(LookupArgs);
template <int IN, int U>
static LookupKernel pickLookupOut(int out) {
  return out == kF32 ? lookupKernel<IN, kF32, U> : out == kF16 ? lookupKernel<IN, kF16, U> : lookupKernel<IN, kBF16, U>;
}
template <int U>
static LookupKernel pickLookup(int in, int out) {
  return in == kF32 ? pickLookupOut<kF32, U>(out) : in == kF16 ? pickLookupOut<kF16, U>(out) : pickLookupOut<kBF16, U>(out);
}

// ------------------------------------------------------------------------------------------------- gradient
//
// 1. Sort. Every token gets a key, its row (or `rows` if it does not count: outside the piece, or padding), and a
//    payload, its source and number. A radix sort from the low digit up, stable and without atomics on positions,
//    puts equal keys side by side in the order source, token: the order of every sum is fixed by the ids and the rows
//    that they name here (where a block of 2. begins in a run depends on how many tokens the rows before have).
// 2. Chunks. The sorted list is cut into chunks of kChunk. A chunk that lies within one row's run is summed by a
//    wave of its own into fp32 scratch, and so are kSuper such chunks: a row that many tokens share (padding that
//    counts, frequent words) is summed by many waves, and again in a fixed order.
// 3. Rows. A wave per group of sorted positions and row piece sums the runs that begin in its group: single tokens up to
//    the first whole chunk, whole chunks' (and chunks of chunks') sums, single tokens after the last.
// Without accumulation the rows that no token names have to become zeros. That is most of the table and most of the
// bytes, and it needs nothing of the sort: all rows are cleared by additional workgroups of the launches of 1.,
// which leave most of the chip idle, and the named rows are written over afterwards.

constexpr int kChunk = 16;         // tokens
constexpr int kSuper = 16;         // chunks
constexpr int kSuperTokens = kChunk * kSuper;
constexpr int kMaxDigitBits = 10;
constexpr int kMaxBins = 1 << kMaxDigitBits;
constexpr int kSrcShift = 28;  // payload: source << 28 | token, so a source has fewer than 2^28 tokens
constexpr uint32_t kTokenMask = (1u << kSrcShift) - 1;

struct GradArgs {
  const char* grads[kMaxSrcs];
  const char* ids[kMaxSrcs];
  uint32_t firstPos[kMaxSrcs + 1];  // the tokens of source r are positions firstPos[r] .. firstPos[r+1] before sorting
  int nsrcs, idBytes;
  size_t gradStride, tableStride;  // bytes
  int64_t firstRow, paddingId;
  uint32_t rows, width, pieces, n;
  float scale;
  bool chunked, supered;  // whether there are sums of chunks, and of chunks of chunks
  char* table;
  // workspace
  uint32_t* keys[2];
  uint32_t* pays[2];
  uint32_t* hist;     // [tiles][bins]
  float* chunkSums;   // [n / kChunk][widthPad]
  float* superSums;   // [n / kSuperTokens][widthPad]
  uint32_t widthPad;  // width rounded up to kVec
};

struct SortPass {
  int from, shift, bits, tiles;  // keys[from] -> keys[from ^ 1]
};

// A share of the clearing of the table: parts [begin, end), done by the launch's workgroups from firstBlock on. A table
// without gaps between its rows is cleared as one range, a part being what a workgroup stores at once; otherwise a part
// is kGapBytes of one row, by a wave.
struct Clear {
  char* at;
  size_t stride;        // of the rows, 0 for one range
  uint64_t bytes;       // of a row, or of the range
  uint64_t rowParts;    // of a row
  uint64_t begin, end;
  uint32_t firstBlock;
};
// How a workgroup clears a range, from a sweep over 1 GiB: workgroups of 4 waves that store 16 bytes a thread once and
// end reach 7.0 TB/s (four stores a thread 6.1, a fixed number of workgroups that walk the range 4.9 to 5.4); a
// workgroup of 16 waves that has its compute unit to itself walks the range with eight stores a thread, each 16 KiB of
// the workgroup in one piece (6.5 TB/s; four stores 6.1, each wave's stores in one piece 5.6).
constexpr uint32_t clearStores(uint32_t waves) { return waves >= 16 ? 8 : 1; }
constexpr uint32_t clearPart(uint32_t waves) { return waves * clearStores(waves) * 1024; }
constexpr uint32_t kGapBytes = 4096;

template <uint32_t WAVES>
__device__ __forceinline__ void clearShare(const Clear& c) {
  const uint32_t lane = threadIdx.x & 63, blocks = gridDim.x - c.firstBlock, block = blockIdx.x - c.firstBlock;
  const u32x4 zero = {0, 0, 0, 0};
  if (c.stride == 0) {
    constexpr uint32_t part = clearPart(WAVES);
    for (uint64_t i = c.begin + block; i < c.end; i += blocks) {
      char* to = c.at + i * part;
      const uint64_t left = c.bytes - i * part;
      if (left >= part) {
#pragma unroll
        for (uint32_t u = 0; u < clearStores(WAVES); u++) store16<2>(to + (u * WAVES * 64 + threadIdx.x) * 16, zero);
      } else {  // the range's last bytes, an even number
        for (uint32_t p = threadIdx.x; p < (uint32_t)left / 16; p += WAVES * 64) store16<2>(to + p * 16, zero);
        for (uint32_t p = (uint32_t)left / 16 * 8 + threadIdx.x; p < (uint32_t)left / 2; p += WAVES * 64) storeElem<2>(to, p, 0);
      }
    }
    return;
  }
  for (uint64_t i = c.begin + (uint64_t)block * WAVES + (uint32_t)waveInBlock(); i < c.end; i += (uint64_t)blocks * WAVES) {
    const uint64_t row = i / c.rowParts, part = i - row * c.rowParts;
    char* to = c.at + row * c.stride + part * kGapBytes;
    const uint32_t left = part + 1 < c.rowParts ? kGapBytes : (uint32_t)(c.bytes - part * kGapBytes);
    for (uint32_t p = lane; p < left / 16; p += 64) store16<2>(to + p * 16, zero);
    for (uint32_t p = left / 16 * 8 + lane; p < left / 2; p += 64) storeElem<2>(to, p, 0);
  }
}

// The keys and payloads of S positions before sorting (of the last one, for positions behind it). The ids are loaded
// without conditions, all of them at once: under one, each load would be waited for by itself.
template <int S>
__device__ __forceinline__ void keysOfTokens(const GradArgs& a, const uint32_t (&pos)[S], uint32_t (&key)[S], uint32_t (&pay)[S]) {
  const char* at[S];
#pragma unroll
  for (int k = 0; k < S; k++) {
    const uint32_t p = pos[k] < a.n ? pos[k] : a.n - 1;
    uint32_t r = 0, first = 0;
    const char* ids = a.ids[0];
#pragma unroll
    for (int i = 1; i < kMaxSrcs; i++) {
      const bool behind = i < a.nsrcs && p >= a.firstPos[i];
      r = behind ? (uint32_t)i : r;
      ids = behind ? a.ids[i] : ids;
      first = behind ? a.firstPos[i] : first;
    }
    pay[k] = (r << kSrcShift) | (p - first);
    at[k] = ids + (size_t)(p - first) * a.idBytes;
  }
  int64_t id[S];
  if (a.idBytes == 8) {
#pragma unroll
    for (int k = 0; k < S; k++) id[k] = *(const DFCCL_GLOBAL int64_t*)at[k];
  } else {
#pragma unroll
    for (int k = 0; k < S; k++) id[k] = *(const DFCCL_GLOBAL int32_t*)at[k];
  }
#pragma unroll
  for (int k = 0; k < S; k++) {
    const int64_t row = rowOf(id[k], a.firstRow, a.rows);
    key[k] = row >= 0 && id[k] != a.paddingId ? (uint32_t)row : a.rows;
  }
}
__device__ __forceinline__ uint32_t payOf(const GradArgs& a, uint32_t pos) {
  uint32_t r = 0, first = 0;
#pragma unroll
  for (int i = 1; i < kMaxSrcs; i++)
    if (i < a.nsrcs && pos >= a.firstPos[i]) {
      r = (uint32_t)i;
      first = a.firstPos[i];
    }
  return (r << kSrcShift) | (pos - first);
}

// A strip's 64 keys of one wave: every lane's rank among the strip's keys of its digit, found with a ballot per bit,
// and their number (`same`, a mask). Lanes without a key are in no mask.
__device__ __forceinline__ uint64_t sameDigit(uint32_t digit, int bits, bool valid) {
  uint64_t same = __ballot(valid);
  for (int b = 0; b < bits; b++) {
    const uint64_t ones = __ballot((digit >> b) & 1u);
    const uint64_t mine = (uint64_t)(int64_t)((int32_t)(digit << (31 - b)) >> 31);  // the lane's bit in all 64
    same &= ~(ones ^ mine);
  }
  return same;
}
// The rank of a strip's keys among the wave's keys of the same digit so far, whose counts are kept in LDS.
template <typename C>
__device__ __forceinline__ uint32_t rankInWave(C* count, uint32_t digit, int bits, bool valid, int lane) {
  const uint64_t same = sameDigit(digit, bits, valid);
  const uint64_t before = same & ((1ull << lane) - 1);
  const uint32_t old = count[digit];
  DFCCL_WAVE_LDS_SYNC();  // (every lane has read the count before the first of its digit raises it)
  if (valid && before == 0) count[digit] = (C)(old + (uint32_t)__builtin_popcountll(same));
  DFCCL_WAVE_LDS_SYNC();
  return old + (uint32_t)__builtin_popcountll(before);
}
__device__ __forceinline__ uint32_t waveScan(uint32_t v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t from = __shfl(v, (lane - d) & 63);
    if (lane >= d) v += from;
  }
  return v;
}

// ---- a few thousand tokens: sorted by one workgroup in LDS, one launch instead of two per digit. Bound by the latency
// of its steps and by the instructions of one compute unit (a ballot per bit and 64 keys): 12 us for 3600 tokens and 14
// bits, where counts and scatters take 21; 40 us for 13000 tokens, where those take 22.
constexpr int kSmallThreads = 1024;
constexpr int kSmallWaves = kSmallThreads / 64;
constexpr int kSmallStrips = 4;
// (a host build sets lower limits, to reach with few tokens what lies beyond them)
#ifndef DFCCL_SORT_SMALL_MAX
#define DFCCL_SORT_SMALL_MAX (kSmallThreads * kSmallStrips)
#endif
#ifndef DFCCL_SUPER_MIN
#define DFCCL_SUPER_MIN 8192
#endif
constexpr uint32_t kSmallMax = DFCCL_SORT_SMALL_MAX, kSuperMin = DFCCL_SUPER_MIN;
static_assert(kSmallMax <= kSmallThreads * kSmallStrips, "one workgroup sorts no more");
constexpr int kSmallDigitBits = 10;
constexpr int kSmallBins = 1 << kSmallDigitBits;
static_assert(kSmallBins == kSmallThreads, "a thread per bin");

__global__ __launch_bounds__(kSmallThreads) void sortSmallKernel(GradArgs a, int keyBits, Clear c) {
  constexpr int S = kSmallStrips;
  struct Shared {
    uint32_t key[kSmallThreads * S];
    uint16_t pos[kSmallThreads * S];  // before sorting
    uint16_t count[kSmallWaves][kSmallBins];
    uint32_t waveTotal[kSmallWaves];
  };
  static_assert(kSmallThreads * S < 65536, "positions and counts are held in 16 bits");
  DFCCL_WG_SHARED(Shared, sh);
  if (blockIdx.x >= c.firstBlock) {
    clearShare<kSmallWaves>(c);
    return;
  }
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = waveInBlock();
  const uint32_t start = (uint32_t)wave * (64 * S);
  uint32_t key[S], pos[S], rank[S];
#pragma unroll
  for (int k = 0; k < S; k++) pos[k] = start + k * 64 + lane;
  if (start < a.n) keysOfTokens<S>(a, pos, key, rank);  // (payloads are made from positions at the end)
  const int passes = (keyBits + kSmallDigitBits - 1) / kSmallDigitBits, bits = (keyBits + passes - 1) / passes;
  for (int pass = 0; pass < passes; pass++) {
    const int shift = pass * bits;
    const uint32_t mask = (1u << bits) - 1;
    const int bins = 1 << bits;
    if (tid < bins) {
#pragma unroll
      for (int w = 0; w < kSmallWaves; w++) sh.count[w][tid] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < S; k++)
      if (start + k * 64 < a.n)
        rank[k] = rankInWave(sh.count[wave], (key[k] >> shift) & mask, bits, start + k * 64 + lane < a.n, lane);
    __syncthreads();
    // a digit's keys begin behind all keys of smaller digits, a wave's behind the same digit's of the waves before
    uint32_t mine = 0;
    if (tid < bins) {
#pragma unroll
      for (int w = 0; w < kSmallWaves; w++) mine += sh.count[w][tid];
    }
    const uint32_t sum = waveScan(mine, lane);
    if (lane == 63) sh.waveTotal[wave] = sum;
    __syncthreads();
    uint32_t at = sum - mine;
    for (int w = 0; w < wave; w++) at += sh.waveTotal[w];
    if (tid < bins) {
#pragma unroll
      for (int w = 0; w < kSmallWaves; w++) {
        const uint32_t n = sh.count[w][tid];
        sh.count[w][tid] = (uint16_t)at;
        at += n;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < S; k++)
      if (start + k * 64 + lane < a.n) {
        const uint32_t to = sh.count[wave][(key[k] >> shift) & mask] + rank[k];
        sh.key[to] = key[k];
        sh.pos[to] = (uint16_t)pos[k];
      }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < S; k++) {
      const uint32_t at = start + k * 64 + lane;
      if (at < a.n) {
        key[k] = sh.key[at];
        pos[k] = sh.pos[at];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < S; k++) {
    const uint32_t at = start + k * 64 + lane;
    if (at < a.n) {
      a.keys[0][at] = key[k];
      a.pays[0][at] = payOf(a, pos[k]);
    }
  }
}

// ---- more tokens: tiles, a count and a scatter per digit (4 and 7 us at 13000 tokens, of which the launches are half)
constexpr int kSortThreads = 256;
constexpr int kSortWaves = kSortThreads / 64;
// 64-key strips of a wave of a tile: few enough that the tokens spread over several workgroups, many enough that there are
// few histograms, which every tile adds up for itself. Calls that add to 131072 rows of 8 columns (two digits): 16384
// tokens 35 us with 2 strips and 36 with 4, 24576 tokens 40 and 39; 65536 tokens 56 us with 4 and 68 with 16, 131072
// tokens 84 with either, 262144 tokens 139 and 119. Beyond, tiles and so histograms grow with the tokens, and what all
// tiles read of them with the square: 1 M tokens (256 tiles) 0.31 ms, 4 M 1.0 ms, 16 M (4096 tiles) 6.6 ms.
static int stripsOf(uint64_t n) { return n <= 16u * 1024 ? 2 : n <= 64u * 1024 ? 4 : 16; }

// The keys and payloads of a tile's strips before the first pass, a few strips at a time.
template <int S>
__device__ __forceinline__ void tileKeys(const GradArgs& a, const uint32_t (&pos)[S], uint32_t (&key)[S], uint32_t (&pay)[S]) {
  constexpr int N = S < 4 ? S : 4;
#pragma unroll
  for (int g = 0; g < S; g += N) {
    uint32_t p[N], k[N], y[N];
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = pos[g + i];
    keysOfTokens<N>(a, p, k, y);
#pragma unroll
    for (int i = 0; i < N; i++) {
      key[g + i] = k[i];
      pay[g + i] = y[i];
    }
  }
}

template <int S, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sortCountKernel(GradArgs a, SortPass p, Clear c) {
  struct Shared {
    uint32_t count[kMaxBins];
  };
  DFCCL_WG_SHARED(Shared, sh);
  if (blockIdx.x >= c.firstBlock) {
    clearShare<kSortWaves>(c);
    return;
  }
  const int tid = (int)threadIdx.x, tile = (int)blockIdx.x, bins = 1 << p.bits;
  for (int i = tid; i < bins; i += kSortThreads) sh.count[i] = 0;
  __syncthreads();
  uint32_t pos[S], key[S], pay[S];  // (positions of a launch fit 32 bits: there are fewer than 2^31 tokens)
#pragma unroll
  for (int k = 0; k < S; k++) pos[k] = (uint32_t)tile * (kSortThreads * S) + k * kSortThreads + tid;
  if constexpr (FIRST) {
    tileKeys<S>(a, pos, key, pay);
  } else {
#pragma unroll
    for (int k = 0; k < S; k++) key[k] = a.keys[p.from][pos[k] < a.n ? pos[k] : a.n - 1];
  }
#pragma unroll
  for (int k = 0; k < S; k++)
    if (pos[k] < a.n)
      __hip_atomic_fetch_add(&sh.count[(key[k] >> p.shift) & (bins - 1)], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  __syncthreads();
  for (int i = tid; i < bins; i += kSortThreads) a.hist[(size_t)tile * bins + i] = sh.count[i];
}

// Stable scatter of a tile: a key goes behind all keys of smaller digits, its digit's keys in the tiles before, in
// the waves before, in the wave's strips before, and in the lanes before.
template <int S, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sortScatterKernel(GradArgs a, SortPass p, Clear c) {
  struct Shared {
    uint32_t count[kSortWaves][kMaxBins];
    uint32_t base[kMaxBins];
    uint32_t total[kMaxBins];
    uint32_t waveTotal[kSortWaves];
  };
  DFCCL_WG_SHARED(Shared, sh);
  if (blockIdx.x >= c.firstBlock) {
    clearShare<kSortWaves>(c);
    return;
  }
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = waveInBlock(), tile = (int)blockIdx.x, bins = 1 << p.bits;
  uint32_t pos[S], key[S], pay[S], rank[S];
#pragma unroll
  for (int k = 0; k < S; k++) pos[k] = (uint32_t)tile * (kSortThreads * S) + (uint32_t)wave * (64 * S) + k * 64 + lane;
  if constexpr (FIRST) {
    tileKeys<S>(a, pos, key, pay);
  } else {
#pragma unroll
    for (int k = 0; k < S; k++) {
      const uint32_t at = pos[k] < a.n ? pos[k] : a.n - 1;
      key[k] = a.keys[p.from][at];
      pay[k] = a.pays[p.from][at];
    }
  }
  for (int i = tid; i < kMaxBins; i += kSortThreads) {
    uint32_t before = 0, total = 0;
    if (i < bins) {
#pragma unroll 8
      for (int t = 0; t < p.tiles; t++) {
        const uint32_t h = a.hist[(size_t)t * bins + i];
        before += t < tile ? h : 0;
        total += h;
      }
    }
    sh.base[i] = before;
    sh.total[i] = total;
#pragma unroll
    for (int w = 0; w < kSortWaves; w++) sh.count[w][i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < S; k++)
    rank[k] = rankInWave(sh.count[wave], (key[k] >> p.shift) & (uint32_t)(bins - 1), p.bits, pos[k] < a.n, lane);
  constexpr int per = kMaxBins / kSortThreads;
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < per; i++) mine += sh.total[tid * per + i];
  const uint32_t sum = waveScan(mine, lane);
  if (lane == 63) sh.waveTotal[wave] = sum;
  __syncthreads();
  uint32_t at = sum - mine;
  for (int w = 0; w < wave; w++) at += sh.waveTotal[w];
#pragma unroll
  for (int i = 0; i < per; i++) {
    const int bin = tid * per + i;
    uint32_t next = at + sh.base[bin];
    at += sh.total[bin];
#pragma unroll
    for (int w = 0; w < kSortWaves; w++) {  // the waves' counts become where the waves' keys begin
      const uint32_t n = sh.count[w][bin];
      sh.count[w][bin] = next;
      next += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < S; k++)
    if (pos[k] < a.n) {
      const uint32_t to = sh.count[wave][(key[k] >> p.shift) & (uint32_t)(bins - 1)] + rank[k];
      a.keys[p.from ^ 1][to] = key[k];
      a.pays[p.from ^ 1][to] = pay[k];
    }
}

// ---- sums

// A lane's eight columns of a row. Where they would reach beyond the row's end the lane loads the row's last eight
// elements instead and stores only its own of them: every lane's loads are the same single instruction, none is under
// a condition, and so all of them can be in flight. Rows of fewer than eight elements (NARROW) are put together from
// elements.
struct Columns {
  uint32_t at, slot;  // first column that is loaded; place in fp32 scratch (which has whole vectors)
  int count, shift;   // elements of a narrow row; how many of the eight are not the lane's (8: none is)
};
template <bool NARROW>
__device__ __forceinline__ Columns columnsOf(uint32_t width, uint32_t piece, int lane) {
  Columns c;
  c.slot = piece * kPieceElems + (uint32_t)lane * kVec;
  if constexpr (NARROW) {
    c.at = 0;
    c.count = c.slot == 0 ? (int)width : 0;
    c.shift = c.slot == 0 ? 0 : kVec;
  } else {
    c.at = c.slot < width - kVec ? c.slot : width - kVec;
    c.count = kVec;
    c.shift = c.slot - c.at < (uint32_t)kVec ? (int)(c.slot - c.at) : kVec;
  }
  return c;
}
template <int DT, bool NARROW>
__device__ __forceinline__ Raw8<DT> loadColumns(const char* row, const Columns& c) {
  const char* p = row + (size_t)c.at * typeSize(DT);
  if constexpr (!NARROW) return loadRaw8<DT>(p);
  Raw8<DT> r{};
#pragma unroll 1
  for (int j = c.count - 1; j >= 0; j--) {  // (in from the low end)
    const uint32_t e = (uint32_t)loadElem<typeSize(DT)>(p, j);
    u32x4 w = r.w[0];
    if constexpr (DT == kF32) {
      u32x4 h = r.w[1];
      r.w[1] = u32x4{w.w, h.x, h.y, h.z};
      r.w[0] = u32x4{e, w.x, w.y, w.z};
    } else {
      r.w[0] = u32x4{(w.x << 16) | e, (w.y << 16) | (w.x >> 16), (w.z << 16) | (w.y >> 16), (w.w << 16) | (w.z >> 16)};
    }
  }
  return r;
}
template <int DT, bool NARROW>
__device__ __forceinline__ void storeColumns(char* row, const Columns& c, const Raw8<DT>& r) {
  char* p = row + (size_t)c.at * typeSize(DT);
  if (!NARROW && c.shift == 0) {
    store16<typeSize(DT)>(p, r.w[0]);
    if constexpr (DT == kF32) store16<4>(p + 16, r.w[1]);
  } else if (c.shift < kVec) {
#pragma unroll
    for (int j = 0; j < kVec; j++)
      if (j >= c.shift && j < c.count) {
        if constexpr (DT == kF32) storeElem<4>(p, j, r.w[j / 4][j % 4]);
        else storeElem<2>(p, j, (r.w[0][j / 2] >> (16 * (j % 2))) & 0xffffu);
      }
  }
}
// Where the gradient rows of the tokens are whose payloads the lanes hold. A lane picks its source's pointer out of the
// kernel's arguments for itself, and the wave takes a token's address from its lane: a load of the pointer, scalar or
// not, would have to be waited for before the row's.
struct TokenRows {
  uint32_t lo, hi;
};
__device__ __forceinline__ TokenRows rowsOf(const GradArgs& a, uint32_t pay) {
  const char* base = a.grads[0];
#pragma unroll
  for (uint32_t r = 1; r < kMaxSrcs; r++) base = (pay >> kSrcShift) == r ? a.grads[r] : base;
  const uint64_t at = (uint64_t)(uintptr_t)base + (uint64_t)(pay & kTokenMask) * a.gradStride;
  return TokenRows{(uint32_t)at, (uint32_t)(at >> 32)};
}
__device__ __forceinline__ const char* rowOfLane(const TokenRows& r, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)r.lo, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)r.hi, lane);
  return (const char*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// acc += the gradients of the `count` tokens whose rows lanes from .. from + count - 1 hold, this lane's eight columns, in
// order. None of the loads is under a condition (the last few, less than AHEAD, repeat the last token's), or the compiler
// would wait for each by itself.
template <int GT, bool NARROW, int AHEAD>
__device__ __forceinline__ void addBatch(const TokenRows& rows, int from, int count, const Columns& c, float (&acc)[kVec]) {
  Raw8<GT> raw[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; i++) raw[i] = loadColumns<GT, NARROW>(rowOfLane(rows, from + (i < count ? i : count - 1)), c);
#pragma unroll
  for (int i = 0; i < AHEAD; i++)
    if (i < count) {
      float f[kVec];
      widen8<GT>(raw[i], f);
#pragma unroll
      for (int j = 0; j < kVec; j++) acc[j] += f[j];
    }
}
template <int GT, bool NARROW, int AHEAD>
__device__ __forceinline__ void addTokens(const TokenRows& rows, int from, int count, const Columns& c, float (&acc)[kVec]) {
  int p = 0;
  for (; p + AHEAD <= count; p += AHEAD) addBatch<GT, NARROW, AHEAD>(rows, from + p, AHEAD, c, acc);
  for (; p < count; p += 4) addBatch<GT, NARROW, 4>(rows, from + p, count - p < 4 ? count - p : 4, c, acc);
}
// acc += rows [begin, end) of fp32 scratch
__device__ __forceinline__ void addSums(const float* sums, uint32_t widthPad, uint32_t begin, uint32_t end, uint32_t slot,
                                        float (&acc)[kVec]) {
  if (slot >= widthPad) return;
  constexpr int kAhead = 8;
  for (uint32_t c = begin; c < end; c += kAhead) {
    Raw8<kF32> raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++)
      raw[i] = loadRaw8<kF32>((const char*)(sums + (size_t)(c + i < end ? c + i : end - 1) * widthPad + slot));
#pragma unroll
    for (int i = 0; i < kAhead; i++)
      if (c + i < end) {
        float f[kVec];
        widen8<kF32>(raw[i], f);
#pragma unroll
        for (int j = 0; j < kVec; j++) acc[j] += f[j];
      }
  }
}

// (twice as many take the registers of two waves per SIMD and gain nothing)
template <int GT>
constexpr int kTokensAhead = GT == kF32 ? 4 : 8;

// One wave per (chunk, piece): the chunk's sum if all of it belongs to one row. Chunks of 16 tokens and of 16 chunks: a run
// then ends in at most 15 tokens, 15 chunks on either side, so the wave that joins it waits for few loads in turn (with
// 32 and 32 the most frequent of 16384 tokens kept its wave for 20 us more).
template <int GT, bool NARROW>
__global__ __launch_bounds__(kRowThreads) void chunkKernel(GradArgs a, int sorted) {
  const int lane = (int)(threadIdx.x & 63);
  const uint32_t* keys = a.keys[sorted];
  const uint64_t items = (uint64_t)(a.n / kChunk) * a.pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * kRowWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kRowWaves) {
    const uint32_t chunk = (uint32_t)(item / a.pieces), piece = (uint32_t)(item % a.pieces), begin = chunk * kChunk;
    uint32_t mine = keys[begin + (lane & (kChunk - 1))], pays = a.pays[sorted][begin + (lane & (kChunk - 1))];
    DFCCL_LOADED(mine);
    DFCCL_LOADED(pays);
    const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)mine, 0);
    const uint32_t last = (uint32_t)__builtin_amdgcn_readlane((int)mine, kChunk - 1);
    if (key >= a.rows || last != key) continue;
    const Columns cols = columnsOf<NARROW>(a.width, piece, lane);
    float acc[kVec] = {};
    addTokens<GT, NARROW, kTokensAhead<GT>>(rowsOf(a, pays), 0, kChunk, cols, acc);
    if (cols.shift < kVec) store8<kF32>((char*)(a.chunkSums + (size_t)chunk * a.widthPad + cols.slot), acc);
  }
}
// One wave per (chunk of chunks, piece)
__global__ __launch_bounds__(kRowThreads) void superKernel(GradArgs a, int sorted) {
  const int lane = (int)(threadIdx.x & 63);
  const uint32_t* keys = a.keys[sorted];
  const uint64_t items = (uint64_t)(a.n / kSuperTokens) * a.pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * kRowWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kRowWaves) {
    const uint32_t super = (uint32_t)(item / a.pieces), piece = (uint32_t)(item % a.pieces);
    uint32_t first = keys[super * kSuperTokens], last = keys[super * kSuperTokens + kSuperTokens - 1];
    DFCCL_LOADED(first);
    DFCCL_LOADED(last);
    const uint32_t key = uniform(first);
    if (key >= a.rows || uniform(last) != key) continue;
    const uint32_t col = piece * kPieceElems + lane * kVec;
    float acc[kVec] = {};
    addSums(a.chunkSums, a.widthPad, super * kSuper, (super + 1) * kSuper, col, acc);
    if (col < a.widthPad) store8<kF32>((char*)(a.superSums + (size_t)super * a.widthPad + col), acc);
  }
}

// The end of a run that is known to reach `lo`: the keys are sorted, so 64 lanes look at 64 places between lo and hi
// and the search goes on between two of them.
__device__ __forceinline__ uint32_t endOfRun(const uint32_t* keys, uint32_t key, uint32_t lo, uint32_t hi, int lane) {
  while (lo < hi) {
    const uint32_t step = (hi - lo + 63) / 64;
    const uint64_t at = (uint64_t)lo + (uint64_t)lane * step;
    const int in = __builtin_popcountll(__ballot(at < hi && keys[at < hi ? at : lo] == key));
    if (in == 0) break;  // (the run ends at lo)
    const uint64_t next = (uint64_t)lo + (uint64_t)in * step;
    lo += (uint32_t)(in - 1) * step + 1;
    if (next < hi) hi = (uint32_t)next;
  }
  return lo;
}

// One wave per (group of kGroup sorted positions, piece): the runs that begin in the group. A lane each reads the keys
// from the one before the group on and the payloads from the group's first on, so after one load it is known where
// runs begin and end and whom they sum; then the group's rows (and the table's, if they are added to) are in flight
// together. Only the group's last run may go on behind it. Bound by HBM where the table is large: it reads and writes
// the rows (190 MB of them in 55 us at 16384 tokens) while the 256 MB of cleared rows that the last cache level still
// holds are written back. Four positions a wave: 55 us, two 68; a position a wave, with the lanes' loads one after the
// other: 71.
constexpr int kGroup = 4;
static_assert(kChunk % kGroup == 0, "a group lies within one chunk");

template <int GT, int TT, bool ADD, bool NARROW>
__global__ __launch_bounds__(kRowThreads) void rowsKernel(GradArgs a, int sorted) {
  const int lane = (int)(threadIdx.x & 63);
  const uint32_t *keys = a.keys[sorted], *pays = a.pays[sorted];
  const uint64_t items = (uint64_t)((a.n + (kGroup - 1)) / kGroup) * a.pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * kRowWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kRowWaves) {
    const uint64_t group = item / a.pieces;
    const Columns cols = columnsOf<NARROW>(a.width, (uint32_t)(item - group * a.pieces), lane);
    const uint32_t p0 = (uint32_t)group * kGroup;
    const uint64_t at = (uint64_t)p0 + (uint32_t)lane;
    uint32_t window = at >= 1 && at - 1 < a.n ? keys[at - 1] : a.rows;  // lane l: position p0 - 1 + l
    uint32_t mine = at < a.n ? pays[at] : 0;                            // lane l: position p0 + l
    DFCCL_LOADED(window);
    DFCCL_LOADED(mine);
    uint32_t key[kGroup + 1];
    bool begins[kGroup], ours[kGroup];  // ours: of a run that begins in the group
    uint32_t before = (uint32_t)__builtin_amdgcn_readlane((int)window, 0);
    bool any = false;
#pragma unroll
    for (int i = 0; i <= kGroup; i++) key[i] = (uint32_t)__builtin_amdgcn_readlane((int)window, i + 1);
#pragma unroll
    for (int i = 0; i < kGroup; i++) {
      begins[i] = key[i] < a.rows && key[i] != before;
      ours[i] = begins[i] || (any && key[i] < a.rows);  // (a run that began in the group goes on, or another begins)
      any = any || begins[i];
      before = key[i];
    }
    if (!any) continue;
    // Positions that are not ours load what the first one that begins a run does (nothing is under a condition: see
    // addBatch), and every sum is complete before the first is stored: loads and stores are counted together, and a
    // wait for a load behind a store is one for the store.
    int some = 0;
    uint32_t someKey = 0;
#pragma unroll
    for (int i = kGroup - 1; i >= 0; i--)
      if (begins[i]) {
        some = i;
        someKey = key[i];
      }
    const TokenRows tokens = rowsOf(a, mine);
    Raw8<GT> raw[kGroup];
    Raw8<TT> old[kGroup], out[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; i++) raw[i] = loadColumns<GT, NARROW>(rowOfLane(tokens, ours[i] ? i : some), cols);
    if constexpr (ADD) {
#pragma unroll
      for (int i = 0; i < kGroup; i++)
        old[i] = loadColumns<TT, NARROW>(a.table + (size_t)(begins[i] ? key[i] : someKey) * a.tableStride, cols);
    }
    float acc[kVec] = {}, was[kVec] = {};
    bool ends[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; i++) {
      float f[kVec];
      widen8<GT>(raw[i], f);
#pragma unroll
      for (int j = 0; j < kVec; j++) acc[j] = begins[i] ? f[j] : acc[j] + f[j];
      if constexpr (ADD) {
        widen8<TT>(old[i], f);
#pragma unroll
        for (int j = 0; j < kVec; j++) was[j] = begins[i] ? f[j] : was[j];
      }
      ends[i] = ours[i] && (i == kGroup - 1 || key[i + 1] != key[i]);
      if (i == kGroup - 1 && ours[i] && key[i + 1] == key[i]) {
        // The group's last run goes on. It began at `pos`, its end is in sight unless it is long.
        uint32_t pos = p0;
#pragma unroll
        for (int k = 1; k < kGroup; k++)
          if (begins[k]) pos = p0 + k;
        const uint64_t same = __ballot(window == key[i]) >> 1;  // bit b: position p0 + b
        const uint64_t on = ~(same >> kGroup);                  // (bits 63 - kGroup and up are out of sight: set)
        uint32_t end = p0 + kGroup + (uint32_t)__builtin_ctzll(on);
        if (end == p0 + 63) end = endOfRun(keys, key[i], end, a.n, lane);
        const uint32_t c0 = (pos + kChunk - 1) / kChunk, c1 = end / kChunk;
        if (!a.chunked || c0 >= c1) {  // (then it ends within the 64 positions whose payloads are here)
          addTokens<GT, NARROW, kTokensAhead<GT>>(tokens, kGroup, (int)(end - p0) - kGroup, cols, acc);
        } else {
          const uint64_t behind = (uint64_t)c1 * kChunk + (uint32_t)lane;
          const uint32_t rest = behind < end ? pays[behind] : 0;
          if (c0 * kChunk == pos) {  // the chunk's sum has the group's tokens, too
#pragma unroll
            for (int j = 0; j < kVec; j++) acc[j] = 0.0f;
          } else {
            addTokens<GT, NARROW, kTokensAhead<GT>>(tokens, kGroup, (int)(c0 * kChunk - p0) - kGroup, cols, acc);
          }
          const uint32_t s0 = (c0 + kSuper - 1) / kSuper, s1 = c1 / kSuper;
          if (!a.supered || s0 >= s1) {
            addSums(a.chunkSums, a.widthPad, c0, c1, cols.slot, acc);
          } else {
            addSums(a.chunkSums, a.widthPad, c0, s0 * kSuper, cols.slot, acc);
            addSums(a.superSums, a.widthPad, s0, s1, cols.slot, acc);
            addSums(a.chunkSums, a.widthPad, s1 * kSuper, c1, cols.slot, acc);
          }
          addTokens<GT, NARROW, kTokensAhead<GT>>(rowsOf(a, rest), 0, (int)(end - c1 * kChunk), cols, acc);
        }
      }
      float sum[kVec];
#pragma unroll
      for (int j = 0; j < kVec; j++) sum[j] = ADD ? was[j] + acc[j] * a.scale : acc[j] * a.scale;
      out[i] = narrow8<TT>(sum);
    }
#pragma unroll
    for (int i = 0; i < kGroup; i++)
      if (ends[i]) storeColumns<TT, NARROW>(a.table + (size_t)key[i] * a.tableStride, cols, out[i]);
  }
}

typedef void (*SortKernel)(GradArgs, SortPass, Clear);
template <int S, bool FIRST>
static SortKernel pickSortS(bool scatter) {
  return scatter ? sortScatterKernel<S, FIRST> : sortCountKernel<S, FIRST>;
}
static SortKernel pickSort(bool scatter, int strips, bool first) {
  if (strips == 2) return first ? pickSortS<2, true>(scatter) : pickSortS<2, false>(scatter);
  if (strips == 4) return first ? pickSortS<4, true>(scatter) : pickSortS<4, false>(scatter);
  return first ? pickSortS<16, true>(scatter) : pickSortS<16, false>(scatter);
}
typedef void (*RowsKernel)(GradArgs, int);
template <bool NARROW>
static RowsKernel pickChunkN(int gt) {
  return gt == kF32 ? chunkKernel<kF32, NARROW> : gt == kF16 ? chunkKernel<kF16, NARROW> : chunkKernel<kBF16, NARROW>;
}
static RowsKernel pickChunk(int gt, bool narrow) { return narrow ? pickChunkN<true>(gt) : pickChunkN<false>(gt); }
template <int GT, bool ADD, bool NARROW>
static RowsKernel pickRowsT(int tt) {
  return tt == kF32   ? rowsKernel<GT, kF32, ADD, NARROW>
         : tt == kF16 ? rowsKernel<GT, kF16, ADD, NARROW>
                      : rowsKernel<GT, kBF16, ADD, NARROW>;
}
template <bool ADD, bool NARROW>
static RowsKernel pickRowsG(int gt, int tt) {
  return gt == kF32   ? pickRowsT<kF32, ADD, NARROW>(tt)
         : gt == kF16 ? pickRowsT<kF16, ADD, NARROW>(tt)
                      : pickRowsT<kBF16, ADD, NARROW>(tt);
}
static RowsKernel pickRows(int gt, int tt, bool accumulate, bool narrow) {
  if (narrow) return accumulate ? pickRowsG<true, true>(gt, tt) : pickRowsG<false, true>(gt, tt);
  return accumulate ? pickRowsG<true, false>(gt, tt) : pickRowsG<false, false>(gt, tt);
}

// Plan of a gradient call from its sizes: how it is sorted and where the workspace's parts begin.
struct GradPlan {
  bool small, chunked, supered;
  int keyBits, passes, digitBits, strips, tiles;
  size_t keys[2], pays[2], hist, chunkSums, superSums, bytes;
};
static GradPlan planGrad(uint64_t n, size_t rows, size_t width) {
  GradPlan p{};
  p.keyBits = 1;
  while (p.keyBits < 32 && ((uint64_t)rows >> p.keyBits) != 0) p.keyBits++;  // keys are 0 .. rows
  p.small = n <= kSmallMax;
  p.passes = (p.keyBits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digitBits = (p.keyBits + p.passes - 1) / p.passes;
  p.strips = stripsOf(n);
  const uint64_t tile = (uint64_t)kSortThreads * p.strips;
  p.tiles = (int)std::max<uint64_t>(1, (n + tile - 1) / tile);
  // Runs of fewer than 64 tokens need no chunks. Chunks of chunks pay for their launch once a run may have several
  // hundred chunks.
  p.chunked = n >= 64;
  p.supered = n >= kSuperMin;
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  const size_t widthPad = (width + kVec - 1) / kVec * kVec;
  for (int i = 0; i < (p.small ? 1 : 2); i++) {
    p.keys[i] = take(n * 4);
    p.pays[i] = take(n * 4);
  }
  if (!p.small) p.hist = take(((size_t)p.tiles << p.digitBits) * 4);
  if (p.chunked) p.chunkSums = take(n / kChunk * widthPad * 4);
  if (p.supered) p.superSums = take(n / kSuperTokens * widthPad * 4);
  p.bytes = std::max<size_t>(at, 256);
  return p;
}

// rows and widths stay below 2^31 and rows * pieces, tokens * pieces below 2^63
static bool gradSizes(int nsrcs, const size_t* tokens, size_t rows, size_t width, uint64_t* n) {
  if (nsrcs < 1 || nsrcs > kMaxSrcs || tokens == nullptr) return false;
  if (rows > 0x7ffffffeull || width > 0x7ffffff0ull) return false;
  *n = 0;
  for (int r = 0; r < nsrcs; r++) {
    if (tokens[r] > kTokenMask) return false;
    *n += tokens[r];
  }
  return *n <= 0x7fffffffull;
}

}  // namespace dfccl

using namespace dfccl;

#define DFCCL_API extern "C" __attribute__((visibility("default")))

DFCCL_API ncclResult_t dfcclEmbeddingLookup(const void* table, ncclDataType_t tableType, size_t rows, size_t tableStride,
                                            int64_t firstRow, const void* ids, ncclDataType_t idType, size_t tokens,
                                            size_t width, double scale, void* out, ncclDataType_t outType,
                                            size_t outStride, void* stream) {
  if (!rowType((int)tableType) || !rowType((int)outType)) return ncclInvalidArgument;
  if (idType != ncclInt32 && idType != ncclInt64) return ncclInvalidArgument;
  if (rows > 0x7ffffffeull || width > 0x7ffffff0ull || tokens > 0x7fffffffull) return ncclInvalidArgument;
  if (tableStride < width || outStride < width || firstRow < 0) return ncclInvalidArgument;
  if (tokens == 0 || width == 0) return ncclSuccess;
  if ((table == nullptr && rows > 0) || ids == nullptr || out == nullptr) return ncclInvalidArgument;
  LookupArgs a{};
  a.table = (const char*)table;
  a.ids = (const char*)ids;
  a.out = (char*)out;
  a.firstRow = firstRow;
  a.rows = (int64_t)rows;
  a.tableStride = tableStride * typeSize((int)tableType);
  a.outStride = outStride * typeSize((int)outType);
  a.tokens = tokens;
  a.width = (uint32_t)width;
  a.pieces = (uint32_t)((width + kPieceElems - 1) / kPieceElems);
  a.idBytes = idType == ncclInt64 ? 8 : 4;
  a.scale = (float)scale;
  constexpr int U = 2;
  // two rows a wave once that still fills the chip (256 CUs, 32 waves each), see lookupKernel; below, one row a wave:
  // a few rows are bound by latency, which more waves with less each hide better
  const bool many = (uint64_t)tokens * a.pieces >= (uint64_t)U * 256 * 32;
  const uint64_t waves = (uint64_t)((tokens + (many ? U : 1) - 1) / (many ? U : 1)) * a.pieces;
  LookupKernel fn = many ? pickLookup<U>((int)tableType, (int)outType) : pickLookup<1>((int)tableType, (int)outType);
  DFCCL_LAUNCH_BLOCKS(fn, gridFor(waves), kRowThreads, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? ncclSuccess : ncclUnhandledCudaError;
}

DFCCL_API ncclResult_t dfcclEmbeddingGradWorkspace(int nsrcs, const size_t* tokens, size_t rows, size_t width,
                                                   size_t* bytes) {
  uint64_t n = 0;
  if (bytes == nullptr || !gradSizes(nsrcs, tokens, rows, width, &n)) return ncclInvalidArgument;
  *bytes = planGrad(n, rows, width).bytes;
  return ncclSuccess;
}

DFCCL_API ncclResult_t dfcclEmbeddingGrad(const void* const* grads, const void* const* ids, const size_t* tokens, int nsrcs,
                                          ncclDataType_t gradType, size_t gradStride, ncclDataType_t idType,
                                          int64_t firstRow, size_t rows, size_t width, int64_t paddingId, double scale,
                                          int accumulate, void* tableGrad, ncclDataType_t tableType, size_t tableStride,
                                          void* workspace, size_t workspaceBytes, void* stream) {
  uint64_t n = 0;
  if (!rowType((int)gradType) || !rowType((int)tableType)) return ncclInvalidArgument;
  if (idType != ncclInt32 && idType != ncclInt64) return ncclInvalidArgument;
  if (!gradSizes(nsrcs, tokens, rows, width, &n)) return ncclInvalidArgument;
  if (gradStride < width || tableStride < width || firstRow < 0) return ncclInvalidArgument;
  if (grads == nullptr || ids == nullptr) return ncclInvalidArgument;
  for (int r = 0; r < nsrcs; r++)
    if (tokens[r] > 0 && width > 0 && (grads[r] == nullptr || ids[r] == nullptr)) return ncclInvalidArgument;
  if (rows == 0 || width == 0 || (accumulate && n == 0)) return ncclSuccess;
  if (tableGrad == nullptr) return ncclInvalidArgument;
  const GradPlan p = planGrad(n, rows, width);
  if (workspace == nullptr || workspaceBytes < p.bytes || ((uintptr_t)workspace & 15u) != 0) return ncclInvalidArgument;
  GradArgs a{};
  uint32_t at = 0;
  for (int r = 0; r < kMaxSrcs; r++) {
    a.grads[r] = r < nsrcs ? (const char*)grads[r] : nullptr;
    a.ids[r] = r < nsrcs ? (const char*)ids[r] : nullptr;
    a.firstPos[r] = at;
    if (r < nsrcs) at += (uint32_t)tokens[r];
  }
  a.firstPos[kMaxSrcs] = at;
  a.nsrcs = nsrcs;
  a.idBytes = idType == ncclInt64 ? 8 : 4;
  a.gradStride = gradStride * typeSize((int)gradType);
  a.tableStride = tableStride * typeSize((int)tableType);
  a.firstRow = firstRow;
  a.paddingId = paddingId;
  a.rows = (uint32_t)rows;
  a.width = (uint32_t)width;
  a.pieces = (uint32_t)((width + kPieceElems - 1) / kPieceElems);
  a.n = (uint32_t)n;
  a.scale = (float)scale;
  a.table = (char*)tableGrad;
  char* ws = (char*)workspace;
  for (int i = 0; i < 2; i++) {
    a.keys[i] = (uint32_t*)(ws + p.keys[i]);
    a.pays[i] = (uint32_t*)(ws + p.pays[i]);
  }
  a.chunked = p.chunked;
  a.supered = p.supered;
  a.hist = (uint32_t*)(ws + p.hist);
  a.chunkSums = (float*)(ws + p.chunkSums);
  a.superSums = (float*)(ws + p.superSums);
  a.widthPad = (uint32_t)((width + kVec - 1) / kVec * kVec);

  // the table's clearing, in equal shares over the launches of the sort
  const bool narrow = width < kVec;
  const uint32_t sortWaves = p.small ? kSmallWaves : kSortWaves;
  const int launches = p.small ? 1 : 2 * p.passes;
  Clear clear{};
  uint64_t clearParts = 0;
  if (!accumulate) {
    const size_t rowBytes = width * typeSize((int)tableType);
    clear.at = a.table;
    if (a.tableStride == rowBytes) {
      clear.bytes = (uint64_t)rowBytes * rows;
      clearParts = (clear.bytes + clearPart(sortWaves) - 1) / clearPart(sortWaves);
    } else {
      clear.stride = a.tableStride;
      clear.bytes = rowBytes;
      clear.rowParts = (rowBytes + kGapBytes - 1) / kGapBytes;
      clearParts = clear.rowParts * rows;
    }
  }
  int launch = 0;
  // the share of the next launch, whose own work takes `blocks` workgroups; returns the launch's grid
  auto share = [&](unsigned blocks) {
    clear.begin = clearParts * launch / launches;
    clear.end = clearParts * (launch + 1) / launches;
    clear.firstBlock = blocks;
    launch++;
    const uint64_t parts = clear.end - clear.begin, want = clear.stride == 0 ? parts : (parts + sortWaves - 1) / sortWaves;
    return blocks + (unsigned)std::min<uint64_t>(want, p.small ? 256 : kMaxGrid);
  };
  const hipStream_t st = (hipStream_t)stream;
  int from = 0;
  if (p.small) {
    const unsigned grid = share(1);
    DFCCL_LAUNCH_BLOCKS(sortSmallKernel, grid, kSmallThreads, st, a, p.keyBits, clear);
  }
  for (int pass = 0; !p.small && pass < p.passes; pass++, from ^= 1) {
    const SortPass s{from, pass * p.digitBits, p.digitBits, p.tiles};
    for (int scatter = 0; scatter < 2; scatter++) {
      const unsigned grid = share((unsigned)p.tiles);
      DFCCL_LAUNCH_BLOCKS(pickSort(scatter != 0, p.strips, pass == 0), grid, kSortThreads, st, a, s, clear);
    }
  }
  if (p.chunked)
    DFCCL_LAUNCH_BLOCKS(pickChunk((int)gradType, narrow), gridFor(n / kChunk * a.pieces), kRowThreads, st, a, from);
  if (p.supered)
    DFCCL_LAUNCH_BLOCKS(superKernel, gridFor(n / kSuperTokens * a.pieces), kRowThreads, st, a, from);
  if (n > 0)
    DFCCL_LAUNCH_BLOCKS(pickRows((int)gradType, (int)tableType, accumulate != 0, narrow),
                        gridFor((n + kGroup - 1) / kGroup * a.pieces), kRowThreads, st, a, from);
  return hipGetLastError() == hipSuccess ? ncclSuccess : ncclUnhandledCudaError;
}

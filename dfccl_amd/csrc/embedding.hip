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

// One wave takes one piece (512 elements) of U tokens' rows: the U ids, then the U loads are in flight together.
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
        store8<OUT>(a.out + (t0 + u) * a.outStride + (size_t)col * typeSize(OUT), f);
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
//    puts equal keys side by side in the order source, token: the order of every sum is fixed by the ids alone.
// 2. Chunks. The sorted list is cut into chunks of kChunk. A chunk that lies within one row's run is summed by a
//    wave of its own into fp32 scratch, and so are kChunk such chunks: a row that many tokens share (padding that
//    counts, frequent words) is summed by many waves, and again in a fixed order.
// 3. Rows. A wave per row piece adds up its run: single tokens up to the first whole chunk, whole chunks' (and
//    chunks of chunks') sums, single tokens after the last. Each row is written once; a row without tokens gets
//    zeros (or is left alone when accumulating).

constexpr int kChunk = 32;
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
  char* table;
  // workspace
  uint32_t* keys[2];
  uint32_t* pays[2];
  uint32_t* hist;      // [tiles][bins]
  int32_t* rowBegin;   // position of a row's first token in the sorted list, -1 without one
  uint32_t* rowEnd;    // behind its last
  float* chunkSums;    // [n / kChunk][widthPad]
  float* superSums;    // [n / kChunk^2][widthPad]
  uint32_t widthPad;   // width rounded up to kVec
};

struct SortPass {
  int from, shift, bits, tiles;  // keys[from] -> keys[from ^ 1]
};

__device__ __forceinline__ void keyOfToken(const GradArgs& a, uint32_t pos, uint32_t& key, uint32_t& pay) {
  int r = 0;
  const char* ids = a.ids[0];
  uint32_t first = 0;
#pragma unroll
  for (int i = 1; i < kMaxSrcs; i++)
    if (i < a.nsrcs && pos >= a.firstPos[i]) {
      r = i;
      ids = a.ids[i];
      first = a.firstPos[i];
    }
  const uint32_t t = pos - first;
  const int64_t id = loadId(ids, a.idBytes, t), row = rowOf(id, a.firstRow, a.rows);
  key = row >= 0 && id != a.paddingId ? (uint32_t)row : a.rows;
  pay = ((uint32_t)r << kSrcShift) | t;
}

constexpr int kSortThreads = 256;
constexpr int kSortWaves = kSortThreads / 64;
// positions of a tile: short enough that a few thousand tokens spread over several workgroups, long enough that
// the sum over the tiles' histograms, which every tile makes for itself, stays short
constexpr int kShortStrips = 4, kLongStrips = 16;

// Digit counts of every tile; the first pass also clears the rows' index with the workgroups behind the tiles.
template <int S, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sortCountKernel(GradArgs a, SortPass p) {
  struct Shared {
    uint32_t count[kMaxBins];
  };
  DFCCL_WG_SHARED(Shared, sh);
  const int tid = (int)threadIdx.x, tile = (int)blockIdx.x, bins = 1 << p.bits;
  if (FIRST && tile >= p.tiles) {
    for (uint64_t i = (uint64_t)(tile - p.tiles) * kSortThreads + tid; i < a.rows;
         i += (uint64_t)(gridDim.x - p.tiles) * kSortThreads)
      a.rowBegin[i] = -1;
    return;
  }
  for (int i = tid; i < bins; i += kSortThreads) sh.count[i] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < S; k++) {
    const uint64_t pos = (uint64_t)tile * (kSortThreads * S) + k * kSortThreads + tid;
    if (pos < a.n) {
      uint32_t key, pay;
      if constexpr (FIRST) keyOfToken(a, (uint32_t)pos, key, pay);
      else key = a.keys[p.from][pos];
      __hip_atomic_fetch_add(&sh.count[(key >> p.shift) & (bins - 1)], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
  __syncthreads();
  for (int i = tid; i < bins; i += kSortThreads) a.hist[(size_t)tile * bins + i] = sh.count[i];
}

// Stable scatter of a tile. A lane's rank among the tile's keys of the same digit: the equal digits of the waves
// before, of this wave's strips before, and of the lanes before it in its strip (found with a ballot per bit).
template <int S, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sortScatterKernel(GradArgs a, SortPass p) {
  struct Shared {
    uint32_t count[kSortWaves][kMaxBins];
    uint32_t base[kMaxBins];
    uint32_t total[kMaxBins];
    uint32_t waveTotal[kSortWaves];
  };
  DFCCL_WG_SHARED(Shared, sh);
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = waveInBlock(), tile = (int)blockIdx.x, bins = 1 << p.bits;
  for (int i = tid; i < kSortWaves * kMaxBins; i += kSortThreads) sh.count[i / kMaxBins][i % kMaxBins] = 0;
  __syncthreads();
  uint32_t key[S], pay[S], rank[S];
  const uint64_t start = (uint64_t)tile * (kSortThreads * S) + (uint64_t)wave * (64 * S) + lane;
#pragma unroll
  for (int k = 0; k < S; k++) {
    const uint64_t pos = start + k * 64;
    key[k] = pay[k] = 0;
    if (pos < a.n) {
      if constexpr (FIRST) keyOfToken(a, (uint32_t)pos, key[k], pay[k]);
      else {
        key[k] = a.keys[p.from][pos];
        pay[k] = a.pays[p.from][pos];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < S; k++) {
    const bool valid = start + k * 64 < a.n;
    const uint32_t d = (key[k] >> p.shift) & (uint32_t)(bins - 1);
    uint64_t same = __ballot(valid);
    for (int b = 0; b < p.bits; b++) {
      const bool one = (d >> b) & 1u;
      const uint64_t ones = __ballot(one);
      same &= one ? ones : ~ones;
    }
    const uint64_t before = same & ((1ull << lane) - 1);
    const uint32_t old = sh.count[wave][d];
    DFCCL_WAVE_LDS_SYNC();  // (every lane has read the count before the first of its digit raises it)
    if (valid && before == 0) sh.count[wave][d] = old + (uint32_t)__builtin_popcountll(same);
    DFCCL_WAVE_LDS_SYNC();
    rank[k] = old + (uint32_t)__builtin_popcountll(before);
  }
  // where the tile's keys of each digit begin: all keys of smaller digits, then this digit's in the tiles before
  for (int i = tid; i < kMaxBins; i += kSortThreads) {
    uint32_t before = 0, total = 0;
    if (i < bins)
      for (int t = 0; t < p.tiles; t++) {
        const uint32_t h = a.hist[(size_t)t * bins + i];
        before += t < tile ? h : 0;
        total += h;
      }
    sh.base[i] = before;
    sh.total[i] = total;
  }
  __syncthreads();
  constexpr int per = kMaxBins / kSortThreads;
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < per; i++) mine += sh.total[tid * per + i];
  uint32_t sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t from = __shfl(sum, (lane - d) & 63);
    if (lane >= d) sum += from;
  }
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
      const uint32_t c = sh.count[w][bin];
      sh.count[w][bin] = next;
      next += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < S; k++)
    if (start + k * 64 < a.n) {
      const uint32_t to = sh.count[wave][(key[k] >> p.shift) & (uint32_t)(bins - 1)] + rank[k];
      a.keys[p.from ^ 1][to] = key[k];
      a.pays[p.from ^ 1][to] = pay[k];
    }
}

// acc += the gradients of sorted positions [begin, end), this lane's eight columns, in order; eight loads in flight
template <int GT>
__device__ __forceinline__ void addTokens(const GradArgs& a, const uint32_t* pays, uint32_t begin, uint32_t end,
                                          uint32_t col, float (&acc)[kVec]) {
  constexpr int kAhead = 8;
  const bool full = col + kVec <= a.width;
  const int left = (int)a.width - (int)col;
  for (uint32_t p = begin; p < end; p += kAhead) {
    Raw8<GT> raw[kAhead];
    if (full) {
#pragma unroll
      for (int i = 0; i < kAhead; i++)
        if (p + i < end) {
          const uint32_t pay = uniform(pays[p + i]);
          raw[i] = loadRaw8<GT>(a.grads[pay >> kSrcShift] + (size_t)(pay & kTokenMask) * a.gradStride +
                                (size_t)col * typeSize(GT));
        }
#pragma unroll
      for (int i = 0; i < kAhead; i++)
        if (p + i < end) {
          float f[kVec];
          widen8<GT>(raw[i], f);
#pragma unroll
          for (int j = 0; j < kVec; j++) acc[j] += f[j];
        }
    } else if (left > 0) {
      for (int i = 0; i < kAhead && p + i < end; i++) {
        const uint32_t pay = uniform(pays[p + i]);
        float f[kVec];
        loadTail<GT>(a.grads[pay >> kSrcShift] + (size_t)(pay & kTokenMask) * a.gradStride + (size_t)col * typeSize(GT),
                     left, f);
#pragma unroll
        for (int j = 0; j < kVec; j++) acc[j] += f[j];
      }
    }
  }
}
// acc += rows [begin, end) of fp32 scratch
__device__ __forceinline__ void addSums(const float* sums, uint32_t widthPad, uint32_t begin, uint32_t end, uint32_t col,
                                        float (&acc)[kVec]) {
  if (col >= widthPad) return;
  constexpr int kAhead = 4;
  for (uint32_t c = begin; c < end; c += kAhead) {
    Raw8<kF32> raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++)
      if (c + i < end) raw[i] = loadRaw8<kF32>((const char*)(sums + (size_t)(c + i) * widthPad + col));
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

// One wave per (chunk, piece): the chunk's sum if all of it belongs to one row; the first piece's waves also note
// where rows begin and end.
template <int GT>
__global__ __launch_bounds__(kRowThreads) void chunkKernel(GradArgs a, int sorted) {
  const int lane = (int)(threadIdx.x & 63);
  const uint32_t* keys = a.keys[sorted];
  const uint32_t chunks = (a.n + kChunk - 1) / kChunk;
  const uint64_t items = (uint64_t)chunks * a.pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * kRowWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kRowWaves) {
    const uint32_t chunk = (uint32_t)(item / a.pieces), piece = (uint32_t)(item % a.pieces), begin = chunk * kChunk;
    if (piece == 0 && lane < kChunk && begin + lane < a.n) {
      const uint32_t pos = begin + lane, key = keys[pos];
      if (key < a.rows) {
        if (pos == 0 || keys[pos - 1] != key) a.rowBegin[key] = (int32_t)pos;
        if (pos + 1 == a.n || keys[pos + 1] != key) a.rowEnd[key] = pos + 1;
      }
    }
    if (a.n - begin < kChunk) continue;
    const uint32_t key = uniform(keys[begin]);
    if (key >= a.rows || uniform(keys[begin + kChunk - 1]) != key) continue;
    const uint32_t col = piece * kPieceElems + lane * kVec;
    float acc[kVec] = {};
    addTokens<GT>(a, a.pays[sorted], begin, begin + kChunk, col, acc);
    if (col < a.widthPad) store8<kF32>((char*)(a.chunkSums + (size_t)chunk * a.widthPad + col), acc);
  }
}
// One wave per (chunk of chunks, piece)
__global__ __launch_bounds__(kRowThreads) void superKernel(GradArgs a, int sorted) {
  const int lane = (int)(threadIdx.x & 63);
  const uint32_t* keys = a.keys[sorted];
  const uint32_t supers = a.n / (kChunk * kChunk);
  const uint64_t items = (uint64_t)supers * a.pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * kRowWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kRowWaves) {
    const uint32_t super = (uint32_t)(item / a.pieces), piece = (uint32_t)(item % a.pieces);
    const uint32_t begin = super * (kChunk * kChunk), key = uniform(keys[begin]);
    if (key >= a.rows || uniform(keys[begin + kChunk * kChunk - 1]) != key) continue;
    const uint32_t col = piece * kPieceElems + lane * kVec;
    float acc[kVec] = {};
    addSums(a.chunkSums, a.widthPad, super * kChunk, (super + 1) * kChunk, col, acc);
    if (col < a.widthPad) store8<kF32>((char*)(a.superSums + (size_t)super * a.widthPad + col), acc);
  }
}

// acc = the sum of a row's run [begin, end)
template <int GT>
__device__ __forceinline__ void sumRun(const GradArgs& a, const uint32_t* pays, uint32_t begin, uint32_t end, uint32_t col,
                                       float (&acc)[kVec]) {
  const uint32_t c0 = (begin + kChunk - 1) / kChunk, c1 = end / kChunk;
  if (c0 >= c1) {
    addTokens<GT>(a, pays, begin, end, col, acc);
    return;
  }
  addTokens<GT>(a, pays, begin, c0 * kChunk, col, acc);
  const uint32_t s0 = (c0 + kChunk - 1) / kChunk, s1 = c1 / kChunk;
  if (s0 >= s1) {
    addSums(a.chunkSums, a.widthPad, c0, c1, col, acc);
  } else {
    addSums(a.chunkSums, a.widthPad, c0, s0 * kChunk, col, acc);
    addSums(a.superSums, a.widthPad, s0, s1, col, acc);
    addSums(a.chunkSums, a.widthPad, s1 * kChunk, c1, col, acc);
  }
  addTokens<GT>(a, pays, c1 * kChunk, end, col, acc);
}

template <int TT>
__device__ __forceinline__ void writeRow(const GradArgs& a, uint32_t row, uint32_t col, bool accumulate, float (&acc)[kVec]) {
  char* to = a.table + (size_t)row * a.tableStride + (size_t)col * typeSize(TT);
  const int left = (int)a.width - (int)col;
#pragma unroll
  for (int j = 0; j < kVec; j++) acc[j] *= a.scale;
  if (left >= kVec) {
    if (accumulate) {
      float old[kVec];
      widen8<TT>(loadRaw8<TT>(to), old);
#pragma unroll
      for (int j = 0; j < kVec; j++) acc[j] += old[j];
    }
    store8<TT>(to, acc);
  } else if (left > 0) {
    if (accumulate) {
      float old[kVec];
      loadTail<TT>(to, left, old);
#pragma unroll
      for (int j = 0; j < kVec; j++) acc[j] += old[j];
    }
    storeTail<TT>(to, left, acc);
  }
}

// Every row of the piece: kRowsPerWave rows' index is read at once.
constexpr int kRowsPerWave = 4;
template <int GT, int TT>
__global__ __launch_bounds__(kRowThreads) void denseRowsKernel(GradArgs a, int sorted) {
  const int lane = (int)(threadIdx.x & 63);
  const uint64_t groups = ((uint64_t)a.rows + kRowsPerWave - 1) / kRowsPerWave, items = groups * a.pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * kRowWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kRowWaves) {
    const uint64_t row0 = item / a.pieces * kRowsPerWave;
    const uint32_t col = (uint32_t)(item % a.pieces) * kPieceElems + (uint32_t)lane * kVec;
    int32_t begin[kRowsPerWave];
#pragma unroll
    for (int i = 0; i < kRowsPerWave; i++) begin[i] = row0 + i < a.rows ? uniform(a.rowBegin[row0 + i]) : -1;
#pragma unroll
    for (int i = 0; i < kRowsPerWave; i++) {
      if (row0 + i >= a.rows) break;
      float acc[kVec] = {};
      if (begin[i] >= 0) sumRun<GT>(a, a.pays[sorted], (uint32_t)begin[i], uniform(a.rowEnd[row0 + i]), col, acc);
      writeRow<TT>(a, (uint32_t)(row0 + i), col, false, acc);
    }
  }
}
// The rows that tokens name: a wave per (position, piece) that goes on where its position begins a run.
template <int GT, int TT>
__global__ __launch_bounds__(kRowThreads) void namedRowsKernel(GradArgs a, int sorted) {
  const int lane = (int)(threadIdx.x & 63);
  const uint32_t* keys = a.keys[sorted];
  const uint64_t items = (uint64_t)a.n * a.pieces;
  for (uint64_t item = (uint64_t)blockIdx.x * kRowWaves + waveInBlock(); item < items;
       item += (uint64_t)gridDim.x * kRowWaves) {
    const uint32_t pos = (uint32_t)(item / a.pieces), key = uniform(keys[pos]);
    if (key >= a.rows || (pos > 0 && uniform(keys[pos - 1]) == key)) continue;
    const uint32_t col = (uint32_t)(item % a.pieces) * kPieceElems + (uint32_t)lane * kVec;
    float acc[kVec] = {};
    sumRun<GT>(a, a.pays[sorted], pos, uniform(a.rowEnd[key]), col, acc);
    writeRow<TT>(a, key, col, true, acc);
  }
}

typedef void (*GradKernel)(GradArgs, int);
static GradKernel pickChunk(int gt) {
  return gt == kF32 ? chunkKernel<kF32> : gt == kF16 ? chunkKernel<kF16> : chunkKernel<kBF16>;
}
template <int GT>
static GradKernel pickRowsT(int tt, bool accumulate) {
  if (accumulate)
    return tt == kF32 ? namedRowsKernel<GT, kF32> : tt == kF16 ? namedRowsKernel<GT, kF16> : namedRowsKernel<GT, kBF16>;
  return tt == kF32 ? denseRowsKernel<GT, kF32> : tt == kF16 ? denseRowsKernel<GT, kF16> : denseRowsKernel<GT, kBF16>;
}
static GradKernel pickRows(int gt, int tt, bool accumulate) {
  return gt == kF32 ? pickRowsT<kF32>(tt, accumulate) : gt == kF16 ? pickRowsT<kF16>(tt, accumulate) : pickRowsT<kBF16>(tt, accumulate);
}

// Plan of a gradient call from its sizes: digits, tiles and where the workspace's parts begin.
struct GradPlan {
  int passes, digitBits, tiles;
  bool longTiles;
  size_t keys[2], pays[2], hist, rowBegin, rowEnd, chunkSums, superSums, bytes;
};
static GradPlan planGrad(uint64_t n, size_t rows, size_t width) {
  GradPlan p{};
  int bits = 1;
  while (bits < 32 && ((uint64_t)rows >> bits) != 0) bits++;  // keys are 0 .. rows
  p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digitBits = (bits + p.passes - 1) / p.passes;
  p.longTiles = n > 64u * 1024;
  const uint64_t tile = (uint64_t)kSortThreads * (p.longTiles ? kLongStrips : kShortStrips);
  p.tiles = (int)std::max<uint64_t>(1, (n + tile - 1) / tile);
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  const size_t widthPad = (width + kVec - 1) / kVec * kVec;
  for (int i = 0; i < 2; i++) {
    p.keys[i] = take(n * 4);
    p.pays[i] = take(n * 4);
  }
  p.hist = take(((size_t)p.tiles << p.digitBits) * 4);
  p.rowBegin = take(rows * 4);
  p.rowEnd = take(rows * 4);
  p.chunkSums = take(n / kChunk * widthPad * 4);
  p.superSums = take(n / (kChunk * kChunk) * widthPad * 4);
  p.bytes = at;
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
  constexpr int U = 4;
  // four rows a wave once that still fills the chip (256 CUs, 32 waves each); below, one row a wave
  const bool many = (uint64_t)tokens * a.pieces >= 4u * 256 * 32;
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
  a.hist = (uint32_t*)(ws + p.hist);
  a.rowBegin = (int32_t*)(ws + p.rowBegin);
  a.rowEnd = (uint32_t*)(ws + p.rowEnd);
  a.chunkSums = (float*)(ws + p.chunkSums);
  a.superSums = (float*)(ws + p.superSums);
  a.widthPad = (uint32_t)((width + kVec - 1) / kVec * kVec);

  const hipStream_t st = (hipStream_t)stream;
  int from = 0;
  for (int pass = 0; pass < p.passes; pass++, from ^= 1) {
    SortPass s;
    s.from = from;
    s.shift = pass * p.digitBits;
    s.bits = p.digitBits;
    s.tiles = p.tiles;
    const unsigned tiles = (unsigned)p.tiles;
    if (pass == 0) {
      const unsigned clear = accumulate ? 0u : (unsigned)std::min<size_t>((rows + 4095) / 4096, 1024);
      DFCCL_LAUNCH_BLOCKS((p.longTiles ? sortCountKernel<kLongStrips, true> : sortCountKernel<kShortStrips, true>),
                          tiles + clear, kSortThreads, st, a, s);
      if (n == 0) break;
      DFCCL_LAUNCH_BLOCKS((p.longTiles ? sortScatterKernel<kLongStrips, true> : sortScatterKernel<kShortStrips, true>), tiles,
                          kSortThreads, st, a, s);
    } else {
      DFCCL_LAUNCH_BLOCKS((p.longTiles ? sortCountKernel<kLongStrips, false> : sortCountKernel<kShortStrips, false>), tiles,
                          kSortThreads, st, a, s);
      DFCCL_LAUNCH_BLOCKS((p.longTiles ? sortScatterKernel<kLongStrips, false> : sortScatterKernel<kShortStrips, false>), tiles,
                          kSortThreads, st, a, s);
    }
  }
  if (n > 0) {
    const uint64_t chunks = (n + kChunk - 1) / kChunk;
    DFCCL_LAUNCH_BLOCKS(pickChunk((int)gradType), gridFor(chunks * a.pieces), kRowThreads, st, a, from);
    const uint64_t supers = n / (kChunk * kChunk);
    if (supers > 0) DFCCL_LAUNCH_BLOCKS(superKernel, gridFor(supers * a.pieces), kRowThreads, st, a, from);
  }
  const uint64_t waves = (accumulate ? n : ((uint64_t)rows + kRowsPerWave - 1) / kRowsPerWave) * a.pieces;
  DFCCL_LAUNCH_BLOCKS(pickRows((int)gradType, (int)tableType, accumulate != 0), gridFor(waves), kRowThreads, st, a, from);
  return hipGetLastError() == hipSuccess ? ncclSuccess : ncclUnhandledCudaError;
}

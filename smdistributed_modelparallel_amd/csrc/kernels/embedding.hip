// Token embedding: y[t] = scale * W[id_t - start] (+ P[pos_t]), and the gradients of both tables.
//
// Forward: a gather, bound by HBM: it writes every row and reads it from the table (or the
// caches, for frequent tokens).  The sum is formed in fp32 and rounded once.
//
// Backward: dW[v] = scale * sum of dy[t] over the tokens with id_t = v, in token order and in
// fp32, so that the result does not depend on the order in which blocks run.  The tokens are
// brought into the order of their rows first (bound by latency: 27 us for 65536 tokens), then every
// row of dy is read once and every row of dW written once (bound by HBM).
//
// Measured, 65536 tokens, 50257 x 1600 bf16, with a table of 2048 positions: forward 73 us after other work,
// 65 us of a table that was read just before; sums and zeros of both tables 118 us (580 MB, 4.9 TB/s); joins
// 9 us.  One block for each row of the table,
// which looked for its tokens in all ids, took 3400 us.
#include "kernels.h"
#include "vec8.h"

namespace smpk {
namespace {

constexpr int kT = 256;
constexpr int64_t kMostBlocks = (1ll << 32) / kT;  // a grid's threads stay below 2^32
// Longest list that is ordered in one launch.  The whole gradient of lists of a vocabulary of 50257, 8 bf16
// columns, so and by radix passes: 8192 tokens 40 and 51 us, 16384 51 and 57 us, 24576 59 us both, 65536 93
// and 58 us.
constexpr int64_t kRangeTokens = 16384;
constexpr int64_t kRangeBlocks = 256;  // blocks of that launch: one for each CU

// Row of a table for one token of a list with ids; `rows` where the id is not one of its rows.
__device__ __forceinline__ uint32_t row_of(const IndexList& l, int64_t t) {
  const int64_t id = l.wide ? static_cast<const int64_t*>(l.ids)[t] : static_cast<const int32_t*>(l.ids)[t];
  const uint64_t r = static_cast<uint64_t>(id) - static_cast<uint64_t>(l.start);
  return static_cast<uint32_t>(r < static_cast<uint64_t>(l.rows) ? r : l.rows);
}

constexpr int kPerThread = 4;  // vectors of a thread, all loads in flight together

// Vectors of the output in order, kT * kPerThread of them a block: all lanes are busy at any width.
// Threads past the end and tokens without a row load row 0 and drop it: no branch separates the
// loads.  slice: an XCD (every kXcds-th block) takes `slice` blocks of each sequence, the same
// positions of all of them (or nearly: in whole blocks), so that its L2 holds their rows.  32 x 1000 tokens of 1600
// bf16: 30 us, and 40 us with the blocks in order; 32 x 2048, whose sequences are multiples of kXcds
// blocks in any case: 65 us both; 64 x 512, whose are not quite: 32 and 28 us.
constexpr uint32_t kXcds = 8;
template <typename T, bool FULL>
__global__ void __launch_bounds__(kT) emb_fwd(IndexList ids, const T* __restrict__ w, int64_t w_stride, float scale,
                                              int foreign_zero, IndexList pos, const T* __restrict__ p,
                                              int64_t p_stride, T* __restrict__ y, int n, int d, uint32_t per_row,
                                              uint32_t reciprocal, uint32_t slice) {
  uint32_t block = blockIdx.x;
  if (slice != 0 && block < gridDim.x / (kXcds * slice) * (kXcds * slice)) {
    const uint32_t k = block / kXcds, sequence = k / slice;
    block = (sequence * kXcds + block % kXcds) * slice + (k - sequence * slice);
  }
  const int64_t v0 = static_cast<int64_t>(block) * (kT * kPerThread);
  const int t0 = static_cast<int>(v0 / per_row);
  const uint32_t r0 = static_cast<uint32_t>(v0 - static_cast<int64_t>(t0) * per_row);
  int t[kPerThread], c[kPerThread];
  int64_t id[kPerThread], at[kPerThread];
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const uint32_t off = r0 + u * kT + threadIdx.x;
    uint32_t q = __umulhi(off, reciprocal), r = off - q * per_row;  // reciprocal rounded down: q may be one short
    q += r >= per_row ? 1 : 0;
    r -= r >= per_row ? per_row : 0;
    t[u] = t0 + static_cast<int>(q);
    c[u] = static_cast<int>(r) * kCols;
  }
  if (ids.wide) {
#pragma unroll
    for (int u = 0; u < kPerThread; ++u) id[u] = static_cast<const int64_t*>(ids.ids)[t[u] < n ? t[u] : 0];
  } else {
#pragma unroll
    for (int u = 0; u < kPerThread; ++u) id[u] = static_cast<const int32_t*>(ids.ids)[t[u] < n ? t[u] : 0];
  }
  if (p != nullptr) {
    if (pos.ids == nullptr) {
      const uint32_t period = static_cast<uint32_t>(pos.period), first = static_cast<uint32_t>(t0) % period;
#pragma unroll
      for (int u = 0; u < kPerThread; ++u) {
        uint32_t k = first + static_cast<uint32_t>(t[u] - t0);
        if (k >= period) k -= period;
        at[u] = k < period ? k : k % period;  // (a block spans several periods)
      }
    } else if (pos.wide) {
#pragma unroll
      for (int u = 0; u < kPerThread; ++u) at[u] = static_cast<const int64_t*>(pos.ids)[t[u] < n ? t[u] : 0];
    } else {
#pragma unroll
      for (int u = 0; u < kPerThread; ++u) at[u] = static_cast<const int32_t*>(pos.ids)[t[u] < n ? t[u] : 0];
    }
  }
  Raw8<T> a[kPerThread], b[kPerThread];
  bool held[kPerThread];
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const int64_t row = id[u] - ids.start;
    held[u] = row >= 0 && row < ids.rows;
    read8<FULL>(w + (held[u] ? row : 0) * w_stride + c[u], d - c[u], a[u]);
  }
  if (p != nullptr) {
#pragma unroll
    for (int u = 0; u < kPerThread; ++u) {
      const bool ok = at[u] >= 0 && at[u] < pos.rows;
      read8<FULL>(p + (ok ? at[u] : 0) * p_stride + c[u], d - c[u], b[u]);
      at[u] = ok;
    }
  }
  const float none = foreign_zero ? 0.f : NAN;
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    float o[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) o[j] = held[u] ? at8(a[u], j) * scale : none;
    if (p != nullptr) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) o[j] += at[u] ? at8(b[u], j) : NAN;
    }
    if (t[u] < n) write8<FULL, false>(y + static_cast<int64_t>(t[u]) * d + c[u], d - c[u], o);
  }
}

// ----------------------------------------------------------------------- sorting the tokens
// Stable radix sort of (row, token), least significant digit first: a row number has at most 10
// bits a pass, so a vocabulary of up to 2^20 rows takes two.  A block of 16 waves owns a
// consecutive run of the items, each wave a consecutive part of it; the waves count their digits,
// the counts become the places of each wave's items, and the wave walks over its items once more,
// 64 at a time, in order.  No place depends on the order in which anything runs.  65536 tokens:
// 5.0 us to count and 8.7 us to place, each pass; both are the latency of few blocks.  Every block reads the
// counts of all: 256 blocks up to 2 M tokens, more above.  Gradient of 8 bf16 columns: 2^22 tokens 0.58 ms,
// 2^24 2.2 ms, 2^27 39 ms.
constexpr int kWaves = 16;
constexpr int kSortThreads = kWaves * 64;
constexpr int kMaxBits = 10;

struct SortItems {
  IndexList ids;  // first pass: keys and tokens come from the ids
  uint32_t skip;  // row without a gradient; none of them: `rows`
  const uint32_t* keys;  // later passes (null in the first)
  const int32_t* tokens;
  uint32_t* keys_out;
  int32_t* tokens_out;
  int64_t n, per_block;  // per_block: a multiple of kSortThreads
  int shift, bits;
  uint8_t* marks;  // null, or [rows rounded up to 16]: 1 for every row that has a token
};

// Rows' keys are their numbers; tokens without a row come last, with the key `rows`.
__device__ __forceinline__ uint32_t key_of(const SortItems& a, int64_t i) {
  if (a.keys != nullptr) return a.keys[i];
  const uint32_t r = row_of(a.ids, i);
  return r == a.skip ? static_cast<uint32_t>(a.ids.rows) : r;
}

__device__ __forceinline__ void wave_run(const SortItems& a, int block, int64_t& s, int64_t& e) {
  const int64_t part = a.per_block / kWaves;
  s = static_cast<int64_t>(block) * a.per_block + (threadIdx.x >> 6) * part;
  e = s + part < a.n ? s + part : a.n;
}

constexpr int kRounds = 8;  // 64-item rounds of a wave: at most 8192 items a block

// Counts a wave's next 64 items; returns how many of the wave's items of the same digit come before
// this lane's.  Equal digits are counted together: a list may hold one token thousands of times.
__device__ __forceinline__ int count_items(int digit, bool valid, int bits, int32_t* cnt) {
  const int lane = threadIdx.x & 63;
  uint64_t same = __ballot(valid);  // the lanes with this lane's digit
  const int one = __builtin_amdgcn_readlane(digit, __ffsll(static_cast<unsigned long long>(same | 1ull << 63)) - 1);
  const int steps = __ballot(valid && digit != one) == 0 ? 0 : bits;  // runs of one token need no matching
  for (int b = 0; b < steps; ++b) {
    const uint32_t mine = static_cast<uint32_t>(static_cast<int32_t>(static_cast<uint32_t>(digit) << (31 - b)) >> 31);
    const uint64_t m = __ballot(mine != 0);
    same &= ~(m ^ (static_cast<uint64_t>(mine) << 32 | mine));
  }
  const int first = valid ? __ffsll(static_cast<unsigned long long>(same)) - 1 : lane;
  int at = 0;
  if (valid && lane == first) at = atomicAdd(&cnt[digit], __popcll(same));
  return __shfl(at, first, 64) + __popcll(same & ((1ull << lane) - 1));
}

// The first pass also clears the marks that its second launch sets for every row with a token.
__device__ __forceinline__ void clear_marks(const SortItems& a, int block, int blocks) {
  if (a.marks == nullptr || a.keys != nullptr) return;
  const int64_t words = (a.ids.rows + 15) / 16;  // (the workspace is a multiple of 16 bytes)
  for (int64_t i = static_cast<int64_t>(block) * kSortThreads + threadIdx.x; i < words;
       i += static_cast<int64_t>(blocks) * kSortThreads)
    reinterpret_cast<uint4*>(a.marks)[i] = make_uint4(0, 0, 0, 0);
}

__global__ void __launch_bounds__(kSortThreads) emb_sort_count(SortItems a, int32_t* __restrict__ counts) {
  __shared__ int32_t cnt[1 << kMaxBits];
  const int bins = 1 << a.bits;
  for (int d = threadIdx.x; d < bins; d += kSortThreads) cnt[d] = 0;
  clear_marks(a, blockIdx.x, gridDim.x);
  __syncthreads();
  int64_t s, e;
  wave_run(a, blockIdx.x, s, e);
  uint32_t keys[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = s + r * 64 + (threadIdx.x & 63);
    keys[r] = i < e ? key_of(a, i) : 0u;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (s + r * 64 < e)
      count_items((keys[r] >> a.shift) & (bins - 1), s + r * 64 + (threadIdx.x & 63) < e, a.bits, cnt);
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) counts[static_cast<int64_t>(blockIdx.x) * bins + d] = cnt[d];
}

template <int BITS>
struct SortLds {
  int32_t cnt[kWaves][1 << BITS];
  int32_t total[1 << BITS], before[1 << BITS];
  int32_t wave_total[kWaves];
};

// cnt[w][d], the items of digit d in wave w, becomes the place of the first of them: after all items
// of smaller digits (anywhere), and of digit d in earlier blocks (`before`) and waves.
template <int BITS>
__device__ __forceinline__ void counts_to_places(SortLds<BITS>& lds, int bins, bool one_block) {
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  int c[kWaves], total = 0;
  if (tid < bins) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      c[w] = lds.cnt[w][tid];
      total += c[w];
    }
    if (!one_block) total = lds.total[tid];
  }
  int incl = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(incl, o, 64);
    if (lane >= o) incl += v;
  }
  if (lane == 63) lds.wave_total[wid] = incl;
  __syncthreads();
  if (tid < bins) {
    int base = incl - total + (one_block ? 0 : lds.before[tid]);
    for (int w = 0; w < wid; ++w) base += lds.wave_total[w];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      lds.cnt[w][tid] = base;
      base += c[w];
    }
  }
  __syncthreads();
}

// One pass over the items of one block; counts [blocks][bins] of all blocks.
__global__ void __launch_bounds__(kSortThreads) emb_sort_place(SortItems a, const int32_t* __restrict__ counts) {
  __shared__ SortLds<kMaxBits> lds;
  const int bins = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int blocks = gridDim.x, block = blockIdx.x;
  for (int d = lane; d < bins; d += 64) lds.cnt[wid][d] = 0;
  if (tid < bins) lds.total[tid] = lds.before[tid] = 0;
  __syncthreads();
  int64_t s, e;
  wave_run(a, block, s, e);
  // every thread adds up one digit of some blocks
  int all = 0, earlier = 0;
  const int my_digit = tid & (bins - 1), step = kSortThreads >> a.bits;
#pragma unroll 8
  for (int b = tid >> a.bits; b < blocks; b += step) {
    const int c = counts[(static_cast<int64_t>(b) << a.bits) + my_digit];
    all += c;
    earlier += b < block ? c : 0;
  }
  atomicAdd(&lds.total[my_digit], all);
  atomicAdd(&lds.before[my_digit], earlier);
  uint32_t keys[kRounds];
  int32_t token[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = s + r * 64 + lane;
    keys[r] = i < e ? key_of(a, i) : 0u;
    token[r] = a.tokens != nullptr && i < e ? a.tokens[i] : static_cast<int32_t>(i);
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (s + r * 64 < e)
      rank[r] = count_items((keys[r] >> a.shift) & (bins - 1), s + r * 64 + lane < e, a.bits, lds.cnt[wid]);
  __syncthreads();
  counts_to_places(lds, bins, false);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (s + r * 64 + lane >= e) continue;
    const int at = lds.cnt[wid][(keys[r] >> a.shift) & (bins - 1)] + rank[r];
    a.keys_out[at] = keys[r];
    a.tokens_out[at] = token[r];
    if (a.marks != nullptr && a.keys == nullptr && keys[r] < a.ids.rows) a.marks[keys[r]] = 1;
  }
}

// The whole order in one launch, for vocabularies and lists that are not too large: every block
// owns a range of rows and reads all ids twice -- from the caches, which hold them -- once to count
// the tokens of its rows (and of the rows before, which say where its part of the list begins),
// once to place them.  Waves and their items are taken in order, as above.
template <int BITS>
__global__ void __launch_bounds__(kSortThreads) emb_sort_ranges(SortItems a, int range) {
  __shared__ SortLds<BITS> lds;
  __shared__ int32_t below[kWaves], valid_ids[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, bins = 1 << a.bits;
  const uint32_t lo = blockIdx.x * static_cast<uint32_t>(range), none = static_cast<uint32_t>(a.ids.rows);
  const uint32_t mine_end = none - lo < static_cast<uint32_t>(range) ? none - lo : range;  // its rows: lo + [0, mine_end)
  for (int d = lane; d < bins; d += 64) lds.cnt[wid][d] = 0;  // (its own wave's: no barrier)
  const int64_t part = (a.n + kWaves - 1) / kWaves, s = wid * part, e = s + part < a.n ? s + part : a.n;
  int less = 0, held = 0;
  for (int64_t i0 = s; i0 < e; i0 += 64 * kRounds) {
    uint32_t key[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int64_t i = i0 + r * 64 + lane;
      key[r] = i < e ? key_of(a, i) : none;
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      less += __popcll(__ballot(key[r] < lo));
      held += __popcll(__ballot(key[r] != none));
      if (key[r] - lo < mine_end) atomicAdd(&lds.cnt[wid][key[r] - lo], 1);
    }
  }
  if (lane == 0) {
    below[wid] = less;
    valid_ids[wid] = held;
  }
  __syncthreads();
  int first = 0, live = 0;
  for (int w = 0; w < kWaves; ++w) {
    first += below[w];
    live += valid_ids[w];
  }
  if (a.marks != nullptr && tid < static_cast<int>(mine_end)) {
    int total = 0;
    for (int w = 0; w < kWaves; ++w) total += lds.cnt[w][tid];
    a.marks[lo + tid] = total != 0;
  }
  counts_to_places(lds, bins, true);
  for (int64_t i0 = s; i0 < e; i0 += 64 * kRounds) {
    uint32_t key[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int64_t i = i0 + r * 64 + lane;
      key[r] = i < e ? key_of(a, i) : none;
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const bool mine = key[r] - lo < mine_end;
      if (__ballot(mine) == 0) continue;
      const int at = first + count_items(mine ? static_cast<int>(key[r] - lo) : 0, mine, a.bits, lds.cnt[wid]);
      if (mine) {
        a.keys_out[at] = key[r];
        a.tokens_out[at] = static_cast<int32_t>(i0 + r * 64 + lane);
      }
    }
  }
  // the places of the tokens without a row, a part for each block
  for (int64_t i = live + static_cast<int64_t>(blockIdx.x) * kSortThreads + tid; i < a.n;
       i += static_cast<int64_t>(gridDim.x) * kSortThreads)
    a.keys_out[i] = none;
}

// --------------------------------------------------------------------- sums over the sorted tokens
// The sorted list is cut into chunks of the same number of tokens, whatever rows they belong to.
// A chunk adds up each run of one row; a run that lies in the chunk is that row's gradient, the
// others leave a partial sum: slot 0 for the run that began in an earlier chunk, slot 1 for the
// one that begins here and goes on.  A second kernel adds a row's partials in chunk order.
struct Sorted {
  const uint32_t* keys;  // null: the list of positions, `batch` tokens each, `period` apart
  const int32_t* tokens;
  int64_t n, rows, batch, period;
  __device__ __forceinline__ uint32_t key(int64_t j) const {
    return keys != nullptr ? keys[j] : static_cast<uint32_t>(j) / static_cast<uint32_t>(batch);
  }
  __device__ __forceinline__ int64_t token(int64_t j, uint32_t k) const {
    return keys != nullptr ? tokens[j] : (j - k * batch) * period + k;
  }
};

// dw row = scale * sum, or that added to the row
template <bool FULL, typename T>
__device__ __forceinline__ void write_row(T* p, int left, float (&sum)[kCols], float scale, int accumulate) {
  if (accumulate) {
    Raw8<T> r;
    read8<FULL>(p, left, r);
#pragma unroll
    for (int j = 0; j < kCols; ++j) sum[j] = fmaf(sum[j], scale, at8(r, j));
  } else {
#pragma unroll
    for (int j = 0; j < kCols; ++j) sum[j] *= scale;
  }
  write8<FULL, sizeof(T) == 2>(p, left, sum);  // (fp32 lanes fill half lines: through the caches)
}

// What a launch has to do for one table: blocks [first, first + blocks) add up its tokens, then
// [clear, clear + clears) clear rows, `windows` of them in all.
struct Work {
  Sorted l;
  void* dw;
  float* part;
  const uint8_t* marks;
  float scale;
  int accumulate, chunk;
  int64_t first, blocks, clear, clears, windows;
  int stream;  // zeros past the caches
};

constexpr int kZeroRows = 16;
// Cleared rows of a table that the caches hold (256 MB, of which the reads need a part) go through
// them: 62 MB of fp32 15.7 us against 21.7 us past them; 155 MB of fp16 35.2 us against 28.9 us.  Of bf16
// tables alone, replayed, the zeros past the caches are ahead earlier: 64 MB 25 and 22 us for the whole
// gradient, 96 MB 30 and 26 us, 128 MB 36 and 30 us.
constexpr int64_t kCached = 96ll << 20;

// 512 columns of the rows of a bit mask, every fourth of them for this wave, become zero; `at`: the
// first row and column, `left` columns to the row's end.  Whole vectors go as 16 consecutive bytes a
// lane, so that every store fills whole lines (past the caches, half lines of fp32 took 388 us where
// whole ones take 146 us).
template <bool FULL, bool STREAM, typename T>
__device__ __forceinline__ void zero_rows(uint64_t rows, T* at, int64_t left, int d) {
  constexpr int M = 16 / sizeof(T);
  const int lane = threadIdx.x & 63;
  const float zero[kCols] = {};
  const Word4 none = {0, 0, 0, 0};
  for (int k = 0; rows != 0; ++k, rows &= rows - 1) {
    if (k % (kT / 64) != static_cast<int>(threadIdx.x >> 6)) continue;
    T* const row = at + static_cast<int64_t>(__ffsll(static_cast<unsigned long long>(rows)) - 1) * d;
    if constexpr (FULL) {
#pragma unroll
      for (int u = 0; u < kCols / M; ++u) {
        const int c = (u * 64 + lane) * M;
        if (c >= left) continue;
        Word4* const q = reinterpret_cast<Word4*>(row + c);
        if (STREAM) {
          __builtin_nontemporal_store(none, q);
        } else {
          *q = none;
        }
      }
    } else if (lane * kCols < left) {
      write8<FULL, STREAM>(row + lane * kCols, static_cast<int>(left) - lane * kCols, zero);
    }
  }
}

// A dense gradient: windows of 16 rows x 512 columns, of which the rows without a token are cleared
// (marks null: the rows from `period` on).  One window a block in tables of up to kClears of them.
constexpr int64_t kClears = 1 << 21;
template <bool FULL, typename T>
__device__ __forceinline__ void clear_rows(const Work& wk, int64_t block, int slabs, T* dw, int d) {
  const Sorted& l = wk.l;
  const int lane = threadIdx.x & 63;
  for (; block < wk.windows; block += wk.clears) {
    const int64_t window = block / slabs, r0 = window * kZeroRows, mine = r0 + lane;
    const int c = static_cast<int>(block - window * slabs) * 64 * kCols;
    const bool empty = lane < kZeroRows && mine < l.rows &&
                       (l.n == 0 || (wk.marks != nullptr ? wk.marks[mine] == 0 : mine >= l.period));
    const uint64_t rows = __ballot(empty);  // the same in all waves
    T* const at = dw + r0 * d + c;
    if (wk.stream) {  // (two loops: the compiler would make one store of two that differ in this alone)
      zero_rows<FULL, true>(rows, at, d - c, d);
    } else {
      zero_rows<FULL, false>(rows, at, d - c, d);
    }
  }
}

__device__ __forceinline__ Work work_of(const Work& a, const Work& b) {
  const int64_t i = blockIdx.x;
  return (i >= b.first && i < b.first + b.blocks) || i >= b.clear ? b : a;
}

// A wave takes a chunk of at most 64 tokens and 512 columns.  Lane i knows the i-th token; a run is
// followed with scalar registers, so the branches cost nothing, and the gradient rows of one
// batch are loaded while those of the batch before are added.
template <typename T, bool FULL>
__global__ void __launch_bounds__(kT) emb_bwd_wide(Work w0, Work w1, const T* __restrict__ dy, int d, int slabs) {
  constexpr int kAhead = sizeof(T) == 4 ? 4 : 8;
  const Work wk = work_of(w0, w1);
  const Sorted l = wk.l;
  T* const dw = static_cast<T*>(wk.dw);
  float* const part = wk.part;
  const float scale = wk.scale;
  const int accumulate = wk.accumulate, chunk = wk.chunk;
  if (static_cast<int64_t>(blockIdx.x) >= wk.clear) {
    clear_rows<FULL>(wk, blockIdx.x - wk.clear, slabs, dw, d);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) - wk.first) * (kT / 64) +
                       __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int64_t ch = unit / slabs;
  const int c = (static_cast<int>(unit - ch * slabs) * 64 + lane) * kCols, left = d - c;
  const int64_t j0 = ch * chunk, j1 = j0 + chunk < l.n ? j0 + chunk : l.n;
  const int from = left > 0 ? c : 0;  // lanes past the row's end load its first vector and drop it
  if (j0 >= l.n) return;
  const int m = static_cast<int>(j1 - j0);
  const uint32_t none = static_cast<uint32_t>(l.rows);
  const uint32_t my_key = lane < m ? l.key(j0 + lane) : none;
  const int my_token = lane < m ? static_cast<int>(l.token(j0 + lane, my_key)) : 0;
  const uint32_t before = j0 > 0 ? l.key(j0 - 1) : none, after = j1 < l.n ? l.key(j1) : none;
  auto key_at = [&](int i) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(my_key), i)); };
  // tokens with a row: those without come last
  const int live = __popcll(__ballot(lane < m && my_key != none));
  if (live == 0) return;
  Raw8<T> buf[2][kAhead];
  auto fetch = [&](int i, Raw8<T> (&r)[kAhead]) {  // (past the last token: that token again, dropped)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t t = __builtin_amdgcn_readlane(my_token, i + u < live ? i + u : live - 1);
      read8<FULL>(dy + t * d + from, left, r[u]);
    }
  };
  uint32_t cur = key_at(0);
  bool head = before == cur;
  float sum[kCols];
#pragma unroll
  for (int q = 0; q < kCols; ++q) sum[q] = 0.f;
  auto add = [&](int i, const Raw8<T> (&r)[kAhead]) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u >= live) break;
      const uint32_t k = key_at(i + u);
      if (k != cur) {
        if (left > 0) {
          if (head) {
            write8<FULL, false>(part + (2 * ch) * d + c, left, sum);
          } else {
            write_row<FULL>(dw + static_cast<int64_t>(cur) * d + c, left, sum, scale, accumulate);
          }
        }
        head = false;
        cur = k;
#pragma unroll
        for (int q = 0; q < kCols; ++q) sum[q] = 0.f;
      }
#pragma unroll
      for (int q = 0; q < kCols; ++q) sum[q] += at8(r[u], q);
    }
  };
  fetch(0, buf[0]);
  for (int i = 0; i < live; i += 2 * kAhead) {
    fetch(i + kAhead, buf[1]);
    add(i, buf[0]);
    fetch(i + 2 * kAhead, buf[0]);
    add(i + kAhead, buf[1]);
  }
  if (left <= 0) return;
  const bool tail = live == m && after == cur;
  if (head || tail) {
    write8<FULL, false>(part + (2 * ch + (head ? 0 : 1)) * d + c, left, sum);
  } else {
    write_row<FULL>(dw + static_cast<int64_t>(cur) * d + c, left, sum, scale, accumulate);
  }
}

// The same for rows of at most 256 columns: `lanes` threads (a power of two) hold a chunk's
// columns, kT / lanes chunks a block.
template <typename T, bool FULL>
__global__ void __launch_bounds__(kT) emb_bwd_narrow(Work w0, Work w1, const T* __restrict__ dy, int d, int lanes) {
  constexpr int kAhead = 8;
  const Work wk = work_of(w0, w1);
  const Sorted l = wk.l;
  T* const dw = static_cast<T*>(wk.dw);
  float* const part = wk.part;
  const float scale = wk.scale;
  const int accumulate = wk.accumulate, chunk = wk.chunk;
  if (static_cast<int64_t>(blockIdx.x) >= wk.clear) {
    clear_rows<FULL>(wk, blockIdx.x - wk.clear, 1, dw, d);
    return;
  }
  const int64_t ch = (static_cast<int64_t>(blockIdx.x) - wk.first) * (kT / lanes) + threadIdx.x / lanes;
  const int c = threadIdx.x % lanes * kCols;
  const int left = d - c;
  const int64_t j0 = ch * chunk, j1 = j0 + chunk < l.n ? j0 + chunk : l.n;
  if (j0 >= l.n || left <= 0) return;
  const uint32_t none = static_cast<uint32_t>(l.rows);
  uint32_t cur = l.key(j0);
  bool head = j0 > 0 && l.key(j0 - 1) == cur;
  float sum[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) sum[j] = 0.f;
  for (int64_t j = j0; j < j1; j += kAhead) {
    uint32_t key[kAhead];
    Raw8<T> row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) key[u] = j + u < j1 ? l.key(j + u) : none;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (key[u] != none) read8<FULL>(dy + l.token(j + u, key[u]) * d + c, left, row[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (key[u] != cur && j + u < j1) {
        if (head) {
          write8<FULL, false>(part + (2 * ch) * d + c, left, sum);
        } else {
          write_row<FULL>(dw + static_cast<int64_t>(cur) * d + c, left, sum, scale, accumulate);
        }
        head = false;
        cur = key[u];
#pragma unroll
        for (int q = 0; q < kCols; ++q) sum[q] = 0.f;
      }
      if (key[u] != none) {
#pragma unroll
        for (int q = 0; q < kCols; ++q) sum[q] += at8(row[u], q);
      }
    }
    if (cur == none) return;  // only tokens without a row follow
  }
  const bool tail = j1 < l.n && l.key(j1) == cur;
  if (head || tail) {
    write8<FULL, false>(part + (2 * ch + (head ? 0 : 1)) * d + c, left, sum);
  } else {
    write_row<FULL>(dw + static_cast<int64_t>(cur) * d + c, left, sum, scale, accumulate);
  }
}

// ------------------------------------------------------------------------------- short lists
// The whole backward of a short list in one launch and without a workspace.  Every block owns a range of
// rows: it reads all ids, keeps its own tokens in order, adds up each row's -- a wave for 512 columns
// or, for rows of many tokens, all waves -- and clears the rows without a token.  512 tokens of 512
// bf16 into 5000 rows: 6 us, with the launches above 14 us; all of them into one row: 16 and 15 us.  A
// training call of 231 tokens of 512 fp32, which is bound by the host: 61 us, 68 us with them.
constexpr int kShortTokens = 512;
constexpr int kShortRange = 1024;   // rows of a block
constexpr int kShortBlocks = 1024;  // of a table

struct ShortTable {
  IndexList ids;
  uint32_t skip;
  void* dw;
  float scale;
  int accumulate, range, blocks;
};
struct ShortTables {
  ShortTable t[2];
  const void* dy;
  int n, d;
};

// Adds the gradients of the list's tokens [q0, q1) that belong to `row`, in order.
template <typename T, bool FULL>
__device__ __forceinline__ void add_tokens(const uint16_t* rows, const uint16_t* tokens, int row, int q0, int q1,
                                           const T* __restrict__ dy, int d, int from, int left, float (&sum)[kCols]) {
  constexpr int kAhead = 8;
  for (; q0 < q1; q0 += 64) {
    const int q = q0 + static_cast<int>(threadIdx.x & 63);
    const int token = q < q1 ? tokens[q] : 0;
    uint64_t on = __ballot(q < q1 && rows[q < q1 ? q : 0] == row);
    while (on != 0) {
      const int live = __popcll(on);
      Raw8<T> r[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {  // (past the last token: that one again, dropped)
        const int i = __ffsll(static_cast<unsigned long long>(on)) - 1;
        read8<FULL>(dy + static_cast<int64_t>(__builtin_amdgcn_readlane(token, i)) * d + from, left, r[k]);
        if (k + 1 < live) on &= on - 1;
      }
      if (live <= kAhead) on = 0;
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[j] += k < live ? at8(r[k], j) : 0.f;
    }
  }
}

template <typename T, bool FULL>
__global__ void __launch_bounds__(kT) emb_bwd_short(ShortTables a) {
  constexpr int kWaves = kT / 64, kItems = kShortTokens / kT, kHeavy = 32;
  __shared__ int held_by[kShortRange];  // tokens of a row
  __shared__ uint16_t rows[kShortTokens], tokens[kShortTokens];
  __shared__ uint16_t light[kShortTokens], heavy[kShortTokens / kHeavy];  // rows with tokens
  __shared__ int count[kItems][kWaves], lights, heavies;
  __shared__ float part[kWaves][kCols][64];
  const bool second = static_cast<int>(blockIdx.x) >= a.t[0].blocks;
  const ShortTable& t = second ? a.t[1] : a.t[0];
  const int block = static_cast<int>(blockIdx.x) - (second ? a.t[0].blocks : 0);
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), d = a.d;
  const int64_t lo = static_cast<int64_t>(block) * t.range;
  const int range = static_cast<int>(t.ids.rows - lo < t.range ? t.ids.rows - lo : t.range);
  for (int i = tid; i < range; i += kT) held_by[i] = 0;
  if (tid == 0) lights = heavies = 0;
  int mine[kItems];  // row of the range, or -1
  uint64_t mask[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int i = k * kT + tid;
    mine[k] = -1;
    if (i < a.n) {
      const uint32_t r = t.ids.ids != nullptr ? row_of(t.ids, i)
                                              : static_cast<uint32_t>(i) % static_cast<uint32_t>(t.ids.period);
      if (r != t.skip && r < t.ids.rows && r >= lo && r - lo < range) mine[k] = static_cast<int>(r - lo);
    }
    mask[k] = __ballot(mine[k] >= 0);
    if (lane == 0) count[k][wid] = __popcll(mask[k]);
  }
  __syncthreads();
  int m = 0;
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w == wid && mine[k] >= 0) {
        const int at = m + __popcll(mask[k] & ((1ull << lane) - 1));
        rows[at] = static_cast<uint16_t>(mine[k]);
        tokens[at] = static_cast<uint16_t>(k * kT + tid);
        atomicAdd(&held_by[mine[k]], 1);
      }
      m += count[k][w];
    }
  }
  __syncthreads();
  // (the order of these lists is not fixed, and decides no sum)
  if (m > 0) {
    for (int i = tid; i < range; i += kT) {
      const int n = held_by[i];
      if (n > kHeavy) {
        heavy[atomicAdd(&heavies, 1)] = static_cast<uint16_t>(i);
      } else if (n > 0) {
        light[atomicAdd(&lights, 1)] = static_cast<uint16_t>(i);
      }
    }
  }
  __syncthreads();
  const T* const __restrict__ dy = static_cast<const T*>(a.dy);
  T* const dw = static_cast<T*>(t.dw) + lo * d;
  const int slabs = (d + 64 * kCols - 1) / (64 * kCols);
  for (int u = wid; u < lights * slabs; u += kWaves) {
    const int p = u / slabs, c = ((u - p * slabs) * 64 + lane) * kCols, left = d - c;
    const int row = __builtin_amdgcn_readfirstlane(light[p]);
    float sum[kCols] = {};
    add_tokens<T, FULL>(rows, tokens, row, 0, m, dy, d, left > 0 ? c : 0, left, sum);
    if (left > 0) write_row<FULL>(dw + static_cast<int64_t>(row) * d + c, left, sum, t.scale, t.accumulate);
  }
  // rows of many tokens: a part of the list for each wave
  const int quarter = (m + kWaves - 1) / kWaves;
  for (int u = 0; u < heavies * slabs; ++u) {
    const int p = u / slabs, c = ((u - p * slabs) * 64 + lane) * kCols, left = d - c;
    const int row = __builtin_amdgcn_readfirstlane(heavy[p]), q0 = wid * quarter;
    float sum[kCols] = {};
    add_tokens<T, FULL>(rows, tokens, row, q0, q0 + quarter < m ? q0 + quarter : m, dy, d, left > 0 ? c : 0, left, sum);
#pragma unroll
    for (int j = 0; j < kCols; ++j) part[wid][j][lane] = sum[j];
    __syncthreads();
    if (wid == 0 && left > 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w)
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[j] += part[w][j][lane];
      write_row<FULL>(dw + static_cast<int64_t>(row) * d + c, left, sum, t.scale, t.accumulate);
    }
    __syncthreads();
  }
  if (t.accumulate) return;
  const float zero[kCols] = {};
  const int per_row = (d + kCols - 1) / kCols;
  for (int v = tid; v < range * per_row; v += kT) {
    const int row = v / per_row, c = (v - row * per_row) * kCols;
    if (held_by[row] == 0) write8<FULL, false>(dw + static_cast<int64_t>(row) * d + c, d - c, zero);
  }
}

// Block b joins the run that begins in chunk b and goes on behind it.
template <typename T, bool FULL>
__global__ void __launch_bounds__(kT) emb_bwd_join(Sorted l, const float* __restrict__ part, int d, int chunk, int lanes,
                                                   float scale, T* __restrict__ dw, int accumulate) {
  constexpr int kBatch = 4;
  __shared__ float buf[kT][kCols];
  const int tid = threadIdx.x, lane = tid % lanes, g = tid / lanes, groups = kT / lanes;
  const int c = (blockIdx.y * lanes + lane) * kCols, left = d - c;
  const int64_t ch = blockIdx.x, j0 = ch * chunk, j1 = j0 + chunk;
  if (j1 >= l.n) return;
  const uint32_t k = l.key(j1);
  if (k >= l.rows || l.key(j1 - 1) != k || (j0 > 0 && l.key(j0) == k && l.key(j0 - 1) == k)) return;
  int64_t last = ch + 1;  // the run's last chunk: 64 chunks' first keys at a time
  for (;;) {
    const int64_t j = (last + 1 + (tid & 63)) * chunk;
    const uint64_t on = __ballot(j < l.n && l.key(j) == k);
    const int more = on == ~0ull ? 64 : __ffsll(static_cast<unsigned long long>(~on)) - 1;
    last += more;
    if (more < 64) break;
  }
  float sum[kCols];
#pragma unroll
  for (int q = 0; q < kCols; ++q) sum[q] = 0.f;
  if (left > 0) {
    for (int64_t m = ch + g; m <= last; m += kBatch * groups) {
      Raw8<float> r[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t k0 = m + u * groups < last ? m + u * groups : last;  // (past the end: dropped)
        read8<FULL>(part + (2 * k0 + (k0 == ch ? 1 : 0)) * d + c, left, r[u]);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (m + u * groups > last) break;
#pragma unroll
        for (int q = 0; q < kCols; ++q) sum[q] += at8(r[u], q);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < kCols; ++q) buf[tid][q] = sum[q];
  __syncthreads();
  if (g != 0 || left <= 0) return;
  for (int m = 1; m < groups; ++m) {
#pragma unroll
    for (int q = 0; q < kCols; ++q) sum[q] += buf[m * lanes + lane][q];
  }
  write_row<FULL>(dw + static_cast<int64_t>(k) * d + c, left, sum, scale, accumulate);
}

}  // namespace

int embedding_fwd(int dt, const IndexList& ids, const void* w, int64_t w_stride, float scale, int foreign_zero,
                  const IndexList& pos, const void* p, int64_t p_stride, void* y, int64_t n, int64_t d,
                  hipStream_t s) {
  if (n <= 0 || d <= 0) return 0;
  const int64_t per_row = (d + kCols - 1) / kCols;
  const int64_t blocks = (n * per_row + kT * kPerThread - 1) / (kT * kPerThread);
  if (blocks >= kMostBlocks || n > 0x7fffffff - kT * kPerThread) return -3;
  const uint32_t reciprocal = per_row == 1 ? 0xffffffffu : static_cast<uint32_t>((1ull << 32) / per_row);
  uint32_t slice = 0;
  if (p != nullptr && pos.ids == nullptr)
    slice = static_cast<uint32_t>((pos.period * per_row + kXcds * kT * kPerThread / 2) / (kXcds * kT * kPerThread));
  SMPK_DISPATCH(dt, T, {
    const auto kernel = d % kCols == 0 ? emb_fwd<T, true> : emb_fwd<T, false>;
    kernel<<<static_cast<unsigned>(blocks), kT, 0, s>>>(ids, static_cast<const T*>(w), w_stride, scale, foreign_zero, pos,
                                                       static_cast<const T*>(p), p_stride, static_cast<T*>(y),
                                                       static_cast<int>(n), static_cast<int>(d),
                                                       static_cast<uint32_t>(per_row), reciprocal, slice);
  });
  return static_cast<int>(hipGetLastError());
}

// bytes: of a dense gradient to be written, 0 if it is added to
bool embedding_bwd_short(int64_t n, int64_t d, int64_t rows, int64_t bytes) {
  // one block may have to add up all tokens; the zeros of a table that the caches do not hold need
  // other stores
  return n > 0 && n <= kShortTokens && n * d <= 1 << 18 && rows <= kShortBlocks * kShortRange && bytes <= kCached;
}

EmbeddingPlan embedding_bwd_plan(int64_t n, int64_t d, int64_t rows, int64_t batch) {
  EmbeddingPlan p{};
  if (n <= 0) {  // nothing to order, to add up or to join: rows are cleared at most
    p.one_launch = 1;
    p.chunk = 16;
    return p;
  }
  int bits = 1;
  while ((rows >> bits) != 0) ++bits;  // the keys 0 .. rows
  p.range = static_cast<int>((rows + kRangeBlocks - 1) / kRangeBlocks);
  p.one_launch = n <= kRangeTokens && p.range <= 1 << kMaxBits;
  if (p.one_launch) {
    bits = 1;
    while ((1 << bits) < p.range) ++bits;
    p.passes = 1;
    p.bits = bits;
    p.per_block = 0;
    p.sort_blocks = (rows + p.range - 1) / p.range;
  } else {
    p.passes = (bits + kMaxBits - 1) / kMaxBits;
    p.bits = (bits + p.passes - 1) / p.passes;
    // runs of 2048 tokens or, above 256 blocks, whose counts every block reads, of up to 8192
    // (kRounds rounds of 16 waves)
    constexpr int64_t kMost = kRounds * kSortThreads;
    int64_t parts = (n + 2047) / 2048;
    if (parts > 256) parts = (n + kMost - 1) / kMost > 256 ? (n + kMost - 1) / kMost : 256;
    p.per_block = ((n + parts - 1) / parts + kSortThreads - 1) / kSortThreads * kSortThreads;
    p.sort_blocks = (n + p.per_block - 1) / p.per_block;
  }
  int64_t c = 16;  // tokens of a chunk: long ones leave fewer partial sums, short ones more to run at once
  // (narrow rows share their blocks' lanes: the same time at 16, of many more blocks)
  while (d > 32 * kCols && c < 64 && n / (c * 2) >= 1024) c *= 2;
  // positions of up to 64 sequences: whole runs in a chunk, which leave nothing to join
  p.join = !(batch > 0 && batch <= 64);
  if (!p.join) c = c < batch ? batch : c / batch * batch;
  p.chunk = static_cast<int>(c);
  p.chunks = (n + c - 1) / c;
  return p;
}

namespace {

// The order of a table's tokens: sorted, unless they are positions.
int sort_tokens(const EmbeddingGrad& t, int64_t n, Sorted& l, hipStream_t s) {
  const EmbeddingPlan& p = t.plan;
  l = Sorted{nullptr, nullptr, n, t.ids.rows, t.ids.period > 0 ? n / t.ids.period : 1, t.ids.period};
  if (t.ids.ids == nullptr || n <= 0) return 0;
  SortItems a;
  a.ids = t.ids;
  a.skip = static_cast<uint32_t>(t.skip >= 0 && t.skip < t.ids.rows ? t.skip : t.ids.rows);
  a.keys = nullptr;
  a.tokens = nullptr;
  a.n = n;
  a.per_block = p.per_block;
  a.shift = 0;
  a.bits = p.bits;
  a.keys_out = t.keys;
  a.tokens_out = t.tokens;
  a.marks = t.accumulate ? nullptr : t.marks;
  if (p.one_launch) {
    const auto kernel = p.bits <= 8 ? emb_sort_ranges<8> : emb_sort_ranges<kMaxBits>;
    kernel<<<static_cast<unsigned>(p.sort_blocks), kSortThreads, 0, s>>>(a, p.range);
  } else {
    for (int q = 0; q < p.passes; ++q) {
      const int to = (p.passes - 1 - q) & 1;
      a.keys_out = t.keys + to * n;
      a.tokens_out = t.tokens + to * n;
      emb_sort_count<<<static_cast<unsigned>(p.sort_blocks), kSortThreads, 0, s>>>(a, t.counts);
      emb_sort_place<<<static_cast<unsigned>(p.sort_blocks), kSortThreads, 0, s>>>(a, t.counts);
      a.keys = a.keys_out;
      a.tokens = a.tokens_out;
      a.shift += a.bits;
    }
  }
  l.keys = t.keys;
  l.tokens = t.tokens;
  return static_cast<int>(hipGetLastError());
}

}  // namespace

int embedding_bwd(int dt, const void* dy, int64_t n, int64_t d, const EmbeddingGrad* tables, int count, hipStream_t s) {
  if (d <= 0 || count < 1 || count > 2) return -5;
  int lanes = 1;  // of a narrow chunk, and of a joining block's column slab
  while (lanes < kT && lanes * kCols < d) lanes *= 2;
  const bool wide = lanes >= 64, full = d % kCols == 0;
  const int join_lanes = wide ? 64 : lanes;  // four partial rows at once
  const int64_t slabs = (d + 64 * kCols - 1) / (64 * kCols);
  const int64_t join_slabs = (d + join_lanes * kCols - 1) / (join_lanes * kCols);
  const int64_t units = wide ? kT / 64 : kT / lanes;
  Work w[2];
  int64_t grid = 0;
  for (int i = 0; i < count; ++i) {
    const EmbeddingGrad& t = tables[i];
    const int rc = sort_tokens(t, n, w[i].l, s);
    if (rc != 0) return rc;
    w[i].dw = t.dw;
    w[i].part = t.part;
    w[i].marks = w[i].l.keys != nullptr ? t.marks : nullptr;
    w[i].scale = t.scale;
    w[i].accumulate = t.accumulate;
    w[i].chunk = t.plan.chunk;
    w[i].stream = w[i].l.rows * d * (dt == F32 ? 4 : 2) > kCached;
    w[i].first = grid;
    w[i].blocks = ((wide ? t.plan.chunks * slabs : t.plan.chunks) + units - 1) / units;
    grid += w[i].blocks;
  }
  for (int i = 0; i < count; ++i) {
    w[i].clear = grid;
    w[i].windows = tables[i].accumulate ? 0 : (w[i].l.rows + kZeroRows - 1) / kZeroRows * slabs;
    w[i].clears = w[i].windows < kClears ? w[i].windows : kClears;
    grid += w[i].clears;
  }
  if (count == 1) {
    w[1] = w[0];
    w[1].first = w[1].clear = grid;
    w[1].blocks = 0;
  }
  if (grid >= kMostBlocks || join_slabs > 65535) return -3;
  if (grid == 0) return 0;
  SMPK_DISPATCH(dt, T, {
    if (wide) {
      const auto kernel = full ? emb_bwd_wide<T, true> : emb_bwd_wide<T, false>;
      kernel<<<static_cast<unsigned>(grid), kT, 0, s>>>(w[0], w[1], static_cast<const T*>(dy), static_cast<int>(d),
                                                       static_cast<int>(slabs));
    } else {
      const auto kernel = full ? emb_bwd_narrow<T, true> : emb_bwd_narrow<T, false>;
      kernel<<<static_cast<unsigned>(grid), kT, 0, s>>>(w[0], w[1], static_cast<const T*>(dy), static_cast<int>(d),
                                                       lanes);
    }
    for (int i = 0; i < count; ++i) {
      const EmbeddingPlan& p = tables[i].plan;
      if (!p.join || p.chunks <= 1) continue;
      const auto kernel = full ? emb_bwd_join<T, true> : emb_bwd_join<T, false>;
      kernel<<<dim3(static_cast<unsigned>(p.chunks), static_cast<unsigned>(join_slabs)), kT, 0, s>>>(
          w[i].l, w[i].part, static_cast<int>(d), p.chunk, join_lanes, w[i].scale, static_cast<T*>(w[i].dw),
          w[i].accumulate);
    }
  });
  return static_cast<int>(hipGetLastError());
}

int embedding_bwd_of_short(int dt, const void* dy, int64_t n, int64_t d, const EmbeddingGrad* tables, int count,
                           hipStream_t s) {
  if (d <= 0 || count < 1 || count > 2 || n <= 0 || n > kShortTokens) return -5;
  ShortTables a{};
  a.dy = dy;
  a.n = static_cast<int>(n);
  a.d = static_cast<int>(d);
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    const EmbeddingGrad& t = tables[i];
    const int64_t rows = t.ids.rows, range = (rows + kShortBlocks - 1) / kShortBlocks;
    if (rows < 1 || range > kShortRange || range * d > 0x7fffffff) return -4;
    a.t[i].ids = t.ids;
    a.t[i].skip = static_cast<uint32_t>(t.skip >= 0 && t.skip < rows ? t.skip : rows);
    a.t[i].dw = t.dw;
    a.t[i].scale = t.scale;
    a.t[i].accumulate = t.accumulate;
    a.t[i].range = static_cast<int>(range);
    a.t[i].blocks = static_cast<int>((rows + range - 1) / range);
    blocks += a.t[i].blocks;
  }
  SMPK_DISPATCH(dt, T, {
    const auto kernel = d % kCols == 0 ? emb_bwd_short<T, true> : emb_bwd_short<T, false>;
    kernel<<<static_cast<unsigned>(blocks), kT, 0, s>>>(a);
  });
  return static_cast<int>(hipGetLastError());
}

}  // namespace smpk

// Token embedding: y[t] = scale * W[id_t - start] (+ P[pos_t]), and the gradients of both tables.
//
// Forward: a gather, bound by HBM: it writes every row and reads it from the table (or the
// caches, for the frequent tokens).  The sum is formed in fp32 and rounded once.
//
// Backward: dW[v] = scale * sum of dy[t] over the tokens with id_t = v, in token order and in
// fp32, so that the result does not depend on the order in which blocks run.
#include "common.h"
#include "kernels.h"

namespace smpk {
namespace {

constexpr int kT = 256;
constexpr int64_t kShortSort = 16384;

// Row of a table for one token, or -1 where the id is not one of its rows.
__device__ __forceinline__ int64_t row_of(const IndexList& l, int64_t t) {
  int64_t id;
  if (l.ids == nullptr) {
    id = t % l.period;
  } else {
    id = l.wide ? static_cast<const int64_t*>(l.ids)[t] : static_cast<const int32_t*>(l.ids)[t];
  }
  id -= l.start;
  return id >= 0 && id < l.rows ? id : -1;
}

template <typename T, int N>
struct Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_pack(const T* p, float (&o)[N]) {
  if constexpr (N > 1) {
    const Vec16<T> a = load16(p);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = to_f32(a.v[j]);
  } else {
    o[0] = to_f32(*p);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const float (&o)[N]) {
  if constexpr (N > 1) {
    Vec16<T> a;
#pragma unroll
    for (int j = 0; j < N; ++j) a.v[j] = from_f32<T>(o[j]);
    store16(p, a);
  } else {
    *p = from_f32<T>(o[0]);
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(kT) emb_fwd(IndexList ids, const T* __restrict__ w, int64_t w_stride, float scale,
                                              int foreign_zero, IndexList pos, const T* __restrict__ p,
                                              int64_t p_stride, T* __restrict__ y, int64_t n, int d) {
  const int per_row = d / N;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kT + threadIdx.x;
  if (i >= n * per_row) return;
  const int64_t t = i / per_row;
  const int c = static_cast<int>(i - t * per_row) * N;
  const int64_t r = row_of(ids, t);
  float o[N];
  if (r >= 0) {
    load_pack<T, N>(w + r * w_stride + c, o);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= scale;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = foreign_zero ? 0.f : NAN;
  }
  if (p != nullptr) {
    const int64_t q = row_of(pos, t);
    float a[N];
    if (q >= 0) {
      load_pack<T, N>(p + q * p_stride + c, a);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) a[j] = NAN;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] += a[j];
  }
  store_pack<T, N>(y + t * d + c, o);
}

// ----------------------------------------------------------------------- sorting the tokens
// Stable radix sort of (row, token), least significant digit first: a row number has at most 10
// bits a pass, so a vocabulary of up to 2^20 rows takes two.  A block of 16 waves owns a
// consecutive run of the items, each wave a consecutive part of it; the waves count their digits,
// the counts become the places of each wave's items, and the wave walks over its items once more,
// 64 at a time, in order.  No place depends on the order in which anything runs.
constexpr int kWaves = 16;
constexpr int kSortThreads = kWaves * 64;
constexpr int kMaxBits = 10;

struct SortItems {
  IndexList ids;  // first pass: keys and tokens come from the ids
  int64_t skip;
  const uint32_t* keys;  // later passes (null in the first)
  const int32_t* tokens;
  uint32_t* keys_out;
  int32_t* tokens_out;
  int64_t n, per_block;  // per_block: a multiple of kSortThreads
  int shift, bits;
};

// Rows' keys are their numbers; tokens without a row come last, with the key `rows`.
__device__ __forceinline__ uint32_t key_of(const SortItems& a, int64_t i) {
  if (a.keys != nullptr) return a.keys[i];
  const int64_t r = row_of(a.ids, i);
  return static_cast<uint32_t>(r < 0 || r == a.skip ? a.ids.rows : r);
}

__device__ __forceinline__ void wave_run(const SortItems& a, int block, int64_t& s, int64_t& e) {
  const int64_t part = a.per_block / kWaves;
  s = static_cast<int64_t>(block) * a.per_block + (threadIdx.x >> 6) * part;
  e = s + part < a.n ? s + part : a.n;
}

__global__ void __launch_bounds__(kSortThreads) emb_sort_count(SortItems a, int32_t* __restrict__ counts) {
  __shared__ int32_t cnt[1 << kMaxBits];
  const int bins = 1 << a.bits;
  for (int d = threadIdx.x; d < bins; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  int64_t s, e;
  wave_run(a, blockIdx.x, s, e);
  for (int64_t i = s + (threadIdx.x & 63); i < e; i += 64) atomicAdd(&cnt[(key_of(a, i) >> a.shift) & (bins - 1)], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) counts[static_cast<int64_t>(blockIdx.x) * bins + d] = cnt[d];
}

// One pass of one block.  counts [blocks][bins]: of all blocks (a single block needs none).
__device__ __forceinline__ void sort_pass(const SortItems& a, const int32_t* counts, int blocks, int block,
                                          int32_t (*cnt)[1 << kMaxBits], int32_t* wave_total) {
  const int bins = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  for (int d = lane; d < bins; d += 64) cnt[wid][d] = 0;
  __syncthreads();
  int64_t s, e;
  wave_run(a, block, s, e);
  for (int64_t i = s + lane; i < e; i += 64) atomicAdd(&cnt[wid][(key_of(a, i) >> a.shift) & (bins - 1)], 1);
  __syncthreads();
  // thread d owns digit d: items with smaller digits anywhere, then of this digit in earlier blocks
  int total = 0, before = 0;
  if (tid < bins) {
    if (blocks == 1) {
      for (int w = 0; w < kWaves; ++w) total += cnt[w][tid];
    } else {
      for (int b = 0; b < blocks; ++b) {
        const int c = counts[static_cast<int64_t>(b) * bins + tid];
        total += c;
        before += b < block ? c : 0;
      }
    }
  }
  int incl = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(incl, o, 64);
    if (lane >= o) incl += v;
  }
  if (lane == 63) wave_total[wid] = incl;
  __syncthreads();
  int base = incl - total + before;
  for (int w = 0; w < wid; ++w) base += wave_total[w];
  if (tid < bins) {
    for (int w = 0; w < kWaves; ++w) {
      const int c = cnt[w][tid];
      cnt[w][tid] = base;
      base += c;
    }
  }
  __syncthreads();
  for (int64_t i0 = s; i0 < e; i0 += 64) {
    const int64_t i = i0 + lane;
    const bool valid = i < e;
    const uint32_t key = valid ? key_of(a, i) : 0u;
    const int digit = (key >> a.shift) & (bins - 1);
    uint64_t same = __ballot(valid);  // the lanes with this lane's digit
    for (int b = 0; b < a.bits; ++b) {
      const bool one = (digit >> b) & 1;
      const uint64_t m = __ballot(one);
      same &= one ? m : ~m;
    }
    const int first = valid ? __ffsll(static_cast<unsigned long long>(same)) - 1 : lane;
    int at = 0;
    if (valid && lane == first) at = atomicAdd(&cnt[wid][digit], __popcll(same));
    at = __shfl(at, first, 64) + __popcll(same & ((1ull << lane) - 1));
    if (valid) {
      a.keys_out[at] = key;
      a.tokens_out[at] = a.tokens != nullptr ? a.tokens[i] : static_cast<int32_t>(i);
    }
  }
}

__global__ void __launch_bounds__(kSortThreads) emb_sort_place(SortItems a, const int32_t* __restrict__ counts) {
  __shared__ int32_t cnt[kWaves][1 << kMaxBits];
  __shared__ int32_t wave_total[kWaves];
  sort_pass(a, counts, gridDim.x, blockIdx.x, cnt, wave_total);
}

// All passes of a short list in one block; the result lies in keys_out / tokens_out.
__global__ void __launch_bounds__(kSortThreads) emb_sort_short(SortItems a, uint32_t* keys2, int32_t* tokens2,
                                                               int passes) {
  __shared__ int32_t cnt[kWaves][1 << kMaxBits];
  __shared__ int32_t wave_total[kWaves];
  uint32_t* k[2] = {a.keys_out, keys2};
  int32_t* t[2] = {a.tokens_out, tokens2};
  for (int p = 0; p < passes; ++p) {
    const int to = (passes - 1 - p) & 1;
    a.keys_out = k[to];
    a.tokens_out = t[to];
    sort_pass(a, nullptr, 1, 0, cnt, wave_total);
    __syncthreads();
    a.keys = k[to];
    a.tokens = t[to];
    a.shift += a.bits;
  }
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

constexpr int kCols = 8;    // columns of a thread
constexpr int kAhead = 8;  // rows whose loads are in flight together

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Any16 {
  T v[16 / sizeof(T)];
};
template <typename T>
struct Raw8 {
  Any16<T> a[kCols * sizeof(T) / 16];
};

template <typename T>
__device__ __forceinline__ void read8(const T* p, int left, Raw8<T>& r) {
  constexpr int M = 16 / sizeof(T);
  if (left >= kCols) {
#pragma unroll
    for (int k = 0; k < kCols / M; ++k) __builtin_memcpy(&r.a[k], p + k * M, 16);
  } else {
#pragma unroll
    for (int j = 0; j < kCols; ++j) r.a[j / M].v[j % M] = j < left ? p[j] : from_f32<T>(0.f);
  }
}
template <typename T>
__device__ __forceinline__ float at8(const Raw8<T>& r, int j) {
  constexpr int M = 16 / sizeof(T);
  return to_f32(r.a[j / M].v[j % M]);
}
template <typename T>
__device__ __forceinline__ void write8(T* p, int left, const float (&o)[kCols]) {
  constexpr int M = 16 / sizeof(T);
  if (left >= kCols) {
#pragma unroll
    for (int k = 0; k < kCols / M; ++k) {
      Any16<T> a;
#pragma unroll
      for (int j = 0; j < M; ++j) a.v[j] = from_f32<T>(o[k * M + j]);
      __builtin_memcpy(p + k * M, &a, 16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (j < left) p[j] = from_f32<T>(o[j]);
  }
}

// dw row = scale * sum, or that added to the row
template <typename T>
__device__ __forceinline__ void write_row(T* p, int left, float (&sum)[kCols], float scale, int accumulate) {
  if (accumulate) {
    Raw8<T> r;
    read8(p, left, r);
#pragma unroll
    for (int j = 0; j < kCols; ++j) sum[j] = fmaf(sum[j], scale, at8(r, j));
  } else {
#pragma unroll
    for (int j = 0; j < kCols; ++j) sum[j] *= scale;
  }
  write8(p, left, sum);
}

// `lanes` threads (a power of two) hold a chunk's columns, kT / lanes chunks a block
template <typename T>
__global__ void __launch_bounds__(kT) emb_bwd_chunks(Sorted l, const T* __restrict__ dy, int d, int chunk, int lanes,
                                                     float scale, T* __restrict__ dw, int accumulate,
                                                     float* __restrict__ part) {
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * (kT / lanes) + threadIdx.x / lanes;
  const int c = (blockIdx.y * lanes + threadIdx.x % lanes) * kCols;
  const int left = d - c;
  const int64_t j0 = ch * chunk, j1 = j0 + chunk < l.n ? j0 + chunk : l.n;
  if (j0 >= l.n || left <= 0) return;
  uint32_t cur = l.key(j0);
  bool head = j0 > 0 && l.key(j0 - 1) == cur;
  float sum[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) sum[j] = 0.f;
  for (int64_t j = j0; j < j1; j += kAhead) {
    uint32_t key[kAhead];
    Raw8<T> row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) key[u] = j + u < j1 ? l.key(j + u) : static_cast<uint32_t>(l.rows);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (key[u] < l.rows) read8(dy + l.token(j + u, key[u]) * d + c, left, row[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (key[u] != cur && j + u < j1) {
        if (head) {
          write8(part + (2 * ch) * d + c, left, sum);
        } else {
          write_row(dw + static_cast<int64_t>(cur) * d + c, left, sum, scale, accumulate);
        }
        head = false;
        cur = key[u];
#pragma unroll
        for (int q = 0; q < kCols; ++q) sum[q] = 0.f;
      }
      if (key[u] < l.rows) {
#pragma unroll
        for (int q = 0; q < kCols; ++q) sum[q] += at8(row[u], q);
      }
    }
    if (cur >= l.rows) return;  // only tokens without a row follow
  }
  const bool tail = j1 < l.n && l.key(j1) == cur;
  if (head || tail) {
    write8(part + (2 * ch + (head ? 0 : 1)) * d + c, left, sum);
  } else {
    write_row(dw + static_cast<int64_t>(cur) * d + c, left, sum, scale, accumulate);
  }
}

// the first place whose key is not below k
__device__ __forceinline__ int64_t lower_bound(const Sorted& l, uint32_t k) {
  if (l.keys == nullptr) {
    const int64_t j = static_cast<int64_t>(k) * l.batch;
    return j < l.n ? j : l.n;
  }
  int64_t lo = 0, hi = l.n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (l.keys[mid] < k) {
      lo = mid + 1;
    } else {
      hi = mid;
    }
  }
  return lo;
}

constexpr int kZeroRows = 64;  // rows of a block that clears what no token touched

// Blocks 0 .. chunks - 1 join the run that begins in that chunk and goes on behind it; further
// blocks (a dense gradient) write zeros to the rows that no token has.
template <typename T>
__global__ void __launch_bounds__(kT) emb_bwd_join(Sorted l, const float* __restrict__ part, int d, int chunk,
                                                   int64_t chunks, int lanes, float scale, T* __restrict__ dw,
                                                   int accumulate) {
  __shared__ float buf[kT][kCols];
  const int tid = threadIdx.x, lane = tid % lanes, g = tid / lanes, groups = kT / lanes;
  const int c = (blockIdx.y * lanes + lane) * kCols, left = d - c;
  if (blockIdx.x >= chunks) {
    const int64_t r0 = (blockIdx.x - chunks) * kZeroRows;
    const int64_t mine = r0 + (tid & 63);
    bool empty = false;
    if (mine < l.rows) {
      const int64_t j = lower_bound(l, static_cast<uint32_t>(mine));
      empty = j >= l.n || l.key(j) != mine;
    }
    const uint64_t rows = __ballot(empty);  // the same in all waves
    const float zero[kCols] = {};
    for (int r = g; r < kZeroRows; r += groups)
      if (((rows >> r) & 1) && left > 0) write8(dw + (r0 + r) * d + c, left, zero);
    return;
  }
  const int64_t ch = blockIdx.x, j0 = ch * chunk, j1 = j0 + chunk;
  if (j1 >= l.n) return;
  const uint32_t k = l.key(j1);
  if (k >= l.rows || l.key(j1 - 1) != k || (j0 > 0 && l.key(j0) == k && l.key(j0 - 1) == k)) return;
  const int64_t last = (lower_bound(l, k + 1) - 1) / chunk;  // the run's last chunk
  float sum[kCols];
#pragma unroll
  for (int q = 0; q < kCols; ++q) sum[q] = 0.f;
  if (left > 0) {
    for (int64_t m = ch + g; m <= last; m += groups) {
      Raw8<float> r;
      read8(part + (2 * m + (m == ch ? 1 : 0)) * d + c, left, r);
#pragma unroll
      for (int q = 0; q < kCols; ++q) sum[q] += at8(r, q);
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
  write_row(dw + static_cast<int64_t>(k) * d + c, left, sum, scale, accumulate);
}

bool packs(int64_t d, int64_t stride, const void* p, int es) {
  return (d * es) % 16 == 0 && (stride * es) % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

}  // namespace

int embedding_fwd(int dt, const IndexList& ids, const void* w, int64_t w_stride, float scale, int foreign_zero,
                  const IndexList& pos, const void* p, int64_t p_stride, void* y, int64_t n, int64_t d,
                  hipStream_t s) {
  if (n <= 0 || d <= 0) return 0;
  SMPK_DISPATCH(dt, T, {
    const int es = sizeof(T);
    const bool vec = packs(d, w_stride, w, es) && packs(d, d, y, es) && (p == nullptr || packs(d, p_stride, p, es));
    const int64_t items = n * (vec ? d / Vec16<T>::N : d);
    const int64_t blocks = (items + kT - 1) / kT;
    if (blocks > 0x7fffffff) return -3;
    if (vec) {
      emb_fwd<T, Vec16<T>::N><<<static_cast<unsigned>(blocks), kT, 0, s>>>(
          ids, static_cast<const T*>(w), w_stride, scale, foreign_zero, pos, static_cast<const T*>(p), p_stride,
          static_cast<T*>(y), n, static_cast<int>(d));
    } else {
      emb_fwd<T, 1><<<static_cast<unsigned>(blocks), kT, 0, s>>>(
          ids, static_cast<const T*>(w), w_stride, scale, foreign_zero, pos, static_cast<const T*>(p), p_stride,
          static_cast<T*>(y), n, static_cast<int>(d));
    }
  });
  return static_cast<int>(hipGetLastError());
}

EmbeddingPlan embedding_bwd_plan(int64_t n, int64_t d, int64_t rows, bool sorted) {
  EmbeddingPlan p;
  int bits = 1;
  while ((rows >> bits) != 0) ++bits;  // the keys 0 .. rows
  p.passes = sorted ? 0 : (bits + kMaxBits - 1) / kMaxBits;
  p.bits = sorted ? 0 : (bits + p.passes - 1) / p.passes;
  // one block sorts a short list alone, in one launch; longer ones go in runs of 2048 tokens or,
  // above 256 blocks, whose counts every block reads, in longer runs
  const int64_t parts = n <= kShortSort ? 1 : ((n + 2047) / 2048 < 256 ? (n + 2047) / 2048 : 256);
  p.per_block = ((n + parts - 1) / parts + kSortThreads - 1) / kSortThreads * kSortThreads;
  p.sort_blocks = n > 0 ? (n + p.per_block - 1) / p.per_block : 0;
  int64_t c = 16;  // tokens of a chunk: long ones leave fewer partial sums, short ones more to run at once
  while (c < 64 && n / (c * 2) >= 1024) c *= 2;
  p.chunk = static_cast<int>(c);
  p.chunks = (n + c - 1) / c;
  return p;
}

int embedding_bwd(int dt, const IndexList& ids, const void* dy, int64_t n, int64_t d, float scale, int64_t skip,
                  void* dw, int accumulate, const EmbeddingPlan& p, uint32_t* keys, int32_t* tokens, int32_t* counts,
                  float* part, hipStream_t s) {
  if (ids.rows <= 0 || d <= 0 || (n <= 0 && accumulate)) return 0;
  Sorted l{nullptr, nullptr, n, ids.rows, ids.period > 0 ? n / ids.period : 1, ids.period};
  if (ids.ids != nullptr && n > 0) {
    SortItems a;
    a.ids = ids;
    a.skip = skip;
    a.keys = nullptr;
    a.tokens = nullptr;
    a.n = n;
    a.per_block = p.per_block;
    a.shift = 0;
    a.bits = p.bits;
    a.keys_out = keys;
    a.tokens_out = tokens;
    if (p.sort_blocks == 1) {
      emb_sort_short<<<1, kSortThreads, 0, s>>>(a, keys + n, tokens + n, p.passes);
    } else {
      for (int q = 0; q < p.passes; ++q) {
        const int to = (p.passes - 1 - q) & 1;
        a.keys_out = keys + to * n;
        a.tokens_out = tokens + to * n;
        emb_sort_count<<<static_cast<unsigned>(p.sort_blocks), kSortThreads, 0, s>>>(a, counts);
        emb_sort_place<<<static_cast<unsigned>(p.sort_blocks), kSortThreads, 0, s>>>(a, counts);
        a.keys = a.keys_out;
        a.tokens = a.tokens_out;
        a.shift += a.bits;
      }
    }
    l.keys = keys;
    l.tokens = tokens;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return static_cast<int>(e);
  }
  int lanes = 1;
  while (lanes < kT && lanes * kCols < d) lanes *= 2;
  const unsigned slabs = static_cast<unsigned>((d + lanes * kCols - 1) / (lanes * kCols));
  const int64_t per = kT / lanes, zero = accumulate ? 0 : (ids.rows + kZeroRows - 1) / kZeroRows;
  if (slabs > 65535 || p.chunks + zero > 0x7fffffff) return -3;
  SMPK_DISPATCH(dt, T, {
    if (p.chunks > 0)
      emb_bwd_chunks<T><<<dim3(static_cast<unsigned>((p.chunks + per - 1) / per), slabs), kT, 0, s>>>(
          l, static_cast<const T*>(dy), static_cast<int>(d), p.chunk, lanes, scale, static_cast<T*>(dw), accumulate,
          part);
    if (p.chunks + zero > 0)
      emb_bwd_join<T><<<dim3(static_cast<unsigned>(p.chunks + zero), slabs), kT, 0, s>>>(
          l, part, static_cast<int>(d), p.chunk, p.chunks, lanes, scale, static_cast<T*>(dw), accumulate);
  });
  return static_cast<int>(hipGetLastError());
}

}  // namespace smpk

// The norms around a transformer block in one pass over the hidden state:
//
//   h = N2(x)  (x: the block's output; no norm: h = x)     N(v) = (v - mean) * rstd * w + b
//   s = residual + alpha * g * h                           root-mean-square norms: mean = 0
//   y = N1(s)  (the next block's input)
//
// and backward, with dS = ds + N1^T(dy):
//
//   d residual = dS,  dh = alpha g dS,  dg = alpha sum dS h,  dx = N2^T(dh),
//   dw1 = sum dy n1, db1 = sum dy, dw2 = sum dh n2, db2 = sum dh      (n: normalised values)
//   N^T(d) = rstd * (d w - mean(d w) - n mean(d w n))
//
// Bound by HBM: forward reads x, residual and writes s, y; backward reads x, residual, dy, ds and
// writes two gradients.  A row stays in registers from its load to its store.  The norm is taken
// of s before s is rounded, and the backward forms the same fp32 s again from x and residual --
// it has to read x in any case, and s in 16 bits would cost the fp32 weight gradients 1e-3 of
// their value.
//
// A thread holds 8 consecutive elements of a row (V times that for wide rows).  Rows of up to 256
// elements share a wave: 8, 16 or 32 lanes each (40 M elements in rows of 64 bf16: 56 us forward,
// 297 us with a wave for each).  Forward, rows of up to 2048 elements belong to one wave each: no
// barrier, and the rows of a CU's waves overlap freely.  Wider rows, and all wider rows of the
// backward, belong to a team of waves.
//
// Measured, bf16: 16384 x 1600 with a gate, forward 45 us (4.7 TB/s), backward 65 us (4.8 TB/s);
// 16384 x 4096 root-mean-square with fp32 weights, 105 us and 168 us (4.8 TB/s); a copy of 1 GiB
// reaches 5.1 TB/s.
#include "kernels.h"
#include "vec8.h"

namespace smpk {
namespace {

// How a row splits into vectors: into whole ones; into whole ones of which the last begins before the
// end of the one before it, whose elements both hold and write -- the same values -- and one counts in
// the sums over the row; or, in rows of less than one vector, element by element.  40 M bf16 elements in
// rows of 1601: 69 us forward, 125 us backward; with the last vector element by element 84 and 181 us.
enum Rows { kWhole, kOverlap, kShort };

// First column of a thread's vector; `left`, at most kCols for the last one, from there to the row's end.
template <int R>
__device__ __forceinline__ int column(int vector, int d, int& left) {
  const int c = vector * kCols;
  left = d - c;
  return R == kOverlap && left < kCols ? d - kCols : c;
}

// Element j counts in sums over the row.
template <int R>
__device__ __forceinline__ bool counts(int j, int left) {
  return R == kWhole || (R == kOverlap ? j + left >= kCols : j < left);
}

// A vector that may be absent (`other` then) and of either T or fp32.
template <int R, typename T>
__device__ __forceinline__ void read_opt(const void* p, bool f32, int64_t at, int left, float other, float (&o)[kCols]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < kCols; ++j) o[j] = other;
  } else if (f32) {
    read8<R != kShort>(static_cast<const float*>(p) + at, left, o);
  } else {
    read8<R != kShort>(static_cast<const T*>(p) + at, left, o);
  }
}

// Sums over a team: SUB lanes of a wave (8, 16 or 32; 0: whole waves).
template <int SUB>
struct Team {
  float* smem;  // [2][2][16]
  int first, waves, slot;  // `slot` alternates so that one barrier suffices

  __device__ __forceinline__ static float in_wave(float v) {
    if constexpr (SUB == 0) {
      return wave_sum_fixed(v);
    } else {
#pragma unroll
      for (int o = 1; o < SUB; o <<= 1) v += __shfl_xor(v, o, 64);
      return v;
    }
  }
  __device__ __forceinline__ void sum2(float& a, float& b) {
    a = in_wave(a);
    b = in_wave(b);
    if (SUB != 0 || waves == 1) return;
    float* s = smem + slot * 32;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) {
      s[threadIdx.x >> 6] = a;
      s[16 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.f;
    for (int k = 0; k < waves; ++k) {
      a += s[first + k];
      b += s[16 + first + k];
    }
  }
  __device__ __forceinline__ void sum1(float& a) {
    a = in_wave(a);
    if (SUB != 0 || waves == 1) return;
    float* s = smem + slot * 32;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
    __syncthreads();
    a = 0.f;
    for (int k = 0; k < waves; ++k) a += s[first + k];
  }
};

// Mean, then the mean square of the differences: values of any offset keep their deviation.
template <int V, int R, int SUB>
__device__ __forceinline__ void moments(const float (&v)[V][kCols], const int (&left)[V], int d, float eps, bool rms,
                                        Team<SUB>& team, float& mean, float& rstd) {
  mean = 0.f;
  if (!rms) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int j = 0; j < kCols; ++j) a += counts<R>(j, left[k]) ? v[k][j] : 0.f;
    team.sum1(a);
    mean = a / d;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    if (left[k] <= 0) continue;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const float c = counts<R>(j, left[k]) ? v[k][j] - mean : 0.f;
      q = fmaf(c, c, q);
    }
  }
  team.sum1(q);
  rstd = rsqrtf(q / d + eps);
}

// threads_of_row threads for a row: SUB, 64 (and blockDim.x / that rows a block), or all of the block
template <typename T, int V, int R, int SUB>
__global__ void __launch_bounds__(1024) block_norm_fwd(BlockNormArgs a, int threads_of_row) {
  __shared__ float smem[64];
  const int team_size = SUB != 0 ? SUB : threads_of_row;
  const int tid = threadIdx.x, lane = team_size <= 64 ? tid & (team_size - 1) : tid;
  Team<SUB> team{smem, 0, team_size / 64, 0};
  int64_t row = blockIdx.x;
  if (SUB != 0) row = row * (blockDim.x / team_size) + tid / team_size;
  if (SUB == 0 && team_size == 64) row = row * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(tid >> 6);
  row += a.first_row;
  if (row >= a.rows) return;  // (all lanes of their own rows: no barrier or sum follows for them)
  int col[V], left[V];
  float s[V][kCols], h[V][kCols];
  Raw8<T> rs[V], rh[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = col[k] = column<R>(k * team_size + lane, a.d, left[k]);
    if (left[k] <= 0) continue;
    if (a.x != nullptr) read8<R != kShort>(static_cast<const T*>(a.x) + row * a.d + c, left[k], rh[k]);
    read8<R != kShort>(static_cast<const T*>(a.res) + row * a.d + c, left[k], rs[k]);
  }
#pragma unroll
  for (int k = 0; k < V; ++k)
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      h[k][j] = left[k] > 0 && a.x != nullptr ? at8(rh[k], j) : 0.f;
      s[k][j] = left[k] > 0 ? at8(rs[k], j) : 0.f;
    }
  float mean2 = 0.f, rstd2 = 1.f, mean1, rstd1;
  if (a.x != nullptr) {
    if (a.pw != nullptr) moments<V, R, SUB>(h, left, a.d, a.eps, a.rms, team, mean2, rstd2);
    const int64_t gate_row = a.gate != nullptr ? row / a.gate_rows * a.d : 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = col[k];
      if (left[k] <= 0) continue;
      float w[kCols], b[kCols], g[kCols];
      read_opt<R, T>(a.pw, a.w_f32, c, left[k], 1.f, w);
      read_opt<R, T>(a.pb, a.w_f32, c, left[k], 0.f, b);
      read_opt<R, T>(a.gate, a.gate_f32, gate_row + c, left[k], 1.f, g);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const float v = fmaf((h[k][j] - mean2) * rstd2, w[j], b[j]);
        s[k][j] = fmaf(a.alpha * g[j], v, s[k][j]);
      }
      write8<R != kShort, true>(static_cast<T*>(a.s) + row * a.d + c, left[k], s[k]);
    }
  }
  moments<V, R, SUB>(s, left, a.d, a.eps, a.rms, team, mean1, rstd1);
  if (lane == 0 && a.stats != nullptr)
    reinterpret_cast<float4*>(a.stats)[row] = make_float4(mean1, rstd1, mean2, rstd2);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = col[k];
    if (left[k] <= 0) continue;
    float w[kCols], b[kCols];
    read_opt<R, T>(a.w, a.w_f32, c, left[k], 1.f, w);
    read_opt<R, T>(a.b, a.w_f32, c, left[k], 0.f, b);
#pragma unroll
    for (int j = 0; j < kCols; ++j) w[j] = fmaf((s[k][j] - mean1) * rstd1, w[j], b[j]);
    write8<R != kShort, true>(static_cast<T*>(a.y) + row * a.d + c, left[k], w);
  }
}

// A unit (one team) takes consecutive rows of one gate row.  split > 1: `split` units share the rows
// of a gate row; split == 1: a unit takes whole gate rows, `units` apart.
struct Walk {
  int row, gate;
  int at, count;  // at-th of the unit's `count` rows of this gate row
  bool live;
  __device__ __forceinline__ Walk(const BlockNormArgs& a, int unit) {
    const int rows = static_cast<int>(a.gate_rows), split = static_cast<int>(a.split);
    const int chunk = (rows + split - 1) / split, first = unit % split * chunk;
    gate = unit / split;
    at = 0;
    count = rows - first < chunk ? rows - first : chunk;
    live = gate < a.groups && count > 0;
    row = live ? gate * rows + first : 0;
  }
  // the gate row ends with this row, and all of it was this unit's
  __device__ __forceinline__ bool last(const BlockNormArgs& a) const { return a.split == 1 && at == count - 1; }
  __device__ __forceinline__ void next(const BlockNormArgs& a, int units) {
    ++row;
    if (++at < count) return;
    at = 0;
    live = live && a.split == 1 && a.groups - gate > units;
    gate = live ? gate + units : 0;
    row = gate * static_cast<int>(a.gate_rows);
  }
};

enum { kW1, kB1, kW2, kB2, kG, kSums };

// A whole gate row's gradient, alpha * sum.
template <typename T, int R>
__device__ __forceinline__ void write_gate(const BlockNormArgs& a, int64_t gate, int c, int left, float (&sum)[kCols]) {
#pragma unroll
  for (int j = 0; j < kCols; ++j) sum[j] *= a.alpha;
  if (a.gate_f32) {
    write8<R != kShort, true>(static_cast<float*>(a.dgate) + gate * a.d + c, left, sum);
  } else {
    write8<R != kShort, true>(static_cast<T*>(a.dgate) + gate * a.d + c, left, sum);
  }
}

// A row's loads, issued while the row before is worked on.
template <typename T>
struct RowData {
  Raw8<T> x, res, dy, ds;
  float4 st;
};

template <typename T, int R>
__device__ __forceinline__ void load_row(const BlockNormArgs& a, int64_t row, int c, int left, RowData<T>& r) {
  if (left <= 0) return;
  const int64_t at = row * a.d + c;
  read8<R != kShort>(static_cast<const T*>(a.res) + at, left, r.res);
  if (a.x != nullptr) read8<R != kShort>(static_cast<const T*>(a.x) + at, left, r.x);
  if (a.dy != nullptr) read8<R != kShort>(static_cast<const T*>(a.dy) + at, left, r.dy);
  if (a.ds != nullptr) read8<R != kShort>(static_cast<const T*>(a.ds) + at, left, r.ds);
}

template <typename T, int R>
__device__ __forceinline__ void fetch(const BlockNormArgs& a, const Walk& t, int c, int left, RowData<T>& r) {
  if (!t.live || left <= 0) return;
  r.st = reinterpret_cast<const float4*>(a.stats)[t.row];
  load_row<T, R>(a, t.row, c, left, r);
}

// Rows of up to 6144 elements, one vector a thread, with the column sums in registers.  The weights
// stay there too, in their own type W (T or fp32): a unit works on many rows.  These registers
// allow 12 waves a CU.
template <typename T, typename W, int R, int SUB>
__global__ void __launch_bounds__(768) block_norm_bwd(BlockNormArgs a, int threads_of_row, int iterations) {
  // past the caches where the stores fill whole lines, or nearly: rows of 1601 bf16 125 us so, 127 us
  // stored normally, but rows of 101 174 and 152 us, and of 1600 fp32 226 and 211 us
  constexpr bool kStream = sizeof(T) == 2 && (R == kWhole || SUB == 0);
  extern __shared__ float lds[];  // [64] reductions, then [team_size * kCols] to join the teams' sums
  const int team_size = SUB != 0 ? SUB : threads_of_row;
  const int tid = threadIdx.x, teams = blockDim.x / team_size;
  const int tm = SUB != 0 ? tid / team_size : __builtin_amdgcn_readfirstlane(tid / team_size);
  int left;
  const int lane = tid - tm * team_size, c = column<R>(lane, a.d, left);
  Team<SUB> team{lds, tm * (team_size / 64), team_size / 64, 0};
  const int unit = blockIdx.x * teams + tm, units = gridDim.x * teams;
  float sum[kSums][kCols];
  Raw8<W> w, pw, pb;
  float ag[kCols];  // alpha * gate
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    w.v[j] = pw.v[j] = from_f32<W>(1.f);
    pb.v[j] = from_f32<W>(0.f);
    ag[j] = a.alpha;
#pragma unroll
    for (int q = 0; q < kSums; ++q) sum[q][j] = 0.f;
  }
  if (left > 0) {
    read8<R != kShort>(static_cast<const W*>(a.w) + c, left, w);
    if (a.pw != nullptr) read8<R != kShort>(static_cast<const W*>(a.pw) + c, left, pw);
    if (a.pb != nullptr) read8<R != kShort>(static_cast<const W*>(a.pb) + c, left, pb);
  }
  int gate_now = -1;
  RowData<T> r;
  Walk t(a, unit);
  fetch<T, R>(a, t, c, left, r);

  for (int i = 0; i < iterations; ++i) {
    if (a.gate != nullptr && t.live && t.gate != gate_now && left > 0) {
      gate_now = t.gate;
      read_opt<R, T>(a.gate, a.gate_f32, static_cast<int64_t>(t.gate) * a.d + c, left, 1.f, ag);
#pragma unroll
      for (int j = 0; j < kCols; ++j) ag[j] *= a.alpha;
    }
    float n1[kCols], n2[kCols], dy[kCols], ds[kCols];
    const float4 st = r.st;
    const bool live = t.live && left > 0;
    float p = 0.f, q = 0.f;
    if (live) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        n1[j] = at8(r.res, j);
        n2[j] = 0.f;
        ds[j] = a.ds != nullptr ? at8(r.ds, j) : 0.f;
      }
      if (a.x != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          n2[j] = (at8(r.x, j) - st.z) * st.w;
          n1[j] = fmaf(ag[j], fmaf(n2[j], at8(pw, j), at8(pb, j)), n1[j]);
        }
      }
      if (a.dy != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          const float g = at8(r.dy, j);
          n1[j] = (n1[j] - st.x) * st.y;
          sum[kW1][j] = fmaf(g, n1[j], sum[kW1][j]);
          sum[kB1][j] += g;
          dy[j] = g * at8(w, j);
          const float own = counts<R>(j, left) ? dy[j] : 0.f;
          p += own;
          q = fmaf(own, n1[j], q);
        }
      }
    }
    const int64_t at = static_cast<int64_t>(t.row) * a.d + c;
    const int gate = t.gate;
    const bool last = t.last(a);
    t.next(a, units);
    if (i + 1 < iterations) fetch<T, R>(a, t, c, left, r);
    if (a.dy != nullptr) {
      team.sum2(p, q);
      p = a.rms ? 0.f : p / a.d;
      q /= a.d;
    }
    float u = 0.f, v = 0.f;
    if (live) {
      if (a.dy != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) ds[j] = fmaf(st.y, dy[j] - p - n1[j] * q, ds[j]);
      }
      if (a.dres != nullptr) write8<R != kShort, kStream>(static_cast<T*>(a.dres) + at, left, ds);
      if (a.x != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          sum[kG][j] = fmaf(ds[j], fmaf(n2[j], at8(pw, j), at8(pb, j)), sum[kG][j]);
          const float dh = ds[j] * ag[j];
          sum[kW2][j] = fmaf(dh, n2[j], sum[kW2][j]);
          sum[kB2][j] += dh;
          ds[j] = dh * at8(pw, j);  // the gradient of n2; of x itself without a norm
          const float own = counts<R>(j, left) ? ds[j] : 0.f;
          u += own;
          v = fmaf(own, n2[j], v);
        }
      }
    }
    if (a.pw != nullptr) {
      team.sum2(u, v);
      u = a.rms ? 0.f : u / a.d;
      v /= a.d;
    } else {
      u = v = 0.f;
    }
    if (live && a.x != nullptr) {
      if (a.dx != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) ds[j] = st.w * (ds[j] - u - n2[j] * v);
        write8<R != kShort, kStream>(static_cast<T*>(a.dx) + at, left, ds);
      }
      if (a.gate_direct && last) {
        write_gate<T, R>(a, gate, c, left, sum[kG]);
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[kG][j] = 0.f;
      }
    }
  }

  // partial sums: of the teams together for the vectors, of each unit for its gate row
#pragma unroll
  for (int j = 0; j < kCols; ++j) sum[kG][j] *= a.alpha;
  if (a.gate_part != nullptr && left > 0)
    write8<R != kShort, false>(a.gate_part + static_cast<int64_t>(unit) * a.d + c, left, sum[kG]);
#pragma unroll
  for (int q = 0; q < kSums; ++q) {
    if (a.part[q] == nullptr) continue;
    for (int m = teams - 1; m > 0; --m) {
      float* buf = lds + 64;
      __syncthreads();
      if (tm == m) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) buf[j * team_size + lane] = sum[q][j];
      }
      __syncthreads();
      if (tm == 0) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[q][j] += buf[j * team_size + lane];
      }
    }
    if (tm == 0 && left > 0) write8<R != kShort, false>(a.part[q] + static_cast<int64_t>(blockIdx.x) * a.d + c, left, sum[q]);
  }
}

// Wider rows, whose elements leave no registers for the column sums: one row a block.  What the
// column sums need of a row's reductions goes to a.pq.
template <typename T, int V, int R>
__global__ void __launch_bounds__(1024) block_norm_bwd_rows(BlockNormArgs a) {
  __shared__ float smem[64];
  const int team_size = blockDim.x, lane = threadIdx.x;
  Team<0> team{smem, 0, team_size / 64, 0};
  const int64_t row = a.first_row + blockIdx.x, gate_row = a.gate != nullptr ? row / a.gate_rows * a.d : 0;
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  RowData<T> r[V];  // all loads first
  float n1[V][kCols], n2[V][kCols], dy[V][kCols], ds[V][kCols];
  int col[V], left[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = col[k] = column<R>(k * team_size + lane, a.d, left[k]);
    load_row<T, R>(a, row, c, left[k], r[k]);
  }
  float p = 0.f, q = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = col[k];
    if (left[k] <= 0) continue;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      n1[k][j] = at8(r[k].res, j);
      n2[k][j] = a.x != nullptr ? at8(r[k].x, j) : 0.f;
      dy[k][j] = a.dy != nullptr ? at8(r[k].dy, j) : 0.f;
      ds[k][j] = a.ds != nullptr ? at8(r[k].ds, j) : 0.f;
    }
    if (a.x != nullptr) {
      float pw[kCols], pb[kCols], g[kCols];
      read_opt<R, T>(a.pw, a.w_f32, c, left[k], 1.f, pw);
      read_opt<R, T>(a.pb, a.w_f32, c, left[k], 0.f, pb);
      read_opt<R, T>(a.gate, a.gate_f32, gate_row + c, left[k], 1.f, g);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        n2[k][j] = (n2[k][j] - st.z) * st.w;
        n1[k][j] = fmaf(a.alpha * g[j], fmaf(n2[k][j], pw[j], pb[j]), n1[k][j]);
      }
    }
    if (a.dy != nullptr) {
      float w[kCols];
      read_opt<R, T>(a.w, a.w_f32, c, left[k], 1.f, w);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        n1[k][j] = (n1[k][j] - st.x) * st.y;
        dy[k][j] *= w[j];
        const float own = counts<R>(j, left[k]) ? dy[k][j] : 0.f;
        p += own;
        q = fmaf(own, n1[k][j], q);
      }
    }
  }
  if (a.dy != nullptr) {
    team.sum2(p, q);
    p = a.rms ? 0.f : p / a.d;
    q /= a.d;
  }
  if (lane == 0) reinterpret_cast<float2*>(a.pq)[row] = make_float2(p, q);
  float u = 0.f, v = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = col[k];
    if (left[k] <= 0) continue;
    if (a.dy != nullptr) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) ds[k][j] = fmaf(st.y, dy[k][j] - p - n1[k][j] * q, ds[k][j]);
    }
    if (a.dres != nullptr) write8<R != kShort, true>(static_cast<T*>(a.dres) + row * a.d + c, left[k], ds[k]);
    if (a.x == nullptr) continue;
    float pw[kCols], g[kCols];
    read_opt<R, T>(a.pw, a.w_f32, c, left[k], 1.f, pw);
    read_opt<R, T>(a.gate, a.gate_f32, gate_row + c, left[k], 1.f, g);
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      ds[k][j] = a.alpha * g[j] * ds[k][j] * pw[j];
      const float own = counts<R>(j, left[k]) ? ds[k][j] : 0.f;
      u += own;
      v = fmaf(own, n2[k][j], v);
    }
  }
  if (a.dx == nullptr) return;
  if (a.pw != nullptr) {
    team.sum2(u, v);
    u = a.rms ? 0.f : u / a.d;
    v /= a.d;
  } else {
    u = v = 0.f;
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = col[k];
    if (left[k] <= 0) continue;
#pragma unroll
    for (int j = 0; j < kCols; ++j) ds[k][j] = st.w * (ds[k][j] - u - n2[k][j] * v);
    write8<R != kShort, true>(static_cast<T*>(a.dx) + row * a.d + c, left[k], ds[k]);
  }
}

// The column sums of wide rows: a thread takes 8 columns of a unit's rows and forms n1, n2 and dS
// again from the rows and their reductions.  blockIdx.y: the unit.
template <typename T, int R>
__global__ void __launch_bounds__(256) block_norm_bwd_columns(BlockNormArgs a, int iterations) {
  int left;
  const int c = column<R>(blockIdx.x * 256 + threadIdx.x, a.d, left);
  if (left <= 0) return;
  const int unit = blockIdx.y, units = gridDim.y;
  float w[kCols], pw[kCols], pb[kCols], ag[kCols], sum[kSums][kCols];
  read_opt<R, T>(a.w, a.w_f32, c, left, 1.f, w);
  read_opt<R, T>(a.pw, a.w_f32, c, left, 1.f, pw);
  read_opt<R, T>(a.pb, a.w_f32, c, left, 0.f, pb);
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    ag[j] = a.alpha;
#pragma unroll
    for (int q = 0; q < kSums; ++q) sum[q][j] = 0.f;
  }
  int gate_now = -1;
  Walk t(a, unit);
  RowData<T> r;
  float2 pq = make_float2(0.f, 0.f);
  auto load = [&] {
    fetch<T, R>(a, t, c, left, r);
    if (t.live) pq = reinterpret_cast<const float2*>(a.pq)[t.row];
  };
  load();
  for (int i = 0; i < iterations && t.live; ++i) {
    if (a.gate != nullptr && t.gate != gate_now) {
      gate_now = t.gate;
      read_opt<R, T>(a.gate, a.gate_f32, static_cast<int64_t>(t.gate) * a.d + c, left, 1.f, ag);
#pragma unroll
      for (int j = 0; j < kCols; ++j) ag[j] *= a.alpha;
    }
    const RowData<T> now = r;
    const float4 st = now.st;
    const float p = pq.x, q = pq.y;
    const bool last = t.last(a);
    const int gate = t.gate;
    t.next(a, units);
    if (i + 1 < iterations) load();
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const float n2 = a.x != nullptr ? (at8(now.x, j) - st.z) * st.w : 0.f;
      const float h = fmaf(n2, pw[j], pb[j]);
      const float s = a.x != nullptr ? fmaf(ag[j], h, at8(now.res, j)) : at8(now.res, j);
      const float n1 = (s - st.x) * st.y, dy = a.dy != nullptr ? at8(now.dy, j) : 0.f;
      float d = a.ds != nullptr ? at8(now.ds, j) : 0.f;
      if (a.dy != nullptr) d = fmaf(st.y, dy * w[j] - p - n1 * q, d);
      const float dh = d * ag[j];
      sum[kW1][j] = fmaf(dy, n1, sum[kW1][j]);
      sum[kB1][j] += dy;
      sum[kG][j] = fmaf(d, h, sum[kG][j]);
      sum[kW2][j] = fmaf(dh, n2, sum[kW2][j]);
      sum[kB2][j] += dh;
    }
    if (a.gate_direct && last) {
      write_gate<T, R>(a, gate, c, left, sum[kG]);
#pragma unroll
      for (int j = 0; j < kCols; ++j) sum[kG][j] = 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < kCols; ++j) sum[kG][j] *= a.alpha;
  if (a.gate_part != nullptr) write8<R != kShort, false>(a.gate_part + static_cast<int64_t>(unit) * a.d + c, left, sum[kG]);
#pragma unroll
  for (int q = 0; q < kSums; ++q)
    if (a.part[q] != nullptr) write8<R != kShort, false>(a.part[q] + static_cast<int64_t>(unit) * a.d + c, left, sum[q]);
}

// out[g][c] = (or +=) the sum over `split` partial rows; 32 columns x 32 row groups a block.  9 us for two
// vectors of 256 partial rows and 16 gate rows of 4096.
__global__ void __launch_bounds__(1024) block_norm_join(BlockNormJoin l, int d) {
  __shared__ float buf[32][33];
  int64_t g = blockIdx.y;
  int i = 0;
  while (g >= l.item[i].groups) g -= l.item[i++].groups;  // (the grid has one y for each group of each item)
  const BlockNormJoin::Item& it = l.item[i];
  const int x = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  float v = 0.f;
  if (c < d) {
#pragma unroll 4
    for (int64_t k = r; k < it.split; k += 32) v += it.part[(g * it.split + k) * d + c];
  }
  buf[r][x] = v;
  __syncthreads();
  if (r != 0 || c >= d) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) v += buf[k][x];
  const int64_t at = g * d + c;
  switch (it.dt) {
    case F32: {
      float* o = static_cast<float*>(it.out) + at;
      *o = it.accumulate ? *o + v : v;
      break;
    }
    case F16: {
      f16* o = static_cast<f16*>(it.out) + at;
      *o = from_f32<f16>(it.accumulate ? to_f32(*o) + v : v);
      break;
    }
    default: {
      bf16* o = static_cast<bf16*>(it.out) + at;
      *o = from_f32<bf16>(it.accumulate ? to_f32(*o) + v : v);
    }
  }
}

constexpr int64_t kMaxWidth = 16384;
// Widest row whose column sums stay in registers: one vector a thread in the 12 waves of a CU.  Above
// it the sums spill: 40 M elements in rows of 12288 fp32 took 842 us in one pass, 208 us in two.
// At 8192 bf16 one pass takes 155 us in spite of its spills, two take 178 us; one rule for both types.
constexpr int64_t kMaxSummed = 6144;

// Threads of a row of up to 32 vectors: lanes of one wave, which takes several rows then.
int sub_of(int64_t vectors) { return vectors <= 8 ? 8 : vectors <= 16 ? 16 : vectors <= 32 ? 32 : 0; }

// Rows in launches of at most 2^28 threads: a grid has to stay below 2^32, and a launch of that size
// takes 100 us or more.  launch(arguments, blocks)
template <typename F>
void in_parts(BlockNormArgs a, int64_t rows_of_block, int64_t threads, const F& launch) {
  const int64_t most = (1ll << 28) / threads;
  for (; a.first_row < a.rows; a.first_row += most * rows_of_block) {
    const int64_t blocks = (a.rows - a.first_row + rows_of_block - 1) / rows_of_block;
    launch(a, static_cast<unsigned>(blocks < most ? blocks : most));
  }
}

}  // namespace

int block_norm_fwd(int dt, const BlockNormArgs& a, hipStream_t s) {
  if (a.d < 1 || a.d > kMaxWidth) return -4;
  if (a.rows <= 0) return 0;
  const int64_t vectors = (a.d + kCols - 1) / kCols;
  const bool wave = vectors <= 256;
  const int sub = sub_of(vectors);
  const int v = vectors <= 64 ? 1 : vectors <= 128 ? 2 : wave ? 4 : vectors <= 1024 ? 1 : 2;
  const int team = sub ? sub : wave ? 64 : static_cast<int>(((vectors + v - 1) / v + 63) / 64 * 64);
  const int threads = wave ? 256 : team;
  SMPK_DISPATCH(dt, T, {
    const bool whole = a.d % kCols == 0;
    const auto kernel =
        sub == 8    ? (whole ? block_norm_fwd<T, 1, kWhole, 8>
                             : a.d > kCols ? block_norm_fwd<T, 1, kOverlap, 8> : block_norm_fwd<T, 1, kShort, 8>)
        : sub == 16 ? (whole ? block_norm_fwd<T, 1, kWhole, 16> : block_norm_fwd<T, 1, kOverlap, 16>)
        : sub == 32 ? (whole ? block_norm_fwd<T, 1, kWhole, 32> : block_norm_fwd<T, 1, kOverlap, 32>)
        : v == 1    ? (whole ? block_norm_fwd<T, 1, kWhole, 0> : block_norm_fwd<T, 1, kOverlap, 0>)
        : v == 2    ? (whole ? block_norm_fwd<T, 2, kWhole, 0> : block_norm_fwd<T, 2, kOverlap, 0>)
                    : (whole ? block_norm_fwd<T, 4, kWhole, 0> : block_norm_fwd<T, 4, kOverlap, 0>);
    in_parts(a, wave ? 256 / team : 1, threads,
             [&](const BlockNormArgs& part, unsigned blocks) { kernel<<<blocks, threads, 0, s>>>(part, team); });
  });
  return static_cast<int>(hipGetLastError());
}

int block_norm_bwd_plan(int64_t rows, int64_t d, int64_t gate_rows, BlockNormPlan& p) {
  if (d < 1 || d > kMaxWidth || rows < 1 || rows > 0x7fffffff) return -4;
  const int64_t vectors = (d + kCols - 1) / kCols;
  p.two_pass = d > kMaxSummed;
  p.team = p.two_pass ? 256 : sub_of(vectors) ? sub_of(vectors) : static_cast<int>((vectors + 63) / 64 * 64);
  // teams of a block: as many waves as a CU holds, in three blocks of 4 waves or, for wider teams, in
  // one; LDS joins their sums, so that partial rows are fewer than units
  const int teams = p.two_pass ? 1 : p.team <= 256 ? 256 / p.team : 768 / p.team;
  p.threads = p.team * teams;
  int64_t units = (p.two_pass ? 1024 / ((vectors + 255) / 256) : p.team <= 256 ? 768 : 256) * teams;
  if (units > rows) units = rows;
  const int64_t groups = rows / gate_rows;
  p.split = units / groups;
  if (p.split < 1) p.split = 1;
  if (p.split > gate_rows) p.split = gate_rows;
  const int64_t used = p.split > 1 ? p.split * groups : (units < groups ? units : groups);
  p.blocks = (used + teams - 1) / teams;
  p.units = p.blocks * teams;
  p.iterations = p.split > 1 ? (gate_rows + p.split - 1) / p.split : (groups + p.units - 1) / p.units * gate_rows;
  p.lds = static_cast<int>((64 + (teams > 1 ? p.team * kCols : 0)) * sizeof(float));
  return 0;
}

namespace {
template <typename T, typename W, int R>
void launch_bwd(const BlockNormArgs& a, const BlockNormPlan& p, hipStream_t s) {
  const int iterations = static_cast<int>(p.iterations);
  if (p.two_pass) {
    const int64_t vectors = (a.d + kCols - 1) / kCols;
    const int v = vectors <= 1024 ? 1 : 2;
    const auto kernel = v == 1 ? block_norm_bwd_rows<T, 1, R> : block_norm_bwd_rows<T, 2, R>;
    const unsigned threads = static_cast<unsigned>(((vectors + v - 1) / v + 63) / 64 * 64);
    in_parts(a, 1, threads, [&](const BlockNormArgs& part, unsigned blocks) { kernel<<<blocks, threads, 0, s>>>(part); });
    bool sums = a.gate_direct || a.gate_part != nullptr;
    for (float* q : a.part) sums = sums || q != nullptr;
    if (!sums) return;
    const unsigned columns = static_cast<unsigned>((vectors + 255) / 256);
    block_norm_bwd_columns<T, R><<<dim3(columns, static_cast<unsigned>(p.units)), 256, 0, s>>>(a, iterations);
    return;
  }
  const auto kernel = p.team == 8    ? block_norm_bwd<T, W, R, 8>
                      : p.team == 16 ? block_norm_bwd<T, W, R, 16>
                      : p.team == 32 ? block_norm_bwd<T, W, R, 32>
                                     : block_norm_bwd<T, W, R, 0>;
  kernel<<<static_cast<unsigned>(p.blocks), p.threads, p.lds, s>>>(a, p.team, iterations);
}
template <typename T, typename W>
void launch_bwd_of(const BlockNormArgs& a, const BlockNormPlan& p, hipStream_t s) {
  if (a.d % kCols == 0) {
    launch_bwd<T, W, kWhole>(a, p, s);
  } else if (a.d > kCols) {
    launch_bwd<T, W, kOverlap>(a, p, s);
  } else {
    block_norm_bwd<T, W, kShort, 8><<<static_cast<unsigned>(p.blocks), p.threads, p.lds, s>>>(
        a, p.team, static_cast<int>(p.iterations));
  }
}
}  // namespace

int block_norm_bwd(int dt, const BlockNormArgs& a, const BlockNormPlan& p, hipStream_t s) {
  if (a.rows <= 0) return 0;
  if (p.two_pass && a.pq == nullptr) return -5;
  SMPK_DISPATCH(dt, T, {
    if (a.w_f32) {
      launch_bwd_of<T, float>(a, p, s);
    } else {
      launch_bwd_of<T, T>(a, p, s);
    }
  });
  return static_cast<int>(hipGetLastError());
}

int block_norm_join(const BlockNormJoin& l, int d, hipStream_t s) {
  if (l.count <= 0) return 0;
  int64_t groups = 0;
  for (int i = 0; i < l.count; ++i) groups += l.item[i].groups;
  if (groups > 65535) return -3;
  block_norm_join<<<dim3((d + 31) / 32, static_cast<unsigned>(groups)), 1024, 0, s>>>(l, d);
  return static_cast<int>(hipGetLastError());
}

}  // namespace smpk

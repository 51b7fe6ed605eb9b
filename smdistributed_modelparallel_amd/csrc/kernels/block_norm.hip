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
// A thread holds 8 consecutive elements of a row (V times that for wide rows).  Forward, rows of up
// to 2048 elements belong to one wave each: no barrier, and the rows of a CU's waves overlap freely.
// Wider rows, and all rows of the backward, belong to a team of waves.
#include "kernels.h"
#include "vec8.h"

namespace smpk {
namespace {

template <bool FULL>
__device__ __forceinline__ bool in_row(int j, int left) {
  return FULL || j < left;
}

// A vector that may be absent (`other` then) and of either T or fp32.
template <bool FULL, typename T>
__device__ __forceinline__ void read_opt(const void* p, bool f32, int64_t at, int left, float other, float (&o)[kCols]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < kCols; ++j) o[j] = other;
  } else if (f32) {
    read8<FULL>(static_cast<const float*>(p) + at, left, o);
  } else {
    read8<FULL>(static_cast<const T*>(p) + at, left, o);
  }
}

// Sums over a team of `waves` waves; `slot` alternates so that one barrier suffices.
struct Team {
  float* smem;  // [2][2][16]
  int first, waves, slot;
  __device__ __forceinline__ void sum2(float& a, float& b) {
    a = wave_sum_fixed(a);
    b = wave_sum_fixed(b);
    if (waves == 1) return;
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
    a = wave_sum_fixed(a);
    if (waves == 1) return;
    float* s = smem + slot * 32;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
    __syncthreads();
    a = 0.f;
    for (int k = 0; k < waves; ++k) a += s[first + k];
  }
};

// Mean, then the mean square of the differences: values of any offset keep their deviation.
template <int V, bool FULL>
__device__ __forceinline__ void moments(const float (&v)[V][kCols], const int (&left)[V], int d, float eps, bool rms,
                                        Team& team, float& mean, float& rstd) {
  mean = 0.f;
  if (!rms) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int j = 0; j < kCols; ++j) a += v[k][j];  // (zero past the row's end)
    team.sum1(a);
    mean = a / d;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    if (left[k] <= 0) continue;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const float c = in_row<FULL>(j, left[k]) ? v[k][j] - mean : 0.f;
      q = fmaf(c, c, q);
    }
  }
  team.sum1(q);
  rstd = rsqrtf(q / d + eps);
}

// team_size threads for a row: 64 (and blockDim.x / 64 rows a block), or all of the block
template <typename T, int V, bool FULL>
__global__ void __launch_bounds__(1024) block_norm_fwd(BlockNormArgs a, int team_size) {
  __shared__ float smem[64];
  const int tid = threadIdx.x, lane = team_size == 64 ? tid & 63 : tid;
  Team team{smem, 0, team_size / 64, 0};
  const int64_t row = team_size == 64
                          ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(tid >> 6)
                          : blockIdx.x;
  if (row >= a.rows) return;  // (whole waves of their own rows: no barrier follows for them)
  int left[V];
  float s[V][kCols], h[V][kCols];
  Raw8<T> rs[V], rh[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * team_size + lane) * kCols;
    left[k] = a.d - c;
    if (left[k] <= 0) continue;
    if (a.x != nullptr) read8<FULL>(static_cast<const T*>(a.x) + row * a.d + c, left[k], rh[k]);
    read8<FULL>(static_cast<const T*>(a.res) + row * a.d + c, left[k], rs[k]);
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
    if (a.pw != nullptr) moments<V, FULL>(h, left, a.d, a.eps, a.rms, team, mean2, rstd2);
    const int64_t gate_row = a.gate != nullptr ? row / a.gate_rows * a.d : 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * team_size + lane) * kCols;
      if (left[k] <= 0) continue;
      float w[kCols], b[kCols], g[kCols];
      read_opt<FULL, T>(a.pw, a.w_f32, c, left[k], 1.f, w);
      read_opt<FULL, T>(a.pb, a.w_f32, c, left[k], 0.f, b);
      read_opt<FULL, T>(a.gate, a.gate_f32, gate_row + c, left[k], 1.f, g);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const float v = fmaf((h[k][j] - mean2) * rstd2, w[j], b[j]);
        s[k][j] = in_row<FULL>(j, left[k]) ? fmaf(a.alpha * g[j], v, s[k][j]) : 0.f;
      }
      write8<FULL, true>(static_cast<T*>(a.s) + row * a.d + c, left[k], s[k]);
    }
  }
  moments<V, FULL>(s, left, a.d, a.eps, a.rms, team, mean1, rstd1);
  if (lane == 0 && a.stats != nullptr)
    reinterpret_cast<float4*>(a.stats)[row] = make_float4(mean1, rstd1, mean2, rstd2);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * team_size + lane) * kCols;
    if (left[k] <= 0) continue;
    float w[kCols], b[kCols];
    read_opt<FULL, T>(a.w, a.w_f32, c, left[k], 1.f, w);
    read_opt<FULL, T>(a.b, a.w_f32, c, left[k], 0.f, b);
#pragma unroll
    for (int j = 0; j < kCols; ++j) w[j] = fmaf((s[k][j] - mean1) * rstd1, w[j], b[j]);
    write8<FULL, true>(static_cast<T*>(a.y) + row * a.d + c, left[k], w);
  }
}

// A unit (one team) takes consecutive rows of one gate row.  split > 1: `split` units share the rows
// of a gate row; split == 1: a unit takes whole gate rows, `units` apart.
struct Walk {
  int64_t row, gate;
  int64_t at, count;  // at-th of the unit's `count` rows of this gate row
  bool live;
  __device__ __forceinline__ Walk(const BlockNormArgs& a, int64_t unit) {
    const int64_t chunk = (a.gate_rows + a.split - 1) / a.split, first = unit % a.split * chunk;
    gate = unit / a.split;
    at = 0;
    count = a.gate_rows - first < chunk ? a.gate_rows - first : chunk;
    live = gate < a.groups && count > 0;
    row = gate * a.gate_rows + first;
  }
  // the gate row ends with this row, and all of it was this unit's
  __device__ __forceinline__ bool last(const BlockNormArgs& a) const { return a.split == 1 && at == count - 1; }
  __device__ __forceinline__ void next(const BlockNormArgs& a, int64_t units) {
    ++row;
    if (++at < count) return;
    at = 0;
    gate += units;
    row = gate * a.gate_rows;
    live = live && a.split == 1 && gate < a.groups;
  }
};

enum { kW1, kB1, kW2, kB2, kG, kSums };

// A row's loads, issued while the row before is worked on.
template <typename T, int V>
struct RowData {
  Raw8<T> x[V], res[V], dy[V], ds[V];
  float4 st;
};

template <typename T, int V, bool FULL>
__device__ __forceinline__ void fetch(const BlockNormArgs& a, const Walk& t, int team_size, int lane, RowData<T, V>& r) {
  if (!t.live) return;
  r.st = reinterpret_cast<const float4*>(a.stats)[t.row];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * team_size + lane) * kCols, left = a.d - c;
    if (left <= 0) continue;
    const int64_t at = t.row * a.d + c;
    read8<FULL>(static_cast<const T*>(a.res) + at, left, r.res[k]);
    if (a.x != nullptr) read8<FULL>(static_cast<const T*>(a.x) + at, left, r.x[k]);
    if (a.dy != nullptr) read8<FULL>(static_cast<const T*>(a.dy) + at, left, r.dy[k]);
    if (a.ds != nullptr) read8<FULL>(static_cast<const T*>(a.ds) + at, left, r.ds[k]);
  }
}

// The weights stay in registers, in their own type W (T or fp32): a unit works on many rows.
template <typename T, typename W, int V, bool FULL, int THREADS>
__global__ void __launch_bounds__(THREADS) block_norm_bwd(BlockNormArgs a, int team_size, int64_t iterations) {
  extern __shared__ float lds[];  // [64] reductions, then [team_size * kCols * V] to join the teams' sums
  const int tid = threadIdx.x, teams = blockDim.x / team_size;
  const int tm = __builtin_amdgcn_readfirstlane(tid / team_size), lane = tid - tm * team_size;  // (whole waves)
  Team team{lds, tm * (team_size / 64), team_size / 64, 0};
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * teams + tm, units = static_cast<int64_t>(gridDim.x) * teams;
  float sum[kSums][V][kCols];
  Raw8<W> w[V], pw[V], pb[V];
  float ag[V][kCols];  // alpha * gate
  int left[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * team_size + lane) * kCols;
    left[k] = a.d - c;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      w[k].v[j] = pw[k].v[j] = from_f32<W>(1.f);
      pb[k].v[j] = from_f32<W>(0.f);
      ag[k][j] = a.alpha;
    }
    if (left[k] > 0) {
      read8<FULL>(static_cast<const W*>(a.w) + c, left[k], w[k]);
      if (a.pw != nullptr) read8<FULL>(static_cast<const W*>(a.pw) + c, left[k], pw[k]);
      if (a.pb != nullptr) read8<FULL>(static_cast<const W*>(a.pb) + c, left[k], pb[k]);
    }
#pragma unroll
    for (int q = 0; q < kSums; ++q)
#pragma unroll
      for (int j = 0; j < kCols; ++j) sum[q][k][j] = 0.f;
  }
  int64_t gate_now = -1;
  RowData<T, V> r;
  Walk t(a, unit);
  fetch<T, V, FULL>(a, t, team_size, lane, r);

  for (int64_t i = 0; i < iterations; ++i) {
    if (a.gate != nullptr && t.live && t.gate != gate_now) {
      gate_now = t.gate;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = (k * team_size + lane) * kCols;
        if (left[k] <= 0) continue;
        read_opt<FULL, T>(a.gate, a.gate_f32, t.gate * a.d + c, left[k], 1.f, ag[k]);
#pragma unroll
        for (int j = 0; j < kCols; ++j) ag[k][j] *= a.alpha;
      }
    }
    float n1[V][kCols], n2[V][kCols], dy[V][kCols], ds[V][kCols];
    const float4 st = r.st;
    float p = 0.f, q = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (left[k] <= 0 || !t.live) continue;
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        n1[k][j] = at8(r.res[k], j);
        n2[k][j] = 0.f;
        ds[k][j] = a.ds != nullptr ? at8(r.ds[k], j) : 0.f;
      }
      if (a.x != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          n2[k][j] = in_row<FULL>(j, left[k]) ? (at8(r.x[k], j) - st.z) * st.w : 0.f;
          n1[k][j] = fmaf(ag[k][j], fmaf(n2[k][j], at8(pw[k], j), at8(pb[k], j)), n1[k][j]);
        }
      }
      if (a.dy != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          const float g = at8(r.dy[k], j);
          n1[k][j] = in_row<FULL>(j, left[k]) ? (n1[k][j] - st.x) * st.y : 0.f;
          sum[kW1][k][j] = fmaf(g, n1[k][j], sum[kW1][k][j]);
          sum[kB1][k][j] += g;
          dy[k][j] = g * at8(w[k], j);
          p += dy[k][j];
          q = fmaf(dy[k][j], n1[k][j], q);
        }
      }
    }
    const Walk now = t;
    const bool last = now.last(a);
    t.next(a, units);
    if (i + 1 < iterations) fetch<T, V, FULL>(a, t, team_size, lane, r);
    if (a.dy != nullptr) {
      team.sum2(p, q);
      p = a.rms ? 0.f : p / a.d;
      q /= a.d;
    }
    float u = 0.f, v = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (left[k] <= 0 || !now.live) continue;
      const int64_t at = now.row * a.d + (k * team_size + lane) * kCols;
      if (a.dy != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) ds[k][j] = fmaf(st.y, dy[k][j] - p - n1[k][j] * q, ds[k][j]);
      }
      if (a.dres != nullptr) write8<FULL, true>(static_cast<T*>(a.dres) + at, left[k], ds[k]);
      if (a.x == nullptr) continue;
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const float s = in_row<FULL>(j, left[k]) ? ds[k][j] : 0.f;
        sum[kG][k][j] = fmaf(s, fmaf(n2[k][j], at8(pw[k], j), at8(pb[k], j)), sum[kG][k][j]);
        const float dh = s * ag[k][j];
        sum[kW2][k][j] = fmaf(dh, n2[k][j], sum[kW2][k][j]);
        sum[kB2][k][j] += dh;
        ds[k][j] = dh * at8(pw[k], j);  // the gradient of n2; of x itself without a norm
        u += ds[k][j];
        v = fmaf(ds[k][j], n2[k][j], v);
      }
    }
    if (a.pw != nullptr) {
      team.sum2(u, v);
      u = a.rms ? 0.f : u / a.d;
      v /= a.d;
    } else {
      u = v = 0.f;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * team_size + lane) * kCols;
      if (left[k] <= 0 || !now.live || a.x == nullptr) continue;
      if (a.dx != nullptr) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) ds[k][j] = st.w * (ds[k][j] - u - n2[k][j] * v);
        write8<FULL, true>(static_cast<T*>(a.dx) + now.row * a.d + c, left[k], ds[k]);
      }
      if (a.gate_direct && last) {  // a whole gate row's sum is complete
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[kG][k][j] *= a.alpha;
        if (a.gate_f32) {
          write8<FULL, true>(static_cast<float*>(a.dgate) + now.gate * a.d + c, left[k], sum[kG][k]);
        } else {
          write8<FULL, true>(static_cast<T*>(a.dgate) + now.gate * a.d + c, left[k], sum[kG][k]);
        }
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[kG][k][j] = 0.f;
      }
    }
  }

  // partial sums: of the teams together for the vectors, of each unit for its gate row
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * team_size + lane) * kCols;
#pragma unroll
    for (int j = 0; j < kCols; ++j) sum[kG][k][j] *= a.alpha;
    if (a.gate_part != nullptr && c < a.d) write8<FULL, false>(a.gate_part + unit * a.d + c, a.d - c, sum[kG][k]);
  }
#pragma unroll
  for (int q = 0; q < kSums; ++q) {
    if (a.part[q] == nullptr) continue;
    for (int m = teams - 1; m > 0; --m) {
      float* buf = lds + 64;
      __syncthreads();
      if (tm == m) {
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
          for (int j = 0; j < kCols; ++j) buf[(k * kCols + j) * team_size + lane] = sum[q][k][j];
      }
      __syncthreads();
      if (tm == 0) {
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
          for (int j = 0; j < kCols; ++j) sum[q][k][j] += buf[(k * kCols + j) * team_size + lane];
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * team_size + lane) * kCols;
      if (tm == 0 && c < a.d)
        write8<FULL, false>(a.part[q] + static_cast<int64_t>(blockIdx.x) * a.d + c, a.d - c, sum[q][k]);
    }
  }
}

// out[g][c] = (or +=) the sum over `split` partial rows; 32 columns x 32 row groups a block
__global__ void __launch_bounds__(1024) block_norm_join(BlockNormJoin l, int d) {
  __shared__ float buf[32][33];
  const BlockNormJoin::Item& it = l.item[blockIdx.y];
  const int64_t g = blockIdx.z;
  if (g >= it.groups) return;
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

// Teams of the backward: one vector a thread up to 4096 elements, two beyond.
int team_of(int64_t d, int& v) {
  const int64_t vectors = (d + kCols - 1) / kCols;
  v = vectors <= 512 ? 1 : 2;
  return static_cast<int>(((vectors + v - 1) / v + 63) / 64 * 64);
}

constexpr int64_t kMaxWidth = 16384;

}  // namespace

int block_norm_fwd(int dt, const BlockNormArgs& a, hipStream_t s) {
  if (a.d < 1 || a.d > kMaxWidth) return -4;
  if (a.rows <= 0) return 0;
  const int64_t vectors = (a.d + kCols - 1) / kCols;
  const bool wave = vectors <= 256;
  const int v = vectors <= 64 ? 1 : vectors <= 128 ? 2 : wave ? 4 : vectors <= 1024 ? 1 : 2;
  const int team = wave ? 64 : static_cast<int>(((vectors + v - 1) / v + 63) / 64 * 64);
  const int64_t blocks = wave ? (a.rows + 3) / 4 : a.rows;
  if (blocks > 0x7fffffff) return -3;
  SMPK_DISPATCH(dt, T, {
    const bool full = a.d % kCols == 0;
    const auto kernel = v == 1   ? (full ? block_norm_fwd<T, 1, true> : block_norm_fwd<T, 1, false>)
                        : v == 2 ? (full ? block_norm_fwd<T, 2, true> : block_norm_fwd<T, 2, false>)
                                 : (full ? block_norm_fwd<T, 4, true> : block_norm_fwd<T, 4, false>);
    kernel<<<static_cast<unsigned>(blocks), wave ? 256 : team, 0, s>>>(a, team);
  });
  return static_cast<int>(hipGetLastError());
}

int block_norm_bwd_plan(int64_t rows, int64_t d, int64_t gate_rows, BlockNormPlan& p) {
  if (d < 1 || d > kMaxWidth || rows < 1) return -4;
  int v;
  p.team = team_of(d, v);
  const int teams = p.team >= 256 ? 1 : 256 / p.team;  // LDS joins their sums: fewer partial rows than units
  p.threads = p.team * teams;
  int64_t units = (p.team > 256 ? 512 : 768) * teams;
  if (units > rows) units = rows;
  const int64_t groups = rows / gate_rows;
  p.split = units / groups;
  if (p.split < 1) p.split = 1;
  if (p.split > gate_rows) p.split = gate_rows;
  const int64_t used = p.split > 1 ? p.split * groups : (units < groups ? units : groups);
  p.blocks = (used + teams - 1) / teams;
  p.units = p.blocks * teams;
  p.iterations = p.split > 1 ? (gate_rows + p.split - 1) / p.split : (groups + p.units - 1) / p.units * gate_rows;
  p.lds = static_cast<int>((64 + (teams > 1 ? p.team * kCols * v : 0)) * sizeof(float));
  return 0;
}

namespace {
template <typename T, typename W>
void launch_bwd(const BlockNormArgs& a, const BlockNormPlan& p, hipStream_t s) {
  const bool full = a.d % kCols == 0;
  int v;
  team_of(a.d, v);
  const auto kernel = v == 1 ? (full ? block_norm_bwd<T, W, 1, true, 512> : block_norm_bwd<T, W, 1, false, 512>)
                      : p.threads <= 512
                          ? (full ? block_norm_bwd<T, W, 2, true, 512> : block_norm_bwd<T, W, 2, false, 512>)
                          : (full ? block_norm_bwd<T, W, 2, true, 1024> : block_norm_bwd<T, W, 2, false, 1024>);
  kernel<<<static_cast<unsigned>(p.blocks), p.threads, p.lds, s>>>(a, p.team, p.iterations);
}
}  // namespace

int block_norm_bwd(int dt, const BlockNormArgs& a, const BlockNormPlan& p, hipStream_t s) {
  if (a.rows <= 0) return 0;
  SMPK_DISPATCH(dt, T, {
    if (a.w_f32) {
      launch_bwd<T, float>(a, p, s);
    } else {
      launch_bwd<T, T>(a, p, s);
    }
  });
  return static_cast<int>(hipGetLastError());
}

int block_norm_join(const BlockNormJoin& l, int d, hipStream_t s) {
  if (l.count <= 0) return 0;
  int64_t groups = 1;
  for (int i = 0; i < l.count; ++i) groups = l.item[i].groups > groups ? l.item[i].groups : groups;
  if (groups > 65535) return -3;
  block_norm_join<<<dim3((d + 31) / 32, l.count, static_cast<unsigned>(groups)), 1024, 0, s>>>(l, d);
  return static_cast<int>(hipGetLastError());
}

}  // namespace smpk

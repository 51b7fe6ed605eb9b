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
// A thread holds kN = 8 consecutive elements of a row (times V for the widest rows); a team of
// threads, a multiple of 64, holds the row.  Rows of odd widths start off 16 bytes: the hardware
// loads and stores 16 bytes at any address, so only the last, partial vector of a row goes
// element by element.
#include "common.h"
#include "kernels.h"

namespace smpk {
namespace {

constexpr int kN = 8;

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned16 {
  T v[16 / sizeof(T)];
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, float (&o)[kN]) {
  if (left >= kN) {
    constexpr int M = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < kN; k += M) {
      Unaligned16<T> a;
      __builtin_memcpy(&a, p + k, 16);
#pragma unroll
      for (int j = 0; j < M; ++j) o[k + j] = to_f32(a.v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; ++j) o[j] = j < left ? to_f32(p[j]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int left, const float (&o)[kN]) {
  if (left >= kN) {
    constexpr int M = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < kN; k += M) {
      Unaligned16<T> a;
#pragma unroll
      for (int j = 0; j < M; ++j) a.v[j] = from_f32<T>(o[k + j]);
      __builtin_memcpy(p + k, &a, 16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; ++j)
      if (j < left) p[j] = from_f32<T>(o[j]);
  }
}

// A vector that may be absent (`other` then) and of either T or fp32.
template <typename T>
__device__ __forceinline__ void load_opt(const void* p, bool f32, int64_t at, int left, float other, float (&o)[kN]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < kN; ++j) o[j] = other;
  } else if (f32) {
    load8(static_cast<const float*>(p) + at, left, o);
  } else {
    load8(static_cast<const T*>(p) + at, left, o);
  }
}

// Sums of two values over a team of `waves` waves; `slot` alternates so that one barrier suffices.
struct Team {
  float* smem;  // [2][2][16]
  int first, waves, slot;
  __device__ __forceinline__ void sum2(float& a, float& b) {
    a = wave_sum(a);
    b = wave_sum(b);
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
};

template <int V>
__device__ __forceinline__ void moments(const float (&v)[V][kN], const int (&left)[V], int d, float eps, bool rms,
                                        Team& team, float& mean, float& rstd) {
  mean = 0.f;
  float unused = 0.f;
  if (!rms) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int j = 0; j < kN; ++j) a += v[k][j];  // (zero past the row's end)
    team.sum2(a, unused);
    mean = a / d;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k)
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      const float c = j < left[k] ? v[k][j] - mean : 0.f;
      q = fmaf(c, c, q);
    }
  team.sum2(q, unused);
  rstd = rsqrtf(q / d + eps);
}

template <typename T, int V>
__global__ void __launch_bounds__(1024) block_norm_fwd(BlockNormArgs a, int team_size) {
  __shared__ float smem[64];
  const int tid = threadIdx.x, teams = blockDim.x / team_size, lane = tid % team_size, tm = tid / team_size;
  Team team{smem, tm * (team_size / 64), team_size / 64, 0};
  const int64_t row = static_cast<int64_t>(blockIdx.x) * teams + tm;
  const bool live = row < a.rows;  // a team past the end only joins the barriers
  int left[V];
  float s[V][kN], h[V][kN];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * team_size + lane) * kN;
    left[k] = live ? a.d - c : 0;
#pragma unroll
    for (int j = 0; j < kN; ++j) s[k][j] = h[k][j] = 0.f;
    if (left[k] > 0) {
      load8(static_cast<const T*>(a.res) + row * a.d + c, left[k], s[k]);
      if (a.x != nullptr) load8(static_cast<const T*>(a.x) + row * a.d + c, left[k], h[k]);
    }
  }
  float mean2 = 0.f, rstd2 = 1.f, mean1, rstd1;
  if (a.x != nullptr) {
    if (a.pw != nullptr) moments(h, left, a.d, a.eps, a.rms, team, mean2, rstd2);
    const int64_t gate_row = a.gate != nullptr && live ? row / a.gate_rows * a.d : 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * team_size + lane) * kN;
      if (left[k] <= 0) continue;
      float w[kN], b[kN], g[kN];
      load_opt<T>(a.pw, a.w_f32, c, left[k], 1.f, w);
      load_opt<T>(a.pb, a.w_f32, c, left[k], 0.f, b);
      load_opt<T>(a.gate, a.gate_f32, gate_row + c, left[k], 1.f, g);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const float v = fmaf((h[k][j] - mean2) * rstd2, w[j], b[j]);
        s[k][j] = j < left[k] ? fmaf(a.alpha * g[j], v, s[k][j]) : 0.f;
      }
      store8(static_cast<T*>(a.s) + row * a.d + c, left[k], s[k]);
    }
  }
  moments(s, left, a.d, a.eps, a.rms, team, mean1, rstd1);
  if (live && lane == 0 && a.stats != nullptr)
    reinterpret_cast<float4*>(a.stats)[row] = make_float4(mean1, rstd1, mean2, rstd2);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * team_size + lane) * kN;
    if (left[k] <= 0) continue;
    float w[kN], b[kN];
    load_opt<T>(a.w, a.w_f32, c, left[k], 1.f, w);
    load_opt<T>(a.b, a.w_f32, c, left[k], 0.f, b);
#pragma unroll
    for (int j = 0; j < kN; ++j) w[j] = fmaf((s[k][j] - mean1) * rstd1, w[j], b[j]);
    store8(static_cast<T*>(a.y) + row * a.d + c, left[k], w);
  }
}

// A unit (one team) takes rows of one gate row only.  split > 1: `split` units share the rows of
// a gate row; split == 1: a unit takes whole gate rows, `units` apart.
struct Turn {
  int64_t row;
  bool live, last;  // last: the gate row ends with this row (split == 1)
  int64_t gate;
};
__device__ __forceinline__ Turn turn_of(const BlockNormArgs& a, int64_t unit, int64_t units, int64_t i) {
  Turn t;
  const int64_t groups = a.rows / a.gate_rows;
  if (a.split > 1) {
    const int64_t chunk = (a.gate_rows + a.split - 1) / a.split, j = unit % a.split * chunk + i;
    t.gate = unit / a.split;
    t.live = t.gate < groups && i < chunk && j < a.gate_rows;
    t.row = t.gate * a.gate_rows + j;
    t.last = false;
  } else {
    const int64_t j = i % a.gate_rows;
    t.gate = unit + i / a.gate_rows * units;
    t.live = t.gate < groups;
    t.row = t.gate * a.gate_rows + j;
    t.last = j == a.gate_rows - 1;
  }
  return t;
}

enum { kW1, kB1, kW2, kB2, kG, kSums };

template <typename T, int V>
__global__ void __launch_bounds__(1024) block_norm_bwd(BlockNormArgs a, int team_size, int64_t iterations) {
  extern __shared__ float lds[];  // [64] reductions, then [team_size * kN * V] to join the teams' sums
  const int tid = threadIdx.x, teams = blockDim.x / team_size, lane = tid % team_size, tm = tid / team_size;
  Team team{lds, tm * (team_size / 64), team_size / 64, 0};
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * teams + tm, units = static_cast<int64_t>(gridDim.x) * teams;
  float sum[kSums][V][kN];
#pragma unroll
  for (int q = 0; q < kSums; ++q)
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int j = 0; j < kN; ++j) sum[q][k][j] = 0.f;

  for (int64_t i = 0; i < iterations; ++i) {
    const Turn t = turn_of(a, unit, units, i);
    float n1[V][kN], n2[V][kN], dy[V][kN], ds[V][kN];
    int left[V];
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    if (t.live) st = reinterpret_cast<const float4*>(a.stats)[t.row];
    float p = 0.f, q = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * team_size + lane) * kN;
      left[k] = t.live ? a.d - c : 0;
#pragma unroll
      for (int j = 0; j < kN; ++j) n1[k][j] = n2[k][j] = dy[k][j] = ds[k][j] = 0.f;
      if (left[k] <= 0) continue;
      const int64_t at = t.row * a.d + c;
      float w[kN], b[kN], g[kN], pw[kN];
      load8(static_cast<const T*>(a.res) + at, left[k], n1[k]);
      if (a.ds != nullptr) load8(static_cast<const T*>(a.ds) + at, left[k], ds[k]);
      if (a.x != nullptr) {
        load8(static_cast<const T*>(a.x) + at, left[k], n2[k]);
        load_opt<T>(a.pw, a.w_f32, c, left[k], 1.f, pw);
        load_opt<T>(a.pb, a.w_f32, c, left[k], 0.f, b);
        load_opt<T>(a.gate, a.gate_f32, t.gate * a.d + c, left[k], 1.f, g);
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          n2[k][j] = j < left[k] ? (n2[k][j] - st.z) * st.w : 0.f;
          n1[k][j] = fmaf(a.alpha * g[j], fmaf(n2[k][j], pw[j], b[j]), n1[k][j]);
        }
      }
      if (a.dy != nullptr) {
        load8(static_cast<const T*>(a.dy) + at, left[k], dy[k]);
        load_opt<T>(a.w, a.w_f32, c, left[k], 1.f, w);
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          n1[k][j] = j < left[k] ? (n1[k][j] - st.x) * st.y : 0.f;
          sum[kW1][k][j] = fmaf(dy[k][j], n1[k][j], sum[kW1][k][j]);
          sum[kB1][k][j] += dy[k][j];
          dy[k][j] *= w[j];
          p += dy[k][j];
          q = fmaf(dy[k][j], n1[k][j], q);
        }
      }
    }
    if (a.dy != nullptr) {
      team.sum2(p, q);
      p = a.rms ? 0.f : p / a.d;
      q /= a.d;
    }
    float u = 0.f, v = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * team_size + lane) * kN;
      if (left[k] <= 0) continue;
      const int64_t at = t.row * a.d + c;
      if (a.dy != nullptr) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
          ds[k][j] = fmaf(st.y, dy[k][j] - p - n1[k][j] * q, ds[k][j]);
      }
      if (a.dres != nullptr) store8(static_cast<T*>(a.dres) + at, left[k], ds[k]);
      if (a.x == nullptr) continue;
      float b[kN], g[kN], pw[kN];
      load_opt<T>(a.pw, a.w_f32, c, left[k], 1.f, pw);
      load_opt<T>(a.pb, a.w_f32, c, left[k], 0.f, b);
      load_opt<T>(a.gate, a.gate_f32, t.gate * a.d + c, left[k], 1.f, g);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const float as = j < left[k] ? a.alpha * ds[k][j] : 0.f;
        sum[kG][k][j] = fmaf(as, fmaf(n2[k][j], pw[j], b[j]), sum[kG][k][j]);
        const float dh = as * g[j];
        sum[kW2][k][j] = fmaf(dh, n2[k][j], sum[kW2][k][j]);
        sum[kB2][k][j] += dh;
        ds[k][j] = dh * pw[j];  // the gradient of n2; of x itself without a norm
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
      const int c = (k * team_size + lane) * kN;
      if (left[k] <= 0 || a.x == nullptr) continue;
      if (a.dx != nullptr) {
#pragma unroll
        for (int j = 0; j < kN; ++j) ds[k][j] = st.w * (ds[k][j] - u - n2[k][j] * v);
        store8(static_cast<T*>(a.dx) + t.row * a.d + c, left[k], ds[k]);
      }
      if (a.gate_direct && t.last) {  // a whole gate row's sum is complete
        if (a.gate_f32) {
          store8(static_cast<float*>(a.dgate) + t.gate * a.d + c, left[k], sum[kG][k]);
        } else {
          store8(static_cast<T*>(a.dgate) + t.gate * a.d + c, left[k], sum[kG][k]);
        }
#pragma unroll
        for (int j = 0; j < kN; ++j) sum[kG][k][j] = 0.f;
      }
    }
  }

  // partial sums: of the teams together for the vectors, of each unit for its gate row
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * team_size + lane) * kN;
    if (a.gate_part != nullptr && c < a.d) store8(a.gate_part + unit * a.d + c, a.d - c, sum[kG][k]);
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
          for (int j = 0; j < kN; ++j) buf[(k * kN + j) * team_size + lane] = sum[q][k][j];
      }
      __syncthreads();
      if (tm == 0) {
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
          for (int j = 0; j < kN; ++j) sum[q][k][j] += buf[(k * kN + j) * team_size + lane];
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * team_size + lane) * kN;
      if (tm == 0 && c < a.d) store8(a.part[q] + static_cast<int64_t>(blockIdx.x) * a.d + c, a.d - c, sum[q][k]);
    }
  }
}

// out[g][c] = (or +=) the sum over `split` partial rows; 64 columns x 16 row groups a block
__global__ void __launch_bounds__(1024) block_norm_join(BlockNormJoin l, int d) {
  __shared__ float buf[16][64];
  const BlockNormJoin::Item& it = l.item[blockIdx.y];
  const int64_t g = blockIdx.z;
  if (g >= it.groups) return;
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), r = threadIdx.x >> 6;
  float v = 0.f;
  if (c < d)
    for (int64_t k = r; k < it.split; k += 16) v += it.part[(g * it.split + k) * d + c];
  buf[r][threadIdx.x & 63] = v;
  __syncthreads();
  if (r != 0 || c >= d) return;
  for (int k = 1; k < 16; ++k) v += buf[k][threadIdx.x];
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

// threads of a team and vectors a thread holds; false: the row is too wide
bool team_for(int64_t d, int& team, int& v) {
  const int64_t vectors = (d + kN - 1) / kN;
  v = vectors <= 1024 ? 1 : 2;
  const int64_t t = ((vectors + v - 1) / v + 63) / 64 * 64;
  team = static_cast<int>(t);
  return t <= 1024;
}

}  // namespace

int block_norm_fwd(int dt, const BlockNormArgs& a, hipStream_t s) {
  int team, v;
  if (!team_for(a.d, team, v)) return -4;
  if (a.rows <= 0) return 0;
  const int teams = team >= 256 ? 1 : 256 / team;
  const int64_t blocks = (a.rows + teams - 1) / teams;
  if (blocks > 0x7fffffff) return -3;
  SMPK_DISPATCH(dt, T, {
    if (v == 1) {
      block_norm_fwd<T, 1><<<static_cast<unsigned>(blocks), team * teams, 0, s>>>(a, team);
    } else {
      block_norm_fwd<T, 2><<<static_cast<unsigned>(blocks), team * teams, 0, s>>>(a, team);
    }
  });
  return static_cast<int>(hipGetLastError());
}

int block_norm_bwd_plan(int64_t rows, int64_t d, int64_t gate_rows, BlockNormPlan& p) {
  int v;
  if (!team_for(d, p.team, v)) return -4;
  const int teams = 1024 / p.team;  // LDS joins their sums: fewer partial rows than units
  p.threads = p.team * teams;
  int64_t units = 512 * teams;
  if (units > rows) units = rows;
  const int64_t groups = rows / gate_rows;
  p.split = units / groups;
  if (p.split < 1) p.split = 1;
  if (p.split > gate_rows) p.split = gate_rows;
  const int64_t used = p.split > 1 ? p.split * groups : (units < groups ? units : groups);
  p.blocks = (used + teams - 1) / teams;
  p.units = p.blocks * teams;
  p.iterations = p.split > 1 ? (gate_rows + p.split - 1) / p.split : (groups + p.units - 1) / p.units * gate_rows;
  p.lds = static_cast<int>((64 + (teams > 1 ? p.team * kN * v : 0)) * sizeof(float));
  return 0;
}

int block_norm_bwd(int dt, const BlockNormArgs& a, const BlockNormPlan& p, hipStream_t s) {
  if (a.rows <= 0) return 0;
  SMPK_DISPATCH(dt, T, {
    if ((a.d + kN - 1) / kN <= 1024) {
      block_norm_bwd<T, 1><<<static_cast<unsigned>(p.blocks), p.threads, p.lds, s>>>(a, p.team, p.iterations);
    } else {
      block_norm_bwd<T, 2><<<static_cast<unsigned>(p.blocks), p.threads, p.lds, s>>>(a, p.team, p.iterations);
    }
  });
  return static_cast<int>(hipGetLastError());
}

int block_norm_join(const BlockNormJoin& l, int d, hipStream_t s) {
  if (l.count <= 0) return 0;
  int64_t groups = 1;
  for (int i = 0; i < l.count; ++i) groups = l.item[i].groups > groups ? l.item[i].groups : groups;
  if (groups > 65535) return -3;
  block_norm_join<<<dim3((d + 63) / 64, l.count, static_cast<unsigned>(groups)), 1024, 0, s>>>(l, d);
  return static_cast<int>(hipGetLastError());
}

}  // namespace smpk

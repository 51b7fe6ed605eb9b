// The norm of all gradients of a model at once, and the gradients scaled down to a largest norm.
//
// norm = scale * sqrt(sum g^2) or scale * max |g|; out = g * scale * min(1, max_norm / (norm + 1e-6)).
// Bound by HBM: every gradient is read for the norm, and read again and written for the clip.
// Measured, 1.56 G bf16 elements in 579 tensors: norm 0.57 ms (5.5 TB/s), clip 1.31 ms (4.7 TB/s, the
// rate of a copy of that size).
//
// The tensors come as a table in the kernel's arguments (kGradList of them a launch): no copy to
// the device precedes a launch, and a captured launch holds its table.  A tensor is cut into
// chunks of the same size for all, one block each; a block leaves one partial, and the partials
// are added in a fixed order -- the same bits on every run.  Squares are summed in 64 bits: no
// finite gradient overflows or underflows the sum, and the conversions stay far below the time
// of the memory reads.  Maxima are taken on the bits of |g|, whose order as unsigned integers
// puts infinities above all numbers and NaN above them: a NaN is never lost.
#include "kernels.h"
#include "vec8.h"

namespace smpk {
namespace {

constexpr int kT = 256;
constexpr int kAhead = 4;  // vectors of 8 elements whose loads a thread has in flight together

struct Chunk {
  int t;          // tensor in the table
  int64_t s, e;  // its elements [s, e)
};

__device__ __forceinline__ Chunk chunk_of(const GradList& l, uint32_t b, int64_t size) {
  int lo = 0, hi = l.count;  // first[lo] <= b < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.first[mid] <= b) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  Chunk c;
  c.t = lo;
  c.s = static_cast<int64_t>(b - l.first[lo]) * size;
  c.e = c.s + size < l.n[lo] ? c.s + size : l.n[lo];
  return c;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double wave_max_bits(double v) {  // non-negative or NaN: ordered by their bits
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double w = __shfl_xor(v, o, 64);
    v = __double_as_longlong(w) > __double_as_longlong(v) ? w : v;
  }
  return v;
}

// all threads get the block's sum or largest value
template <bool INF>
__device__ __forceinline__ double block_join(double v, double* smem) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
  v = INF ? wave_max_bits(v) : wave_sum(v);
  __syncthreads();
  if (lane == 0) smem[wid] = v;
  __syncthreads();
  v = lane < nw ? smem[lane] : 0.0;
  return INF ? wave_max_bits(v) : wave_sum(v);
}

template <bool INF>
struct Acc {
  double sum = 0.0;
  uint32_t top = 0;
  __device__ __forceinline__ void add(float x) {
    if (INF) {
      const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
      top = b > top ? b : top;
    } else {
      const double d = x;
      sum = fma(d, d, sum);
    }
  }
  __device__ __forceinline__ double value() const { return INF ? static_cast<double>(__uint_as_float(top)) : sum; }
};

template <typename T, bool INF>
__device__ __forceinline__ void accumulate(const T* p, int64_t n, Acc<INF>& a) {
  int64_t i = static_cast<int64_t>(threadIdx.x) * kCols;
  for (; i + (kAhead - 1) * kT * kCols + kCols <= n; i += kAhead * kT * kCols) {
    Raw8<T> r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) read8<true>(p + i + u * kT * kCols, kCols, r[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int j = 0; j < kCols; ++j) a.add(at8(r[u], j));
  }
  for (; i < n; i += kT * kCols) {
    const int left = n - i < kCols ? static_cast<int>(n - i) : kCols;
    float x[kCols];
    read8<false>(p + i, left, x);  // (zeros past the end)
#pragma unroll
    for (int j = 0; j < kCols; ++j) a.add(x[j]);
  }
}

template <bool INF>
__global__ void __launch_bounds__(kT) grad_partials(GradList l, int64_t size, double* __restrict__ part) {
  __shared__ double smem[kT / 64];
  const Chunk c = chunk_of(l, blockIdx.x, size);
  Acc<INF> a;
  const int64_t n = c.e - c.s;
  switch (l.dt[c.t]) {
    case F32:
      accumulate<float, INF>(static_cast<const float*>(l.p[c.t]) + c.s, n, a);
      break;
    case F16:
      accumulate<f16, INF>(static_cast<const f16*>(l.p[c.t]) + c.s, n, a);
      break;
    default:
      accumulate<bf16, INF>(static_cast<const bf16*>(l.p[c.t]) + c.s, n, a);
  }
  const double v = block_join<INF>(a.value(), smem);
  if (threadIdx.x == 0) part[l.first_chunk + blockIdx.x] = v;
}

// All partials joined by one block, in an order that depends on their number alone, not on the
// block's: every block of a launch gets the same bits.  Returns scale^2 * sum, or scale * max.
template <bool INF>
__device__ __forceinline__ double join(const double* part, int64_t n, double scale, double* smem) {
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    const double w = part[i];
    if (INF) {
      v = __double_as_longlong(w) > __double_as_longlong(v) ? w : v;
    } else {
      v += w;
    }
  }
  v = block_join<INF>(v, smem);
  return INF ? v * scale : v * scale * scale;
}

// What each gradient is multiplied by: scale, less where the norm is above max_norm.
template <bool INF>
__device__ __forceinline__ float factor_of(double power, double scale, double max_norm) {
  const double f = max_norm / ((INF ? power : sqrt(power)) + 1e-6);
  return static_cast<float>((f > 1.0 ? 1.0 : f) * scale);  // (a NaN stays)
}

template <bool INF>
__global__ void __launch_bounds__(1024) grad_join(const double* __restrict__ part, int64_t n, double scale,
                                                  double max_norm, double* __restrict__ power,
                                                  float* __restrict__ norm, float* __restrict__ factor) {
  __shared__ double smem[16];
  const double p = join<INF>(part, n, scale, smem);
  if (threadIdx.x == 0) {
    *power = p;
    *norm = static_cast<float>(INF ? p : sqrt(p));
    if (factor != nullptr) *factor = factor_of<INF>(p, scale, max_norm);
  }
}

template <typename T, typename O>
__device__ __forceinline__ void scale_chunk(const T* p, O* o, int64_t n, float f) {
  int64_t i = static_cast<int64_t>(threadIdx.x) * kCols;
  for (; i + (kAhead - 1) * kT * kCols + kCols <= n; i += kAhead * kT * kCols) {
    Raw8<T> r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) read8<true>(p + i + u * kT * kCols, kCols, r[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float x[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) x[j] = at8(r[u], j) * f;
      write8<true, false>(o + i + u * kT * kCols, kCols, x);
    }
  }
  for (; i < n; i += kT * kCols) {
    const int left = n - i < kCols ? static_cast<int>(n - i) : kCols;
    float x[kCols];
    read8<false>(p + i, left, x);
#pragma unroll
    for (int j = 0; j < kCols; ++j) x[j] *= f;
    write8<false, false>(o + i, left, x);
  }
}

template <typename T>
__device__ __forceinline__ void scale_to(const T* p, void* o, int odt, int64_t s, int64_t n, float f) {
  switch (odt) {
    case F32:
      scale_chunk(p + s, static_cast<float*>(o) + s, n, f);
      break;
    case F16:
      scale_chunk(p + s, static_cast<f16*>(o) + s, n, f);
      break;
    default:
      scale_chunk(p + s, static_cast<bf16*>(o) + s, n, f);
  }
}

// Last chunk first: what the norm read last is what the caches still hold.
__device__ __forceinline__ void scale_one(const GradList& l, int64_t size, float f) {
  const Chunk c = chunk_of(l, l.first[l.count] - 1 - blockIdx.x, size);
  const int64_t n = c.e - c.s;
  if (f == 1.f && l.p[c.t] == l.o[c.t]) return;  // in place and within the norm: nothing to change
  switch (l.dt[c.t]) {
    case F32:
      scale_to(static_cast<const float*>(l.p[c.t]), l.o[c.t], l.odt[c.t], c.s, n, f);
      break;
    case F16:
      scale_to(static_cast<const f16*>(l.p[c.t]), l.o[c.t], l.odt[c.t], c.s, n, f);
      break;
    default:
      scale_to(static_cast<const bf16*>(l.p[c.t]), l.o[c.t], l.odt[c.t], c.s, n, f);
  }
}

__global__ void __launch_bounds__(kT) grad_scale(GradList l, int64_t size, const float* __restrict__ factor) {
  scale_one(l, size, *factor);
}

// The same for few partials: each block joins them itself, which saves the launch of grad_join.
template <bool INF>
__global__ void __launch_bounds__(kT) grad_join_scale(GradList l, int64_t size, const double* __restrict__ part,
                                                      int64_t n, double scale, double max_norm,
                                                      double* __restrict__ power, float* __restrict__ norm) {
  __shared__ double smem[kT / 64];
  const double p = join<INF>(part, n, scale, smem);
  if (l.first_chunk == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
    *power = p;
    *norm = static_cast<float>(INF ? p : sqrt(p));
  }
  scale_one(l, size, factor_of<INF>(p, scale, max_norm));
}

}  // namespace

int64_t grad_chunk_size(int64_t total) {
  // about 4096 chunks for a large model (16 blocks for each CU), none below 16384 elements
  const int64_t size = (total / 4096 + 2047) / 2048 * 2048;
  return size < 16384 ? 16384 : size;
}

int grad_partials(const GradList& l, int64_t size, int inf, double* part, hipStream_t s) {
  const uint32_t blocks = l.first[l.count];
  if (blocks == 0) return 0;
  if (inf) {
    grad_partials<true><<<blocks, kT, 0, s>>>(l, size, part);
  } else {
    grad_partials<false><<<blocks, kT, 0, s>>>(l, size, part);
  }
  return static_cast<int>(hipGetLastError());
}

int grad_join(const double* part, int64_t n, int inf, double scale, double max_norm, double* power, float* norm,
              float* factor, hipStream_t s) {
  if (inf) {
    grad_join<true><<<1, 1024, 0, s>>>(part, n, scale, max_norm, power, norm, factor);
  } else {
    grad_join<false><<<1, 1024, 0, s>>>(part, n, scale, max_norm, power, norm, factor);
  }
  return static_cast<int>(hipGetLastError());
}

int grad_scale(const GradList& l, int64_t size, const float* factor, hipStream_t s) {
  const uint32_t blocks = l.first[l.count];
  if (blocks == 0) return 0;
  grad_scale<<<blocks, kT, 0, s>>>(l, size, factor);
  return static_cast<int>(hipGetLastError());
}

int grad_join_scale(const GradList& l, int64_t size, const double* part, int64_t n, int inf, double scale,
                    double max_norm, double* power, float* norm, hipStream_t s) {
  const uint32_t blocks = l.first[l.count];
  if (blocks == 0) return 0;
  const auto kernel = inf ? grad_join_scale<true> : grad_join_scale<false>;
  kernel<<<blocks, kT, 0, s>>>(l, size, part, n, scale, max_norm, power, norm);
  return static_cast<int>(hipGetLastError());
}

}  // namespace smpk

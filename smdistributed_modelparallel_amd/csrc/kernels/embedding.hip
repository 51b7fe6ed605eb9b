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

// One block per table row: it looks for its tokens in all of the list, kT at a time, and adds
// their gradient rows in token order.
template <typename T, int N>
__global__ void __launch_bounds__(kT) emb_bwd_scan(IndexList ids, const T* __restrict__ dy, int64_t n, int d,
                                                   float scale, int64_t skip, T* __restrict__ dw, int accumulate) {
  __shared__ int list[kT];
  __shared__ int wave_count[kT / 64];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  for (int c0 = 0; c0 < d; c0 += kT * N) {
    const int c = c0 + threadIdx.x * N;
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    bool any = false;
    for (int64_t t0 = 0; t0 < n; t0 += kT) {
      const int64_t t = t0 + threadIdx.x;
      const bool mine = t < n && row != skip && row_of(ids, t) == row;
      const uint64_t m = __ballot(mine);
      __syncthreads();
      if (lane == 0) wave_count[wid] = __popcll(m);
      __syncthreads();
      int base = 0, total = 0;
      for (int k = 0; k < kT / 64; ++k) {
        if (k < wid) base += wave_count[k];
        total += wave_count[k];
      }
      if (mine) list[base + __popcll(m & ((1ull << lane) - 1))] = threadIdx.x;
      __syncthreads();
      any |= total > 0;
      if (c < d) {
        for (int k = 0; k < total; ++k) {
          float g[N];
          load_pack<T, N>(dy + (t0 + list[k]) * d + c, g);
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] += g[j];
        }
      }
    }
    if (c < d && (any || !accumulate)) {
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] *= scale;
      if (accumulate) {
        float g[N];
        load_pack<T, N>(dw + row * d + c, g);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += g[j];
      }
      store_pack<T, N>(dw + row * d + c, acc);
    }
  }
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

int embedding_bwd(int dt, const IndexList& ids, const void* dy, int64_t n, int64_t d, float scale, int64_t skip,
                  void* dw, int accumulate, hipStream_t s) {
  if (ids.rows <= 0 || d <= 0 || (n <= 0 && accumulate)) return 0;
  SMPK_DISPATCH(dt, T, {
    const int es = sizeof(T);
    if (packs(d, d, dy, es) && packs(d, d, dw, es)) {
      emb_bwd_scan<T, Vec16<T>::N><<<static_cast<unsigned>(ids.rows), kT, 0, s>>>(
          ids, static_cast<const T*>(dy), n, static_cast<int>(d), scale, skip, static_cast<T*>(dw), accumulate);
    } else {
      emb_bwd_scan<T, 1><<<static_cast<unsigned>(ids.rows), kT, 0, s>>>(
          ids, static_cast<const T*>(dy), n, static_cast<int>(d), scale, skip, static_cast<T*>(dw), accumulate);
    }
  });
  return static_cast<int>(hipGetLastError());
}

}  // namespace smpk

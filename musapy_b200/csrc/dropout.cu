// Dropout whose mask is never stored: y = x * keep / (1 - p), keep drawn from
// a counter (philox.cuh), so the backward pass is the same call on the
// gradient with the same seed and offset. No counterpart in the reference.
//
// A thread takes eight elements, one counter, per step: one 16-byte load and
// store of a 16-bit type, two of float. The counter's ~70 integer instructions
// need no loaded value, so they run while the load is under way; eight blocks
// per SM keep enough loads in flight (2^28 f16: 172 us at one counter per
// thread and step and 8 blocks, 194 us at two and 6, 181 us at four and 4; a
// block per 2048 elements instead of a grid of 64 per SM: 187 us).
// Bound: memory (one read and one write per element); 6.2 TB/s at 2^28 f16, 6.5
// TB/s at 2^27 f32.
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "philox.cuh"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kThreads = 256;

template <class T>
struct Eight {
  static constexpr int kWords = (int)sizeof(T) / 2;
  union {
    uint4 w[kWords];
    T v[8];
  };
  MPB_D Eight() {}
};

// What stays is scaled in float and rounded once.
template <class T>
MPB_D void drop_eight(Eight<T>& x, const uint4& w, const Dropper& d) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = to_f(x.v[j]) * d.up;
    x.v[j] = Cvt<T>::from(stays(d, w, j) ? v : 0.0f);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads, 8) k_dropout(const T* __restrict__ x, T* __restrict__ y, int64_t n,
                                                         Dropper d) {
  const int64_t whole = n / 8, stride = (int64_t)gridDim.x * kThreads;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t b = at; b < whole; b += stride) {
    constexpr int N = Eight<T>::kWords;
    Eight<T> v;
#pragma unroll
    for (int k = 0; k < N; ++k) v.w[k] = ld_stream16((const char*)x + (b * N + k) * 16);
    drop_eight(v, philox(d, (uint64_t)b), d);
#pragma unroll
    for (int k = 0; k < N; ++k) st_stream16((char*)y + (b * N + k) * 16, v.w[k]);
  }
  const int64_t i = whole * 8 + at;  // the last elements, fewer than eight
  if (i < n) y[i] = keeps(d, (uint64_t)i) ? Cvt<T>::from(to_f(x[i]) * d.up) : Cvt<T>::from(0.0f);
}

// Addresses that no 16-byte access may use: a thread still takes one counter per step.
template <class T>
__global__ void __launch_bounds__(kThreads) k_dropout_any(const T* __restrict__ x, T* __restrict__ y, int64_t n,
                                                          Dropper d) {
  const int64_t blocks = (n + 7) / 8;
  for (int64_t b = (int64_t)blockIdx.x * kThreads + threadIdx.x; b < blocks; b += (int64_t)gridDim.x * kThreads) {
    const uint4 w = philox(d, (uint64_t)b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t i = b * 8 + j;
      if (i < n) y[i] = stays(d, w, j) ? Cvt<T>::from(to_f(x[i]) * d.up) : Cvt<T>::from(0.0f);
    }
  }
}

template <class T>
int launch_dropout(const void* x, void* y, int64_t n, const Dropper& d, cudaStream_t s) {
  const int64_t want = ((n + 7) / 8 + kThreads - 1) / kThreads, cap = (int64_t)sm_count() * 64;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  if (d.all) return cuda_check(cudaMemsetAsync(y, 0, (size_t)n * sizeof(T), s), "dropout");
  if (((uintptr_t)x | (uintptr_t)y) % 16 == 0) k_dropout<T><<<grid, kThreads, 0, s>>>((const T*)x, (T*)y, n, d);
  else k_dropout_any<T><<<grid, kThreads, 0, s>>>((const T*)x, (T*)y, n, d);
  return launch_check("dropout");
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" int mpb_dropout(int64_t n, const void* x, int dtype, double p, uint64_t seed, uint64_t offset, void* y,
                           mpb_stream_t stream) {
  if (n < 0) return fail(MPB_ERR_SHAPE, "dropout: negative length %lld", (long long)n);
  if (!(p >= 0.0 && p <= 1.0)) return fail(MPB_ERR_INVALID, "dropout: probability %g outside [0, 1]", p);
  if (n > 0 && (!x || !y)) return fail(MPB_ERR_INVALID, "dropout: null pointer");
  const Dropper d = make_dropper(p, seed, offset);
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case MPB_F32: return n ? launch_dropout<float>(x, y, n, d, s) : MPB_OK;
    case MPB_F16: return n ? launch_dropout<__half>(x, y, n, d, s) : MPB_OK;
    case MPB_BF16: return n ? launch_dropout<__nv_bfloat16>(x, y, n, d, s) : MPB_OK;
    default: return fail(MPB_ERR_DTYPE, "dropout: dtype %d not supported (float16, bfloat16, float32)", dtype);
  }
}

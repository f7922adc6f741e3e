// Dropout whose mask is never stored: y = x * keep / (1 - p), keep drawn from
// a counter (philox.cuh), so the backward pass is the same call on the
// gradient with the same seed and offset. No counterpart in the reference.
//
// Bound: memory (one read and one write per element).
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "philox.cuh"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kThreads = 256;

// A thread takes eight elements, one counter, per step.
template <class T>
__global__ void __launch_bounds__(kThreads) k_dropout(const T* __restrict__ x, T* __restrict__ y, int64_t n,
                                                      Dropper d) {
  const int64_t blocks = (n + 7) / 8;
  for (int64_t b = (int64_t)blockIdx.x * kThreads + threadIdx.x; b < blocks; b += (int64_t)gridDim.x * kThreads) {
    const uint4 w = philox(d, (uint64_t)b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t i = b * 8 + j;
      if (i < n) y[i] = half_of(w, j) >= d.drop ? Cvt<T>::from(to_f(x[i]) * d.up) : Cvt<T>::from(0.0f);
    }
  }
}

template <class T>
int launch_dropout(const void* x, void* y, int64_t n, const Dropper& d, cudaStream_t s) {
  const int64_t want = ((n + 7) / 8 + kThreads - 1) / kThreads, cap = (int64_t)sm_count() * 64;
  k_dropout<T><<<(unsigned)(want < cap ? want : cap), kThreads, 0, s>>>((const T*)x, (T*)y, n, d);
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

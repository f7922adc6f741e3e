// Packs of elements and block reductions shared by the row kernels (norms,
// dropout, policy loss) and the gated scan. All arithmetic is in float:
// 16-bit elements are widened on load and rounded once (to nearest even) on
// store.
#pragma once
#include "common.cuh"

namespace mpb {

// N elements of T (N * sizeof(T) a multiple of 4, at most 16 bytes) moved by one load or store;
// the address is a multiple of the pack's size.
template <int BYTES> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

template <class T, int N>
struct Pack {
  using W = typename Word<sizeof(T) * N>::type;
  union {
    W w;
    T v[N];
  };
  MPB_D Pack() {}
};

template <class T>
MPB_D float to_f(T x) {
  return Cvt<float>::from(x);
}

MPB_D float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
MPB_D float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Sum over the block, the same value in every thread (fixed order: lanes by
// butterfly, warps in a butterfly again). `red` holds 32 floats; the caller
// separates uses of the same `red` by a barrier, or alternates two of them.
MPB_D float block_sum(float v, float* red) {
  v = warp_sum(v);
  const int warps = (blockDim.x + 31) >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum(lane < warps ? red[lane] : 0.0f);
}

// sigmoid(g) and 1 - sigmoid(g), both to full relative precision: e^-|g| never
// overflows and neither result is a difference of nearly equal numbers.
MPB_D void sigmoid2(float g, float& s, float& one_minus) {
  const float e = __expf(-fabsf(g));
  const float r = __fdividef(1.0f, 1.0f + e);
  const float q = e * r;
  s = g >= 0.0f ? r : q;
  one_minus = g >= 0.0f ? q : r;
  if (g != g) s = one_minus = g;
}

}  // namespace mpb

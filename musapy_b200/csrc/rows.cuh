// Packs of elements and block reductions shared by the row kernels (norms,
// dropout, policy loss) and the gated scan. All arithmetic is in float:
// 16-bit elements are widened on load and rounded once (to nearest even) on
// store.
#pragma once
#include "common.cuh"
#include <type_traits>

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

// One or two floats. Two go through the packed f32x2 instructions of sm_100,
// which do in one issue slot what takes two: the kernels here are close enough
// to the issue limit for that to matter.
template <int V> struct FloatsOf;
template <> struct FloatsOf<1> { using type = float; };
template <> struct FloatsOf<2> { using type = float2; };
template <int V> using Floats = typename FloatsOf<V>::type;

MPB_D float vadd(float a, float b) { return a + b; }
MPB_D float2 vadd(float2 a, float2 b) { return __fadd2_rn(a, b); }
MPB_D float vmul(float a, float b) { return a * b; }
MPB_D float2 vmul(float2 a, float2 b) { return __fmul2_rn(a, b); }
MPB_D float vfma(float a, float b, float c) { return fmaf(a, b, c); }
MPB_D float2 vfma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
template <int V> MPB_D Floats<V> vset(float c);
template <> MPB_D float vset<1>(float c) { return c; }
template <> MPB_D float2 vset<2>(float c) { return make_float2(c, c); }
MPB_D float vget(float a, int) { return a; }
MPB_D float vget(float2 a, int i) { return i ? a.y : a.x; }
MPB_D void vput(float& a, int, float v) { a = v; }
MPB_D void vput(float2& a, int i, float v) { (i ? a.y : a.x) = v; }

MPB_D float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
MPB_D float rcpf(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
MPB_D float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
constexpr float kMinusLog2e = -1.44269504088896340736f;

// s = sigmoid(g) = 1 / (1 + e) and 1 - s = e s with e = 2^(-g log2 e): neither is
// a difference of nearly equal numbers, so both keep their relative precision:
// a few units in the last place, and what the rounding of -g log2 e to float
// makes of e, up to |g| units of 2^-24. FINE takes that out again: x being the rounded
// argument, e = 2^x (1 + t) with t = -g - x ln 2, which is exact enough in two fused
// multiply-adds. It is for gates in 32 bits; the results of 16-bit gates are
// rounded to far more than the 2^-17 that |g| units come to at most.
// e is held at 2^126, and its 2^-126 is taken off s again: a gate of -inf gives an
// exact 0, and a sigmoid that is not below 2^-102 does not notice. NaN stays NaN.
constexpr float kLeastSigmoid = 1.1754943508222875e-38f;  // 2^-126
constexpr float kMinusLn2 = -0.69314718055994530942f;
constexpr float kMinusLn2Rest = (float)(-0.69314718055994530942 - (double)kMinusLn2);
template <bool FINE>
MPB_D void sigmoid2(float g, float& s, float& one_minus) {
  const float x = g * kMinusLog2e;
  float e = ex2f(min_nan(x, 126.0f));
  if (FINE) {
    const float t = fmaf(x, kMinusLn2Rest, fmaf(x, kMinusLn2, -g));
    e = fmaf(e, fabsf(x) > 126.0f ? 0.0f : t, e);
  }
  const float r = rcpf(1.0f + e);
  s = r - kLeastSigmoid;
  one_minus = e * r;
}
template <bool FINE>
MPB_D void sigmoid2(float2 g, float2& s, float2& one_minus) {
  const float2 x = vmul(g, vset<2>(kMinusLog2e));
  float2 e = make_float2(ex2f(min_nan(x.x, 126.0f)), ex2f(min_nan(x.y, 126.0f)));
  if (FINE) {
    float2 t = vfma(x, vset<2>(kMinusLn2Rest), vfma(x, vset<2>(kMinusLn2), make_float2(-g.x, -g.y)));
    t = make_float2(fabsf(x.x) > 126.0f ? 0.0f : t.x, fabsf(x.y) > 126.0f ? 0.0f : t.y);
    e = vfma(e, t, e);
  }
  const float2 d = vadd(e, vset<2>(1.0f)), r = make_float2(rcpf(d.x), rcpf(d.y));
  s = vadd(r, vset<2>(-kLeastSigmoid));
  one_minus = vmul(e, r);
}

// Elements of a pack as floats, and back.
template <class T>
MPB_D float unpack(const Pack<T, 1>& p) { return to_f(p.v[0]); }
MPB_D float2 unpack(const Pack<float, 2>& p) { return make_float2(p.v[0], p.v[1]); }
MPB_D float2 unpack(const Pack<__half, 2>& p) { return __half22float2(__halves2half2(p.v[0], p.v[1])); }
MPB_D float2 unpack(const Pack<__nv_bfloat16, 2>& p) {
  return make_float2(__uint_as_float(p.w << 16), __uint_as_float(p.w & 0xffff0000u));
}
template <class T>
MPB_D Pack<T, 1> pack(float a) {
  Pack<T, 1> p;
  p.v[0] = Cvt<T>::from(a);
  return p;
}
template <class T>
MPB_D Pack<T, 2> pack(float2 a) {
  Pack<T, 2> p;
  if constexpr (sizeof(T) == 4) {
    p.v[0] = a.x;
    p.v[1] = a.y;
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __float22half2_rn(a);
    p.w = *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __float22bfloat162_rn(a);
    p.w = *reinterpret_cast<const uint32_t*>(&h);
  }
  return p;
}

}  // namespace mpb

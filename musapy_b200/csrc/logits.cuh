// What the losses over rows of logits share (policy loss, distillation): sums of
// exponentials folded as a row arrives, 16 bytes of logits at a time, and the
// tokens in a mask.
#pragma once
#include "rows.cuh"

namespace mpb {

// Tokens in the mask, the same value in every thread: counted before, or here,
// 16 bytes at a time where the mask is aligned.
MPB_D float tokens_in_mask(const uint8_t* mask, int64_t N, const float* counted, float* red) {
  if (!mask) return (float)N;
  if (counted) return *counted;
  int n = 0;
  const int64_t words = (uintptr_t)mask % 16 == 0 ? N / 16 : 0;
  auto set = [](uint32_t v) { return __popc((v | ((v & 0x7f7f7f7fu) + 0x7f7f7f7fu)) & 0x80808080u); };  // bytes that are not 0
#pragma unroll 4
  for (int64_t w = threadIdx.x; w < words; w += blockDim.x) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(mask) + w);
    n += set(v.x) + set(v.y) + set(v.z) + set(v.w);
  }
  for (int64_t i = words * 16 + threadIdx.x; i < N; i += blockDim.x) n += mask[i] ? 1 : 0;
  return block_sum((float)n, red);
}

MPB_D float block_max(float v, float* red) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_max(lane < (int)(blockDim.x >> 5) ? red[lane] : -INFINITY);
}

// e^(z - base) of one value; with another c than log2 e, 2^(c (z - base)).
MPB_D float exp_from(float z, float minus_base, float c = -kMinusLog2e) { return ex2f((z + minus_base) * c); }

// e^(z - base) of many. Near: 2^(z c + k) with c = log2 e (over a temperature) and k = -base c, one
// fused multiply-add each; k is rounded, which scales all of them alike, and
// fix() is the factor that takes this out of them again. Far from zero, where
// the rounding of k is no small number, the difference is taken first.
constexpr float kNear = 65536.0f;  // k is off by at most 2^-8 below it
template <bool NEAR>
struct Exponent {
  float base, k, c;
  MPB_D explicit Exponent(float b, float factor = -kMinusLog2e) : base(b), k(-b * factor), c(factor) {}
  MPB_D float fix() const { return NEAR ? ex2f(-fmaf(base, c, k)) : 1.0f; }
  MPB_D float2 operator()(float2 z) const {
    const float2 x = NEAR ? vfma(z, vset<2>(c), vset<2>(k)) : vmul(vadd(z, vset<2>(-base)), vset<2>(c));
    return make_float2(ex2f(x.x), ex2f(x.y));
  }
};
// f with the form that goes with the base.
template <class F>
MPB_D void with_exponent(float base, F f) {
  if (fabsf(base) <= kNear) f(Exponent<true>(base));
  else f(Exponent<false>(base));
}
template <class F>
MPB_D void with_exponent(float base, float c, F f) {
  if (fabsf(base) * c <= kNear) f(Exponent<true>(base, c));
  else f(Exponent<false>(base, c));
}

// 16 bytes of logits as pairs of floats.
template <class T>
struct Sixteen {
  static constexpr int kElems = 16 / (int)sizeof(T), kPairs = kElems / 2;
  union {
    uint4 w;
    T v[kElems];
    typename Word<2 * sizeof(T)>::type pair[kPairs];
  };
  MPB_D explicit Sixteen(uint4 q) : w(q) {}
  MPB_D float2 get(int i) const {
    Pack<T, 2> p;
    p.w = pair[i];
    return unpack(p);
  }
  MPB_D void put(int i, float2 f) { pair[i] = pack<T>(f).w; }
};

// The pairwise larger of 16 bytes of elements, and the largest of them as float.
template <class T>
MPB_D uint4 larger(uint4 a, uint4 b) {
  auto two = [](uint32_t x, uint32_t y) -> uint32_t {
    if constexpr (std::is_same<T, float>::value) {
      return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&x), *reinterpret_cast<__half2*>(&y));
      return *reinterpret_cast<const uint32_t*>(&m);
    } else {
      const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&x), *reinterpret_cast<__nv_bfloat162*>(&y));
      return *reinterpret_cast<const uint32_t*>(&m);
    }
  };
  return make_uint4(two(a.x, b.x), two(a.y, b.y), two(a.z, b.z), two(a.w, b.w));
}
template <class T>
MPB_D float largest(uint4 a) {
  const Sixteen<T> x(a);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < Sixteen<T>::kPairs; ++i) m = fmaxf(m, fmaxf(x.get(i).x, x.get(i).y));
  return m;
}
// 16 bytes of -inf: in the place of words that a thread does not have.
template <class T>
MPB_D uint4 no_words() {
  const uint32_t w = std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

// The larger maximum, and the sum of exponentials taken from it. -inf with a
// sum of zero is the empty set.
struct Fold {
  float top, sum;
  MPB_D void join(float t, float s, float c = -kMinusLog2e) {
    const float m = fmaxf(top, t), b = m == -INFINITY ? 0.0f : m;
    sum = sum * exp_from(top, -b, c) + s * exp_from(t, -b, c);
    top = m;
  }
};

MPB_D void copy_word16(uint32_t dst, const uint4* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

}  // namespace mpb

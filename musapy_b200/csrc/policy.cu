// Clipped policy loss with a KL term, from logits, with its gradient in the
// same call. For token i with logits z, target t, advantage A, mask m (no
// counterpart in the reference):
//
//   logp = z_t - log sum_j e^z_j          rho = e^(logp - old)
//   L_i  = -min(rho A, clip(rho, 1 - lo, 1 + hi) A) + beta (e^q - q - 1),   q = ref - logp
//   loss = sum m_i L_i / max(1, sum m_i)
//   dloss/dz_j = g_i ([j = t] - e^(z_j - lse)),
//   g_i = m_i / max(1, sum m) * ((clipped ? 0 : -rho A) + beta (1 - e^q))
//
// Tokens outside the mask take no part whatever their logits and targets
// hold: their gradient rows, logp and kl are zero. A target outside the
// vocabulary makes its token's values NaN.
//
// A token's logits are read once: a cluster of 1 to 8 blocks copies the row into
// its shared memory, in 16-byte words that each thread takes for itself (so no
// barrier guards them), folds maximum and sum of exponentials as the copies
// arrive, joins them over the cluster, and turns the row into its gradient
// from shared memory. Blocks of 64 KB leave room for three per SM, so one row's
// copies run under another's stores. Rows of at most 4 KB are a warp's,
// held in registers. Rows that are too long for eight
// blocks, or whose gradient is aligned otherwise than the logits, take three
// passes over global memory.
//
// Bound: memory (logits read, gradient written); next to it the two exponentials
// per element, 119 us each for 4096 x 131072 at 16 per clock and SM. Measured,
// loss and gradient: 4096 x 131072 bf16 423 us (5.1 TB/s), 2048 x 131072 f32 370 us
// (5.8 TB/s), 8192 x 32000 bf16 195 us (5.4 TB/s), 65536 x 1000 bf16 67 us (3.9 TB/s);
// the loss alone, half the bytes, 250 us (4.3 TB/s), 221, 119 and 45 us. Three passes
// over global memory took 1314 us for the first; blocks of 32 KB, six per SM,
// 463 us; one maximum and one rescaling per 16-byte word instead of four, and
// bounds checked per word, 571 us.
#include <cooperative_groups.h>
#include "async_copy.cuh"
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kThreads = 512;

struct PolicyArgs {
  int64_t N, V;
  const void* logits;
  int64_t l_sr;  // row stride, elements
  const void* targets;
  int targets64;
  const float *old_logp, *adv, *ref_logp;
  const uint8_t* mask;
  float lo, hi, beta, grad_scale;
  float *loss, *logp, *kl;
  uint8_t* clipped;
  void* grad;
  float* each;         // per-token loss, scratch
  const float* count;  // tokens in the mask, where a kernel before has counted them
};

// What a token brings besides its logits, loaded before they are waited for.
struct Token {
  float adv, old, ref;
  MPB_D Token(const PolicyArgs& p, int64_t i) : adv(p.adv[i]), old(p.old_logp[i]), ref(p.ref_logp ? p.ref_logp[i] : 0.0f) {}
};

// What a token's logp makes of the loss: its value, kl, clipped and d loss / d logp (without the mean's divisor).
// rho and e^q may be beyond float where they count for nothing: an advantage of
// zero makes rho A zero for every finite exponent, a coefficient of zero leaves
// the KL term out.
MPB_D void token_terms(const PolicyArgs& p, const Token& token, float logp, float& value, float& kl, bool& clipped,
                       float& slope) {
  const float a = token.adv, x = logp - token.old, rho = expf(x);
  clipped = (a > 0.0f && rho > 1.0f + p.hi) || (a < 0.0f && rho < 1.0f - p.lo);
  const float bound = a > 0.0f ? 1.0f + p.hi : 1.0f - p.lo;
  const float gain = a == 0.0f && fabsf(x) < INFINITY ? 0.0f : rho * a;
  value = clipped ? -bound * a : -gain;
  slope = clipped ? 0.0f : -gain;
  kl = 0.0f;
  if (p.ref_logp) {
    const float q = token.ref - logp, em = expm1f(q);
    kl = em - q;
    if (p.beta != 0.0f) {
      value = fmaf(p.beta, kl, value);
      slope = fmaf(-p.beta, em, slope);
    }
  }
}

// Tokens in the mask, the same value in every thread: counted before, or here,
// 16 bytes at a time where the mask is aligned.
MPB_D float tokens_in_mask(const PolicyArgs& p, float* red) {
  if (!p.mask) return (float)p.N;
  if (p.count) return *p.count;
  int n = 0;
  const int64_t words = (uintptr_t)p.mask % 16 == 0 ? p.N / 16 : 0;
  auto set = [](uint32_t v) { return __popc((v | ((v & 0x7f7f7f7fu) + 0x7f7f7f7fu)) & 0x80808080u); };  // bytes that are not 0
#pragma unroll 4
  for (int64_t w = threadIdx.x; w < words; w += blockDim.x) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.mask) + w);
    n += set(v.x) + set(v.y) + set(v.z) + set(v.w);
  }
  for (int64_t i = words * 16 + threadIdx.x; i < p.N; i += blockDim.x) n += p.mask[i] ? 1 : 0;
  return block_sum((float)n, red);
}

MPB_D float block_max(float v, float* red) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_max(lane < (int)(blockDim.x >> 5) ? red[lane] : -INFINITY);
}

// A masked token: zeros.
template <class T>
MPB_D void write_masked(const PolicyArgs& p, int64_t i, int64_t from, int64_t to, int tid, int threads) {
  T* g = (T*)p.grad + i * p.V;
  if (p.grad) {
    // whole 16-byte words where the row has them
    constexpr int E = 16 / sizeof(T);
    const int64_t head = (int64_t)((16 - ((uintptr_t)(g + from) & 15)) & 15) / (int64_t)sizeof(T);
    const int64_t body = from + (head < to - from ? head : to - from), words = (to - body) / E;
    for (int64_t j = from + tid; j < body; j += threads) g[j] = Cvt<T>::from(0.0f);
    for (int64_t w = tid; w < words; w += threads) st_stream16(g + body + w * E, make_uint4(0, 0, 0, 0));
    for (int64_t j = body + words * E + tid; j < to; j += threads) g[j] = Cvt<T>::from(0.0f);
  }
  if (from == 0 && tid == 0) {
    p.each[i] = p.logp[i] = p.kl[i] = 0.0f;
    p.clipped[i] = 0;
  }
}

MPB_D int64_t target_of(const PolicyArgs& p, int64_t i) {
  return p.targets64 ? ((const int64_t*)p.targets)[i] : ((const int32_t*)p.targets)[i];
}

// e^(z - base) of one value.
MPB_D float exp_from(float z, float minus_base) { return ex2f((z + minus_base) * -kMinusLog2e); }

// e^(z - base) of many. Near: 2^(z c + k) with c = log2 e and k = -base c, one
// fused multiply-add each; k is rounded, which scales all of them alike, and
// fix() is the factor that takes this out of them again. Far from zero, where
// the rounding of k is no small number, the difference is taken first.
constexpr float kNear = 65536.0f;  // k is off by at most 2^-8 below it
template <bool NEAR>
struct Exponent {
  float base, k;
  MPB_D explicit Exponent(float b) : base(b), k(b * kMinusLog2e) {}
  MPB_D float fix() const { return NEAR ? ex2f(-fmaf(base, -kMinusLog2e, k)) : 1.0f; }
  MPB_D float2 operator()(float2 z) const {
    const float2 x = NEAR ? vfma(z, vset<2>(-kMinusLog2e), vset<2>(k))
                          : vmul(vadd(z, vset<2>(-base)), vset<2>(-kMinusLog2e));
    return make_float2(ex2f(x.x), ex2f(x.y));
  }
};
// f with the form that goes with the base.
template <class F>
MPB_D void with_exponent(float base, F f) {
  if (fabsf(base) <= kNear) f(Exponent<true>(base));
  else f(Exponent<false>(base));
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
  MPB_D void join(float t, float s) {
    const float m = fmaxf(top, t), b = m == -INFINITY ? 0.0f : m;
    sum = sum * exp_from(top, -b) + s * exp_from(t, -b);
    top = m;
  }
};

constexpr int kRowThreads = 256;
constexpr int kGroups = 4;  // in which a block's copies arrive
constexpr int kBatch = 4;   // words a thread folds at once: one maximum, one rescaling of its sum
constexpr int kMostBlocks = 8;

MPB_D void copy_word16(uint32_t dst, const uint4* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Block `rank` of the row's cluster takes `per` 16-byte words of it. The
// elements before the first aligned word and after the last, fewer than a word
// each, go to the first threads of rank 0.
template <class T>
__global__ void __launch_bounds__(kRowThreads, 3) k_policy_row(PolicyArgs p, int per, int blocks) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint4 words[];
  __shared__ float red[2][32];
  __shared__ float2 folds[kMostBlocks];
  constexpr int E = 16 / (int)sizeof(T);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = blocks > 1 ? (int)cluster.block_rank() : 0;
  const int64_t i = blockIdx.x / blocks;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const T* z = (const T*)p.logits + i * p.l_sr;
  int64_t head = (int64_t)((16 - ((uintptr_t)z & 15)) & 15) / (int64_t)sizeof(T);
  if (head > p.V) head = p.V;
  const int64_t all_words = (p.V - head) / E, tail = head + all_words * E;
  const int64_t w0 = (int64_t)rank * per;
  const int mine = (int)(all_words - w0 < per ? (all_words > w0 ? all_words - w0 : 0) : per);
  const int64_t t = target_of(p, i);
  const Token token(p, i);
  if (p.mask && !p.mask[i]) {  // the whole cluster leaves here
    const int64_t from = rank == 0 ? 0 : head + w0 * E, to = rank == blocks - 1 ? p.V : head + (w0 + per) * E;
    write_masked<T>(p, i, from < p.V ? from : p.V, to < p.V ? to : p.V, threadIdx.x, blockDim.x);
    return;
  }
  // every block of the cluster runs (nothing is made visible by this)
  if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const uint4* src = reinterpret_cast<const uint4*>(z + head) + w0;
  const uint32_t dst = smem_u32(words);
  const int each = (mine + threads - 1) / threads;
  const int quarter = (each + kGroups * kBatch - 1) / (kGroups * kBatch) * kBatch;  // words per thread and group
  // the usual block: sixteen words for every thread, no bounds to check
  const bool full = mine == kGroups * kBatch * threads;
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    if (full) {
#pragma unroll
      for (int k = q * kBatch; k < (q + 1) * kBatch; ++k) copy_word16(dst + (tid + k * threads) * 16, src + tid + k * threads);
    } else {
      for (int k = q * quarter; k < (q + 1) * quarter; ++k)
        if (tid + k * threads < mine) copy_word16(dst + (tid + k * threads) * 16, src + tid + k * threads);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // meanwhile: the elements at the ends, the target's logit, the tokens in the mask
  const int64_t ends = head + (p.V - tail);
  const int64_t end_at = tid < head ? tid : tail + (tid - head);
  const bool has_end = rank == 0 && tid < ends;
  Fold f{-INFINITY, 0.0f};
  float end = 0.0f;
  if (has_end) {
    end = to_f(z[end_at]);
    f.top = end == -INFINITY ? -INFINITY : fmaxf(end, -INFINITY);
    f.sum = exp_from(end, -(end == -INFINITY ? 0.0f : end));
  }
  const bool valid = t >= 0 && t < p.V;
  const float zt = valid ? to_f(z[t]) : 0.0f;
  const float count = p.grad ? tokens_in_mask(p, red[0]) : 1.0f;
  auto fold_batch = [&](const uint4 (&v)[kBatch]) {
    uint4 most = v[0];
#pragma unroll
    for (int j = 1; j < kBatch; ++j) most = larger<T>(most, v[j]);
    const float m = fmaxf(f.top, largest<T>(most)), b = m == -INFINITY ? 0.0f : m;
    f.sum *= exp_from(f.top, -b);
    f.top = m;
    with_exponent(b, [&](auto e) {
      float2 s = vset<2>(0.0f);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const Sixteen<T> x(v[j]);
#pragma unroll
        for (int i = 0; i < Sixteen<T>::kPairs; ++i) s = vadd(s, e(x.get(i)));
      }
      f.sum = fmaf(s.x + s.y, e.fix(), f.sum);
    });
  };
  auto fold_group = [&](int q) {
    uint4 v[kBatch];
    if (full) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) v[j] = words[tid + (q * kBatch + j) * threads];
      fold_batch(v);
      return;
    }
    for (int k = q * quarter; k < (q + 1) * quarter; k += kBatch) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int w = tid + (k + j) * threads;
        v[j] = w < mine ? words[w] : no_words<T>();
      }
      fold_batch(v);
    }
  };
  asm volatile("cp.async.wait_group 3;" ::: "memory");
  fold_group(0);
  asm volatile("cp.async.wait_group 2;" ::: "memory");
  fold_group(1);
  asm volatile("cp.async.wait_group 1;" ::: "memory");
  fold_group(2);
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  fold_group(3);
  // over the block: the maximum, then the sums taken from it, in a fixed order
  __shared__ float tops[32];
  const float wtop = warp_max(f.top);
  if (lane == 0) tops[warp] = wtop;
  __syncthreads();
  const int warps = threads >> 5;
  const float top = warp_max(lane < warps ? tops[lane] : -INFINITY), base = top == -INFINITY ? 0.0f : top;
  float sum = block_sum(f.sum * exp_from(f.top, -base), red[1]);
  float all_top = top;
  if (blocks > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < blocks) *cluster.map_shared_rank(&folds[rank], tid) = make_float2(top, sum);
    cluster.sync();
    Fold c{folds[0].x, folds[0].y};
    for (int k = 1; k < blocks; ++k) c.join(folds[k].x, folds[k].y);
    all_top = c.top;
    sum = c.sum;
  }
  const float all_base = all_top == -INFINITY ? 0.0f : all_top;
  const float logp = valid ? zt - all_base - logf(sum) : NAN;
  float value, kl, slope;
  bool clipped;
  token_terms(p, token, logp, value, kl, clipped, slope);
  if (rank == 0 && tid == 0) {
    p.each[i] = value;
    p.logp[i] = logp;
    p.kl[i] = kl;
    p.clipped[i] = clipped;
  }
  if (!p.grad) return;
  T* g = (T*)p.grad + i * p.V;
  slope *= p.grad_scale / count;
  const float down = -slope / sum;
  uint4* out = reinterpret_cast<uint4*>(g + head) + w0;
  with_exponent(all_base, [&](auto e) {
    const float2 by = vset<2>(down * e.fix());
    auto word = [&](int w) {
      Sixteen<T> x(words[w]);
#pragma unroll
      for (int j = 0; j < Sixteen<T>::kPairs; ++j) x.put(j, vmul(e(x.get(j)), by));
      st_stream16(out + w, x.w);
    };
    if (full) {
#pragma unroll
      for (int k = 0; k < kGroups * kBatch; ++k) word(tid + k * threads);
    } else {
      for (int w = tid; w < mine; w += threads) word(w);
    }
  });
  if (has_end) g[end_at] = Cvt<T>::from(fmaf(down, exp_from(end, -all_base), end_at == t ? slope : 0.0f));
  // the target's element again, by the thread that has written its word
  const int64_t tw = valid && t >= head && t < tail ? (t - head) / E - w0 : -1;
  if (tw >= 0 && tw < mine && tw % threads == tid)
    g[t] = Cvt<T>::from(fmaf(down, exp_from(zt, -all_base), slope));
}

// A warp per token, its logits in registers: rows of at most kLaneWords 16-byte
// words per lane.
constexpr int kLaneWords = 8;
constexpr int kWarpRows = 8;  // warps, tokens, per block

template <class T>
__global__ void __launch_bounds__(kWarpRows * 32) k_policy_warp(PolicyArgs p) {
  __shared__ float red[32];
  constexpr int E = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t i = (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5);
  const float count = p.grad ? tokens_in_mask(p, red) : 1.0f;
  if (i >= p.N) return;
  const Token token(p, i);
  if (p.mask && !p.mask[i]) {
    write_masked<T>(p, i, 0, p.V, lane, 32);
    return;
  }
  const T* z = (const T*)p.logits + i * p.l_sr;
  int head = (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T);
  if (head > p.V) head = (int)p.V;
  const int words = ((int)p.V - head) / E, tail = head + words * E;
  const uint4* src = reinterpret_cast<const uint4*>(z + head);
  uint4 v[kLaneWords];
#pragma unroll
  for (int k = 0; k < kLaneWords; ++k) v[k] = lane + k * 32 < words ? ld_stream16(src + lane + k * 32) : no_words<T>();
  const int end_at = lane < head ? lane : tail + (lane - head);
  const bool has_end = lane < head + ((int)p.V - tail);
  const float end = has_end ? to_f(z[end_at]) : -INFINITY;
  const int64_t t = target_of(p, i);
  const bool valid = t >= 0 && t < p.V;
  const float zt = valid ? to_f(z[t]) : 0.0f;
  uint4 most = v[0];
#pragma unroll
  for (int k = 1; k < kLaneWords; ++k) most = larger<T>(most, v[k]);
  const float top = warp_max(fmaxf(largest<T>(most), end)), base = top == -INFINITY ? 0.0f : top;
  float sum = has_end ? exp_from(end, -base) : 0.0f;
  with_exponent(base, [&](auto e) {
    float2 s = vset<2>(0.0f);
#pragma unroll
    for (int k = 0; k < kLaneWords; ++k) {
      const Sixteen<T> x(v[k]);
      if (k * 32 < words)
#pragma unroll
        for (int j = 0; j < Sixteen<T>::kPairs; ++j) s = vadd(s, e(x.get(j)));
    }
    sum = fmaf(s.x + s.y, e.fix(), sum);
  });
  sum = warp_sum(sum);
  const float logp = valid ? zt - base - logf(sum) : NAN;
  float value, kl, slope;
  bool clipped;
  token_terms(p, token, logp, value, kl, clipped, slope);
  if (lane == 0) {
    p.each[i] = value;
    p.logp[i] = logp;
    p.kl[i] = kl;
    p.clipped[i] = clipped;
  }
  if (!p.grad) return;
  T* g = (T*)p.grad + i * p.V;
  slope *= p.grad_scale / count;
  const float down = -slope / sum;
  uint4* out = reinterpret_cast<uint4*>(g + head);
  with_exponent(base, [&](auto e) {
    const float2 by = vset<2>(down * e.fix());
#pragma unroll
    for (int k = 0; k < kLaneWords; ++k)
      if (lane + k * 32 < words) {
        Sixteen<T> x(v[k]);
#pragma unroll
        for (int j = 0; j < Sixteen<T>::kPairs; ++j) x.put(j, vmul(e(x.get(j)), by));
        st_stream16(out + lane + k * 32, x.w);
      }
  });
  if (has_end) g[end_at] = Cvt<T>::from(fmaf(down, exp_from(end, -base), end_at == t ? slope : 0.0f));
  // the target's element again, by the lane that has written its word
  if (valid && t >= head && t < tail && (t - head) / E % 32 == lane)
    g[t] = Cvt<T>::from(fmaf(down, exp_from(zt, -base), slope));
}

// One block per token, three passes over its logits: maximum, sum, gradient.
template <class T>
__global__ void __launch_bounds__(kThreads) k_policy_passes(PolicyArgs p) {
  __shared__ float red[3][32];
  const int64_t i = blockIdx.x;
  const T* z = (const T*)p.logits + i * p.l_sr;
  T* g = p.grad ? (T*)p.grad + i * p.V : nullptr;
  if (p.mask && !p.mask[i]) {
    write_masked<T>(p, i, 0, p.V, threadIdx.x, blockDim.x);
    return;
  }
  const float count = tokens_in_mask(p, red[0]);
  float top = -INFINITY;
  for (int64_t j = threadIdx.x; j < p.V; j += kThreads) top = fmaxf(top, to_f(z[j]));
  top = block_max(top, red[1]);
  float sum = 0.0f;
  const float base = top == -INFINITY ? 0.0f : top;
  for (int64_t j = threadIdx.x; j < p.V; j += kThreads) sum += exp_from(to_f(z[j]), -base);
  sum = block_sum(sum, red[2]);
  const int64_t t = target_of(p, i);
  const bool valid = t >= 0 && t < p.V;
  const Token token(p, i);
  const float logp = valid ? to_f(z[t]) - base - logf(sum) : NAN;
  float value, kl, slope;
  bool clipped;
  token_terms(p, token, logp, value, kl, clipped, slope);
  if (threadIdx.x == 0) {
    p.each[i] = value;
    p.logp[i] = logp;
    p.kl[i] = kl;
    p.clipped[i] = clipped;
  }
  if (!g) return;
  slope *= p.grad_scale / count;
  const float down = -slope / sum;
  for (int64_t j = threadIdx.x; j < p.V; j += kThreads)
    g[j] = Cvt<T>::from(fmaf(down, exp_from(to_f(z[j]), -base), j == t ? slope : 0.0f));
}

// The mean over the mask, in a fixed order.
__global__ void __launch_bounds__(1024) k_policy_mean(PolicyArgs p) {
  __shared__ float red[2][32];
  const float count = tokens_in_mask(p, red[0]);
  float v = 0.0f;
#pragma unroll 4
  for (int64_t w = threadIdx.x; w < p.N / 4; w += 1024) {
    const float4 f = reinterpret_cast<const float4*>(p.each)[w];
    v += (f.x + f.y) + (f.z + f.w);
  }
  const int64_t last = p.N / 4 * 4 + threadIdx.x;
  if (last < p.N) v += p.each[last];
  v = block_sum(v, red[1]);
  if (threadIdx.x == 0) *p.loss = v / fmaxf(1.0f, count);
}

__global__ void __launch_bounds__(1024) k_policy_count(PolicyArgs p, float* count) {
  __shared__ float red[32];
  const float n = tokens_in_mask(p, red);
  if (threadIdx.x == 0) *count = n;
}

// ------------------------------------------------------------------- host
constexpr int64_t kPart = kRowThreads * kGroups * kBatch;
constexpr int kMostBytes = 208 << 10;   // of a row, where eight blocks have to do

// Every block counts the tokens in the mask itself while its copies are under
// way, as long as that is two loads for each of its threads; of more tokens the
// number is taken by a kernel before.
int count_before(PolicyArgs& p, int threads, cudaStream_t s) {
  if (!p.mask || !p.grad || p.N <= 32 * threads) return MPB_OK;
  float* count = p.each + p.N;
  k_policy_count<<<1, 1024, 0, s>>>(p, count);
  p.count = count;
  return launch_check("policy_loss");
}

template <class T>
int launch_policy(PolicyArgs& p, cudaStream_t s) {
  if (p.N > 0) {
    const int64_t size = sizeof(T), words = p.V * size / 16 > 0 ? p.V * size / 16 : 1;
    // parts of sixteen words for each of 256 threads (64 KB, three blocks per SM); longer rows share by eight
    int64_t blocks64 = (words + kPart - 1) / kPart;
    const int blocks = blocks64 < kMostBlocks ? (int)blocks64 : kMostBlocks;
    const int64_t per = blocks64 <= kMostBlocks ? (words < kPart ? words : kPart) : (words + blocks - 1) / blocks;
    const bool same = !p.grad || (((uintptr_t)p.logits - (uintptr_t)p.grad) % 16 == 0 && (p.l_sr - p.V) * size % 16 == 0);
    if (same && words <= kLaneWords * 32) {
      if (int rc = count_before(p, kWarpRows * 32, s)) return rc;
      k_policy_warp<T><<<(unsigned)((p.N + kWarpRows - 1) / kWarpRows), kWarpRows * 32, 0, s>>>(p);
      if (int rc = launch_check("policy_loss")) return rc;
    } else if (same && per * 16 <= kMostBytes && p.N * blocks <= 0x7fffffffLL) {
      const int bytes = (int)per * 16;
      int threads = (int)((per / (kGroups * kBatch) + 31) / 32 * 32);
      threads = threads < 32 ? 32 : threads > kRowThreads ? kRowThreads : threads;
      if (int rc = count_before(p, threads, s)) return rc;
      if (int rc = allow_smem<k_policy_row<T>, kMostBytes>("policy_loss")) return rc;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(p.N * blocks));
      cfg.blockDim = dim3((unsigned)threads);
      cfg.dynamicSmemBytes = (size_t)bytes;
      cfg.stream = s;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)blocks;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (int rc = launch_check_pdl(cudaLaunchKernelEx(&cfg, k_policy_row<T>, p, (int)per, blocks), "policy_loss"))
        return rc;
    } else {
      if (int rc = count_before(p, kThreads, s)) return rc;
      k_policy_passes<T><<<(unsigned)p.N, kThreads, 0, s>>>(p);
      if (int rc = launch_check("policy_loss")) return rc;
    }
  }
  k_policy_mean<<<1, 1024, 0, s>>>(p);
  return launch_check("policy_loss");
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" {

size_t mpb_policy_loss_scratch_bytes(int64_t N, int64_t V, int dtype) {
  return N > 0 ? ((size_t)N + 1) * sizeof(float) : 0;  // the tokens' losses, their number
}

int mpb_policy_loss(int64_t N, int64_t V, const void* logits, int dtype, int64_t l_sr, const void* targets,
                    int targets_dtype, const float* old_logp, const float* advantages, const float* ref_logp,
                    const void* mask, double clip_low, double clip_high, double kl_coef, double grad_scale, float* loss,
                    float* logp, float* kl, void* clipped, void* dlogits, void* scratch, size_t scratch_bytes,
                    mpb_stream_t stream) {
  if (N < 0 || V < 0) return fail(MPB_ERR_SHAPE, "policy_loss: negative extent");
  if (N > 0x7fffffffLL || (N > 0 && V == 0))
    return fail(MPB_ERR_SHAPE, "policy_loss: %lld tokens over %lld words", (long long)N, (long long)V);
  if (targets_dtype != MPB_I64 && targets_dtype != MPB_I32)
    return fail(MPB_ERR_DTYPE, "policy_loss: targets dtype %d not supported (int32, int64)", targets_dtype);
  if (!(clip_low >= 0.0) || !(clip_high >= 0.0)) return fail(MPB_ERR_INVALID, "policy_loss: negative clip range");
  if (!loss || (N > 0 && (!logits || !targets || !old_logp || !advantages || !logp || !kl || !clipped)))
    return fail(MPB_ERR_INVALID, "policy_loss: null pointer");
  const size_t need = mpb_policy_loss_scratch_bytes(N, V, dtype);
  if (need > scratch_bytes || (need && !scratch))
    return fail(MPB_ERR_SCRATCH, "policy_loss: %zu bytes of scratch, %zu needed", scratch_bytes, need);
  if (need && (uintptr_t)scratch % 16 != 0) return fail(MPB_ERR_INVALID, "policy_loss: scratch not 16-byte aligned");
  PolicyArgs p = {};
  p.N = N, p.V = V, p.logits = logits, p.l_sr = l_sr, p.targets = targets, p.targets64 = targets_dtype == MPB_I64;
  p.old_logp = old_logp, p.adv = advantages, p.ref_logp = ref_logp, p.mask = (const uint8_t*)mask;
  p.lo = (float)clip_low, p.hi = (float)clip_high, p.beta = (float)kl_coef, p.grad_scale = (float)grad_scale;
  p.loss = loss, p.logp = logp, p.kl = kl, p.clipped = (uint8_t*)clipped, p.grad = dlogits, p.each = (float*)scratch;
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case MPB_F32: return launch_policy<float>(p, s);
    case MPB_F16: return launch_policy<__half>(p, s);
    case MPB_BF16: return launch_policy<__nv_bfloat16>(p, s);
    default: return fail(MPB_ERR_DTYPE, "policy_loss: dtype %d not supported (float16, bfloat16, float32)", dtype);
  }
}

}  // extern "C"

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
// Bound: memory (logits read, gradient written).
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
  float* each;  // per-token loss, scratch
};

// What a token's logp makes of the loss: its value, kl, clipped and d loss / d logp (without the mean's divisor).
MPB_D void token_terms(const PolicyArgs& p, int64_t i, float logp, float& value, float& kl, bool& clipped, float& slope) {
  const float a = p.adv[i], rho = __expf(logp - p.old_logp[i]);
  clipped = (a > 0.0f && rho > 1.0f + p.hi) || (a < 0.0f && rho < 1.0f - p.lo);
  const float bound = a > 0.0f ? 1.0f + p.hi : 1.0f - p.lo;
  value = -(clipped ? bound : rho) * a;
  slope = clipped ? 0.0f : -rho * a;
  kl = 0.0f;
  if (p.ref_logp) {
    const float q = p.ref_logp[i] - logp, em = expm1f(q);
    kl = em - q;
    value = fmaf(p.beta, kl, value);
    slope = fmaf(-p.beta, em, slope);
  }
}

MPB_D float tokens_in_mask(const PolicyArgs& p, float* red) {
  float n = 0.0f;
  if (!p.mask) return (float)p.N;
  for (int64_t i = threadIdx.x; i < p.N; i += blockDim.x) n += p.mask[i] ? 1.0f : 0.0f;
  return block_sum(n, red);
}

MPB_D float block_max(float v, float* red) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_max(lane < (int)(blockDim.x >> 5) ? red[lane] : -INFINITY);
}

// One block per token, three passes over its logits: maximum, sum, gradient.
template <class T>
__global__ void __launch_bounds__(kThreads) k_policy(PolicyArgs p) {
  __shared__ float red[3][32];
  const int64_t i = blockIdx.x;
  const T* z = (const T*)p.logits + i * p.l_sr;
  T* g = p.grad ? (T*)p.grad + i * p.V : nullptr;
  if (p.mask && !p.mask[i]) {
    if (g)
      for (int64_t j = threadIdx.x; j < p.V; j += kThreads) g[j] = Cvt<T>::from(0.0f);
    if (threadIdx.x == 0) {
      p.each[i] = p.logp[i] = p.kl[i] = 0.0f;
      p.clipped[i] = 0;
    }
    return;
  }
  const float count = tokens_in_mask(p, red[0]);
  float top = -INFINITY;
  for (int64_t j = threadIdx.x; j < p.V; j += kThreads) top = fmaxf(top, to_f(z[j]));
  top = block_max(top, red[1]);
  float sum = 0.0f;
  const float base = top == -INFINITY ? 0.0f : top;
  for (int64_t j = threadIdx.x; j < p.V; j += kThreads) sum += __expf(to_f(z[j]) - base);
  sum = block_sum(sum, red[2]);
  const int64_t t = p.targets64 ? ((const int64_t*)p.targets)[i] : ((const int32_t*)p.targets)[i];
  const bool valid = t >= 0 && t < p.V;
  const float logp = valid ? to_f(z[t]) - base - logf(sum) : NAN;
  float value, kl, slope;
  bool clipped;
  token_terms(p, i, logp, value, kl, clipped, slope);
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
    g[j] = Cvt<T>::from(fmaf(down, __expf(to_f(z[j]) - base), j == t ? slope : 0.0f));
}

// The mean over the mask, in a fixed order.
__global__ void __launch_bounds__(1024) k_policy_mean(PolicyArgs p) {
  __shared__ float red[2][32];
  const float count = tokens_in_mask(p, red[0]);
  float v = 0.0f;
  for (int64_t i = threadIdx.x; i < p.N; i += 1024) v += p.each[i];
  v = block_sum(v, red[1]);
  if (threadIdx.x == 0) *p.loss = v / fmaxf(1.0f, count);
}

template <class T>
int launch_policy(const PolicyArgs& p, cudaStream_t s) {
  if (p.N > 0) {
    k_policy<T><<<(unsigned)p.N, kThreads, 0, s>>>(p);
    if (int rc = launch_check("policy_loss")) return rc;
  }
  k_policy_mean<<<1, 1024, 0, s>>>(p);
  return launch_check("policy_loss");
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" {

size_t mpb_policy_loss_scratch_bytes(int64_t N, int64_t V, int dtype) { return N > 0 ? (size_t)N * sizeof(float) : 0; }

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

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
// from shared memory. Blocks of up to 72 KB leave room for three per SM, so one
// row's copies run under another's stores. Rows that are too long for eight
// blocks, or whose gradient is aligned otherwise than the logits, take three
// passes over global memory.
//
// Bound: memory (logits read, gradient written).
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
  if (p.count) return *p.count;
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

// A masked token: zeros.
template <class T>
MPB_D void write_masked(const PolicyArgs& p, int64_t i, int64_t from, int64_t to) {
  T* g = (T*)p.grad + i * p.V;
  if (p.grad) {
    // whole 16-byte words where the row has them
    constexpr int E = 16 / sizeof(T);
    const int64_t head = (int64_t)((16 - ((uintptr_t)(g + from) & 15)) & 15) / (int64_t)sizeof(T);
    const int64_t body = from + (head < to - from ? head : to - from), words = (to - body) / E;
    for (int64_t j = from + threadIdx.x; j < body; j += blockDim.x) g[j] = Cvt<T>::from(0.0f);
    for (int64_t w = threadIdx.x; w < words; w += blockDim.x) st_stream16(g + body + w * E, make_uint4(0, 0, 0, 0));
    for (int64_t j = body + words * E + threadIdx.x; j < to; j += blockDim.x) g[j] = Cvt<T>::from(0.0f);
  }
  if (from == 0 && threadIdx.x == 0) {
    p.each[i] = p.logp[i] = p.kl[i] = 0.0f;
    p.clipped[i] = 0;
  }
}

MPB_D int64_t target_of(const PolicyArgs& p, int64_t i) {
  return p.targets64 ? ((const int64_t*)p.targets)[i] : ((const int32_t*)p.targets)[i];
}

// e^(z - base) of a pair.
MPB_D float2 exp_from(float2 z, float2 minus_base) {
  const float2 d = vmul(vadd(z, minus_base), vset<2>(-kMinusLog2e));
  return make_float2(ex2f(d.x), ex2f(d.y));
}
MPB_D float exp_from(float z, float minus_base) { return ex2f((z + minus_base) * -kMinusLog2e); }

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
  MPB_D float top() const {
    float2 m = get(0);
#pragma unroll
    for (int i = 1; i < kPairs; ++i) m = make_float2(fmaxf(m.x, get(i).x), fmaxf(m.y, get(i).y));
    return fmaxf(m.x, m.y);
  }
};

// The larger maximum, and the sum of exponentials taken from it. -inf with a
// sum of zero is the empty set.
struct Fold {
  float top, sum;
  MPB_D float base() const { return top == -INFINITY ? 0.0f : top; }
  MPB_D void join(float t, float s) {
    const float m = fmaxf(top, t), b = m == -INFINITY ? 0.0f : m;
    sum = sum * exp_from(top, -b) + s * exp_from(t, -b);
    top = m;
  }
};

constexpr int kRowThreads = 256;
constexpr int kGroups = 4;  // in which a block's copies arrive
constexpr int kMostBlocks = 8;

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
  if (p.mask && !p.mask[i]) {  // the whole cluster leaves here
    const int64_t from = rank == 0 ? 0 : head + w0 * E, to = rank == blocks - 1 ? p.V : head + (w0 + per) * E;
    write_masked<T>(p, i, from < p.V ? from : p.V, to < p.V ? to : p.V);
    return;
  }
  if (blocks > 1) cluster.barrier_arrive();  // every block of the cluster runs
  const uint4* src = reinterpret_cast<const uint4*>(z + head) + w0;
  const uint32_t dst = smem_u32(words);
  const int each = (mine + threads - 1) / threads, quarter = (each + kGroups - 1) / kGroups;
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    for (int k = q * quarter; k < (q + 1) * quarter; ++k) {
      const int w = tid + k * threads;
      if (w < mine)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + w * 16), "l"(src + w) : "memory");
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
  const int64_t t = target_of(p, i);
  const bool valid = t >= 0 && t < p.V;
  const float zt = valid ? to_f(z[t]) : 0.0f;
  const float count = p.grad ? tokens_in_mask(p, red[0]) : 1.0f;
  auto fold_group = [&](int q) {
    float top = -INFINITY;
    for (int k = q * quarter; k < (q + 1) * quarter; ++k) {
      const int w = tid + k * threads;
      if (w < mine) top = fmaxf(top, Sixteen<T>(words[w]).top());
    }
    const float m = fmaxf(f.top, top), b = m == -INFINITY ? 0.0f : m;
    f.sum *= exp_from(f.top, -b);
    f.top = m;
    const float2 from = vset<2>(-b);
    float2 s = vset<2>(0.0f);
    for (int k = q * quarter; k < (q + 1) * quarter; ++k) {
      const int w = tid + k * threads;
      if (w < mine) {
        const Sixteen<T> x(words[w]);
#pragma unroll
        for (int j = 0; j < Sixteen<T>::kPairs; ++j) s = vadd(s, exp_from(x.get(j), from));
      }
    }
    f.sum += s.x + s.y;
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
    cluster.barrier_wait();
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
  token_terms(p, i, logp, value, kl, clipped, slope);
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
  const float2 from = vset<2>(-all_base), by = vset<2>(down);
  uint4* out = reinterpret_cast<uint4*>(g + head) + w0;
#pragma unroll 4
  for (int w = tid; w < mine; w += threads) {
    Sixteen<T> x(words[w]);
#pragma unroll
    for (int j = 0; j < Sixteen<T>::kPairs; ++j) x.put(j, vmul(exp_from(x.get(j), from), by));
    st_stream16(out + w, x.w);
  }
  if (has_end) g[end_at] = Cvt<T>::from(fmaf(down, exp_from(end, -all_base), end_at == t ? slope : 0.0f));
  // the target's element again, by the thread that has written its word
  const int64_t tw = valid && t >= head && t < tail ? (t - head) / E - w0 : -1;
  if (tw >= 0 && tw < mine && tw % threads == tid)
    g[t] = Cvt<T>::from(fmaf(down, exp_from(zt, -all_base), slope));
}

// One block per token, three passes over its logits: maximum, sum, gradient.
template <class T>
__global__ void __launch_bounds__(kThreads) k_policy_passes(PolicyArgs p) {
  __shared__ float red[3][32];
  const int64_t i = blockIdx.x;
  const T* z = (const T*)p.logits + i * p.l_sr;
  T* g = p.grad ? (T*)p.grad + i * p.V : nullptr;
  if (p.mask && !p.mask[i]) {
    write_masked<T>(p, i, 0, p.V);
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
    g[j] = Cvt<T>::from(fmaf(down, exp_from(to_f(z[j]), -base), j == t ? slope : 0.0f));
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

__global__ void __launch_bounds__(1024) k_policy_count(PolicyArgs p, float* count) {
  __shared__ float red[32];
  const float n = tokens_in_mask(p, red);
  if (threadIdx.x == 0) *count = n;
}

// ------------------------------------------------------------------- host
// Up to here every block counts the tokens in the mask itself while its copies
// are under way (a byte each, from L2); beyond, a kernel before does.
constexpr int64_t kCountedByAll = 8192;
constexpr int kBlockBytes = 72 << 10;   // of a row, three blocks per SM
constexpr int kMostBytes = 208 << 10;   // of a row, where eight blocks have to do

template <class T>
int allow_smem(int bytes) {
  static int allowed[64] = {};
  int dev = 0;
  if (int rc = cuda_check(cudaGetDevice(&dev), "policy_loss")) return rc;
  if (bytes <= (40 << 10) || (dev >= 0 && dev < 64 && allowed[dev] >= bytes)) return MPB_OK;
  if (int rc = cuda_check(cudaFuncSetAttribute(k_policy_row<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                          "policy_loss"))
    return rc;
  if (dev >= 0 && dev < 64) allowed[dev] = bytes;
  return MPB_OK;
}

template <class T>
int launch_policy(PolicyArgs& p, cudaStream_t s) {
  if (p.N > 0) {
    if (p.mask && p.N > kCountedByAll) {
      float* count = p.each + p.N;
      k_policy_count<<<1, 1024, 0, s>>>(p, count);
      if (int rc = launch_check("policy_loss")) return rc;
      p.count = count;
    }
    const int64_t size = sizeof(T), words = p.V * size / 16 + 1;
    int blocks = 1;
    while (blocks < kMostBlocks && (words + blocks - 1) / blocks * 16 > kBlockBytes) blocks *= 2;
    const int64_t per = (words + blocks - 1) / blocks;
    const bool same = !p.grad || (((uintptr_t)p.logits - (uintptr_t)p.grad) % 16 == 0 && (p.l_sr - p.V) * size % 16 == 0);
    if (same && per * 16 <= kMostBytes && p.N * blocks <= 0x7fffffffLL) {
      const int bytes = (int)per * 16;
      int threads = (int)((per / 4 + 31) / 32 * 32);
      threads = threads < 64 ? 64 : threads > kRowThreads ? kRowThreads : threads;
      if (int rc = allow_smem<T>(bytes)) return rc;
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

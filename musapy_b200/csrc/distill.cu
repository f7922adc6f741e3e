// Distillation from a teacher's top logits, with its gradient in the same call
// (no counterpart in the reference). For token i with logits z, the teacher's K
// logits t_k at the vocabulary's places id_k, temperature tau and mask m:
//
//   p = softmax(t / tau) over the K entries      q = softmax(z / tau)
//   kl_i = sum_k p_k (log p_k - log q_(id_k))
//   loss = tau^2 sum m_i kl_i / max(1, sum m_i)
//   dloss/dz_v = m_i tau / max(1, sum m) (q_v - sum_(k: id_k = v) p_k)
//
// An entry whose teacher logit is -inf is left out whatever its place; a token
// whose entries are all left out has no teacher: zeros, though it counts in the
// mean. An entry that takes part with a place outside the vocabulary makes its
// token's values NaN. Tokens outside the mask give zeros whatever they hold.
//
// The row goes the way of the policy loss (policy.cu): a cluster of blocks holds it
// in shared memory, so that it is read once; maximum and sum are folded as its copies arrive
// and joined over the cluster. The teacher's entries, a few hundred bytes, are worked
// on while the copies are under way: their softmax, and for each place the sum of the
// entries that name it, so that the places are written once and in no order that
// could matter. A row that does not fit, or is aligned otherwise than its gradient,
// takes three passes over global memory.
//
// Bound: memory, with two exponentials per logit beside it. 4096 x 131072 bf16 with 64 entries 492 us (4.4 TB/s), 511 x 32003 float
// with 20 entries 33 us on the GPU (4.0 TB/s). The teacher's softmax costs a block three barriers before it folds:
// 497 us with its first entries asked for before the row's copies, 507 behind them; left to one warp while the others
// fold, 536. The policy loss, without a teacher, takes 430 for the same logits.
#include <cooperative_groups.h>
#include "async_copy.cuh"
#include "common.cuh"
#include "internal.h"
#include "logits.cuh"
#include "musapy_b200.h"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kRowThreads = 256;
constexpr int kGroups = 4;  // in which a block's copies arrive
constexpr int kBatch = 4;   // words a thread folds at once
constexpr int kMostBlocks = 8;
constexpr int kMostTop = 1024;  // entries of a teacher's list
constexpr int kPassThreads = 512;

struct DistillArgs {
  int64_t N, V;
  const void* logits;
  int64_t l_sr;
  const void* ids;
  int ids64, K;
  const void* teacher;
  int teacher_dt;
  const uint8_t* mask;
  float tau, grad_scale;
  float *loss, *kl;
  void* grad;
  float* each;         // per-token loss, scratch
  const float* count;  // tokens in the mask, where a kernel before has counted them
};

// A token's teacher in shared memory.
struct Teacher {
  float top, log_sum;  // of the entries over tau
  bool any, bad;       // an entry takes part; one of them is outside the vocabulary
};

MPB_D float teacher_logit(const DistillArgs& p, int64_t at) {
  if (p.teacher_dt == MPB_F32) return ((const float*)p.teacher)[at];
  if (p.teacher_dt == MPB_F16) return to_f(((const __half*)p.teacher)[at]);
  return to_f(((const __nv_bfloat16*)p.teacher)[at]);
}

MPB_D int64_t teacher_id(const DistillArgs& p, int64_t at) {
  return p.ids64 ? ((const int64_t*)p.ids)[at] : ((const int32_t*)p.ids)[at];
}

// A thread's first entry, asked for before the row: behind the row's copies it would arrive last.
struct FirstEntry {
  float x;
  int64_t id;
  MPB_D FirstEntry(const DistillArgs& p, int64_t i) : x(-INFINITY), id(0) {
    if ((int)threadIdx.x < p.K) x = teacher_logit(p, i * p.K + threadIdx.x), id = teacher_id(p, i * p.K + threadIdx.x);
  }
};

// ids (-1: left out), and p: each entry's share. Every thread of the block takes part; red: two of 32 floats.
MPB_D Teacher load_teacher(const DistillArgs& p, int64_t i, const FirstEntry& first, int* ids, float* share, float (*red)[32]) {
  const int tid = threadIdx.x, threads = blockDim.x;
  const float per = 1.0f / p.tau;
  Teacher t;
  float top = -INFINITY;
  bool bad = false, nan = false;
  for (int k = tid; k < p.K; k += threads) {
    const float x = k == tid ? first.x : teacher_logit(p, i * p.K + k);
    const int64_t id = k == tid ? first.id : teacher_id(p, i * p.K + k);
    const bool in = x != -INFINITY, inside = id >= 0 && id < p.V;
    bad |= in && !inside;
    nan |= x != x;
    ids[k] = in && inside ? (int)id : -1;
    share[k] = x;
    top = fmaxf(top, x);
  }
  t.top = block_max(top, red[0]);
  t.bad = __syncthreads_or(bad || nan);
  t.any = t.top != -INFINITY || t.bad;
  const float base = t.top == -INFINITY ? 0.0f : t.top;
  float sum = 0.0f;
  for (int k = tid; k < p.K; k += threads) {
    const float e = expf((share[k] - base) * per);
    share[k] = e;
    sum += e;
  }
  sum = block_sum(sum, red[1]);
  t.log_sum = logf(sum);
  const float down = sum > 0.0f ? 1.0f / sum : 0.0f;
  for (int k = tid; k < p.K; k += threads) {
    const float e = share[k] * down;
    share[k] = e;
    if (e == 0.0f) ids[k] = -1;
  }
  __syncthreads();
  return t;
}

// The sum of the entries that name entry k's place, in their order; false when an earlier one names it.
MPB_D bool place_sum(const DistillArgs& p, const int* ids, const float* share, int k, float& sum) {
  const int id = ids[k];
  sum = 0.0f;
  if (id < 0) return false;
  int first = k;
  for (int j = p.K - 1; j >= 0; --j)
    if (ids[j] == id) {
      sum += share[j];
      first = j;
    }
  return first == k;
}

// An entry's term of kl: p (log p - log q), both logs from their row's maximum.
MPB_D float entry_term(const DistillArgs& p, const Teacher& t, float share, float x, float z, float z_top, float z_log_sum) {
  const float per = 1.0f / p.tau;
  return share * (((x - t.top) * per - t.log_sum) - ((z - z_top) * per - z_log_sum));
}

template <class T>
MPB_D void zero_row(const DistillArgs& p, int64_t i, int64_t from, int64_t to, int tid, int threads) {
  if (p.grad) {
    T* g = (T*)p.grad + i * p.V;
    constexpr int E = 16 / sizeof(T);
    const int64_t head = (int64_t)((16 - ((uintptr_t)(g + from) & 15)) & 15) / (int64_t)sizeof(T);
    const int64_t body = from + (head < to - from ? head : to - from), words = (to - body) / E;
    for (int64_t j = from + tid; j < body; j += threads) g[j] = Cvt<T>::from(0.0f);
    for (int64_t w = tid; w < words; w += threads) st_stream16(g + body + w * E, make_uint4(0, 0, 0, 0));
    for (int64_t j = body + words * E + tid; j < to; j += threads) g[j] = Cvt<T>::from(0.0f);
  }
  if (from == 0 && tid == 0) p.each[i] = p.kl[i] = 0.0f;
}

// The cluster's block `rank` holds `per` 16-byte words of the row; the elements before the first aligned word and behind
// the last go to the first threads of rank 0.
template <class T>
__global__ void __launch_bounds__(kRowThreads, 3) k_distill_row(DistillArgs p, int per, int blocks) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint4 words[];
  __shared__ float red[4][32], share[kMostTop], tops[32];
  __shared__ int ids[kMostTop];
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
    zero_row<T>(p, i, from < p.V ? from : p.V, to < p.V ? to : p.V, tid, threads);
    return;
  }
  const FirstEntry first(p, i);
  // every block of the cluster runs (nothing is made visible by this)
  if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const uint4* src = reinterpret_cast<const uint4*>(z + head) + w0;
  const uint32_t dst = smem_u32(words);
  const int each = (mine + threads - 1) / threads;
  const int quarter = (each + kGroups * kBatch - 1) / (kGroups * kBatch) * kBatch;  // words per thread and group
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
  // meanwhile: the teacher, the elements at the ends, the tokens in the mask
  const float c = -kMinusLog2e / p.tau;
  const int64_t ends = head + (p.V - tail);
  const int64_t end_at = tid < head ? tid : tail + (tid - head);
  const bool has_end = rank == 0 && tid < ends;
  Fold f{-INFINITY, 0.0f};
  float end = 0.0f;
  if (has_end) {
    end = to_f(z[end_at]);
    f.top = end == -INFINITY ? -INFINITY : fmaxf(end, -INFINITY);
    f.sum = exp_from(end, -(end == -INFINITY ? 0.0f : end), c);
  }
  const float count = p.grad ? tokens_in_mask(p.mask, p.N, p.count, red[0]) : 1.0f;
  const Teacher t = load_teacher(p, i, first, ids, share, red + 1);
  auto fold_batch = [&](const uint4 (&v)[kBatch]) {
    uint4 most = v[0];
#pragma unroll
    for (int j = 1; j < kBatch; ++j) most = larger<T>(most, v[j]);
    const float m = fmaxf(f.top, largest<T>(most)), b = m == -INFINITY ? 0.0f : m;
    f.sum *= exp_from(f.top, -b, c);
    f.top = m;
    with_exponent(b, c, [&](auto e) {
      float2 s = vset<2>(0.0f);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const Sixteen<T> x(v[j]);
#pragma unroll
        for (int n = 0; n < Sixteen<T>::kPairs; ++n) s = vadd(s, e(x.get(n)));
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
  const float wtop = warp_max(f.top);
  if (lane == 0) tops[warp] = wtop;
  __syncthreads();
  const int warps = threads >> 5;
  const float top = warp_max(lane < warps ? tops[lane] : -INFINITY), base = top == -INFINITY ? 0.0f : top;
  float sum = block_sum(f.sum * exp_from(f.top, -base, c), red[3]);
  float all_top = top;
  if (blocks > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < blocks) *cluster.map_shared_rank(&folds[rank], tid) = make_float2(top, sum);
    cluster.sync();
    Fold a{folds[0].x, folds[0].y};
    for (int k = 1; k < blocks; ++k) a.join(folds[k].x, folds[k].y, c);
    all_top = a.top;
    sum = a.sum;
  }
  const float all_base = all_top == -INFINITY ? 0.0f : all_top;
  if (rank == 0) {  // the token's divergence
    const float log_sum = logf(sum);
    float v = 0.0f;
    for (int k = tid; k < p.K; k += threads)
      if (ids[k] >= 0) v += entry_term(p, t, share[k], teacher_logit(p, i * p.K + k), to_f(z[ids[k]]), all_base, log_sum);
    v = block_sum(v, red[1]);
    if (tid == 0) {
      if (t.bad) v = NAN;
      p.kl[i] = v;
      p.each[i] = v;
    }
  }
  if (!p.grad) return;
  T* g = (T*)p.grad + i * p.V;
  const float by = t.bad ? NAN : t.any ? p.grad_scale * p.tau / count : 0.0f, down = t.any ? by / sum : 0.0f;
  uint4* out = reinterpret_cast<uint4*>(g + head) + w0;
  with_exponent(all_base, c, [&](auto e) {
    const float2 w2 = vset<2>(down * e.fix());
    auto word = [&](int w) {
      Sixteen<T> x(words[w]);
#pragma unroll
      for (int j = 0; j < Sixteen<T>::kPairs; ++j) x.put(j, vmul(e(x.get(j)), w2));
      st_stream16(out + w, x.w);
    };
    if (!t.any) {
      for (int w = tid; w < mine; w += threads) st_stream16(out + w, make_uint4(0, 0, 0, 0));
    } else if (full) {
#pragma unroll
      for (int k = 0; k < kGroups * kBatch; ++k) word(tid + k * threads);
    } else {
      for (int w = tid; w < mine; w += threads) word(w);
    }
  });
  if (has_end) g[end_at] = Cvt<T>::from(t.any ? down * exp_from(end, -all_base, c) : 0.0f);
  // the teacher's places again, behind the words that hold them
  __syncthreads();
  const int64_t lo = head + w0 * E, hi = lo + (int64_t)mine * E;
  for (int k = tid; k < p.K; k += threads) {
    const int id = ids[k];
    if (!(id >= lo && id < hi) && !(rank == 0 && id >= 0 && (id < head || id >= tail))) continue;
    float s;
    if (place_sum(p, ids, share, k, s)) g[id] = Cvt<T>::from(fmaf(down, exp_from(to_f(z[id]), -all_base, c), -by * s));
  }
}

// One block per token, three passes over its logits.
template <class T>
__global__ void __launch_bounds__(kPassThreads) k_distill_passes(DistillArgs p) {
  __shared__ float red[4][32], share[kMostTop];
  __shared__ int ids[kMostTop];
  const int64_t i = blockIdx.x;
  const T* z = (const T*)p.logits + i * p.l_sr;
  if (p.mask && !p.mask[i]) {
    zero_row<T>(p, i, 0, p.V, threadIdx.x, blockDim.x);
    return;
  }
  const float c = -kMinusLog2e / p.tau;
  const float count = p.grad ? tokens_in_mask(p.mask, p.N, p.count, red[0]) : 1.0f;
  const Teacher t = load_teacher(p, i, FirstEntry(p, i), ids, share, red + 1);
  float top = -INFINITY;
  for (int64_t j = threadIdx.x; j < p.V; j += kPassThreads) top = fmaxf(top, to_f(z[j]));
  top = block_max(top, red[3]);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int64_t j = threadIdx.x; j < p.V; j += kPassThreads) sum += exp_from(to_f(z[j]), -base, c);
  __syncthreads();
  sum = block_sum(sum, red[0]);
  const float log_sum = logf(sum);
  float v = 0.0f;
  for (int k = threadIdx.x; k < p.K; k += kPassThreads)
    if (ids[k] >= 0) v += entry_term(p, t, share[k], teacher_logit(p, i * p.K + k), to_f(z[ids[k]]), base, log_sum);
  v = block_sum(v, red[2]);
  if (threadIdx.x == 0) {
    if (t.bad) v = NAN;
    p.kl[i] = v;
    p.each[i] = v;
  }
  if (!p.grad) return;
  T* g = (T*)p.grad + i * p.V;
  const float by = t.bad ? NAN : t.any ? p.grad_scale * p.tau / count : 0.0f, down = t.any ? by / sum : 0.0f;
  for (int64_t j = threadIdx.x; j < p.V; j += kPassThreads)
    g[j] = Cvt<T>::from(t.any ? down * exp_from(to_f(z[j]), -base, c) : 0.0f);
  __syncthreads();
  for (int k = threadIdx.x; k < p.K; k += kPassThreads) {
    float s;
    if (place_sum(p, ids, share, k, s)) g[ids[k]] = Cvt<T>::from(fmaf(down, exp_from(to_f(z[ids[k]]), -base, c), -by * s));
  }
}

// The mean over the mask, in a fixed order.
__global__ void __launch_bounds__(1024) k_distill_mean(DistillArgs p) {
  __shared__ float red[2][32];
  const float count = tokens_in_mask(p.mask, p.N, p.count, red[0]);
  float v = 0.0f;
#pragma unroll 4
  for (int64_t w = threadIdx.x; w < p.N / 4; w += 1024) {
    const float4 f = reinterpret_cast<const float4*>(p.each)[w];
    v += (f.x + f.y) + (f.z + f.w);
  }
  const int64_t last = p.N / 4 * 4 + threadIdx.x;
  if (last < p.N) v += p.each[last];
  v = block_sum(v, red[1]);
  if (threadIdx.x == 0) *p.loss = p.tau * p.tau * v / fmaxf(1.0f, count);
}

__global__ void __launch_bounds__(1024) k_distill_count(DistillArgs p, float* count) {
  __shared__ float red[32];
  const float n = tokens_in_mask(p.mask, p.N, nullptr, red);
  if (threadIdx.x == 0) *count = n;
}

constexpr int64_t kPart = kRowThreads * kGroups * kBatch;
constexpr int kMostBytes = 208 << 10;  // of a row, where eight blocks have to do

// Every block counts the tokens in the mask itself while its copies are under
// way, as long as that is two loads for each of its threads.
int count_before(DistillArgs& p, int threads, cudaStream_t s) {
  if (!p.mask || !p.grad || p.N <= 32 * threads) return MPB_OK;
  float* count = p.each + p.N;
  k_distill_count<<<1, 1024, 0, s>>>(p, count);
  p.count = count;
  return launch_check("distill_loss");
}

template <class T>
int launch_distill(DistillArgs& p, cudaStream_t s) {
  if (p.N > 0) {
    const int64_t size = sizeof(T), words = p.V * size / 16 > 0 ? p.V * size / 16 : 1;
    // parts of sixteen words for each of 256 threads (64 KB, three blocks per SM); longer rows share by eight
    int64_t blocks64 = (words + kPart - 1) / kPart;
    const int blocks = blocks64 < kMostBlocks ? (int)blocks64 : kMostBlocks;
    const int64_t per = blocks64 <= kMostBlocks ? (words < kPart ? words : kPart) : (words + blocks - 1) / blocks;
    const bool same = !p.grad || (((uintptr_t)p.logits - (uintptr_t)p.grad) % 16 == 0 && (p.l_sr - p.V) * size % 16 == 0);
    if (same && per * 16 <= kMostBytes && p.N * blocks <= 0x7fffffffLL) {
      const int bytes = (int)per * 16;
      int threads = (int)((per / (kGroups * kBatch) + 31) / 32 * 32);
      threads = threads < 32 ? 32 : threads > kRowThreads ? kRowThreads : threads;
      if (int rc = count_before(p, threads, s)) return rc;
      if (int rc = allow_smem<k_distill_row<T>, kMostBytes>("distill_loss")) return rc;
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
      cfg.numAttrs = blocks > 1 ? 1 : 0;
      if (int rc = launch_check_pdl(cudaLaunchKernelEx(&cfg, k_distill_row<T>, p, (int)per, blocks), "distill_loss"))
        return rc;
    } else {
      if (int rc = count_before(p, kPassThreads, s)) return rc;
      k_distill_passes<T><<<(unsigned)p.N, kPassThreads, 0, s>>>(p);
      if (int rc = launch_check("distill_loss")) return rc;
    }
  }
  k_distill_mean<<<1, 1024, 0, s>>>(p);
  return launch_check("distill_loss");
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" {

size_t mpb_distill_loss_scratch_bytes(int64_t N) { return N > 0 ? ((size_t)N + 1) * sizeof(float) : 0; }

int mpb_distill_loss(int64_t N, int64_t V, int64_t K, const void* logits, int dtype, int64_t l_sr, const void* ids,
                     int ids_dtype, const void* teacher, int teacher_dtype, const void* mask, double temperature,
                     double grad_scale, float* loss, float* kl, void* dlogits, void* scratch, size_t scratch_bytes,
                     mpb_stream_t stream) {
  if (N < 0 || V < 0 || K < 0) return fail(MPB_ERR_SHAPE, "distill_loss: negative extent");
  if (N > 0x7fffffffLL || V > 0x7fffffffLL || (N > 0 && V == 0))
    return fail(MPB_ERR_SHAPE, "distill_loss: %lld tokens over %lld words", (long long)N, (long long)V);
  if (K > kMostTop) return fail(MPB_ERR_SHAPE, "distill_loss: %lld entries per token (at most %d)", (long long)K, kMostTop);
  if (ids_dtype != MPB_I64 && ids_dtype != MPB_I32)
    return fail(MPB_ERR_DTYPE, "distill_loss: ids dtype %d not supported (int32, int64)", ids_dtype);
  if (teacher_dtype != MPB_F32 && teacher_dtype != MPB_F16 && teacher_dtype != MPB_BF16)
    return fail(MPB_ERR_DTYPE, "distill_loss: teacher dtype %d not supported (float16, bfloat16, float32)", teacher_dtype);
  if (!(temperature >= 1e-3 && temperature <= 1e3))
    return fail(MPB_ERR_INVALID, "distill_loss: temperature %g outside [0.001, 1000]", temperature);
  if (!loss || (N > 0 && (!logits || !kl || (K > 0 && (!ids || !teacher)))))
    return fail(MPB_ERR_INVALID, "distill_loss: null pointer");
  const size_t need = mpb_distill_loss_scratch_bytes(N);
  if (need > scratch_bytes || (need && !scratch))
    return fail(MPB_ERR_SCRATCH, "distill_loss: %zu bytes of scratch, %zu needed", scratch_bytes, need);
  if (need && (uintptr_t)scratch % 16 != 0) return fail(MPB_ERR_INVALID, "distill_loss: scratch not 16-byte aligned");
  DistillArgs p = {};
  p.N = N, p.V = V, p.logits = logits, p.l_sr = l_sr, p.ids = ids, p.ids64 = ids_dtype == MPB_I64, p.K = (int)K;
  p.teacher = teacher, p.teacher_dt = teacher_dtype, p.mask = (const uint8_t*)mask;
  p.tau = (float)temperature, p.grad_scale = (float)grad_scale;
  p.loss = loss, p.kl = kl, p.grad = dlogits, p.each = (float*)scratch;
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case MPB_F32: return launch_distill<float>(p, s);
    case MPB_F16: return launch_distill<__half>(p, s);
    case MPB_BF16: return launch_distill<__nv_bfloat16>(p, s);
    default: return fail(MPB_ERR_DTYPE, "distill_loss: dtype %d not supported (float16, bfloat16, float32)", dtype);
  }
}

}  // extern "C"

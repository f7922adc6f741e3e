// Embedding lookup with a scale, and the table's gradient (no counterpart in the reference):
//
//   out_n = scale table[token_n]          dtable[v] = scale sum_(n: token_n = v) dout_n
//
// A token outside the table gives a row of NaN and no gradient.
//
// The gradient sums each row's tokens in their order, so that it does not depend on how the
// blocks run: tokens are sorted (stable, by digits of up to nine bits), and what
// names one row lies together. A row named by at most kPart tokens is summed by one group
// of threads; a longer list is cut into parts, whose sums are joined in their order by
// the block that finishes last. A new table is written once, rows that no token names
// as zeros; a gradient that is there already is added to, where tokens name it.
//
// Bound: memory. Up to kSmall tokens one block sorts them, in shared memory; more
// are sorted by two kernels per digit.
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kThreads = 256;
constexpr int kWords = 4;     // of a row that a thread has under way
constexpr int kPart = 32;     // tokens of a row that are summed by one group of threads
constexpr int kMostBits = 9;  // of a digit
constexpr int kMostBins = 1 << kMostBits;
constexpr int kTileTokens = 2048;
constexpr int kSortThreads = 1024;
constexpr int kSmall = 8192;

MPB_D int64_t token_of(const void* tokens, int wide, int64_t n) {
  return wide ? ((const int64_t*)tokens)[n] : (int64_t)((const int32_t*)tokens)[n];
}

// ------------------------------------------------------------- lookup
struct Lookup {
  int64_t N, V, D;
  const void* table;
  int64_t t_sr;
  const void* tokens;
  int wide;
  float scale;
  void* out;
};

// E elements are one access; `lanes` threads (a power of two) take a row.
template <class T, int E>
__global__ void __launch_bounds__(kThreads) k_embed_rows(Lookup p, int lanes) {
  const int64_t n = (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  if (n >= p.N) return;
  const int64_t t = token_of(p.tokens, p.wide, n);
  const bool in = t >= 0 && t < p.V;
  using P = Pack<T, E>;
  const auto* src = reinterpret_cast<const typename P::W*>((const T*)p.table + (in ? t : 0) * p.t_sr);
  auto* dst = reinterpret_cast<typename P::W*>((T*)p.out + n * p.D);
  const int64_t words = p.D / E;
  for (int64_t w = threadIdx.x & (lanes - 1); w < words; w += (int64_t)lanes * kWords) {
    P x[kWords];
#pragma unroll
    for (int k = 0; k < kWords; ++k)
      if (in && w + k * lanes < words) x[k].w = src[w + k * lanes];
#pragma unroll
    for (int k = 0; k < kWords; ++k)
      if (w + k * lanes < words) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[k].v[e] = Cvt<T>::from(in ? to_f(x[k].v[e]) * p.scale : NAN);
        dst[w + k * lanes] = x[k].w;
      }
  }
}

// --------------------------------------------------------------- sort
struct Sorted {
  int64_t N;
  int V;            // also the key of a token outside the table
  const void* tokens;
  int wide;
  int *keys, *at;   // sorted tokens, and where they stand
  int *first, *end; // per row of the table, its tokens among the sorted; null when not asked for
  int *counters;    // cleared here
  int64_t n_counters;
};

MPB_D int key_of(const Sorted& p, int64_t n) {
  const int64_t t = token_of(p.tokens, p.wide, n);
  return t >= 0 && t < p.V ? (int)t : p.V;
}

// Ranks of a warp's 32 keys of one digit among those before them in the warp; count: the warp's counters.
MPB_D int warp_rank(uint16_t* count, int digit, bool on) {
  const unsigned all = __ballot_sync(0xffffffffu, on), same = __match_any_sync(0xffffffffu, on ? digit : -1) & all;
  const int lane = threadIdx.x & 31;
  int before = 0;
  if (on) before = count[digit];
  __syncwarp();
  if (on && lane == 31 - __clz(same)) count[digit] = (uint16_t)(before + __popc(same));
  __syncwarp();
  return before + __popc(same & ((1u << lane) - 1));
}

// Exclusive sums of one value per thread over the block; total in every thread.
template <int THREADS>
MPB_D int block_scan(int v, int* red, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) red[warp] = x;
  __syncthreads();
  int s = lane < THREADS / 32 ? red[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  total = __shfl_sync(0xffffffffu, s, 31);
  const int before = warp ? __shfl_sync(0xffffffffu, s, warp - 1) : 0;
  __syncthreads();
  return before + x - v;
}

// At most kSmall tokens, by one block: each warp has a run of them, each thread eight.
constexpr int kRounds = kSmall / kSortThreads;
constexpr int kSortBytes = kSmall * 4 + kSmall * 2 + (kSortThreads / 32) * kMostBins * 2;

__global__ void __launch_bounds__(kSortThreads) k_embed_sort(Sorted p, int bits, int passes) {
  extern __shared__ __align__(16) int shared[];
  __shared__ int red[32], base[kMostBins];
  constexpr int kWarps = kSortThreads / 32;
  int* keys = shared;
  uint16_t* at = reinterpret_cast<uint16_t*>(keys + kSmall);
  uint16_t* counts = at + kSmall;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = (int)p.N, bins = 1 << bits;
  for (int64_t i = tid; i < p.n_counters; i += kSortThreads) p.counters[i] = 0;
  int key[kRounds], from[kRounds], to[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int i = (warp * kRounds + r) * 32 + lane;
    from[r] = i;
    key[r] = i < n ? key_of(p, i) : 0;
  }
  for (int pass = 0; pass < passes; ++pass) {
    for (int i = tid; i < kWarps * bins; i += kSortThreads) counts[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = (warp * kRounds + r) * 32 + lane;
      to[r] = warp_rank(counts + warp * bins, key[r] >> (pass * bits) & (bins - 1), i < n);
    }
    __syncthreads();
    int total = 0, all;
    if (tid < bins)
      for (int w = 0; w < kWarps; ++w) {
        const int c = counts[w * bins + tid];
        counts[w * bins + tid] = (uint16_t)total;
        total += c;
      }
    const int start = block_scan<kSortThreads>(total, red, all);
    if (tid < bins) base[tid] = start;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = (warp * kRounds + r) * 32 + lane;
      if (i < n) {
        const int digit = key[r] >> (pass * bits) & (bins - 1), o = to[r] + base[digit] + counts[warp * bins + digit];
        keys[o] = key[r];
        at[o] = (uint16_t)from[r];
      }
    }
    __syncthreads();
    if (pass + 1 < passes) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const int i = (warp * kRounds + r) * 32 + lane;
        key[r] = i < n ? keys[i] : 0;
        from[r] = i < n ? at[i] : 0;
      }
      __syncthreads();
    }
  }
  for (int i = tid; i < n; i += kSortThreads) {
    const int k = keys[i];
    p.keys[i] = k;
    p.at[i] = at[i];
    if (p.first && k < p.V) {
      if (i == 0 || keys[i - 1] != k) p.first[k] = i;
      if (i + 1 == n || keys[i + 1] != k) p.end[k] = i + 1;
    }
  }
}

// More tokens: a block per kTileTokens. The digits of a tile, counted; the first pass also clears what later kernels need.
__global__ void __launch_bounds__(kThreads) k_embed_count(Sorted p, const int* keys, int* counts, int shift, int bits) {
  __shared__ int bin[kMostBins];
  const int bins = 1 << bits, tid = threadIdx.x;
  for (int i = tid; i < bins; i += kThreads) bin[i] = 0;
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * kTileTokens;
  for (int i = tid; i < kTileTokens && n0 + i < p.N; i += kThreads)
    atomicAdd(&bin[(keys ? keys[n0 + i] : key_of(p, n0 + i)) >> shift & (bins - 1)], 1);
  if (!keys) {
    const int64_t step = (int64_t)gridDim.x * kThreads, i0 = (int64_t)blockIdx.x * kThreads + tid;
    for (int64_t i = i0; i < p.n_counters; i += step) p.counters[i] = 0;
    if (p.first)
      for (int64_t i = i0; i < p.V; i += step) p.first[i] = p.end[i] = 0;
  }
  __syncthreads();
  for (int i = tid; i < bins; i += kThreads) counts[(int64_t)blockIdx.x * bins + i] = bin[i];
}

// A tile's tokens to their places: behind the smaller digits of all tiles, the same digit of the tiles before, and of
// the tokens before in the tile.
__global__ void __launch_bounds__(kThreads) k_embed_place(Sorted p, const int* keys, const int* at, int* keys_to, int* at_to,
                                                          const int* counts, int shift, int bits) {
  constexpr int kWarps = kThreads / 32, kSteps = kTileTokens / kThreads;
  __shared__ int base[kMostBins], red[32];
  __shared__ uint16_t mine[kWarps * kMostBins];
  const int bins = 1 << bits, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kWarps * bins; i += kThreads) mine[i] = 0;
  int before[kMostBins / kThreads], total[kMostBins / kThreads], sum = 0;
#pragma unroll
  for (int k = 0; k < kMostBins / kThreads; ++k) {
    const int b = tid * (kMostBins / kThreads) + k;
    before[k] = total[k] = 0;
    if (b < bins)
      for (unsigned t = 0; t < gridDim.x; ++t) {
        const int c = counts[(int64_t)t * bins + b];
        if (t < blockIdx.x) before[k] += c;
        total[k] += c;
      }
    sum += total[k];
  }
  int all, start = block_scan<kThreads>(sum, red, all);
#pragma unroll
  for (int k = 0; k < kMostBins / kThreads; ++k) {
    const int b = tid * (kMostBins / kThreads) + k;
    if (b < bins) base[b] = start + before[k];
    start += total[k];
  }
  const int64_t n0 = (int64_t)blockIdx.x * kTileTokens;
  int key[kSteps], to[kSteps];
#pragma unroll
  for (int r = 0; r < kSteps; ++r) {
    const int64_t i = n0 + (warp * kSteps + r) * 32 + lane;
    key[r] = i >= p.N ? 0 : keys ? keys[i] : key_of(p, i);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSteps; ++r) {
    const int64_t i = n0 + (warp * kSteps + r) * 32 + lane;
    to[r] = warp_rank(mine + warp * bins, key[r] >> shift & (bins - 1), i < p.N);
  }
  __syncthreads();
  for (int b = tid; b < bins; b += kThreads) {
    int s = 0;
    for (int w = 0; w < kWarps; ++w) {
      const int c = mine[w * bins + b];
      mine[w * bins + b] = (uint16_t)s;
      s += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSteps; ++r) {
    const int64_t i = n0 + (warp * kSteps + r) * 32 + lane;
    if (i >= p.N) continue;
    const int digit = key[r] >> shift & (bins - 1), o = base[digit] + mine[warp * bins + digit] + to[r];
    keys_to[o] = key[r];
    at_to[o] = at ? at[i] : (int)i;
  }
}

__global__ void __launch_bounds__(kThreads) k_embed_ends(Sorted p) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= p.N) return;
  const int k = p.keys[i];
  if (k >= p.V) return;
  if (i == 0 || p.keys[i - 1] != k) p.first[k] = (int)i;
  if (i + 1 == p.N || p.keys[i + 1] != k) p.end[k] = (int)i + 1;
}

// ----------------------------------------------------------- gradient
struct Sums {
  int64_t N, D;
  int V;
  const void* dout;
  int64_t d_sr;
  const int *keys, *at, *first, *end;
  float scale;
  float* table;
  bool into;
  float* parts;   // sums of the parts of long lists, one row each
  int* counters;  // per place of a part and tile of columns: parts that are done
  int64_t part_blocks;
  int tiles;      // of columns
};

// acc += the E columns from `c` of the tokens sorted at [s, e), in their order.
template <class T, int E>
MPB_D void sum_rows(const Sums& p, int s, int e, int64_t c, float (&acc)[E]) {
  constexpr int kAhead = 8;
  using P = Pack<T, E>;
  const T* x = (const T*)p.dout + c;
  for (int i = s; i < e; i += kAhead) {
    P v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k < e) v[k].w = *reinterpret_cast<const typename P::W*>(x + (int64_t)p.at[i + k] * p.d_sr);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k < e) {
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] += to_f(v[k].v[j]);
      }
  }
}

template <int E>
MPB_D void put_row(const Sums& p, int row, int64_t c, const float (&acc)[E]) {
  float* to = p.table + (int64_t)row * p.D + c;
  if constexpr (E % 4 == 0) {
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      float4 v = make_float4(acc[j] * p.scale, acc[j + 1] * p.scale, acc[j + 2] * p.scale, acc[j + 3] * p.scale);
      float4* at = reinterpret_cast<float4*>(to + j);
      if (p.into) {
        const float4 o = *at;
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
      }
      *at = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) to[j] = p.into ? to[j] + acc[j] * p.scale : acc[j] * p.scale;
  }
}

// The end of the list of row `key` that sorted place s belongs to, and its begin, looked for in growing steps.
MPB_D int list_end(const Sums& p, int s, int key) {
  int64_t at = s, step = 1;  // keys[at] == key
  while (at + step < p.N && p.keys[at + step] == key) at += step, step <<= 1;
  for (; step; step >>= 1)
    if (at + step < p.N && p.keys[at + step] == key) at += step;
  return (int)at + 1;
}
MPB_D int list_begin(const Sums& p, int s, int key) {
  int64_t at = s, step = 1;
  while (at - step >= 0 && p.keys[at - step] == key) at -= step, step <<= 1;
  for (; step; step >>= 1)
    if (at - step >= 0 && p.keys[at - step] == key) at -= step;
  return (int)at;
}

// Where the part that begins at sorted place i keeps its sum: a list longer than kPart begins, and one of its later parts
// begins, at most once among kPart neighbouring places.
MPB_D int64_t part_place(int i, bool begins) { return (int64_t)(i / kPart) * 2 + (begins ? 1 : 0); }

// The first blocks take the parts of long lists, one each; the others the rows: of the whole table, or the lists' first
// tokens. `lanes` threads (a power of two, a warp at least) take a tile of a row.
template <class T, int E>
__global__ void __launch_bounds__(kThreads) k_embed_sums(Sums p, int lanes) {
  if (blockIdx.x < p.part_blocks) {
    __shared__ bool last;
    const int tile = (int)(blockIdx.x % p.tiles);
    const int64_t place = blockIdx.x / p.tiles;
    const int w0 = (int)(place >> 1) * kPart, w1 = (int)min((int64_t)w0 + kPart, p.N), n = (int)p.N;
    int i, key, s, e;
    if (place & 1) {  // a long list that begins here reaches behind these places
      if (w1 >= n) return;
      key = p.keys[w1 - 1];
      if (p.keys[w1] != key) return;
      s = list_begin(p, w1 - 1, key);
      if (s < w0) return;
      i = s;
    } else {  // the list that the first place is of
      key = p.keys[w0];
      s = list_begin(p, w0, key);
      i = s + (w0 - s + kPart - 1) / kPart * kPart;
      if (i == s || i >= w1 || p.keys[i] != key) return;
    }
    if (key >= p.V) return;
    e = list_end(p, i, key);
    if (e - s <= kPart) return;
    const int64_t c0 = (int64_t)tile * kThreads * E, c = c0 + threadIdx.x * E;
    const bool on = c < p.D;
    float acc[E] = {};
    if (on) {
      sum_rows<T, E>(p, i, min(e, i + kPart), c, acc);
      float* to = p.parts + place * p.D + c;
#pragma unroll
      for (int j = 0; j < E; ++j) to[j] = acc[j];
    }
    __threadfence();
    __syncthreads();
    const int parts = (e - s + kPart - 1) / kPart;
    if (threadIdx.x == 0) last = atomicAdd(&p.counters[part_place(s, true) / 2 * p.tiles + tile], 1) == parts - 1;
    __syncthreads();
    if (!last || !on) return;
    __threadfence();
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] = 0.0f;
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
      const float* from = p.parts + part_place(s + k * kPart, k == 0) * p.D + c;
#pragma unroll
      for (int j = 0; j < E; ++j) acc[j] += __ldcg(from + j);
    }
    put_row<E>(p, key, c, acc);
    return;
  }
  const int64_t block = blockIdx.x - p.part_blocks, item = block / p.tiles * (kThreads / lanes) + threadIdx.x / lanes;
  const int tile = (int)(block % p.tiles);
  int row, s, e;
  if (p.into) {
    if (item >= p.N) return;
    s = (int)item;
    row = p.keys[s];
    if (row >= p.V || (s > 0 && p.keys[s - 1] == row)) return;
    e = list_end(p, s, row);
  } else {
    if (item >= p.V) return;
    row = (int)item;
    s = p.first[row];
    e = p.end[row];
  }
  if (e - s > kPart) return;
  const int64_t c = ((int64_t)tile * lanes + (threadIdx.x & (lanes - 1))) * E;
  if (c >= p.D) return;
  float acc[E] = {};
  sum_rows<T, E>(p, s, e, c, acc);
  put_row<E>(p, row, c, acc);
}

// ------------------------------------------------------------------- host
// Threads of a row: enough for `words`, a power of two.
int lanes_for(int64_t words, int least) {
  int lanes = least;
  while (lanes < kThreads && lanes < words) lanes *= 2;
  return lanes;
}

template <class T>
int launch_lookup(const Lookup& p, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool wide = ((uintptr_t)p.table | (uintptr_t)p.out) % 16 == 0 && p.D % E == 0 && p.t_sr % E == 0;
  const int64_t words = wide ? p.D / E : p.D;
  const int lanes = lanes_for((words + kWords - 1) / kWords, 8), rows = kThreads / lanes;
  const unsigned grid = (unsigned)((p.N + rows - 1) / rows);
  if (wide) k_embed_rows<T, E><<<grid, kThreads, 0, s>>>(p, lanes);
  else k_embed_rows<T, 1><<<grid, kThreads, 0, s>>>(p, lanes);
  return launch_check("embedding");
}

struct Digits {
  int bits, passes;
  explicit Digits(int64_t V) {  // keys 0 .. V
    int all = 1;
    while (all < 31 && (1LL << all) <= V) ++all;
    passes = (all + kMostBits - 1) / kMostBits;
    bits = (all + passes - 1) / passes;
  }
};

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

struct Scratch {
  size_t keys, at, keys2, at2, counts, first, end, counters, parts, bytes;
  int64_t n_counters;
  Scratch(int64_t N, int64_t V, int64_t D, bool into) {
    const size_t n = round16((size_t)N * 4);
    const int64_t windows = (N + kPart - 1) / kPart, col_tiles = (D + kThreads - 1) / kThreads;
    const bool small = N <= kSmall;
    keys = 0, at = n, keys2 = 2 * n, at2 = keys2 + (small ? 0 : n), counts = at2 + (small ? 0 : n);
    first = counts + (small ? 0 : round16((size_t)((N + kTileTokens - 1) / kTileTokens) * kMostBins * 4));
    end = first + (into ? 0 : round16((size_t)V * 4));
    counters = end + (into ? 0 : round16((size_t)V * 4));
    n_counters = windows * col_tiles;
    parts = counters + round16((size_t)n_counters * 4);
    bytes = parts + (N > kPart ? (size_t)windows * 2 * D * 4 : 0);
  }
};

int sort_tokens(Sorted& p, char* scratch, const Scratch& w, cudaStream_t s) {
  const Digits g(p.V);
  if (p.N <= kSmall) {
    if (p.first)
      if (int rc = cuda_check(cudaMemsetAsync(p.first, 0, w.counters - w.first, s), "embedding_backward")) return rc;
    if (int rc = allow_smem<k_embed_sort, kSortBytes>("embedding_backward")) return rc;
    k_embed_sort<<<1, kSortThreads, kSortBytes, s>>>(p, g.bits, g.passes);
    return launch_check("embedding_backward");
  }
  int *a_keys = p.keys, *a_at = p.at, *b_keys = (int*)(scratch + w.keys2), *b_at = (int*)(scratch + w.at2);
  const unsigned tiles = (unsigned)((p.N + kTileTokens - 1) / kTileTokens);
  int* counts = (int*)(scratch + w.counts);
  if (g.passes % 2 == 0) std::swap(a_keys, b_keys), std::swap(a_at, b_at);  // the last pass writes to p.keys
  const int *from_keys = nullptr, *from_at = nullptr;
  for (int k = 0; k < g.passes; ++k) {
    k_embed_count<<<tiles, kThreads, 0, s>>>(p, from_keys, counts, k * g.bits, g.bits);
    k_embed_place<<<tiles, kThreads, 0, s>>>(p, from_keys, from_at, a_keys, a_at, counts, k * g.bits, g.bits);
    if (int rc = launch_check("embedding_backward")) return rc;
    from_keys = a_keys, from_at = a_at;
    std::swap(a_keys, b_keys), std::swap(a_at, b_at);
  }
  if (p.first) k_embed_ends<<<(unsigned)((p.N + kThreads - 1) / kThreads), kThreads, 0, s>>>(p);
  return launch_check("embedding_backward");
}

template <class T, int E>
int launch_sums(Sums& p, cudaStream_t s) {
  const int64_t words = (p.D + E - 1) / E;
  const int lanes = lanes_for(words, 32);  // fewer than a block's only where they cover the row
  p.tiles = (int)((words + kThreads - 1) / kThreads);
  p.part_blocks = p.N > kPart ? (p.N + kPart - 1) / kPart * 2 * p.tiles : 0;
  const int64_t items = p.into ? p.N : p.V, groups = kThreads / lanes;
  const int64_t blocks = p.part_blocks + (items + groups - 1) / groups * p.tiles;
  if (blocks > 0x7fffffffLL) return fail(MPB_ERR_SHAPE, "embedding_backward: %lld blocks are too many for one call", (long long)blocks);
  if (blocks == 0) return MPB_OK;
  k_embed_sums<T, E><<<(unsigned)blocks, kThreads, 0, s>>>(p, lanes);
  return launch_check("embedding_backward");
}

template <class T>
int launch_gradient(Sums& p, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool wide = ((uintptr_t)p.dout | (uintptr_t)p.table) % 16 == 0 && p.D % E == 0 && p.d_sr % E == 0;
  return wide ? launch_sums<T, E>(p, s) : launch_sums<T, 1>(p, s);
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" {

int mpb_embedding(int64_t N, int64_t V, int64_t D, const void* table, int dtype, int64_t t_sr, const void* tokens,
                  int tokens_dtype, double scale, void* out, mpb_stream_t stream) {
  if (N < 0 || V < 0 || D < 0) return fail(MPB_ERR_SHAPE, "embedding: negative extent");
  if (N > 0x7fffffffLL) return fail(MPB_ERR_SHAPE, "embedding: %lld tokens are too many for one call", (long long)N);
  if (tokens_dtype != MPB_I64 && tokens_dtype != MPB_I32)
    return fail(MPB_ERR_DTYPE, "embedding: tokens dtype %d not supported (int32, int64)", tokens_dtype);
  if (dtype != MPB_F32 && dtype != MPB_F16 && dtype != MPB_BF16)
    return fail(MPB_ERR_DTYPE, "embedding: dtype %d not supported (float16, bfloat16, float32)", dtype);
  if (N * D == 0) return MPB_OK;
  if ((V > 0 && !table) || !tokens || !out) return fail(MPB_ERR_INVALID, "embedding: null pointer");
  const Lookup p = {N, V, D, table, t_sr, tokens, tokens_dtype == MPB_I64, (float)scale, out};
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case MPB_F32: return launch_lookup<float>(p, s);
    case MPB_F16: return launch_lookup<__half>(p, s);
    default: return launch_lookup<__nv_bfloat16>(p, s);
  }
}

size_t mpb_embedding_backward_scratch_bytes(int64_t N, int64_t V, int64_t D, int into) {
  return N > 0 && V > 0 && D > 0 ? Scratch(N, V, D, into != 0).bytes : 0;
}

int mpb_embedding_backward(int64_t N, int64_t V, int64_t D, const void* dout, int dtype, int64_t d_sr, const void* tokens,
                           int tokens_dtype, double scale, int into, float* dtable, void* scratch, size_t scratch_bytes,
                           mpb_stream_t stream) {
  const char* name = "embedding_backward";
  if (N < 0 || V < 0 || D < 0) return fail(MPB_ERR_SHAPE, "%s: negative extent", name);
  if (N > 0x7fffffffLL - kPart || V > 0x7ffffffeLL)
    return fail(MPB_ERR_SHAPE, "%s: %lld tokens over %lld rows are too many for one call", name, (long long)N, (long long)V);
  if (tokens_dtype != MPB_I64 && tokens_dtype != MPB_I32)
    return fail(MPB_ERR_DTYPE, "%s: tokens dtype %d not supported (int32, int64)", name, tokens_dtype);
  if (dtype != MPB_F32 && dtype != MPB_F16 && dtype != MPB_BF16)
    return fail(MPB_ERR_DTYPE, "%s: dtype %d not supported (float16, bfloat16, float32)", name, dtype);
  if (V * D == 0) return MPB_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (!dtable || (N > 0 && (!dout || !tokens))) return fail(MPB_ERR_INVALID, "%s: null pointer", name);
  if (N == 0) return into ? MPB_OK : cuda_check(cudaMemsetAsync(dtable, 0, (size_t)V * D * 4, s), name);
  const Scratch w(N, V, D, into != 0);
  if (w.bytes > scratch_bytes || !scratch)
    return fail(MPB_ERR_SCRATCH, "%s: %zu bytes of scratch, %zu needed", name, scratch_bytes, w.bytes);
  if ((uintptr_t)scratch % 16 != 0) return fail(MPB_ERR_INVALID, "%s: scratch not 16-byte aligned", name);
  char* at = (char*)scratch;
  Sorted o = {N, (int)V, tokens, tokens_dtype == MPB_I64, (int*)(at + w.keys), (int*)(at + w.at),
              into ? nullptr : (int*)(at + w.first), into ? nullptr : (int*)(at + w.end), (int*)(at + w.counters), w.n_counters};
  if (int rc = sort_tokens(o, at, w, s)) return rc;
  Sums p = {N, D, (int)V, dout, d_sr, o.keys, o.at, o.first, o.end, (float)scale, dtable, into != 0, (float*)(at + w.parts),
            o.counters, 0, 1};
  switch (dtype) {
    case MPB_F32: return launch_gradient<float>(p, s);
    case MPB_F16: return launch_gradient<__half>(p, s);
    default: return launch_gradient<__nv_bfloat16>(p, s);
  }
}

}  // extern "C"

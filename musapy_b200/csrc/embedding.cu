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
// Bound: memory. Up to kFew tokens need no sort, up to kSmall are sorted by one kernel, more by two for each digit, and three from
// 2^18 on.
// Lookup of 32768 rows of 4096 bf16: 82 us (6.5 TB/s); 64 rows 2.3 us on the GPU. Gradient of 32768 tokens of 32000 x 2048 from
// bf16: 130 us, of which the sums 98 (4.1 TB/s; they wait on three loads in a row: the list, its tokens, their rows) and the sort 27; of 4097 of
// 50257 x 769 float, added: 24 us on the GPU, sort 6, sums 18 (rows that begin at no 16-byte boundary go by single elements).
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kThreads = 256;
constexpr int kWords = 4;     // of a row that a thread has under way
// Tokens of a row that are summed by one group of threads. Of 32768 tokens of 32000 x 2048 bf16, and of 4097 of 50257 x 769
// float: 98 and 17.7 us for the sums at 32, 121 and 20.8 at 16, 161 and 27 at 8; at 64, not
// taken up, the calls take 142 instead of 148 and 37 instead of 39 us.
constexpr int kPart = 32;
constexpr int kMostBits = 9;  // of a digit
constexpr int kMostBins = 1 << kMostBits;
constexpr int kTileTokens = 2048;
// Tiles whose counts each block of the sort sums by itself: quadratic, where a scan of them is one more launch per digit. 32000 rows of
// 8 from 128 tiles: 134 us, scanned 137; 256: 237 and 217; 8192: 20.7 and 7.5 ms.
constexpr int kFewTiles = 128;
// Tokens that one kernel sorts, by counting. 32000 rows of 64, a new table: 2048, 4097, 6000 and 8192 tokens 32, 35, 42 and 45 us, by digits
// 51, 52, 53 and 55.
constexpr int kSmall = 8192;
constexpr int kSmallBytes = (kSmall + 32) * 8;

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

// Ranks of a warp's 32 keys of one digit among those before them in the warp; count: the warp's counters. Who has the
// same digit is found by a vote for each of its bits (the instruction that matches whole words took 5 times as long).
MPB_D int warp_rank(uint16_t* count, int digit, int bits, bool on) {
  unsigned same = __ballot_sync(0xffffffffu, on);
  for (int b = 0; b < bits; ++b) {
    const bool set = digit >> b & 1;
    const unsigned with = __ballot_sync(0xffffffffu, set);
    same &= set ? with : ~with;
  }
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

// At most kSmall tokens: a token's place is the number of tokens that sort before it, counted against all of them: a
// key and its index are one number, so that is a comparison for each. A block finds the places of 32 tokens, each of
// its warps against an eighth of the keys; it takes all keys into shared memory. 4097 tokens: 6.1 us, where one
// block sorting them by digits took 12.8. C: a number that holds key and index.
template <class C>
__global__ void __launch_bounds__(kThreads) k_embed_rank(Sorted p) {
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ int part[kThreads / 32][32];
  C* all = reinterpret_cast<C*>(shared);
  constexpr int kAtOnce = 16 / (int)sizeof(C), kWarps = kThreads / 32;
  const int n = (int)p.N, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = ((n + kWarps - 1) / kWarps + kAtOnce - 1) / kAtOnce * kAtOnce;  // of keys, for a warp
#pragma unroll 8
  for (int i = tid; i < run * kWarps; i += kThreads) all[i] = i < n ? (C)key_of(p, i) * kSmall + i : ~(C)0;
  if (blockIdx.x == 0)
    for (int64_t i = tid; i < p.n_counters; i += kThreads) p.counters[i] = 0;
  __syncthreads();
  const int mine = blockIdx.x * 32 + lane;
  const C own = mine < n ? all[mine] : 0;
  int before = 0;
  const uint4* w = reinterpret_cast<const uint4*>(all + warp * run);
#pragma unroll 8
  for (int i = 0; i < run / kAtOnce; ++i) {
    union { uint4 q; C c[kAtOnce]; } x;
    x.q = w[i];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) before += x.c[k] < own ? 1 : 0;
  }
  part[warp][lane] = before;
  __syncthreads();
  if (warp != 0 || mine >= n) return;
#pragma unroll
  for (int k = 1; k < kWarps; ++k) before += part[k][lane];
  p.keys[before] = (int)(own / kSmall);
  p.at[before] = mine;
}

// More tokens: a block per kTileTokens. The digits of a tile, counted; the first pass also clears what later kernels need.
__global__ void __launch_bounds__(kThreads) k_embed_count(Sorted p, const int* keys, int* counts, int shift, int bits) {
  __shared__ int bin[kMostBins];
  const int bins = 1 << bits, tid = threadIdx.x;
  for (int i = tid; i < bins; i += kThreads) bin[i] = 0;
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * kTileTokens;
  int key[kTileTokens / kThreads];
#pragma unroll
  for (int k = 0; k < kTileTokens / kThreads; ++k) {
    const int64_t i = n0 + tid + k * kThreads;
    key[k] = i >= p.N ? -1 : keys ? keys[i] : key_of(p, i);
  }
#pragma unroll
  for (int k = 0; k < kTileTokens / kThreads; ++k)
    if (key[k] >= 0) atomicAdd(&bin[key[k] >> shift & (bins - 1)], 1);
  if (!keys) {
    const int64_t step = (int64_t)gridDim.x * kThreads, i0 = (int64_t)blockIdx.x * kThreads + tid;
    for (int64_t i = i0; i < p.n_counters; i += step) p.counters[i] = 0;
    if (p.first)
      for (int64_t i = i0; i < p.V; i += step) p.first[i] = p.end[i] = 0;
  }
  __syncthreads();
  for (int i = tid; i < bins; i += kThreads) counts[(int64_t)blockIdx.x * bins + i] = bin[i];
}

// The counts of many tiles, per digit: in the place of each the sum of those before it, and the sum of all. A block takes 32
// digits; each of its warps a run of tiles.
constexpr int kStartWarps = 32;
__global__ void __launch_bounds__(kStartWarps * 32) k_embed_starts(int* counts, int* totals, int tiles, int bins) {
  constexpr int kAhead = 8;
  __shared__ int sums[kStartWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x * 32 + lane;
  const int run = (tiles + kStartWarps - 1) / kStartWarps, t0 = min(warp * run, tiles), t1 = min(t0 + run, tiles);
  const bool on = b < bins;
  int sum = 0;
#pragma unroll 8
  for (int t = t0; t < t1; ++t)
    if (on) sum += counts[(int64_t)t * bins + b];
  sums[warp][lane] = sum;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += sums[w][lane];
  if (!on) return;
  if (warp == kStartWarps - 1) totals[b] = before + sum;
  for (int t = t0; t < t1; t += kAhead) {
    int c[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (t + k < t1) c[k] = counts[(int64_t)(t + k) * bins + b];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (t + k < t1) counts[(int64_t)(t + k) * bins + b] = before, before += c[k];
  }
}

// A tile's tokens to their places: behind the smaller digits of all tiles, the same digit of the tiles before, and of
// the tokens before in the tile. The tiles' counts, of few tiles, are summed by every block; with totals they have been.
__global__ void __launch_bounds__(kThreads) k_embed_place(Sorted p, const int* keys, const int* at, int* keys_to, int* at_to,
                                                          const int* counts, const int* totals, int shift, int bits) {
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
    if (b < bins && totals)
      before[k] = counts[(int64_t)blockIdx.x * bins + b], total[k] = totals[b];
    else if (b < bins)
#pragma unroll 8
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
    to[r] = warp_rank(mine + warp * bins, key[r] >> shift & (bins - 1), bits, i < p.N);
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
  bool add, by_list;  // to what is there; the rows are found as the lists' begins, not as all of the table's
  float* parts;   // sums of the parts of long lists, one row each
  int* counters;  // per place of a part and tile of columns: parts that are done
  int64_t part_blocks;
  int tiles;      // of columns, for a part
};

// kCols accesses of E columns, `lanes` apart from column word w on, summed over a list of tokens, in their
// order (at: where the n of them stand); several rows are under way at once.
template <int E> constexpr int cols_of() { return E > 4 ? 2 : 4; }
template <class T, int E, int kCols>
MPB_D void sum_rows(const Sums& p, const int* at, int n, int64_t w, int lanes, float (&acc)[kCols][E]) {
  constexpr int kAhead = E > 4 ? 2 : 4;
  using P = Pack<T, E>;
  const int64_t words = p.D / E;
  const auto* x = reinterpret_cast<const typename P::W*>(p.dout);
  const int64_t step = p.d_sr / E;
#pragma unroll
  for (int c = 0; c < kCols; ++c)
#pragma unroll
    for (int j = 0; j < E; ++j) acc[c][j] = 0.0f;
  for (int i = 0; i < n; i += kAhead) {
    P v[kAhead][kCols];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k < n) {
        const auto* row = x + (int64_t)at[i + k] * step;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          if (w + c * lanes < words) v[k][c].w = row[w + c * lanes];
      }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k < n) {
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int j = 0; j < E; ++j) acc[c][j] += to_f(v[k][c].v[j]);
      }
  }
}

// What the table's gradient holds already, or zeros.
template <int E, bool ADD>
MPB_D void old_row(const Sums& p, int row, int64_t c, float (&old)[E]) {
  const float* from = p.table + (int64_t)row * p.D + c;
  if constexpr (E % 4 == 0) {
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      const float4 o = ADD ? *reinterpret_cast<const float4*>(from + j) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      old[j] = o.x, old[j + 1] = o.y, old[j + 2] = o.z, old[j + 3] = o.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) old[j] = ADD ? from[j] : 0.0f;
  }
}
template <int E, bool ADD>
MPB_D void put_row(const Sums& p, int row, int64_t c, const float (&old)[E], const float (&acc)[E]) {
  float* to = p.table + (int64_t)row * p.D + c;
  float v[E];
#pragma unroll
  for (int j = 0; j < E; ++j) v[j] = ADD ? old[j] + acc[j] * p.scale : acc[j] * p.scale;
  if constexpr (E % 4 == 0) {
#pragma unroll
    for (int j = 0; j < E; j += 4) *reinterpret_cast<float4*>(to + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) to[j] = v[j];
  }
}

// The end of the list of row `key` that begins at s, looked for in growing steps.
MPB_D int list_end(const Sums& p, int s, int key) {
  int64_t at = s, step = 1;  // keys[at] == key
  while (at + step < p.N && p.keys[at + step] == key) at += step, step <<= 1;
  for (; step; step >>= 1)
    if (at + step < p.N && p.keys[at + step] == key) at += step;
  return (int)at + 1;
}
// How many places behind (way 1) or before (-1) sorted place s are of the same list: by the whole block, 256
// places at a time, in growing steps where that is not the end of it.
MPB_D int list_reach(const Sums& p, int s, int key, int way) {
  auto same = [&](int64_t from, int64_t step) {
    const int64_t i = s + way * (from + step * (threadIdx.x + 1));
    return __syncthreads_count(i >= 0 && i < p.N && p.keys[i] == key);
  };
  int64_t step = 1;
  int n;
  while ((n = same(0, step)) == kThreads) step *= kThreads;
  int64_t reach = n * step;
  while (step > 1) {
    step /= kThreads;
    reach += same(reach, step) * step;
  }
  return (int)reach;
}

// Where the part that begins at sorted place i keeps its sum: a list longer than kPart begins, and one of its later parts
// begins, at most once among kPart neighbouring places.
MPB_D int64_t part_place(int i, bool begins) { return (int64_t)(i / kPart) * 2 + (begins ? 1 : 0); }

// The first blocks take the parts of long lists, one tile of columns each; the others the rows: of the whole table, or
// the lists' first tokens. `lanes` threads (a power of two, a warp at least) walk a row's columns.
template <class T, int E, bool ADD>
__global__ void __launch_bounds__(kThreads) k_embed_sums(Sums p, int lanes) {
  constexpr int kCols = cols_of<E>();
  const int64_t words = p.D / E;
  float acc[kCols][E];
  if (blockIdx.x < p.part_blocks) {
    __shared__ bool last;
    const int tile = (int)(blockIdx.x % p.tiles);
    const int64_t place = blockIdx.x / p.tiles;
    const int w0 = (int)(place >> 1) * kPart, w1 = (int)min((int64_t)w0 + kPart, p.N), n = (int)p.N;
    // a long list that begins here reaches behind these places; the list that the first place is of
    const bool begins = place & 1;
    if (begins && w1 >= n) return;
    const int key = p.keys[begins ? w1 - 1 : w0];
    if (key >= p.V || (begins && p.keys[w1] != key)) return;
    const int s = (begins ? w1 - 1 : w0) - list_reach(p, begins ? w1 - 1 : w0, key, -1);
    const int i = begins ? s : s + (w0 - s + kPart - 1) / kPart * kPart;
    if (begins ? s < w0 : i == s || i >= w1 || p.keys[i] != key) return;
    const int e = i + 1 + list_reach(p, i, key, 1);
    if (e - s <= kPart) return;
    // each warp sums four of the part's rows, so that all of them are under way at once, and the warps' sums are added
    // in their order
    constexpr int kWarps = kThreads / 32, kEach = kPart / kWarps, kValues = 32 * kCols * E;
    __shared__ int rows[kPart];
    __shared__ float sums[kWarps][kValues];
    const int have = min(e - i, kPart), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if ((int)threadIdx.x < have) rows[threadIdx.x] = p.at[i + threadIdx.x];
    __syncthreads();
    sum_rows<T, E, kCols>(p, rows + warp * kEach, min(have - warp * kEach, kEach), (int64_t)tile * 32 * kCols + lane, 32, acc);
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) sums[warp][(c * E + j) * 32 + lane] = acc[c][j];
    __syncthreads();
    auto column = [&](int v) { return (((int64_t)tile * kCols + v / 32 / E) * 32 + v % 32) * E + v / 32 % E; };
#pragma unroll
    for (int v = threadIdx.x; v < kValues; v += kThreads)
      if (column(v) < p.D) {
        float x = sums[0][v];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) x += sums[k][v];
        p.parts[place * p.D + column(v)] = x;
      }
    __threadfence();
    __syncthreads();
    const int parts = (e - s + kPart - 1) / kPart;
    if (threadIdx.x == 0) last = atomicAdd(&p.counters[part_place(s, true) / 2 * p.tiles + tile], 1) == parts - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (int v = threadIdx.x; v < kValues; v += kThreads) {
      const int64_t c = column(v);
      if (c >= p.D) continue;
      float* to = p.table + (int64_t)key * p.D + c;
      const float old = ADD ? *to : 0.0f;
      float x = 0.0f;
#pragma unroll 8
      for (int k = 0; k < parts; ++k) x += __ldcg(p.parts + part_place(s + k * kPart, k == 0) * p.D + c);
      *to = ADD ? old + x * p.scale : x * p.scale;
    }
    return;
  }
  const int64_t item = (blockIdx.x - p.part_blocks) * (kThreads / lanes) + threadIdx.x / lanes;
  int row, s, e;
  if (p.by_list) {
    if (item >= p.N) return;
    s = (int)item;
    row = p.keys[s];
    const int before = s > 0 ? p.keys[s - 1] : -1, after = s + 1 < p.N ? p.keys[s + 1] : -1;
    asm volatile("prefetch.global.L1 [%0];" ::"l"(p.at + s));
    if (row >= p.V || before == row) return;
    e = after == row ? list_end(p, s + 1, row) : s + 1;
  } else {
    if (item >= p.V) return;
    row = (int)item;
    s = p.first[row];
    e = p.end[row];
  }
  if (e - s > kPart) return;
  for (int64_t w = threadIdx.x & (lanes - 1); w < words; w += (int64_t)kCols * lanes) {
    float old[kCols][E];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (w + c * lanes < words) old_row<E, ADD>(p, row, (w + c * lanes) * E, old[c]);
    sum_rows<T, E, kCols>(p, p.at + s, e - s, w, lanes, acc);
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (w + c * lanes < words) put_row<E, ADD>(p, row, (w + c * lanes) * E, old[c], acc[c]);
  }
}

// At most kFew tokens need no sort: the block of a token that no earlier one equals looks through all of them, and sums
// what names its row. One kernel instead of two to four: 17 tokens of 69 channels: 9 us a call, 16 with the sort.
constexpr int kFew = 128;
struct Few {
  Sums s;
  const void* tokens;
  int wide;
};
template <class T, int E, bool ADD>
__global__ void __launch_bounds__(kThreads) k_embed_few(Few f) {
  constexpr int kCols = cols_of<E>();
  __shared__ int key[kFew], list[kFew], found[kFew / 32];
  const Sums& p = f.s;
  const int n = (int)(blockIdx.x / p.tiles), tile = (int)(blockIdx.x % p.tiles), tid = threadIdx.x, N = (int)p.N;
  if (tid < kFew) {
    const int64_t t = tid < N ? token_of(f.tokens, f.wide, tid) : -1;
    key[tid] = t >= 0 && t < p.V ? (int)t : -1;
  }
  __syncthreads();
  const int own = key[n];
  const bool same = tid < kFew && key[tid] == own;
  const unsigned which = __ballot_sync(0xffffffffu, same);
  if (tid < kFew && tid % 32 == 0) found[tid / 32] = __popc(which);
  if (__syncthreads_or(same && tid < n) || own < 0) return;
  int at = __popc(which & ((1u << tid % 32) - 1)), count = 0;
#pragma unroll
  for (int w = 0; w < kFew / 32; ++w) {
    if (w < tid / 32) at += found[w];
    count += found[w];
  }
  if (same) list[at] = tid;
  __syncthreads();
  const int64_t words = p.D / E, w = (int64_t)tile * kCols * kThreads + tid;
  float acc[kCols][E], old[kCols][E];
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    if (w + c * kThreads < words) old_row<E, ADD>(p, own, (w + c * kThreads) * E, old[c]);
  sum_rows<T, E, kCols>(p, list, count, w, kThreads, acc);
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    if (w + c * kThreads < words) put_row<E, ADD>(p, own, (w + c * kThreads) * E, old[c], acc[c]);
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
  size_t keys, at, keys2, at2, counts, totals, first, end, counters, parts, bytes;
  int64_t n_counters;
  Scratch(int64_t N, int64_t V, int64_t D, bool by_list) {
    const size_t n = round16((size_t)N * 4);
    const int64_t windows = (N + kPart - 1) / kPart, col_tiles = (D + 127) / 128;  // at most: a tile has 128 columns and more
    const bool small = N <= kSmall;
    keys = 0, at = n, keys2 = 2 * n, at2 = keys2 + (small ? 0 : n), counts = at2 + (small ? 0 : n);
    totals = counts + (small ? 0 : round16((size_t)((N + kTileTokens - 1) / kTileTokens) * kMostBins * 4));
    first = totals + (small ? 0 : kMostBins * 4);
    end = first + (by_list ? 0 : round16((size_t)V * 4));
    counters = end + (by_list ? 0 : round16((size_t)V * 4));
    n_counters = windows * col_tiles;
    parts = counters + round16((size_t)n_counters * 4);
    bytes = parts + (N > kPart ? (size_t)windows * 2 * D * 4 : 0);
  }
};

int sort_tokens(Sorted& p, char* scratch, const Scratch& w, cudaStream_t s) {
  if (p.N <= kSmall) {
    const unsigned blocks = (unsigned)((p.N + 31) / 32);
    const int64_t most = (p.N + 31) / 32 * 32 + 32;  // keys with what fills up the warps' runs
    if ((int64_t)(p.V + 1) * kSmall <= 0xffffffffLL) {
      if (int rc = allow_smem<k_embed_rank<uint32_t>, kSmallBytes>("embedding_backward")) return rc;
      k_embed_rank<uint32_t><<<blocks, kThreads, (size_t)most * 4, s>>>(p);
    } else {
      if (int rc = allow_smem<k_embed_rank<uint64_t>, kSmallBytes>("embedding_backward")) return rc;
      k_embed_rank<uint64_t><<<blocks, kThreads, (size_t)most * 8, s>>>(p);
    }
    if (int rc = launch_check("embedding_backward")) return rc;
    if (!p.first) return MPB_OK;
    if (int rc = cuda_check(cudaMemsetAsync(p.first, 0, w.counters - w.first, s), "embedding_backward")) return rc;
    k_embed_ends<<<(unsigned)((p.N + kThreads - 1) / kThreads), kThreads, 0, s>>>(p);
    return launch_check("embedding_backward");
  }
  const Digits g(p.V);
  int *a_keys = p.keys, *a_at = p.at, *b_keys = (int*)(scratch + w.keys2), *b_at = (int*)(scratch + w.at2);
  const unsigned tiles = (unsigned)((p.N + kTileTokens - 1) / kTileTokens);
  int *counts = (int*)(scratch + w.counts), *totals = tiles > kFewTiles ? (int*)(scratch + w.totals) : nullptr;
  if (g.passes % 2 == 0) std::swap(a_keys, b_keys), std::swap(a_at, b_at);  // the last pass writes to p.keys
  const int *from_keys = nullptr, *from_at = nullptr;
  for (int k = 0; k < g.passes; ++k) {
    k_embed_count<<<tiles, kThreads, 0, s>>>(p, from_keys, counts, k * g.bits, g.bits);
    if (totals) k_embed_starts<<<((1u << g.bits) + 31) / 32, kStartWarps * 32, 0, s>>>(counts, totals, (int)tiles, 1 << g.bits);
    k_embed_place<<<tiles, kThreads, 0, s>>>(p, from_keys, from_at, a_keys, a_at, counts, totals, k * g.bits, g.bits);
    if (int rc = launch_check("embedding_backward")) return rc;
    from_keys = a_keys, from_at = a_at;
    std::swap(a_keys, b_keys), std::swap(a_at, b_at);
  }
  if (p.first) k_embed_ends<<<(unsigned)((p.N + kThreads - 1) / kThreads), kThreads, 0, s>>>(p);
  return launch_check("embedding_backward");
}

template <class T, int E>
int launch_sums(Sums& p, cudaStream_t s) {
  constexpr int kCols = cols_of<E>();
  const int64_t words = p.D / E;
  const int lanes = lanes_for((words + kCols - 1) / kCols, 32);
  p.tiles = (int)((words + kCols * 32 - 1) / (kCols * 32));
  p.part_blocks = p.N > kPart ? (p.N + kPart - 1) / kPart * 2 * p.tiles : 0;
  const int64_t items = p.by_list ? p.N : p.V, groups = kThreads / lanes;
  const int64_t blocks = p.part_blocks + (items + groups - 1) / groups;
  if (blocks > 0x7fffffffLL) return fail(MPB_ERR_SHAPE, "embedding_backward: %lld blocks are too many for one call", (long long)blocks);
  if (p.add) k_embed_sums<T, E, true><<<(unsigned)blocks, kThreads, 0, s>>>(p, lanes);
  else k_embed_sums<T, E, false><<<(unsigned)blocks, kThreads, 0, s>>>(p, lanes);
  return launch_check("embedding_backward");
}

template <class T, int E>
int launch_few(Few& f, cudaStream_t s) {
  constexpr int kCols = cols_of<E>();
  const int64_t words = f.s.D / E, tiles = (words + kCols * kThreads - 1) / (kCols * kThreads);
  if (tiles * f.s.N > 0x7fffffffLL) return fail(MPB_ERR_SHAPE, "embedding_backward: %lld channels are too many for one call", (long long)f.s.D);
  f.s.tiles = (int)tiles;
  const unsigned grid = (unsigned)(tiles * f.s.N);
  if (f.s.add) k_embed_few<T, E, true><<<grid, kThreads, 0, s>>>(f);
  else k_embed_few<T, E, false><<<grid, kThreads, 0, s>>>(f);
  return launch_check("embedding_backward");
}

template <class T>
int launch_gradient(Sums& p, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool wide = ((uintptr_t)p.dout | (uintptr_t)p.table) % 16 == 0 && p.D % E == 0 && p.d_sr % E == 0;
  return wide ? launch_sums<T, E>(p, s) : launch_sums<T, 1>(p, s);
}
template <class T>
int launch_gradient(Few& f, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const Sums& p = f.s;
  const bool wide = ((uintptr_t)p.dout | (uintptr_t)p.table) % 16 == 0 && p.D % E == 0 && p.d_sr % E == 0;
  return wide ? launch_few<T, E>(f, s) : launch_few<T, 1>(f, s);
}

// A new table of more rows than tokens name is cleared first, and written again where tokens name it: half as many
// tokens as rows at most write half of it twice. Of more tokens each row's list is looked up and written once. Tokens for an eighth, a
// half, three quarters and all of 32000 rows of 2048 bf16: cleared 80, 122, 140 and 155 us, looked up 103, 127, 138 and
// 144; of 50257 x 768: 73, 129, 159 and 188, and 106, 148, 166 and 182.
bool by_list(int64_t N, int64_t V, bool into) { return into || N <= kFew || N <= V / 2; }

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
  return N > kFew && V > 0 && D > 0 ? Scratch(N, V, D, by_list(N, V, into != 0)).bytes : 0;
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
  const bool listed = by_list(N, V, into != 0), few = N <= kFew;
  const Scratch w(N, V, D, listed);
  const size_t need = few ? 0 : w.bytes;
  if (need > scratch_bytes || (need && !scratch))
    return fail(MPB_ERR_SCRATCH, "%s: %zu bytes of scratch, %zu needed", name, scratch_bytes, need);
  if (need && (uintptr_t)scratch % 16 != 0) return fail(MPB_ERR_INVALID, "%s: scratch not 16-byte aligned", name);
  if (listed && !into)
    if (int rc = cuda_check(cudaMemsetAsync(dtable, 0, (size_t)V * D * 4, s), name)) return rc;
  if (few) {
    Few f = {{N, D, (int)V, dout, d_sr, nullptr, nullptr, nullptr, nullptr, (float)scale, dtable, into != 0, true, nullptr, nullptr, 0, 1},
             tokens, tokens_dtype == MPB_I64};
    switch (dtype) {
      case MPB_F32: return launch_gradient<float>(f, s);
      case MPB_F16: return launch_gradient<__half>(f, s);
      default: return launch_gradient<__nv_bfloat16>(f, s);
    }
  }
  char* at = (char*)scratch;
  Sorted o = {N, (int)V, tokens, tokens_dtype == MPB_I64, (int*)(at + w.keys), (int*)(at + w.at),
              listed ? nullptr : (int*)(at + w.first), listed ? nullptr : (int*)(at + w.end), (int*)(at + w.counters), w.n_counters};
  if (int rc = sort_tokens(o, at, w, s)) return rc;
  Sums p = {N, D, (int)V, dout, d_sr, o.keys, o.at, o.first, o.end, (float)scale, dtable, into != 0, listed,
            (float*)(at + w.parts), o.counters, 0, 1};
  switch (dtype) {
    case MPB_F32: return launch_gradient<float>(p, s);
    case MPB_F16: return launch_gradient<__half>(p, s);
    default: return launch_gradient<__nv_bfloat16>(p, s);
  }
}

}  // extern "C"

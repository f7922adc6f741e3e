// Linear attention with a decay for each head. Per sequence and head, with q_t,
// k_t of DK channels, v_t of DV, log-decay g_t (no counterpart in the reference):
//
//   S_t = e^(g_t) S_(t-1) + k_t v_t'      o_t = scale S_t' q_t
//
// in chunks of 64 steps. With G the running sum of g inside a chunk, D_ij =
// e^(G_i - G_j) for j <= i and zero elsewhere, S the state before the chunk and
// U the gradient of the state behind it:
//
//   o_i  = scale (sum_j D_ij (q_i k_j) v_j + e^(G_i) S' q_i)
//   S   <- e^(G_C) S + sum_j e^(G_C - G_j) k_j v_j'
//   dq_i = scale (sum_j D_ij (do_i v_j) k_j + e^(G_i) S do_i)
//   dk_j = scale sum_i D_ij (do_i v_j) q_i + e^(G_C - G_j) U v_j
//   dv_j = scale sum_i D_ij (q_i k_j) do_i + e^(G_C - G_j) U' k_j
//   U   <- e^(G_C) U + scale sum_i e^(G_i) q_i do_i'
//   dg_t = sum_(j<t<=i) M_ij + sum_(i>=t) a_i + sum_(j<t) b_j + e^(G_C) <U, S>
//
// with M = scale D (q k') (do v') and a_i = q_i dq_i, b_j = k_j dk_j of the terms
// with S and U: what passes through step t. Only that is added, nothing is taken away again, so that a strong decay's
// gradient, as small as the decay, is right to float precision among large ones (row sums less column sums of M lost it whole
// from log-decays of -16 on).
//
// Products run on the tensor cores with operands of bf16 and sums in float. A
// bf16 input is one such operand; a float16 input is the sum of two, a float of three,
// and so is what a float weight makes of an input. Scores and states that reach a 16-bit result alone are two
// (16 bits: the result's own rounding is what remains). Products of pieces whose
// place together is past the result's precision are left out.
//
// This file has the kernels of any type, layout and width up to 256: the states at the
// chunks' borders (k_la_states, over segments that k_la_join joins), from which
// all chunks' outputs (k_la_output) and gradients (k_la_gradients) follow side by side; the step;
// and the gradients of bf16 heads of up to 128 channels (k_la_gradients_wide). bf16 rows of 16-byte words are walked by
// linear_attention_walk.cu, without storing states going forward.
//
// Bound: forward and backward move 0.5 GB each way at most for what takes them hundreds of us; they wait on their own
// tiles (synchronous loads, two barriers a tile, splits into pieces), at 8 warps per SM: gradients of 4 x 4096 x 16 heads of 128 bf16
// 726 us (1.3 TB/s under the profiler, tensor cores 0.25), 1 x 19250 x 3 heads of 128 and 64 float, all of the backward pass, 733 us.
// The step is bound by memory: 64 x 16 heads of 128 x 128, 134 MB, 24.6 us (5.5 TB/s).
#include "common.cuh"
#include "internal.h"
#include "linear_attention.cuh"
#include "musapy_b200.h"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kThreads = 128;
constexpr int kPlane = kChunk * kPitch;

using bf16 = __nv_bfloat16;

template <class T> struct RawPieces;
template <> struct RawPieces<bf16> { static constexpr int n = 1; };
template <> struct RawPieces<__half> { static constexpr int n = 2; };
template <> struct RawPieces<float> { static constexpr int n = 3; };

// What a product that only reaches a result of type T has to keep: the scores' pieces (P), the states' (S).
// 16-bit types: 16 bits of both, so that the result is off by its own rounding (with scores of 8 bits a bf16 result
// was off by 2.35e-3 of its norm, where its rounding is 1.66e-3). float: 24.
template <class T> struct Keep;
template <> struct Keep<bf16> { static constexpr int P = 2, S = 2; };
template <> struct Keep<__half> { static constexpr int P = 2, S = 2; };
template <> struct Keep<float> { static constexpr int P = 3, S = 3; };
constexpr int kExact = 3;  // 24 bits: what reaches a result of 32 bits

// ------------------------------------------------------------ tiles
// x as the sum of N bf16 numbers, each the rounding of what is left.
template <int N>
MPB_D void split(float x, bf16 (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = __float2bfloat16_rn(x);
    x -= __bfloat162float(p[i]);
  }
}

// Eight neighbouring elements of a row as floats, zero from `have` on.
template <class T>
MPB_D void load8(const T* src, int have, bool wide, float (&x)[8]) {
  if (wide && have >= 8) {
    constexpr int W = (int)sizeof(T) / 2, E = 16 / (int)sizeof(T);
    union { uint4 w[W]; T v[W * E]; } u;
#pragma unroll
    for (int i = 0; i < W; ++i) u.w[i] = *(reinterpret_cast<const uint4*>(src) + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f(u.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < have ? to_f(src[i]) : 0.0f;
  }
}

template <int N>
MPB_D void store8(bf16* dst, const float (&x)[8]) {
  union { uint4 w; bf16 v[8]; } u[N];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bf16 p[N];
    split<N>(x[i], p);
#pragma unroll
    for (int n = 0; n < N; ++n) u[n].v[i] = p[n];
  }
#pragma unroll
  for (int n = 0; n < N; ++n) *reinterpret_cast<uint4*>(dst + n * kPlane) = u[n].w;
}

// A tile of 64 steps and 64 channels in N planes; steps from `rows` on and channels from `cols` on are zero.
// With weights each step is multiplied by its own; a weight of zero leaves it out whatever it holds.
template <class T, int N, bool WEIGHTED>
MPB_D void load_tile(bf16* dst, const T* src, int64_t step, int rows, int cols, bool wide, const float* w) {
#pragma unroll
  for (int k = 0; k < kChunk * kTile / 8 / kThreads; ++k) {
    const int at = threadIdx.x + k * kThreads, r = at >> 3, c = (at & 7) * 8;
    float x[8];
    const float by = WEIGHTED ? w[r] : 1.0f;
    load8(src + r * step + c, r < rows && by != 0.0f ? cols - c : 0, wide, x);
    if (WEIGHTED) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= by;
    }
    store8<N>(dst + r * kPitch + c, x);
  }
}

// Where a state of a chunk comes from: what its segment has summed up, and the state before the segment times the
// decay since.
struct StateTile {
  const float *own, *start;  // start == nullptr: nothing before
  float since;
  MPB_D float4 get(int64_t at) const {
    float4 a = *reinterpret_cast<const float4*>(own + at);
    if (start && since != 0.0f) {
      const float4 b = *reinterpret_cast<const float4*>(start + at);
      a.x = fmaf(since, b.x, a.x), a.y = fmaf(since, b.y, a.y), a.z = fmaf(since, b.z, a.z), a.w = fmaf(since, b.w, a.w);
    }
    return a;
  }
};

// 64 x 64 of a state (pitch `dvp`, a multiple of 16) in N planes, zero outside.
template <int N, class F>
MPB_D void load_state(bf16* dst, const StateTile& s, int64_t at, int dvp, int rows, int cols, F each) {
#pragma unroll
  for (int k = 0; k < kChunk * kTile / 8 / kThreads; ++k) {
    const int i = threadIdx.x + k * kThreads, r = i >> 3, c = (i & 7) * 8;
    float x[8] = {};
    if (r < rows && c < cols) {
      const float4 a = s.get(at + (int64_t)r * dvp + c), b = s.get(at + (int64_t)r * dvp + c + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
    each(k, x);
    store8<N>(dst + r * kPitch + c, x);
  }
}

// ----------------------------------------------------------- products
// acc (16 x 8 NT of a warp) += A B over 64: A's rows from `m`, B's columns from `n0`. TA: A lies with its rows as columns,
// TB: B lies with the summed index as rows. Pieces pa, pb with pa + pb < L take part.
template <int NT, bool TA, bool TB, int PA, int PB, int L>
MPB_D void multiply(float (&acc)[NT][4], const bf16* A, int m, const bf16* B, int n0 = 0) {
  const int lane = threadIdx.x & 31, r = lane & 7, lo = (lane >> 3 & 1) * 8, hi = (lane >> 4) * 8;
  const uint32_t a_at = smem_addr(A) + 2 * (TA ? (hi + r) * kPitch + m + lo : (m + lo + r) * kPitch + hi);
  const uint32_t b_at = smem_addr(B) + 2 * (TB ? (lo + r) * kPitch + hi + n0 : (hi + r + n0) * kPitch + lo);
  if constexpr (PA > 1 && PB > 1) {
    // The tensor core cuts a sum where others round: the small products come first, of all steps, only the large ones meet
    // the sum at its size, and what is summed already is added outside. (Errors of float inputs: 1.2e-6 with the pieces of
    // each step together, 6e-7 in this order, 3e-7 with the sum added outside.)
    float sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[n][i] = 0.0f;
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int p = 0; p < PA; ++p) {
          const int q = l - p;
          if (q < 0 || q >= PB) continue;
          uint32_t a[4];
          ldmatrix4<TA>(a, a_at + 2 * (p * kPlane + (TA ? 16 * k * kPitch : 16 * k)));
#pragma unroll
          for (int n = 0; n < NT / 2; ++n) {
            uint32_t b[4];
            ldmatrix4<TB>(b, b_at + 2 * (q * kPlane + (TB ? 16 * k * kPitch + 16 * n : 16 * n * kPitch + 16 * k)));
            mma_bf16(sum[2 * n], a, b[0], b[1]);
            mma_bf16(sum[2 * n + 1], a, b[2], b[3]);
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] += sum[n][i];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t a[PA][4];
#pragma unroll
      for (int p = 0; p < PA; ++p) ldmatrix4<TA>(a[p], a_at + 2 * (p * kPlane + (TA ? 16 * k * kPitch : 16 * k)));
#pragma unroll
      for (int n = 0; n < NT / 2; ++n) {
#pragma unroll
        for (int q = 0; q < PB; ++q) {
          uint32_t b[4];
          ldmatrix4<TB>(b, b_at + 2 * (q * kPlane + (TB ? 16 * k * kPitch + 16 * n : 16 * n * kPitch + 16 * k)));
#pragma unroll
          for (int p = 0; p < PA; ++p)
            if (p + q < L) {
              mma_bf16(acc[2 * n], a[p], b[0], b[1]);
              mma_bf16(acc[2 * n + 1], a[p], b[2], b[3]);
            }
        }
      }
    }
  }
}

template <int NT>
MPB_D void clear(float (&acc)[NT][4]) {
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
}

// f(row, col, values of the row's two neighbouring columns) for what a thread holds of its warp's 16 x 64.
template <class F>
MPB_D void each_pair(float (&acc)[8][4], F f) {
  const int lane = threadIdx.x & 31, row = (threadIdx.x >> 5) * 16 + (lane >> 2), col = (lane & 3) * 2;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    f(row, n * 8 + col, acc[n][0], acc[n][1]);
    f(row + 8, n * 8 + col, acc[n][2], acc[n][3]);
  }
}

template <int N>
MPB_D void store_pair(bf16* dst, int row, int col, float x, float y) {
  bf16 a[N], b[N];
  split<N>(x, a);
  split<N>(y, b);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const __nv_bfloat162 v(a[n], b[n]);
    *reinterpret_cast<__nv_bfloat162*>(dst + n * kPlane + row * kPitch + col) = v;
  }
}

// Writes a warp's 16 x 64 of a result (row pitch `step`), rows and columns inside only.
template <class O>
MPB_D void write_tile(O* dst, int64_t step, int rows, int cols, float (&acc)[8][4]) {
  const bool pairs = ((uintptr_t)dst / sizeof(O) | (uintptr_t)step) % 2 == 0;
  each_pair(acc, [&](int r, int c, float x, float y) {
    if (r >= rows) return;
    O* p = dst + r * step + c;
    if (pairs && c + 1 < cols) {
      *reinterpret_cast<typename Word<2 * sizeof(O)>::type*>(p) = pack<O>(make_float2(x, y)).w;
    } else {
      if (c < cols) p[0] = Cvt<O>::from(x);
      if (c + 1 < cols) p[1] = Cvt<O>::from(y);
    }
  });
}

// ------------------------------------------------------------- states
// The states at the chunks' borders: before each chunk (REV: behind each, of the gradient), as sums over the chunk's
// segment alone; `first` is what the first segment begins with. One block has 64 x 64 of a head's state in registers
// and walks a segment's chunks. since: the decay from the segment's begin to each chunk, ends: the segments' sums.
struct States {
  Shape d;
  Input x, y;  // k and v, or q and do
  Decay g;
  const float* first;
  float scale;
  float *at, *since, *ends, *last;  // last: the final state, where one segment gives it
  int* status = nullptr;            // cleared: nothing here waits
};

template <class T, bool REV>
__global__ void __launch_bounds__(kThreads) k_la_states(States p) {
  extern __shared__ __align__(16) bf16 tiles[];
  constexpr int PT = RawPieces<T>::n;
  __shared__ ChunkDecay cd;
  bf16 *A = tiles, *Bt = tiles + kExact * kPlane;
  const Shape& d = p.d;
  const int tk = (d.dkp + kTile - 1) / kTile, tv = (d.dvp + kTile - 1) / kTile;
  int64_t i = blockIdx.x;
  const int iv = (int)(i % tv);
  i /= tv;
  const int ik = (int)(i % tk);
  i /= tk;
  const int seg = (int)(i % d.segments);
  const int64_t bh = i / d.segments;
  const int h = (int)(bh % d.H);
  const int64_t b = bh / d.H;
  const int c0 = seg * d.per, c1 = min(d.chunks, c0 + d.per);
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.status = MPB_OK;
  const bool begins = REV ? c1 == d.chunks : seg == 0;
  const int64_t tile = (int64_t)ik * kTile * d.dvp + iv * kTile;
  const int rows = d.dkp - ik * kTile, cols = d.dvp - iv * kTile;
  const int64_t size = (int64_t)d.dkp * d.dvp;

  float S[8][4];
  clear(S);
  if (begins && p.first) {
    const float* f = p.first + bh * d.DK * d.DV;
    const int r0 = ik * kTile, q0 = iv * kTile;
    each_pair(S, [&](int r, int c, float& x, float& y) {
      if (r0 + r < d.DK) {
        if (q0 + c < d.DV) x = f[(int64_t)(r0 + r) * d.DV + q0 + c];
        if (q0 + c + 1 < d.DV) y = f[(int64_t)(r0 + r) * d.DV + q0 + c + 1];
      }
    });
  }
  float since = 1.0f;
  auto put = [&](float* to) {
    each_pair(S, [&](int r, int c, float x, float y) {
      if (r < rows && c < cols) *reinterpret_cast<float2*>(to + tile + (int64_t)r * d.dvp + c) = make_float2(x, y);
    });
  };
  for (int n = 0; n < c1 - c0; ++n) {
    const int c = REV ? c1 - 1 - n : c0 + n;
    const int64_t t0 = (int64_t)c * kChunk;
    const int steps = (int)min((int64_t)kChunk, d.T - t0);
    if (threadIdx.x < 32) cd.fill(p.g.p + b * p.g.sb + t0 * p.g.st + h * p.g.sh, p.g.st, steps);
    if (p.at) put(p.at + (bh * d.chunks + c) * size);
    if (ik == 0 && iv == 0 && threadIdx.x == 0) p.since[bh * d.chunks + c] = since;
    __syncthreads();
    // the first operand carries the decays: k to the chunk's end, q from its start
    const float by = REV ? p.scale : 1.0f;
    if (threadIdx.x < kChunk) cd.weight[threadIdx.x] = by * (REV ? cd.into[threadIdx.x] : cd.rest[threadIdx.x]);
    __syncthreads();
    load_tile<T, kExact, true>(A, p.x.at<T>(b, t0, h / d.share) + ik * kTile, p.x.st, steps, d.DK - ik * kTile, p.x.wide,
                               cd.weight);
    load_tile<T, PT, false>(Bt, p.y.at<T>(b, t0, h) + iv * kTile, p.y.st, steps, d.DV - iv * kTile, p.y.wide, nullptr);
    __syncthreads();
    float E[8][4];
    clear(E);
    multiply<8, true, true, kExact, PT, kExact>(E, A, (threadIdx.x >> 5) * 16, Bt);
    const float all = cd.all;
    if (all == 0.0f) {  // a state that is dropped may hold anything
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) S[k][j] = E[k][j];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) S[k][j] = fmaf(all, S[k][j], E[k][j]);
    }
    since = all == 0.0f ? 0.0f : since * all;  // one that overflowed is dropped too
    __syncthreads();
  }
  if (d.segments > 1) {
    put(p.ends + (bh * d.segments + seg) * size);
    if (ik == 0 && iv == 0 && threadIdx.x == 0) p.since[(bh + d.B * d.H) * d.chunks + seg] = since;
  } else if (p.last) {
    float* to = p.last + bh * d.DK * d.DV;
    const int r0 = ik * kTile, q0 = iv * kTile;
    each_pair(S, [&](int r, int c, float x, float y) {
      if (r0 + r < d.DK) {
        if (q0 + c < d.DV) to[(int64_t)(r0 + r) * d.DV + q0 + c] = x;
        if (q0 + c + 1 < d.DV) to[(int64_t)(r0 + r) * d.DV + q0 + c + 1] = y;
      }
    });
  }
}

// The segments' sums become the states before them, in place; the last one goes to `last`. A thread has four neighbouring
// elements of one head's state, loads the sums of eight segments at once and then runs through them.
constexpr int kJoinAhead = 8;
template <bool REV>
__global__ void __launch_bounds__(128) k_la_join(States p) {
  const Shape& d = p.d;
  const int size = d.dkp * d.dvp, i = (blockIdx.x * 128 + threadIdx.x) * 4;
  if (i >= size) return;
  const int r = i / d.dvp, c = i % d.dvp;
  for (int64_t bh = blockIdx.y; bh < d.B * d.H; bh += gridDim.y) {
    const float* decay = p.since + (bh + d.B * d.H) * d.chunks;
    float4* ends = reinterpret_cast<float4*>(p.ends + bh * d.segments * size + i);
    auto seg = [&](int n) { return REV ? d.segments - 1 - n : n; };
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int n0 = 0; n0 < d.segments; n0 += kJoinAhead) {
      float4 own[kJoinAhead];
      float a[kJoinAhead];
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k)
        if (n0 + k < d.segments) own[k] = ends[(int64_t)seg(n0 + k) * (size / 4)], a[k] = decay[seg(n0 + k)];
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k)
        if (n0 + k < d.segments) {
          ends[(int64_t)seg(n0 + k) * (size / 4)] = s;
          if (n0 + k > 0 && a[k] != 0.0f) {
            own[k].x = fmaf(a[k], s.x, own[k].x), own[k].y = fmaf(a[k], s.y, own[k].y);
            own[k].z = fmaf(a[k], s.z, own[k].z), own[k].w = fmaf(a[k], s.w, own[k].w);
          }
          s = own[k];
        }
    }
    if (p.last && r < d.DK) {
      float* to = p.last + bh * d.DK * d.DV + (int64_t)r * d.DV + c;
      if (c < d.DV) to[0] = s.x;
      if (c + 1 < d.DV) to[1] = s.y;
      if (c + 2 < d.DV) to[2] = s.z;
      if (c + 3 < d.DV) to[3] = s.w;
    }
  }
}

struct StateSet {
  const float *at, *since, *ends;
  MPB_D StateTile of(const Shape& d, int64_t bh, int c, bool rev) const {
    const int64_t size = (int64_t)d.dkp * d.dvp;
    const int seg = c / d.per;
    const bool begins = rev ? seg == d.segments - 1 : seg == 0;
    return {at + (bh * d.chunks + c) * size, begins ? nullptr : ends + (bh * d.segments + seg) * size,
            since[bh * d.chunks + c]};
  }
};

// ------------------------------------------------------------ outputs
struct Outputs {
  Shape d;
  Input q, k, v;
  Decay g;
  float scale;
  StateSet s;
  void* o;
};

// One block: 64 channels of v for one chunk of a head.
template <class T>
__global__ void __launch_bounds__(kThreads) k_la_output(Outputs p) {
  extern __shared__ __align__(16) bf16 tiles[];
  constexpr int PT = RawPieces<T>::n, PP = Keep<T>::P, PS = Keep<T>::S;
  __shared__ ChunkDecay cd;
  bf16 *X = tiles, *Y = X + PT * kPlane, *Z = Y + PT * kPlane;
  const Shape& d = p.d;
  const int tk = (d.dkp + kTile - 1) / kTile, tv = (d.dvp + kTile - 1) / kTile;
  int64_t i = blockIdx.x;
  const int iv = (int)(i % tv);
  i /= tv;
  const int c = (int)(i % d.chunks);
  const int64_t bh = i / d.chunks;
  const int h = (int)(bh % d.H), m = (threadIdx.x >> 5) * 16;
  const int64_t b = bh / d.H, t0 = (int64_t)c * kChunk;
  const int steps = (int)min((int64_t)kChunk, d.T - t0);
  if (threadIdx.x < 32) cd.fill(p.g.p + b * p.g.sb + t0 * p.g.st + h * p.g.sh, p.g.st, steps);
  const StateTile s = p.s.of(d, bh, c, false);
  float P[8][4], O[8][4];
  clear(P);
  clear(O);
  for (int ik = 0; ik < tk; ++ik) {
    const int k0 = ik * kTile;
    load_tile<T, PT, false>(X, p.q.at<T>(b, t0, h / d.share) + k0, p.q.st, steps, d.DK - k0, p.q.wide, nullptr);
    load_tile<T, PT, false>(Y, p.k.at<T>(b, t0, h / d.share) + k0, p.k.st, steps, d.DK - k0, p.k.wide, nullptr);
    load_state<PS>(Z, s, (int64_t)k0 * d.dvp + iv * kTile, d.dvp, d.dkp - k0, d.dvp - iv * kTile, [](int, float (&)[8]) {});
    __syncthreads();
    multiply<8, false, false, PT, PT, kExact>(P, X, m, Y);
    multiply<8, false, true, PT, PS, PS>(O, X, m, Z);
    __syncthreads();
  }
  each_pair(O, [&](int r, int, float& x, float& y) {
    const float by = cd.into[r] * p.scale;
    x = by != 0.0f ? x * by : 0.0f;
    y = by != 0.0f ? y * by : 0.0f;
  });
  // the scores of a warp's rows go where q was: rows of its own, read by it alone
  bf16* S = X;
  static_assert(PP <= 2 * PT, "the scores' planes fit those of q and k");
  each_pair(P, [&](int r, int j, float x, float y) {
    store_pair<PP>(S, r, j, cd.pair(r, j) * x * p.scale, cd.pair(r, j + 1) * y * p.scale);
  });
  load_tile<T, PT, false>(Z, p.v.at<T>(b, t0, h) + iv * kTile, p.v.st, steps, d.DV - iv * kTile, p.v.wide, nullptr);
  __syncthreads();
  multiply<8, false, true, PP, PT, PP>(O, S, m, Z);
  write_tile((T*)p.o + ((b * d.T + t0) * d.H + h) * d.DV + iv * kTile, (int64_t)d.H * d.DV, steps, d.DV - iv * kTile, O);
}

// ---------------------------------------------------------- gradients
struct Gradients {
  Shape d;
  Input q, k, v, g_o;
  Decay g;
  float scale;
  StateSet s, u;
  void *dq, *dk;  // (B, T, H, DK) floats where heads share, else results
  void* dv;
  float *dg, *dg_chunk;  // per step, or the sums of chunks
};

// Sums of M (a chunk's pairs of steps) over the columns before column t, for a warp's rows from t on: what each pair of
// steps passes through step t. each_row takes the next 8 columns of a thread's row, of which it has the two at t; before: the sum of
// the columns before those.
struct Passing {
  float at[2] = {0.0f, 0.0f};
  MPB_D void each_row(int row, int t, float m0, float m1, float& before) {
    const int l = threadIdx.x & 3;
    float run = m0 + m1;
    float x = __shfl_up_sync(0xffffffffu, run, 1, 4);
    if (l >= 1) run += x;
    x = __shfl_up_sync(0xffffffffu, run, 2, 4);
    if (l >= 2) run += x;
    x = __shfl_up_sync(0xffffffffu, run, 1, 4);
    const float first = before + (l ? x : 0.0f);
    before += __shfl_sync(0xffffffffu, run, 3, 4);
    if (row >= t) at[0] += first;
    if (row >= t + 1) at[1] += first + m0;
  }
  // over the warp's rows; in every thread
  MPB_D void join() {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      for (int o = 4; o < 32; o <<= 1) at[e] += __shfl_xor_sync(0xffffffffu, at[e], o);
  }
};

// The decays' gradients of a chunk, by one warp: each lane has two steps. near: what the chunk's pairs pass through them; `back`
// counts for the steps up to it and `fore` for those behind; `through` is <U, S>.
MPB_D void write_decay(const Gradients& p, const ChunkDecay& cd, int64_t b, int h, int c, int steps, const float (&near)[2],
                       const float (&back)[2], const float (&fore)[2], float through) {
  const int lane = threadIdx.x & 31, t = 2 * lane;
  float after = back[0] + back[1], before = fore[0] + fore[1];
  for (int o = 1; o < 32; o <<= 1) {
    const float x = __shfl_down_sync(0xffffffffu, after, o), y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane + o < 32) after += x;
    if (lane >= o) before += y;
  }
  // without its own: the neighbour's, not a difference
  after = __shfl_down_sync(0xffffffffu, after, 1);
  before = __shfl_up_sync(0xffffffffu, before, 1);
  if (lane == 31) after = 0.0f;
  if (lane == 0) before = 0.0f;
  const float all_pass = cd.all != 0.0f ? cd.all * through : 0.0f;
  float out[2] = {near[0] + (after + back[1] + back[0]) + before + all_pass, near[1] + (after + back[1]) + (before + fore[0]) + all_pass};
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (cd.resets(t + e)) out[e] = 0.0f;
    if (t + e < steps) {
      if (p.dg) p.dg[(b * p.d.T + (int64_t)c * kChunk + t + e) * p.d.H + h] = out[e];
      sum += out[e];
    }
  }
  sum = warp_sum(sum);
  if (p.dg_chunk && lane == 0) p.dg_chunk[(b * p.d.chunks + c) * p.d.H + h] = sum;
}

template <class T, class O>
__global__ void __launch_bounds__(kThreads) k_la_gradients(Gradients p) {
  extern __shared__ __align__(16) bf16 tiles[];
  constexpr int PT = RawPieces<T>::n, PP = Keep<T>::P, PS = Keep<T>::S;
  __shared__ ChunkDecay cd;
  __shared__ float passing[4][kChunk], far_q[kChunk], far_k[kChunk], through[4];
  bf16 *X = tiles, *Y = X + PT * kPlane, *Z = Y + PT * kPlane, *W = Z + kExact * kPlane;
  // the scores are used before U comes to W in three planes, those of the gradients beside it
  bf16 *Pt = W, *Rt = W + kExact * kPlane;
  static_assert(PP <= kExact, "the scores' planes fit those of U");
  const Shape& d = p.d;
  const int tk = (d.dkp + kTile - 1) / kTile, tv = (d.dvp + kTile - 1) / kTile;
  const int c = (int)(blockIdx.x % d.chunks), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = warp * 16;
  const int64_t bh = blockIdx.x / d.chunks;
  const int h = (int)(bh % d.H), hq = h / d.share;
  const int64_t b = bh / d.H, t0 = (int64_t)c * kChunk;
  const int steps = (int)min((int64_t)kChunk, d.T - t0);
  if (threadIdx.x < 32) cd.fill(p.g.p + b * p.g.sb + t0 * p.g.st + h * p.g.sh, p.g.st, steps);
  const StateTile s = p.s.of(d, bh, c, false), u = p.u.of(d, bh, c, true);
  auto load = [&](bf16* to, const Input& x, int head, int first, int all) {
    load_tile<T, PT, false>(to, x.at<T>(b, t0, head) + first, x.st, steps, all - first, x.wide, nullptr);
  };
  // the scores, and those of the gradients
  float P[8][4], R[8][4];
  clear(P);
  clear(R);
  for (int ik = 0; ik < tk; ++ik) {
    load(X, p.q, hq, ik * kTile, d.DK);
    load(Y, p.k, hq, ik * kTile, d.DK);
    __syncthreads();
    multiply<8, false, false, PT, PT, kExact>(P, X, m, Y);
    __syncthreads();
  }
  for (int iv = 0; iv < tv; ++iv) {
    load(X, p.g_o, h, iv * kTile, d.DV);
    load(Y, p.v, h, iv * kTile, d.DV);
    __syncthreads();
    multiply<8, false, false, PT, PT, kExact>(R, X, m, Y);
    __syncthreads();
  }
  {
    float before[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      Passing pass;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int r = m + (lane >> 2) + 8 * a, j = n * 8 + (lane & 3) * 2;
        float pr[2], rr[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float by = cd.pair(r, j + e) * p.scale;
          pr[e] = by * P[n][2 * a + e];
          rr[e] = by * R[n][2 * a + e];
        }
        pass.each_row(r, j, pr[0] * R[n][2 * a], pr[1] * R[n][2 * a + 1], before[a]);
        store_pair<PP>(Pt, r, j, pr[0], pr[1]);
        store_pair<PP>(Rt, r, j, rr[0], rr[1]);
      }
      pass.join();
      if (lane < 4) passing[warp][n * 8 + lane * 2] = pass.at[0], passing[warp][n * 8 + lane * 2 + 1] = pass.at[1];
    }
  }
  auto weigh = [&](float (&acc)[8][4], const float* w, float by) {
    each_pair(acc, [&](int r, int, float& x, float& y) {
      const float f = w[r] * by;
      x = f != 0.0f ? x * f : 0.0f;
      y = f != 0.0f ? y * f : 0.0f;
    });
  };
  // dv
  for (int iv = 0; iv < tv; ++iv) {
    float acc[8][4];
    clear(acc);
    for (int ik = 0; ik < tk; ++ik) {
      __syncthreads();
      load(Y, p.k, hq, ik * kTile, d.DK);
      load_state<PS>(Z, u, (int64_t)ik * kTile * d.dvp + iv * kTile, d.dvp, d.dkp - ik * kTile, d.dvp - iv * kTile,
                     [](int, float (&)[8]) {});
      __syncthreads();
      multiply<8, false, true, PT, PS, PS>(acc, Y, m, Z);
    }
    weigh(acc, cd.rest, 1.0f);
    load(X, p.g_o, h, iv * kTile, d.DV);
    __syncthreads();
    multiply<8, true, true, PP, PT, PP>(acc, Pt, m, X);
    write_tile((T*)p.dv + ((b * d.T + t0) * d.H + h) * d.DV + iv * kTile, (int64_t)d.H * d.DV, steps, d.DV - iv * kTile, acc);
    __syncthreads();
  }
  // dq and dk
  float fq[2] = {0.0f, 0.0f}, fk[2] = {0.0f, 0.0f}, pass = 0.0f;
  for (int ik = 0; ik < tk; ++ik) {
    float aq[8][4], ak[8][4];
    clear(aq);
    clear(ak);
    for (int iv = 0; iv < tv; ++iv) {
      __syncthreads();
      load(X, p.g_o, h, iv * kTile, d.DV);
      load(Y, p.v, h, iv * kTile, d.DV);
      float held[4][8];
      const int64_t at = (int64_t)ik * kTile * d.dvp + iv * kTile;
      load_state<kExact>(Z, s, at, d.dvp, d.dkp - ik * kTile, d.dvp - iv * kTile, [&](int k, float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) held[k][e] = x[e];
      });
      load_state<kExact>(W, u, at, d.dvp, d.dkp - ik * kTile, d.dvp - iv * kTile, [&](int k, float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) pass = fmaf(held[k][e], x[e], pass);
      });
      __syncthreads();
      multiply<8, false, false, PT, kExact, kExact>(aq, X, m, Z);
      multiply<8, false, false, PT, kExact, kExact>(ak, Y, m, W);
    }
    weigh(aq, cd.into, p.scale);
    weigh(ak, cd.rest, 1.0f);
    __syncthreads();
    load(X, p.q, hq, ik * kTile, d.DK);
    load(Y, p.k, hq, ik * kTile, d.DK);
    __syncthreads();
    auto dot = [&](float (&acc)[8][4], const bf16* x, float (&sum)[2]) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const bf16* at = x + (m + (lane >> 2) + 8 * a) * kPitch + n * 8 + (lane & 3) * 2;
          float v0 = 0.0f, v1 = 0.0f;
#pragma unroll
          for (int q = PT - 1; q >= 0; --q) {
            v0 += __bfloat162float(at[q * kPlane]);
            v1 += __bfloat162float(at[q * kPlane + 1]);
          }
          sum[a] = fmaf(v0, acc[n][2 * a], sum[a]);
          sum[a] = fmaf(v1, acc[n][2 * a + 1], sum[a]);
        }
    };
    dot(aq, X, fq);
    dot(ak, Y, fk);
    multiply<8, false, true, PP, PT, PP>(aq, Rt, m, Y);
    multiply<8, true, true, PP, PT, PP>(ak, Rt, m, X);
    const int64_t to = ((b * d.T + t0) * d.H + h) * d.DK + ik * kTile;
    write_tile((O*)p.dq + to, (int64_t)d.H * d.DK, steps, d.DK - ik * kTile, aq);
    write_tile((O*)p.dk + to, (int64_t)d.H * d.DK, steps, d.DK - ik * kTile, ak);
  }
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    for (int o = 1; o < 4; o <<= 1) {
      fq[a] += __shfl_xor_sync(0xffffffffu, fq[a], o);
      fk[a] += __shfl_xor_sync(0xffffffffu, fk[a], o);
    }
    if ((lane & 3) == 0) {
      far_q[m + (lane >> 2) + 8 * a] = fq[a];
      far_k[m + (lane >> 2) + 8 * a] = fk[a];
    }
  }
  pass = warp_sum(pass);
  if (lane == 0) through[warp] = pass;
  __syncthreads();
  if (warp != 0) return;
  float near[2], back[2], fore[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int t = 2 * lane + e;
    near[e] = (passing[0][t] + passing[1][t]) + (passing[2][t] + passing[3][t]);
    back[e] = far_q[t];
    fore[e] = far_k[t];
  }
  write_decay(p, cd, b, h, c, steps, near, back, fore, (through[0] + through[1]) + (through[2] + through[3]));
}

// The same for bf16 heads of up to 64 NK and 64 NV channels: all of the chunk's q, k, v and do stay in shared memory,
// copied there at once, and the two states pass through it once, a tile of 64 x 64 at a time, the next one on its way to registers
// meanwhile. Eight warps: 16 rows and half of a tile's columns each. 4 x 4096 x 16 heads of 128: 726 us, where the kernel above, which
// loads a tile whenever it needs one, takes 1313.
constexpr int kWideThreads = 256;

// A tile of 64 x 64 by asynchronous copies, zeros outside.
MPB_D void copy_tile(bf16* dst, const bf16* src, int64_t step, int rows, int cols) {
#pragma unroll
  for (int k = 0; k < kChunk * kTile / 8 / kWideThreads; ++k) {
    const int at = threadIdx.x + k * kWideThreads, r = at >> 3, c = (at & 7) * 8;
    const int have = r < rows ? min(max(cols - c, 0), 8) * 2 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst + r * kPitch + c)),
                 "l"(have ? src + r * step + c : src), "r"(have)
                 : "memory");
  }
}

template <int NK, int NV, class O>
__global__ void __launch_bounds__(kWideThreads, 1) k_la_gradients_wide(Gradients p) {
  extern __shared__ __align__(16) bf16 tiles[];
  __shared__ ChunkDecay cd;
  __shared__ float rows_m[kChunk], passing[4][kChunk], far_q[2][kChunk], far_k[2][kChunk], through[8];
  bf16 *Q = tiles, *K = Q + NK * kPlane, *V = K + NK * kPlane, *G = V + NV * kPlane, *Z = G + NV * kPlane, *W = Z + kExact * kPlane;
  constexpr int PP = Keep<bf16>::P;
  bf16 *Pt = W + kExact * kPlane, *Rt = Pt + PP * kPlane;
  const Shape& d = p.d;
  const int c = (int)(blockIdx.x % d.chunks), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int m = (warp & 3) * 16, side = warp >> 2, n0 = side * 32;
  const int64_t bh = blockIdx.x / d.chunks;
  const int h = (int)(bh % d.H), hq = h / d.share;
  const int64_t b = bh / d.H, t0 = (int64_t)c * kChunk;
  const int steps = (int)min((int64_t)kChunk, d.T - t0);
  for (int i = 0; i < NK; ++i) {
    copy_tile(Q + i * kPlane, p.q.at<bf16>(b, t0, hq) + i * kTile, p.q.st, steps, d.DK - i * kTile);
    copy_tile(K + i * kPlane, p.k.at<bf16>(b, t0, hq) + i * kTile, p.k.st, steps, d.DK - i * kTile);
  }
  for (int i = 0; i < NV; ++i) {
    copy_tile(V + i * kPlane, p.v.at<bf16>(b, t0, h) + i * kTile, p.v.st, steps, d.DV - i * kTile);
    copy_tile(G + i * kPlane, p.g_o.at<bf16>(b, t0, h) + i * kTile, p.g_o.st, steps, d.DV - i * kTile);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  // the states: a thread has 8 neighbouring columns of rows r and r + 32 of a tile
  const StateTile s = p.s.of(d, bh, c, false), u = p.u.of(d, bh, c, true);
  const int sr = threadIdx.x >> 3, sc = (threadIdx.x & 7) * 8;
  float xs[2][8], xu[2][8];
  auto fetch = [&](int tile) {
    const int ik = tile / NV, iv = tile % NV;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = ik * kTile + sr + 32 * k, col = iv * kTile + sc;
      const bool in = r < d.dkp && col < d.dvp;
      const int64_t at = (int64_t)r * d.dvp + col;
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f), a = in ? s.get(at + j) : zero, e = in ? u.get(at + j) : zero;
        xs[k][j] = a.x, xs[k][j + 1] = a.y, xs[k][j + 2] = a.z, xs[k][j + 3] = a.w;
        xu[k][j] = e.x, xu[k][j + 1] = e.y, xu[k][j + 2] = e.z, xu[k][j + 3] = e.w;
      }
    }
  };
  fetch(0);
  if (threadIdx.x < 32) cd.fill(p.g.p + b * p.g.sb + t0 * p.g.st + h * p.g.sh, p.g.st, steps);
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  const int row = m + (lane >> 2), col = n0 + (lane & 3) * 2;
  {
    float P[4][4], R[4][4];
    clear(P);
    clear(R);
#pragma unroll
    for (int i = 0; i < NK; ++i) multiply<4, false, false, 1, 1, 1>(P, Q + i * kPlane, m, K + i * kPlane, n0);
#pragma unroll
    for (int i = 0; i < NV; ++i) multiply<4, false, false, 1, 1, 1>(R, G + i * kPlane, m, V + i * kPlane, n0);
    float before[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      Passing pass;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int r = row + 8 * a, j = n * 8 + col;
        float pr[2], rr[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float by = cd.pair(r, j + e) * p.scale;
          pr[e] = by * P[n][2 * a + e];
          rr[e] = by * R[n][2 * a + e];
        }
        pass.each_row(r, j, pr[0] * R[n][2 * a], pr[1] * R[n][2 * a + 1], before[a]);
        store_pair<PP>(Pt, r, j, pr[0], pr[1]);
        store_pair<PP>(Rt, r, j, rr[0], rr[1]);
      }
      pass.join();
      if (lane < 4)
#pragma unroll
        for (int e = 0; e < 2; ++e) passing[warp & 3][n0 + n * 8 + lane * 2 + e] = pass.at[e];
    }
    if (side == 0 && (lane & 3) == 0) rows_m[row] = before[0], rows_m[row + 8] = before[1];
  }
  auto weigh = [&](float (&acc)[4][4], const float* w, float by) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const float f = w[row + 8 * a] * by;
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) acc[n][2 * a + e] = f != 0.0f ? acc[n][2 * a + e] * f : 0.0f;
    }
  };
  auto write = [&](auto* dst, int64_t step, int cols, float (&acc)[4][4]) {
    using T = typename std::remove_pointer<decltype(dst)>::type;
    const bool pairs = ((uintptr_t)dst / sizeof(T) | (uintptr_t)step) % 2 == 0;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int r = row + 8 * a, j = n * 8 + col;
        if (r >= steps) continue;
        T* to = dst + r * step + j;
        if (pairs && j + 1 < cols) {
          *reinterpret_cast<typename Word<2 * sizeof(T)>::type*>(to) = pack<T>(make_float2(acc[n][2 * a], acc[n][2 * a + 1])).w;
        } else {
          if (j < cols) to[0] = Cvt<T>::from(acc[n][2 * a]);
          if (j + 1 < cols) to[1] = Cvt<T>::from(acc[n][2 * a + 1]);
        }
      }
  };
  auto dot = [&](float (&acc)[4][4], const bf16* x, float (&sum)[2]) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t two = *reinterpret_cast<const uint32_t*>(x + (row + 8 * a) * kPitch + n * 8 + col);
        sum[a] = fmaf(__uint_as_float(two << 16), acc[n][2 * a], sum[a]);
        sum[a] = fmaf(__uint_as_float(two & 0xffff0000u), acc[n][2 * a + 1], sum[a]);
      }
  };
  float fq[2] = {0.0f, 0.0f}, fk[2] = {0.0f, 0.0f}, pass = 0.0f, dv[NV][4][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) clear(dv[i]);
#pragma unroll
  for (int ik = 0; ik < NK; ++ik) {
    float aq[4][4], ak[4][4];
    clear(aq);
    clear(ak);
#pragma unroll
    for (int iv = 0; iv < NV; ++iv) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) pass = fmaf(xs[k][j], xu[k][j], pass);
        store8<kExact>(Z + (sr + 32 * k) * kPitch + sc, xs[k]);
        store8<kExact>(W + (sr + 32 * k) * kPitch + sc, xu[k]);
      }
      if (ik * NV + iv + 1 < NK * NV) fetch(ik * NV + iv + 1);
      __syncthreads();
      multiply<4, false, false, 1, kExact, kExact>(aq, G + iv * kPlane, m, Z, n0);
      multiply<4, false, false, 1, kExact, kExact>(ak, V + iv * kPlane, m, W, n0);
      multiply<4, false, true, 1, Keep<bf16>::S, Keep<bf16>::S>(dv[iv], K + ik * kPlane, m, W, n0);
    }
    weigh(aq, cd.into, p.scale);
    weigh(ak, cd.rest, 1.0f);
    dot(aq, Q + ik * kPlane, fq);
    dot(ak, K + ik * kPlane, fk);
    multiply<4, false, true, PP, 1, PP>(aq, Rt, m, K + ik * kPlane, n0);
    multiply<4, true, true, PP, 1, PP>(ak, Rt, m, Q + ik * kPlane, n0);
    const int64_t to = ((b * d.T + t0) * d.H + h) * d.DK + ik * kTile;
    write((O*)p.dq + to, (int64_t)d.H * d.DK, d.DK - ik * kTile, aq);
    write((O*)p.dk + to, (int64_t)d.H * d.DK, d.DK - ik * kTile, ak);
  }
#pragma unroll
  for (int iv = 0; iv < NV; ++iv) {
    weigh(dv[iv], cd.rest, 1.0f);
    multiply<4, true, true, PP, 1, PP>(dv[iv], Pt, m, G + iv * kPlane, n0);
    write((bf16*)p.dv + ((b * d.T + t0) * d.H + h) * d.DV + iv * kTile, (int64_t)d.H * d.DV, d.DV - iv * kTile, dv[iv]);
  }
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    for (int o = 1; o < 4; o <<= 1) {
      fq[a] += __shfl_xor_sync(0xffffffffu, fq[a], o);
      fk[a] += __shfl_xor_sync(0xffffffffu, fk[a], o);
    }
    if ((lane & 3) == 0) {
      far_q[side][row + 8 * a] = fq[a];
      far_k[side][row + 8 * a] = fk[a];
    }
  }
  pass = warp_sum(pass);
  if (lane == 0) through[warp] = pass;
  __syncthreads();
  if (warp != 0) return;
  float near[2], back[2], fore[2];
  // the second half's steps: also what the first half's columns pass to the rows from there on
  const float own = rows_m[2 * lane + 1];
  float rest = rows_m[2 * lane] + own;
  for (int o = 1; o < 32; o <<= 1) {
    const float x = __shfl_down_sync(0xffffffffu, rest, o);
    if (lane + o < 32) rest += x;
  }
  const float next = __shfl_down_sync(0xffffffffu, rest, 1);
  const float half[2] = {lane >= 16 ? rest : 0.0f, lane >= 16 ? (lane < 31 ? next : 0.0f) + own : 0.0f};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int t = 2 * lane + e;
    near[e] = (passing[0][t] + passing[1][t]) + (passing[2][t] + passing[3][t]) + half[e];
    back[e] = far_q[0][t] + far_q[1][t];
    fore[e] = far_k[0][t] + far_k[1][t];
  }
  float all_pass = 0.0f;
  for (int k = 0; k < 8; ++k) all_pass += through[k];
  write_decay(p, cd, b, h, c, steps, near, back, fore, all_pass);
}

// Sums over the heads that share one, in their order: (rows, heads, share, n) floats to (rows, heads, n).
template <class T>
__global__ void __launch_bounds__(256) k_la_unshare(const float* x, T* y, int64_t total, int share, int n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t r = i / n;
  const float* at = x + r * share * n + (i - r * n);
  float s = 0.0f;
  for (int k = 0; k < share; ++k) s += at[(int64_t)k * n];
  y[i] = Cvt<T>::from(s);
}

// A head's decay gradient from the chunks' sums, in a fixed order.
__global__ void __launch_bounds__(256) k_la_decay_sum(const float* x, float* y, int64_t rows, int H) {
  __shared__ float red[32];
  float s = 0.0f;
  for (int64_t r = threadIdx.x; r < rows; r += 256) s += x[r * H + blockIdx.x];
  s = block_sum(s, red);
  if (threadIdx.x == 0) y[blockIdx.x] = s;
}

// --------------------------------------------------------- one token
struct Step {
  int64_t B;
  int H, share, DK, DV;
  Input q, k, v;
  Decay g;
  float scale;
  float* state;
  void* o;
};

constexpr int kStepThreads = 256;
constexpr int kStepRows = 8;  // of the state that a thread has under way

// A block updates the state of one head: a thread takes V neighbouring columns of every (256 / lanes)-th row. The state is
// read and written once and not looked at again soon: evict-first, in both directions.
template <class T, int V>
__global__ void __launch_bounds__(kStepThreads) k_la_step(Step p) {
  __shared__ float qs[kMostChannels], ks[kMostChannels], part[kStepThreads * V];
  const int64_t bh = blockIdx.x, b = bh / p.H;
  const int h = (int)(bh % p.H), lanes = (p.DV + V - 1) / V, groups = kStepThreads / lanes;
  const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes, c = lane * V;
  const bool on = group < groups;
  float* S = p.state + bh * p.DK * p.DV + c;
  using W = typename Word<4 * V>::type;
  union Cell { W w; float f[V]; };
  auto load = [&](Cell (&x)[kStepRows], int r0) {
#pragma unroll
    for (int k = 0; k < kStepRows; ++k)
      if (r0 + k * groups < p.DK) {
        const W* at = reinterpret_cast<const W*>(S + (int64_t)(r0 + k * groups) * p.DV);
        if constexpr (V == 4) x[k].w = ld_stream16(at);
        else x[k].w = *at;
      }
  };
  Cell x[kStepRows];
  if (on) load(x, group);
  for (int i = threadIdx.x; i < p.DK; i += kStepThreads) {
    qs[i] = to_f(p.q.at<T>(b, 0, h / p.share)[i]) * p.scale;
    ks[i] = to_f(p.k.at<T>(b, 0, h / p.share)[i]);
  }
  const float a = expf(p.g.p[b * p.g.sb + h * p.g.sh]);
  float v[V], o[V];
  const T* vp = p.v.at<T>(b, 0, h);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = on && c + j < p.DV ? to_f(vp[c + j]) : 0.0f, o[j] = 0.0f;
  __syncthreads();
  if (on) {
    for (int r0 = group; r0 < p.DK; r0 += kStepRows * groups) {
      if (r0 != group) load(x, r0);
#pragma unroll
      for (int k = 0; k < kStepRows; ++k) {
        const int r = r0 + k * groups;
        if (r >= p.DK) break;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[k].f[j] = fmaf(ks[r], v[j], a != 0.0f ? a * x[k].f[j] : 0.0f);
          o[j] = fmaf(qs[r], x[k].f[j], o[j]);
        }
        W* at = reinterpret_cast<W*>(S + (int64_t)r * p.DV);
        if constexpr (V == 4) st_stream16(at, x[k].w);
        else *at = x[k].w;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) part[(group * lanes + lane) * V + j] = o[j];
  }
  __syncthreads();
  T* out = (T*)p.o + bh * p.DV;
  for (int i = threadIdx.x; i < p.DV; i += kStepThreads) {
    float s = 0.0f;
    for (int g = 0; g < groups; ++g) s += part[g * lanes * V + i];
    out[i] = Cvt<T>::from(s);
  }
}

// ------------------------------------------------------------------- host
size_t round32(size_t n) { return (n + 31) / 32 * 32; }

Shape make_shape(int64_t B, int64_t T, int64_t H, int64_t Hq, int64_t DK, int64_t DV) {
  Shape d = {};
  d.B = B, d.T = T, d.H = (int)H, d.share = (int)(H / Hq), d.DK = (int)DK, d.DV = (int)DV;
  d.dkp = (d.DK + 15) / 16 * 16, d.dvp = (d.DV + 15) / 16 * 16;
  d.chunks = (int)((T + kChunk - 1) / kChunk);
  // Few heads: a row's chunks are walked in segments side by side, down to single chunks, until about four blocks wait
  // on each of 148 SMs. (3 x 777 x 6 heads of 40 float16: 43 us a call, 55 with at least four chunks in a segment.)
  const int64_t blocks = B * H * ((d.dkp + kTile - 1) / kTile) * ((d.dvp + kTile - 1) / kTile);
  int64_t want = 4 * 148 / (blocks > 0 ? blocks : 1), most = d.chunks;
  if (want > most) want = most;
  d.per = want > 1 ? (int)((d.chunks + want - 1) / want) : d.chunks;
  d.segments = d.per > 0 ? (d.chunks + d.per - 1) / d.per : 1;
  return d;
}

// The scratch of one direction's states: without `kept`, those of the segments alone.
struct StateScratch {
  size_t at, since, ends, bytes;
  StateScratch(const Shape& d, size_t from, bool kept) {
    const size_t bh = (size_t)d.B * d.H, size = (size_t)d.dkp * d.dvp * 4;
    at = from;
    since = at + (kept ? bh * d.chunks * size : 0);
    ends = since + round32(bh * d.chunks * 2 * 4);
    bytes = ends + (d.segments > 1 ? bh * d.segments * size : 0);
  }
};
constexpr size_t kStatusBytes = 32;  // the status word leads the scratch

// Whether the walk of whole rows may be taken, as far as the layout does not decide: of every length. Calls of 1, 128 and 512
// steps of 64 heads of 128, forward: 13, 16 and 66 us, by the kernels of chunks 25, 44 and 111; backward: 58, 67 and 185,
// and 92, 123 and 281. It loses where few heads have the four chunks from which rows are cut: 4 heads of 128, 256 steps forward 48 us, and 36.
bool may_walk(int dtype, int64_t DK, int64_t DV, bool aligned) { return aligned && dtype == MPB_BF16 && DK <= 128 && DV <= 128 && DV % 8 == 0; }

// The walk's segments: as many as give every SM (148) a block. They cost a walk more over k and v. Rows of 8192 steps of 128
// channels, forward, 4, 37, 74 and 75 heads: 62, 243, 425 and 451 us; in one segment 416, 432, 449 and 449; in segments for two blocks per SM, which
// run one after the other, 92, 267, 461 and 546.
Shape walk_shape(Shape d) {
  const int64_t heads = d.B * d.H;
  int64_t want = heads > 0 ? 148 / heads : 1, most = d.chunks / 2;
  if (want > most) want = most;
  d.per = want > 1 ? (int)((d.chunks + want - 1) / want) : d.chunks;
  d.segments = d.per > 0 ? (d.chunks + d.per - 1) / d.per : 1;
  return d;
}

Input make_input(const void* p, int64_t sb, int64_t st, int64_t sh, size_t e) {
  return {p, sb, st, sh, (uintptr_t)p % 16 == 0 && (sb * (int64_t)e) % 16 == 0 && (st * (int64_t)e) % 16 == 0 && (sh * (int64_t)e) % 16 == 0};
}

int join_states(const States& p, bool rev, cudaStream_t s) {
  const Shape& d = p.d;
  if (d.segments == 1) return MPB_OK;
  const int64_t heads = d.B * d.H;
  const dim3 blocks((unsigned)((d.dkp * d.dvp / 4 + 127) / 128), (unsigned)(heads < 65535 ? heads : 65535));
  if (rev) k_la_join<true><<<blocks, 128, 0, s>>>(p);
  else k_la_join<false><<<blocks, 128, 0, s>>>(p);
  return launch_check("linear_attention");
}

// The states of p's chunks (p.at null: of its segments alone).
template <class T, bool REV>
int run_states(const States& p, bool walk, int* status, cudaStream_t s) {
  constexpr int kStatesBytes = (kExact + RawPieces<T>::n) * kPlane * 2;
  const Shape& d = p.d;
  if (walk) {
    const Walk w = {d, {}, p.x, p.y, p.g, p.first, nullptr, p.scale, nullptr, REV, p.at, p.since, p.ends, p.last, status};
    if (int rc = walk_states(w, s)) return rc;
  } else {
    const int64_t tiles = (int64_t)((d.dkp + kTile - 1) / kTile) * ((d.dvp + kTile - 1) / kTile);
    if (int rc = allow_smem<k_la_states<T, REV>, kStatesBytes>("linear_attention")) return rc;
    States q = p;
    q.status = status;
    k_la_states<T, REV><<<(unsigned)(d.B * d.H * d.segments * tiles), kThreads, kStatesBytes, s>>>(q);
    if (int rc = launch_check("linear_attention")) return rc;
  }
  return join_states(p, REV, s);
}

template <class T>
int run_forward(Shape d, const Input& q, const Input& k, const Input& v, const Decay& g, const float* first, float scale,
                void* o, float* state, bool walk, char* scratch, cudaStream_t s) {
  int* status = (int*)scratch;
  if (walk) d = walk_shape(d);
  const StateScratch w(d, kStatusBytes, !walk);
  States st = {d, k, v, g, first, 1.0f, walk ? nullptr : (float*)(scratch + w.at), (float*)(scratch + w.since),
               (float*)(scratch + w.ends), state};
  if (walk) {
    if (int rc = cuda_check(cudaMemsetAsync(status, 0, kStatusBytes, s), "linear_attention")) return rc;
    if (d.segments > 1)
      if (int rc = run_states<T, false>(st, true, status, s)) return rc;
    const Walk p = {d, q, k, v, g, first, st.ends, scale, o, false, nullptr, nullptr, nullptr, d.segments > 1 ? nullptr : state, status};
    return walk_outputs(p, s);
  }
  if (int rc = run_states<T, false>(st, false, status, s)) return rc;
  constexpr int PT = RawPieces<T>::n, PS = Keep<T>::S;
  constexpr int kOutputBytes = (2 * PT + (PT > PS ? PT : PS)) * kPlane * 2;
  Outputs out = {d, q, k, v, g, scale, {st.at, st.since, st.ends}, o};
  if (int rc = allow_smem<k_la_output<T>, kOutputBytes>("linear_attention")) return rc;
  k_la_output<T><<<(unsigned)(d.B * d.H * d.chunks * ((d.dvp + kTile - 1) / kTile)), kThreads, kOutputBytes, s>>>(out);
  return launch_check("linear_attention");
}

// What the gradients need besides the states: per-head dq and dk where heads share one, and the chunks' sums of dg.
struct GradScratch {
  size_t s, u, dq, dk, dg, bytes;
  GradScratch(const Shape& d, bool by_head) {
    const StateScratch a(d, kStatusBytes, true), b(d, a.bytes, true);
    const size_t part = d.share > 1 ? (size_t)d.B * d.T * d.H * d.DK * 4 : 0;
    s = kStatusBytes, u = a.bytes, dq = round32(b.bytes), dk = dq + round32(part), dg = dk + round32(part);
    bytes = dg + (by_head ? round32((size_t)d.B * d.chunks * d.H * 4) : 0);
  }
};

template <int NK, int NV, class O>
int run_wide(const Gradients& p, cudaStream_t s) {
  constexpr int kWideBytes = (2 * NK + 2 * NV + 2 * kExact + 2 * Keep<bf16>::P) * kPlane * 2;
  if (int rc = allow_smem<k_la_gradients_wide<NK, NV, O>, kWideBytes>("linear_attention_backward")) return rc;
  k_la_gradients_wide<NK, NV, O><<<(unsigned)(p.d.B * p.d.H * p.d.chunks), kWideThreads, kWideBytes, s>>>(p);
  return launch_check("linear_attention_backward");
}

// wide: bf16 heads of up to 128 channels, all inputs in 16-byte words.
template <class T, class O>
int run_gradients(const Gradients& p, bool wide, cudaStream_t s) {
  if constexpr (std::is_same<T, bf16>::value) {
    if (wide) {
      if (p.d.DK > 64) return p.d.DV > 64 ? run_wide<2, 2, O>(p, s) : run_wide<2, 1, O>(p, s);
      return p.d.DV > 64 ? run_wide<1, 2, O>(p, s) : run_wide<1, 1, O>(p, s);
    }
  }
  constexpr int kGradBytes = (2 * RawPieces<T>::n + 2 * kExact + Keep<T>::P) * kPlane * 2;
  if (int rc = allow_smem<k_la_gradients<T, O>, kGradBytes>("linear_attention_backward")) return rc;
  k_la_gradients<T, O><<<(unsigned)(p.d.B * p.d.H * p.d.chunks), kThreads, kGradBytes, s>>>(p);
  return launch_check("linear_attention_backward");
}

template <class T>
int run_backward(Gradients p, const float* first, const float* dstate, void* dq, void* dk, float* dg, bool by_head, float* dfirst,
                 bool walk, char* scratch, cudaStream_t s) {
  if (walk) p.d = walk_shape(p.d);
  const Shape& d = p.d;
  const GradScratch w(d, by_head);
  const StateScratch a(d, w.s, true), b(d, w.u, true);
  int* status = (int*)scratch;
  if (walk)
    if (int rc = cuda_check(cudaMemsetAsync(status, 0, kStatusBytes, s), "linear_attention_backward")) return rc;
  States st = {d, p.k, p.v, p.g, first, 1.0f, (float*)(scratch + a.at), (float*)(scratch + a.since), (float*)(scratch + a.ends), nullptr};
  if (int rc = run_states<T, false>(st, walk, status, s)) return rc;
  States ut = {d, p.q, p.g_o, p.g, dstate, p.scale, (float*)(scratch + b.at), (float*)(scratch + b.since), (float*)(scratch + b.ends),
               dfirst};
  if (int rc = run_states<T, true>(ut, walk, status, s)) return rc;
  p.s = {st.at, st.since, st.ends}, p.u = {ut.at, ut.since, ut.ends};
  p.dg = by_head ? nullptr : dg, p.dg_chunk = by_head ? (float*)(scratch + w.dg) : nullptr;
  if (d.share > 1) {
    p.dq = scratch + w.dq, p.dk = scratch + w.dk;
    if (int rc = run_gradients<T, float>(p, walk, s)) return rc;
    const int64_t total = d.B * d.T * (d.H / d.share) * d.DK;
    const unsigned blocks = (unsigned)((total + 255) / 256);
    k_la_unshare<T><<<blocks, 256, 0, s>>>((const float*)p.dq, (T*)dq, total, d.share, d.DK);
    k_la_unshare<T><<<blocks, 256, 0, s>>>((const float*)p.dk, (T*)dk, total, d.share, d.DK);
    if (int rc = launch_check("linear_attention_backward")) return rc;
  } else {
    p.dq = dq, p.dk = dk;
    if (int rc = run_gradients<T, T>(p, walk, s)) return rc;
  }
  if (by_head) {
    k_la_decay_sum<<<(unsigned)d.H, 256, 0, s>>>(p.dg_chunk, dg, d.B * d.chunks, d.H);
    return launch_check("linear_attention_backward");
  }
  return MPB_OK;
}

template <class T>
int run_step(const Step& p, cudaStream_t s) {
  const unsigned grid = (unsigned)(p.B * p.H);
  if (p.DV % 4 == 0) k_la_step<T, 4><<<grid, kStepThreads, 0, s>>>(p);
  else k_la_step<T, 1><<<grid, kStepThreads, 0, s>>>(p);
  return launch_check("linear_attention_step");
}

int check_shape(const char* name, int64_t B, int64_t T, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype) {
  if (dtype != MPB_F32 && dtype != MPB_F16 && dtype != MPB_BF16)
    return fail(MPB_ERR_DTYPE, "%s: dtype %d not supported (float16, bfloat16, float32)", name, dtype);
  if (B < 0 || T < 0 || H < 1 || Hq < 1 || H % Hq != 0)
    return fail(MPB_ERR_SHAPE, "%s: %lld sequences of %lld steps, %lld heads over %lld", name, (long long)B, (long long)T,
                (long long)H, (long long)Hq);
  if (DK < 1 || DV < 1 || DK > kMostChannels || DV > kMostChannels)
    return fail(MPB_ERR_SHAPE, "%s: %lld and %lld channels per head (1 to %d)", name, (long long)DK, (long long)DV, kMostChannels);
  // blocks, and bytes of a state for each chunk, are counted in 64 bits; the grid in 31
  if (H > (1 << 20) || B > (1LL << 31) || T > (1LL << 36) || (double)B * H * ((T + kChunk - 1) / kChunk + 1) * 16 > 2147483647.0)
    return fail(MPB_ERR_SHAPE, "%s: %lld sequences of %lld steps and %lld heads are too many for one call", name, (long long)B,
                (long long)T, (long long)H);
  return MPB_OK;
}

size_t bytes_of(int dtype) { return dtype == MPB_F32 ? 4 : 2; }

int check_scratch(const char* name, size_t need, const void* scratch, size_t bytes) {
  if (need > bytes || (need && !scratch)) return fail(MPB_ERR_SCRATCH, "%s: %zu bytes of scratch, %zu needed", name, bytes, need);
  if (need && (uintptr_t)scratch % 16 != 0) return fail(MPB_ERR_INVALID, "%s: scratch not 16-byte aligned", name);
  return MPB_OK;
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" {

size_t mpb_linear_attention_scratch_bytes(int64_t B, int64_t T, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype,
                                          int backward, int decay_by_head, int aligned) {
  if (check_shape("linear_attention", B, T, H, Hq, DK, DV, dtype) || B * T == 0) return 0;
  Shape d = make_shape(B, T, H, Hq, DK, DV);
  const bool walk = may_walk(dtype, DK, DV, aligned != 0);
  if (walk) d = walk_shape(d);
  return backward ? GradScratch(d, decay_by_head != 0).bytes : StateScratch(d, kStatusBytes, !walk).bytes;
}

int mpb_linear_attention_status(const void* scratch, mpb_stream_t stream) {
  if (!scratch) return MPB_OK;
  int status = MPB_OK;
  if (int rc = cuda_check(cudaMemcpyAsync(&status, scratch, sizeof(int), cudaMemcpyDeviceToHost, (cudaStream_t)stream), "linear_attention"))
    return rc;
  if (int rc = cuda_check(cudaStreamSynchronize((cudaStream_t)stream), "linear_attention")) return rc;
  return status == MPB_ERR_TIMEOUT ? fail(MPB_ERR_TIMEOUT, "linear_attention: a wait between its warps gave up") : MPB_OK;
}

int64_t mpb_linear_attention_wait_limit(int64_t ns) {
  return walk_wait_limit(ns < 0 ? 0 : ns > (int64_t)kMostWaitNs ? (int64_t)kMostWaitNs : ns);
}

int mpb_linear_attention(int64_t B, int64_t T, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype, const void* q,
                         int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                         const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const float* log_decay, int64_t g_sb,
                         int64_t g_st, int64_t g_sh, const float* state0, double scale, void* o, float* state, void* scratch,
                         size_t scratch_bytes, mpb_stream_t stream) {
  const char* name = "linear_attention";
  if (int rc = check_shape(name, B, T, H, Hq, DK, DV, dtype)) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const size_t state_bytes = (size_t)(B * H * DK * DV) * 4;
  if (B == 0) return MPB_OK;
  if (T == 0) {  // the state stays what it was
    if (!state) return MPB_OK;
    if (state0) return cuda_check(cudaMemcpyAsync(state, state0, state_bytes, cudaMemcpyDeviceToDevice, s), name);
    return cuda_check(cudaMemsetAsync(state, 0, state_bytes, s), name);
  }
  if (!q || !k || !v || !log_decay || !o) return fail(MPB_ERR_INVALID, "%s: null pointer", name);
  const Shape d = make_shape(B, T, H, Hq, DK, DV);
  const size_t e = bytes_of(dtype);
  const Input qi = make_input(q, q_sb, q_st, q_sh, e), ki = make_input(k, k_sb, k_st, k_sh, e), vi = make_input(v, v_sb, v_st, v_sh, e);
  const bool walk = may_walk(dtype, DK, DV, (uintptr_t)o % 16 == 0) && walk_takes(d, qi, ki, vi);
  if (int rc = check_scratch(name, mpb_linear_attention_scratch_bytes(B, T, H, Hq, DK, DV, dtype, 0, 0, walk), scratch, scratch_bytes))
    return rc;
  const Decay g = {log_decay, g_sb, g_st, g_sh};
  switch (dtype) {
    case MPB_F32: return run_forward<float>(d, qi, ki, vi, g, state0, (float)scale, o, state, walk, (char*)scratch, s);
    case MPB_F16: return run_forward<__half>(d, qi, ki, vi, g, state0, (float)scale, o, state, walk, (char*)scratch, s);
    default: return run_forward<bf16>(d, qi, ki, vi, g, state0, (float)scale, o, state, walk, (char*)scratch, s);
  }
}

int mpb_linear_attention_backward(int64_t B, int64_t T, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype, const void* dout,
                                  int64_t do_sb, int64_t do_st, int64_t do_sh, const void* q, int64_t q_sb, int64_t q_st,
                                  int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v,
                                  int64_t v_sb, int64_t v_st, int64_t v_sh, const float* log_decay, int64_t g_sb, int64_t g_st,
                                  int64_t g_sh, const float* state0, const float* dstate, double scale, void* dq, void* dk,
                                  void* dv, float* dlog_decay, int decay_by_head, float* dstate0, void* scratch,
                                  size_t scratch_bytes, mpb_stream_t stream) {
  const char* name = "linear_attention_backward";
  if (int rc = check_shape(name, B, T, H, Hq, DK, DV, dtype)) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const size_t state_bytes = (size_t)(B * H * DK * DV) * 4;
  if (B * T == 0) {
    if (decay_by_head && dlog_decay)
      if (int rc = cuda_check(cudaMemsetAsync(dlog_decay, 0, (size_t)H * 4, s), name)) return rc;
    if (B == 0 || !dstate0) return MPB_OK;
    if (dstate) return cuda_check(cudaMemcpyAsync(dstate0, dstate, state_bytes, cudaMemcpyDeviceToDevice, s), name);
    return cuda_check(cudaMemsetAsync(dstate0, 0, state_bytes, s), name);
  }
  if (!dout || !q || !k || !v || !log_decay || !dq || !dk || !dv || !dlog_decay || !dstate0)
    return fail(MPB_ERR_INVALID, "%s: null pointer", name);
  const size_t e = bytes_of(dtype);
  Gradients p = {};
  p.d = make_shape(B, T, H, Hq, DK, DV);
  p.q = make_input(q, q_sb, q_st, q_sh, e), p.k = make_input(k, k_sb, k_st, k_sh, e);
  p.v = make_input(v, v_sb, v_st, v_sh, e), p.g_o = make_input(dout, do_sb, do_st, do_sh, e);
  p.g = {log_decay, g_sb, g_st, g_sh};
  p.scale = (float)scale, p.dv = dv;
  const bool walk = may_walk(dtype, DK, DV, true) && walk_takes(p.d, p.q, p.k, p.v) && walk_takes(p.d, p.q, p.k, p.g_o);
  if (int rc = check_scratch(name, mpb_linear_attention_scratch_bytes(B, T, H, Hq, DK, DV, dtype, 1, decay_by_head, walk), scratch,
                             scratch_bytes))
    return rc;
  const bool by = decay_by_head != 0;
  switch (dtype) {
    case MPB_F32: return run_backward<float>(p, state0, dstate, dq, dk, dlog_decay, by, dstate0, walk, (char*)scratch, s);
    case MPB_F16: return run_backward<__half>(p, state0, dstate, dq, dk, dlog_decay, by, dstate0, walk, (char*)scratch, s);
    default: return run_backward<bf16>(p, state0, dstate, dq, dk, dlog_decay, by, dstate0, walk, (char*)scratch, s);
  }
}

int mpb_linear_attention_step(int64_t B, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype, const void* q, int64_t q_sb,
                              int64_t q_sh, const void* k, int64_t k_sb, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_sh,
                              const float* log_decay, int64_t g_sb, int64_t g_sh, double scale, float* state, void* o,
                              mpb_stream_t stream) {
  const char* name = "linear_attention_step";
  if (int rc = check_shape(name, B, 1, H, Hq, DK, DV, dtype)) return rc;
  if (B == 0) return MPB_OK;
  if (!q || !k || !v || !log_decay || !state || !o) return fail(MPB_ERR_INVALID, "%s: null pointer", name);
  if ((uintptr_t)state % 16 != 0) return fail(MPB_ERR_INVALID, "%s: state not 16-byte aligned", name);
  const size_t e = bytes_of(dtype);
  Step p = {B, (int)H, (int)(H / Hq), (int)DK, (int)DV, make_input(q, q_sb, 0, q_sh, e), make_input(k, k_sb, 0, k_sh, e),
            make_input(v, v_sb, 0, v_sh, e), {log_decay, g_sb, 0, g_sh}, (float)scale, state, o};
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case MPB_F32: return run_step<float>(p, s);
    case MPB_F16: return run_step<__half>(p, s);
    default: return run_step<bf16>(p, s);
  }
}

}  // extern "C"

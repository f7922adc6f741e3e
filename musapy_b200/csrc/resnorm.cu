// Root-mean-square norms before and after a block, fused with the block's
// gate, dropout and residual scale. For every row (no counterpart in the
// reference):
//
//   r_z = (mean z^2 + eps)^-1/2       n = z r_z w_post
//   y   = x + m act(g) n              m = scale, or scale * keep / (1 - p)
//   r_y = (mean y^2 + eps)^-1/2       u = y r_y w_pre
//
// z is what the block computed, y the residual stream after it and u the
// normed input of the next block. Without a branch (z null) y = x: the plain
// norm. Backward, with the gradients dy and du:
//
//   dx = dy + r_y (w_pre du - y^ mean(y^ w_pre du)),          y^ = y r_y
//   dn = dx m act(g),   dz = r_z (w_post dn - z^ mean(z^ w_post dn)),  z^ = z r_z
//   dg = dx m n act'(g),   dw_post = sum dn z^,   dw_pre = sum du y^
//
// Rows run in float; y and u are rounded once from it (u from the unrounded
// y). The backward pass takes y as it was stored and r_z, r_y as the forward
// pass left them.
//
// A row lives in the registers of its threads (a warp or several, up to 512
// threads with 32 elements each) between its reductions, so every input is
// read once and every output written once. At 32 elements per thread, rows above 8192
// elements, the backward pass does not fit 128 registers and spills 130 to 230
// bytes per thread in 16-bit types, 300 to 400 in float, and 700 to 940 where
// bounds are checked or the packs are single elements (forward 80 at most). In the backward pass blocks take
// rows in turn and add the weights' gradients up in shared memory, each thread
// its own columns; a second kernel adds the blocks' sums in a fixed order.
// Rows too long for that (above 16384 elements) are read again for each pass, and
// their column sums are taken by one thread per column over all rows.
//
// Bound: memory. Measured, 16384 x 4096 with a full gate, f32: forward 203 us
// (6.6 TB/s), backward 432 us (5.0 TB/s); bf16: forward 111 us (6.0 TB/s), with
// dropout 130 us, backward 221 us (4.9 TB/s) and 226 us; the plain norm 46 us (5.9
// TB/s) and 123 us (3.3 TB/s), f32 84 and 155 us. 4096 x 16384 bf16: 174 and 281 us.
// 2048 x 32768 bf16 (re-read): 1044 and 5065 us. The backward pass runs
// about 60 instructions per element at 16 warps per SM (the registers of 16
// elements' five inputs and sums): their issue, half of it stalled on the
// row's loads and the two reductions, is what is left above the bytes.
// Tried against earlier forms: copying the next row ahead into shared memory, 243 us
// against 237 (bf16, no dropout) and 576 against 435 us (f32: fewer resident blocks);
// one pack per thread and 512 threads per row, 240 us against 209. That 209 us was
// a warp's packs 32 apart over the whole row; one warp's packs after the other, as
// now, costs 221 us there and saves odd widths a sixth or more. Rows that no 16-byte
// access may use go element by element (16383 x 4095, f32: forward 238 us, backward
// 690 us; bf16: 208 and 630 us) or, 16-bit types of even width, by pairs (16384 x
// 4094 bf16: 142 and 302 us), and with dropout they draw a counter for each element
// or pair (bf16: 436 and 803 us; pairs 242 and 434 us).
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "philox.cuh"
#include "rows.cuh"

namespace mpb {
namespace {

struct NormArgs {
  int64_t R, D;
  const void *x, *z, *gate, *dy, *du, *yin;
  int64_t x_sr, z_sr, g_sr, dy_sr, du_sr, y_sr;  // row strides, elements
  const float *w_post, *w_pre;
  const float* rstd;  // backward: (2, R), or (R) without a branch
  void *y, *u, *dx, *dz, *dgate;
  float *rstd_out, *dw_post, *dw_pre;
  float* part;  // backward scratch
  int gate_kind, act;
  float scale, eps;
  Dropper drop;
  int dropping;
};

constexpr int kThreads = 256;     // a row longer than kInRegisters
constexpr int kRowThreads = 512;  // of a row in registers, at most
constexpr int kPerThread = 32;    // its elements per thread, at most
constexpr int64_t kMostStride = 1 << 29;  // between rows: its bytes are multiplied in 32 bits
constexpr int64_t kInRegisters = (int64_t)kRowThreads * kPerThread;

template <class T>
MPB_D void act_of(int act, float g, float& v, float& slope) {
  if (act == MPB_ACT_LINEAR) {
    v = g;
    slope = 1.0f;
    return;
  }
  float s, om;
  sigmoid2<sizeof(T) == 4>(g, s, om);
  if (act == MPB_ACT_SIGMOID) {
    v = s;
    slope = s * om;
  } else {
    v = g * s;
    slope = s * (1.0f + g * om);
  }
}

template <class T>
MPB_D float gate_at(const NormArgs& p, int64_t r, int64_t c) {
  const T* g = (const T*)p.gate;
  return to_f(p.gate_kind == MPB_GATE_FULL ? g[r * p.g_sr + c] : p.gate_kind == MPB_GATE_ROW ? g[r * p.g_sr] : g[c]);
}

MPB_D float branch_factor(const NormArgs& p, int64_t r, int64_t c) {
  if (!p.dropping) return p.scale;
  return keeps(p.drop, (uint64_t)(r * p.D + c)) ? p.scale * p.drop.up : 0.0f;
}

template <class T>
MPB_D float stream_at(const NormArgs& p, int64_t r, int64_t c, float rz) {
  float y = to_f(((const T*)p.x)[r * p.x_sr + c]);
  if (p.z) {
    const float m = branch_factor(p, r, c);
    if (m != 0.0f) {
      float v = 1.0f, slope;
      if (p.gate_kind != MPB_GATE_NONE) act_of<T>(p.act, gate_at<T>(p, r, c), v, slope);
      y += m * v * (to_f(((const T*)p.z)[r * p.z_sr + c]) * rz * p.w_post[c]);
    }
  }
  return y;
}

// Long rows, one block per row.
template <class T>
__global__ void __launch_bounds__(kThreads) k_norm_long(NormArgs p) {
  __shared__ float red[2][32];
  const int64_t r = blockIdx.x;
  float rz = 0.0f;
  if (p.z) {
    float ss = 0.0f;
    for (int64_t c = threadIdx.x; c < p.D; c += kThreads) {
      const float z = to_f(((const T*)p.z)[r * p.z_sr + c]);
      ss = fmaf(z, z, ss);
    }
    rz = 1.0f / sqrtf(block_sum(ss, red[0]) / (float)p.D + p.eps);
  }
  float ss = 0.0f;
  for (int64_t c = threadIdx.x; c < p.D; c += kThreads) {
    const float y = stream_at<T>(p, r, c, rz);
    ss = fmaf(y, y, ss);
    if (p.y) ((T*)p.y)[r * p.D + c] = Cvt<T>::from(y);
  }
  const float ry = 1.0f / sqrtf(block_sum(ss, red[1]) / (float)p.D + p.eps);
  for (int64_t c = threadIdx.x; c < p.D; c += kThreads)
    ((T*)p.u)[r * p.D + c] = Cvt<T>::from(stream_at<T>(p, r, c, rz) * ry * p.w_pre[c]);
  if (threadIdx.x == 0) {
    if (p.z) p.rstd_out[r] = rz;
    p.rstd_out[(p.z ? p.R : 0) + r] = ry;
  }
}

// Long rows, one block per row: the row's gradients.
template <class T>
__global__ void __launch_bounds__(kThreads) k_norm_bwd_long(NormArgs p) {
  __shared__ float red[3][32];
  const int64_t r = blockIdx.x;
  const float rz = p.z ? p.rstd[r] : 0.0f, ry = p.rstd[(p.z ? p.R : 0) + r];
  const T *du = (const T*)p.du + r * p.du_sr, *y = (const T*)p.yin + r * p.y_sr;
  const T *dy = (const T*)p.dy + r * p.dy_sr, *z = (const T*)p.z + r * p.z_sr;
  float dot = 0.0f;
  if (p.du)
    for (int64_t c = threadIdx.x; c < p.D; c += kThreads)
      dot = fmaf(to_f(du[c]) * p.w_pre[c], to_f(y[c]) * ry, dot);
  const float my = block_sum(dot, red[0]) / (float)p.D;
  auto dx_at = [&](int64_t c) {
    const float base = p.dy ? to_f(dy[c]) : 0.0f;
    return p.du ? base + ry * (to_f(du[c]) * p.w_pre[c] - to_f(y[c]) * ry * my) : base;
  };
  float dotz = 0.0f, dgr = 0.0f;
  for (int64_t c = threadIdx.x; c < p.D; c += kThreads) {
    const float dx = dx_at(c);
    ((T*)p.dx)[r * p.D + c] = Cvt<T>::from(dx);
    if (!p.z) continue;
    const float m = branch_factor(p, r, c);
    float v = 1.0f, slope = 0.0f;
    if (p.gate_kind != MPB_GATE_NONE) act_of<T>(p.act, gate_at<T>(p, r, c), v, slope);
    const float zh = to_f(z[c]) * rz;
    const float d = m == 0.0f ? 0.0f : dx * m;
    if (m != 0.0f) dotz = fmaf(d * v * p.w_post[c], zh, dotz);
    const float dg = m == 0.0f ? 0.0f : d * (zh * p.w_post[c]) * slope;
    if (p.gate_kind == MPB_GATE_FULL) ((T*)p.dgate)[r * p.D + c] = Cvt<T>::from(dg);
    dgr += dg;
  }
  if (!p.z) return;
  const float mz = block_sum(dotz, red[1]) / (float)p.D;
  if (p.gate_kind == MPB_GATE_ROW) {
    dgr = block_sum(dgr, red[2]);
    if (threadIdx.x == 0) ((T*)p.dgate)[r] = Cvt<T>::from(dgr);
  }
  for (int64_t c = threadIdx.x; c < p.D; c += kThreads) {
    const float m = branch_factor(p, r, c);
    float v = 1.0f, slope;
    if (p.gate_kind != MPB_GATE_NONE) act_of<T>(p.act, gate_at<T>(p, r, c), v, slope);
    const float dn = m == 0.0f ? 0.0f : dx_at(c) * m * v;
    ((T*)p.dz)[r * p.D + c] = Cvt<T>::from(rz * (dn * p.w_post[c] - to_f(z[c]) * rz * mz));
  }
}

// One thread per column: the gradients of the weights and of a gate per channel. dx is read back
// from where the row kernel left it.
template <class T>
__global__ void k_norm_bwd_long_cols(NormArgs p) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= p.D) return;
  float wpre = 0.0f, wpost = 0.0f, dgc = 0.0f;
  for (int64_t r = 0; r < p.R; ++r) {
    const float ry = p.rstd[(p.z ? p.R : 0) + r];
    if (p.du) wpre += to_f(((const T*)p.du)[r * p.du_sr + c]) * (to_f(((const T*)p.yin)[r * p.y_sr + c]) * ry);
    if (!p.z) continue;
    const float m = branch_factor(p, r, c);
    if (m == 0.0f) continue;
    float v = 1.0f, slope = 0.0f;
    if (p.gate_kind != MPB_GATE_NONE) act_of<T>(p.act, gate_at<T>(p, r, c), v, slope);
    const float zh = to_f(((const T*)p.z)[r * p.z_sr + c]) * p.rstd[r];
    const float d = p.part[r * p.D + c] * m;
    wpost += d * v * zh;
    dgc += d * zh * p.w_post[c] * slope;
  }
  p.dw_pre[c] = wpre;
  if (p.z) p.dw_post[c] = wpost;
  if (p.gate_kind == MPB_GATE_CHANNEL) ((T*)p.dgate)[c] = Cvt<T>::from(dgc);
}

// dx in float for the column kernel.
template <class T>
__global__ void __launch_bounds__(kThreads) k_norm_bwd_long_dx(NormArgs p) {
  __shared__ float red[32];
  const int64_t r = blockIdx.x;
  const float ry = p.rstd[(p.z ? p.R : 0) + r];
  const T *du = (const T*)p.du + r * p.du_sr, *y = (const T*)p.yin + r * p.y_sr, *dy = (const T*)p.dy + r * p.dy_sr;
  float dot = 0.0f;
  if (p.du)
    for (int64_t c = threadIdx.x; c < p.D; c += kThreads)
      dot = fmaf(to_f(du[c]) * p.w_pre[c], to_f(y[c]) * ry, dot);
  const float my = block_sum(dot, red) / (float)p.D;
  for (int64_t c = threadIdx.x; c < p.D; c += kThreads) {
    const float base = p.dy ? to_f(dy[c]) : 0.0f;
    p.part[r * p.D + c] = p.du ? base + ry * (to_f(du[c]) * p.w_pre[c] - to_f(y[c]) * ry * my) : base;
  }
}

// ------------------------------------------------------- rows in registers
// W elements of T, one or two words of at most 16 bytes, worked on as pairs of
// floats (W == 1: as single ones).
template <class T, int W>
struct Elems {
  static constexpr int kBytes = (int)sizeof(T) * W, kWordBytes = kBytes > 16 ? 16 : kBytes, kWords = kBytes / kWordBytes;
  static constexpr int kPer = W % 2 == 0 ? 2 : 1, kParts = W / kPer;
  using F = Floats<kPer>;
  using Wd = typename Word<kWordBytes>::type;
  union {
    Wd w[kWords];
    T v[W];
    typename Word<(int)sizeof(T) * kPer>::type part[kParts];
  };
  MPB_D Elems() {}
  MPB_D void load(const T* q) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = __ldcs(reinterpret_cast<const Wd*>(q) + k);
  }
  MPB_D void store(T* q) const {
#pragma unroll
    for (int k = 0; k < kWords; ++k) __stcs(reinterpret_cast<Wd*>(q) + k, w[k]);
  }
  MPB_D F get(int i) const {
    Pack<T, kPer> p;
    p.w = part[i];
    return unpack(p);
  }
  MPB_D void put(int i, F f) { part[i] = pack<T>(f).w; }
};

template <class T, int W>
MPB_D void load_floats(const float* q, typename Elems<T, W>::F (&v)[Elems<T, W>::kParts]) {
  if constexpr (W % 4 == 0) {
#pragma unroll
    for (int k = 0; k < W / 4; ++k) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(q) + k);
      v[2 * k] = make_float2(f.x, f.y);
      v[2 * k + 1] = make_float2(f.z, f.w);
    }
  } else if constexpr (W == 2) {
    v[0] = make_float2(__ldg(q), __ldg(q + 1));
  } else {
    v[0] = __ldg(q);
  }
}

// What dropout keeps of W elements from index i on (a multiple of W).
template <int W>
struct Kept {
  uint4 w;
  uint32_t first;
  MPB_D Kept() {}
  MPB_D Kept(const Dropper& d, uint64_t i) : w(drop_words(d, i >> 3)), first((uint32_t)i & 7) {}
  MPB_D bool operator()(const Dropper& d, int j) const {
    if constexpr (W == 8) return stays(d, w, j);
    const uint32_t at = first + j, word = at < 4 ? (at < 2 ? w.x : w.y) : (at < 6 ? w.z : w.w);
    return ((at & 1) ? word : word << 16) >= d.drop;
  }
  // f where kept, g where dropped, of part i
  MPB_D float pick(const Dropper& d, int i, float f, float g) const { return (*this)(d, i) ? f : g; }
  MPB_D float2 pick(const Dropper& d, int i, float2 f, float2 g) const {
    return make_float2((*this)(d, 2 * i) ? f.x : g.x, (*this)(d, 2 * i + 1) ? f.y : g.y);
  }
};

// Row r of an operand, `skip` elements on: the row's stride in bytes fits 32
// bits (checked), so this is one wide multiply-add.
template <class T>
MPB_D const T* row_at(const void* base, int r, int64_t sr, int skip) {
  return reinterpret_cast<const T*>((const char*)base + (int64_t)r * (int)(sr * (int)sizeof(T))) + skip;
}

// Sum over a row's threads: a warp, or the whole block (blockDim.y == 1).
MPB_D float row_sum(float v, float* red) { return blockDim.x == 32 ? warp_sum(v) : block_sum(v, red); }
MPB_D float fold(float v) { return v; }
MPB_D float fold(float2 v) { return v.x + v.y; }

// What dropout keeps of a row. EARLY: drawn while the row's loads are under way,
// where that is a counter per pack; else drawn at each pack. (16384 x 4096 bf16, the
// backward form then: 232 us early, 243 us late; forward, where the words cost a
// resident block, 144 and 130 us.)
template <int W, int NV, bool EARLY>
struct KeptRow {
  static constexpr bool kEarly = EARLY && W == 8;
  Kept<W> all[kEarly ? NV : 1];
  MPB_D KeptRow(const NormArgs& p, int r, int skip) {
    if constexpr (kEarly)
#pragma unroll
      for (int k = 0; k < NV; ++k) all[k] = Kept<W>(p.drop, (uint64_t)((int64_t)r * p.D + skip + k * 32 * W));
  }
  MPB_D Kept<W> at(const NormArgs& p, int r, int k, int c) const {
    if constexpr (kEarly) return all[k];
    else return Kept<W>(p.drop, (uint64_t)((int64_t)r * p.D + c));
  }
};

// The values and slopes of the gate for the pack at column c of row r; `full`
// has been loaded with the row's other operands. One switch for all elements.
template <class T, int W>
MPB_D void gate_pack(const NormArgs& p, const Elems<T, W>& full, int64_t r, int c,
                     typename Elems<T, W>::F (&v)[Elems<T, W>::kParts],
                     typename Elems<T, W>::F (&slope)[Elems<T, W>::kParts]) {
  using E = Elems<T, W>;
  using F = typename E::F;
  constexpr int NP = E::kParts;
  const F one = vset<E::kPer>(1.0f);
  F g[NP];
  if (p.gate_kind == MPB_GATE_FULL) {
#pragma unroll
    for (int i = 0; i < NP; ++i) g[i] = full.get(i);
  } else if (p.gate_kind == MPB_GATE_NONE) {
#pragma unroll
    for (int i = 0; i < NP; ++i) v[i] = one, slope[i] = vset<E::kPer>(0.0f);
    return;
  } else {
    const T* q = p.gate_kind == MPB_GATE_ROW ? (const T*)p.gate + r * p.g_sr : (const T*)p.gate + c;
    const int st = p.gate_kind == MPB_GATE_ROW ? 0 : 1;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < E::kPer; ++j) vput(g[i], j, to_f(q[(i * E::kPer + j) * st]));
  }
  if (p.act == MPB_ACT_LINEAR) {
#pragma unroll
    for (int i = 0; i < NP; ++i) v[i] = g[i], slope[i] = one;
  } else if (p.act == MPB_ACT_SIGMOID) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      F om;
      sigmoid2<sizeof(T) == 4>(g[i], v[i], om);
      slope[i] = vmul(v[i], om);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      F s, om;
      sigmoid2<sizeof(T) == 4>(g[i], s, om);
      v[i] = vmul(g[i], s);
      slope[i] = vmul(s, vfma(g[i], om, one));
    }
  }
}

enum { kPlain = 0, kBranch = 1, kDropped = 2 };  // no branch, a branch, a branch with dropout

// blockDim.x threads per row, blockDim.y rows per block (more than one only
// for rows of a warp). A warp holds 32 NV packs one after the other, a lane every
// 32nd of them: the distances within a thread are constants.
template <class T, int W, int NV, int MODE>
__global__ void __launch_bounds__(kRowThreads) k_norm_rows(NormArgs p) {
  using E = Elems<T, W>;
  using F = typename E::F;
  constexpr int NP = E::kParts;
  __shared__ float red[2][32];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= p.R) return;
  const int r = (int)row, D = (int)p.D, packs = D / W, tid = threadIdx.x;
  const int q0 = (tid >> 5) * 32 * NV + (tid & 31), skip = q0 * W;
  const F zero = vset<E::kPer>(0.0f);
  const T *xr = row_at<T>(p.x, r, p.x_sr, skip), *zr = row_at<T>(p.z, r, p.z_sr, skip);
  const T* gr = row_at<T>(p.gate, r, p.gate_kind == MPB_GATE_FULL ? p.g_sr : 0, skip);
  T *yr = const_cast<T*>(row_at<T>(p.y, r, D, skip)), *ur = const_cast<T*>(row_at<T>(p.u, r, D, skip));
  E x[NV], z[NV], g[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int q = q0 + k * 32;
    if (q < packs) {
      const int at = k * 32 * W;
      if (MODE != kPlain) z[k].load(zr + at);
      x[k].load(xr + at);
      if (MODE != kPlain && p.gate_kind == MPB_GATE_FULL) g[k].load(gr + at);
    }
  }
  const KeptRow<W, NV, false> kept_row(p, r, skip);
  F ss = zero, y[NV][NP];
  float rz = 0.0f;
  if (MODE != kPlain) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (q0 + k * 32 < packs)
#pragma unroll
        for (int i = 0; i < NP; ++i) ss = vfma(z[k].get(i), z[k].get(i), ss);
    rz = 1.0f / sqrtf(row_sum(fold(ss), red[0]) / (float)D + p.eps);
    ss = zero;
  }
  const F factor = vset<E::kPer>(rz * (MODE == kDropped ? p.scale * p.drop.up : p.scale));
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int q = q0 + k * 32;
    if (q < packs) {
      if (MODE == kPlain) {
#pragma unroll
        for (int i = 0; i < NP; ++i) y[k][i] = x[k].get(i);
      } else {
        F w[NP];
        load_floats<T, W>(p.w_post + q * W, w);
        E out;
        F v[NP], slope[NP];
        gate_pack<T, W>(p, g[k], r, q * W, v, slope);
        auto branch = [&](auto kept) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            y[k][i] = kept(i, vfma(vmul(z[k].get(i), w[i]), vmul(v[i], factor), x[k].get(i)), x[k].get(i));
            out.put(i, y[k][i]);
          }
        };
        if constexpr (MODE == kDropped) {
          const Kept<W> kept = kept_row.at(p, r, k, q * W);
          branch([&](int i, F a, F b) { return kept.pick(p.drop, i, a, b); });
        } else {
          branch([](int, F a, F) { return a; });
        }
        out.store(yr + k * 32 * W);
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) ss = vfma(y[k][i], y[k][i], ss);
    }
  }
  const float ry = 1.0f / sqrtf(row_sum(fold(ss), red[1]) / (float)D + p.eps);
  const F up = vset<E::kPer>(ry);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int q = q0 + k * 32;
    if (q < packs) {
      F w[NP];
      load_floats<T, W>(p.w_pre + q * W, w);
      E out;
#pragma unroll
      for (int i = 0; i < NP; ++i) out.put(i, vmul(vmul(y[k][i], up), w[i]));
      out.store(ur + k * 32 * W);
    }
  }
  if (tid == 0) {
    if (MODE != kPlain) p.rstd_out[r] = rz;
    p.rstd_out[(MODE != kPlain ? p.R : 0) + r] = ry;
  }
}

// A thread's column sums in shared memory: W floats of each of its packs, in
// groups of four so that neighbouring threads touch neighbouring banks. Adds
// v * by.
template <class T, int W>
MPB_D void add_columns(float* acc, int slots, int q, const typename Elems<T, W>::F (&v)[Elems<T, W>::kParts],
                       typename Elems<T, W>::F by) {
  if constexpr (W % 4 == 0) {
#pragma unroll
    for (int k = 0; k < W / 4; ++k) {
      float4* a = reinterpret_cast<float4*>(acc) + k * slots + q;
      const float4 f = *a;
      const float2 lo = vfma(v[2 * k], by, make_float2(f.x, f.y)), hi = vfma(v[2 * k + 1], by, make_float2(f.z, f.w));
      *a = make_float4(lo.x, lo.y, hi.x, hi.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) acc[j * slots + q] = fmaf(vget(v[0], j), vget(by, j), acc[j * slots + q]);
  }
}
// Where column c of a row lies among `slots` packs of W.
template <int W>
MPB_D int column_at(int slots, int c) {
  const int q = c / W, j = c % W;
  return W % 4 == 0 ? ((j / 4) * slots + q) * 4 + j % 4 : j * slots + q;
}

// Rows in turn: blockIdx, blockIdx + grid, ... (times blockDim.y). p.part gets
// the block's column sums: w_pre, w_post, gate per channel, each (grid, D).
// ALL: both gradients are given and every thread has all of its packs.
// Factors that a row's elements share are taken out of the products: with
// s = m r_z the element's work is ez = dx z (0 where dropped),
// dw_post += s ez v, dgate = s ez w slope, wn = dx v w,
// dz = m r_z wn - z r_z^3 m mean(ez v w).
template <class T, int W, int NV, int MODE, bool ALL>
__global__ void __launch_bounds__(kRowThreads) k_norm_bwd_rows(NormArgs p) {
  using E = Elems<T, W>;
  using F = typename E::F;
  constexpr int NP = E::kParts, PW = E::kPer;
  extern __shared__ __align__(16) float columns[];
  __shared__ float red[2][3][32];
  const int D = (int)p.D, packs = D / W, tid = threadIdx.x, step = blockDim.x, slots = step * NV;
  const int q0 = (tid >> 5) * 32 * NV + (tid & 31), skip = q0 * W;
  const int sums = MODE == kPlain ? 1 : p.gate_kind == MPB_GATE_CHANNEL ? 3 : 2;
  const F zero = vset<PW>(0.0f), one = vset<PW>(1.0f);
  float* acc = columns + (size_t)threadIdx.y * sums * slots * W;
  for (int i = tid; i < sums * slots * W; i += step) acc[i] = 0.0f;
  if (step == 32) __syncwarp();
  else __syncthreads();
  int side = 0;
  for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < p.R;
       row += (int64_t)gridDim.x * blockDim.y, side ^= 1) {
    const int r = (int)row;
    const T *dyr = row_at<T>(p.dy, r, p.dy_sr, skip), *dur = row_at<T>(p.du, r, p.du_sr, skip);
    const T *yr = row_at<T>(p.yin, r, p.y_sr, skip), *zr = row_at<T>(p.z, r, p.z_sr, skip);
    const T* gr = row_at<T>(p.gate, r, p.gate_kind == MPB_GATE_FULL ? p.g_sr : 0, skip);
    E du[NV], y[NV], dy[NV], z[NV], g[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (ALL || q0 + k * 32 < packs) {
        const int at = k * 32 * W;
        if (ALL || p.du) {
          du[k].load(dur + at);
          y[k].load(yr + at);
        }
        if (ALL || p.dy) dy[k].load(dyr + at);
        if (MODE != kPlain) {
          z[k].load(zr + at);
          if (p.gate_kind == MPB_GATE_FULL) g[k].load(gr + at);
        }
      }
    const float rz = MODE != kPlain ? p.rstd[r] : 0.0f, ry = p.rstd[(MODE != kPlain ? p.R : 0) + r];
    const KeptRow<W, NV, MODE == kDropped> kept_row(p, r, skip);
    float back = 0.0f;  // of y in dx: r_y^3 mean(y w du)
    if (ALL || p.du) {
      F dot = zero;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int q = q0 + k * 32;
        if (ALL || q < packs) {
          F w[NP], c[NP];
          load_floats<T, W>(p.w_pre + q * W, w);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            c[i] = vmul(du[k].get(i), y[k].get(i));
            dot = vfma(c[i], w[i], dot);
          }
          add_columns<T, W>(acc, slots, q, c, vset<PW>(ry));
        }
      }
      back = ry * ry * (ry * (row_sum(fold(dot), red[side][0]) / (float)D));
    }
    const float m = MODE == kDropped ? p.scale * p.drop.up : p.scale, s = m * rz;
    F dotz = zero, dgr = zero, wn[NV][NP];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = q0 + k * 32;
      if (ALL || q < packs) {
        F dx[NP];
        E out;
#pragma unroll
        for (int i = 0; i < NP; ++i) dx[i] = ALL || p.dy ? dy[k].get(i) : zero;
        if (ALL || p.du) {
          F w[NP];
          load_floats<T, W>(p.w_pre + q * W, w);
#pragma unroll
          for (int i = 0; i < NP; ++i)
            dx[i] = vfma(vmul(du[k].get(i), w[i]), vset<PW>(ry), vfma(y[k].get(i), vset<PW>(-back), dx[i]));
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) out.put(i, dx[i]);
        out.store(const_cast<T*>(row_at<T>(p.dx, r, D, skip)) + k * 32 * W);
        if (MODE != kPlain) {
          F w[NP], ezv[NP], dg[NP], v[NP], slope[NP];
          load_floats<T, W>(p.w_post + q * W, w);
          gate_pack<T, W>(p, g[k], r, q * W, v, slope);
          auto branch = [&](auto kept) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              const F ez = vmul(dx[i], z[k].get(i)), dxv = kept(i, vmul(dx[i], v[i])), dgi = vmul(vmul(ez, w[i]), slope[i]);
              ezv[i] = vmul(dxv, z[k].get(i));
              wn[k][i] = vmul(dxv, w[i]);
              dg[i] = kept(i, vmul(dgi, vset<PW>(s)));
              dotz = vfma(ezv[i], w[i], dotz);
              dgr = vadd(dgr, dg[i]);
            }
          };
          if constexpr (MODE == kDropped) {
            const Kept<W> kept = kept_row.at(p, r, k, q * W);
            branch([&](int i, F a) { return kept.pick(p.drop, i, a, zero); });
          } else {
            branch([](int, F a) { return a; });
          }
          add_columns<T, W>(acc + slots * W, slots, q, ezv, vset<PW>(s));
          if (p.gate_kind == MPB_GATE_FULL) {
#pragma unroll
            for (int i = 0; i < NP; ++i) out.put(i, dg[i]);
            out.store(const_cast<T*>(row_at<T>(p.dgate, r, D, skip)) + k * 32 * W);
          } else if (p.gate_kind == MPB_GATE_CHANNEL) {
            add_columns<T, W>(acc + 2 * slots * W, slots, q, dg, one);
          }
        }
      }
    }
    if (MODE != kPlain) {
      const float mz = rz * rz * (s * (row_sum(fold(dotz), red[side][1]) / (float)D));
      if (p.gate_kind == MPB_GATE_ROW) {
        const float sum = row_sum(fold(dgr), red[side][2]);
        if (tid == 0) ((T*)p.dgate)[r] = Cvt<T>::from(sum);
      }
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int q = q0 + k * 32;
        if (ALL || q < packs) {
          E out;
#pragma unroll
          for (int i = 0; i < NP; ++i)
            out.put(i, vfma(z[k].get(i), vset<PW>(-mz), vmul(wn[k][i], vset<PW>(s))));
          out.store(const_cast<T*>(row_at<T>(p.dz, r, D, skip)) + k * 32 * W);
        }
      }
    }
  }
  // the block's sums over its rows of threads, in order
  __syncthreads();
  const int threads = blockDim.x * blockDim.y, me = threadIdx.y * blockDim.x + threadIdx.x;
  for (int s = 0; s < sums; ++s)
    for (int c = me; c < D; c += threads) {
      const int at = s * slots * W + column_at<W>(slots, c);
      float v = 0.0f;
      for (int yy = 0; yy < (int)blockDim.y; ++yy) v += columns[(size_t)yy * sums * slots * W + at];
      p.part[((size_t)s * gridDim.x + blockIdx.x) * D + c] = v;
    }
}

// Adds the blocks' column sums: 32 columns per block, its 32 warps a part of the
// blocks each, in a fixed order.
template <class T>
__global__ void __launch_bounds__(1024) k_norm_columns(NormArgs p, int blocks) {
  __shared__ float part[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x, s = blockIdx.y;
  float v = 0.0f;
  if (c < p.D)
    for (int b = threadIdx.y; b < blocks; b += 32) v += p.part[((size_t)s * blocks + b) * p.D + c];
  part[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = warp_sum(part[threadIdx.x][threadIdx.y]);
  const int mine = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x != 0 || mine >= p.D) return;
  if (s == 0) p.dw_pre[mine] = v;
  else if (s == 1) p.dw_post[mine] = v;
  else ((T*)p.dgate)[mine] = Cvt<T>::from(v);
}

// ------------------------------------------------------------------- host
// How a row is spread: W elements per pack, NV packs per thread.
struct Spread {
  int W, NV;
  unsigned x, y;  // threads per row, rows per block
};

// W: 8 where every row of every operand starts on a 16-byte boundary and D is
// a multiple of 8, else 2 (16-bit types on 4-byte boundaries) or 1. With fewer
// rows than SMs a row takes as many threads as it has packs (a row's latency
// counts); else a thread takes 32 elements forward and 16 (of float 8) backward
// or of narrow packs, what its 128 registers hold, and up to 32 again where 512
// threads need them.
Spread spread_of(int64_t R, int64_t D, int W, bool backward, int size) {
  Spread s;
  s.W = W;
  const int64_t packs = D / W;
  const bool few = R < sm_count();
  const int least = W == 1 ? 8 : W == 2 ? 8 : 1, usual = W == 8 ? (backward ? 4 / size : 4) : 16 / W;
  s.NV = few ? least : packs <= 32 * least ? least : packs <= 64 && W == 8 ? (2 < usual ? 2 : usual) : usual;
  while (s.NV * W < kPerThread && packs > (int64_t)s.NV * kRowThreads) s.NV *= 2;
  const int64_t threads = (packs + s.NV - 1) / s.NV;
  s.x = (unsigned)((threads + 31) / 32 * 32);
  s.y = s.x == 32 && !few ? 4 : 1;
  return s;
}

int sums_of(int mode, int gate_kind) { return mode == kPlain ? 1 : gate_kind == MPB_GATE_CHANNEL ? 3 : 2; }

// Blocks of the backward kernel: what fits the SMs at 128 registers per thread
// (half of that with one pack) and by shared memory, or the rows if they are
// fewer.
int64_t bwd_blocks(const Spread& s, int64_t R, int sums, size_t* smem) {
  *smem = (size_t)s.x * s.NV * s.W * s.y * sizeof(float) * sums;
  int64_t per_sm = (s.NV == 1 ? 2 : 1) * kRowThreads / (s.x * s.y);
  const int64_t by_smem = (int64_t)((224u << 10) / (*smem + 2048));
  if (per_sm > by_smem) per_sm = by_smem;
  if (per_sm < 1) per_sm = 1;
  const int64_t most = per_sm * sm_count(), want = (R + s.y - 1) / s.y;
  return want < most ? want : most;
}

template <class T, int W, int NV, int MODE>
int run_rows(const NormArgs& p, const Spread& sp, bool backward, cudaStream_t s) {
  const dim3 block(sp.x, sp.y);
  if (!backward) {
    k_norm_rows<T, W, NV, MODE><<<(unsigned)((p.R + sp.y - 1) / sp.y), block, 0, s>>>(p);
    return launch_check("gated_residual_norm");
  }
  const char* what = "gated_residual_norm_backward";
  const int sums = sums_of(MODE, p.gate_kind);
  size_t smem;
  const int64_t blocks = bwd_blocks(sp, p.R, sums, &smem);
  auto run = [&](auto all) {
    constexpr auto kernel = k_norm_bwd_rows<T, W, NV, MODE, decltype(all)::value>;
    constexpr int most = kRowThreads * NV * W * (int)sizeof(float) * (MODE == kPlain ? 1 : 3);
    if (int rc = allow_smem<kernel, most>(what)) return rc;
    kernel<<<(unsigned)blocks, block, smem, s>>>(p);
    return (int)MPB_OK;
  };
  const bool all = W == 8 && p.du && p.dy && p.D == (int64_t)W * NV * sp.x;
  if (int rc = all ? run(std::integral_constant<bool, W == 8>()) : run(std::false_type())) return rc;
  if (int rc = launch_check(what)) return rc;
  k_norm_columns<T><<<dim3((unsigned)((p.D + 31) / 32), (unsigned)sums), dim3(32, 32), 0, s>>>(p, (int)blocks);
  return launch_check(what);
}

template <class T, int MODE>
int run_spread(const NormArgs& p, const Spread& sp, bool backward, cudaStream_t s) {
  if (sp.W == 8)
    return sp.NV == 1   ? run_rows<T, 8, 1, MODE>(p, sp, backward, s)
           : sp.NV == 2 ? run_rows<T, 8, 2, MODE>(p, sp, backward, s)
                        : run_rows<T, 8, 4, MODE>(p, sp, backward, s);
  if constexpr (sizeof(T) == 2)
    if (sp.W == 2) return sp.NV == 8 ? run_rows<T, 2, 8, MODE>(p, sp, backward, s) : run_rows<T, 2, 16, MODE>(p, sp, backward, s);
  return sp.NV == 8    ? run_rows<T, 1, 8, MODE>(p, sp, backward, s)
         : sp.NV == 16 ? run_rows<T, 1, 16, MODE>(p, sp, backward, s)
                       : run_rows<T, 1, 32, MODE>(p, sp, backward, s);
}

// Elements per pack that every operand's rows allow.
int width_of(const NormArgs& p, size_t size) {
  const void* ptr[] = {p.x, p.z, p.gate_kind == MPB_GATE_FULL ? p.gate : nullptr, p.dy, p.du, p.yin, p.y, p.u, p.dx, p.dz,
                       p.gate_kind == MPB_GATE_FULL ? p.dgate : nullptr};
  const int64_t st[] = {p.x ? p.x_sr : 0, p.z ? p.z_sr : 0, p.gate_kind == MPB_GATE_FULL ? p.g_sr : 0, p.dy ? p.dy_sr : 0,
                        p.du ? p.du_sr : 0, p.yin ? p.y_sr : 0, p.D};
  const void* weights[] = {p.w_pre, p.w_post};
  auto fits = [&](size_t bytes) {
    for (const void* q : ptr)
      if ((uintptr_t)q % bytes) return false;
    for (int64_t v : st)
      if (v * (int64_t)size % (int64_t)bytes) return false;
    return true;
  };
  bool w16 = true;
  for (const void* q : weights) w16 = w16 && (uintptr_t)q % 16 == 0;
  if (p.D % 8 == 0 && w16 && fits(16)) return 8;
  return size == 2 && p.D % 2 == 0 && fits(4) ? 2 : 1;
}

template <class T>
int launch_rows(const NormArgs& p, bool backward, cudaStream_t s) {
  const Spread sp = spread_of(p.R, p.D, width_of(p, sizeof(T)), backward, (int)sizeof(T));
  return !p.z         ? run_spread<T, kPlain>(p, sp, backward, s)
         : p.dropping ? run_spread<T, kDropped>(p, sp, backward, s)
                      : run_spread<T, kBranch>(p, sp, backward, s);
}

template <class T>
int launch_norm_fwd(const NormArgs& p, cudaStream_t s) {
  if (p.D <= kInRegisters) return launch_rows<T>(p, false, s);
  k_norm_long<T><<<(unsigned)p.R, kThreads, 0, s>>>(p);
  return launch_check("gated_residual_norm");
}

template <class T>
int launch_norm_bwd(const NormArgs& p, cudaStream_t s) {
  const char* what = "gated_residual_norm_backward";
  if (p.R > 0 && p.D <= kInRegisters) return launch_rows<T>(p, true, s);
  if (p.R > 0) {
    k_norm_bwd_long<T><<<(unsigned)p.R, kThreads, 0, s>>>(p);
    if (int rc = launch_check(what)) return rc;
    if (p.z) {
      k_norm_bwd_long_dx<T><<<(unsigned)p.R, kThreads, 0, s>>>(p);
      if (int rc = launch_check(what)) return rc;
    }
  }
  k_norm_bwd_long_cols<T><<<(unsigned)((p.D + 127) / 128), 128, 0, s>>>(p);
  return launch_check(what);
}

int check_norm(const char* what, const NormArgs& p, double dropout) {
  if (p.R < 0 || p.D < 0) return fail(MPB_ERR_SHAPE, "%s: negative extent", what);
  if (p.R > 0x7fffffffLL) return fail(MPB_ERR_SHAPE, "%s: %lld rows", what, (long long)p.R);
  if (p.gate_kind < MPB_GATE_NONE || p.gate_kind > MPB_GATE_CHANNEL)
    return fail(MPB_ERR_INVALID, "%s: unknown gate kind %d", what, p.gate_kind);
  if (p.gate_kind != MPB_GATE_NONE && (!p.gate || !p.z)) return fail(MPB_ERR_INVALID, "%s: null gate or branch", what);
  if (p.act < MPB_ACT_LINEAR || p.act > MPB_ACT_SILU) return fail(MPB_ERR_INVALID, "%s: unknown activation %d", what, p.act);
  if (!(dropout >= 0.0 && dropout <= 1.0))
    return fail(MPB_ERR_INVALID, "%s: dropout %g outside [0, 1]", what, dropout);
  if (p.z && !p.w_post) return fail(MPB_ERR_INVALID, "%s: null w_post", what);
  for (int64_t sr : {p.x_sr, p.z_sr, p.g_sr, p.dy_sr, p.du_sr, p.y_sr})
    if (p.R > 1 && (sr <= -kMostStride || sr >= kMostStride))
      return fail(MPB_ERR_SHAPE, "%s: row stride of %lld elements", what, (long long)sr);
  return MPB_OK;
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" {

int mpb_gated_residual_norm(int64_t R, int64_t D, int dtype, const void* x, int64_t x_sr, const void* z, int64_t z_sr,
                            const void* gate, int64_t g_sr, int gate_kind, int activation, const float* w_post,
                            const float* w_pre, double scale, double eps, double dropout, uint64_t seed,
                            uint64_t offset, void* y, void* u, float* rstd, mpb_stream_t stream) {
  NormArgs p = {};
  p.R = R, p.D = D, p.x = x, p.x_sr = x_sr, p.z = z, p.z_sr = z_sr, p.gate = gate, p.g_sr = g_sr;
  p.gate_kind = gate_kind, p.act = activation, p.w_post = w_post, p.w_pre = w_pre;
  p.scale = (float)scale, p.eps = (float)eps, p.y = y, p.u = u, p.rstd_out = rstd;
  if (int rc = check_norm("gated_residual_norm", p, dropout)) return rc;
  p.drop = make_dropper(dropout, seed, offset);
  p.dropping = p.drop.drop != 0;
  if (dtype != MPB_F32 && dtype != MPB_F16 && dtype != MPB_BF16)
    return fail(MPB_ERR_DTYPE, "gated_residual_norm: dtype %d not supported (float16, bfloat16, float32)", dtype);
  if (R == 0) return MPB_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (D == 0) {  // the factors of a mean of nothing: NaN, which all bits set are
    if (!rstd) return fail(MPB_ERR_INVALID, "gated_residual_norm: null pointer");
    return cuda_check(cudaMemsetAsync(rstd, 0xff, (size_t)R * (z ? 2 : 1) * sizeof(float), s), "gated_residual_norm");
  }
  if (!x || !w_pre || !u || !rstd || (z && !y)) return fail(MPB_ERR_INVALID, "gated_residual_norm: null pointer");
  return dtype == MPB_F32 ? launch_norm_fwd<float>(p, s)
                          : dtype == MPB_F16 ? launch_norm_fwd<__half>(p, s) : launch_norm_fwd<__nv_bfloat16>(p, s);
}

size_t mpb_gated_residual_norm_scratch_bytes(int64_t R, int64_t D, int dtype, int branch, int gate_kind) {
  if (R <= 0 || D <= 0) return 0;
  if (D > kInRegisters) return branch ? (size_t)R * (size_t)D * sizeof(float) : 0;
  const int sums = sums_of(branch ? kBranch : kPlain, gate_kind);
  int64_t most = 0;  // blocks, for any width the addresses may allow
  for (int W : {8, 2, 1}) {
    size_t smem;
    const Spread sp = spread_of(R, (D + W - 1) / W * W, W, true, dtype == MPB_F32 ? 4 : 2);
    const int64_t n = bwd_blocks(sp, R, sums, &smem);
    most = n > most ? n : most;
  }
  return (size_t)most * sums * (size_t)D * sizeof(float);
}

int mpb_gated_residual_norm_backward(int64_t R, int64_t D, int dtype, const void* dy, int64_t dy_sr, const void* du,
                                     int64_t du_sr, const void* y, int64_t y_sr, const void* z, int64_t z_sr,
                                     const void* gate, int64_t g_sr, int gate_kind, int activation,
                                     const float* w_post, const float* w_pre, const float* rstd, double scale,
                                     double dropout, uint64_t seed, uint64_t offset, void* dx, void* dz, void* dgate,
                                     float* dw_post, float* dw_pre, void* scratch, size_t scratch_bytes,
                                     mpb_stream_t stream) {
  const char* what = "gated_residual_norm_backward";
  NormArgs p = {};
  p.R = R, p.D = D, p.dy = dy, p.dy_sr = dy_sr, p.du = du, p.du_sr = du_sr, p.yin = y, p.y_sr = y_sr;
  p.z = z, p.z_sr = z_sr, p.gate = gate, p.g_sr = g_sr, p.gate_kind = gate_kind, p.act = activation;
  p.w_post = w_post, p.w_pre = w_pre, p.rstd = rstd, p.scale = (float)scale;
  p.dx = dx, p.dz = dz, p.dgate = dgate, p.dw_post = dw_post, p.dw_pre = dw_pre, p.part = (float*)scratch;
  if (int rc = check_norm(what, p, dropout)) return rc;
  p.drop = make_dropper(dropout, seed, offset);
  p.dropping = p.drop.drop != 0;
  if (dtype != MPB_F32 && dtype != MPB_F16 && dtype != MPB_BF16)
    return fail(MPB_ERR_DTYPE, "%s: dtype %d not supported (float16, bfloat16, float32)", what, dtype);
  cudaStream_t s = (cudaStream_t)stream;
  if (D == 0) {  // a gate per row has the sum over no channels as its gradient
    if (gate_kind != MPB_GATE_ROW || R == 0) return MPB_OK;
    if (!dgate) return fail(MPB_ERR_INVALID, "%s: null pointer", what);
    return cuda_check(cudaMemsetAsync(dgate, 0, (size_t)R * (dtype == MPB_F32 ? 4 : 2), s), what);
  }
  if (!dw_pre || (z && !dw_post) || (gate_kind != MPB_GATE_NONE && !dgate) || !w_pre)
    return fail(MPB_ERR_INVALID, "%s: null pointer", what);
  if (R > 0 && (!y || !rstd || !dx || (z && !dz))) return fail(MPB_ERR_INVALID, "%s: null pointer", what);
  const size_t need = mpb_gated_residual_norm_scratch_bytes(R, D, dtype, z != nullptr, gate_kind);
  if (need > scratch_bytes || (need && !scratch))
    return fail(MPB_ERR_SCRATCH, "%s: %zu bytes of scratch, %zu needed", what, scratch_bytes, need);
  return dtype == MPB_F32 ? launch_norm_bwd<float>(p, s)
                          : dtype == MPB_F16 ? launch_norm_bwd<__half>(p, s) : launch_norm_bwd<__nv_bfloat16>(p, s);
}

}  // extern "C"

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
// Bound: memory.
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

constexpr int kThreads = 256;

MPB_D void act_of(int act, float g, float& v, float& slope) {
  if (act == MPB_ACT_LINEAR) {
    v = g;
    slope = 1.0f;
    return;
  }
  float s, om;
  sigmoid2(g, s, om);
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
      if (p.gate_kind != MPB_GATE_NONE) act_of(p.act, gate_at<T>(p, r, c), v, slope);
      y += m * v * (to_f(((const T*)p.z)[r * p.z_sr + c]) * rz * p.w_post[c]);
    }
  }
  return y;
}

// One block per row.
template <class T>
__global__ void __launch_bounds__(kThreads) k_norm_fwd(NormArgs p) {
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

// One block per row: the row's gradients.
template <class T>
__global__ void __launch_bounds__(kThreads) k_norm_bwd(NormArgs p) {
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
    if (p.gate_kind != MPB_GATE_NONE) act_of(p.act, gate_at<T>(p, r, c), v, slope);
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
    if (p.gate_kind != MPB_GATE_NONE) act_of(p.act, gate_at<T>(p, r, c), v, slope);
    const float dn = m == 0.0f ? 0.0f : dx_at(c) * m * v;
    ((T*)p.dz)[r * p.D + c] = Cvt<T>::from(rz * (dn * p.w_post[c] - to_f(z[c]) * rz * mz));
  }
}

// One thread per column: the gradients of the weights and of a gate per channel. dx is read back
// from where the row kernel left it.
template <class T>
__global__ void k_norm_bwd_cols(NormArgs p) {
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
    if (p.gate_kind != MPB_GATE_NONE) act_of(p.act, gate_at<T>(p, r, c), v, slope);
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
__global__ void __launch_bounds__(kThreads) k_norm_bwd_dx(NormArgs p) {
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

template <class T>
int launch_norm_fwd(const NormArgs& p, cudaStream_t s) {
  k_norm_fwd<T><<<(unsigned)p.R, kThreads, 0, s>>>(p);
  return launch_check("gated_residual_norm");
}

template <class T>
int launch_norm_bwd(const NormArgs& p, cudaStream_t s) {
  if (p.R > 0) {
    k_norm_bwd<T><<<(unsigned)p.R, kThreads, 0, s>>>(p);
    if (int rc = launch_check("gated_residual_norm_backward")) return rc;
    if (p.z) {
      k_norm_bwd_dx<T><<<(unsigned)p.R, kThreads, 0, s>>>(p);
      if (int rc = launch_check("gated_residual_norm_backward")) return rc;
    }
  }
  k_norm_bwd_cols<T><<<(unsigned)((p.D + 127) / 128), 128, 0, s>>>(p);
  return launch_check("gated_residual_norm_backward");
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
  if (R == 0 || D == 0) return MPB_OK;
  if (!x || !w_pre || !u || !rstd || (z && !y)) return fail(MPB_ERR_INVALID, "gated_residual_norm: null pointer");
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == MPB_F32 ? launch_norm_fwd<float>(p, s)
                          : dtype == MPB_F16 ? launch_norm_fwd<__half>(p, s) : launch_norm_fwd<__nv_bfloat16>(p, s);
}

size_t mpb_gated_residual_norm_scratch_bytes(int64_t R, int64_t D, int dtype, int branch, int gate_kind) {
  return branch ? (size_t)R * (size_t)D * sizeof(float) : 0;
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
  if (D == 0) return MPB_OK;
  if (!dw_pre || (z && !dw_post) || (gate_kind != MPB_GATE_NONE && !dgate) || !w_pre)
    return fail(MPB_ERR_INVALID, "%s: null pointer", what);
  if (R > 0 && (!y || !rstd || !dx || (z && !dz))) return fail(MPB_ERR_INVALID, "%s: null pointer", what);
  const size_t need = mpb_gated_residual_norm_scratch_bytes(R, D, dtype, z != nullptr, gate_kind);
  if (need > scratch_bytes || (need && !scratch))
    return fail(MPB_ERR_SCRATCH, "%s: %zu bytes of scratch, %zu needed", what, scratch_bytes, need);
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == MPB_F32 ? launch_norm_bwd<float>(p, s)
                          : dtype == MPB_F16 ? launch_norm_bwd<__half>(p, s) : launch_norm_bwd<__nv_bfloat16>(p, s);
}

}  // extern "C"

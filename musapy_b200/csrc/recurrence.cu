// Gated linear recurrence along time, forward and backward, and its
// single-token step. For every sequence b and channel d (no counterpart in
// the reference, whose only scan is cumsum):
//
//   a[t] = gate[t]            b[t] = x[t]               (linear)
//   a[t] = sigmoid(gate[t])   b[t] = (1 - a[t]) x[t]    (sigmoid)
//   h[t] = a[t] h[t-1] + b[t],   h[-1] = h0
//
// and backward, with the gradients dh of every h[t] and dstate of the last:
//
//   s[t] = dh[t] + u[t+1],   u[t] = a[t] s[t],   u[T] = dstate,   dh0 = u[0]
//   linear:  dx = s             da = s h[t-1]
//   sigmoid: dx = (1 - a) s     da = s (h[t-1] - x[t]),   dgate = da a (1 - a)
//
// The gate of channel d is number d / (D / H) of H per time step; the gradient
// of a shared gate sums over its channels in a fixed order. The state runs in
// float whatever the element type.
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "rows.cuh"

namespace mpb {
namespace {

struct ScanArgs {
  int64_t B, T, D, H, P;  // P = D / H channels per gate
  const void *x, *gate, *dh, *hsaved;
  int64_t x_sb, x_st, g_sb, g_st, dh_sb, dh_st, h_sb, h_st;  // strides over batch and time, elements
  const float *h0, *dstate;                                  // (B, D) or null
  void* h;                                                   // (B, T, D)
  float* state;                                              // (B, D) or null
  void *dx, *dgate;                                          // (B, T, D), (B, T, H)
  float* dh0;                                                // (B, D) or null
  float* part;                                               // (B, T, H) sums of heads wider than a block
};

constexpr int kThreads = 128;

template <class G, bool SIG>
MPB_D void gate_of(G g, float& a, float& om) {
  if (SIG) {
    sigmoid2(to_f(g), a, om);
  } else {
    a = to_f(g);
    om = 1.0f;
  }
}

// One thread per channel, in time order.
template <class X, class G, bool SIG>
__global__ void __launch_bounds__(kThreads) k_gscan(ScanArgs p) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= p.B * p.D) return;
  const int64_t b = i / p.D, d = i - b * p.D;
  const X* x = (const X*)p.x + b * p.x_sb + d;
  const G* g = (const G*)p.gate + b * p.g_sb + d / p.P;
  X* h = (X*)p.h + b * p.T * p.D + d;
  float s = p.h0 ? p.h0[i] : 0.0f;
#pragma unroll 4
  for (int64_t t = 0; t < p.T; ++t) {
    float a, om;
    gate_of<G, SIG>(g[t * p.g_st], a, om);
    const float v = to_f(x[t * p.x_st]);
    s = SIG ? fmaf(a, s, om * v) : fmaf(a, s, v);
    h[t * p.D] = Cvt<X>::from(s);
  }
  if (p.state) p.state[i] = s;
}

// One block per (sequence, head), its threads over the head's channels, in reverse time order.
template <class X, class G, bool SIG>
__global__ void __launch_bounds__(kThreads) k_gscan_bwd(ScanArgs p) {
  __shared__ float red[2][32];
  const int64_t b = blockIdx.x / p.H, head = blockIdx.x - b * p.H;
  const G* g = (const G*)p.gate + b * p.g_sb + head;
  G* dg = (G*)p.dgate + b * p.T * p.H + head;
  int side = 0;
  for (int64_t c0 = 0; c0 < p.P; c0 += kThreads) {
    const int64_t c = c0 + threadIdx.x, d = head * p.P + c;
    const bool in = c < p.P;
    float u = in && p.dstate ? p.dstate[b * p.D + d] : 0.0f;
    for (int64_t t = p.T - 1; t >= 0; --t) {
      float a, om, da = 0.0f;
      gate_of<G, SIG>(g[t * p.g_st], a, om);
      if (in) {
        const float s = to_f(((const X*)p.dh)[b * p.dh_sb + t * p.dh_st + d]) + u;
        float before = t > 0 ? to_f(((const X*)p.hsaved)[b * p.h_sb + (t - 1) * p.h_st + d])
                             : (p.h0 ? p.h0[b * p.D + d] : 0.0f);
        if (SIG) before -= to_f(((const X*)p.x)[b * p.x_sb + t * p.x_st + d]);
        da = s * before;
        ((X*)p.dx)[(b * p.T + t) * p.D + d] = Cvt<X>::from(SIG ? om * s : s);
        u = a * s;
      }
      if (p.P > 1) {
        da = block_sum(da, red[side]);
        side ^= 1;
      }
      if (threadIdx.x == 0) {
        if (p.P > kThreads) {  // a head wider than the block: each slice of it adds to what the earlier ones left
          float* part = p.part + (b * p.T + t) * p.H + head;
          if (c0) da += *part;
          *part = da;
        }
        if (c0 + kThreads >= p.P) dg[t * p.H] = Cvt<G>::from(SIG ? da * (a * om) : da);
      }
    }
    if (in && p.dh0) p.dh0[b * p.D + d] = u;
  }
}

template <class X, class G, bool SIG>
int launch_fwd(const ScanArgs& p, cudaStream_t s) {
  const int64_t n = p.B * p.D;
  k_gscan<X, G, SIG><<<(unsigned)((n + kThreads - 1) / kThreads), kThreads, 0, s>>>(p);
  return launch_check("gated_scan");
}

template <class X, class G, bool SIG>
int launch_bwd(const ScanArgs& p, cudaStream_t s) {
  k_gscan_bwd<X, G, SIG><<<(unsigned)(p.B * p.H), kThreads, 0, s>>>(p);
  return launch_check("gated_scan_backward");
}

// Calls f<X, G, SIG>() for the element types; false when the pair is not supported.
template <class F>
int by_types(const char* what, int x_dt, int g_dt, int mode, F f) {
  if (mode != MPB_SCAN_LINEAR && mode != MPB_SCAN_SIGMOID) return fail(MPB_ERR_INVALID, "%s: unknown mode %d", what, mode);
  const bool sig = mode == MPB_SCAN_SIGMOID;
#define MPB_SCAN_CASE(XD, GD)                                                                  \
  if (x_dt == XD && g_dt == GD)                                                                \
    return sig ? f(Storage<XD>::type(), Storage<GD>::type(), std::integral_constant<bool, true>()) \
               : f(Storage<XD>::type(), Storage<GD>::type(), std::integral_constant<bool, false>());
  MPB_SCAN_CASE(MPB_F32, MPB_F32)
  MPB_SCAN_CASE(MPB_F16, MPB_F16)
  MPB_SCAN_CASE(MPB_F16, MPB_F32)
  MPB_SCAN_CASE(MPB_BF16, MPB_BF16)
  MPB_SCAN_CASE(MPB_BF16, MPB_F32)
#undef MPB_SCAN_CASE
  return fail(MPB_ERR_DTYPE, "%s: x dtype %d with gate dtype %d not supported", what, x_dt, g_dt);
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t D, int64_t H) {
  if (B < 0 || T < 0 || D < 0 || H < 0) return fail(MPB_ERR_SHAPE, "%s: negative extent", what);
  if (D > 0 && (H < 1 || D % H != 0))
    return fail(MPB_ERR_SHAPE, "%s: %lld gates do not divide %lld channels", what, (long long)H, (long long)D);
  if (B * H > 0x7fffffffLL) return fail(MPB_ERR_SHAPE, "%s: %lld sequences x gates", what, (long long)(B * H));
  return MPB_OK;
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" {

size_t mpb_gated_scan_scratch_bytes(int64_t B, int64_t T, int64_t D, int64_t H, int x_dtype, int gate_dtype,
                                    int backward) {
  return backward && H > 0 && D / H > kThreads ? (size_t)(B * T * H) * sizeof(float) : 0;
}

int mpb_gated_scan(int64_t B, int64_t T, int64_t D, int64_t H, const void* x, int x_dtype, int64_t x_sb, int64_t x_st,
                   const void* gate, int gate_dtype, int64_t g_sb, int64_t g_st, const float* h0, int mode, void* h,
                   float* state, void* scratch, size_t scratch_bytes, mpb_stream_t stream) {
  if (int rc = check_sizes("gated_scan", B, T, D, H)) return rc;
  ScanArgs p = {};
  p.B = B, p.T = T, p.D = D, p.H = H, p.P = H ? D / H : 1;
  p.x = x, p.x_sb = x_sb, p.x_st = x_st, p.gate = gate, p.g_sb = g_sb, p.g_st = g_st;
  p.h0 = h0, p.h = h, p.state = state;
  return by_types("gated_scan", x_dtype, gate_dtype, mode, [&](auto xt, auto gt, auto sig) {
    if (B * D == 0) return (int)MPB_OK;
    if (T > 0 && (!x || !gate || !h)) return fail(MPB_ERR_INVALID, "gated_scan: null pointer");
    return launch_fwd<decltype(xt), decltype(gt), decltype(sig)::value>(p, (cudaStream_t)stream);
  });
}

int mpb_gated_scan_backward(int64_t B, int64_t T, int64_t D, int64_t H, const void* dh, int64_t dh_sb, int64_t dh_st,
                            const void* x, int x_dtype, int64_t x_sb, int64_t x_st, const void* gate, int gate_dtype,
                            int64_t g_sb, int64_t g_st, const void* h, int64_t h_sb, int64_t h_st, const float* h0,
                            const float* dstate, int mode, void* dx, void* dgate, float* dh0, void* scratch,
                            size_t scratch_bytes, mpb_stream_t stream) {
  if (int rc = check_sizes("gated_scan_backward", B, T, D, H)) return rc;
  ScanArgs p = {};
  p.B = B, p.T = T, p.D = D, p.H = H, p.P = H ? D / H : 1;
  p.dh = dh, p.dh_sb = dh_sb, p.dh_st = dh_st, p.x = x, p.x_sb = x_sb, p.x_st = x_st;
  p.gate = gate, p.g_sb = g_sb, p.g_st = g_st, p.hsaved = h, p.h_sb = h_sb, p.h_st = h_st;
  p.h0 = h0, p.dstate = dstate, p.dx = dx, p.dgate = dgate, p.dh0 = dh0, p.part = (float*)scratch;
  const size_t need = mpb_gated_scan_scratch_bytes(B, T, D, H, x_dtype, gate_dtype, 1);
  if (need > scratch_bytes || (need && !scratch))
    return fail(MPB_ERR_SCRATCH, "gated_scan_backward: %zu bytes of scratch, %zu needed", scratch_bytes, need);
  return by_types("gated_scan_backward", x_dtype, gate_dtype, mode, [&](auto xt, auto gt, auto sig) {
    if (B * D == 0) return (int)MPB_OK;
    if (T > 0 && (!dh || !x || !gate || !h || !dx || !dgate))
      return fail(MPB_ERR_INVALID, "gated_scan_backward: null pointer");
    return launch_bwd<decltype(xt), decltype(gt), decltype(sig)::value>(p, (cudaStream_t)stream);
  });
}

int mpb_gated_scan_step(int64_t B, int64_t D, int64_t H, const void* x, int x_dtype, int64_t x_sb, const void* gate,
                        int gate_dtype, int64_t g_sb, int mode, float* state, void* h, mpb_stream_t stream) {
  return mpb_gated_scan(B, 1, D, H, x, x_dtype, x_sb, 0, gate, gate_dtype, g_sb, 0, state, mode, h, state, nullptr, 0,
                        stream);
}

}  // extern "C"

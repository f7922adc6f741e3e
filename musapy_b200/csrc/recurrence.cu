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
//
// One pass over the data, in tiles of 32 lanes x V channels by S x 16 steps.
// A warp holds 16 steps of its channels in registers and folds them to the
// map c -> A c + B that they apply to the state; the block joins the maps of
// its S warps, gets the state that enters the tile, and each warp then runs
// its steps once more from the state that enters them and writes. Where T
// takes several tiles they form a chain: a tile publishes its map, then its
// outgoing state, and takes its incoming state from the nearest earlier tile
// that has published one, applying the maps between them in time order. A
// state passes through the same operations wherever the look-back found it, so
// results do not depend on timing. Tiles are handed out by a ticket, all
// chains' first tiles first, so that a tile waits only for tiles that already
// run, and every wait is bounded. The backward pass is the same walk with time
// reversed, over the map u -> a (u + dh).
//
// Bound: memory.
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "plan.h"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kSteps = 16;               // steps per warp and tile
constexpr int kWarps = 8;                // warps of a full tile
constexpr uint32_t kMap = 1, kState = 2; // what a tile has published

struct ScanArgs {
  int64_t B, T, D, H, P;  // P = D / H channels per gate
  const void *x, *gate, *dh, *hsaved;
  int64_t x_sb, x_st, g_sb, g_st, dh_sb, dh_st, h_sb, h_st;  // strides over batch and time, elements
  const float *h0, *dstate;                                  // (B, D) or null
  void* h;                                                   // (B, T, D)
  float* state;                                              // (B, D) or null
  void *dx, *dgate;                                          // (B, T, D), (B, T, H)
  float* dh0;                                                // (B, D) or null
  // channel groups: a block's 32 lanes
  uint32_t groups;            // per sequence
  uint32_t heads_per, lanes_per, groups_per;  // shared gates: heads per group, lanes per head, groups per head
  uint32_t chains, chunks;    // B * groups, tiles per chain
  FastDiv by_groups, by_groups_per, by_lanes_per, by_chains;
  int steps;                  // of a tile
  // scratch
  uint32_t *ticket, *status, *flags;
  float *map_a, *map_b, *out_state;  // (tiles, channels of a group)
  float* part;                       // (B, T, H, groups_per)
};

template <class G, bool SIG>
MPB_D void gate_of(G g, float& a, float& om) {
  if (SIG) {
    sigmoid2(to_f(g), a, om);
  } else {
    a = to_f(g);
    om = 1.0f;
  }
}

// The state after the map (a, b). A zero state stays out of the product: the
// product of a tile's gates may have overflowed although no state did.
MPB_D float apply(float a, float b, float c) { return c == 0.0f ? b : fmaf(a, c, b); }

// Where a lane works.
struct Lane {
  int64_t b, ch, gate;  // sequence, first channel, its gate
  bool in;
};

template <int V, bool SHARED>
MPB_D Lane place(const ScanArgs& p, uint32_t chain, int lane) {
  uint32_t b, group;
  p.by_groups.divmod(chain, b, group);
  Lane l;
  l.b = b;
  if (!SHARED) {
    l.ch = l.gate = ((int64_t)group * 32 + lane) * V;
    l.in = l.ch < p.D;
  } else if (p.groups_per > 1) {  // a head's channels in several groups
    uint32_t head, part;
    p.by_groups_per.divmod(group, head, part);
    const int64_t c = ((int64_t)part * 32 + lane) * V;
    l.gate = head;
    l.ch = head * p.P + c;
    l.in = c < p.P;
  } else {  // one or several heads in a group
    uint32_t head, at;
    p.by_lanes_per.divmod((uint32_t)lane, head, at);
    l.in = head < p.heads_per && (int64_t)group * p.heads_per + head < p.H;
    l.gate = (int64_t)group * p.heads_per + head;
    l.ch = l.gate * p.P + (int64_t)at * V;
  }
  if (!l.in) l.ch = l.gate = 0;
  return l;
}

MPB_D uint32_t ld_flag(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
MPB_D void st_flag(uint32_t* p, uint32_t v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
MPB_D unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Warp 0 of a tile: the state that enters it, per lane and channel. `first`
// is the state before the chain; (a, b) is the tile's own map, published when
// the tile before has no state yet.
template <int V>
MPB_D void look_back(const ScanArgs& p, uint32_t chain, uint32_t chunk, int lane, const float (&a)[V],
                     const float (&b)[V], float (&carry)[V]) {
  constexpr int C = 32 * V;
  const uint32_t tile = chunk * p.chains + chain;
  auto at = [&](uint32_t k) { return (size_t)(k * p.chains + chain) * C + lane * V; };
  uint32_t back = 0;  // distance - 1 of the nearest tile with a state
  bool found = chunk == 0 || ld_flag(p.flags + tile - p.chains) == kState;
  found = __all_sync(0xffffffffu, found);
  if (!found) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      __stcg(p.map_a + at(chunk) + v, a[v]);
      __stcg(p.map_b + at(chunk) + v, b[v]);
    }
    __threadfence();
    __syncwarp();
    if (lane == 0) st_flag(p.flags + tile, kMap);
    const unsigned long long t0 = now_ns();
    for (;;) {
      // lane i looks at the tile i + 1 before this one; before the chain's
      // first tile stands the initial state
      const uint32_t f = (uint32_t)lane < chunk ? ld_flag(p.flags + tile - (lane + 1) * p.chains) : kState;
      const uint32_t states = __ballot_sync(0xffffffffu, f == kState);
      const uint32_t nothing = __ballot_sync(0xffffffffu, f == 0);
      if (states) {
        back = __ffs(states) - 1;
        if ((nothing & ((1u << back) - 1)) == 0) break;
      }
      const bool late = now_ns() - t0 > 2000000000ull;
      if (__any_sync(0xffffffffu, late)) {  // give up: what follows is marked and NaN
        if (lane == 0) st_flag(p.status, MPB_ERR_TIMEOUT);
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = NAN;
        return;
      }
    }
  }
  __threadfence();
  __syncwarp();
  if (chunk > back)
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = __ldcg(p.out_state + at(chunk - 1 - back) + v);
  for (uint32_t k = chunk - back; k < chunk; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = apply(__ldcg(p.map_a + at(k) + v), __ldcg(p.map_b + at(k) + v), carry[v]);
}

// Joins the maps of the block's warps (a, b: this warp's), gets the state
// `carry` that enters the tile (in: the one before the chain) and returns the
// state that enters the warp's steps.
template <int V>
MPB_D void join(const ScanArgs& p, uint32_t chain, uint32_t chunk, int warp, int lane, const float (&a)[V],
                const float (&b)[V], float (&carry)[V]) {
  constexpr int C = 32 * V;
  __shared__ float sa[kWarps][C], sb[kWarps][C], sc[C];
  const int warps = blockDim.x >> 5;
  if (warps == 1 && p.chunks == 1) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sa[warp][lane * V + v] = a[v];
    sb[warp][lane * V + v] = b[v];
  }
  __syncthreads();
  if (p.chunks > 1) {
    if (warp == 0) {
      float ta[V], tb[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        ta[v] = a[v], tb[v] = b[v];
        for (int w = 1; w < warps; ++w) {
          const float aw = sa[w][lane * V + v];
          tb[v] = apply(aw, sb[w][lane * V + v], tb[v]);
          ta[v] *= aw;
        }
      }
      look_back<V>(p, chain, chunk, lane, ta, tb, carry);
      const uint32_t tile = chunk * p.chains + chain;
      if (chunk + 1 < p.chunks) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          __stcg(p.out_state + (size_t)tile * C + lane * V + v, apply(ta[v], tb[v], carry[v]));
        __threadfence();
        __syncwarp();
        if (lane == 0) st_flag(p.flags + tile, kState);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) sc[lane * V + v] = carry[v];
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = sc[lane * V + v];
  }
  for (int w = 0; w < warp; ++w)
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = apply(sa[w][lane * V + v], sb[w][lane * V + v], carry[v]);
}

// The block's tile: the next ticket, or its index where no tile waits for another.
MPB_D void take_tile(const ScanArgs& p, uint32_t& chain, uint32_t& chunk) {
  uint32_t tile = blockIdx.x;
  if (p.chunks > 1) {
    __shared__ uint32_t mine;
    if (threadIdx.x == 0) mine = atomicAdd(p.ticket, 1u);
    __syncthreads();
    tile = mine;
  }
  p.by_chains.divmod(tile, chunk, chain);
}

template <class X, class G, bool SIG, int V, bool SHARED>
__global__ void __launch_bounds__(kWarps * 32, 2) k_gscan(ScanArgs p) {
  using XP = Pack<X, V>;
  using GP = Pack<G, SHARED ? 1 : V>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t chain, chunk;
  take_tile(p, chain, chunk);
  const Lane l = place<V, SHARED>(p, chain, lane);
  const int64_t t0 = (int64_t)chunk * p.steps + warp * kSteps;
  const int n = l.in ? (int)(p.T - t0 < kSteps ? p.T - t0 : kSteps) : 0;
  const X* x = (const X*)p.x + l.b * p.x_sb + t0 * p.x_st + l.ch;
  const G* g = (const G*)p.gate + l.b * p.g_sb + t0 * p.g_st + l.gate;
  XP xw[kSteps];
  GP gw[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    if (i < n) {
      xw[i].w = *reinterpret_cast<const typename XP::W*>(x + i * p.x_st);
      gw[i].w = *reinterpret_cast<const typename GP::W*>(g + i * p.g_st);
    }
  float carry[V], a[kSteps][V], b[kSteps][V], ma[V], mb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    carry[v] = l.in && p.h0 ? p.h0[l.b * p.D + l.ch + v] : 0.0f;
    ma[v] = 1.0f;
    mb[v] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a[i][v] = 1.0f;
      b[i][v] = 0.0f;
      if (i < n) {
        float om;
        gate_of<G, SIG>(gw[i].v[SHARED ? 0 : v], a[i][v], om);
        b[i][v] = SIG ? om * to_f(xw[i].v[v]) : to_f(xw[i].v[v]);
      }
      ma[v] *= a[i][v];
      mb[v] = fmaf(a[i][v], mb[v], b[i][v]);
    }
  join<V>(p, chain, chunk, warp, lane, ma, mb, carry);
  X* h = (X*)p.h + (l.b * p.T + t0) * p.D + l.ch;
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    if (i < n) {
      XP out;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        carry[v] = fmaf(a[i][v], carry[v], b[i][v]);
        out.v[v] = Cvt<X>::from(carry[v]);
      }
      *reinterpret_cast<typename XP::W*>(h + i * p.D) = out.w;
    }
  if (p.state && n > 0 && t0 + n == p.T)
#pragma unroll
    for (int v = 0; v < V; ++v) p.state[l.b * p.D + l.ch + v] = carry[v];
}

// Sums over the `lanes` (a power of two) neighbours of a lane of kSteps values
// each: every round gives half of the values to the partner and takes its
// half of the others', so 16 shuffles do for 16 values over 32 lanes. On
// return val[0..left) of a lane are the sums of the steps first..first + left,
// the same in the lanes that differ in bits above log2(kSteps).
MPB_D void sum_over_lanes(float (&val)[kSteps], int lane, int lanes, int& first, int& left) {
  first = 0;
  left = kSteps;
#pragma unroll
  for (int half = kSteps / 2, bit = 1; half > 0; half >>= 1, bit <<= 1) {
    if (bit < lanes) {
      const bool up = lane & bit;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float give = up ? val[i] : val[i + half], keep = up ? val[i + half] : val[i];
        val[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
      }
      first += up ? half : 0;
      left = half;
    }
  }
#pragma unroll
  for (int bit = kSteps; bit < 32; bit <<= 1)
    if (bit < lanes) val[0] += __shfl_xor_sync(0xffffffffu, val[0], bit);
}

template <class X, class G, bool SIG, int V, bool SHARED>
__global__ void __launch_bounds__(kWarps * 32, 2) k_gscan_bwd(ScanArgs p) {
  using XP = Pack<X, V>;
  using GP = Pack<G, SHARED ? 1 : V>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t chain, chunk;
  take_tile(p, chain, chunk);
  const Lane l = place<V, SHARED>(p, chain, lane);
  const int64_t r0 = (int64_t)chunk * p.steps + warp * kSteps;  // steps counted from the end
  const int64_t t0 = p.T - 1 - r0;
  const int n = l.in ? (int)(p.T - r0 < kSteps ? p.T - r0 : kSteps) : 0;
  const X* dh = (const X*)p.dh + l.b * p.dh_sb + t0 * p.dh_st + l.ch;
  const X* x = (const X*)p.x + l.b * p.x_sb + t0 * p.x_st + l.ch;
  const X* hs = (const X*)p.hsaved + l.b * p.h_sb + (t0 - 1) * p.h_st + l.ch;
  const G* g = (const G*)p.gate + l.b * p.g_sb + t0 * p.g_st + l.gate;
  XP dw[kSteps], xw[kSteps], hw[kSteps];
  GP gw[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    if (i < n) {
      dw[i].w = *reinterpret_cast<const typename XP::W*>(dh - i * p.dh_st);
      gw[i].w = *reinterpret_cast<const typename GP::W*>(g - i * p.g_st);
    }
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    if (i < n) {
      if (SIG) xw[i].w = *reinterpret_cast<const typename XP::W*>(x - i * p.x_st);
      if (t0 - i > 0) hw[i].w = *reinterpret_cast<const typename XP::W*>(hs - i * p.h_st);
    }
  float carry[V], ma[V], mb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    carry[v] = l.in && p.dstate ? p.dstate[l.b * p.D + l.ch + v] : 0.0f;
    ma[v] = 1.0f;
    mb[v] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    if (i < n)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, om;
        gate_of<G, SIG>(gw[i].v[SHARED ? 0 : v], a, om);
        ma[v] *= a;
        mb[v] = a * (mb[v] + to_f(dw[i].v[v]));
      }
  join<V>(p, chain, chunk, warp, lane, ma, mb, carry);
  X* dx = (X*)p.dx + (l.b * p.T + t0) * p.D + l.ch;
  G* dg = (G*)p.dgate + (l.b * p.T + t0) * p.H + l.gate;
  float sum[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    sum[i] = 0.0f;
    if (i < n) {
      XP out;
      GP gout;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, om;
        gate_of<G, SIG>(gw[i].v[SHARED ? 0 : v], a, om);
        const float s = to_f(dw[i].v[v]) + carry[v];
        float low = t0 - i > 0 ? to_f(hw[i].v[v]) : (p.h0 ? p.h0[l.b * p.D + l.ch + v] : 0.0f);
        if (SIG) low -= to_f(xw[i].v[v]);
        out.v[v] = Cvt<X>::from(SIG ? om * s : s);
        if (SHARED) {
          sum[i] = fmaf(s, low, sum[i]);
        } else {
          gout.v[v] = Cvt<G>::from(SIG ? s * low * (a * om) : s * low);
        }
        carry[v] = a * s;
      }
      *reinterpret_cast<typename XP::W*>(dx - i * p.D) = out.w;
      if (!SHARED) *reinterpret_cast<typename GP::W*>(dg - i * p.H) = gout.w;
    }
  }
  if (p.dh0 && n > 0 && r0 + n == p.T)
#pragma unroll
    for (int v = 0; v < V; ++v) p.dh0[l.b * p.D + l.ch + v] = carry[v];
  if (!SHARED) return;
  // a head's lanes: a power of two of them, or the whole warp (idle lanes add zeros)
  const int lanes = p.heads_per > 1 ? (int)p.lanes_per : 32;
  int first, left;
  sum_over_lanes(sum, lane, lanes, first, left);
  // lanes that hold the same sums: the one with the upper bits clear writes
  const int at = p.heads_per > 1 ? lane & (lanes - 1) : lane;
  const uint32_t group = chain - (uint32_t)l.b * p.groups;
  const int64_t head = p.groups_per > 1 ? (int64_t)p.by_groups_per.div(group)
                                        : (int64_t)group * p.heads_per + (p.heads_per > 1 ? lane / lanes : 0);
  if (at >= kSteps || head >= p.H) return;
  const int64_t bt = (int64_t)p.by_groups.div(chain) * p.T;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int64_t t = t0 - (first + i);
    if (i >= left || t < 0 || r0 + first + i >= p.T) continue;
    if (p.groups_per > 1) {
      p.part[((bt + t) * p.H + head) * p.groups_per + (group - (uint32_t)head * p.groups_per)] = sum[i];
    } else {
      float a, om;
      gate_of<G, SIG>(((const G*)p.gate)[(int64_t)p.by_groups.div(chain) * p.g_sb + t * p.g_st + head], a, om);
      ((G*)p.dgate)[(bt + t) * p.H + head] = Cvt<G>::from(SIG ? sum[i] * (a * om) : sum[i]);
    }
  }
}

// Heads of more channels than a block holds: the sum of their groups' sums, in order.
template <class G, bool SIG>
__global__ void __launch_bounds__(256) k_gscan_heads(ScanArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.B * p.T * p.H) return;
  const int64_t bt = i / p.H, head = i - bt * p.H, b = bt / p.T, t = bt - b * p.T;
  float s = 0.0f;
  for (uint32_t k = 0; k < p.groups_per; ++k) s += p.part[i * p.groups_per + k];
  float a, om;
  gate_of<G, SIG>(((const G*)p.gate)[b * p.g_sb + t * p.g_st + head], a, om);
  ((G*)p.dgate)[i] = Cvt<G>::from(SIG ? s * (a * om) : s);
}

// T == 0: the state passes through.
__global__ void k_gscan_none(const float* in, float* out, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) out[i] = in ? in[i] : 0.0f;
}

// One token: a thread per V channels.
template <class X, class G, bool SIG, int V, bool SHARED>
__global__ void __launch_bounds__(256) k_gscan_step(ScanArgs p, FastDiv by_d, FastDiv by_p) {
  using XP = Pack<X, V>;
  using GP = Pack<G, SHARED ? 1 : V>;
  uint32_t b, d;
  by_d.divmod(blockIdx.x * 256 + threadIdx.x, b, d);
  if (b >= p.B) return;
  d *= V;
  XP xw, out;
  GP gw;
  xw.w = *reinterpret_cast<const typename XP::W*>((const X*)p.x + b * p.x_sb + d);
  gw.w = *reinterpret_cast<const typename GP::W*>((const G*)p.gate + b * p.g_sb + (SHARED ? by_p.div(d) : d));
  float* s = p.state + b * p.D + d;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float a, om;
    gate_of<G, SIG>(gw.v[SHARED ? 0 : v], a, om);
    const float x = to_f(xw.v[v]);
    const float h = fmaf(a, s[v], SIG ? om * x : x);
    s[v] = h;
    out.v[v] = Cvt<X>::from(h);
  }
  *reinterpret_cast<typename XP::W*>((X*)p.h + b * p.D + d) = out.w;
}

// ------------------------------------------------------------------- host
// V = 2: two channels of a 16-bit type per lane, one 4-byte word per step. It
// takes even extents, strides and addresses (of a shared gate's heads too).
bool pairs(const ScanArgs& p, int x_dt, int g_dt, bool backward) {
  if (x_dt == MPB_F32 || p.P % 2 != 0 && p.H != p.D || p.D % 2 != 0) return false;
  auto even = [](const void* q, int64_t sb, int64_t st, size_t word) {
    return (uintptr_t)q % word == 0 && sb % 2 == 0 && st % 2 == 0;
  };
  bool ok = even(p.x, p.x_sb, p.x_st, 4) && even(p.h, 0, 0, 4);
  if (p.H == p.D) ok = ok && even(p.gate, p.g_sb, p.g_st, g_dt == MPB_F32 ? 8 : 4);
  if (backward)
    ok = ok && even(p.dh, p.dh_sb, p.dh_st, 4) && even(p.hsaved, p.h_sb, p.h_st, 4) && even(p.dx, 0, 0, 4) &&
         (p.H != p.D || even(p.dgate, 0, 0, g_dt == MPB_F32 ? 8 : 4));
  return ok;
}

// The channel groups and tiles for V channels per lane.
void lay_out(ScanArgs& p, int V) {
  const int64_t C = 32 * V;
  if (p.H == p.D) {
    p.groups = (uint32_t)((p.D + C - 1) / C);
    p.heads_per = p.lanes_per = p.groups_per = 1;
  } else {
    const int64_t lanes = (p.P + V - 1) / V;
    p.groups_per = (uint32_t)((lanes + 31) / 32);
    p.lanes_per = (uint32_t)(lanes < 32 ? lanes : 32);
    // several heads share a warp where their lanes are a power of two (the sums over them go by lane bits)
    p.heads_per = (lanes & (lanes - 1)) == 0 && lanes < 32 ? (uint32_t)(32 / lanes) : 1;
    p.groups = (uint32_t)(p.groups_per > 1 ? p.H * p.groups_per : (p.H + p.heads_per - 1) / p.heads_per);
  }
  const int64_t warps = (p.T + kSteps - 1) / kSteps;
  p.steps = (int)(warps < kWarps ? warps : kWarps) * kSteps;
  p.chains = (uint32_t)(p.B * p.groups);
  p.chunks = (uint32_t)((p.T + p.steps - 1) / p.steps);
  p.by_groups = FastDiv(p.groups);
  p.by_groups_per = FastDiv(p.groups_per);
  p.by_lanes_per = FastDiv(p.lanes_per);
  p.by_chains = FastDiv(p.chains);
}

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

// Scratch: {ticket, status}, flags (cleared by the call), maps and states of the tiles, sums of wide heads.
size_t scratch_of(ScanArgs& p, int V, bool backward, void* base, size_t* cleared) {
  size_t at = 0;
  char* q = (char*)base;
  *cleared = 0;
  if (p.chunks > 1) {
    const size_t tiles = (size_t)p.chains * p.chunks, data = align16(tiles * 32 * V * sizeof(float));
    p.ticket = (uint32_t*)q;
    p.status = (uint32_t*)(q + 4);
    p.flags = (uint32_t*)(q + 16);
    at = *cleared = align16(16 + tiles * sizeof(uint32_t));
    p.map_a = (float*)(q + at);
    p.map_b = (float*)(q + at + data);
    p.out_state = (float*)(q + at + 2 * data);
    at += 3 * data;
  }
  if (backward && p.groups_per > 1) {
    p.part = (float*)(q + at);
    at += align16((size_t)(p.B * p.T * p.H) * p.groups_per * sizeof(float));
  }
  return at;
}

// Enough for either V: the choice needs addresses and strides.
size_t scratch_need(ScanArgs p, bool backward) {
  size_t most = 0, cleared;
  for (int V = 1; V <= 2; ++V) {
    lay_out(p, V);
    const size_t n = scratch_of(p, V, backward, nullptr, &cleared);
    most = n > most ? n : most;
  }
  return most;
}

int prepare(const char* what, ScanArgs& p, int V, bool backward, void* scratch, cudaStream_t s) {
  lay_out(p, V);
  size_t cleared;
  scratch_of(p, V, backward, scratch, &cleared);
  if (cleared) return cuda_check(cudaMemsetAsync(scratch, 0, cleared, s), what);
  return MPB_OK;
}

template <class X, class G, bool SIG>
int launch_fwd(ScanArgs& p, int V, void* scratch, cudaStream_t s) {
  if (int rc = prepare("gated_scan", p, V, false, scratch, s)) return rc;
  const unsigned grid = p.chains * p.chunks, block = (unsigned)p.steps / kSteps * 32;
  const bool shared = p.H != p.D;
  constexpr int W = sizeof(X) == 2 ? 2 : 1;
  if (V == 2) {
    if (shared) k_gscan<X, G, SIG, W, true><<<grid, block, 0, s>>>(p);
    else k_gscan<X, G, SIG, W, false><<<grid, block, 0, s>>>(p);
  } else {
    if (shared) k_gscan<X, G, SIG, 1, true><<<grid, block, 0, s>>>(p);
    else k_gscan<X, G, SIG, 1, false><<<grid, block, 0, s>>>(p);
  }
  return launch_check("gated_scan");
}

template <class X, class G, bool SIG>
int launch_bwd(ScanArgs& p, int V, void* scratch, cudaStream_t s) {
  if (int rc = prepare("gated_scan_backward", p, V, true, scratch, s)) return rc;
  const unsigned grid = p.chains * p.chunks, block = (unsigned)p.steps / kSteps * 32;
  const bool shared = p.H != p.D;
  constexpr int W = sizeof(X) == 2 ? 2 : 1;
  if (V == 2) {
    if (shared) k_gscan_bwd<X, G, SIG, W, true><<<grid, block, 0, s>>>(p);
    else k_gscan_bwd<X, G, SIG, W, false><<<grid, block, 0, s>>>(p);
  } else {
    if (shared) k_gscan_bwd<X, G, SIG, 1, true><<<grid, block, 0, s>>>(p);
    else k_gscan_bwd<X, G, SIG, 1, false><<<grid, block, 0, s>>>(p);
  }
  if (int rc = launch_check("gated_scan_backward")) return rc;
  if (!shared || p.groups_per == 1) return MPB_OK;
  k_gscan_heads<G, SIG><<<(unsigned)((p.B * p.T * p.H + 255) / 256), 256, 0, s>>>(p);
  return launch_check("gated_scan_backward");
}

template <class X, class G, bool SIG>
int launch_step(const ScanArgs& p, int V, cudaStream_t s) {
  const int64_t n = p.B * (p.D / V);
  const unsigned grid = (unsigned)((n + 255) / 256);
  const FastDiv by_d((uint32_t)(p.D / V)), by_p((uint32_t)p.P);
  const bool shared = p.H != p.D;
  constexpr int W = sizeof(X) == 2 ? 2 : 1;
  if (V == 2) {
    if (shared) k_gscan_step<X, G, SIG, W, true><<<grid, 256, 0, s>>>(p, by_d, by_p);
    else k_gscan_step<X, G, SIG, W, false><<<grid, 256, 0, s>>>(p, by_d, by_p);
  } else {
    if (shared) k_gscan_step<X, G, SIG, 1, true><<<grid, 256, 0, s>>>(p, by_d, by_p);
    else k_gscan_step<X, G, SIG, 1, false><<<grid, 256, 0, s>>>(p, by_d, by_p);
  }
  return launch_check("gated_scan_step");
}

int pass_state(const char* what, const float* in, float* out, int64_t n, cudaStream_t s) {
  if (!out || in == out) return MPB_OK;
  k_gscan_none<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(in, out, n);
  return launch_check(what);
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
  // tiles are counted in 32 bits (at 16 steps of one warp the least a tile covers)
  if (B > 0x7fffffff || T > (int64_t)1 << 40 || D > 0x7fffffff ||
      (double)B * (double)(D + 32) * ((double)T / 128 + 1) > 2.0e9)
    return fail(MPB_ERR_SHAPE, "%s: (%lld, %lld, %lld) is too large", what, (long long)B, (long long)T, (long long)D);
  return MPB_OK;
}

int check_scratch(const char* what, size_t need, const void* scratch, size_t bytes) {
  if (need > bytes || (need && !scratch))
    return fail(MPB_ERR_SCRATCH, "%s: %zu bytes of scratch, %zu needed", what, bytes, need);
  return MPB_OK;
}

}  // namespace
}  // namespace mpb

using namespace mpb;

extern "C" {

size_t mpb_gated_scan_scratch_bytes(int64_t B, int64_t T, int64_t D, int64_t H, int x_dtype, int gate_dtype,
                                    int backward) {
  if (check_sizes("gated_scan", B, T, D, H) != MPB_OK || B * T * D == 0) return 0;
  ScanArgs p = {};
  p.B = B, p.T = T, p.D = D, p.H = H, p.P = D / H;
  return scratch_need(p, backward != 0);
}

int mpb_gated_scan(int64_t B, int64_t T, int64_t D, int64_t H, const void* x, int x_dtype, int64_t x_sb, int64_t x_st,
                   const void* gate, int gate_dtype, int64_t g_sb, int64_t g_st, const float* h0, int mode, void* h,
                   float* state, void* scratch, size_t scratch_bytes, mpb_stream_t stream) {
  const char* what = "gated_scan";
  if (int rc = check_sizes(what, B, T, D, H)) return rc;
  ScanArgs p = {};
  p.B = B, p.T = T, p.D = D, p.H = H, p.P = H ? D / H : 1;
  p.x = x, p.x_sb = x_sb, p.x_st = x_st, p.gate = gate, p.g_sb = g_sb, p.g_st = g_st;
  p.h0 = h0, p.h = h, p.state = state;
  cudaStream_t s = (cudaStream_t)stream;
  return by_types(what, x_dtype, gate_dtype, mode, [&](auto xt, auto gt, auto sig) {
    if (B * D == 0) return (int)MPB_OK;
    if (T == 0) return pass_state(what, h0, state, B * D, s);
    if (!x || !gate || !h) return fail(MPB_ERR_INVALID, "%s: null pointer", what);
    if (int rc = check_scratch(what, scratch_need(p, false), scratch, scratch_bytes)) return rc;
    const int V = pairs(p, x_dtype, gate_dtype, false) ? 2 : 1;
    return launch_fwd<decltype(xt), decltype(gt), decltype(sig)::value>(p, V, scratch, s);
  });
}

int mpb_gated_scan_backward(int64_t B, int64_t T, int64_t D, int64_t H, const void* dh, int64_t dh_sb, int64_t dh_st,
                            const void* x, int x_dtype, int64_t x_sb, int64_t x_st, const void* gate, int gate_dtype,
                            int64_t g_sb, int64_t g_st, const void* h, int64_t h_sb, int64_t h_st, const float* h0,
                            const float* dstate, int mode, void* dx, void* dgate, float* dh0, void* scratch,
                            size_t scratch_bytes, mpb_stream_t stream) {
  const char* what = "gated_scan_backward";
  if (int rc = check_sizes(what, B, T, D, H)) return rc;
  ScanArgs p = {};
  p.B = B, p.T = T, p.D = D, p.H = H, p.P = H ? D / H : 1;
  p.dh = dh, p.dh_sb = dh_sb, p.dh_st = dh_st, p.x = x, p.x_sb = x_sb, p.x_st = x_st;
  p.gate = gate, p.g_sb = g_sb, p.g_st = g_st, p.hsaved = h, p.h_sb = h_sb, p.h_st = h_st;
  p.h0 = h0, p.dstate = dstate, p.dx = dx, p.dgate = dgate, p.dh0 = dh0;
  cudaStream_t s = (cudaStream_t)stream;
  return by_types(what, x_dtype, gate_dtype, mode, [&](auto xt, auto gt, auto sig) {
    if (B * D == 0) return (int)MPB_OK;
    if (T == 0) return pass_state(what, dstate, dh0, B * D, s);
    if (!dh || !x || !gate || !h || !dx || !dgate) return fail(MPB_ERR_INVALID, "%s: null pointer", what);
    if (int rc = check_scratch(what, scratch_need(p, true), scratch, scratch_bytes)) return rc;
    const int V = pairs(p, x_dtype, gate_dtype, true) ? 2 : 1;
    return launch_bwd<decltype(xt), decltype(gt), decltype(sig)::value>(p, V, scratch, s);
  });
}

int mpb_gated_scan_step(int64_t B, int64_t D, int64_t H, const void* x, int x_dtype, int64_t x_sb, const void* gate,
                        int gate_dtype, int64_t g_sb, int mode, float* state, void* h, mpb_stream_t stream) {
  const char* what = "gated_scan_step";
  if (int rc = check_sizes(what, B, 1, D, H)) return rc;
  if (B * D > 0x7fffffffLL) return fail(MPB_ERR_SHAPE, "%s: %lld channels", what, (long long)(B * D));
  ScanArgs p = {};
  p.B = B, p.T = 1, p.D = D, p.H = H, p.P = H ? D / H : 1;
  p.x = x, p.x_sb = x_sb, p.gate = gate, p.g_sb = g_sb, p.h = h, p.state = state;
  return by_types(what, x_dtype, gate_dtype, mode, [&](auto xt, auto gt, auto sig) {
    if (B * D == 0) return (int)MPB_OK;
    if (!x || !gate || !h || !state) return fail(MPB_ERR_INVALID, "%s: null pointer", what);
    const int V = pairs(p, x_dtype, gate_dtype, false) ? 2 : 1;
    return launch_step<decltype(xt), decltype(gt), decltype(sig)::value>(p, V, (cudaStream_t)stream);
  });
}

int mpb_gated_scan_status(const void* scratch, int64_t T, mpb_stream_t stream) {
  uint32_t status = 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (!scratch || T <= kWarps * kSteps) return MPB_OK;  // one tile per chain: nothing waits
  if (int rc = cuda_check(cudaMemcpyAsync(&status, (const char*)scratch + 4, 4, cudaMemcpyDeviceToHost, s), "gated_scan_status"))
    return rc;
  if (int rc = cuda_check(cudaStreamSynchronize(s), "gated_scan_status")) return rc;
  return status ? fail((int)status, "gated_scan: a bounded wait for an earlier tile gave up") : MPB_OK;
}

}  // extern "C"

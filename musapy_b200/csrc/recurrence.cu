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
// One pass over the data, in tiles of 32 lanes x V channels by S warps x 16
// (backward 8 or 16) steps. A warp folds its steps to the map c -> A c + B that they
// apply to the state; the block joins the maps of its warps, and each warp
// then runs its steps once more from the state that enters them and writes.
// A warp copies its own steps' rows into shared memory some tiles ahead
// (cp.async, 16 bytes per lane where the layout allows), so the copies of the
// next tiles are in flight while a tile is computed, and no block barrier
// guards them.
//
// Along time either a block walks a chain (the tiles of 32 V channels of a
// sequence) and carries the state, or, where there are too few chains to
// occupy the GPU that way, the tiles of a chain run at the same time: a tile
// publishes its map, then its outgoing state, and takes its incoming state
// from the nearest earlier tile that has published one, applying the maps
// between them in time order. A state passes through the same operations
// wherever the look-back found it, so results do not depend on timing. Words
// are published without flags or fences: zero means not there yet, and a zero
// value is written as -0. Tiles are handed out by a ticket, all chains' first
// tiles first, so that a tile waits only for tiles that already run, and every
// wait is bounded. The backward pass is the same walk with time reversed, over
// the map u -> a (u + dh).
//
// A product of decays (16 steps of a warp, or a look-back's tile) may leave the
// range of float where the states do not. Above it, with linear gates beyond one,
// the tile's warps run one after the other instead, each from the state that the
// one before it ends with (where that is every tile, (8, 4096, 2048) f32 forward
// takes 332 us instead of 149, a gate per head of 64 in bf16 197 instead of 66, and
// (1, 65536, 1000) f32 by look-back 3.5 ms instead of 239 us). Below it the product
// is zero or a few bits: what is lost is below 2^-126 of the state before.
//
// Bound: memory by the bytes; what is reached is set by the latency of a tile
// (its barrier, the maps' join, in a look-back two round trips to L2) at 16
// warps per SM (8 where kRing says so), which is what the registers and the copies
// under way leave. Measured, (8, 4096, 2048) bf16 sigmoid, 256 chains: walked
// forward 78 us (5.1 TB/s), backward 150 us (5.4 TB/s); f32 linear 153 us (5.3 TB/s)
// and 205 us (6.5 TB/s); 32 gates for heads of 64, bf16 linear, 66 us (4.1 TB/s) and
// 104 us (3.9 TB/s). With 96 to 128 chains an SM has one block: 0.45 to 0.64 of the
// copy rate for the first, 0.33 to 0.54 for the last. By look-back (1, 65536, 1000)
// f32 linear: 239 us (3.3 TB/s) and 418 us; (1, 4096, 2048) bf16 sigmoid 27 and 41 us.
// Forms tried against earlier ones of 83 us forward and 161 us backward: one 4-byte
// copy per lane instead of 16 bytes 112 us forward; values in registers from plain
// loads, no copies ahead, 266 us; 16 warps of 8 (backward 4) steps instead of 8 of
// 16 (8) 109 and 223 us, the join and the places of a tile being done by twice the
// threads. Warps in turn through the unrolled steps instead of a short loop of their
// own cost heads backward 115 us.
#include "async_copy.cuh"
#include "common.cuh"
#include "internal.h"
#include "musapy_b200.h"
#include "plan.h"
#include "rows.cuh"

namespace mpb {
namespace {

constexpr int kWarps = 8;       // warps of a full tile
constexpr int kFwd = 16;        // steps per warp and tile, forward
// Steps per warp and tile, backward. The more, the fewer joins; 16 where two tiles
// of that many fit a block's share of shared memory: three inputs of one word
// per step. (Linear, a gate per head of 64, bf16, T = 4096: 74 us with 16 steps and
// 98 us with 8 at 128 chains, 104 and 129 us at 256, but 43 us with either by
// look-back at 32; f32 with a gate per channel 55 and 64 us at 128 chains, 100 and 97
// at 256. Sigmoid, four inputs, (8, 4096, 2048) bf16, in an earlier form: 172 us with
// 16 and 161 with 8.)
constexpr int bwd_steps(bool sig, int gate_bytes, int V, bool shared) {
  return !sig && (shared || gate_bytes * V <= 4) ? 16 : 8;
}
// Shared memory of a walk's block for tiles under way, two blocks per SM. A look-back
// always has three tiles under way; where a tile takes 48 KB (16-bit inputs with a
// 32-bit gate per channel; linear, backward, 16 steps) that leaves one block per SM.
constexpr int kRing = 96 << 10;

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
  FastDiv by_groups, by_groups_per, by_lanes_per, by_chains, by_heads_per;
  int steps;                  // of a tile
  int walk;                   // a block takes whole chains
  int wide;                   // every input's rows can be copied 16 bytes at a time
  // scratch
  uint32_t *ticket, *status;
  uint64_t* maps;    // (tiles, channels of a group): {A, B}
  uint32_t* states;  // (tiles, channels of a group): the state after the tile
  float* part;       // (B, T, H, groups_per)
};

// The decay a and what the input is weighted with, om, of a gate of type G.
template <bool SIG, class G, class F>
MPB_D void gate_of(F g, F& a, F& om) {
  if constexpr (SIG) {
    sigmoid2<sizeof(G) == 4>(g, a, om);
  } else {
    a = om = g;
  }
}
// Of a gate's pack; one that the lane's channels share is evaluated once.
template <bool SIG, int V, class G, int N>
MPB_D void gates_of(const Pack<G, N>& g, Floats<V>& a, Floats<V>& om) {
  if constexpr (N == 1 && V == 2) {
    float sa, so;
    gate_of<SIG, G>(to_f(g.v[0]), sa, so);
    a = vset<V>(sa);
    om = vset<V>(so);
  } else {
    gate_of<SIG, G>(unpack(g), a, om);
  }
}

// Whether a map's values are numbers on every channel of the lane (zero times an
// infinity or a NaN is NaN). Linear gates above one may take a product of decays
// out of the range of float where no state leaves it: such a map stands for nothing.
template <int V>
MPB_D bool numbers(Floats<V> a, Floats<V> b) {
  const Floats<V> zero = vfma(a, vset<V>(0.0f), vmul(b, vset<V>(0.0f)));
  return vget(zero, 0) + vget(zero, V - 1) == 0.0f;
}

// Where a lane works.
struct Lane {
  int64_t b, ch, gate;  // sequence, first channel, its gate
  int64_t ch0, end;     // the warp's first channel and the one after its last
  int64_t head;         // the warp's first gate
  int slot;             // the lane's gate among the warp's
  bool in;
};

template <int V, bool SHARED>
MPB_D Lane place(const ScanArgs& p, uint32_t chain, int lane) {
  uint32_t b, group;
  p.by_groups.divmod(chain, b, group);
  Lane l;
  l.b = b;
  if (!SHARED) {
    l.ch = l.gate = l.head = ((int64_t)group * 32 + lane) * V;
    l.slot = 0;
    l.ch0 = (int64_t)group * 32 * V;
    l.end = p.D;
    l.in = l.ch < p.D;
  } else if (p.groups_per > 1) {  // a head's channels in several groups
    uint32_t head, part;
    p.by_groups_per.divmod(group, head, part);
    const int64_t c = ((int64_t)part * 32 + lane) * V;
    l.gate = l.head = head;
    l.slot = 0;
    l.ch = head * p.P + c;
    l.ch0 = head * p.P + (int64_t)part * 32 * V;
    l.end = (head + 1) * p.P;
    l.in = c < p.P;
  } else {  // one or several heads in a group
    uint32_t head, at;
    p.by_lanes_per.divmod((uint32_t)lane, head, at);
    l.in = head < p.heads_per && (int64_t)group * p.heads_per + head < p.H;
    l.head = (int64_t)group * p.heads_per;
    l.gate = l.head + head;
    l.slot = l.in ? (int)head : 0;
    l.ch0 = l.head * p.P;
    l.end = (l.head + p.heads_per < p.H ? l.head + p.heads_per : p.H) * p.P;
    l.ch = l.gate * p.P + (int64_t)at * V;
  }
  if (!l.in) l.ch = l.gate = 0;
  return l;
}

MPB_D uint32_t ld_word(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
MPB_D uint64_t ld_word(const uint64_t* p) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
MPB_D void st_word(uint32_t* p, uint32_t v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
MPB_D void st_word(uint64_t* p, uint64_t v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
MPB_D unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
constexpr unsigned long long kPatience = 2000000000ull;  // ns a wait lasts at most

// A value as a word that is never zero, and back (+0 for -0).
MPB_D uint32_t state_word(float v) {
  const uint32_t w = __float_as_uint(v);
  return w ? w : 0x80000000u;
}
MPB_D uint64_t map_word(float a, float b) {
  const uint64_t w = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
  return w ? w : 0x80000000ull;
}

// A word some other tile publishes, when it is there; false when the wait ran out.
template <class W>
MPB_D bool await(const W* p, W& w) {
  w = ld_word(p);
  if (w) return true;
  const unsigned long long t0 = now_ns();
  do {
    w = ld_word(p);
    if (w) return true;
  } while (now_ns() - t0 < kPatience);
  return false;
}

// Warp 0 of a tile: the state that enters it, per lane and channel (carry
// holds the one before the chain). early: the words of the tile before as seen
// some time ago.
template <int V>
MPB_D void look_back(const ScanArgs& p, uint32_t chain, uint32_t chunk, int lane, uint32_t (&early)[V],
                     float (&carry)[V]) {
  constexpr int C = 32 * V;
  if (chunk == 0) return;
  auto at = [&](uint32_t k) { return (size_t)(k * p.chains + chain) * C + lane * V; };
  bool there = true;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (!early[v]) early[v] = ld_word(p.states + at(chunk - 1) + v);
    there = there && early[v];
  }
  if (__all_sync(0xffffffffu, there)) {
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = __uint_as_float(early[v]) + 0.0f;
    return;
  }
  // lane i looks at the first channel of the tile i + 1 before this one;
  // before the chain's first tile stands the initial state
  uint32_t back;
  bool ok = true;
  const unsigned long long t0 = now_ns();
  for (;;) {
    const bool before = (uint32_t)lane >= chunk;
    const size_t q = before ? 0 : (size_t)((chunk - 1 - lane) * p.chains + chain) * C;
    const uint32_t states = __ballot_sync(0xffffffffu, before || ld_word(p.states + q) != 0);
    const uint32_t nothing = __ballot_sync(0xffffffffu, !before && ld_word(p.maps + q) == 0);
    if (states) {
      back = __ffs(states) - 1;
      if ((nothing & ((1u << back) - 1)) == 0) break;
    }
    if (__any_sync(0xffffffffu, now_ns() - t0 > kPatience)) {
      ok = false;
      back = 0;
      break;
    }
  }
  // The other channels' words of those tiles are there or about to be. The
  // state and the first maps are fetched together: one round trip.
  constexpr int kTogether = 8;
  uint32_t state[V] = {};
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (chunk > back && ok) state[v] = ld_word(p.states + at(chunk - 1 - back) + v);
  for (uint32_t k0 = chunk - back, first = 1; first || k0 < chunk; k0 += kTogether, first = 0) {
    uint64_t w[kTogether][V];
#pragma unroll
    for (int i = 0; i < kTogether; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) w[i][v] = k0 + i < chunk ? ld_word(p.maps + at(k0 + i) + v) : 0;
    if (first && chunk > back && ok)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (!state[v]) ok = await(p.states + at(chunk - 1 - back) + v, state[v]) && ok;
        carry[v] = __uint_as_float(state[v]) + 0.0f;
      }
#pragma unroll
    for (int i = 0; i < kTogether; ++i)
      if (k0 + i < chunk)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (!w[i][v]) ok = ok && await(p.maps + at(k0 + i) + v, w[i][v]);
          carry[v] = fmaf(__uint_as_float((uint32_t)w[i][v]), carry[v], __uint_as_float((uint32_t)(w[i][v] >> 32)));
        }
  }
  if (!ok) {  // gave up: what follows is marked and NaN
    st_word(p.status, MPB_ERR_TIMEOUT);
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = NAN;
  }
}

template <int V>
struct Shared {
  // the warps' maps, of three tiles in turn
  __align__(8) float a[3][kWarps][32 * V];
  __align__(8) float b[3][kWarps][32 * V];
  __align__(8) float carry[32 * V];
  uint32_t tiles[4];
  int turns;  // of a look-back's tile: its warps run in turn
};

// The state after warp w's steps.
template <int V>
MPB_D Floats<V> through(const Shared<V>& sh, int side, int w, int lane, Floats<V> c) {
  return vfma(*reinterpret_cast<const Floats<V>*>(&sh.a[side][w][lane * V]), c,
              *reinterpret_cast<const Floats<V>*>(&sh.b[side][w][lane * V]));
}

template <int V>
MPB_D void put_map(Shared<V>& sh, int side, int warp, int lane, Floats<V> a, Floats<V> b) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sh.a[side][warp][lane * V + v] = vget(a, v);
    sh.b[side][warp][lane * V + v] = vget(b, v);
  }
}

// Warps in turn, where a warp's map is not made of numbers: each waits for the
// state that the one before it ends with. To start: the state that enters the
// warp's steps, for the first warp the tile's. To end: the state after the steps.
template <int V>
MPB_D void start_turn(const Shared<V>& sh, int warp, int lane, Floats<V>& in) {
  for (int w = 0; w < warp; ++w) __syncthreads();
  if (warp) in = *reinterpret_cast<const Floats<V>*>(&sh.carry[lane * V]);
}
template <int V>
MPB_D void end_turn(Shared<V>& sh, int warp, int lane, Floats<V> in) {
  *reinterpret_cast<Floats<V>*>(&sh.carry[lane * V]) = in;
  for (int w = warp; w < (int)(blockDim.x >> 5); ++w) __syncthreads();
}

// A walk's tile: joins the maps of the block's warps (a, b: this warp's). carry:
// the state that enters the tile and, on return, the one that leaves it (of
// a single warp the caller's steps end there). Returns in `in` the state that
// enters the warp's steps. With TURNS, true and nothing joined (in = carry) where a
// map is not sound: the warps run in turn.
template <int V, bool TURNS>
MPB_D bool join(Shared<V>& sh, int side, int warp, int lane, bool sound, Floats<V> a, Floats<V> b, Floats<V>& carry,
                Floats<V>& in) {
  const int warps = blockDim.x >> 5;
  in = carry;
  if (warps == 1) return false;
  put_map<V>(sh, side, warp, lane, a, b);
  if constexpr (TURNS) {
    if (__syncthreads_or(!sound)) return true;
  } else {
    __syncthreads();
  }
  if (warps == kWarps) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) in = carry;
      carry = through<V>(sh, side, w, lane, carry);
    }
  } else {
    for (int w = 0; w < warps; ++w) {
      if (w == warp) in = carry;
      carry = through<V>(sh, side, w, lane, carry);
    }
  }
  return false;
}

// cp.async of the word that holds the element(s): 4 bytes for one 32-bit or
// two 16-bit elements, 8 for two 32-bit ones. Of a single 16-bit element the
// aligned word around it is taken (an address of 2 modulo 4 is never the start
// of an allocation; at 0 modulo 4 only the element's two bytes are read).
template <int BYTES>
MPB_D void copy_word(uint32_t dst, const void* src) {
  if constexpr (BYTES == 8) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
  } else if constexpr (BYTES == 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
  } else {
    const uintptr_t q = (uintptr_t)src;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(q & ~(uintptr_t)3),
                 "r"((q & 2) ? 4 : 2)
                 : "memory");
  }
}
MPB_D void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
MPB_D void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// p + st as one 64-bit add (the compiler would multiply for every step).
template <class T>
MPB_D T* ahead_by(T* p, int64_t st) {
  uint64_t q = (uint64_t)p;
  asm("add.s64 %0, %0, %1;" : "+l"(q) : "l"(st));
  return (T*)q;
}

// Stores through a pointer that ahead_by has moved: it is global memory.
template <class T, int N>
MPB_D void put_global(char* p, const Pack<T, N>& v) {
  if constexpr (sizeof(T) * N == 8) {
    asm volatile("st.global.v2.u32 [%0], {%1, %2};" ::"l"(p), "r"(v.w.x), "r"(v.w.y) : "memory");
  } else if constexpr (sizeof(T) * N == 4) {
    asm volatile("st.global.u32 [%0], %1;" ::"l"(p), "r"(*reinterpret_cast<const uint32_t*>(&v.w)) : "memory");
  } else {
    asm volatile("st.global.u16 [%0], %1;" ::"l"(p), "h"(v.w) : "memory");
  }
}

// One input of a tile: N elements of T per step, in words of shared memory
// [step][thread].
template <class T, int N>
struct Column {
  static constexpr int kElems = (int)sizeof(T) * N;        // bytes used
  static constexpr int kWord = kElems < 4 ? 4 : kElems;    // bytes kept
  static constexpr uint32_t bytes(int steps) { return (uint32_t)steps * kWarps * 32 * kWord; }
  // n of STEPS steps, st bytes apart
  template <int STEPS>
  static MPB_D void copy(uint32_t base, const char* src, int64_t st, int n) {
    base += threadIdx.x * kWord;
    if (n >= STEPS) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        copy_word<kElems>(base + i * kWarps * 32 * kWord, src);
        src = ahead_by(src, st);
      }
    } else {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (i < n) copy_word<kElems>(base + i * kWarps * 32 * kWord, src);
        src = ahead_by(src, st);
      }
    }
  }
  // 16 bytes at a time, a warp's rows of 32 words by as many lanes as a row
  // takes: a quarter of the copies. src: the lane's part of the warp's first row;
  // `mine`: it lies inside the row.
  static constexpr int kLanes = kElems * 2;  // of 16 bytes, for a row of 32 lanes' elements
  static constexpr int kRows = 32 / kLanes;  // rows per copy of the warp
  template <int STEPS>
  static MPB_D void copy_wide(uint32_t base, const char* src, int64_t st, int n, bool mine) {
    const int lane = threadIdx.x & 31, row = lane / kLanes;
    base += (row * kWarps * 32 + (threadIdx.x & ~31)) * kWord + lane % kLanes * 16;
#pragma unroll
    for (int j = 0; j < STEPS; j += kRows) {
      if (mine && row + j < n)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + j * kWarps * 32 * kWord), "l"(src) : "memory");
      src = ahead_by(src, st * kRows);
    }
  }
  // half: of a single 16-bit element, bit 1 of its address
  static MPB_D Pack<T, N> get(const char* base, int i, uint32_t half) {
    Pack<T, N> v;
    const char* q = base + (i * kWarps * 32 + threadIdx.x) * kWord;
    if constexpr (kElems < 4) q += half & 2;
    v.w = *reinterpret_cast<const typename Pack<T, N>::W*>(q);
    return v;
  }
};

// The gates of a warp's steps where channels share them: a word per step and
// head of the warp, copied by one lane each and read by all of the head's.
template <class G, int STEPS>
struct HeadGates {
  static constexpr int kElems = (int)sizeof(G);
  static MPB_D uint32_t at(int e) { return ((threadIdx.x >> 5) * STEPS * 32 + e) * 4; }
  // src: the gate of the warp's first head at its first step
  static MPB_D void copy(uint32_t base, const char* src, int64_t st, int n, int per, int heads, FastDiv by_per) {
    for (int e = threadIdx.x & 31; e < STEPS * per; e += 32) {
      uint32_t i, j;
      by_per.divmod((uint32_t)e, i, j);
      if ((int)i < n && (int)j < heads) copy_word<kElems>(base + at(e), src + i * st + j * kElems);
    }
  }
  static MPB_D Pack<G, 1> get(const char* base, int e, uint32_t half) {
    Pack<G, 1> v;
    const char* q = base + at(e);
    if constexpr (kElems < 4) q += half & 2;
    v.w = *reinterpret_cast<const typename Pack<G, 1>::W*>(q);
    return v;
  }
};

// The tiles of a walk, in order: the chunks of chain blockIdx, then of chain
// blockIdx + grid, ...
struct Order {
  uint32_t chain, chunk;
  MPB_D Order() : chain(blockIdx.x), chunk(0) {}
  MPB_D bool here(const ScanArgs& p) const { return chain < p.chains; }
  MPB_D void next(const ScanArgs& p) {
    if (++chunk == p.chunks) {
      chunk = 0;
      chain += gridDim.x;
    }
  }
};

// Where a thread's words of a tile lie.
template <int PER, int N>
struct Place {
  const char* at[N];
  int left;       // steps from the warp's first one to the end of the sequence; 0 on an idle lane
  int end;        // the same on every lane
  int heads;      // gates of the warp, where channels share them
  uint32_t wide;  // wide_lane
  // Along a chain: the next chunk.
  MPB_D void move(const ScanArgs& p, const int64_t (&st)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) at[k] += st[k] * p.steps;
    left -= p.steps;
    end -= p.steps;
  }
  MPB_D int steps() const { return left < PER ? left : PER; }
};

// The tiles of a look-back, taken by ticket. Work on a tile is in two parts: its
// map is published one tile before its state is asked for, so that the wait
// for one tile's state runs under the folding of the next tile's map, and
// the tiles of a chain find each other's maps ready.
//   front(o, stage, side)  folds tile o's maps into sh side
//   first(o, c)            the state before the chain, warp 0 (of the first 32 chunks:
//                          as far as a look-back reaches)
//   rest(o, stage, in, in_turn)  runs the warp's steps from the state `in` to the one after them
//   copy(it, stage)        copies the block's tile number `it`, and commits
// With TURNS, a tile whose map is not made of numbers publishes none: the tiles
// after it wait for its state, which its last warp publishes.
template <int V, bool TURNS, class Front, class First, class Rest, class Copy>
MPB_D void look_back_tiles(const ScanArgs& p, Shared<V>& sh, int warp, int lane, Front front, First first, Rest rest,
                           Copy copy) {
  constexpr int C = 32 * V;
  const uint32_t total = p.chains * p.chunks;
  struct At {
    uint32_t chain, chunk;
  };
  auto tile = [&](int it, At& o) {  // false when there is none
    const uint32_t t = sh.tiles[it & 3];
    p.by_chains.divmod(t, o.chunk, o.chain);
    return t < total;
  };
  // The first tickets are taken one after the other, so that every running
  // block has its first tile before any has its second: a tile's predecessors
  // are then worked on at the same time, not behind others.
  for (int s = 0; s < 3; ++s) {
    if (threadIdx.x == 0) sh.tiles[s] = atomicAdd(p.ticket, 1u);
    __syncthreads();
    At o;
    copy(tile(s, o), o.chain, o.chunk, s);
  }
  At cur, nxt;
  float ta[V], tb[V];  // the tile's map, warp 0
  bool sound = true;   // on every lane
  auto publish = [&](const At& o, int side) {
    bool mine = true;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ta[v] = sh.a[side][0][lane * V + v], tb[v] = sh.b[side][0][lane * V + v];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float aw = sh.a[side][w][lane * V + v];
        tb[v] = fmaf(aw, tb[v], sh.b[side][w][lane * V + v]);
        ta[v] *= aw;
      }
      mine = mine && numbers<1>(ta[v], tb[v]);
    }
    if (TURNS) sound = __all_sync(0xffffffffu, mine);
    if (o.chunk + 1 < p.chunks && sound)
#pragma unroll
      for (int v = 0; v < V; ++v)
        st_word(p.maps + (size_t)(o.chunk * p.chains + o.chain) * C + lane * V + v, map_word(ta[v], tb[v]));
  };
  bool have = tile(0, cur);
  copies_wait<2>();
  __syncwarp();  // the words that other lanes have copied
  if (have) front(cur.chain, cur.chunk, 0, 0);
  __syncthreads();
  if (have && warp == 0) publish(cur, 0);
  int stage = 0;
  for (int it = 0; have; ++it) {
    const int after = stage == 2 ? 0 : stage + 1;
    const bool more = tile(it + 1, nxt);
    if (threadIdx.x == 0) sh.tiles[(it + 3) & 3] = atomicAdd(p.ticket, 1u);
    uint32_t early[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
      early[v] = warp == 0 && cur.chunk > 0
                     ? ld_word(p.states + (size_t)((cur.chunk - 1) * p.chains + cur.chain) * C + lane * V + v)
                     : 0;
    copies_wait<1>();
    __syncwarp();
    if (more) front(nxt.chain, nxt.chunk, after, after);
    __syncthreads();
    if (warp == 0) {
      const bool whole = sound;
      float a[V], b[V], c[V];
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = ta[v], b[v] = tb[v];
      if (more) publish(nxt, after);
      first(cur.chain, cur.chunk, c);
      look_back<V>(p, cur.chain, cur.chunk, lane, early, c);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (cur.chunk + 1 < p.chunks && whole)
          st_word(p.states + (size_t)(cur.chunk * p.chains + cur.chain) * C + lane * V + v, state_word(fmaf(a[v], c[v], b[v])));
        sh.carry[lane * V + v] = c[v];
      }
      if (TURNS && lane == 0) sh.turns = !whole;
    }
    __syncthreads();
    const bool turns = TURNS && sh.turns;
    Floats<V> in = vset<V>(0.0f);
    if (!turns || warp == 0) in = *reinterpret_cast<const Floats<V>*>(&sh.carry[lane * V]);
    if (!turns) {
      for (int w = 0; w < warp; ++w) in = through<V>(sh, stage, w, lane, in);
      rest(cur.chain, cur.chunk, stage, in, std::false_type());
    } else if constexpr (TURNS) {
      start_turn<V>(sh, warp, lane, in);
      rest(cur.chain, cur.chunk, stage, in, std::true_type());
      if (warp == kWarps - 1 && cur.chunk + 1 < p.chunks)
#pragma unroll
        for (int v = 0; v < V; ++v)
          st_word(p.states + (size_t)(cur.chunk * p.chains + cur.chain) * C + lane * V + v, state_word(vget(in, v)));
      end_turn<V>(sh, warp, lane, in);
    }
    __syncwarp();  // the stage has been read by every lane
    At far;
    copy(tile(it + 3, far), far.chain, far.chunk, stage);
    cur = nxt;
    have = more;
    stage = after;
  }
}

// Where a lane's copies of a column start, from the first row's start; st: bytes between steps.
template <class C, class T>
MPB_D const char* at_lane(const ScanArgs& p, const char* row, const Lane& l, int64_t st, int lane) {
  return p.wide ? row + l.ch0 * (int)sizeof(T) + lane % C::kLanes * 16 + lane / C::kLanes * st : row + l.ch * (int)sizeof(T);
}
template <class C, int STEPS>
MPB_D void copy_column(const ScanArgs& p, uint32_t base, const char* src, int64_t st, int left, int end, uint32_t wide) {
  if (p.wide) C::template copy_wide<STEPS>(base, src, st, end, wide >> (C::kElems / 4) & 1);
  else C::template copy<STEPS>(base, src, st, left);
}
// Bit n: the lane's 16 bytes of a row of 32 words of 4 n bytes lie inside the warp's channels.
template <int V>
MPB_D uint32_t wide_lane(const Lane& l, int lane) {
  uint32_t bits = 0;
#pragma unroll
  for (int n = 1; n <= 2; ++n) {
    const int per = 4 * V / n;  // channels in 16 bytes of such a row
    if (per > 0 && l.ch0 + (lane % (8 * n)) * per < l.end) bits |= 1u << n;
  }
  return bits;
}

template <class X, class G, int V, bool SHARED>
struct FwdTile {
  using CX = Column<X, V>;
  using CG = Column<G, SHARED ? 1 : V>;
  using HG = HeadGates<G, kFwd>;
  static constexpr uint32_t kG = CX::bytes(kFwd), kBytes = kG + CG::bytes(kFwd);
  static constexpr int kStages = kRing / kBytes < 3 ? kRing / kBytes : 3;  // of a walk
  static_assert(kStages >= 2, "a tile is copied while another is computed");
};

// What the forward kernels share: copies, and the decay and input of a step.
template <class X, class G, bool SIG, int V, bool SHARED>
struct Forward {
  using Tile = FwdTile<X, G, V, SHARED>;
  const ScanArgs& p;
  const int64_t in_st[2], out_st;
  const int lane, warp;
  int gate_slot;
  uint32_t half_x, half_g;  // bit 1 of the addresses of single 16-bit elements at step 0
  size_t state_at;
  MPB_D explicit Forward(const ScanArgs& args)
      : p(args), in_st{args.x_st * (int64_t)sizeof(X), args.g_st * (int64_t)sizeof(G)}, out_st(args.D * (int64_t)sizeof(X)),
        lane(threadIdx.x & 31), warp(threadIdx.x >> 5) {}
  MPB_D void inputs(uint32_t chain, uint32_t chunk, Place<kFwd, 2>& f) const {
    const Lane l = place<V, SHARED>(p, chain, lane);
    const int64_t t0 = (int64_t)chunk * p.steps + warp * kFwd;
    const char* x = (const char*)((const X*)p.x + l.b * p.x_sb + t0 * p.x_st);
    const char* g = (const char*)((const G*)p.gate + l.b * p.g_sb + t0 * p.g_st);
    f.at[0] = at_lane<typename Tile::CX, X>(p, x, l, in_st[0], lane);
    f.at[1] = SHARED ? g + l.head * sizeof(G) : at_lane<typename Tile::CG, G>(p, g, l, in_st[1], lane);
    f.wide = wide_lane<V>(l, lane);
    f.end = (int)(p.T - t0);
    f.left = l.in ? f.end : 0;
    f.heads = SHARED ? (int)(p.H - l.head < p.heads_per ? p.H - l.head : p.heads_per) : 0;
  }
  MPB_D void copy(uint32_t base, const Place<kFwd, 2>& f) const {
    copy_column<typename Tile::CX, kFwd>(p, base, f.at[0], in_st[0], f.left, f.end, f.wide);
    if constexpr (SHARED) Tile::HG::copy(base + Tile::kG, f.at[1], in_st[1], f.end, (int)p.heads_per, f.heads, p.by_heads_per);
    else copy_column<typename Tile::CG, kFwd>(p, base + Tile::kG, f.at[1], in_st[1], f.left, f.end, f.wide);
  }
  MPB_D void output(uint32_t chain, uint32_t chunk, Place<kFwd, 1>& f) {
    const Lane l = place<V, SHARED>(p, chain, lane);
    const int64_t t0 = (int64_t)chunk * p.steps + warp * kFwd;
    f.at[0] = (const char*)((const X*)p.h + (l.b * p.T + t0) * p.D + l.ch);
    f.left = l.in ? (int)(p.T - t0) : 0;
    state_at = (size_t)(l.b * p.D + l.ch);
    sub_words(l);
  }
  MPB_D void sub_words(const Lane& l) {
    gate_slot = l.slot;
    half_x = (uint32_t)(uintptr_t)((const X*)p.x + l.b * p.x_sb + l.ch);
    half_g = (uint32_t)(uintptr_t)((const G*)p.gate + l.b * p.g_sb + l.gate);
  }
  // t0: the warp's first step in the tile
  MPB_D void step(const char* mine, int i, uint32_t t0, Floats<V>& a, Floats<V>& b) const {
    const Floats<V> x = unpack(Tile::CX::get(mine, i, half_x + (t0 + i) * (uint32_t)in_st[0]));
    const uint32_t half = half_g + (t0 + i) * (uint32_t)in_st[1];
    Floats<V> om;
    if constexpr (SHARED) gates_of<SIG, V>(Tile::HG::get(mine + Tile::kG, i * (int)p.heads_per + gate_slot, half), a, om);
    else gates_of<SIG, V>(Tile::CG::get(mine + Tile::kG, i, half), a, om);
    b = SIG ? vmul(om, x) : x;
  }
  // Runs f(i) over the warp's steps of a tile; f returns the state to write.
  template <class F>
  MPB_D void write(const Place<kFwd, 1>& to, Floats<V>& in, F f) const {
    const int n = to.steps();
    char* h = const_cast<char*>(to.at[0]);
    if (__all_sync(0xffffffffu, n == kFwd)) {
#pragma unroll
      for (int i = 0; i < kFwd; ++i) {
        f(i);
        put_global(h, pack<X>(in));
        h = ahead_by(h, out_st);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kFwd; ++i)
        if (i < n) {
          f(i);
          put_global(h, pack<X>(in));
          h = ahead_by(h, out_st);
        }
    }
    ended(to, n, in);
  }
  // The same for a warp in turn, in short code.
  MPB_D void write_in_turn(const char* mine, uint32_t t0, const Place<kFwd, 1>& to, Floats<V>& in) const {
    const int n = to.steps();
    char* h = const_cast<char*>(to.at[0]);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      Floats<V> a, b;
      step(mine, i, t0, a, b);
      in = vfma(a, in, b);
      put_global(h, pack<X>(in));
      h = ahead_by(h, out_st);
    }
    ended(to, n, in);
  }
  MPB_D void ended(const Place<kFwd, 1>& to, int n, Floats<V> in) const {
    if (p.state && n > 0 && n == to.left)
#pragma unroll
      for (int v = 0; v < V; ++v) p.state[state_at + v] = vget(in, v);
  }
};

template <class X, class G, bool SIG, int V, bool SHARED>
__global__ void __launch_bounds__(kWarps * 32, 2) k_gscan_walk(ScanArgs p) {
  using Tile = FwdTile<X, G, V, SHARED>;
  constexpr int NST = Tile::kStages;
  extern __shared__ __align__(16) char ring[];
  __shared__ Shared<V> sh;
  Forward<X, G, SIG, V, SHARED> fw(p);
  const uint32_t base = smem_u32(ring);
  if (p.status && blockIdx.x == 0 && threadIdx.x == 0) *p.status = MPB_OK;  // nothing waits
  Order cur, ahead;
  Place<kFwd, 2> from;
  Place<kFwd, 1> to;
  const int64_t out_st[1] = {fw.out_st};
  auto copy = [&](int s) {  // the walk's next tile into stage s
    if (ahead.here(p)) {
      if (ahead.chunk == 0) fw.inputs(ahead.chain, 0, from);
      else from.move(p, fw.in_st);
      fw.copy(base + s * Tile::kBytes, from);
      ahead.next(p);
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) copy(s);
  int stage = 0;
  Floats<V> carry = vset<V>(0.0f);
  for (int it = 0; cur.here(p); ++it) {
    __syncwarp();  // the stage that is filled next has been read by every lane
    copy(stage == 0 ? NST - 1 : stage - 1);
    if (cur.chunk == 0) {
      fw.output(cur.chain, 0, to);
#pragma unroll
      for (int v = 0; v < V; ++v) vput(carry, v, to.left > 0 && p.h0 ? p.h0[fw.state_at + v] : 0.0f);
    } else {
      to.move(p, out_st);
    }
    copies_wait<NST - 1>();
    __syncwarp();  // the words that other lanes have copied
    const char* mine = ring + stage * Tile::kBytes;
    const uint32_t t0 = cur.chunk * p.steps + fw.warp * kFwd;
    // Steps after the last are computed from whatever the ring holds: nothing
    // follows them in the chain, and they are not written.
    Floats<V> a[kFwd], b[kFwd], ma = vset<V>(1.0f), mb = vset<V>(0.0f), in;
#pragma unroll
    for (int i = 0; i < kFwd; ++i) {
      fw.step(mine, i, t0, a[i], b[i]);
      ma = vmul(ma, a[i]);
      mb = vfma(a[i], mb, b[i]);
    }
    const bool sound = SIG || to.left < kFwd || numbers<V>(ma, mb);
    const bool turns = join<V, !SIG>(sh, it & 1, fw.warp, fw.lane, sound, ma, mb, carry, in);
    if (turns) {
      start_turn<V>(sh, fw.warp, fw.lane, in);
      fw.write_in_turn(mine, t0, to, in);
      end_turn<V>(sh, fw.warp, fw.lane, in);
      carry = *reinterpret_cast<const Floats<V>*>(&sh.carry[fw.lane * V]);
    } else {
      fw.write(to, in, [&](int i) { in = vfma(a[i], in, b[i]); });
    }
    if (blockDim.x == 32) carry = in;
    cur.next(p);
    stage = stage + 1 == NST ? 0 : stage + 1;
  }
}

template <class X, class G, bool SIG, int V, bool SHARED>
__global__ void __launch_bounds__(kWarps * 32, 2) k_gscan_far(ScanArgs p) {
  using Tile = FwdTile<X, G, V, SHARED>;
  extern __shared__ __align__(16) char ring[];
  __shared__ Shared<V> sh;
  Forward<X, G, SIG, V, SHARED> fw(p);
  const uint32_t base = smem_u32(ring);
  auto t0_of = [&](uint32_t chunk) { return chunk * p.steps + fw.warp * kFwd; };
  look_back_tiles<V, !SIG>(
      p, sh, fw.warp, fw.lane,
      [&](uint32_t chain, uint32_t chunk, int stage, int side) {
        const Lane l = place<V, SHARED>(p, chain, fw.lane);
        fw.sub_words(l);
        Floats<V> ma = vset<V>(1.0f), mb = vset<V>(0.0f);
#pragma unroll
        for (int i = 0; i < kFwd; ++i) {
          Floats<V> a, b;
          fw.step(ring + stage * Tile::kBytes, i, t0_of(chunk), a, b);
          ma = vmul(ma, a);
          mb = vfma(a, mb, b);
        }
        // steps after the last and idle lanes were computed from whatever the ring held
        if (!SIG && !(l.in && p.T - t0_of(chunk) >= kFwd)) ma = vset<V>(1.0f), mb = vset<V>(0.0f);
        put_map<V>(sh, side, fw.warp, fw.lane, ma, mb);
      },
      [&](uint32_t chain, uint32_t chunk, float (&c)[V]) {
        const Lane l = place<V, SHARED>(p, chain, fw.lane);
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = chunk < 32 && l.in && p.h0 ? p.h0[l.b * p.D + l.ch + v] : 0.0f;
      },
      [&](uint32_t chain, uint32_t chunk, int stage, Floats<V>& in, auto in_turn) {
        Place<kFwd, 1> to;
        fw.output(chain, chunk, to);
        if constexpr (decltype(in_turn)::value) {
          fw.write_in_turn(ring + stage * Tile::kBytes, t0_of(chunk), to, in);
        } else {
          fw.write(to, in, [&](int i) {
            Floats<V> a, b;
            fw.step(ring + stage * Tile::kBytes, i, t0_of(chunk), a, b);
            in = vfma(a, in, b);
          });
        }
      },
      [&](bool is, uint32_t chain, uint32_t chunk, int stage) {
        if (is) {
          Place<kFwd, 2> from;
          fw.inputs(chain, chunk, from);
          fw.copy(base + stage * Tile::kBytes, from);
        }
        copies_commit();
      });
}

// Sums over the `lanes` (a power of two) neighbours of a lane of N values
// each: every round gives half of the values to the partner and takes its
// half of the others', so 16 shuffles do for 16 values over 32 lanes. On
// return val[0..left) of a lane are the sums of the steps first..first + left,
// the same in the lanes that differ in bits from log2(N) on.
template <int N>
MPB_D void sum_over_lanes(float (&val)[N], int lane, int lanes, int& first, int& left) {
  first = 0;
  left = N;
#pragma unroll
  for (int half = N / 2, bit = 1; half > 0; half >>= 1, bit <<= 1) {
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
  for (int bit = N; bit < 32; bit <<= 1)
    if (bit < lanes) val[0] += __shfl_xor_sync(0xffffffffu, val[0], bit);
}

template <class X, class G, bool SIG, int V, bool SHARED>
struct BwdTile {
  static constexpr int kBwd = bwd_steps(SIG, (int)sizeof(G), V, SHARED);
  using CX = Column<X, V>;
  using CG = Column<G, SHARED ? 1 : V>;
  using HG = HeadGates<G, kBwd>;
  static constexpr uint32_t kH = CX::bytes(kBwd), kX = 2 * kH, kG = SIG ? 3 * kH : kX, kBytes = kG + CG::bytes(kBwd);
  static constexpr int kStages = kRing / kBytes < 3 ? kRing / kBytes : 3;  // of a walk
  static_assert(kStages >= 2, "a tile is copied while another is computed");
};

// As Forward, from the last step to the first. The gate is taken from shared
// memory twice rather than kept (backward moves twice the bytes per element,
// so the second exponential fits beside them).
template <class X, class G, bool SIG, int V, bool SHARED>
struct Backward {
  using Tile = BwdTile<X, G, SIG, V, SHARED>;
  static constexpr int kBwd = Tile::kBwd;
  const ScanArgs& p;
  const int64_t in_st[4], out_st[2];
  const int lane, warp;
  int gate_slot;
  uint32_t half0[4];  // bit 1 of the addresses of single 16-bit elements at the sequence's last step
  size_t state_at;
  MPB_D explicit Backward(const ScanArgs& args)
      : p(args), in_st{-args.dh_st * (int64_t)sizeof(X), -args.h_st * (int64_t)sizeof(X), -args.x_st * (int64_t)sizeof(X),
                       -args.g_st * (int64_t)sizeof(G)},
        out_st{-args.D * (int64_t)sizeof(X), -args.H * (int64_t)sizeof(G)}, lane(threadIdx.x & 31), warp(threadIdx.x >> 5) {}
  MPB_D void inputs(uint32_t chain, uint32_t chunk, Place<kBwd, 4>& f) const {
    const Lane l = place<V, SHARED>(p, chain, lane);
    const int64_t r0 = (int64_t)chunk * p.steps + warp * kBwd, t0 = p.T - 1 - r0;
    auto row = [&](const void* q, int64_t sb, int64_t st, int64_t t) { return (const char*)((const X*)q + l.b * sb + t * st); };
    const char* g = (const char*)((const G*)p.gate + l.b * p.g_sb + t0 * p.g_st);
    f.at[0] = at_lane<typename Tile::CX, X>(p, row(p.dh, p.dh_sb, p.dh_st, t0), l, in_st[0], lane);
    f.at[1] = at_lane<typename Tile::CX, X>(p, row(p.hsaved, p.h_sb, p.h_st, t0 - 1), l, in_st[1], lane);
    f.at[2] = at_lane<typename Tile::CX, X>(p, row(p.x, p.x_sb, p.x_st, t0), l, in_st[2], lane);
    f.at[3] = SHARED ? g + l.head * sizeof(G) : at_lane<typename Tile::CG, G>(p, g, l, in_st[3], lane);
    f.wide = wide_lane<V>(l, lane);
    f.end = (int)(p.T - r0);
    f.left = l.in ? f.end : 0;
    f.heads = SHARED ? (int)(p.H - l.head < p.heads_per ? p.H - l.head : p.heads_per) : 0;
  }
  MPB_D void copy(uint32_t q, const Place<kBwd, 4>& f) const {
    auto column = [&](uint32_t to, int k, int less) {
      copy_column<typename Tile::CX, kBwd>(p, to, f.at[k], in_st[k], f.left - less, f.end - less, f.wide);
    };
    column(q, 0, 0);
    column(q + Tile::kH, 1, 1);  // h[-1] is h0
    if (SIG) column(q + Tile::kX, 2, 0);
    if constexpr (SHARED) Tile::HG::copy(q + Tile::kG, f.at[3], in_st[3], f.end, (int)p.heads_per, f.heads, p.by_heads_per);
    else copy_column<typename Tile::CG, kBwd>(p, q + Tile::kG, f.at[3], in_st[3], f.left, f.end, f.wide);
  }
  MPB_D void sub_words(const Lane& l) {
    gate_slot = l.slot;
    auto bit = [&](const void* q, int64_t sb, int64_t st, int64_t t) {
      return (uint32_t)(uintptr_t)((const X*)q + l.b * sb + t * st + l.ch);
    };
    half0[0] = bit(p.dh, p.dh_sb, p.dh_st, p.T - 1);
    half0[1] = bit(p.hsaved, p.h_sb, p.h_st, p.T - 2);
    half0[2] = bit(p.x, p.x_sb, p.x_st, p.T - 1);
    half0[3] = (uint32_t)(uintptr_t)((const G*)p.gate + l.b * p.g_sb + (p.T - 1) * p.g_st + l.gate);
  }
  MPB_D void output(uint32_t chain, uint32_t chunk, Place<kBwd, 2>& f) {
    const Lane l = place<V, SHARED>(p, chain, lane);
    const int64_t r0 = (int64_t)chunk * p.steps + warp * kBwd, t0 = p.T - 1 - r0;
    f.at[0] = (const char*)((const X*)p.dx + (l.b * p.T + t0) * p.D + l.ch);
    f.at[1] = (const char*)((const G*)p.dgate + (l.b * p.T + t0) * p.H + l.gate);
    f.left = l.in ? (int)(p.T - r0) : 0;
    state_at = (size_t)(l.b * p.D + l.ch);
    sub_words(l);
  }
  // r0: the warp's first step in the tile, counted from the end
  MPB_D uint32_t half(int k, uint32_t r0, int i) const { return half0[k] + (r0 + i) * (uint32_t)in_st[k]; }
  MPB_D void gate_at(const char* mine, int i, uint32_t r0, Floats<V>& a, Floats<V>& om) const {
    if constexpr (SHARED) gates_of<SIG, V>(Tile::HG::get(mine + Tile::kG, i * (int)p.heads_per + gate_slot, half(3, r0, i)), a, om);
    else gates_of<SIG, V>(Tile::CG::get(mine + Tile::kG, i, half(3, r0, i)), a, om);
  }
  MPB_D void fold(const char* mine, uint32_t r0, Floats<V>& ma, Floats<V>& mb) const {
    ma = vset<V>(1.0f), mb = vset<V>(0.0f);
#pragma unroll
    for (int i = 0; i < kBwd; ++i) {
      Floats<V> a, om;
      gate_at(mine, i, r0, a, om);
      ma = vmul(ma, a);
      mb = vmul(a, vadd(mb, unpack(Tile::CX::get(mine, i, half(0, r0, i)))));
    }
  }
  // Step i from `in`, u of the step after, with low = h[t - 1]: writes dx and the gradient of a gate of the lane's
  // own, leaves u in `in` and returns da.
  MPB_D Floats<V> step(const char* mine, int i, uint32_t r0, Floats<V> low, char*& dx, char*& dg, Floats<V>& in) const {
    Floats<V> a, om;
    gate_at(mine, i, r0, a, om);
    const Floats<V> s = vadd(unpack(Tile::CX::get(mine, i, half(0, r0, i))), in);
    if constexpr (SIG) low = vfma(unpack(Tile::CX::get(mine + Tile::kX, i, half(2, r0, i))), vset<V>(-1.0f), low);
    put_global(dx, pack<X>(SIG ? vmul(om, s) : s));
    dx = ahead_by(dx, out_st[0]);
    in = vmul(a, s);
    const Floats<V> da = vmul(s, low);
    if constexpr (!SHARED) {
      put_global(dg, pack<G>(SIG ? vmul(da, vmul(a, om)) : da));
      dg = ahead_by(dg, out_st[1]);
    }
    return da;
  }
  static MPB_D float over_channels(Floats<V> da) { return V == 2 ? vget(da, 0) + vget(da, 1) : vget(da, 0); }
  MPB_D Floats<V> before(const char* mine, int i, uint32_t r0) const {
    return unpack(Tile::CX::get(mine + Tile::kH, i, half(1, r0, i)));
  }
  // h0 before the first step of the sequence, which is the last of `to`
  MPB_D Floats<V> before_any(const char* mine, int i, uint32_t r0, const Place<kBwd, 2>& to) const {
    Floats<V> low = before(mine, i, r0);
    if (to.left - 1 == i)
#pragma unroll
      for (int v = 0; v < V; ++v) vput(low, v, p.h0 ? p.h0[state_at + v] : 0.0f);
    return low;
  }
  MPB_D void ended(const Place<kBwd, 2>& to, int n, Floats<V> in) const {
    if (p.dh0 && n > 0 && n == to.left)
#pragma unroll
      for (int v = 0; v < V; ++v) p.dh0[state_at + v] = vget(in, v);
  }
  // The warp's steps from the state `in` (u of the step after).
  MPB_D void write(const char* mine, uint32_t chain, uint32_t r0, const Place<kBwd, 2>& to, Floats<V>& in) const {
    const int n = to.steps();
    char *dx = const_cast<char*>(to.at[0]), *dg = const_cast<char*>(to.at[1]);
    float sum[kBwd];
    if (__all_sync(0xffffffffu, to.left > kBwd)) {
#pragma unroll
      for (int i = 0; i < kBwd; ++i) sum[i] = over_channels(step(mine, i, r0, before(mine, i, r0), dx, dg, in));
    } else {
#pragma unroll
      for (int i = 0; i < kBwd; ++i) {
        sum[i] = 0.0f;
        if (i < n) sum[i] = over_channels(step(mine, i, r0, before_any(mine, i, r0, to), dx, dg, in));
      }
    }
    ended(to, n, in);
    if constexpr (SHARED) head_sums(sum, chain, r0);
  }
  // The same for a warp in turn, in short code.
  MPB_D void write_in_turn(const char* mine, uint32_t chain, uint32_t r0, const Place<kBwd, 2>& to, Floats<V>& in) const {
    const int n = to.steps();
    char *dx = const_cast<char*>(to.at[0]), *dg = const_cast<char*>(to.at[1]);
    const Heads q(p, chain, lane);
#pragma unroll 1
    for (int i = 0; i < kBwd; ++i) {
      float sum = 0.0f;
      if (i < n) sum = over_channels(step(mine, i, r0, before_any(mine, i, r0, to), dx, dg, in));
      if constexpr (SHARED) {
        for (int bit = 1; bit < q.lanes; bit <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, bit);
        if (q.at == 0) put_head(q, p.T - 1 - (int64_t)r0 - i, sum);
      }
    }
    ended(to, n, in);
  }
  // A head's lanes: a power of two of them, or the whole warp (idle lanes add zeros).
  struct Heads {
    int lanes, at;
    int64_t b, head;
    uint32_t group;
    MPB_D Heads(const ScanArgs& p, uint32_t chain, int lane) {
      lanes = p.heads_per > 1 ? (int)p.lanes_per : 32;
      at = p.heads_per > 1 ? lane & (lanes - 1) : lane;
      b = p.by_groups.div(chain);
      group = chain - (uint32_t)b * p.groups;
      head = p.groups_per > 1 ? (int64_t)p.by_groups_per.div(group)
                              : (int64_t)group * p.heads_per + (p.heads_per > 1 ? lane / lanes : 0);
    }
  };
  // The sum over a head's channels (of the group) at step t.
  MPB_D void put_head(const Heads& q, int64_t t, float sum) const {
    if (t < 0 || q.head >= p.H) return;
    const int64_t bt = q.b * p.T;
    if (p.groups_per > 1) {
      p.part[((bt + t) * p.H + q.head) * p.groups_per + (q.group - (uint32_t)q.head * p.groups_per)] = sum;
    } else {
      float a, om;
      gate_of<SIG, G>(to_f(((const G*)p.gate)[q.b * p.g_sb + t * p.g_st + q.head]), a, om);
      ((G*)p.dgate)[(bt + t) * p.H + q.head] = Cvt<G>::from(SIG ? sum * (a * om) : sum);
    }
  }
  MPB_D void head_sums(float (&sum)[kBwd], uint32_t chain, uint32_t r0) const {
    const Heads q(p, chain, lane);
    int first, left;
    sum_over_lanes(sum, lane, q.lanes, first, left);
    // of the lanes that hold the same sums the one with the upper bits clear writes
    if (q.at >= kBwd) return;
#pragma unroll
    for (int i = 0; i < kBwd; ++i)
      if (i < left) put_head(q, p.T - 1 - (int64_t)r0 - (first + i), sum[i]);
  }
};

template <class X, class G, bool SIG, int V, bool SHARED>
__global__ void __launch_bounds__(kWarps * 32, 2) k_gscan_bwd_walk(ScanArgs p) {
  using Tile = BwdTile<X, G, SIG, V, SHARED>;
  constexpr int NST = Tile::kStages, kBwd = Tile::kBwd;
  extern __shared__ __align__(16) char ring[];
  __shared__ Shared<V> sh;
  Backward<X, G, SIG, V, SHARED> bw(p);
  const uint32_t base = smem_u32(ring);
  if (p.status && blockIdx.x == 0 && threadIdx.x == 0) *p.status = MPB_OK;  // nothing waits
  Order cur, ahead;
  Place<kBwd, 4> from;
  Place<kBwd, 2> to;
  auto copy = [&](int s) {  // the walk's next tile into stage s
    if (ahead.here(p)) {
      if (ahead.chunk == 0) bw.inputs(ahead.chain, 0, from);
      else from.move(p, bw.in_st);
      bw.copy(base + s * Tile::kBytes, from);
      ahead.next(p);
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) copy(s);
  int stage = 0;
  Floats<V> carry = vset<V>(0.0f);
  for (int it = 0; cur.here(p); ++it) {
    __syncwarp();  // the stage that is filled next has been read by every lane
    copy(stage == 0 ? NST - 1 : stage - 1);
    if (cur.chunk == 0) {
      bw.output(cur.chain, 0, to);
#pragma unroll
      for (int v = 0; v < V; ++v) vput(carry, v, to.left > 0 && p.dstate ? p.dstate[bw.state_at + v] : 0.0f);
    } else {
      to.move(p, bw.out_st);
    }
    copies_wait<NST - 1>();
    __syncwarp();  // the words that other lanes have copied
    const char* mine = ring + stage * Tile::kBytes;
    const uint32_t r0 = cur.chunk * p.steps + bw.warp * kBwd;
    Floats<V> ma, mb, in;
    bw.fold(mine, r0, ma, mb);
    const bool sound = SIG || to.left < kBwd || numbers<V>(ma, mb);
    const bool turns = join<V, !SIG>(sh, it & 1, bw.warp, bw.lane, sound, ma, mb, carry, in);
    if (turns) {
      start_turn<V>(sh, bw.warp, bw.lane, in);
      bw.write_in_turn(mine, cur.chain, r0, to, in);
      end_turn<V>(sh, bw.warp, bw.lane, in);
      carry = *reinterpret_cast<const Floats<V>*>(&sh.carry[bw.lane * V]);
    } else {
      bw.write(mine, cur.chain, r0, to, in);
    }
    if (blockDim.x == 32) carry = in;
    cur.next(p);
    stage = stage + 1 == NST ? 0 : stage + 1;
  }
}

template <class X, class G, bool SIG, int V, bool SHARED>
__global__ void __launch_bounds__(kWarps * 32, 2) k_gscan_bwd_far(ScanArgs p) {
  using Tile = BwdTile<X, G, SIG, V, SHARED>;
  constexpr int kBwd = Tile::kBwd;
  extern __shared__ __align__(16) char ring[];
  __shared__ Shared<V> sh;
  Backward<X, G, SIG, V, SHARED> bw(p);
  const uint32_t base = smem_u32(ring);
  auto r0_of = [&](uint32_t chunk) { return chunk * p.steps + bw.warp * kBwd; };
  look_back_tiles<V, !SIG>(
      p, sh, bw.warp, bw.lane,
      [&](uint32_t chain, uint32_t chunk, int stage, int side) {
        const Lane l = place<V, SHARED>(p, chain, bw.lane);
        bw.sub_words(l);
        Floats<V> ma, mb;
        bw.fold(ring + stage * Tile::kBytes, r0_of(chunk), ma, mb);
        if (!SIG && !(l.in && p.T - r0_of(chunk) >= kBwd)) ma = vset<V>(1.0f), mb = vset<V>(0.0f);
        put_map<V>(sh, side, bw.warp, bw.lane, ma, mb);
      },
      [&](uint32_t chain, uint32_t chunk, float (&c)[V]) {
        const Lane l = place<V, SHARED>(p, chain, bw.lane);
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = chunk < 32 && l.in && p.dstate ? p.dstate[l.b * p.D + l.ch + v] : 0.0f;
      },
      [&](uint32_t chain, uint32_t chunk, int stage, Floats<V>& in, auto in_turn) {
        Place<kBwd, 2> to;
        bw.output(chain, chunk, to);
        if constexpr (decltype(in_turn)::value) bw.write_in_turn(ring + stage * Tile::kBytes, chain, r0_of(chunk), to, in);
        else bw.write(ring + stage * Tile::kBytes, chain, r0_of(chunk), to, in);
      },
      [&](bool is, uint32_t chain, uint32_t chunk, int stage) {
        if (is) {
          Place<kBwd, 4> from;
          bw.inputs(chain, chunk, from);
          bw.copy(base + stage * Tile::kBytes, from);
        }
        copies_commit();
      });
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
  gate_of<SIG, G>(to_f(((const G*)p.gate)[b * p.g_sb + t * p.g_st + head]), a, om);
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
  XP xw;
  GP gw;
  xw.w = *reinterpret_cast<const typename XP::W*>((const X*)p.x + b * p.x_sb + d);
  gw.w = *reinterpret_cast<const typename GP::W*>((const G*)p.gate + b * p.g_sb + (SHARED ? by_p.div(d) : d));
  float* s = p.state + b * p.D + d;
  Floats<V> h, a, om;
  const Floats<V> x = unpack(xw);
#pragma unroll
  for (int v = 0; v < V; ++v) vput(h, v, s[v]);
  gates_of<SIG, V>(gw, a, om);
  h = vfma(a, h, SIG ? vmul(om, x) : x);
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = vget(h, v);
  *reinterpret_cast<typename XP::W*>((X*)p.h + b * p.D + d) = pack<X>(h).w;
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

// From this many chains on a block walks a chain; one number for all types, modes and
// directions. T = 4096, walked / by look-back in us, forward then backward:
//   chains   bf16 sigmoid          bf16 linear, per head   f32 linear
//     32      51 / 27    96 / 41    39 / 26    72 / 43      33 / 22   49 / 33
//     64      51 / 43    96 / 70    39 / 38    72 / 64      33 / 37   49 / 55
//     96      51 / 56    97 / 90    39 / 51    73 / 85      35 / 47   51 / 70
//    128      51 / 67    97 / 111   39 / 60    74 / 107     35 / 57   54 / 84
//    160      78 / 78   150 / 129   62 / 69   101 / 129     58 / 65   85 / 97
//    256      78 / 110  150 / 184   66 / 93   104 / 201     75 / 91  100 / 148
// So it loses 12 % for f32 at 64 chains, 8 % for sigmoid backward at 96, and 16 %
// for that at 160, where some SMs walk two chains and some one.
constexpr uint32_t kWalkFrom = 80;

// Copies of 16 bytes: every row of every input starts on such a boundary, and
// so does every head. (Of 16-bit types with two channels per lane; with one the
// words in shared memory are wider than the elements.)
bool wide(const ScanArgs& p, int V, int x_dt, int g_dt, bool backward, bool sig) {
  const int64_t xs = x_dt == MPB_F32 ? 4 : 2, gs = g_dt == MPB_F32 ? 4 : 2;
  if (xs * V < 4) return false;
  auto fits = [](const void* q, int64_t sb, int64_t st, int64_t size) {
    return (uintptr_t)q % 16 == 0 && sb * size % 16 == 0 && st * size % 16 == 0;
  };
  if (p.D * xs % 16 != 0 || (p.H != p.D && p.P * xs % 16 != 0)) return false;
  if ((!backward || sig) && !fits(p.x, p.x_sb, p.x_st, xs)) return false;
  if (p.H == p.D && !fits(p.gate, p.g_sb, p.g_st, gs)) return false;
  return !backward || (fits(p.dh, p.dh_sb, p.dh_st, xs) && fits(p.hsaved, p.h_sb, p.h_st, xs));
}

// The channel groups and tiles for V channels per lane and `per` steps per warp.
void lay_out(ScanArgs& p, int V, int per) {
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
  const int64_t warps = (p.T + per - 1) / per;
  p.steps = (int)(warps < kWarps ? warps : kWarps) * per;
  p.chains = (uint32_t)(p.B * p.groups);
  p.chunks = (uint32_t)((p.T + p.steps - 1) / p.steps);
  p.walk = p.chunks == 1 || p.chains >= kWalkFrom;
  p.by_groups = FastDiv(p.groups);
  p.by_groups_per = FastDiv(p.groups_per);
  p.by_lanes_per = FastDiv(p.lanes_per);
  p.by_heads_per = FastDiv(p.heads_per);
  p.by_chains = FastDiv(p.chains);
}

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

// Scratch: {ticket, status}, states and maps of the tiles (cleared by the call), sums of wide heads.
size_t scratch_of(ScanArgs& p, int V, bool backward, void* base, size_t* cleared) {
  size_t at = 16;
  char* q = (char*)base;
  *cleared = 0;
  if (!p.walk) {
    const size_t words = (size_t)p.chains * p.chunks * 32 * V;
    p.ticket = (uint32_t*)q;
    p.status = (uint32_t*)(q + 4);
    p.maps = (uint64_t*)(q + 16);
    p.states = (uint32_t*)(q + 16 + words * 8);
    at = *cleared = align16(16 + words * 12);
  }
  if (backward && p.groups_per > 1) {
    p.part = (float*)(q + at);
    at += align16((size_t)(p.B * p.T * p.H) * p.groups_per * sizeof(float));
  }
  return at > 16 ? at : 0;
}

// Enough for either V and number of steps: the choice needs addresses, strides and the mode.
size_t scratch_need(ScanArgs p, bool backward) {
  size_t most = 0, cleared;
  for (int V = 1; V <= 2; ++V)
    for (int per : {8, 16}) {
      if (!backward && per != kFwd) continue;
      lay_out(p, V, per);
      const size_t n = scratch_of(p, V, backward, nullptr, &cleared);
      most = n > most ? n : most;
    }
  return most;
}

int prepare(const char* what, ScanArgs& p, int V, int per, bool backward, void* scratch, cudaStream_t s) {
  lay_out(p, V, per);
  size_t cleared;
  if (scratch_need(p, backward)) p.status = (uint32_t*)((char*)scratch + 4);
  scratch_of(p, V, backward, scratch, &cleared);
  if (cleared) return cuda_check(cudaMemsetAsync(scratch, 0, cleared, s), what);
  return MPB_OK;
}

// SMEM: the block's tiles under way.
template <auto kernel, int SMEM>
int launch_tiles(const char* what, const ScanArgs& p, int per, cudaStream_t s) {
  if (int rc = allow_smem<kernel, SMEM>(what)) return rc;
  const uint32_t most = (uint32_t)sm_count() * 2, tiles = p.walk ? p.chains : p.chains * p.chunks;
  kernel<<<tiles < most ? tiles : most, (unsigned)(p.steps / per) * 32, SMEM, s>>>(p);
  return launch_check(what);
}

template <class X, class G, bool SIG, int V, bool SHARED>
int launch_fwd_v(const ScanArgs& p, cudaStream_t s) {
  using Tile = FwdTile<X, G, V, SHARED>;
  const char* what = "gated_scan";
  return p.walk ? launch_tiles<k_gscan_walk<X, G, SIG, V, SHARED>, Tile::kStages * Tile::kBytes>(what, p, kFwd, s)
                : launch_tiles<k_gscan_far<X, G, SIG, V, SHARED>, 3 * Tile::kBytes>(what, p, kFwd, s);
}

template <class X, class G, bool SIG, int V, bool SHARED>
int launch_bwd_v(const ScanArgs& p, cudaStream_t s) {
  using Tile = BwdTile<X, G, SIG, V, SHARED>;
  const char* what = "gated_scan_backward";
  return p.walk ? launch_tiles<k_gscan_bwd_walk<X, G, SIG, V, SHARED>, Tile::kStages * Tile::kBytes>(what, p, Tile::kBwd, s)
                : launch_tiles<k_gscan_bwd_far<X, G, SIG, V, SHARED>, 3 * Tile::kBytes>(what, p, Tile::kBwd, s);
}

template <class X, class G, bool SIG>
int launch_fwd(ScanArgs& p, int V, void* scratch, cudaStream_t s) {
  if (int rc = prepare("gated_scan", p, V, kFwd, false, scratch, s)) return rc;
  constexpr int W = sizeof(X) == 2 ? 2 : 1;
  if (p.H != p.D) return V == 2 ? launch_fwd_v<X, G, SIG, W, true>(p, s) : launch_fwd_v<X, G, SIG, 1, true>(p, s);
  return V == 2 ? launch_fwd_v<X, G, SIG, W, false>(p, s) : launch_fwd_v<X, G, SIG, 1, false>(p, s);
}

template <class X, class G, bool SIG>
int launch_bwd(ScanArgs& p, int V, void* scratch, cudaStream_t s) {
  if (int rc = prepare("gated_scan_backward", p, V, bwd_steps(SIG, (int)sizeof(G), V, p.H != p.D), true, scratch, s)) return rc;
  constexpr int W = sizeof(X) == 2 ? 2 : 1;
  if (p.H == p.D) return V == 2 ? launch_bwd_v<X, G, SIG, W, false>(p, s) : launch_bwd_v<X, G, SIG, 1, false>(p, s);
  if (int rc = V == 2 ? launch_bwd_v<X, G, SIG, W, true>(p, s) : launch_bwd_v<X, G, SIG, 1, true>(p, s)) return rc;
  if (p.groups_per == 1) return MPB_OK;
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
  if (B > 0x7fffffff || T > 0x7ff00000 || D > 0x7fffffff || H > 0x7fffffff ||
      (double)B * (double)(D + 32) * ((double)T / 128 + 1) > 2.0e9)
    return fail(MPB_ERR_SHAPE, "%s: (%lld, %lld, %lld) is too large", what, (long long)B, (long long)T, (long long)D);
  return MPB_OK;
}

int check_scratch(const char* what, size_t need, const void* scratch, size_t bytes) {
  if (need > bytes || (need && !scratch))
    return fail(MPB_ERR_SCRATCH, "%s: %zu bytes of scratch, %zu needed", what, bytes, need);
  if (need && (uintptr_t)scratch % 16 != 0) return fail(MPB_ERR_INVALID, "%s: scratch not 16-byte aligned", what);
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
    p.wide = wide(p, V, x_dtype, gate_dtype, false, mode == MPB_SCAN_SIGMOID);
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
    if (B * D == 0) {  // gates of no channels: sums of nothing
      const int64_t n = B * T * H;
      if (n == 0) return (int)MPB_OK;
      if (!dgate) return fail(MPB_ERR_INVALID, "%s: null pointer", what);
      return cuda_check(cudaMemsetAsync(dgate, 0, (size_t)n * sizeof(gt), s), what);
    }
    if (T == 0) return pass_state(what, dstate, dh0, B * D, s);
    if (!dh || !x || !gate || !h || !dx || !dgate) return fail(MPB_ERR_INVALID, "%s: null pointer", what);
    if (int rc = check_scratch(what, scratch_need(p, true), scratch, scratch_bytes)) return rc;
    const int V = pairs(p, x_dtype, gate_dtype, true) ? 2 : 1;
    p.wide = wide(p, V, x_dtype, gate_dtype, true, mode == MPB_SCAN_SIGMOID);
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

int mpb_gated_scan_status(const void* scratch, mpb_stream_t stream) {
  uint32_t status = 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (!scratch) return MPB_OK;
  if (int rc = cuda_check(cudaMemcpyAsync(&status, (const char*)scratch + 4, 4, cudaMemcpyDeviceToHost, s), "gated_scan_status"))
    return rc;
  if (int rc = cuda_check(cudaStreamSynchronize(s), "gated_scan_status")) return rc;
  return status ? fail((int)status, "gated_scan: a bounded wait for an earlier tile gave up") : MPB_OK;
}

}  // extern "C"

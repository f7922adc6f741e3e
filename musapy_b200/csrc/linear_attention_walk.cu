// Linear attention of bf16 heads of up to 128 channels: a block walks a head's chunks (or those of one segment of
// it) with the state on chip, so that q, k and v are read and o is written once. The formulas are those of
// linear_attention.cu. Per chunk of 64 steps the tensor core makes
//
//   A = q k'           (steps x steps)        -> P = D A, as two bf16 numbers, back to shared memory
//   E = (w k)' v       (channels x channels)  w_j = e^(G_C - G_j); w k as three bf16 numbers that sum to it
//   X' = S' q', Y' = v' P'  (channels of v x steps),  o = scale (e^(G_i) X + Y)
//
// and the state's threads S <- e^(G_C) S + E in float, from which X takes S as two bf16 numbers. Two numbers keep 16 bits, so
// that outputs are off by their own rounding (1.66e-3 of their norm; with P and S rounded once to bf16, 2.35e-3, in 211 us
// instead of 263 for the first case below). The sum and X tie a chunk to the next.
//
// Roles of the block's warps: 8 keep the state (in tensor memory, half a row of channels per thread), 4 write
// outputs (where q was, for a copy to take them), 8 weigh and split k, 4 make P, one copies in (TMA, two or three chunks in
// shared memory), one copies out, one issues the matrix instructions, one makes the decays. They meet at mbarriers; every wait gives up after two seconds, sets the status
// word and ends the block, whose results are NaN.
//
// What it takes: 8 x 4096 x 16 heads of 128, 263 us (2.1 TB/s; 553 MB, 85 us at the copy rate; without this kernel 1464 us);
// 1 x 32768 x 8 heads of 64 in 18 segments 148 us with the walk that finds their states. Without outputs, the states of all chunks
// kept in float, 4 x 4096 x 16 heads of 128 take 100 us (2.7 TB/s; by each thread's own stores 149). The
// tensor core has 40 instructions a chunk, each of which takes 73 cycles by itself whatever its columns up to 128 (its left operand's
// 4 KB come at 64 bytes a cycle), so that both pieces of P are one right operand of 128 columns; those of S, a left
// operand, are two. From one chunk to the next pass X (16 instructions) and the state's sum, which Y and the next scores
// overlap. Issue order E, X, Y, next scores: 279 us for the first case with the L2 flushed, 174 for its heads of 64; X, Y, next scores, E:
// 298 and 206; X, E, Y, next scores: 279 and 180. Three chunks of 128 and 128 channels do not fit beside the pieces; there two are under way.
//
// Operands lie as the copies leave them, rows of 128 bytes in the 128-byte swizzle; what is needed transposed (k, v, S as
// left operands, v as a right one) is read "along the other dim" by the tensor core. Every matrix
// instruction has 128 rows: of operands with 64, the second half is whatever lies behind them in shared memory, and its
// results are not read.
#include <cuda.h>
#include <atomic>
#include "async_copy.cuh"
#include "common.cuh"
#include "internal.h"
#include "linear_attention.cuh"
#include "rows.cuh"

namespace mpb {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kThreads = 28 * 32;
constexpr int kMostStages = 3;  // chunks of q, k, v in shared memory
constexpr int kSlots = 4;    // chunks whose decays are there
constexpr int kPieces = 3;   // of w k: the code takes them to be three
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kColA = 0, kColX = 64, kColY = 128, kColE = 256, kColS = 384;  // Y: of P's two pieces, side by side

// A bounded wait in few instructions: there are many of them, and code in them that reads the clock, though it does not run,
// took the first case above from 270 to 310 us. A try that fails has itself waited for 4 us (3.98 measured, by 1 to 896
// threads at once), so that a number of tries is a time.
constexpr uint32_t kTryNs = 4000;
MPB_D bool mbar_wait_for(uint32_t bar, uint32_t parity, int tries) {
#pragma unroll 1
  for (int i = 0; i < tries; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return false;
}

// ------------------------------------------------------- tensor core
MPB_D void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
MPB_D void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
MPB_D void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
MPB_D void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
MPB_D void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// An operand's descriptor in two halves: the lower one moves with the address, in units of 16 bytes.
struct Operand {
  uint32_t lo, hi;
};
template <bool ADD>
MPB_D void mma(uint32_t d, Operand a, int a_off, Operand b, int b_off, uint32_t idesc) {
  const uint32_t al = a.lo + (uint32_t)(a_off >> 4), bl = b.lo + (uint32_t)(b_off >> 4);
  if (ADD)
    asm volatile(
        "{\n\t.reg .b64 da, db;\n\t.reg .pred p;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.eq.u32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d),
        "r"(al), "r"(a.hi), "r"(bl), "r"(b.hi), "r"(idesc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .b64 da, db;\n\t.reg .pred p;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.u32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d),
        "r"(al), "r"(a.hi), "r"(bl), "r"(b.hi), "r"(idesc)
        : "memory");
}
MPB_D void tmem_load(uint32_t (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
MPB_D void tmem_load(uint32_t (&r)[8], uint32_t at) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at));
}
MPB_D void tmem_store(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
      : "memory");
}
MPB_D void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
MPB_D void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A shared memory operand in the 128-byte swizzle: `group`, bytes between groups of eight rows of 128 bytes; `block`,
// between blocks of 64 elements where the rows run along the other dim.
MPB_D Operand operand(uint32_t at, uint32_t block, uint32_t group) {
  return {((at >> 4) & 0x3fff) | (block >> 4) << 16, (group >> 4) | 1u << 14 | 2u << 29};
}
// bf16 operands, float sums, 128 rows, n columns; ta, tb: an operand whose rows run along its own dim, not the summed one.
constexpr uint32_t instruction(int n, bool ta, bool tb) {
  return 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)ta << 15 | (uint32_t)tb << 16 | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}

MPB_D void tma_tile(uint32_t dst, const CUtensorMap* map, int x, int h, int t, int b, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(h), "r"(t), "r"(b), "r"(bar)
      : "memory");
}

MPB_D void tma_write(const CUtensorMap* map, uint32_t src, int x, int h, int t, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map), "r"(src), "r"(x),
               "r"(h), "r"(t), "r"(b)
               : "memory");
}

// Two floats as two bf16 numbers each: their rounding, and that of what it leaves.
MPB_D void two_pieces(float2 f, uint32_t& high, uint32_t& low) {
  high = pack<bf16>(f).w;
  low = pack<bf16>(vfma(make_float2(__uint_as_float(high << 16), __uint_as_float(high & 0xffff0000u)), vset<2>(-1.0f), f)).w;
}

// ------------------------------------------------------------ layout
enum Bar { kFull0, kFull1, kFull2, kEmpty0, kEmpty1, kEmpty2, kDec0, kDec1, kDec2, kDec3, kADone0, kADone1, kAFree, kPReady, kWReady, kEDone, kEFree, kSReady,
           kXDone, kODone, kOFree, kOReady0, kOReady1, kOReady2, kOEmpty, kFree0, kFree1, kFree2, kFree3, kEnd, kBars };

template <int DK, int DV, bool OUT>
struct Layout {
  static constexpr int kBlock = 64 * 128;  // 64 steps of 64 channels
  static constexpr int q = 0, k = q + (OUT ? DK / 64 * kBlock : 0), v = k + DK / 64 * kBlock, kStage = v + DV / 64 * kBlock;
  // three chunks of 128 and 128 channels do not fit beside the two pieces of S and P
  static constexpr int kStages = OUT && DK + DV == 256 ? 2 : kMostStages;
  // The first piece of w k takes the place of k. A left operand has 128 rows, and where it holds 64 the other half is read
  // from what follows: S behind W, P behind S.
  static constexpr int W = kStages * kStage, S = W + (kPieces - 1) * (DK / 64) * kBlock;
  static constexpr int kPieceS = DV / 64 * DK * 128, P = S + 2 * kPieceS, decays = P + 2 * kBlock;
  static constexpr int bars = decays + kSlots * ((int)sizeof(ChunkDecay) + 15) / 16 * 16, tmem = bars + kBars * 8;
  static constexpr int bytes = tmem + 16 + 1024;  // the copies' rows want 1024-byte alignment
};

struct Maps {
  CUtensorMap q, k, v, o;
};

// What a block leaves that gave up: NaN in the place of all its results, which also reaches what is made from its states.
// (Not inlined: in the kernel's own text it took the first case above from 263 to 280 us.)
template <bool OUT>
__device__ __noinline__ void leave_nan(const Walk& p) {
  const Shape& d = p.d;
  const int seg = (int)(blockIdx.x % d.segments);
  const int64_t bh = blockIdx.x / d.segments, size = (int64_t)d.dkp * d.dvp;
  const int c0 = seg * d.per, c1 = min(d.chunks, c0 + d.per);
  auto fill = [&](float* to, int64_t n) {
    for (int64_t i = threadIdx.x; i < n; i += kThreads) to[i] = NAN;
  };
  if (OUT) {
    const int64_t h = bh % d.H, b = bh / d.H, t1 = min((int64_t)c1 * kChunk, d.T);
    for (int64_t t = (int64_t)c0 * kChunk + threadIdx.x / 32; t < t1; t += kThreads / 32)
      for (int c = threadIdx.x % 32; c < d.DV; c += 32) ((bf16*)p.o)[((b * d.T + t) * d.H + h) * d.DV + c] = __float2bfloat16_rn(NAN);
  }
  if (!OUT && p.at) fill(p.at + (bh * d.chunks + c0) * size, (c1 - c0) * size);
  if (d.segments > 1 && p.ends) fill(p.ends + (bh * d.segments + seg) * size, size);
  if (d.segments == 1 && p.last) fill(p.last + bh * d.DK * d.DV, (int64_t)d.DK * d.DV);
}

template <int DK, int DV, bool OUT>
__global__ void __launch_bounds__(kThreads, 1) k_la_walk(const __grid_constant__ Maps maps, const __grid_constant__ Walk p) {
  using L = Layout<DK, DV, OUT>;
  constexpr int kStages = L::kStages;
  extern __shared__ unsigned char raw[];
  const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u;
  unsigned char* mem = raw + (smem - smem_u32(raw));
  ChunkDecay* decays = reinterpret_cast<ChunkDecay*>(mem + L::decays);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Shape& d = p.d;
  const int seg = (int)(blockIdx.x % d.segments);
  const int64_t bh = blockIdx.x / d.segments;
  const int h = (int)(bh % d.H), hq = h / d.share;
  const int64_t b = bh / d.H;
  const int c0 = seg * d.per, c1 = min(d.chunks, c0 + d.per), n_chunks = c1 - c0;
  auto bar = [&](int i) { return smem + L::bars + 8 * i; };
  auto chunk = [&](int n) { return p.rev ? c1 - 1 - n : c0 + n; };
  bool ok = true;
  // true where the phase of chunk n has come
  auto wait = [&](int i, int n) {
    if (ok) ok = mbar_wait_for(bar(i), (uint32_t)n & 1, p.tries);
    return ok;
  };
  auto wait_warp = [&](int i, int n) {
    ok = __all_sync(0xffffffffu, wait(i, n));
    return ok;
  };
  if (tid == 0) {
    for (int i = 0; i < kBars; ++i) {
      const int count = i >= kDec0 && i <= kDec3 ? 32 : i == kAFree || i == kPReady ? 128 : i == kWReady ? 256
                        : i == kEFree || i == kSReady || (!OUT && i == kOReady0) ? 2 * DK : i == kOFree || (i >= kOReady0 && i <= kOReady2) ? DV
                        : OUT && i >= kEmpty0 && i <= kEmpty2 ? 2
                        : i >= kFree0 && i <= kFree3 ? 2 * DK + (OUT ? DV : 0) : 1;
      mbar_init(bar(i), count);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 26) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem + L::tmem), "n"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(mem + L::tmem);
  const uint32_t quarter = tmem + ((uint32_t)(warp & 3) * 32 << 16);
  const int row = (warp & 3) * 32 + lane;
  constexpr uint32_t kOther = L::kBlock;

  if (warp < 8) {  // ------------------------------------------- the state
    if (row < DK) {
      constexpr int kGroups = DV / 32;  // of 16 columns, of a thread: half of its row of the state
      const int col0 = (warp >> 2) * (DV / 2);
      const int64_t size = (int64_t)d.dkp * d.dvp;
      const float* first = nullptr;
      int pitch = 0;
      bool have = false;
      const bool begins = p.rev ? c1 == d.chunks : seg == 0;
      if (begins) {
        first = p.first + bh * d.DK * d.DV + (int64_t)row * d.DV, pitch = d.DV, have = p.first && row < d.DK;
      } else if (p.starts) {
        first = p.starts + (bh * d.segments + seg) * size + (int64_t)row * d.dvp, pitch = d.dvp, have = row < d.dkp;
      }
      unsigned char* s_row = mem + L::S + row * 128;
      const uint32_t s_tmem = quarter + kColS + col0, e_tmem = quarter + kColE + col0;
      // 16 columns of S to shared memory, as two bf16 numbers each: its rounding, and that of what it leaves
      auto put = [&](int g, const uint32_t (&s)[16]) {
        const int c = col0 + g * 16;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t high[4], low[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) two_pieces(make_float2(__uint_as_float(s[8 * k + 2 * j]), __uint_as_float(s[8 * k + 2 * j + 1])), high[j], low[j]);
          unsigned char* to = s_row + c / 64 * (DK * 128) + ((c / 8 % 8 + k ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(to) = make_uint4(high[0], high[1], high[2], high[3]);
          *reinterpret_cast<uint4*>(to + L::kPieceS) = make_uint4(low[0], low[1], low[2], low[3]);
        }
      };
#pragma unroll 1
      for (int g = 0; g < kGroups; ++g) {
        uint32_t s[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c = col0 + g * 16 + i;
          s[i] = have && c < pitch ? __float_as_uint(first[c]) : 0u;
        }
        tmem_store(s_tmem + g * 16, s);
        if (OUT) put(g, s);
      }
      wait_stores();
      if (OUT) {
        proxy_fence();
        mbar_arrive(bar(kSReady));
      }
      float since = 1.0f;
      // The state before each chunk leaves in float, by a copy of 32 columns each from where S's pieces would be.
      const bool keep = !OUT && p.at;
      for (int n = 0; n < n_chunks; ++n) {
        const int c = chunk(n);
        if (!wait_warp(kDec0 + n % kSlots, n / kSlots)) break;
        const float all = decays[n % kSlots].all;
        if (p.since && row == 0 && col0 == 0) p.since[bh * d.chunks + c] = since;
        since = all == 0.0f ? 0.0f : since * all;  // one that overflowed is dropped too
        if (!wait_warp(kEDone, n)) break;
        fence_after();
        if (keep && n > 0 && !wait_warp(kOEmpty, n - 1)) break;
        uint32_t e[2][16], s[2][16];
        tmem_load(e[0], e_tmem);
        tmem_load(s[0], s_tmem);
        if (OUT && !wait_warp(kXDone, n)) {
          wait_loads();
          break;
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          uint32_t(&eg)[16] = e[g & 1], (&sg)[16] = s[g & 1];
          wait_loads();
          if (g + 1 < kGroups) {
            tmem_load(e[g + 1 & 1], e_tmem + (g + 1) * 16);
            tmem_load(s[g + 1 & 1], s_tmem + (g + 1) * 16);
          } else {
            fence_before();
            mbar_arrive(bar(kEFree));
            mbar_arrive(bar(kFree0 + n % kSlots));
          }
          if (keep) {
            const int c = col0 + g * 16;
            unsigned char* to = mem + L::S + c / 32 * (DK * 128) + row * 128;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(to + ((c / 4 % 8 + i ^ (row & 7)) << 4)) = make_uint4(sg[4 * i], sg[4 * i + 1], sg[4 * i + 2], sg[4 * i + 3]);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sg[i] = all == 0.0f ? eg[i] : __float_as_uint(fmaf(all, __uint_as_float(sg[i]), __uint_as_float(eg[i])));
          tmem_store(s_tmem + g * 16, sg);
          if (OUT) put(g, sg);
        }
        wait_stores();
        if (OUT) {
          proxy_fence();
          fence_before();
          mbar_arrive(bar(kSReady));
        } else if (keep) {
          proxy_fence();
          mbar_arrive(bar(kOReady0));
        }
      }
      if (ok) {
        const bool whole = d.segments == 1;
        float* to = whole ? (p.last ? p.last + bh * d.DK * d.DV + (int64_t)row * d.DV : nullptr)
                          : (p.ends ? p.ends + (bh * d.segments + seg) * size + (int64_t)row * d.dvp : nullptr);
        const int width = row < (whole ? d.DK : d.dkp) && to ? (whole ? d.DV : d.dvp) : 0;
        if (p.ends && !whole && row == 0 && col0 == 0) p.since[(bh + d.B * d.H) * d.chunks + seg] = since;
#pragma unroll 1
        for (int g = 0; g < kGroups; ++g) {
          uint32_t s[16];
          tmem_load(s, s_tmem + g * 16);
          wait_loads();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (col0 + g * 16 + i < width) to[col0 + g * 16 + i] = __uint_as_float(s[i]);
        }
      }
    }
  } else if (warp < 12) {  // ----------------------------------- outputs
    if (OUT && row < DV) {
      const float2 scale = vset<2>(p.scale);
      for (int n = 0; n < n_chunks; ++n) {
        if (!wait_warp(kDec0 + n % kSlots, n / kSlots) || !wait_warp(kODone, n)) break;
        fence_after();
        const float* into = decays[n % kSlots].into;
        // the outputs take the place of q, laid out like it, and are copied from there
        unsigned char* to = mem + (n % kStages) * L::kStage + row / 64 * L::kBlock + row % 8 * 2;
        const int word = row / 8 % 8;
        uint32_t two[32];  // outputs of two steps each
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          uint32_t x[8], y[8], z[8];
          tmem_load(x, quarter + kColX + g * 8);
          tmem_load(y, quarter + kColY + g * 8);
          tmem_load(z, quarter + kColY + 64 + g * 8);
          wait_loads();
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float2 by = *reinterpret_cast<const float2*>(into + g * 8 + i);
            float2 v = make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
            // what a decay of zero has dropped may be anything
            v.x = by.x != 0.0f ? v.x : 0.0f;
            v.y = by.y != 0.0f ? v.y : 0.0f;
            const float2 near = vadd(make_float2(__uint_as_float(y[i]), __uint_as_float(y[i + 1])),
                                     make_float2(__uint_as_float(z[i]), __uint_as_float(z[i + 1])));
            two[g * 4 + i / 2] = pack<bf16>(vmul(vfma(by, v, near), scale)).w;
          }
        }
        // more channels than q has: the place of k too, once the state's sum has been made from it
        if (DV > DK && !wait_warp(kEDone, n)) break;
        fence_before();
        mbar_arrive(bar(kOFree));
        mbar_arrive(bar(kFree0 + n % kSlots));
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const uint32_t x = two[i];
          *reinterpret_cast<uint16_t*>(to + 2 * i * 128 + ((word ^ (2 * i & 7)) << 4)) = (uint16_t)x;
          *reinterpret_cast<uint16_t*>(to + (2 * i + 1) * 128 + ((word ^ (2 * i + 1 & 7)) << 4)) = (uint16_t)(x >> 16);
        }
        proxy_fence();
        mbar_arrive(bar(kOReady0 + n % kStages));
      }
    }
  } else if (warp < 20) {  // ------------------------------ the weighed k
    const int at = tid - 12 * 32;
    constexpr int kWords = DK / 64 * kChunk * 8 / 256;
    for (int n = 0; n < n_chunks; ++n) {
      if (!wait_warp(kDec0 + n % kSlots, n / kSlots) || !wait_warp(kFull0 + n % kStages, n / kStages)) break;
      const ChunkDecay& cd = decays[n % kSlots];
      unsigned char* from = mem + (n % kStages) * L::kStage + L::k + at * 16;
      unsigned char* to = mem + L::W + at * 16;
      union Word { uint4 q; uint32_t pair[4]; };
      Word x[kPieces][kWords];
#pragma unroll
      for (int i = 0; i < kWords; ++i) x[0][i].q = *reinterpret_cast<const uint4*>(from + i * 4096);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const int t = (at / 8 + 32 * i) % kChunk;
        const float by = p.rev ? cd.into[t] * p.scale : cd.rest[t];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 f = make_float2(__uint_as_float(x[0][i].pair[j] << 16), __uint_as_float(x[0][i].pair[j] & 0xffff0000u));
          f = by != 0.0f ? vmul(f, vset<2>(by)) : vset<2>(0.0f);
#pragma unroll
          for (int k = 0; k < kPieces; ++k) {
            const uint32_t h2 = pack<bf16>(f).w;
            x[k][i].pair[j] = h2;
            f = vfma(make_float2(__uint_as_float(h2 << 16), __uint_as_float(h2 & 0xffff0000u)), vset<2>(-1.0f), f);
          }
        }
      }
      // the pieces go where matrix instructions still read: of the chunk before, and the scores
      if ((n > 0 && !wait_warp(kEDone, n - 1)) || (OUT && !wait_warp(kADone0 + (n & 1), n / 2))) break;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        *reinterpret_cast<uint4*>(from + i * 4096) = x[0][i].q;
#pragma unroll
        for (int k = 1; k < kPieces; ++k) *reinterpret_cast<uint4*>(to + (k - 1) * (DK / 64) * L::kBlock + i * 4096) = x[k][i].q;
      }
      proxy_fence();
      mbar_arrive(bar(kWReady));
    }
  } else if ((warp & 3) < 2 && warp < 26) {  // the scores: 32 rows and 32 columns of a warp
    if (OUT) {
      const int half = warp >= 24;  // of the columns
      unsigned char* to = mem + L::P + row * 128;
      for (int n = 0; n < n_chunks; ++n) {
        if (!wait_warp(kDec0 + n % kSlots, n / kSlots) || !wait_warp(kADone0 + (n & 1), n / 2)) break;
        fence_after();
        const ChunkDecay& cd = decays[n % kSlots];
        uint4 w[4] = {}, z[4] = {};
        if ((warp & 3) >= half) {
          uint32_t a[2][16];
          tmem_load(a[0], quarter + kColA + half * 32);
          tmem_load(a[1], quarter + kColA + half * 32 + 16);
          const float hi = cd.hi[row], lo = cd.lo[row];
          const int from = cd.from[row];
          wait_loads();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const int j = half * 32 + c * 4;
            const float4 hj = *reinterpret_cast<const float4*>(cd.hi + j), lj = *reinterpret_cast<const float4*>(cd.lo + j);
            const float e[4] = {ex2f((hi - hj.x) + (lo - lj.x)), ex2f((hi - hj.y) + (lo - lj.y)), ex2f((hi - hj.z) + (lo - lj.z)),
                                ex2f((hi - hj.w) + (lo - lj.w))};
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = j + i <= row && j + i >= from ? e[i] * __uint_as_float(a[c >> 2][(c & 3) * 4 + i]) : 0.0f;
            uint4 &high = w[c >> 1], &low = z[c >> 1];
            if (c & 1) {
              two_pieces(make_float2(f[0], f[1]), high.z, low.z);
              two_pieces(make_float2(f[2], f[3]), high.w, low.w);
            } else {
              two_pieces(make_float2(f[0], f[1]), high.x, low.x);
              two_pieces(make_float2(f[2], f[3]), high.y, low.y);
            }
          }
        }
        fence_before();
        mbar_arrive(bar(kAFree));
        if (n > 0 && !wait_warp(kODone, n - 1)) break;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          unsigned char* at = to + (((half * 4 + c) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(at) = w[c];
          *reinterpret_cast<uint4*>(at + L::kBlock) = z[c];
        }
        proxy_fence();
        mbar_arrive(bar(kPReady));
      }
    }
  } else if (warp == 22) {  // -------------------------------- the copies
    if (lane == 0) {
      int n = 0;
      for (; n < n_chunks; ++n) {
        const int s = n % kStages;
        if (n >= kStages && !wait(kEmpty0 + s, n / kStages - 1)) break;
        const uint32_t at = smem + s * L::kStage;
        const int t0 = chunk(n) * kChunk;
        mbar_expect_tx(bar(kFull0 + s), L::kStage);
        for (int i = 0; i < DK / 64; ++i) {
          if (OUT) tma_tile(at + L::q + i * L::kBlock, &maps.q, i * 64, hq, t0, (int)b, bar(kFull0 + s));
          tma_tile(at + L::k + i * L::kBlock, &maps.k, i * 64, hq, t0, (int)b, bar(kFull0 + s));
        }
        for (int i = 0; i < DV / 64; ++i) tma_tile(at + L::v + i * L::kBlock, &maps.v, i * 64, h, t0, (int)b, bar(kFull0 + s));
      }
      // whatever the others did: the last copy into each place has landed before the block ends
      for (int s = 0; s < kStages && s < n; ++s) mbar_wait(bar(kFull0 + s), (uint32_t)((n - 1 - s) / kStages) & 1);
    }
  } else if (warp == 23) {  // ------------------- the matrix instructions
    if (lane == 0) {
      constexpr uint32_t kScores = instruction(64, false, false), kSum = instruction(DV, true, true), kOut = instruction(64, true, false),
                         kOutTwo = instruction(128, true, false);
      const Operand q0 = operand(smem + L::q, 16, 1024), k0 = operand(smem + L::k, 16, 1024), kt0 = operand(smem + L::k, kOther, 1024),
                    vt0 = operand(smem + L::v, kOther, 1024), w0 = operand(smem + L::W, kOther, 1024),
                    s0 = operand(smem + L::S, DK * 128, 1024), p0 = operand(smem + L::P, 16, 1024);
      auto in_stage = [&](Operand o, int s) { return Operand{o.lo + (uint32_t)(s * (L::kStage >> 4)), o.hi}; };
      constexpr int kPiece = DK / 64 * L::kBlock;
      auto scores = [&](int n, int s) {
        const Operand q = in_stage(q0, s), k = in_stage(k0, s);
        mma<false>(tmem + kColA, q, 0, k, 0, kScores);
#pragma unroll
        for (int i = 1; i < DK / 16; ++i)
          mma<true>(tmem + kColA, q, (i / 4) * L::kBlock + (i % 4) * 32, k, (i / 4) * L::kBlock + (i % 4) * 32, kScores);
        commit(bar(kADone0 + (n & 1)));
      };
      if (OUT && n_chunks > 0 && wait(kFull0, 0)) {
        fence_after();
        scores(0, 0);
      }
      for (int n = 0; n < n_chunks; ++n) {
        const int st = n % kStages, next = (n + 1) % kStages;
        const Operand kt = in_stage(kt0, st), vt = in_stage(vt0, st);
        // where the outputs take the place of k, they still wait for the sum before
        if (OUT && DV > DK && n > 0 && !wait(kOFree, n - 1)) break;
        if (!wait(kWReady, n) || !wait(kFull0 + st, n / kStages)) break;
        if (n > 0 && !wait(kEFree, n - 1)) break;
        fence_after();
        // the small pieces first
        mma<false>(tmem + kColE, w0, kPiece, vt, 0, kSum);
#pragma unroll
        for (int i = 1; i < 4; ++i) mma<true>(tmem + kColE, w0, kPiece + i * 2048, vt, i * 2048, kSum);
#pragma unroll
        for (int i = 0; i < 4; ++i) mma<true>(tmem + kColE, w0, i * 2048, vt, i * 2048, kSum);
#pragma unroll
        for (int i = 0; i < 4; ++i) mma<true>(tmem + kColE, kt, i * 2048, vt, i * 2048, kSum);
        commit(bar(kEDone));
        commit(bar(kEmpty0 + st));
        if (OUT) {
          if (!wait(kSReady, n) || (n > 0 && !wait(kOFree, n - 1))) break;
          fence_after();
          const Operand q = in_stage(q0, st);
          // the smaller piece first
          mma<false>(tmem + kColX, s0, L::kPieceS, q, 0, kOut);
#pragma unroll
          for (int i = 1; i < DK / 16; ++i) mma<true>(tmem + kColX, s0, L::kPieceS + i * 2048, q, (i / 4) * L::kBlock + (i % 4) * 32, kOut);
#pragma unroll
          for (int i = 0; i < DK / 16; ++i) mma<true>(tmem + kColX, s0, i * 2048, q, (i / 4) * L::kBlock + (i % 4) * 32, kOut);
          commit(bar(kXDone));
          if (!wait(kPReady, n)) break;
          fence_after();
          // both pieces of P in one: 128 columns cost what 64 do
          mma<false>(tmem + kColY, vt, 0, p0, 0, kOutTwo);
#pragma unroll
          for (int i = 1; i < 4; ++i) mma<true>(tmem + kColY, vt, i * 2048, p0, i * 32, kOutTwo);
          commit(bar(kODone));
          if (n + 1 < n_chunks) {
            if (!wait(kFull0 + next, (n + 1) / kStages) || !wait(kAFree, n)) break;
            fence_after();
            scores(n + 1, next);
          }
        }
      }
    }
  } else if (warp == 27) {  // ----------------------- the outputs' copies
    if (!OUT && p.at && lane == 0) {
      for (int n = 0; n < n_chunks; ++n) {
        if (!wait(kOReady0, n)) break;
        for (int i = 0; i < DV / 32; ++i)
          if (i * 32 < d.dvp)
            tma_write(&maps.o, smem + L::S + i * (DK * 128), i * 32, 0, chunk(n), (int)bh);
        asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
        mbar_arrive(bar(kOEmpty));
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    if (OUT && lane == 0) {
      for (int n = 0; n < n_chunks; ++n) {
        if (!wait(kOReady0 + n % kStages, n / kStages)) break;
        const uint32_t at = smem + (n % kStages) * L::kStage;
        for (int i = 0; i < DV / 64; ++i)
          if (i * 64 < d.DV) tma_write(&maps.o, at + i * L::kBlock, i * 64, h, chunk(n) * kChunk, (int)b);
        asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
        mbar_arrive(bar(kEmpty0 + n % kStages));
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  } else {  // --------------------------------------------- the decays
    const float* g = p.g.p + b * p.g.sb + h * p.g.sh;
    for (int n = 0; n < n_chunks; ++n) {
      const int64_t t0 = (int64_t)chunk(n) * kChunk;
      if (n >= kSlots && !wait_warp(kFree0 + n % kSlots, n / kSlots - 1)) break;
      decays[n % kSlots].fill(g + t0 * p.g.st, p.g.st, (int)min((int64_t)kChunk, d.T - t0));
      mbar_arrive(bar(kDec0 + n % kSlots));
    }
  }
  if (!ok && p.status) *p.status = MPB_ERR_TIMEOUT;
  __syncwarp();
  // A block that gave up: what it has under way ends before its memory does. The copies have been waited for by the warps
  // that issued them.
  if (__syncthreads_or(!ok)) {
    wait_loads();
    wait_stores();
    if (warp == 23 && lane == 0) {
      commit(bar(kEnd));
      mbar_wait(bar(kEnd), 0);
    }
    leave_nan<OUT>(p);
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 26)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemColumns) : "memory");
}

// ------------------------------------------------------------------- host
std::atomic<uint32_t> wait_limit{kMostWaitNs};

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
  static EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// Boxes of 64 channels and 64 steps of one head of a (B, T, heads, D) array; zeros outside it.
bool encode(CUtensorMap* m, const Input& x, int64_t B, int64_t T, int64_t heads, int64_t D) {
  const EncodeTiled fn = encoder();
  if (!fn) return false;
  // a dim of one step has no stride of its own
  auto bytes = [&](int64_t n, int64_t stride) { return (cuuint64_t)(n > 1 ? stride * 2 : (D * 2 + 15) / 16 * 16); };
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T, (cuuint64_t)B};
  const cuuint64_t strides[3] = {bytes(heads, x.sh), bytes(T, x.st), bytes(B, x.sb)};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)kChunk, 1}, each[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(x.p), dims, strides, box, each,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes of 32 columns and all rows of a (heads, chunks, dkp, dvp) array of states in float.
bool encode_states(CUtensorMap* m, const Walk& p, int rows) {
  const EncodeTiled fn = encoder();
  if (!fn) return false;
  const Shape& d = p.d;
  const cuuint64_t dims[4] = {(cuuint64_t)d.dvp, (cuuint64_t)d.dkp, (cuuint64_t)d.chunks, (cuuint64_t)(d.B * d.H)};
  const cuuint64_t strides[3] = {(cuuint64_t)d.dvp * 4, (cuuint64_t)d.dkp * d.dvp * 4, (cuuint64_t)d.chunks * d.dkp * d.dvp * 4};
  const cuuint32_t box[4] = {32, (cuuint32_t)rows, 1, 1}, each[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.at, dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DK, int DV, bool OUT>
int launch(const Walk& p, cudaStream_t s) {
  const Shape& d = p.d;
  Maps maps;
  const int64_t hq = d.H / d.share;
  if ((OUT && !encode(&maps.q, p.q, d.B, d.T, hq, d.DK)) || !encode(&maps.k, p.k, d.B, d.T, hq, d.DK) ||
      !encode(&maps.v, p.v, d.B, d.T, d.H, d.DV) ||
      (OUT && !encode(&maps.o, {p.o, d.T * d.H * d.DV, (int64_t)d.H * d.DV, d.DV, true}, d.B, d.T, d.H, d.DV)) ||
      (!OUT && p.at && !encode_states(&maps.o, p, DK)))
    return fail(MPB_ERR_CUDA, "linear_attention: the copies' maps cannot be made");
  constexpr int kWalkBytes = Layout<DK, DV, OUT>::bytes;
  if (int rc = allow_smem<k_la_walk<DK, DV, OUT>, kWalkBytes>("linear_attention")) return rc;
  k_la_walk<DK, DV, OUT><<<(unsigned)(d.B * d.H * d.segments), kThreads, kWalkBytes, s>>>(maps, p);
  return launch_check("linear_attention");
}

template <bool OUT>
int launch_for(const Walk& p, cudaStream_t s) {
  const bool k = p.d.DK > 64, v = p.d.DV > 64;
  return k ? (v ? launch<128, 128, OUT>(p, s) : launch<128, 64, OUT>(p, s))
           : (v ? launch<64, 128, OUT>(p, s) : launch<64, 64, OUT>(p, s));
}

}  // namespace

bool walk_takes(const Shape& d, const Input& q, const Input& k, const Input& v) {
  if (d.DK > 128 || d.DV > 128 || d.T >= (1LL << 31) - kChunk || d.B >= (1LL << 31) ) return false;
  for (const Input* x : {&q, &k, &v}) {
    if (!x->wide) return false;
    const int64_t heads = x == &v ? d.H : d.H / d.share;
    if ((d.B > 1 && x->sb <= 0) || (d.T > 1 && x->st <= 0) || (heads > 1 && x->sh <= 0)) return false;
    if (x->sb >= (1LL << 38) || x->st >= (1LL << 38) || x->sh >= (1LL << 38)) return false;
  }
  return true;
}
int walk_outputs(Walk p, cudaStream_t s) {
  p.tries = (int)((wait_limit.load() + kTryNs - 1) / kTryNs);
  return launch_for<true>(p, s);
}
int walk_states(Walk p, cudaStream_t s) {
  p.tries = (int)((wait_limit.load() + kTryNs - 1) / kTryNs);
  return launch_for<false>(p, s);
}
int64_t walk_wait_limit(int64_t ns) { return wait_limit.exchange((uint32_t)ns); }

}  // namespace mpb

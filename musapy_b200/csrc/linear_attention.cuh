// Pieces shared by the linear attention kernels: the decays of a chunk and the
// warp-level matrix instructions.
#pragma once
#include "rows.cuh"

namespace mpb {

constexpr int kChunk = 64;          // steps of a chunk
constexpr int kTile = 64;           // channels of a tile
constexpr int kPitch = 72;          // elements of a tile's row in shared memory: 144 bytes, so eight rows are in eight bank groups
constexpr int kMostChannels = 256;  // of a head

MPB_D uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

template <bool TRANSPOSED>
MPB_D void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANSPOSED)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

MPB_D void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The decays between the steps of a chunk. The running sums of g, in units of
// log2 e, are taken in double and kept as two floats, since the difference of
// two large sums has to be right to float precision. A decay below
// e^-104, which is zero in float (-inf among them), begins anew: sums restart there
// and pairs across it have a decay of exactly zero.
struct alignas(16) ChunkDecay {
  float hi[kChunk], lo[kChunk];
  int from[kChunk];                      // the last step at or before that begins anew, or -1
  float into[kChunk], rest[kChunk], weight[kChunk];  // from before the chunk to a step, from a step to the chunk's end
  float all;                             // over the chunk

  // By one warp; steps from `steps` on do not decay and hold nothing.
  MPB_D void fill(const float* g, int64_t stride, int steps) {
    const int lane = threadIdx.x & 31;
    double sum[2];
    int begin[2];
    float x[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) x[e] = 2 * lane + e < steps ? g[(int64_t)(2 * lane + e) * stride] : 0.0f;
    constexpr float kZero = -104.0f;
    constexpr double kLog2e = 1.4426950408889634074;
    begin[0] = x[0] < kZero ? 2 * lane : -1;
    begin[1] = x[1] < kZero ? 2 * lane + 1 : begin[0];
    sum[0] = x[0] < kZero ? 0.0 : (double)x[0] * kLog2e;
    sum[1] = x[1] < kZero ? 0.0 : sum[0] + (double)x[1] * kLog2e;
    // inclusive over the lanes: a lane that begins anew keeps its own sum
    double run = sum[1];
    int at = begin[1];
    for (int o = 1; o < 32; o <<= 1) {
      const double s = __shfl_up_sync(0xffffffffu, run, o);
      const int b = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o && at < 0) run += s, at = b;
    }
    const double s0 = __shfl_up_sync(0xffffffffu, run, 1);
    const int b0 = __shfl_up_sync(0xffffffffu, at, 1);
    if (lane > 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (begin[e] < 0) sum[e] += s0, begin[e] = b0;
    }
    const double last = __shfl_sync(0xffffffffu, sum[1], 31);
    const int last_begin = __shfl_sync(0xffffffffu, begin[1], 31);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int t = 2 * lane + e;
      hi[t] = (float)sum[e];
      lo[t] = (float)(sum[e] - (double)hi[t]);
      from[t] = begin[e];
      into[t] = begin[e] < 0 ? exp2f((float)sum[e]) : 0.0f;
      rest[t] = t >= last_begin ? exp2f((float)(last - sum[e])) : 0.0f;
    }
    if (lane == 0) all = last_begin < 0 ? exp2f((float)last) : 0.0f;
  }
  MPB_D bool resets(int t) const { return from[t] == t; }
  // From step j to step i; zero for later steps and across a restart.
  MPB_D float pair(int i, int j) const {
    return j <= i && j >= from[i] ? ex2f((hi[i] - hi[j]) + (lo[i] - lo[j])) : 0.0f;
  }
};

struct Shape {
  int64_t B, T;
  int H, share, DK, DV;      // share: heads that share one of q and k
  int chunks, segments, per;  // per: chunks of a segment
  int dkp, dvp;               // channels in the scratch, multiples of 16
};
struct Input {
  const void* p;
  int64_t sb, st, sh;
  bool wide;  // 16-byte loads
  template <class T>
  MPB_D const T* at(int64_t b, int64_t t, int h) const { return (const T*)p + b * sb + t * st + h * sh; }
};
struct Decay {
  const float* p;
  int64_t sb, st, sh;
};

constexpr uint32_t kMostWaitNs = 2000000000;  // of a wait between a block's warps

// The bf16 kernel of whole rows (linear_attention_walk.cu): one block per head of a sequence and segment.
struct Walk {
  Shape d;
  Input q, k, v;       // without outputs q is unused: k and v, or the pair that the state is summed from
  Decay g;
  const float* first;  // the state before the first segment, (DK, DV) per head, or null
  const float* starts; // the states before the other segments, padded; null without outputs: each begins from nothing
  float scale;
  void* o;
  bool rev;
  float *at, *since, *ends, *last;  // as k_la_states leaves them; null where not wanted
  int* status;
  int tries = 0;  // of a wait between the block's warps: set by the two below
};
int64_t walk_wait_limit(int64_t ns);
bool walk_takes(const Shape& d, const Input& q, const Input& k, const Input& v);
int walk_outputs(Walk p, cudaStream_t s);
int walk_states(Walk p, cudaStream_t s);

}  // namespace mpb

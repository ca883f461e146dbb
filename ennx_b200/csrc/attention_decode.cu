// attention_decode.cu -- grouped-query attention of one new token per sequence
// against a key/value cache, writing the new token's key and value.
//
// With p = lengths[b] - 1 the new token's position and R_p its rotation,
//   k_cache[b, p] = R_p k[b], v_cache[b, p] = v[b],
//   o[b, h] = sum_{j <= p} softmax_j(R_p q[b, h] . k_cache[b, j, h/G] / sqrt(128)) v_cache[b, j, h/G].
//
// Bound: HBM, 512 bytes of cache per key and head; the arithmetic is 4 * G
// FLOP per byte pair.  The G query heads of a cache head are the rows of an
// m16n8k16 product, so a key is read once for all of them.  Each warp streams
// 16 keys a step through its own cp.async ring and keeps its own running
// maximum, sum and output, so no barrier stands in the loop.
//
// The rotated query and the weights have more bits than bf16 holds, so both
// enter the products as hi + lo, two bf16 numbers (2^-16 of the value left).
// With at most 8 query heads the tile's other 8 rows carry the lo parts and a
// lane finds both sums in its own accumulators (rows g and g + 8): exactness
// costs no instruction.  9 to 16 heads take a second product each.
//
// Work is counted in steps of 16 keys, numbered over all (sequence, cache head,
// block of kRows query heads), and every WARP takes an equal run of steps
// whatever the lengths are: one long sequence is split over the device and a
// ragged batch is balanced.  A warp needs nobody else: it reads and rotates its
// own query rows, and its copies run ahead from one sequence into the next.
// Where a run begins or ends inside a sequence its partial (maximum, sum,
// output) goes to the workspace in fp32 and a second kernel joins the partials
// in order.  (Runs of blocks, with a merge of their warps and an empty ring at
// the end of each sequence, took 40 us instead of 32 on 32 ragged sequences
// of up to 4096 keys.)  Shorter caches take a block per head, or a cluster of up
// to 8, whose warps share the keys and meet once, and no second kernel.
#include "kernels.cuh"
#include "serve.cuh"

#include <math.h>

namespace ennx {
namespace {

constexpr int D = 128;
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStep = 16;                       // keys of a warp's step
constexpr int kStages = 3;                      // ring depth: 2 steps (16 KB) in flight per warp, 128 KB per SM
constexpr int kStageBytes = 2 * kStep * D * 2;  // K and V rows of one step
constexpr int kWarpRing = kStages * kStageBytes;
constexpr int kLoBytes = 16 * D * 2;            // a warp's lo parts of 16 query rows
constexpr int kSmem = kWarps * (kWarpRing + kLoBytes);
constexpr int kPerSm = 2;                       // blocks resident per SM
constexpr int kPart = D + 2;                    // floats of a partial row: output, maximum, sum
static_assert(kPerSm * (kSmem + 1024) <= 228 * 1024, "blocks of an SM");
static_assert(kWarps * 16 * kPart * 4 <= kWarps * kWarpRing, "the merge buffer overlays the rings");

struct Cache {
  uint16_t *k, *v;
  long long kb, kt, kh, vb, vt, vh;  // strides in elements: sequence, token, head
};
struct Args {
  const uint16_t *q, *knew, *vnew;
  uint16_t* o;
  long long ldq, ldk, ldv, ldo;
  Cache c;
  const int* lengths;
  int batch, room, hkv, group;
  int blocks;  // blocks of kRows query heads per cache head
  float scale_log2;
  int rotate;
  float* partial;
  int longest_first;  // blocks take the sequences in the order of their lengths
};

__device__ __forceinline__ int seq_len(const Args& a, int b) { return min(a.room, max(0, __ldg(a.lengths + b))); }
// steps of one head of a sequence, and its weight in the division of the work:
// a head costs the reading of its query rows beside its steps
__device__ __forceinline__ int head_steps(int len) { return (len + kStep - 1) / kStep; }
constexpr int kHeadCost = 2;
__device__ __forceinline__ int head_weight(int steps) { return steps > 0 ? steps + kHeadCost : 0; }
__device__ __forceinline__ long long seq_weight(const Args& a, int b) {
  return (long long)head_weight(head_steps(seq_len(a, b))) * a.hkv * a.blocks;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_16x8x16(c, a[0], a[1], a[2], a[3], b0, b1);
}
// hi parts of a pair packed, the pair replaced by what is left
__device__ __forceinline__ uint32_t take_hi(float& x, float& y) {
  const uint32_t hi = pack_bf16x2(x, y);
  x -= __uint_as_float(hi << 16);
  y -= __uint_as_float(hi & 0xffff0000u);
  return hi;
}
__device__ __forceinline__ uint32_t cluster_ctas() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ float2 lds_cluster(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
// 16-byte chunk `c` of row `r` in a tile of 256-byte rows
__device__ __forceinline__ uint32_t at(int r, int c) { return (uint32_t)(r * 256 + ((c ^ (r & 7)) << 4)); }

// One warp's work on one (sequence, cache head, block of query heads).
template <int kRows>
struct Head {
  static constexpr int R = kRows / 8;  // rows g (and g + 8) of a lane
  int b, h, hq0, rows, len;            // query heads hq0 .. hq0 + rows - 1
  uint32_t qf[8][4];
  float acc[16][4], m[R], l[R];        // l of this lane's columns
  float sn[2], cs[2];                  // rotation of pairs lane and lane + 32 to position len - 1

  __device__ __forceinline__ void place(const Args& a, int seq, int within, int n) {
    b = seq;
    len = n;
    h = within / a.blocks;
    const int g0 = within % a.blocks * kRows;
    rows = min(kRows, a.group - g0);
    hq0 = h * a.group + g0;
  }

  // Query rows as fragments: rotated, split into hi and lo.  kRows 8: the lo
  // parts are rows 8 .. 15 of the tile; kRows 16: they go to `lo_parts`.
  // The loads come first, all of them, and the rotation's frequencies from
  // shared memory: a load at a time between the shuffles, and frequencies
  // indexed by lane in the parameters, took 4.4 us, a third of a short run.
  __device__ __forceinline__ void start(const Args& a, const double* inv, uint32_t lo_parts, int lane) {
    const int g = lane >> 2, t = lane & 3;
    uint32_t raw[R][4][2][2];  // columns 16 kk + 8 e + 2t, + 1 and those 64 further on
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint16_t* q = a.q + (long long)b * a.ldq + (long long)(hq0 + (g + 8 * r < rows ? g + 8 * r : 0)) * D + 2 * t;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int far = 0; far < 2; ++far)
            raw[r][kk][e][far] = __ldg(reinterpret_cast<const uint32_t*>(q + 16 * kk + 8 * e + 64 * far));
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      sn[e] = 0.0f;
      cs[e] = 1.0f;
      if (a.rotate) rope_sincos(inv[lane + 32 * e], len - 1, &sn[e], &cs[e]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = g + 8 * r < rows;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w1 = raw[r][kk][e][0], w2 = raw[r][kk][e][1];
          float x[2] = {__uint_as_float(w1 << 16), __uint_as_float(w1 & 0xffff0000u)};
          float y[2] = {__uint_as_float(w2 << 16), __uint_as_float(w2 & 0xffff0000u)};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int from = (16 * (kk & 1) + 8 * e + 2 * t + i) & 31;
            const float s = __shfl_sync(0xffffffffu, sn[kk >> 1], from), c = __shfl_sync(0xffffffffu, cs[kk >> 1], from);
            if (a.rotate) rope_turn(x[i], y[i], s, c);
            if (!live) x[i] = y[i] = 0.0f;
          }
          const uint32_t xh = take_hi(x[0], x[1]), yh = take_hi(y[0], y[1]);
          const uint32_t xl = pack_bf16x2(x[0], x[1]), yl = pack_bf16x2(y[0], y[1]);
          qf[kk][2 * e + r] = xh;
          qf[kk + 4][2 * e + r] = yh;
          if constexpr (kRows == 8) {
            qf[kk][2 * e + 1] = xl;
            qf[kk + 4][2 * e + 1] = yl;
          } else {
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(lo_parts + at(g + 8 * r, 2 * kk + e) + 4 * t), "r"(xl) : "memory");
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(lo_parts + at(g + 8 * r, 2 * kk + 8 + e) + 4 * t), "r"(yl) : "memory");
          }
        }
    }
    if constexpr (kRows == 16) __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) { m[r] = -INFINITY; l[r] = 0.0f; }
  }

  // Writes the new token's key and value to the cache and over row `p` of the stage.
  __device__ __forceinline__ void append(const Args& a, uint8_t* st, int p, int lane) {
    uint16_t* kw = a.c.k + (long long)b * a.c.kb + (long long)h * a.c.kh + (long long)(len - 1) * a.c.kt;
    uint16_t* vw = a.c.v + (long long)b * a.c.vb + (long long)h * a.c.vh + (long long)(len - 1) * a.c.vt;
    const uint16_t* kn = a.knew + (long long)b * a.ldk + h * D;
    const uint16_t* vn = a.vnew + (long long)b * a.ldv + h * D;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = lane + 32 * e;
      float x1 = bf16_to_f32(__ldg(kn + d)), x2 = bf16_to_f32(__ldg(kn + d + 64));
      if (a.rotate) rope_turn(x1, x2, sn[e], cs[e]);
      const uint16_t b1 = f32_to_bf16_rne(x1), b2 = f32_to_bf16_rne(x2);
      kw[d] = b1;
      kw[d + 64] = b2;
      *reinterpret_cast<uint16_t*>(st + at(p, d >> 3) + (d & 7) * 2) = b1;
      *reinterpret_cast<uint16_t*>(st + at(p, (d + 64) >> 3) + (d & 7) * 2) = b2;
      const uint16_t w1 = __ldg(vn + d), w2 = __ldg(vn + d + 64);
      vw[d] = w1;
      vw[d + 64] = w2;
      *reinterpret_cast<uint16_t*>(st + kStep * 256 + at(p, d >> 3) + (d & 7) * 2) = w1;
      *reinterpret_cast<uint16_t*>(st + kStep * 256 + at(p, (d + 64) >> 3) + (d & 7) * 2) = w2;
    }
    __syncwarp();
  }

  // keys key0 .. key0 + 15, of which those below len count
  __device__ __forceinline__ void step(const Args& a, uint32_t sk, uint32_t lo_parts, int key0, int lane) {
    const int t = lane & 3;
    const uint32_t sv = sk + kStep * 256;
    float s[2][4] = {}, lo[2][4] = {};  // lo: of the lo parts, kRows 16 (kRows 8 has them in rows 8 .. 15 of s)
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      uint32_t kf[4];
      ldsm4(sk + at((lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)), kf);
      mma(s[0], qf[kk], kf[0], kf[1]);
      mma(s[1], qf[kk], kf[2], kf[3]);
      if (kRows == 16 && a.rotate) {
        uint32_t ql[4];
        ldsm4(lo_parts + at(lane & 15, 2 * kk + (lane >> 4)), ql);
        mma(lo[0], ql, kf[0], kf[1]);
        mma(lo[1], ql, kf[2], kf[3]);
      }
    }
    float alpha[R], ref[R], pr[R][4];  // pr[.]: keys 2t, 2t + 1 of both blocks of 8
    bool moved = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int nb = j >> 1, e = j & 1;
        // an infinite score is what the hi parts say: the lo parts of the same
        // factors may be 0 or of the other sign, and the sum NaN then
        const float hi = s[nb][2 * r + e], rest = kRows == 8 ? s[nb][2 + e] : lo[nb][2 * r + e];
        const float v = fabsf(hi) == INFINITY ? hi : hi + rest;
        pr[r][j] = key0 + nb * 8 + 2 * t + e < len ? v * a.scale_log2 : -INFINITY;
        top = fmaxf(top, pr[r][j]);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float mn = fmaxf(m[r], top);
      ref[r] = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet: every exponent below is -inf
      alpha[r] = ex2(m[r] - ref[r]);
      moved |= alpha[r] != 1.0f;
      m[r] = mn;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int r = 0; r < R; ++r) l[r] *= alpha[r];
#pragma unroll
      for (int nb = 0; nb < 16; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[nb][j] *= alpha[kRows == 8 ? 0 : j >> 1];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pr[r][j] = ex2(pr[r][j] - ref[r]);
        l[r] += pr[r][j];
      }
    uint32_t pf[4], pl[4];
    if constexpr (kRows == 8) {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        pf[2 * nb] = take_hi(pr[0][2 * nb], pr[0][2 * nb + 1]);
        pf[2 * nb + 1] = pack_bf16x2(pr[0][2 * nb], pr[0][2 * nb + 1]);
      }
    } else {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          pf[2 * nb + r] = take_hi(pr[r][2 * nb], pr[r][2 * nb + 1]);
          pl[2 * nb + r] = pack_bf16x2(pr[r][2 * nb], pr[r][2 * nb + 1]);
        }
    }
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      uint32_t vf[4];
      ldsm4t(sv + at(lane & 15, 2 * nb + (lane >> 4)), vf);
      mma(acc[2 * nb], pf, vf[0], vf[1]);
      mma(acc[2 * nb + 1], pf, vf[2], vf[3]);
      if constexpr (kRows == 16) {
        mma(acc[2 * nb], pl, vf[0], vf[1]);
        mma(acc[2 * nb + 1], pl, vf[2], vf[3]);
      }
    }
  }

  // the row sums over the lanes that share a row
  __device__ __forceinline__ void close() {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
  }
  __device__ __forceinline__ float2 value(int r, int nb) const {  // columns 8 nb + 2t, + 1 of row g + 8r
    return kRows == 8 ? make_float2(acc[nb][0] + acc[nb][2], acc[nb][1] + acc[nb][3])
                      : make_float2(acc[nb][2 * r], acc[nb][2 * r + 1]);
  }
  // partial rows, kPart floats each
  __device__ __forceinline__ void put_partial(float* to, int lane) const {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (g + 8 * r < rows) {
        float* row = to + (g + 8 * r) * kPart;
#pragma unroll
        for (int nb = 0; nb < 16; ++nb) *reinterpret_cast<float2*>(row + nb * 8 + 2 * t) = value(r, nb);
        if (t == 0) *reinterpret_cast<float2*>(row + D) = make_float2(m[r], l[r]);
      }
  }
  __device__ __forceinline__ void put_output(const Args& a, int lane) const {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (g + 8 * r < rows) {
        const float inv = 1.0f / l[r];  // every score -inf: 0 / 0, as the softmax
        uint16_t* o = a.o + (long long)b * a.ldo + (long long)(hq0 + g + 8 * r) * D + 2 * t;
#pragma unroll
        for (int nb = 0; nb < 16; ++nb) {
          const float2 v = value(r, nb);
          *reinterpret_cast<uint32_t*>(o + nb * 8) = pack_bf16x2(v.x * inv, v.y * inv);
        }
      }
  }
};

// Keys key0 .. key0 + 15 of one cache head into a stage, zeros from `len` on.
__device__ __forceinline__ void copy_step(const Args& a, const uint16_t* kbase, const uint16_t* vbase, int key0, int len,
                                          uint32_t dst, int lane) {
#pragma unroll
  for (int j = 0; j < kStep / 2; ++j) {
    const int r = 2 * j + (lane >> 4), c = lane & 15, key = key0 + r;
    const bool ok = key < len;
    const long long tok = ok ? key : 0;
    cp_async16(dst + at(r, c), kbase + tok * a.c.kt + c * 8, ok);
    cp_async16(dst + kStep * 256 + at(r, c), vbase + tok * a.c.vt + c * 8, ok);
  }
}
__device__ __forceinline__ const uint16_t* head_base(const uint16_t* cache, long long seq_stride, long long head_stride, int b,
                                                     int h) {
  return cache + (long long)b * seq_stride + (long long)h * head_stride;
}

// Short caches: one block, or a cluster of up to 8, per (sequence, cache head,
// block of query heads); the warps take the steps in turn, are merged per block
// and then over distributed shared memory, row by row.
template <int kRows>
__global__ void __launch_bounds__(kThreads, kPerSm) token_whole_kernel(const __grid_constant__ Args a,
                                                                       const __grid_constant__ RopeTable table) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ double inv[64];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = (int)cluster_ctarank(), cluster = (int)cluster_ctas();
  const int seg = (int)blockIdx.x / cluster, per_seq = a.hkv * a.blocks;
  __shared__ int sequence;
  if (a.rotate && threadIdx.x < 64) inv[threadIdx.x] = rope_inv(table, threadIdx.x);
  if (a.longest_first && (int)threadIdx.x < a.batch) {  // the sequence whose place by length is this one
    const int i = (int)threadIdx.x, own = seq_len(a, i);
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < a.batch; ++j) {
      const int other = seq_len(a, j);
      place += other > own || (other == own && j < i);
    }
    if (place == seg / per_seq) sequence = i;
  }
  __syncthreads();
  uint8_t* mine = smem + warp * kWarpRing;
  const uint32_t ring = smem_u32(mine), lo_parts = smem_u32(smem) + kWarps * kWarpRing + warp * kLoBytes;
  // (in bounds even where lengths that change under the call left no sequence in this place)
  const int b = a.longest_first ? (int)min((uint32_t)sequence, (uint32_t)a.batch - 1u) : seg / per_seq;
  const int len = seq_len(a, b), steps = head_steps(len);
  Head<kRows> s;
  s.place(a, b, seg % per_seq, len);
  const uint16_t *kbase = head_base(a.c.k, a.c.kb, a.c.kh, b, s.h), *vbase = head_base(a.c.v, a.c.vb, a.c.vh, b, s.h);
  const int first = rank * kWarps + warp, stride = cluster * kWarps;  // steps first, first + stride, ..
  const int n = steps > first ? (steps - first + stride - 1) / stride : 0;
  auto fetch = [&](int i) {
    if (i < n) copy_step(a, kbase, vbase, (first + i * stride) * kStep, len, ring + i % kStages * kStageBytes, lane);
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  s.start(a, inv, lo_parts, lane);
  for (int i = 0; i < n; ++i) {
    cp_wait<kStages - 2>();
    __syncwarp();            // the stage is there, and all lanes have read the one before it,
    fetch(i + kStages - 1);  // which is filled again while this one is used
    const int key0 = (first + i * stride) * kStep, p = len - 1 - key0;
    if (a.knew && p >= 0 && p < kStep) s.append(a, mine + i % kStages * kStageBytes, p, lane);
    s.step(a, ring + i % kStages * kStageBytes, lo_parts, key0, lane);
  }
  cp_wait<0>();
  s.close();
  __syncthreads();  // every ring is drained: the merge buffers may overlay them
  float* merge = reinterpret_cast<float*>(smem);  // [warp][row][kPart]
  float* joined = merge + kWarps * 16 * kPart;        // [row][kPart], of this block
  static_assert((kWarps + 1) * 16 * kPart * 4 <= kWarps * kWarpRing, "the merge buffers overlay the rings");
  s.put_partial(merge + warp * 16 * kPart, lane);
  __syncthreads();
  auto put = [&](int row, const float (&y)[4], float sum) {
    const float inv = len > 0 ? 1.0f / sum : 0.0f;  // every score -inf: 0 / 0, as the softmax
    *reinterpret_cast<uint2*>(a.o + (long long)b * a.ldo + (long long)(s.hq0 + row) * D + lane * 4) =
        make_uint2(pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv));
  };
  for (int row = warp; row < s.rows; row += kWarps) {
    float mx = -INFINITY, sum = 0.0f, y[4] = {};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, merge[(w * 16 + row) * kPart + D]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* part = merge + (w * 16 + row) * kPart;
      const float f = ex2(part[D] - ref);
      sum += f * part[D + 1];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += f * part[lane * 4 + e];
    }
    if (cluster == 1) {
      put(row, y, sum);
    } else {
      float* to = joined + row * kPart;
      *reinterpret_cast<float2*>(to + lane * 4) = make_float2(y[0], y[1]);
      *reinterpret_cast<float2*>(to + lane * 4 + 2) = make_float2(y[2], y[3]);
      if (lane == 0) *reinterpret_cast<float2*>(to + D) = make_float2(mx, sum);
    }
  }
  if (cluster == 1) return;
  cluster_sync();
  for (int row = rank + cluster * warp; row < s.rows; row += stride) {
    float2 ml = make_float2(-INFINITY, 0.0f), u[8], v[8];
    if (lane < cluster) ml = lds_cluster(mapa_shared(joined + row * kPart + D, lane));
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < cluster) {
        const uint32_t from = mapa_shared(joined + row * kPart + lane * 4, c);
        u[c] = lds_cluster(from);
        v[c] = lds_cluster(from + 8);
      }
    float mx = ml.x;
#pragma unroll
    for (int off = 4; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));  // lanes 0 .. 7
    mx = __shfl_sync(0xffffffffu, mx, 0);
    const float f = ex2(ml.x - (mx == -INFINITY ? 0.0f : mx));
    float sum = f * ml.y, y[4] = {};
#pragma unroll
    for (int off = 4; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    sum = __shfl_sync(0xffffffffu, sum, 0);
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < cluster) {
        const float fc = __shfl_sync(0xffffffffu, f, c);
        y[0] += fc * u[c].x;
        y[1] += fc * u[c].y;
        y[2] += fc * v[c].x;
        y[3] += fc * v[c].y;
      }
    put(row, y, sum);
  }
  cluster_sync();  // no block leaves while its rows are being read
}

// Any cache: every warp an equal run of all steps.
template <int kRows>
__global__ void __launch_bounds__(kThreads, kPerSm) token_split_kernel(const __grid_constant__ Args a,
                                                                       const __grid_constant__ RopeTable table) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ double inv[64];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (a.rotate && threadIdx.x < 64) inv[threadIdx.x] = rope_inv(table, threadIdx.x);
  __syncthreads();
  uint8_t* mine = smem + warp * kWarpRing;
  const uint32_t ring = smem_u32(mine), lo_parts = smem_u32(smem) + kWarps * kWarpRing + warp * kLoBytes;
  // the join kernel may start its own prologue; it waits for this grid to finish before it reads
  launch_dependents();
  const int per_seq = a.hkv * a.blocks;
  const long long worker = (long long)blockIdx.x * kWarps + warp, workers = (long long)gridDim.x * kWarps;
  long long total = 0;
  for (int i = lane; i < a.batch; i += 32) total += seq_weight(a, i);
#pragma unroll
  for (int off = 16; off; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  const long long per = (total + workers - 1) / workers, first = per * worker;
  int left = (int)min(per, total - first);
  if (left <= 0) return;
  // the sequence that holds step `first`, and the steps before it
  int b = 0;
  long long before = 0;
  for (int b0 = 0;; b0 += 32) {  // ends: first < total
    const long long own = b0 + lane < a.batch ? seq_weight(a, b0 + lane) : 0;
    long long upto = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += up;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, first < before + upto);
    if (hit) {
      const int at_lane = __ffs(hit) - 1;
      b = b0 + at_lane;
      before += __shfl_sync(0xffffffffu, upto - own, at_lane);
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  // where the copies and the products stand
  struct Walk {
    int b, within, step, len, steps;
  };
  auto enter = [&](Walk& w) {
    w.len = seq_len(a, w.b);
    w.steps = head_steps(w.len);
  };
  auto next_head = [&](Walk& w) {  // the next head with keys, while there are steps left
    w.step = 0;
    if (++w.within < per_seq) return;
    w.within = 0;
    do ++w.b;
    while (w.b < a.batch && seq_len(a, w.b) == 0);
    if (w.b < a.batch) enter(w);
  };
  Walk now{b, 0, 0, 0, 0};
  enter(now);
  now.within = (int)((first - before) / head_weight(now.steps));
  int weight_in = (int)((first - before) % head_weight(now.steps));  // of the head, before this run
  now.step = max(0, weight_in - kHeadCost);
  // steps of the run: its weight without that of the heads it opens
  int to_copy = 0;
  {
    Walk w = now;
    int in = weight_in;
    for (int rest = left; rest > 0; in = 0) {
      const int part = min(rest, head_weight(w.steps) - in);
      to_copy += max(0, in + part - kHeadCost) - max(0, in - kHeadCost);
      rest -= part;
      if (rest > 0) next_head(w);
    }
  }
  Walk ahead = now;
  int copied = 0;
  const uint16_t *kbase = nullptr, *vbase = nullptr;
  auto base = [&] {
    const int h = ahead.within / a.blocks;
    kbase = head_base(a.c.k, a.c.kb, a.c.kh, ahead.b, h);
    vbase = head_base(a.c.v, a.c.vb, a.c.vh, ahead.b, h);
  };
  base();
  auto fetch = [&] {
    if (to_copy > 0) {
      copy_step(a, kbase, vbase, ahead.step * kStep, ahead.len, ring + copied % kStages * kStageBytes, lane);
      if (--to_copy > 0 && ++ahead.step == ahead.steps) {
        next_head(ahead);
        base();
      }
    }
    ++copied;
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  Head<kRows> s;
  for (int used = 0; left > 0;) {
    const int part = min(left, head_weight(now.steps) - weight_in);
    const int n = max(0, weight_in + part - kHeadCost) - now.step;
    if (n > 0) {
    s.place(a, now.b, now.within, now.len);
    s.start(a, inv, lo_parts, lane);
    for (int i = 0; i < n; ++i, ++used) {
      cp_wait<kStages - 2>();
      __syncwarp();  // the stage is there, and all lanes have read the one before it,
      fetch();       // which is filled again while this one is used
      const int key0 = (now.step + i) * kStep, p = now.len - 1 - key0;
      if (a.knew && p >= 0 && p < kStep) s.append(a, mine + used % kStages * kStageBytes, p, lane);
      s.step(a, ring + used % kStages * kStageBytes, lo_parts, key0, lane);
    }
    s.close();
    const long long seg = (long long)now.b * per_seq + now.within;
    // a slot per (worker, segment): from one such pair to the next either number grows
    if (n == now.steps) s.put_output(a, lane);
    else s.put_partial(a.partial + (worker + seg) * kRows * kPart, lane);
    }
    left -= part;
    weight_in = 0;
    if (left > 0) next_head(now);
  }
  cp_wait<0>();
}

// Joins the partials of one row of a segment (block): its warps take 32 parts
// each at a time and are joined in order.  A segment of one part was written by
// that part's warp, an empty one gets zeros here.  (One warp for all parts of a
// row took 9 us for 74 of them.)
__global__ void __launch_bounds__(kThreads) token_join_kernel(const __grid_constant__ Args a, int workers, int block_rows) {
  const int seg = blockIdx.x, row = blockIdx.y, per_seq = a.hkv * a.blocks, b = seg / per_seq, within = seg % per_seq;
  const int steps = head_steps(seq_len(a, b)), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the weight before this sequence, and all of it
  __shared__ long long sums[2][kWarps];
  __shared__ float joined[kWarps][kPart];
  long long before = 0, total = 0;
  for (int i = threadIdx.x; i < a.batch; i += kThreads) {
    const long long u = seq_weight(a, i);
    total += u;
    if (i < b) before += u;
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, off);
    before += __shfl_xor_sync(0xffffffffu, before, off);
  }
  if (lane == 0) { sums[0][warp] = total; sums[1][warp] = before; }
  __syncthreads();
  total = before = 0;
  for (int w = 0; w < kWarps; ++w) { total += sums[0][w]; before += sums[1][w]; }
  const long long first = before + (long long)within * head_weight(steps) + kHeadCost;  // its first step
  const long long per = total > 0 ? (total + workers - 1) / workers : 1;
  const long long c0 = first / per;
  const int parts = steps > 0 ? (int)((first + steps - 1) / per - c0) + 1 : 0;
  const int h = within / a.blocks, g0 = within % a.blocks * block_rows;
  // the partials are complete and visible; blocks without any wait too, so
  // that this grid never ends before the one it follows
  wait_previous();
  if (parts == 1 || row >= min(block_rows, a.group - g0)) return;  // block-uniform
  float m = -INFINITY, l = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = warp * 32; c < parts; c += 32 * kWarps) {
    // maxima and sums first, a lane each, then the outputs, all loads independent
    const int n = min(32, parts - c);
    const float* part = a.partial + ((c0 + c + seg) * block_rows + row) * kPart;
    const long long stride = (long long)block_rows * kPart;
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < n) ml = *reinterpret_cast<const float2*>(part + lane * stride + D);
    float mn = fmaxf(m, ml.x);
#pragma unroll
    for (int off = 16; off; off >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
    const float ref = mn == -INFINITY ? 0.0f : mn, f0 = ex2(m - ref), f = ex2(ml.x - ref);
    float sum = f * ml.y;
#pragma unroll
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    l = l * f0 + sum;
    m = mn;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= f0;
#pragma unroll 16
    for (int i = 0; i < n; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      const float2 u = *reinterpret_cast<const float2*>(part + i * stride + lane * 4);
      const float2 v = *reinterpret_cast<const float2*>(part + i * stride + lane * 4 + 2);
      y[0] += fi * u.x;
      y[1] += fi * u.y;
      y[2] += fi * v.x;
      y[3] += fi * v.y;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) joined[warp][lane * 4 + e] = y[e];
  if (lane == 0) { joined[warp][D] = m; joined[warp][D + 1] = l; }
  __syncthreads();
  const int d = threadIdx.x;  // a column each
  static_assert(kThreads == D, "a thread per column");
  float mx = -INFINITY, sum = 0.0f, v = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, joined[w][D]);
  const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float f = ex2(joined[w][D] - ref);
    sum += f * joined[w][D + 1];
    v += f * joined[w][d];
  }
  const float inv = parts > 0 ? 1.0f / sum : 0.0f;  // every score -inf: 0 / 0, as the softmax
  a.o[(long long)b * a.ldo + (long long)(h * a.group + g0 + row) * D + d] = f32_to_bf16_rne(v * inv);
}

// query heads per block of rows: 8 leave room for the lo parts in the tile,
// more heads share one reading of the cache by 16
int block_rows(int group) { return group <= 8 ? 8 : 16; }

int split_grid() { return kPerSm * sm_count(); }

int64_t segments(int64_t batch, int hq, int hkv) {
  const int group = hq / hkv, rows = block_rows(group);
  return batch * hkv * ((group + rows - 1) / rows);
}

// Blocks of a head: one for each 128 tokens of room, 8 at most and two per SM
// over all heads (some more in rooms of more than 2048 tokens per block); a
// single one up to 256 tokens, where a cluster's start and meeting cost more (64
// keys 3.8 us, 5.2 in a cluster; 300 keys 6.1 and 5.2; 4096 keys 37 and 9.5).  0:
// the cache is split over the device.  That is for rooms of more than 2048
// tokens per block, where the longest sequence alone would last longer than a
// split and its second kernel (one sequence of 16 query heads on 4: 4096 keys 9.5
// us and 17.4 split, 8192 keys 13.7 and 18.8, 16384 keys 22.9 and 20.9; 64 heads
// with 4096 keys 25 and 32; 32 ragged sequences of up to 4096 keys 28 and 32, 24
// of up to 8192 32 and 38).  The lengths are on the device, so the room decides:
// one long sequence among empty ones takes up to 21 us instead of 11.
int whole_cluster(int64_t segs, int room) {
  int n = 1;
  while (n < 8 && room > 256 && room > 128 * n &&
         (n * segs <= sm_count() || (n * segs <= 2 * sm_count() && room > 2048 * n)))
    n *= 2;
  return room <= 2048 * n ? n : 0;
}
// With more blocks than SMs the longest sequences start first (32 ragged
// sequences of up to 4096 keys 30.1 -> 28.3 us, 24 of up to 8192 with two blocks
// each 47 -> 42; sequences of one length lose 0.4 us), where a thread per
// sequence can find the order.
bool longest_first(int64_t segs, int cluster, int batch) {
  return segs * cluster > sm_count() && batch > 1 && batch <= kThreads;
}

template <int kRows>
int32_t launch_whole(const Args& a, const RopeTable& table, int64_t segs, int cluster, int dev, cudaStream_t s) {
  static SharedMemorySetup setup;
  ENNX_TRY(allow_shared_memory(setup, dev, token_whole_kernel<kRows>, kSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(segs * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute together;
  together.id = cudaLaunchAttributeClusterDimension;
  together.val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = &together;
  cfg.numAttrs = 1;
  ENNX_CUDA(cudaLaunchKernelEx(&cfg, token_whole_kernel<kRows>, a, table), "token attention");
  ENNX_LAUNCH_CHECK("token attention");
  return ENNX_B200_OK;
}
template <int kRows>
int32_t launch_split(const Args& a, const RopeTable& table, int64_t segs, int dev, cudaStream_t s) {
  static SharedMemorySetup setup;
  ENNX_TRY(allow_shared_memory(setup, dev, token_split_kernel<kRows>, kSmem));
  token_split_kernel<kRows><<<(unsigned)split_grid(), kThreads, kSmem, s>>>(a, table);
  ENNX_LAUNCH_CHECK("token attention");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)segs, (unsigned)(a.group < kRows ? a.group : kRows));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  ENNX_CUDA(cudaLaunchKernelEx(&cfg, token_join_kernel, a, split_grid() * kWarps, kRows), "token attention join");
  ENNX_LAUNCH_CHECK("token attention join");
  return ENNX_B200_OK;
}
template <int kRows>
int32_t launch(const Args& a, const RopeTable& table, int64_t segs, int cluster, int dev, cudaStream_t s) {
  return cluster ? launch_whole<kRows>(a, table, segs, cluster, dev, s) : launch_split<kRows>(a, table, segs, dev, s);
}

}  // namespace
}  // namespace ennx

using namespace ennx;

extern "C" {

size_t ennx_b200_gqa_attention_decode_workspace_size(int32_t batch, int32_t room, int32_t hq, int32_t hkv) {
  if (batch <= 0 || hkv <= 0 || hq <= 0 || hq % hkv) return 0;
  const int64_t segs = segments(batch, hq, hkv);
  if (whole_cluster(segs, room)) return 0;
  return ((size_t)segs + (size_t)split_grid() * kWarps) * block_rows(hq / hkv) * kPart * sizeof(float);
}

int32_t ennx_b200_gqa_attention_decode(const ennx_b200_decode_attention* p, float rope_theta, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  cudaStream_t s = (cudaStream_t)stream;
  if (!p) return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: null parameters");
  if (p->batch < 0 || p->room <= 0 || p->hq <= 0 || p->hkv <= 0 || p->hq % p->hkv)
    return set_error(ENNX_B200_INVALID_ARGUMENT,
                     "attention_decode: room must be positive and Hq a positive multiple of Hkv");
  if (!(rope_theta >= 0.0f) || isinf(rope_theta))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: rope_theta must be finite and not negative");
  if (p->batch == 0) return ENNX_B200_OK;
  if (!p->q || !p->o || !p->k_cache || !p->v_cache || !p->lengths)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: null argument");
  if (!p->k != !p->v) return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: k and v come together");
  if (p->ld_q < (int64_t)p->hq * D || p->ld_o < (int64_t)p->hq * D ||
      (p->k && (p->ld_k < (int64_t)p->hkv * D || p->ld_v < (int64_t)p->hkv * D)))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: a row stride is shorter than its heads");
  const int64_t strides = p->k_seq | p->k_token | p->k_head | p->v_seq | p->v_token | p->v_head;
  if (strides < 0) return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: a cache stride is negative");
  if ((strides | p->ld_q | p->ld_o) % 8 ||
      (((uintptr_t)p->k_cache | (uintptr_t)p->v_cache | (uintptr_t)p->q | (uintptr_t)p->o) & 15u))
    return set_error(ENNX_B200_INVALID_ARGUMENT,
                     "attention_decode: caches, q and o must be 16-byte aligned with strides of a multiple of 8");
  const auto shared = [&](int64_t seq, int64_t token, int64_t head) {
    return (p->batch > 1 && !seq) || (p->room > 1 && !token) || (p->hkv > 1 && !head);
  };
  if (p->k && (shared(p->k_seq, p->k_token, p->k_head) || shared(p->v_seq, p->v_token, p->v_head)))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: a cache that takes k and v cannot have strides of 0");
  if (p->k && p->k_cache == p->v_cache)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: k_cache and v_cache that take k and v must be apart");
  const int group = p->hq / p->hkv, rows = block_rows(group), blocks = (group + rows - 1) / rows;
  const int64_t segs = segments(p->batch, p->hq, p->hkv);
  // a warp's run and the columns of a row are counted in 32 bits
  if (p->hq > 0x7fffffff / D || segs > 0x7fffffffLL - 65536 || segs * (p->room / kStep + 1 + kHeadCost) / ((int64_t)split_grid() * kWarps) > 0x7fffff00LL)
    return set_error(ENNX_B200_UNSUPPORTED, "attention_decode: too many heads");
  const size_t need = ennx_b200_gqa_attention_decode_workspace_size(p->batch, p->room, p->hq, p->hkv);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u)))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: a 16-byte aligned workspace of %zu bytes required",
                     need);
  const auto rows_at = [&](const uint16_t* at, int64_t ld, int heads) {
    return Memory::rows(at, p->batch, ld * 2, (int64_t)heads * D * 2);
  };
  const auto cache_at = [&](const uint16_t* at, int64_t seq, int64_t token, int64_t head) {
    return Memory{at, D * 2, {p->batch, p->room, p->hkv}, {seq * 2, token * 2, head * 2}};
  };
  const Memory mq = rows_at(p->q, p->ld_q, p->hq), mo = rows_at(p->o, p->ld_o, p->hq);
  const Memory mk = rows_at(p->k, p->ld_k, p->hkv), mv = rows_at(p->v, p->ld_v, p->hkv);
  const Memory kc = cache_at(p->k_cache, p->k_seq, p->k_token, p->k_head);
  const Memory vc = cache_at(p->v_cache, p->v_seq, p->v_token, p->v_head), ml = Memory::bytes(p->lengths, (int64_t)p->batch * 4);
  const bool in_place = p->o == p->q && (p->ld_o == p->ld_q || p->batch == 1);
  if (!in_place && share_bytes(mo, mq))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: o must be q itself or not overlap it");
  for (const Memory& m : {mk, mv, kc, vc, ml})
    if (share_bytes(mo, m))
      return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: o must not overlap k, v, the caches or lengths");
  if (p->k) {
    if (shares_own_bytes(kc) || shares_own_bytes(vc))
      return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: rows of a cache that takes k and v must not overlap");
    if (share_bytes(kc, vc))
      return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: k_cache and v_cache that take k and v must be apart");
    for (const Memory& m : {mq, mk, mv, ml})
      if (share_bytes(kc, m) || share_bytes(vc, m))
        return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: caches that take k and v must not overlap q, k, v or lengths");
  }
  const int cluster = whole_cluster(segs, p->room);
  const Args a{p->q, p->k, p->v, p->o, p->ld_q, p->ld_k, p->ld_v, p->ld_o,
               {p->k_cache, p->v_cache, p->k_seq, p->k_token, p->k_head, p->v_seq, p->v_token, p->v_head},
               p->lengths, p->batch, p->room, p->hkv, group, blocks, 1.4426950408889634f / sqrtf((float)D),
               rope_theta > 0.0f, (float*)workspace, longest_first(segs, cluster, p->batch)};
  const RopeTable& table = rope_table(rope_theta > 0.0f ? rope_theta : 1.0f);
  int dev = 0;
  int* status = nullptr;
  ENNX_TRY(serving_device(&dev, &status));
  return rows == 8 ? launch<8>(a, table, segs, cluster, dev, s) : launch<16>(a, table, segs, cluster, dev, s);
}

}  // extern "C"

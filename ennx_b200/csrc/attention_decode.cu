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
// maximum, sum and output, so no barrier stands in the loop; warps are merged
// once per sequence and head.
//
// The rotated query and the weights have more bits than bf16 holds, so both
// enter the products as hi + lo, two bf16 numbers (2^-16 of the value left).
// With at most 8 query heads the tile's other 8 rows carry the lo parts and a
// lane finds both sums in its own accumulators (rows g and g + 8): exactness
// costs no instruction.  9 to 16 heads take a second product each.
//
// Work is cut into units of 64 keys, numbered over all (sequence, cache head,
// block of kRows query heads), and every block takes an equal run of units
// whatever the lengths are: one long sequence is split over all blocks and a
// ragged batch is balanced.  Where a run ends inside a sequence its partial
// (maximum, sum, output) goes to the workspace in fp32 and a second kernel
// joins the partials in order.
#include "kernels.cuh"
#include "serve.cuh"

#include <math.h>

namespace ennx {
namespace {

constexpr int D = 128;
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStep = 16;                  // keys per warp step
constexpr int kUnit = kStep * kWarps;      // keys per unit of work
constexpr int kStages = 3;                 // ring depth: 2 steps (16 KB) in flight per warp, 128 KB per SM
constexpr int kStageBytes = 2 * kStep * D * 2;  // K and V rows of one step
constexpr int kRing = kWarps * kStages * kStageBytes;
constexpr int kQBytes = 16 * D * 2;
constexpr int kSmem = kRing + 2 * kQBytes;  // the second tile: lo parts where the heads fill the first
constexpr int kPerSm = 2;                  // blocks resident per SM (2 x 100 KB of shared memory)
static_assert(kWarps * 16 * (D + 2) * 4 <= kRing, "the merge buffer overlays the ring");

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
};

__device__ __forceinline__ int seq_len(const Args& a, int b) { return min(a.room, max(0, __ldg(a.lengths + b))); }
__device__ __forceinline__ long long seq_units(const Args& a, int b) {
  return (long long)((seq_len(a, b) + kUnit - 1) / kUnit) * a.hkv * a.blocks;
}

// Sum over sequences of their units, and (target >= 0) the sequence that
// holds unit `target` with the units before it.  By every thread of a block
// of kThreads threads.
__device__ long long scan_units(const Args& a, long long target, int* seq, long long* before) {
  __shared__ long long warp_sum[kWarps];
  __shared__ int hit_seq;
  __shared__ long long hit_before;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long run = 0;
  __syncthreads();  // an earlier call's results have been read
  if (threadIdx.x == 0) { hit_seq = -1; hit_before = 0; }
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + (int)threadIdx.x;
    const long long mine = b < a.batch ? seq_units(a, b) : 0;
    long long inc = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += up;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    long long first = run + inc - mine;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) first += warp_sum[w];
      run += warp_sum[w];
    }
    if (mine > 0 && target >= first && target < first + mine) { hit_seq = b; hit_before = first; }
  }
  __syncthreads();
  *seq = hit_seq;
  *before = hit_before;
  return run;
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
__device__ __forceinline__ void turn(float& x1, float& x2, float s, float c) {
  const float y1 = x1 * c - x2 * s;
  x2 = x2 * c + x1 * s;
  x1 = y1;
}
// hi parts of a pair packed, the pair replaced by what is left
__device__ __forceinline__ uint32_t take_hi(float& x, float& y) {
  const uint32_t hi = pack_bf16x2(x, y);
  x -= __uint_as_float(hi << 16);
  y -= __uint_as_float(hi & 0xffff0000u);
  return hi;
}
// 16-byte chunk `c` of row `r` in a tile of 256-byte rows
__device__ __forceinline__ uint32_t at(int r, int c) { return (uint32_t)(r * 256 + ((c ^ (r & 7)) << 4)); }

// kSplit: block = an equal run of all units, partials where a run ends inside
// a segment; otherwise block = one whole (sequence, cache head, head block).
template <bool kSplit, int kRows>
__global__ void __launch_bounds__(kThreads, kPerSm) token_attention_kernel(const __grid_constant__ Args a,
                                                                           const __grid_constant__ RopeTable table) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ float rot[2][64];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * kStages * kStageBytes;
  const uint32_t sq = smem_u32(smem) + kRing;
  float* merge = reinterpret_cast<float*>(smem);  // [warp][16][D + 2] over the ring, used with the ring drained

  int b;
  long long seg, left;
  int unit;  // first unit within the segment
  if constexpr (kSplit) {
    // the join kernel may start its own prologue; it waits for this grid to finish before it reads
    launch_dependents();
    long long before, total = scan_units(a, -1, &b, &before);
    const long long per = (total + gridDim.x - 1) / gridDim.x, first = per * blockIdx.x;
    left = min(per, total - first);
    if (left <= 0) return;
    scan_units(a, first, &b, &before);
    const int n = (seq_len(a, b) + kUnit - 1) / kUnit;
    const long long in_seq = first - before;
    seg = (long long)b * a.hkv * a.blocks + in_seq / n;
    unit = (int)(in_seq % n);
  } else {
    seg = blockIdx.x;
    b = (int)(seg / (a.hkv * a.blocks));
    unit = 0;
    left = (seq_len(a, b) + kUnit - 1) / kUnit;
  }

  while (true) {
    const int len = seq_len(a, b), units = (len + kUnit - 1) / kUnit;
    const int within = (int)(seg - (long long)b * a.hkv * a.blocks);
    const int h = within / a.blocks, g0 = (within % a.blocks) * kRows;
    const int rows = min(kRows, a.group - g0), hq0 = h * a.group + g0;  // query heads hq0 .. hq0 + rows - 1
    const int n = (int)min((long long)(units - unit), left);
    const uint16_t* kbase = a.c.k + (long long)b * a.c.kb + (long long)h * a.c.kh;
    const uint16_t* vbase = a.c.v + (long long)b * a.c.vb + (long long)h * a.c.vh;

    auto fetch = [&](int i) {  // keys of step i of this warp, zeros behind the last one
      if (i < n) {
        const int key0 = (unit + i) * kUnit + warp * kStep;
        const uint32_t dst = ring + (i % kStages) * kStageBytes;
#pragma unroll
        for (int j = 0; j < kStep / 2; ++j) {
          const int r = 2 * j + (lane >> 4), c = lane & 15, key = key0 + r;
          const bool ok = key < len;
          const long long tok = ok ? key : 0;
          cp_async16(dst + at(r, c), kbase + tok * a.c.kt + c * 8, ok);
          cp_async16(dst + kStep * 256 + at(r, c), vbase + tok * a.c.vt + c * 8, ok);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(i);

    // the segment's query rows, rotated, to shared memory as hi and lo
    if (a.rotate && threadIdx.x < 64) rope_sincos(table, threadIdx.x, len - 1, &rot[0][threadIdx.x], &rot[1][threadIdx.x]);
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * 64; i += kThreads) {
      const int r = i >> 6, d = i & 63;
      float x[2] = {0.0f, 0.0f};
      if (r < rows) {
        const uint16_t* src = a.q + (long long)b * a.ldq + (hq0 + r) * D + d;
        x[0] = bf16_to_f32(__ldg(src));
        x[1] = bf16_to_f32(__ldg(src + 64));
        if (a.rotate) turn(x[0], x[1], rot[0][d], rot[1][d]);
      }
      uint8_t* row = smem + kRing;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = (d + 64 * e) >> 3, byte = (d & 7) * 2;
        const uint16_t hi = f32_to_bf16_rne(x[e]), lo = f32_to_bf16_rne(x[e] - bf16_to_f32(hi));
        *reinterpret_cast<uint16_t*>(row + at(r, c) + byte) = hi;
        *reinterpret_cast<uint16_t*>(row + (kRows == 8 ? at(r + 8, c) : kQBytes + at(r, c)) + byte) = lo;
      }
    }
    __syncthreads();
    uint32_t qf[8][4];
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) ldsm4(sq + at(lane & 15, 2 * kk + (lane >> 4)), qf[kk]);

    float acc[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    // heads g (and g + 8); l of this lane's columns
    constexpr int R = kRows / 8;
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) { m[r] = -INFINITY; l[r] = 0.0f; }

    for (int i = 0; i < n; ++i) {
      cp_wait<kStages - 2>();
      __syncwarp();
      const uint32_t sk = ring + (i % kStages) * kStageBytes, sv = sk + kStep * 256;
      const int key0 = (unit + i) * kUnit + warp * kStep;
      const int p = len - 1 - key0;  // the new token's row of this step, if it is in it
      if (a.knew && p >= 0 && p < kStep) {
        // row p of the cache is written here and replaced in the copy just read
        uint8_t* st = smem + warp * kStages * kStageBytes + (i % kStages) * kStageBytes;
        uint16_t* kw = a.c.k + (long long)b * a.c.kb + (long long)h * a.c.kh + (long long)(len - 1) * a.c.kt;
        uint16_t* vw = a.c.v + (long long)b * a.c.vb + (long long)h * a.c.vh + (long long)(len - 1) * a.c.vt;
        const uint16_t* kn = a.knew + (long long)b * a.ldk + h * D;
        const uint16_t* vn = a.vnew + (long long)b * a.ldv + h * D;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = lane + 32 * e;
          float x1 = bf16_to_f32(__ldg(kn + d)), x2 = bf16_to_f32(__ldg(kn + d + 64));
          if (a.rotate) turn(x1, x2, rot[0][d], rot[1][d]);
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
      float s[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        uint32_t kf[4];
        ldsm4(sk + at((lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)), kf);
        mma(s[0], qf[kk], kf[0], kf[1]);
        mma(s[1], qf[kk], kf[2], kf[3]);
        if (kRows == 16 && a.rotate) {
          uint32_t ql[4];
          ldsm4(sq + kQBytes + at(lane & 15, 2 * kk + (lane >> 4)), ql);
          mma(s[0], ql, kf[0], kf[1]);
          mma(s[1], ql, kf[2], kf[3]);
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
          const float v = kRows == 8 ? s[nb][e] + s[nb][2 + e] : s[nb][2 * r + e];
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
      __syncwarp();  // all lanes have read the stage that the next fetch overwrites
      fetch(i + kStages - 1);
    }
    cp_wait<0>();
    __syncthreads();  // every ring is drained: the merge buffer may overlay it
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      const int row = g + 8 * r;
      float* mr = merge + (warp * 16 + row) * (D + 2);
      if (row < rows) {
#pragma unroll
        for (int nb = 0; nb < 16; ++nb)
          *reinterpret_cast<float2*>(mr + nb * 8 + 2 * t) =
              kRows == 8 ? make_float2(acc[nb][0] + acc[nb][2], acc[nb][1] + acc[nb][3])
                         : make_float2(acc[nb][2 * r], acc[nb][2 * r + 1]);
        if (t == 0) { mr[D] = m[r]; mr[D + 1] = l[r]; }
      }
    }
    __syncthreads();
    const bool whole = !kSplit || n == units;
    const int per_row = kThreads / 16;  // threads of one row
    for (int row = threadIdx.x / per_row; row < rows; row += 16) {
      float mx = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, merge[(w * 16 + row) * (D + 2) + D]);
      const float ref = mx == -INFINITY ? 0.0f : mx;
      float f[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* mr = merge + (w * 16 + row) * (D + 2);
        f[w] = ex2(mr[D] - ref);
        sum += f[w] * mr[D + 1];
      }
      const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
      float* part = kSplit ? a.partial + ((long long)blockIdx.x + seg) * 16 * (D + 2) + row * (D + 2) : nullptr;
      uint16_t* orow = a.o + (long long)b * a.ldo + (hq0 + row) * D;
      for (int d = (threadIdx.x % per_row) * 2; d < D; d += 2 * per_row) {
        float y0 = 0.0f, y1 = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 v = *reinterpret_cast<const float2*>(merge + (w * 16 + row) * (D + 2) + d);
          y0 += f[w] * v.x;
          y1 += f[w] * v.y;
        }
        if (whole) *reinterpret_cast<uint32_t*>(orow + d) = pack_bf16x2(y0 * inv, y1 * inv);
        else *reinterpret_cast<float2*>(part + d) = make_float2(y0, y1);
      }
      if (!whole && threadIdx.x % per_row == 0) *reinterpret_cast<float2*>(part + D) = make_float2(mx, sum);
    }
    left -= n;
    if (left <= 0) return;
    __syncthreads();  // the ring and the query rows are free again
    ++seg;
    unit = 0;
    if (seg == (long long)(b + 1) * a.hkv * a.blocks) {
      do ++b;
      while (b < a.batch && seq_len(a, b) == 0);
      if (b >= a.batch) return;  // not reached: `left` counts the units there are
      seg = (long long)b * a.hkv * a.blocks;
    }
  }
}

// Joins the partials of one segment (block) in the order of its keys; one
// warp per query head.  A segment of one part was written by that part's
// block, an empty one gets zeros here.
__global__ void __launch_bounds__(kThreads) token_join_kernel(const __grid_constant__ Args a, int grid, int block_rows) {
  const int seg = blockIdx.x, per_seq = a.hkv * a.blocks, b = seg / per_seq, within = seg % per_seq;
  const int len = seq_len(a, b), units = (len + kUnit - 1) / kUnit;
  // the units before this sequence, and all of them
  long long mine = 0, total;
  {
    __shared__ long long sums[2][kWarps];
    long long all = 0;
    for (int i = threadIdx.x; i < a.batch; i += kThreads) {
      const long long u = seq_units(a, i);
      all += u;
      if (i < b) mine += u;
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, off);
      mine += __shfl_xor_sync(0xffffffffu, mine, off);
    }
    if ((threadIdx.x & 31) == 0) { sums[0][threadIdx.x >> 5] = all; sums[1][threadIdx.x >> 5] = mine; }
    __syncthreads();
    total = mine = 0;
    for (int w = 0; w < kWarps; ++w) { total += sums[0][w]; mine += sums[1][w]; }
  }
  const long long first = mine + (long long)within * units;
  const long long per = total > 0 ? (total + grid - 1) / grid : 1;
  const long long c0 = first / per, c1 = units > 0 ? (first + units - 1) / per : c0;
  const int h = within / a.blocks, g0 = (within % a.blocks) * block_rows;
  const int rows = min(block_rows, a.group - g0), lane = threadIdx.x & 31;
  // the partials are complete and visible; blocks without any wait too, so
  // that this grid never ends before the one it follows
  wait_previous();
  if (units > 0 && c0 == c1) return;
  for (int row = threadIdx.x >> 5; row < rows; row += kWarps) {
    float m = -INFINITY, l = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (units > 0)
      for (long long c = c0; c <= c1; ++c) {
        const float* part = a.partial + (c + seg) * 16 * (D + 2) + row * (D + 2);
        const float2 ml = *reinterpret_cast<const float2*>(part + D);
        const float2 v0 = *reinterpret_cast<const float2*>(part + lane * 4);
        const float2 v1 = *reinterpret_cast<const float2*>(part + lane * 4 + 2);
        const float mn = fmaxf(m, ml.x), ref = mn == -INFINITY ? 0.0f : mn;
        const float f0 = ex2(m - ref), f1 = ex2(ml.x - ref);
        l = l * f0 + ml.y * f1;
        y[0] = y[0] * f0 + v0.x * f1;
        y[1] = y[1] * f0 + v0.y * f1;
        y[2] = y[2] * f0 + v1.x * f1;
        y[3] = y[3] * f0 + v1.y * f1;
        m = mn;
      }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    uint16_t* orow = a.o + (long long)b * a.ldo + (h * a.group + g0 + row) * D + lane * 4;
    *reinterpret_cast<uint2*>(orow) = make_uint2(pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv));
  }
}

// Caches of up to this many tokens are not split: at 1024 keys one block per
// head takes about as long as a split and its join together.
constexpr int kWholeRoom = 1024;

// query heads per block of rows: 8 leave room for the lo parts in the tile,
// more heads share one reading of the cache by 16
int block_rows(int group) { return group <= 8 ? 8 : 16; }

int split_grid() { return kPerSm * sm_count(); }

template <int kRows>
int32_t launch(const Args& a, const RopeTable& table, bool split, int64_t segs, int dev, cudaStream_t s) {
  static SharedMemorySetup setup[2];
  const auto kernel = split ? token_attention_kernel<true, kRows> : token_attention_kernel<false, kRows>;
  ENNX_TRY(allow_shared_memory(setup[split], dev, kernel, kSmem));
  kernel<<<split ? (unsigned)split_grid() : (unsigned)segs, kThreads, kSmem, s>>>(a, table);
  ENNX_LAUNCH_CHECK("token attention");
  return ENNX_B200_OK;
}

}  // namespace
}  // namespace ennx

using namespace ennx;

extern "C" {

size_t ennx_b200_gqa_attention_decode_workspace_size(int32_t batch, int32_t room, int32_t hq, int32_t hkv) {
  if (batch <= 0 || hkv <= 0 || hq <= 0 || hq % hkv || room <= kWholeRoom) return 0;
  const int rows = block_rows(hq / hkv);
  const size_t segs = (size_t)batch * hkv * ((hq / hkv + rows - 1) / rows);
  return (segs + split_grid()) * 16 * (D + 2) * sizeof(float);
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
  if ((strides | p->ld_q | p->ld_o) % 8 || (((uintptr_t)p->k_cache | (uintptr_t)p->v_cache | (uintptr_t)p->o) & 15u))
    return set_error(ENNX_B200_INVALID_ARGUMENT,
                     "attention_decode: caches and o must be 16-byte aligned with strides of a multiple of 8");
  const int group = p->hq / p->hkv, rows = block_rows(group), blocks = (group + rows - 1) / rows;
  const int64_t segs = (int64_t)p->batch * p->hkv * blocks;
  if (segs > 0x7fffffffLL - 65536) return set_error(ENNX_B200_UNSUPPORTED, "attention_decode: too many heads");
  const size_t need = ennx_b200_gqa_attention_decode_workspace_size(p->batch, p->room, p->hq, p->hkv);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u)))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_decode: a 16-byte aligned workspace of %zu bytes required",
                     need);
  const Args a{p->q, p->k, p->v, p->o, p->ld_q, p->ld_k, p->ld_v, p->ld_o,
               {p->k_cache, p->v_cache, p->k_seq, p->k_token, p->k_head, p->v_seq, p->v_token, p->v_head},
               p->lengths, p->batch, p->room, p->hkv, group, blocks, 1.4426950408889634f / sqrtf((float)D),
               rope_theta > 0.0f, (float*)workspace};
  const RopeTable& table = rope_table(rope_theta > 0.0f ? rope_theta : 1.0f);
  int dev = 0;
  int* status = nullptr;
  ENNX_TRY(serving_device(&dev, &status));
  ENNX_TRY(rows == 8 ? launch<8>(a, table, need != 0, segs, dev, s) : launch<16>(a, table, need != 0, segs, dev, s));
  if (!need) return ENNX_B200_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)segs);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  ENNX_CUDA(cudaLaunchKernelEx(&cfg, token_join_kernel, a, split_grid(), rows), "token attention join");
  ENNX_LAUNCH_CHECK("token attention join");
  return ENNX_B200_OK;
}

}  // extern "C"

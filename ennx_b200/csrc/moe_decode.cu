// moe_decode.cu -- the mixture-of-experts layer for a few tokens (at most 64).
//
//   l = W_r x;  e_1 .. e_k the largest logits (strict '>': the lower expert
//   wins a tie), gate_r = softmax over those k;
//   y = residual + sum_r gate_r W_d[e_r] (silu(W_g[e_r] x) * W_u[e_r] x).
//
// Bound: HBM.  A weight of a picked expert is read once and used by the few
// tokens that picked it, so the layer is as fast as those weights stream in;
// the grouped GEMM path of the full layer spends its time on permuting rows
// and on tiles of 128 tokens instead.
//
// Three kernels in one programmatic-launch chain: router logits; gate/up
// products with SwiGLU; down products with the weighted sum.  The last two
// give every block an equal share of the weight rows whatever the routing is
// (gate/up: an equal run of the picked experts' columns; down: an equal share
// of the output rows over all picked experts, so a block owns its outputs and
// sums the experts in a fixed order without atomics).  Each block derives the
// routing from the logits itself, which costs less than another launch.
//
// Products run on m16n8k16 with weight rows as the 16 rows and tokens as the
// 8 columns; each warp streams its own weight tiles through a ring of bulk
// copies, a row (512 bytes) each: copying with a 16-byte instruction per lane
// instead took 6 times the instructions and was bound by them (64 tokens 212
// us).  k is permuted the same way in both operands so that a lane's fragments
// are 16 contiguous bytes.
#include "kernels.cuh"
#include "serve.cuh"

#include <math.h>

namespace ennx {
namespace {

constexpr int kTokens = 64, kTopK = 8, kExperts = 256;
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kChunk = 32;       // k of one 64-byte piece per row: two products of 16
constexpr int kTileChunks = 8;   // chunks of a warp's tile
constexpr int kStages = 3;       // two tiles of 8 KB in flight per warp, 128 KB per SM
// Rows of a tile in shared memory, in pairs 1088 bytes apart, the second row
// 576 bytes behind the first: the two rows of an 8-lane phase, 64 bytes each,
// then lie on different banks wherever the phase starts.
__device__ __forceinline__ constexpr uint32_t row_at(int r) { return (uint32_t)((r >> 1) * 1088 + (r & 1) * 576); }
constexpr int tile_bytes(int rows) { return (rows + 1) / 2 * 1088; }

struct Layer {
  const uint16_t *x, *w_router, *w_gate_up, *w_down, *residual;
  uint16_t* y;
  int* index;     // nullable
  float* gate;    // nullable
  float* logits;  // [tokens][experts]
  uint16_t* act;  // [tokens * top_k][width], rows expert by expert
  int tokens, hidden, experts, top_k, width;
  int* status;
};

// A warp's ring of weight tiles, filled by one bulk copy per row.
struct Ring {
  uint8_t* base;
  uint64_t* full;
  int stage_bytes, fetched, used;
  bool bad;  // a wait gave up: later ones are not tried again, the results are void
  __device__ __forceinline__ void init(uint8_t* at, uint64_t* bars, int bytes, int lane) {
    base = at; full = bars; stage_bytes = bytes; fetched = used = 0; bad = false;
    if (lane < kStages) mbar_init(full + lane, 1);
    fence_barrier_init();
    fence_proxy_async();
    __syncwarp();
  }
  // lane r < 16 copies row r from `src` where `ok`; the same `bytes` per row
  __device__ __forceinline__ void fetch(const uint16_t* src, bool ok, int bytes, int lane) {
    const int at = fetched % kStages;
    const uint32_t copies = __popc(__ballot_sync(0xffffffffu, ok));
    if (lane == 0) mbar_arrive_expect_tx(full + at, copies * bytes);
    __syncwarp();
    if (ok) bulk_copy(smem_u32(base) + at * stage_bytes + row_at(lane), src, bytes, full + at);
    ++fetched;
  }
  __device__ __forceinline__ uint32_t wait(int* status) {  // the next tile's address
    const int at = used % kStages;
    if (!bad) bad = !mbar_wait(full + at, (used / kStages) & 1, status);
    ++used;
    return smem_u32(base) + at * stage_bytes;
  }
};

// ---------------------------------------------------------------------------
// router logits: block = 4 experts x 8 tokens, a thread 8 k at a time.  Each
// logit is an fp32 sum over the threads' short chains (8 or 16 products at
// hidden 2048) joined as a tree.
// ---------------------------------------------------------------------------
constexpr int kRE = 4, kRT = 8;
__global__ void __launch_bounds__(kThreads) token_router_kernel(const __grid_constant__ Layer p) {
  launch_dependents();
  __shared__ float part[kWarps][kRE][kRT];
  const int e0 = blockIdx.x * kRE, t0 = blockIdx.y * kRT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float acc[kRE][kRT] = {};
  for (int c = threadIdx.x; c < p.hidden / 8; c += kThreads) {
    uint4 w[kRE];
#pragma unroll
    for (int e = 0; e < kRE; ++e)
      w[e] = e0 + e < p.experts ? ldg_stream_v4(p.w_router + (long long)(e0 + e) * p.hidden + c * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < kRT; ++t) {
      if (t0 + t < p.tokens) {
        const uint4 xv = __ldg(reinterpret_cast<const uint4*>(p.x + (long long)(t0 + t) * p.hidden + c * 8));
        const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
        for (int e = 0; e < kRE; ++e) {
          const uint32_t ww[4] = {w[e].x, w[e].y, w[e].z, w[e].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[e][t] = fmaf(__uint_as_float(xw[j] << 16), __uint_as_float(ww[j] << 16), acc[e][t]);
            acc[e][t] = fmaf(__uint_as_float(xw[j] & 0xffff0000u), __uint_as_float(ww[j] & 0xffff0000u), acc[e][t]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kRT; ++t)
    if (t0 + t < p.tokens) {
#pragma unroll
      for (int e = 0; e < kRE; ++e) {
        float v = acc[e][t];
#pragma unroll
        for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        if (lane == 0) part[warp][e][t] = v;
      }
    }
  __syncthreads();
  const int e = threadIdx.x / kRT, t = threadIdx.x % kRT;
  if (e < kRE && e0 + e < p.experts && t0 + t < p.tokens) {
    float v[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v[w] = part[w][e][t];
    p.logits[(t0 + t) * p.experts + e0 + e] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  }
}

// ---------------------------------------------------------------------------
// routing of all tokens, by every block for itself
// ---------------------------------------------------------------------------
struct Plan {
  float gates[kTokens * kTopK];     // of pick r of token t at t * kTopK + r
  uint8_t picks[kTokens * kTopK];
  uint32_t takers[kExperts][2];     // tokens that picked an expert, a bit each
  int active;                       // experts that some token picked
  uint8_t expert[kExperts];         // active expert a
  uint16_t first[kExperts + 1];     // its first slot; slots run expert by expert, token by token
  uint16_t slot[kTokens * kTopK];   // t * kTopK + r of a slot
  int scan[kWarps][2];
  __device__ __forceinline__ int token(int i) const { return slot[i] / kTopK; }
  __device__ __forceinline__ float gate(int i) const { return gates[slot[i]]; }
};

// NaN sorts below everything, so that it never displaces a number
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return v != v ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ void make_plan(const Layer& p, Plan& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kPer = kExperts / 32;
  for (int i = threadIdx.x; i < 2 * kExperts; i += kThreads) s.takers[i >> 1][i & 1] = 0u;
  for (int t = warp; t < p.tokens; t += kWarps) {
    float v[kPer];
    uint32_t key[kPer];  // 0 with `taken`: picked already or no expert
    uint32_t taken = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = i * 32 + lane;
      v[i] = e < p.experts ? __ldcg(p.logits + t * p.experts + e) : 0.0f;
      key[i] = order_key(v[i]);
      if (e >= p.experts) taken |= 1u << i;
    }
    float top = 0.0f, sum = 0.0f, mine = 0.0f;
    int pick = 0;
    for (int r = 0; r < p.top_k; ++r) {
      uint32_t best = 0;
      int at = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i * 32 < p.experts && !(taken >> i & 1u) && (at == 0x7fffffff || key[i] > best)) {
          best = key[i];
          at = i * 32 + lane;
        }
      const uint32_t m = __reduce_max_sync(0xffffffffu, at == 0x7fffffff ? 0u : best);
      const int e = __reduce_min_sync(0xffffffffu, at != 0x7fffffff && best == m ? at : 0x7fffffff);
      float val = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (e == i * 32 + lane) {
          taken |= 1u << i;
          val = v[i];
        }
      val = __shfl_sync(0xffffffffu, val, e & 31);
      if (r == 0) top = val;
      const float g = expf(val - top);
      sum += g;
      if (lane == r) {
        mine = g;
        pick = e;
      }
    }
    if (lane < p.top_k) {
      s.picks[t * kTopK + lane] = (uint8_t)pick;
      s.gates[t * kTopK + lane] = mine / sum;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.tokens * p.top_k; i += kThreads) {
    const int t = i / p.top_k, e = s.picks[t * kTopK + i % p.top_k];
    atomicOr(&s.takers[e][t >> 5], 1u << (t & 31));
  }
  __syncthreads();
  static_assert(kThreads == kExperts, "a thread per expert");
  const uint32_t lo = s.takers[threadIdx.x][0], hi = s.takers[threadIdx.x][1];
  const int n = __popc(lo) + __popc(hi);
  int slots = n, actives = n > 0;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, slots, off), b = __shfl_up_sync(0xffffffffu, actives, off);
    if (lane >= off) { slots += a; actives += b; }
  }
  if (lane == 31) { s.scan[warp][0] = slots; s.scan[warp][1] = actives; }
  __syncthreads();
  for (int w = 0; w < warp; ++w) { slots += s.scan[w][0]; actives += s.scan[w][1]; }
  if (threadIdx.x == kThreads - 1) {
    s.active = actives;
    s.first[actives] = (uint16_t)slots;
  }
  if (n > 0) {
    int slot = slots - n;
    s.expert[actives - 1] = (uint8_t)threadIdx.x;
    s.first[actives - 1] = (uint16_t)slot;
    for (int t = 0; t < p.tokens; ++t)
      if ((t < 32 ? lo >> t : hi >> (t - 32)) & 1u) {
        int at = t * kTopK;
        for (int r = 0; r < p.top_k; ++r)
          if (s.picks[t * kTopK + r] == threadIdx.x) at = t * kTopK + r;
        s.slot[slot++] = (uint16_t)at;
      }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------
// gate/up: a block takes an equal run of the (picked expert, column) list.  A
// tile is 8 columns (8 gate rows and their 8 up rows) x all k, the k split
// over the warps; kN blocks of 8 tokens at a time stay in registers.
// ---------------------------------------------------------------------------
template <int kN>
struct GateUpShared {
  uint8_t ring[kWarps][kStages][tile_bytes(16)];
  float4 red[2][kWarps][kN][32];
  uint64_t full[kWarps][kStages];
  Plan plan;
};

template <int kN>
__global__ void __launch_bounds__(kThreads, 1) token_gate_up_kernel(const __grid_constant__ Layer p) {
  extern __shared__ __align__(128) uint8_t smem[];
  GateUpShared<kN>& sh = *reinterpret_cast<GateUpShared<kN>*>(smem);
  Plan& s = sh.plan;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  Ring ring;
  ring.init(sh.ring[warp][0], sh.full[warp], tile_bytes(16), lane);
  wait_previous();
  launch_dependents();
  make_plan(p, s);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.tokens * p.top_k; i += kThreads) {
      const int at = i / p.top_k * kTopK + i % p.top_k;
      if (p.index) p.index[i] = s.picks[at];
      if (p.gate) p.gate[i] = s.gates[at];
    }

  const long long columns = (long long)s.active * p.width;
  const long long begin = columns * blockIdx.x / gridDim.x, end = columns * (blockIdx.x + 1) / gridDim.x;
  if (begin >= end) return;
  const int a_first = (int)(begin / p.width), a_last = (int)((end - 1) / p.width);
  const int c_first = (int)(begin - (long long)a_first * p.width), c_last = (int)(end - (long long)a_last * p.width);
  const int chunks = p.hidden / kChunk, passes = (chunks + kWarps * kTileChunks - 1) / (kWarps * kTileChunks);
  const int per = ((chunks + passes - 1) / passes + kWarps - 1) / kWarps;  // chunks of a warp in a pass

  // tiles in order: expert, group of kN * 8 tokens, 8 columns, k pass
  struct Walk {
    int a, c, c_begin, c_end, group, groups, pass;
  };
  auto enter = [&](Walk& w) {  // first tile of expert w.a
    w.c = w.c_begin = w.a == a_first ? c_first : 0;
    w.c_end = w.a == a_last ? c_last : p.width;
    w.groups = (s.first[w.a + 1] - s.first[w.a] + kN * 8 - 1) / (kN * 8);
    w.group = w.pass = 0;
  };
  auto next = [&](Walk& w) -> bool {  // false behind the last tile
    if (++w.pass < passes) return true;
    w.pass = 0;
    w.c += 8;
    if (w.c < w.c_end) return true;
    w.c = w.c_begin;
    if (++w.group < w.groups) return true;
    if (++w.a > a_last) return false;
    enter(w);
    return true;
  };
  auto chunk0 = [&](int pass) { return (pass * kWarps + warp) * per; };
  auto valid = [&](int pass) { return max(0, min(per, chunks - chunk0(pass))); };  // chunks of this warp's tile

  Walk ahead, now;
  ahead.a = a_first;
  enter(ahead);
  now = ahead;
  bool more = true;
  auto fetch = [&] {
    if (!more) return;
    const int col = ahead.c + (lane & 7), row = (col >> 7) * 256 + (lane >> 3) * 128 + (col & 127), n = valid(ahead.pass);
    const uint16_t* w = p.w_gate_up + ((long long)s.expert[ahead.a] * 2 * p.width + row) * p.hidden + chunk0(ahead.pass) * kChunk;
    ring.fetch(w, lane < 16 && col < ahead.c_end && n > 0, n * 64, lane);
    more = next(ahead);
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  uint4 xf[kTileChunks][kN];
  bool reload = true;
  float acc[kN][4];
  for (int done = 0;;) {
    const int n_chunks = valid(now.pass), first = s.first[now.a] + now.group * kN * 8, last = s.first[now.a + 1];
    if (reload) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int slot = first + n * 8 + g;
        const bool ok = slot < last;
        const uint16_t* x = p.x + (ok ? (long long)s.token(slot) * p.hidden : 0) + chunk0(now.pass) * kChunk + t * 8;
#pragma unroll
        for (int j = 0; j < kTileChunks; ++j)
          xf[j][n] = ok && j < n_chunks ? __ldg(reinterpret_cast<const uint4*>(x + j * kChunk)) : make_uint4(0, 0, 0, 0);
      }
    }
    if (now.pass == 0) {
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][j] = 0.0f;
    }
    const uint32_t tile = ring.wait(p.status) + row_at(g) + 16 * t;  // row g + 8: row_at(8) further on
#pragma unroll
    for (int j = 0; j < kTileChunks; ++j) {
      if (j < n_chunks) {
        const uint4 a = lds128(tile + 64 * j), b = lds128(tile + row_at(8) + 64 * j);
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          mma_16x8x16(acc[n], a.x, b.x, a.y, b.y, xf[j][n].x, xf[j][n].y);
          mma_16x8x16(acc[n], a.z, b.z, a.w, b.w, xf[j][n].z, xf[j][n].w);
        }
      }
    }
    __syncwarp();
    fetch();
    if (now.pass == passes - 1) {
      float4(&buf)[kWarps][kN][32] = sh.red[done & 1];
      ++done;
#pragma unroll
      for (int n = 0; n < kN; ++n) buf[warp][n][lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
      // one barrier a tile: the other buffer is written again only after the
      // next barrier, which every reader of this one reaches first
      __syncthreads();
      if (warp < kN) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 u = buf[w][warp][lane];
          v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
        }
        const int col = now.c + g, slot = first + warp * 8 + 2 * t;
        if (col < now.c_end) {
          // rounded to bf16 for the second product: at most 2^-8 of a value
          uint16_t* h = p.act + (long long)slot * p.width + col;
          if (slot < last) h[0] = f32_to_bf16_rne(v.x / (1.0f + expf(-v.x)) * v.z);
          if (slot + 1 < last) h[p.width] = f32_to_bf16_rne(v.y / (1.0f + expf(-v.y)) * v.w);
        }
      }
    }
    const int a = now.a, group = now.group;
    if (!next(now)) break;
    reload = passes > 1 || now.a != a || now.group != group;
  }
}

// ---------------------------------------------------------------------------
// down: a block owns an equal share of the output rows (kRows at a time: 14 of
// the 16 of a product, 2048 rows over 148 blocks, keep the sums of 64 tokens
// in shared memory beside the ring) over all picked experts; experts go round
// the warps, a warp's tile is kRows rows x 256 k.
// ---------------------------------------------------------------------------
constexpr int kRows = 14;
struct DownShared {
  uint8_t ring[kWarps][kStages][tile_bytes(kRows)];
  uint64_t full[kWarps][kStages];
  Plan plan;
  float sums[1];  // [warp][token][kRows]
};

template <int kN>
__global__ void __launch_bounds__(kThreads, 1) token_down_kernel(const __grid_constant__ Layer p) {
  extern __shared__ __align__(128) uint8_t smem[];
  DownShared& sh = *reinterpret_cast<DownShared*>(smem);
  Plan& s = sh.plan;
  const int span = p.tokens * kRows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  float* sums = sh.sums + warp * span;
  Ring ring;
  ring.init(sh.ring[warp][0], sh.full[warp], tile_bytes(kRows), lane);
  // the router grid has finished (every gate/up block waited for it before it
  // let this grid start), so the routing and the first weights can be fetched
  // while the gate/up products are still running
  make_plan(p, s);
  const int chunks = p.width / kChunk, passes = (chunks + kTileChunks - 1) / kTileChunks;
  const int row_begin = (int)((long long)p.hidden * blockIdx.x / gridDim.x);
  const int row_end = (int)((long long)p.hidden * (blockIdx.x + 1) / gridDim.x);
  bool waited = false;

  for (int row0 = row_begin; row0 < row_end; row0 += kRows) {
    const int rows = min(kRows, row_end - row0);
    struct Walk {
      int a, group, pass;
    };
    auto next = [&](Walk& w) -> bool {
      if (++w.pass < passes) return true;
      w.pass = 0;
      if (++w.group * kN * 8 < s.first[w.a + 1] - s.first[w.a]) return true;
      w.group = 0;
      w.a += kWarps;
      return w.a < s.active;
    };
    Walk ahead{warp, 0, 0}, now = ahead;
    bool more = warp < s.active;
    auto fetch = [&] {
      if (!more) return;
      const int k0 = ahead.pass * kTileChunks, n = min(kTileChunks, chunks - k0);
      const uint16_t* w = p.w_down + ((long long)s.expert[ahead.a] * p.hidden + row0 + lane) * p.width + k0 * kChunk;
      ring.fetch(w, lane < rows, n * 64, lane);
      more = next(ahead);
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch();
    for (int i = lane; i < span; i += 32) sums[i] = 0.0f;
    if (!waited) {
      wait_previous();  // the activations are complete and visible
      waited = true;
    }
    __syncwarp();
    float acc[kN][4];
    while (warp < s.active) {
      const int first = s.first[now.a] + now.group * kN * 8, last = s.first[now.a + 1];
      const int k0 = now.pass * kTileChunks, n_chunks = min(kTileChunks, chunks - k0);
      uint4 hf[kTileChunks][kN];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const bool ok = first + n * 8 + g < last;
        const uint16_t* h = p.act + (ok ? (long long)(first + n * 8 + g) * p.width : 0) + k0 * kChunk + t * 8;
#pragma unroll
        for (int j = 0; j < kTileChunks; ++j)
          hf[j][n] = ok && j < n_chunks ? __ldcg(reinterpret_cast<const uint4*>(h + j * kChunk)) : make_uint4(0, 0, 0, 0);
      }
      if (now.pass == 0) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[n][j] = 0.0f;
      }
      // rows 14 and 15 of the product are not copied: whatever lies there
      // (the next tile's first bytes) enters only their own sums
      const uint32_t tile = ring.wait(p.status) + row_at(g) + 16 * t;
#pragma unroll
      for (int j = 0; j < kTileChunks; ++j) {
        if (j < n_chunks) {
          const uint4 a = lds128(tile + 64 * j), b = lds128(tile + (g < kRows - 8 ? row_at(8) : 0u) + 64 * j);
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            mma_16x8x16(acc[n], a.x, b.x, a.y, b.y, hf[j][n].x, hf[j][n].y);
            mma_16x8x16(acc[n], a.z, b.z, a.w, b.w, hf[j][n].z, hf[j][n].w);
          }
        }
      }
      __syncwarp();
      fetch();
      if (now.pass == passes - 1) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int slot = first + n * 8 + 2 * t + e;
            if (slot < last) {
              float* to = sums + s.token(slot) * kRows + g;
              const float gate = s.gate(slot);
              to[0] += gate * acc[n][e];
              if (g < kRows - 8) to[8] += gate * acc[n][2 + e];
            }
          }
        __syncwarp();
      }
      if (!next(now)) break;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < span; i += kThreads) {
      const int tok = i / kRows, r = i % kRows;
      if (r < rows) {
        const long long at = (long long)tok * p.hidden + row0 + r;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += sh.sums[w * span + i];
        if (p.residual) v += bf16_to_f32(p.residual[at]);
        p.y[at] = f32_to_bf16_rne(v);
      }
    }
    __syncthreads();
  }
  if (!waited) wait_previous();  // no grid of the chain ends before the one it follows
}

constexpr size_t down_smem(int tokens) { return sizeof(DownShared) + sizeof(float) * kWarps * tokens * kRows; }
static_assert(sizeof(GateUpShared<2>) <= 227 * 1024 && down_smem(kTokens) <= 227 * 1024, "shared memory of one block");

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename K>
int32_t launch_after(SharedMemorySetup& setup, int dev, K kernel, size_t smem, size_t most, const Layer& p, cudaStream_t s) {
  ENNX_TRY(allow_shared_memory(setup, dev, kernel, (int)most));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sm_count());
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  ENNX_CUDA(cudaLaunchKernelEx(&cfg, kernel, p), "few-token moe");
  ENNX_LAUNCH_CHECK("few-token moe");
  return ENNX_B200_OK;
}
template <int kN>
int32_t launch_experts(const Layer& p, int dev, cudaStream_t s) {
  static SharedMemorySetup setup[2];
  constexpr size_t smem = sizeof(GateUpShared<kN>);
  ENNX_TRY(launch_after(setup[0], dev, token_gate_up_kernel<kN>, smem, smem, p, s));
  return launch_after(setup[1], dev, token_down_kernel<kN>, down_smem(p.tokens), down_smem(kTokens), p, s);
}

}  // namespace
}  // namespace ennx

using namespace ennx;

extern "C" {

size_t ennx_b200_moe_layer_decode_workspace_size(int64_t tokens, int32_t experts, int32_t top_k, int32_t expert_width) {
  if (tokens <= 0 || tokens > kTokens || experts <= 0 || top_k <= 0 || expert_width <= 0) return 0;
  return round256(sizeof(float) * tokens * experts) + round256(sizeof(uint16_t) * tokens * top_k * expert_width);
}

int32_t ennx_b200_moe_layer_decode(const uint16_t* x, const uint16_t* w_router, const uint16_t* w_gate_up,
                                   const uint16_t* w_down, int64_t tokens, int32_t hidden, int32_t experts,
                                   int32_t top_k, int32_t expert_width, const uint16_t* residual, uint16_t* y,
                                   int32_t* index, float* gate, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  cudaStream_t s = (cudaStream_t)stream;
  if (tokens < 0) return set_error(ENNX_B200_INVALID_ARGUMENT, "moe_layer_decode: negative token count");
  if (top_k < 1 || top_k > kTopK || top_k > experts)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "moe_layer_decode: top_k must be in [1, min(8, experts)]");
  if (tokens > kTokens || experts > kExperts)
    return set_error(ENNX_B200_UNSUPPORTED, "moe_layer_decode: at most %d tokens and %d experts", kTokens, kExperts);
  if (hidden <= 0 || hidden % 64 || expert_width <= 0 || expert_width % 128)
    return set_error(ENNX_B200_UNSUPPORTED,
                     "moe_layer_decode: hidden must be a multiple of 64 and the expert width of 128");
  if (tokens == 0) return ENNX_B200_OK;
  if (!x || !w_router || !w_gate_up || !w_down || !y)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "moe_layer_decode: null argument");
  if (((uintptr_t)x | (uintptr_t)w_router | (uintptr_t)w_gate_up | (uintptr_t)w_down) & 15u)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "moe_layer_decode: x and the weights must be 16-byte aligned");
  const size_t need = ennx_b200_moe_layer_decode_workspace_size(tokens, experts, top_k, expert_width);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "moe_layer_decode: a 16-byte aligned workspace of %zu bytes required",
                     need);
  int dev = 0;
  int* status = nullptr;
  ENNX_TRY(serving_device(&dev, &status));
  const Layer p{x, w_router, w_gate_up, w_down, residual, y, index, gate, (float*)workspace,
                (uint16_t*)((uint8_t*)workspace + round256(sizeof(float) * tokens * experts)),
                (int)tokens, hidden, experts, top_k, expert_width, status};
  const dim3 router((unsigned)((experts + kRE - 1) / kRE), (unsigned)((tokens + kRT - 1) / kRT));
  token_router_kernel<<<router, kThreads, 0, s>>>(p);
  ENNX_LAUNCH_CHECK("few-token router");
  return tokens <= 8 ? launch_experts<1>(p, dev, s) : launch_experts<2>(p, dev, s);
}

}  // extern "C"

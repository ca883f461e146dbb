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
// Three kernels in one programmatic-launch chain: router; gate/up products
// with SwiGLU; down products with the weighted sum.  The last two give every
// block an equal share of the weight rows whatever the routing is (gate/up: an
// equal run of the picked experts' columns; down: an equal share of the output
// rows over all picked experts, so a block owns its outputs and sums the
// experts in a fixed order without atomics).  Each block sorts the picks by
// expert for itself, about a microsecond, which costs less than another launch.
//
// Products run on m16n8k16 with weight rows as the 16 rows and tokens as the
// 8 columns; each warp streams its own weight tiles through a ring of bulk
// copies, a row (512 bytes) each: copying with a 16-byte instruction per lane
// instead took 6 times the instructions and was bound by them (the layer for 64
// tokens 212 us).  k is permuted the same way in both operands so that a lane's
// fragments are 16 contiguous bytes.
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
  uint8_t* picks;  // [tokens][kTopK]
  float* gates;    // [tokens][kTopK]
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
  __device__ __forceinline__ void drain(int* status) {  // after a wait that gave up: no copy may land behind the block
    if (!bad) return;
    for (int i = max(0, fetched - kStages); i < fetched; ++i) mbar_wait(full + i % kStages, (i / kStages) & 1, status);
  }
};

// ---------------------------------------------------------------------------
// router: a cluster of 8 blocks takes 8 tokens; each block forms the logits of
// an eighth of the experts, block r gathers those of token r over distributed
// shared memory and picks.  A logit is an fp32 sum: a thread's chain of 8
// products (16 at hidden 4096), joined as a tree.
// ---------------------------------------------------------------------------
constexpr int kCluster = 8;

// NaN sorts below everything, so that it never displaces a number
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return v != v ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Sum of N values over the lanes, N a power of two up to 64: each exchange
// halves the values a lane holds while it can, so lane l ends with the N / 32
// values from l * N / 32 on (N < 32: value l * N / 32, in all its lanes).
template <int N, int kOff = 16>
__device__ __forceinline__ void spread_sum(float* v, int lane) {
  if constexpr (kOff > 0) {
    if constexpr (N > 1) {
      const bool upper = lane & kOff;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float send = upper ? v[i] : v[i + N / 2], keep = upper ? v[i + N / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, kOff);
      }
      spread_sum<N / 2, kOff / 2>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], kOff);
      spread_sum<1, kOff / 2>(v, lane);
    }
  }
}

template <int kT>  // tokens of a cluster
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads)
    token_router_kernel(const __grid_constant__ Layer p) {
  constexpr int kE = 8, kV = kE * kT;  // experts at a time, sums at a time
  constexpr int kHeld = kV >= 32 ? kV / 32 : 1, kRepeat = kV >= 32 ? 1 : 32 / kV;  // values a lane ends with, lanes of a value
  __shared__ float part[kWarps][kV];
  __shared__ float logits[kExperts];
  cluster_arrive();  // waited for before the first store to another block, which has to have started by then
  bool met = false;
  launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = (int)cluster_ctarank();
  const int t0 = (int)(blockIdx.x / kCluster) * kT;
  const int per = (p.experts + kCluster - 1) / kCluster, e_end = min(p.experts, (rank + 1) * per);
  for (int e0 = rank * per; e0 < e_end; e0 += kE) {
    float acc[kV] = {};
    for (int c = threadIdx.x; c < p.hidden / 8; c += kThreads) {
      uint4 x[kT];
#pragma unroll
      for (int t = 0; t < kT; ++t)
        x[t] = t0 + t < p.tokens ? __ldg(reinterpret_cast<const uint4*>(p.x + (long long)(t0 + t) * p.hidden + c * 8))
                                 : make_uint4(0, 0, 0, 0);
      uint4 w[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e)
        w[e] = e0 + e < e_end ? ldg_stream_v4(p.w_router + (long long)(e0 + e) * p.hidden + c * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const uint32_t ww[4] = {w[e].x, w[e].y, w[e].z, w[e].w};
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          const uint32_t xw[4] = {x[t].x, x[t].y, x[t].z, x[t].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[e * kT + t] = fmaf(__uint_as_float(xw[j] << 16), __uint_as_float(ww[j] << 16), acc[e * kT + t]);
            acc[e * kT + t] = fmaf(__uint_as_float(xw[j] & 0xffff0000u), __uint_as_float(ww[j] & 0xffff0000u), acc[e * kT + t]);
          }
        }
      }
    }
    spread_sum<kV>(acc, lane);
    __syncthreads();  // the sums of the experts before have been read
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (lane % kRepeat == 0) part[warp][lane / kRepeat * kHeld + i] = acc[i];
    __syncthreads();
    if (!met) {  // block-uniform
      cluster_wait();
      met = true;
    }
    if (threadIdx.x < kV) {
      float v[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v[w] = part[w][threadIdx.x];
      const float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      const int e = e0 + (int)threadIdx.x / kT, t = (int)threadIdx.x % kT;
      if (e < e_end)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(&logits[e], (uint32_t)t)), "f"(sum) : "memory");
    }
  }
  if (!met) cluster_wait();  // a block without experts
  cluster_sync();  // every block has all logits of its token; nothing remote is touched behind it
  const int tok = t0 + rank;
  if (rank >= kT || tok >= p.tokens || warp != 0) return;
  constexpr int kPer = kExperts / 32;
  float v[kPer];
  uint32_t key[kPer], taken = 0;  // taken: picked already, or no expert
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = i * 32 + lane;
    v[i] = e < p.experts ? logits[e] : 0.0f;
    key[i] = order_key(v[i]);
    if (e >= p.experts) taken |= 1u << i;
  }
  float top = 0.0f, mine = 0.0f;
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
    const uint32_t m = __reduce_max_sync(0xffffffffu, best);
    const int e = __reduce_min_sync(0xffffffffu, best == m ? at : 0x7fffffff);
    if ((e & 31) == lane) taken |= 1u << (e >> 5);
    if (lane == r) pick = e;
  }
  if (lane < p.top_k) mine = logits[pick];
  top = __shfl_sync(0xffffffffu, mine, 0);
  const float g = lane < p.top_k ? expf(mine - top) : 0.0f;
  float sum = g;
#pragma unroll
  for (int off = 4; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);  // lanes 0 .. 7
  if (lane < p.top_k) {
    p.picks[tok * kTopK + lane] = (uint8_t)pick;
    p.gates[tok * kTopK + lane] = g / sum;
    if (p.index) p.index[tok * p.top_k + lane] = pick;
    if (p.gate) p.gate[tok * p.top_k + lane] = g / sum;
  }
}

// ---------------------------------------------------------------------------
// picks of all tokens sorted by expert, by every block for itself
// ---------------------------------------------------------------------------
struct Plan {
  float gates[kTokens * kTopK];  // of pick r of token t at t * kTopK + r
  uint32_t takers[kExperts][2];  // tokens that picked an expert, a bit each
  uint16_t start[kExperts];      // first slot of an expert
  int active;                    // experts that some token picked
  uint8_t expert[kExperts];      // active expert a
  uint16_t first[kExperts + 1];  // its first slot; slots run expert by expert, token by token
  uint16_t groups[kExperts + 1];  // groups of tokens of the active experts before it
  uint16_t slot[kTokens * kTopK];  // t * kTopK + r of a slot
  uint16_t scan[kWarps][3];
  __device__ __forceinline__ int token(int i) const { return slot[i] / kTopK; }
  __device__ __forceinline__ float gate(int i) const { return gates[slot[i]]; }
};

// by every thread of a block; those behind the first kThreads only keep step
template <int kGroup>  // tokens of a group
__device__ __forceinline__ void make_plan(const Layer& p, Plan& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool works = threadIdx.x < kThreads;
  constexpr int kMine = kTokens * kTopK / kThreads;
  int pick[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {  // pick r of token t, -1 behind the last
    const int at = threadIdx.x + i * kThreads;
    const bool ok = works && at / kTopK < p.tokens && at % kTopK < p.top_k;
    pick[i] = ok ? (int)__ldcg(p.picks + at) : -1;
    if (ok) s.gates[at] = __ldcg(p.gates + at);
  }
  static_assert(kThreads == kExperts, "a thread per expert");
  if (works) s.takers[threadIdx.x][0] = s.takers[threadIdx.x][1] = 0u;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int t = (threadIdx.x + i * kThreads) / kTopK;
    if (pick[i] >= 0) atomicOr(&s.takers[pick[i]][t >> 5], 1u << (t & 31));
  }
  __syncthreads();
  const int n = works ? __popc(s.takers[threadIdx.x][0]) + __popc(s.takers[threadIdx.x][1]) : 0;
  const int own = (n + kGroup - 1) / kGroup;
  int slots = n, actives = n > 0, groups = own;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, slots, off), b = __shfl_up_sync(0xffffffffu, actives, off);
    const int c = __shfl_up_sync(0xffffffffu, groups, off);
    if (lane >= off) { slots += a; actives += b; groups += c; }
  }
  if (works && lane == 31) {
    s.scan[warp][0] = (uint16_t)slots;
    s.scan[warp][1] = (uint16_t)actives;
    s.scan[warp][2] = (uint16_t)groups;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps - 1; ++w)
    if (w < warp) { slots += s.scan[w][0]; actives += s.scan[w][1]; groups += s.scan[w][2]; }
  if (works) s.start[threadIdx.x] = (uint16_t)(slots - n);
  if (threadIdx.x == kThreads - 1) {
    s.active = actives;
    s.first[actives] = (uint16_t)slots;
    s.groups[actives] = (uint16_t)groups;
  }
  if (n > 0) {
    s.expert[actives - 1] = (uint8_t)threadIdx.x;
    s.first[actives - 1] = (uint16_t)(slots - n);
    s.groups[actives - 1] = (uint16_t)(groups - own);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = threadIdx.x + i * kThreads, t = at / kTopK;
    if (pick[i] >= 0) {
      const uint32_t lo = s.takers[pick[i]][0], hi = s.takers[pick[i]][1], below = (1u << (t & 31)) - 1u;
      s.slot[s.start[pick[i]] + (t < 32 ? __popc(lo & below) : __popc(lo) + __popc(hi & below))] = (uint16_t)at;
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------
// gate/up: a block takes an equal run of the (picked expert, column) list, an
// expert's columns counted once per group of its tokens (counted once, a block
// of an expert with 17 tokens or more took twice as long as the others: the
// layer for 64 tokens with one such expert 193 us, now 136).  A tile is 8 columns (8 gate rows and their 8 up rows) x all k, the k split
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
  constexpr bool kOneGroup = kN == 1;  // at most 8 tokens: every expert has one
  make_plan<kN * 8>(p, s);
  const long long units = (long long)(kOneGroup ? s.active : s.groups[s.active]) * p.width;
  const long long begin = units * blockIdx.x / gridDim.x, end = units * (blockIdx.x + 1) / gridDim.x;
  if (begin >= end) return;
  // expert and column of a place in the list
  auto find = [&](int group) {  // the expert that holds a group
    if constexpr (kOneGroup) return group;
    int lo = 0, hi = s.active;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (s.groups[mid] <= group) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  auto column = [&](long long at, int a) {
    if constexpr (kOneGroup) return (int)(at - (long long)a * p.width);
    return (int)(at - (long long)s.groups[a] * p.width) / (s.groups[a + 1] - s.groups[a]);
  };
  const int a_first = find((int)(begin / p.width)), c_first = column(begin, a_first);
  int a_last = find((int)((end - 1) / p.width)), c_last = column(end, a_last);
  if (c_last == 0 && a_last > a_first) {  // the first column of the last expert is the next block's
    --a_last;
    c_last = p.width;
  }
  if (a_first == a_last && c_first >= c_last) return;
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
    __syncwarp();  // all lanes have read the tile before this one,
    fetch();       // whose place is filled again while this one is used
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
          // weighted here, so that the down products only add up, and rounded
          // to bf16 for them: at most 2^-8 of a value
          uint16_t* h = p.act + (long long)slot * p.width + col;
          if (slot < last) h[0] = f32_to_bf16_rne(s.gate(slot) * (v.x / (1.0f + expf(-v.x)) * v.z));
          if (slot + 1 < last) h[p.width] = f32_to_bf16_rne(s.gate(slot + 1) * (v.y / (1.0f + expf(-v.y)) * v.w));
        }
      }
    }
    const int a = now.a, group = now.group;
    if (!next(now)) break;
    reload = passes > 1 || now.a != a || now.group != group;
  }
  ring.drain(p.status);
}

// ---------------------------------------------------------------------------
// down: a block owns an equal share of the output rows (kRows at a time: 14 of
// the 16 of a product, 2048 rows over 148 blocks, keep the sums of 64 tokens
// in shared memory beside the ring) over all picked experts.  Four warps copy
// tiles in turn, one picked expert after the other: kRows weight rows x 768 k
// and the activations of the expert's tokens (at expert width 768 both are
// contiguous runs).  A warp issues a copy in 30 ns, so one warp alone would
// hold the 15 copies of a tile to 1 us, twice their time on the bus.  The
// eight others work in two teams that take every second tile: a tile's chain of
// lookups, products and sums lasts longer than its bytes (0.74 us against 0.49
// with one team of eight), so two are under way at a time.  A team splits its
// tile's k and each warp keeps its own sums of all tokens, so nothing is joined
// before the end.
//
// kDirect (at most kN * 8 tokens): the columns of a product are the tokens, an
// expert's other columns are zero, and the sums stay in registers over all
// experts.  Otherwise the columns are the tokens that picked the expert and
// are added to sums in shared memory, all of a lane's old values read before
// the first is written.
// ---------------------------------------------------------------------------
constexpr int kRows = 14, kPassChunks = 24, kWeightPitch = kPassChunks * 64 + 64, kActPitch = kPassChunks * 64;
constexpr int kTeams = 2, kTeam = kWarps / kTeams;
constexpr int kMine = kPassChunks / kTeam;  // chunks of a warp in a tile
constexpr int kCopyWarps = 4, kDownThreads = kThreads + 32 * kCopyWarps;
template <int kN>
struct DownShared {
  // Tiles in the ring.  A waiter tells two phases of a barrier apart only by
  // parity, so the same copying warp and the same team have to serve a stage
  // every time: the depth is a multiple of both numbers.
  static constexpr int kDepth = 4;
  static_assert(kDepth % kCopyWarps == 0 && kDepth % kTeams == 0, "every phase of a stage is seen by its waiters");
  struct Tile {
    uint8_t weights[kRows * kWeightPitch];
    uint8_t act[kN * 8 * kActPitch];
  } ring[kDepth];
  uint64_t full[kDepth], free[kDepth];
  Plan plan;
  float sums[1];  // [warp][token][kRows]
};
__device__ __forceinline__ float lds_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

template <int kN, bool kDirect>
__global__ void __launch_bounds__(kDownThreads, 1) token_down_kernel(const __grid_constant__ Layer p) {
  using Shared = DownShared<kN>;
  constexpr int kDepth = Shared::kDepth;
  extern __shared__ __align__(128) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  Plan& s = sh.plan;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  if (threadIdx.x < kDepth) {
    mbar_init(&sh.full[threadIdx.x], 2);  // the weights' bytes and the activations'
    mbar_init(&sh.free[threadIdx.x], kTeam);
    fence_barrier_init();
    fence_proxy_async();
  }
  // the router grid has finished (every gate/up block waited for it before it
  // let this grid start), so the routing and the first weights can be fetched
  // while the gate/up products are still running
  make_plan<kN * 8>(p, s);
  const int chunks = p.width / kChunk, passes = (chunks + kPassChunks - 1) / kPassChunks;
  const int row_begin = (int)((long long)p.hidden * blockIdx.x / gridDim.x);
  const int row_end = (int)((long long)p.hidden * (blockIdx.x + 1) / gridDim.x);

  // tiles in order: 14 rows, expert, group of kN * 8 of its tokens, k pass
  struct Walk {
    int row0, a, first, pass;  // first: slot of the group's first token
  };
  auto next = [&](Walk& w) -> bool {  // false behind the last tile of these rows
    if (++w.pass < passes) return true;
    w.pass = 0;
    w.first += kN * 8;
    if (w.first < s.first[w.a + 1]) return true;
    if (++w.a == s.active) return false;
    w.first = s.first[w.a];
    return true;
  };
  if (warp >= kWarps) {
    bool waited = false;
    auto copy_act = [&](const Walk& w, int at) {
      const int rows = min(kN * 8, s.first[w.a + 1] - w.first), bytes = min(kPassChunks, chunks - w.pass * kPassChunks) * 64;
      uint64_t* full = &sh.full[at % kDepth];
      const uint32_t dst = smem_u32(sh.ring[at % kDepth].act);
      const uint16_t* src = p.act + (long long)w.first * p.width + w.pass * kPassChunks * kChunk;
      if (lane == 0) mbar_arrive_expect_tx(full, rows * bytes);
      __syncwarp();
      if (passes == 1 && bytes == kActPitch) {
        if (lane == 0) bulk_copy(dst, src, rows * bytes, full);
      } else if (lane < rows) {
        bulk_copy(dst + lane * kActPitch, src + (long long)lane * p.width, bytes, full);
      }
    };
    Walk held{}, w{row_begin, 0, 0, 0};
    int held_at = -1, last_at = -1;
    for (int at = 0; w.row0 < row_end; ++at) {
      if (at % kCopyWarps == warp - kWarps) {
        const int stage = at % kDepth, bytes = min(kPassChunks, chunks - w.pass * kPassChunks) * 64;
        const int rows = min(kRows, row_end - w.row0);
        const uint16_t* src = p.w_down + ((long long)s.expert[w.a] * p.hidden + w.row0 + lane) * p.width + w.pass * kPassChunks * kChunk;
        // a second tile of this warp: what the first one left is sent before it can wait for the ring
        if (held_at >= 0) {
          wait_previous();
          waited = true;
          copy_act(held, held_at);
          held_at = -1;
        }
        if (!mbar_wait(&sh.free[stage], ((at / kDepth) & 1) ^ 1u, p.status)) break;
        last_at = at;
        if (lane == 0) mbar_arrive_expect_tx(&sh.full[stage], rows * bytes);
        __syncwarp();
        if (lane < rows) bulk_copy(smem_u32(sh.ring[stage].weights) + lane * kWeightPitch, src, bytes, &sh.full[stage]);
        if (waited) {
          copy_act(w, at);
        } else {
          held = w;
          held_at = at;
        }
      }
      if (!next(w)) w = Walk{w.row0 + kRows, 0, 0, 0};
    }
    if (held_at >= 0) {
      wait_previous();
      copy_act(held, held_at);
    }
    // no copy may land behind the block, whose other warps skip their waits
    // once one has given up; the warp's earlier copies came before this one's
    static_assert(kDepth == kCopyWarps, "a copying warp has one stage");
    if (last_at >= 0) mbar_wait(&sh.full[last_at % kDepth], (last_at / kDepth) & 1, p.status);
    return;
  }

  const int span = p.tokens * kRows;
  float* sums = sh.sums + warp * span;
  const uint32_t mine = smem_u32(sums) + g * 4;
  if constexpr (!kDirect) {
    for (int i = lane; i < span; i += 32) sums[i] = 0.0f;
    __syncwarp();
  }
  wait_previous();  // no grid of the chain ends before the one it follows
  bool bad = false;  // a wait gave up: later ones are not tried again, the results are void
  int at = 0;
  for (int row0 = row_begin; row0 < row_end; row0 += kRows) {
    float total[kN][4] = {};  // kDirect
    Walk w{row0, 0, 0, 0};
    bool more = true;
    for (; more; ++at, more = next(w)) {
      if (at % kTeams != warp / kTeam) continue;
      const int stage = at % kDepth, n_chunks = chunks - w.pass * kPassChunks, first = w.first, last = s.first[w.a + 1];
      // where this lane's column of the activations lies; columns without a
      // token read row 0 and are replaced by zeros
      uint32_t column[kN];
      bool live[kN], any[kN];  // any: some column of the block has a token
      uint32_t to[kN][2];
      float acc[kN][4] = {}, old[kN][4];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if constexpr (kDirect) {
          const uint32_t takers = s.takers[s.expert[w.a]][0];
          live[n] = takers >> (n * 8 + g) & 1u;
          any[n] = takers >> (n * 8) & 255u;
          column[n] = live[n] ? __popc(takers & ((1u << (n * 8 + g)) - 1u)) : 0u;
        } else {
          live[n] = first + n * 8 + g < last;
          any[n] = first + n * 8 < last;
          column[n] = live[n] ? n * 8 + g : 0u;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int slot = first + n * 8 + 2 * t + e;
            to[n][e] = slot < last ? mine + s.token(slot) * (kRows * 4) : 0u;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            old[n][j] = 0.0f;
            if (to[n][j & 1] && (j < 2 || g < kRows - 8)) old[n][j] = lds_f32(to[n][j & 1] + 32 * (j >> 1));
          }
        }
      }
      if (!bad) bad = !mbar_wait(&sh.full[stage], (at / kDepth) & 1, p.status);
      // rows behind the block's last (and 14, 15) are not copied: what lies
      // there enters only sums that are not used
      const uint32_t tile = smem_u32(sh.ring[stage].weights) + g * kWeightPitch + 16 * t + warp % kTeam * 64;
      const uint32_t act = smem_u32(sh.ring[stage].act) + 16 * t + warp % kTeam * 64;
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        if (warp % kTeam + j * kTeam < n_chunks) {
          const uint4 u = lds128(tile + j * kTeam * 64);
          const uint4 v = lds128(tile + (g < kRows - 8 ? 8 * kWeightPitch : 0) + j * kTeam * 64);
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            if (!any[n]) continue;
            uint4 h = lds128(act + column[n] * kActPitch + j * kTeam * 64);
            if (!live[n]) h = make_uint4(0, 0, 0, 0);
            mma_16x8x16(acc[n], u.x, v.x, u.y, v.y, h.x, h.y);
            mma_16x8x16(acc[n], u.z, v.z, u.w, v.w, h.z, h.w);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.free[stage]);
      if constexpr (kDirect) {
        // only tokens of the expert: another's zeros times an infinite weight are no zeros
        const uint32_t takers = s.takers[s.expert[w.a]][0];
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (takers >> (n * 8 + 2 * t + (j & 1)) & 1u) total[n][j] += acc[n][j];
      } else {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (to[n][j & 1] && (j < 2 || g < kRows - 8))
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(to[n][j & 1] + 32 * (j >> 1)), "f"(old[n][j] + acc[n][j]) : "memory");
        __syncwarp();
      }
    }
    if constexpr (kDirect) {
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = n * 8 + 2 * t + (j & 1), r = g + 8 * (j >> 1);
          if (tok < p.tokens && r < kRows) sums[tok * kRows + r] = total[n][j];
        }
    }
    const int rows = min(kRows, row_end - row0);
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    for (int i = threadIdx.x; i < span; i += kThreads) {
      const int tok = i / kRows, r = i % kRows;
      if (r < rows) {
        const long long out = (long long)tok * p.hidden + row0 + r;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) v += sh.sums[k * span + i];
        if (p.residual) v += bf16_to_f32(p.residual[out]);
        p.y[out] = f32_to_bf16_rne(v);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    if constexpr (!kDirect) {
      for (int i = lane; i < span; i += 32) sums[i] = 0.0f;
      __syncwarp();
    }
  }
}

template <int kN>
constexpr size_t down_smem(int tokens) { return sizeof(DownShared<kN>) + sizeof(float) * kWarps * tokens * kRows; }
static_assert(sizeof(GateUpShared<2>) <= 227 * 1024 && down_smem<2>(kTokens) <= 227 * 1024, "shared memory of one block");

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename K>
int32_t launch_after(SharedMemorySetup& setup, int dev, K kernel, int threads, size_t smem, size_t most, const Layer& p,
                     cudaStream_t s) {
  ENNX_TRY(allow_shared_memory(setup, dev, kernel, (int)most));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sm_count());
  cfg.blockDim = dim3((unsigned)threads);
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
template <int kN, bool kDirect>
int32_t launch_experts(const Layer& p, int dev, cudaStream_t s) {
  static SharedMemorySetup setup[2];
  constexpr size_t smem = sizeof(GateUpShared<kN>);
  ENNX_TRY(launch_after(setup[0], dev, token_gate_up_kernel<kN>, kThreads, smem, smem, p, s));
  return launch_after(setup[1], dev, token_down_kernel<kN, kDirect>, kDownThreads, down_smem<kN>(p.tokens),
                      down_smem<kN>(kDirect ? kN * 8 : kTokens), p, s);
}

}  // namespace
}  // namespace ennx

using namespace ennx;

extern "C" {

size_t ennx_b200_moe_layer_decode_workspace_size(int64_t tokens, int32_t experts, int32_t top_k, int32_t expert_width) {
  if (tokens <= 0 || tokens > kTokens || experts <= 0 || top_k <= 0 || expert_width <= 0) return 0;
  return round256((sizeof(float) + 1) * kTokens * kTopK) + round256(sizeof(uint16_t) * tokens * top_k * expert_width);
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
  const int64_t row = (int64_t)hidden * 2, picks = tokens * top_k;
  const Memory read[] = {Memory::bytes(x, tokens * row), Memory::bytes(w_router, experts * row),
                         Memory::bytes(w_gate_up, experts * row * 2 * expert_width),
                         Memory::bytes(w_down, experts * row * expert_width), Memory::bytes(residual, tokens * row)};
  const Memory written[] = {Memory::bytes(y, tokens * row), Memory::bytes(index, picks * 4), Memory::bytes(gate, picks * 4),
                            Memory::bytes(workspace, (int64_t)need)};
  for (const Memory& w : written) {
    for (const Memory& r : read)
      if (share_bytes(w, r) && !(w.base == y && r.base == residual && y == residual))
        return set_error(ENNX_B200_INVALID_ARGUMENT,
                         "moe_layer_decode: outputs and workspace must not overlap x or the weights, nor the residual (y may be it)");
    for (const Memory& other : written)
      if (&w != &other && share_bytes(w, other))
        return set_error(ENNX_B200_INVALID_ARGUMENT, "moe_layer_decode: outputs and workspace must not overlap");
  }
  int dev = 0;
  int* status = nullptr;
  ENNX_TRY(serving_device(&dev, &status));
  float* gates = (float*)workspace;
  const Layer p{x, w_router, w_gate_up, w_down, residual, y, index, gate, (uint8_t*)(gates + kTokens * kTopK), gates,
                (uint16_t*)((uint8_t*)workspace + round256((sizeof(float) + 1) * kTokens * kTopK)),
                (int)tokens, hidden, experts, top_k, expert_width, status};
  if (tokens == 1) token_router_kernel<1><<<kCluster, kThreads, 0, s>>>(p);
  else token_router_kernel<8><<<(unsigned)(kCluster * ((tokens + 7) / 8)), kThreads, 0, s>>>(p);
  ENNX_LAUNCH_CHECK("few-token router");
  if (tokens <= 8) return launch_experts<1, true>(p, dev, s);
  return tokens <= 16 ? launch_experts<2, true>(p, dev, s) : launch_experts<2, false>(p, dev, s);
}

}  // extern "C"

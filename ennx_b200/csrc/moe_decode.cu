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
// 8 columns; each warp streams its own weight tiles through a cp.async ring
// (two 8 KB tiles in flight per warp, 128 KB per SM).  k is permuted the same
// way in both operands so that a lane's fragments are 16 contiguous bytes.
#include "kernels.cuh"
#include "serve.cuh"

#include <math.h>

namespace ennx {
namespace {

constexpr int kTokens = 64, kTopK = 8, kExperts = 256;
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kChunk = 32;               // k of one 64-byte piece per row: two mma steps
constexpr int kTileChunks = 8;           // chunks of a warp's tile
constexpr int kPitch = kTileChunks * 64;  // bytes of a tile row
constexpr int kTileBytes = 16 * kPitch;
constexpr int kStages = 3;
constexpr int kRing = kWarps * kStages * kTileBytes;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Layer {
  const uint16_t *x, *w_router, *w_gate_up, *w_down, *residual;
  uint16_t* y;
  int* index;     // nullable
  float* gate;    // nullable
  float* logits;  // [tokens][experts]
  uint16_t* act;  // [tokens * top_k][width], rows expert by expert
  int tokens, hidden, experts, top_k, width;
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

// piece (16 bytes) c of row r of a ring tile: rows 512 bytes apart would put
// the two rows of a quarter-warp on the same banks, so odd rows swap halves
__device__ __forceinline__ uint32_t piece(int r, int c) { return (uint32_t)(r * kPitch + ((c ^ ((r & 1) << 2)) << 4)); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// ---------------------------------------------------------------------------
// gate/up: a block takes an equal run of the (picked expert, column) list.  A
// tile is 8 columns (8 gate rows and their 8 up rows) x all k, the k split
// over the warps; kN blocks of 8 tokens at a time stay in registers.
// ---------------------------------------------------------------------------
template <int kN>
__global__ void __launch_bounds__(kThreads, 1) token_gate_up_kernel(const __grid_constant__ Layer p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  float4* red = reinterpret_cast<float4*>(smem + kRing);  // [2][warp][kN][lane]
  Plan& s = *reinterpret_cast<Plan*>(smem + kRing + 2 * kWarps * kN * 32 * sizeof(float4));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * kStages * kTileBytes;
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
  const int chunks = p.hidden / kChunk, passes = (chunks + kWarps * kTileChunks - 1) / (kWarps * kTileChunks);
  const int per = ((chunks + passes - 1) / passes + kWarps - 1) / kWarps;  // chunks of a warp in a pass

  // tiles in order: expert, group of kN * 8 tokens, 8 columns, k pass
  struct Tile {
    int a, c, pass, group;  // c: column within the expert
  };
  auto last_column = [&](int a) { return (int)min((long long)p.width, end - (long long)a * p.width); };
  auto first_column = [&](int a) { return (int)max(0LL, begin - (long long)a * p.width); };
  auto next = [&](Tile& w) -> bool {  // false behind the last tile
    if (++w.pass < passes) return true;
    w.pass = 0;
    w.c += 8;
    if (w.c < last_column(w.a)) return true;
    w.c = first_column(w.a);
    if (++w.group * kN * 8 < s.first[w.a + 1] - s.first[w.a]) return true;
    w.group = 0;
    ++w.a;
    w.c = 0;
    return (long long)w.a * p.width < end;
  };
  auto chunk0 = [&](int pass) { return (pass * kWarps + warp) * per; };

  Tile ahead{(int)(begin / p.width), (int)(begin % p.width), 0, 0}, now = ahead;
  bool more = true;
  int fetched = 0;
  auto fetch = [&] {
    if (more) {
      const uint16_t* w = p.w_gate_up + (long long)s.expert[ahead.a] * 2 * p.width * p.hidden;
      const uint32_t dst = ring + (fetched % kStages) * kTileBytes;
      const int c_end = last_column(ahead.a), k0 = chunk0(ahead.pass);
      const bool k_ok = (lane >> 2) < per && k0 + (lane >> 2) < chunks;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int col = ahead.c + (r & 7), row = (col >> 7) * 256 + (r >> 3) * 128 + (col & 127);
        const bool ok = k_ok && col < c_end;
        cp_async16(dst + piece(r, lane), w + (ok ? (long long)row * p.hidden + k0 * kChunk + lane * 8 : 0), ok);
      }
      more = next(ahead);
    }
    ++fetched;
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  uint4 xf[kTileChunks][kN];
  int have_a = -1, have_group = -1, have_pass = -1;
  float acc[kN][4];
  for (int i = 0, done = 0;; ++i) {
    if (now.a != have_a || now.group != have_group || now.pass != have_pass) {
      have_a = now.a; have_group = now.group; have_pass = now.pass;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int slot = s.first[now.a] + (now.group * kN + n) * 8 + g;
        const bool ok = slot < s.first[now.a + 1];
        const uint16_t* x = p.x + (ok ? (long long)s.token(slot) * p.hidden : 0) + chunk0(now.pass) * kChunk + t * 8;
#pragma unroll
        for (int j = 0; j < kTileChunks; ++j)
          xf[j][n] = ok && j < per && chunk0(now.pass) + j < chunks ? __ldg(reinterpret_cast<const uint4*>(x + j * kChunk))
                                                                 : make_uint4(0, 0, 0, 0);
      }
    }
    if (now.pass == 0) {
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][j] = 0.0f;
    }
    cp_wait<kStages - 2>();
    __syncwarp();
    const uint32_t tile = ring + (i % kStages) * kTileBytes;
#pragma unroll
    for (int j = 0; j < kTileChunks; ++j) {
      if (j < per) {
        const uint4 a = lds128(tile + piece(g, 4 * j + t)), b = lds128(tile + piece(g + 8, 4 * j + t));
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          mma(acc[n], a.x, b.x, a.y, b.y, xf[j][n].x, xf[j][n].y);
          mma(acc[n], a.z, b.z, a.w, b.w, xf[j][n].z, xf[j][n].w);
        }
      }
    }
    __syncwarp();
    fetch();
    if (now.pass == passes - 1) {
      float4* buf = red + (done & 1) * kWarps * kN * 32;
      ++done;
#pragma unroll
      for (int n = 0; n < kN; ++n)
        buf[(warp * kN + n) * 32 + lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
      // one barrier a tile: the other buffer is written again only after the
      // next barrier, which every reader of this one reaches first
      __syncthreads();
      if (warp < kN) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 u = buf[(w * kN + warp) * 32 + lane];
          v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
        }
        const int col = now.c + g, slot = s.first[now.a] + (now.group * kN + warp) * 8 + 2 * t;
        if (col < last_column(now.a)) {
          // rounded to bf16 for the second product: at most 2^-8 of a value
          uint16_t* h = p.act + (long long)slot * p.width + col;
          if (slot < s.first[now.a + 1]) h[0] = f32_to_bf16_rne(v.x / (1.0f + expf(-v.x)) * v.z);
          if (slot + 1 < s.first[now.a + 1]) h[p.width] = f32_to_bf16_rne(v.y / (1.0f + expf(-v.y)) * v.w);
        }
      }
    }
    if (!next(now)) break;
  }
  cp_wait<0>();
}

// ---------------------------------------------------------------------------
// down: a block owns an equal share of the output rows (kRows at a time: 14 of
// the 16 of a product, 2048 rows over 148 blocks, keep the sums of 64 tokens
// in shared memory beside the ring) over all picked experts; experts go round
// the warps, a warp's tile is kRows rows x 256 k.
// ---------------------------------------------------------------------------
constexpr int kRows = 14;
template <int kN>
__global__ void __launch_bounds__(kThreads, 1) token_down_kernel(const __grid_constant__ Layer p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  float* sums = reinterpret_cast<float*>(smem + kRing);  // [warp][token][kRows]
  const int span = p.tokens * kRows;
  Plan& s = *reinterpret_cast<Plan*>(smem + kRing + sizeof(float) * kWarps * span);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * kStages * kTileBytes;
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
    struct Tile {
      int a, group, pass;
    };
    auto next = [&](Tile& w) -> bool {
      if (++w.pass < passes) return true;
      w.pass = 0;
      if (++w.group * kN * 8 < s.first[w.a + 1] - s.first[w.a]) return true;
      w.group = 0;
      w.a += kWarps;
      return w.a < s.active;
    };
    Tile ahead{warp, 0, 0}, now = ahead;
    bool more = warp < s.active;
    int fetched = 0;
    auto fetch = [&] {
      if (more) {
        const uint16_t* w = p.w_down + ((long long)s.expert[ahead.a] * p.hidden + row0) * p.width;
        const uint32_t dst = ring + (fetched % kStages) * kTileBytes;
        const int k0 = ahead.pass * kTileChunks;
        const bool k_ok = k0 + (lane >> 2) < chunks;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool ok = k_ok && r < rows;
          cp_async16(dst + piece(r, lane), w + (ok ? (long long)r * p.width + k0 * kChunk + lane * 8 : 0), ok);
        }
        more = next(ahead);
      }
      ++fetched;
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch();
    for (int i = lane; i < span; i += 32) sums[warp * span + i] = 0.0f;
    if (!waited) {
      wait_previous();  // the activations are complete and visible
      waited = true;
    }
    __syncwarp();
    float acc[kN][4];
    for (int i = 0; warp < s.active; ++i) {
      const int first = s.first[now.a] + now.group * kN * 8, last = s.first[now.a + 1];
      uint4 hf[kTileChunks][kN];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const bool ok = first + n * 8 + g < last;
        const uint16_t* h = p.act + (ok ? (long long)(first + n * 8 + g) * p.width : 0) + now.pass * kTileChunks * kChunk + t * 8;
#pragma unroll
        for (int j = 0; j < kTileChunks; ++j)
          hf[j][n] = ok && now.pass * kTileChunks + j < chunks ? __ldcg(reinterpret_cast<const uint4*>(h + j * kChunk))
                                                                : make_uint4(0, 0, 0, 0);
      }
      if (now.pass == 0) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[n][j] = 0.0f;
      }
      cp_wait<kStages - 2>();
      __syncwarp();
      const uint32_t tile = ring + (i % kStages) * kTileBytes;
#pragma unroll
      for (int j = 0; j < kTileChunks; ++j) {
        const uint4 a = lds128(tile + piece(g, 4 * j + t)), b = lds128(tile + piece(g + 8, 4 * j + t));
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          mma(acc[n], a.x, b.x, a.y, b.y, hf[j][n].x, hf[j][n].y);
          mma(acc[n], a.z, b.z, a.w, b.w, hf[j][n].z, hf[j][n].w);
        }
      }
      __syncwarp();
      fetch();
      if (now.pass == passes - 1) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int slot = first + n * 8 + 2 * t + (j & 1), row = g + 8 * (j >> 1);
            if (slot < last && row < kRows) sums[warp * span + s.token(slot) * kRows + row] += s.gate(slot) * acc[n][j];
          }
        __syncwarp();
      }
      if (!next(now)) break;
    }
    cp_wait<0>();
    __syncthreads();
    for (int i = threadIdx.x; i < span; i += kThreads) {
      const int tok = i / kRows, r = i % kRows;
      if (r < rows) {
        const long long at = (long long)tok * p.hidden + row0 + r;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += sums[w * span + i];
        if (p.residual) v += bf16_to_f32(p.residual[at]);
        p.y[at] = f32_to_bf16_rne(v);
      }
    }
    __syncthreads();
  }
  if (!waited) wait_previous();  // no grid of the chain ends before the one it follows
}

template <int kN>
constexpr size_t gate_up_smem() { return kRing + 2 * kWarps * kN * 32 * sizeof(float4) + sizeof(Plan); }
constexpr size_t down_smem(int tokens) { return kRing + sizeof(float) * kWarps * tokens * kRows + sizeof(Plan); }
static_assert(gate_up_smem<2>() <= 227 * 1024, "gate/up shared memory");
static_assert(down_smem(kTokens) <= 227 * 1024, "down shared memory");

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename K>
int32_t launch_after(K kernel, int grid, size_t smem, const Layer& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
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
  Layer p{x, w_router, w_gate_up, w_down, residual, y, index, gate, (float*)workspace,
          (uint16_t*)((uint8_t*)workspace + round256(sizeof(float) * tokens * experts)),
          (int)tokens, hidden, experts, top_k, expert_width};
  static bool attr[64];
  int dev = 0;
  ENNX_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= 64) return set_error(ENNX_B200_UNSUPPORTED, "device index %d out of range", dev);
  if (!attr[dev]) {
    const auto most = cudaFuncAttributeMaxDynamicSharedMemorySize;
    ENNX_CUDA(cudaFuncSetAttribute(token_gate_up_kernel<1>, most, (int)gate_up_smem<1>()), "few-token moe smem");
    ENNX_CUDA(cudaFuncSetAttribute(token_gate_up_kernel<2>, most, (int)gate_up_smem<2>()), "few-token moe smem");
    ENNX_CUDA(cudaFuncSetAttribute(token_down_kernel<1>, most, (int)down_smem(kTokens)), "few-token moe smem");
    ENNX_CUDA(cudaFuncSetAttribute(token_down_kernel<2>, most, (int)down_smem(kTokens)), "few-token moe smem");
    attr[dev] = true;
  }
  const dim3 router((unsigned)((experts + kRE - 1) / kRE), (unsigned)((tokens + kRT - 1) / kRT));
  token_router_kernel<<<router, kThreads, 0, s>>>(p);
  ENNX_LAUNCH_CHECK("few-token router");
  const int grid = sm_count();
  if (tokens <= 8) {
    ENNX_TRY(launch_after(token_gate_up_kernel<1>, grid, gate_up_smem<1>(), p, s));
    return launch_after(token_down_kernel<1>, grid, down_smem((int)tokens), p, s);
  }
  ENNX_TRY(launch_after(token_gate_up_kernel<2>, grid, gate_up_smem<2>(), p, s));
  return launch_after(token_down_kernel<2>, grid, down_smem((int)tokens), p, s);
}

}  // extern "C"

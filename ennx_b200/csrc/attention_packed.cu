// attention_packed.cu -- causal grouped-query attention over packed prompts of
// different lengths, on tcgen05 tensor cores.
//
// Sequence s of the packed rows is [cu[s], cu[s+1]); with lo(i) the first row
// of row i's sequence and kv = h / (Hq / Hkv),
//   o[i, h] = sum_{lo(i) <= j <= i} softmax_j(q[i, h] . k[j, kv] / sqrt(128)) v[j, kv].
//
// Bound: the tensor cores and, next to them, one exp2 per score.  Query tiles
// are 128 consecutive PACKED rows whatever sequences they belong to, so a
// sequence boundary costs no tile of its own: a tile reads the key tiles from
// lo(its first row) to its own diagonal and every row masks the keys outside
// [lo(i), i].  With a tile per sequence instead, prompts shorter than 128
// tokens would each occupy a whole tile.
//
// One CTA = two 128-row query tiles (A: rows q0..q0+127, B: q0+128..q0+255)
// of one query head, key/value tiles of 128 keys on the same 128-row grid,
// shared by both.  Tensor memory: S_A | O_A | S_B | O_B, 128 fp32 columns
// each.  Warp roles: 0 TMA producer (two slots of K and of V); 1 one
// thread issues tcgen05.mma (S = Q K^T; O += P V with P from tensor memory);
// 4..11 softmax, four warps per query tile, a thread per row, statistics in
// fp32, P rounded to bf16 (at most 2^-8 relative, random in sign, below the
// rounding of the bf16 output).
//
// A key tile costs each query tile 1024 clocks of tensor work and, at 16 exp2 a
// clock, 1024 clocks of the exponential unit; one query tile's products run
// under the other's softmax.  What bounds the loop is the chain of one query
// tile, S -> softmax (2100 clocks) -> O += P V -> next S, 3700 clocks of which
// 2048 are the two tiles' products.  P is handed over in two halves so that its
// product starts under the second half, and no two threads share a row (two
// per row and an exchange of maxima under a barrier: 16384 tokens 1.19 ms for
// 1.04 then).  S in halves of 64 keys, one ahead of the other, breaks the
// chain, but a 128 x 64 x 16 product lasts 48 clocks instead of 32 and both
// softmaxes then compete for issue slots: 0.92 ms for 0.87.  A part of the
// exponentials as a polynomial on the FMA units changed nothing.
//
// A block takes over the next item of the grid that has not started
// (clusterlaunchcontrol), as late as its last key tile: barriers and tensor
// memory are set up once and the next Q and K arrive while the last softmax
// runs (ragged 16384 tokens 210 -> 203 us).
//
// Measured in a stream of calls: one prompt of 16384 tokens, 16 heads on 4: 0.99
// ms, 1110 TFLOP/s at the power limit (0.87 ms in single calls after a pause); 12
// ragged prompts of 16384 tokens 221 us, 765 TFLOP/s of visible scores.
//
// Masked places may hold anything: masked scores are replaced, not added to,
// but a masked V row still meets P = 0 in the MMA and an infinity or NaN there
// makes 0 * inf = NaN.  Rows behind the last sequence are cleared in shared
// memory; a non-finite output whose scores are numbers, and which no visible
// value explains, is recomputed by `careful_row`, which reads visible keys only.
// That is slow, 0.15 us a key and row with 32 rows one after the other (16384
// tokens whose last value is infinite 77 ms), but falls to the rows of the tiles
// that hold a bad value only.
#include "kernels.cuh"
#include "serve.cuh"

#include <math.h>

namespace ennx {

namespace {

constexpr int D = 128, BQ = 128, BKV = 128;
constexpr int SUB = 128 * 128;  // bytes of one 128-row x 64-column bf16 sub-tile
constexpr int TILE = 2 * SUB;   // 128 rows x 128 columns
// three groups of four warps: producer and MMA (two warps idle), softmax of
// tile A, softmax of tile B; the first gives registers to the others, whose
// threads hold 128 scores (56 + 2 * 224 = 3 * 168, what the block starts with)
constexpr int SOFTMAX_WARPS = 8;
constexpr int FEW_REGS = 56, MANY_REGS = 224;
constexpr int THREADS = 128 + 32 * SOFTMAX_WARPS;
static_assert(FEW_REGS + 2 * MANY_REGS <= 3 * 168 && THREADS == 384, "registers of the block");
constexpr int BARS = 320;
constexpr int SMEM = 6 * TILE /*Q_A, Q_B, 2 K, 2 V*/ + 1024 + BARS;
constexpr uint32_t IDESC_QK = idesc_bf16_f32(128, 128);
constexpr uint32_t IDESC_PV = idesc_bf16_f32(128, 128) | (1u << 16);  // B (V) MN-major
constexpr float kRescaleThreshold = 8.0f;  // log2 units: rescale O only when the max grows by > 2^8

// D[tmem] (+)= A[tmem] * B[smem desc]^T, kind::f16
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ bool elect_one() {  // one lane of the (converged) warp
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// Takes over a block of this grid that has not started: the answer, 16 bytes,
// completes on `bar`.  After an answer of "none" it must not be asked again.
__device__ __forceinline__ void request_block(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ int answered_block(const uint4* answer) {  // its blockIdx.x, -1: none
  int x;
  asm volatile(
      "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 a, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, a;\n\t}"
      : "=r"(x) : "r"(smem_u32(answer)) : "memory");
  return x;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float low(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
// Packed rows: [begin, end) belong to sequences, clamped to the rows there are.
struct Packing {
  const int* cu;
  int nseq, rows;
  __device__ __forceinline__ int begin() const { return max(0, __ldg(cu)); }
  __device__ __forceinline__ int end() const { return min(rows, __ldg(cu + nseq)); }
  // first row of row r's sequence, r itself for a row of no sequence; in
  // [0, r] whatever cu holds, so every index made from it stays in bounds
  __device__ __forceinline__ int first_row(int r) const {
    if (r >= end() || __ldg(cu) > r) return r;
    int lo = 0, hi = nseq;  // last s with cu[s] <= r (empty sequences before it skipped)
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (__ldg(cu + mid) <= r) lo = mid;
      else hi = mid;
    }
    return min(r, max(0, __ldg(cu + lo)));
  }
};

struct Operands {
  const uint16_t *q, *k, *v;
  uint16_t* o;
  long long ldq, ldk, ldv, ldo;
};

// A work item: the grid index whose head and rows it takes, -1 behind the
// last, and the first rows of the sequences that hold its tiles' first rows.
struct Item {
  int index, first[2];
};
struct Bars {
  uint4 next;  // what the request for another item answered
  uint64_t next_full, item_full[2], item_free[2];
  uint64_t q_full, q_free, k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2][2] /*[tile][half of the keys]*/, o_done[2];
  Item item[2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Bars) <= BARS, "the barriers fit their place");

// Output of one (row, head), by one warp, reading visible keys only; every sum
// in fp32.  Keys come four at a time, their loads together.
__device__ __noinline__ void careful_row(const Operands& t, int row, int lo, int h, int kvh, float scale_log2, int lane) {
  constexpr int kKeys = 4;
  auto two = [](uint32_t w, float& a, float& b) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  };
  const uint2 qw = *reinterpret_cast<const uint2*>(t.q + (long long)row * t.ldq + h * D + lane * 4);
  float q[4], m = -INFINITY, l = 0.0f, a[4] = {};
  two(qw.x, q[0], q[1]);
  two(qw.y, q[2], q[3]);
  for (int j0 = lo; j0 <= row; j0 += kKeys) {
    uint2 kw[kKeys], vw[kKeys];
#pragma unroll
    for (int u = 0; u < kKeys; ++u) {
      const long long j = min(j0 + u, row);  // those behind the row are left out below
      kw[u] = *reinterpret_cast<const uint2*>(t.k + j * t.ldk + kvh * D + lane * 4);
      vw[u] = *reinterpret_cast<const uint2*>(t.v + j * t.ldv + kvh * D + lane * 4);
    }
    float s[kKeys], v[kKeys][4], mn = m, more = 0.0f;
#pragma unroll
    for (int u = 0; u < kKeys; ++u) {
      float k[4];
      two(kw[u].x, k[0], k[1]);
      two(kw[u].y, k[2], k[3]);
      two(vw[u].x, v[u][0], v[u][1]);
      two(vw[u].y, v[u][2], v[u][3]);
      s[u] = fmaf(q[3], k[3], fmaf(q[2], k[2], fmaf(q[1], k[1], q[0] * k[0])));
    }
#pragma unroll
    for (int off = 16; off; off >>= 1)
#pragma unroll
      for (int u = 0; u < kKeys; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], off);
#pragma unroll
    for (int u = 0; u < kKeys; ++u) {
      s[u] = j0 + u <= row ? s[u] * scale_log2 : -INFINITY;
      mn = fmaxf(mn, s[u]);
    }
    const float ref = mn == -INFINITY ? 0.0f : mn, alpha = ex2(m - ref);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] *= alpha;
#pragma unroll
    for (int u = 0; u < kKeys; ++u)
      if (j0 + u <= row) {
        const float p = ex2(s[u] - ref);
        more += p;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = fmaf(p, v[u][i], a[i]);
      }
    l = l * alpha + more;
    m = mn;
  }
  const float inv = 1.0f / l;  // every visible score -inf: 0 / 0
  *reinterpret_cast<uint2*>(t.o + (long long)row * t.ldo + h * D + lane * 4) =
      make_uint2(pack_bf16x2(a[0] * inv, a[1] * inv), pack_bf16x2(a[2] * inv, a[3] * inv));
}

// A set of the columns of a head, a bit each.
struct Columns {
  uint32_t w[4];
  __device__ __forceinline__ void add(const Columns& o, bool where) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] |= where ? o.w[i] : 0u;
  }
};
// the set that byte b of a lane of 16, columns 8 * lane .. 8 * lane + 7, makes with the 15 beside it
__device__ __forceinline__ Columns columns_of(uint32_t b, int first_lane) {
  Columns c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c.w[i] = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) c.w[i] |= __shfl_sync(0xffffffffu, b, first_lane + 4 * i + j) << (8 * j);
  }
  return c;
}

// Do outputs `bad` of a lane's row, whose scores are numbers, have to be
// recomputed?  The warp reads the values of keys [from, to), which its tiles
// covered, once for its 32 rows; the row sees those in [lo, row].  A visible NaN
// makes its column NaN and a visible infinity makes it what it is; a masked one
// (which met a weight of 0) makes it NaN wrongly.  A column without either is
// recomputed too: its sum passed the range of fp32.  (Without this look every
// row that saw an infinity for real was recomputed: 16384 tokens of 16 heads
// behind one of them 278 ms, now 3.2.)
__device__ __forceinline__ bool has_to_be_redone(const Operands& t, Columns bad, int row, int lo, int from, int to, int kvh,
                                              int lane) {
  constexpr int kLoads = 8, kKeys = 2 * kLoads;  // two keys a load, 16 lanes each
  Columns seen{}, seen_nan{}, masked{};
  const uint16_t* v = t.v + kvh * D + (lane & 15) * 8;
  for (int j0 = from; j0 < to; j0 += kKeys) {
    uint4 x[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const long long j = min(j0 + 2 * u + (lane >> 4), to - 1);
      x[u] = *reinterpret_cast<const uint4*>(v + j * t.ldv);
    }
    uint32_t any = 0u;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) any |= __vcmpeq2(w[i] & 0x7f807f80u, 0x7f807f80u);
    }
    if (!__any_sync(0xffffffffu, any != 0u)) continue;
#pragma unroll 1
    for (int u = 0; u < kLoads; ++u) {
      const long long j = min(j0 + 2 * u + (lane >> 4), to - 1);
      const uint4 y = *reinterpret_cast<const uint4*>(v + j * t.ldv);
      const uint32_t w[4] = {y.x, y.y, y.z, y.w};
      uint32_t wild = 0u, nan = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t b = w[i] >> (16 * e) & 0x7fffu;
          wild |= (b >= 0x7f80u ? 1u : 0u) << (2 * i + e);
          nan |= (b > 0x7f80u ? 1u : 0u) << (2 * i + e);
        }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int key = min(j0 + 2 * u + half, to - 1);
        const bool visible = key >= lo && key <= row;
        const Columns cw = columns_of(wild, 16 * half), cn = columns_of(nan, 16 * half);
        seen.add(cw, visible);
        seen_nan.add(cn, visible);
        masked.add(cw, !visible);
      }
    }
  }
  uint32_t redo = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) redo |= bad.w[i] & ~seen_nan.w[i] & (masked.w[i] | ~seen.w[i]);
  return redo != 0u;
}

// A warp's rows whose outputs are not finite although their scores are numbers
// (`wild`); those outputs stand in global memory and, times 1 / inv, at o_col.
__device__ __noinline__ void repair_rows(const Operands& t, uint32_t o_col, float inv, bool wild, int row, int lo, int from,
                                         int to, int h, int kvh, float scale_log2) {
  const int lane = threadIdx.x & 31;
  Columns bad;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t ov[32];
    tmem_ld32(o_col + c * 32, ov);
    tmem_ld_wait();
    bad.w[c] = 0u;
#pragma unroll
    for (int i = 0; i < 32; ++i) bad.w[c] |= (isfinite(__uint_as_float(ov[i]) * inv) ? 0u : 1u) << i;
  }
  const bool again = has_to_be_redone(t, bad, row, lo, from, to, kvh, lane);
  uint32_t redo = __ballot_sync(0xffffffffu, wild && again);
  __syncwarp();  // the rows' first outputs are written
  while (redo) {
    const int src = __ffs(redo) - 1;
    redo &= redo - 1;
    careful_row(t, __shfl_sync(0xffffffffu, row, src), __shfl_sync(0xffffffffu, lo, src), h, kvh, scale_log2, lane);
  }
}

// All roles wait while rows are recomputed, 5.6 us per key of a sequence for
// the 32 rows of a warp (131072 keys 0.74 s).  So waits are bounded by the usual
// limit and nearly four times that for the longest sequence there can be.
unsigned long long wait_limit_ns(int64_t rows) { return kWaitLimitNs + 20000ull * (unsigned long long)rows; }

struct True { static constexpr bool value = true; };
struct False { static constexpr bool value = false; };

__global__ void __launch_bounds__(THREADS, 1)
    prompt_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Operands t, Packing pk,
                            int heads, int group, float scale_log2, unsigned long long limit_ns, int* err) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* base = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sQ = base;           // [2] tiles
  uint8_t* sK = sQ + 2 * TILE;  // [2] ring slots
  uint8_t* sV = sK + 2 * TILE;  // [2] ring slots
  Bars& bar = *reinterpret_cast<Bars*>(sV + 2 * TILE);

  // Later rows first, all heads of a block of rows next to one another: the
  // last items to start are then the packing's first rows, which see few keys
  // whatever the lengths are (with heads outside items of any cost
  // start last: ragged 16384 tokens 254 us, so 210), and the heads that
  // share a cache head share its tiles in L2.
  const int items = (int)gridDim.x;
  auto row_of = [&](int index) { return (items - 1 - index) / heads * (2 * BQ); };
  auto head_of = [&](int index) { return (items - 1 - index) % heads; };
  const int end = pk.end();
  if (row_of((int)blockIdx.x) >= end) {  // block-uniform: rows behind the last sequence stay as they are
    wait_previous();
    return;
  }
  // from lane 0, so that the compiler knows it to be the same in a warp
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  auto load_q = [&](int index) {
    const int q0 = row_of(index), h = head_of(index), nq = q0 + BQ < end ? 2 : 1;
    mbar_arrive_expect_tx(&bar.q_full, nq * TILE);
    for (int x = 0; x < nq; ++x) {
      tma_load_2d(sQ + x * TILE, &tmQ, &bar.q_full, h * D, q0 + x * BQ);
      tma_load_2d(sQ + x * TILE + SUB, &tmQ, &bar.q_full, h * D + 64, q0 + x * BQ);
    }
  };

  if (threadIdx.x == 0) {
    mbar_init(&bar.next_full, 1);
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.q_free, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.item_full[i], 1);
      mbar_init(&bar.item_free[i], 1 + SOFTMAX_WARPS);
      mbar_init(&bar.k_full[i], 1);
      mbar_init(&bar.k_free[i], 1);
      mbar_init(&bar.v_full[i], 1);
      mbar_init(&bar.v_free[i], 1);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_full[i][0], 4);
      mbar_init(&bar.p_full[i][1], 4);
      mbar_init(&bar.o_done[i], 1);
    }
    bar.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
    wait_previous();
    load_q((int)blockIdx.x);
  }
  if (warp == 1) { tmem_alloc(&bar.tmem_base, 512); tmem_relinquish(); }
  if (threadIdx.x >= 64 && threadIdx.x < 66) {
    const int x = (int)threadIdx.x - 64;
    bar.item[0].first[x] = pk.first_row(row_of((int)blockIdx.x) + x * BQ);
    bar.item[0].index = (int)blockIdx.x;
  }
  wait_previous();  // q and k are rotated; what stands above reads neither
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem_base;  // S_A: 0, O_A: 128, S_B: 256, O_B: 384
  volatile int* abort_flag = &bar.abort_flag;
  // key tiles on the 128-row grid, numbered from the one that holds A's first
  // key: tile x uses [js[x], je[x]), its diagonal tile last; B may be empty
  struct Tiles {
    int q0, h, kt0, js[2], je[2], nt;
  };
  auto tiles_of = [&](const Item& it) {
    Tiles w;
    w.q0 = row_of(it.index);
    w.h = head_of(it.index);
    w.kt0 = it.first[0] / BKV;
    const bool two = w.q0 + BQ < end;
    w.js[0] = 0;
    w.js[1] = two ? max(0, it.first[1] / BKV - w.kt0) : 0;
    w.je[0] = w.q0 < end ? w.q0 / BKV + 1 - w.kt0 : 0;
    w.je[1] = two ? w.q0 / BKV + 2 - w.kt0 : 0;
    w.nt = two ? w.je[1] : w.je[0];
    return w;
  };
  auto wait = [&](uint64_t* b, uint32_t parity) {
    return mbar_wait(b, parity, err, limit_ns);
  };
  // by a whole warp, the same answer in every lane
  auto warp_wait = [&](uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, wait(b, parity)) != 0; };
  // the n-th item of this block, by a whole warp; index -1: no more
  auto take_item = [&](int n) {
    Item it{-1, {0, 0}};
    if (__any_sync(0xffffffffu, *abort_flag) || !warp_wait(&bar.item_full[n & 1], (n >> 1) & 1)) return it;
    it = bar.item[n & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar.item_free[n & 1]);
    it.index = __shfl_sync(0xffffffffu, it.index, 0);  // (see `warp`)
    it.first[0] = __shfl_sync(0xffffffffu, it.first[0], 0);
    it.first[1] = __shfl_sync(0xffffffffu, it.first[1], 0);
    return it;
  };

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW_REGS));
  if (warp == 0) {
    if (lane == 0) {
      int tiles = 0, k_tiles = 0, loads = 1, asked = 0;  // V and K tiles, Q loads and requests so far
      bool ok = true;
      Item it = bar.item[0];
      mbar_arrive(&bar.item_full[0]);
      for (int n = 0;; ++n) {
        const Tiles w = tiles_of(it);
        const int kvh = w.h / group;
        auto ask = [&] {
          fence_proxy_async();  // the answer before has been read
          mbar_arrive_expect_tx(&bar.next_full, sizeof(uint4));
          request_block(&bar.next, &bar.next_full);
          ++asked;
        };
        if (n > 0 && w.nt > 0) {
          ok = wait(&bar.q_free, (loads & 1) ^ 1);
          if (!ok) break;
          load_q(it.index);
          ++loads;
        }
        for (int j = 0; j < w.nt; ++j, ++tiles) {
          // late, so that blocks with little left take what is left
          if (j == w.nt - 1) ask();
          const int s = tiles & 1;
          const int krow = (w.kt0 + j) * BKV;
          const uint32_t empty = ((tiles >> 1) & 1) ^ 1u;
          uint8_t* k = sK + s * TILE;
          uint8_t* v = sV + s * TILE;
          ok = !*abort_flag && wait(&bar.k_free[s], empty);
          if (!ok) break;
          mbar_arrive_expect_tx(&bar.k_full[s], TILE);
          tma_load_2d(k, &tmK, &bar.k_full[s], kvh * D, krow);
          tma_load_2d(k + SUB, &tmK, &bar.k_full[s], kvh * D + 64, krow);
          ++k_tiles;
          ok = wait(&bar.v_free[s], empty);
          if (!ok) break;
          mbar_arrive_expect_tx(&bar.v_full[s], TILE);
          tma_load_2d(v, &tmV, &bar.v_full[s], kvh * D, krow);
          tma_load_2d(v + SUB, &tmV, &bar.v_full[s], kvh * D + 64, krow);
        }
        if (!ok) break;
        if (w.nt == 0) ask();
        ok = wait(&bar.next_full, n & 1);
        if (!ok) break;
        it.index = answered_block(&bar.next);
        if (it.index >= 0)
          for (int x = 0; x < 2; ++x) it.first[x] = pk.first_row(row_of(it.index) + x * BQ);
        const int m = n + 1;
        ok = wait(&bar.item_free[m & 1], ((m >> 1) & 1) ^ 1);
        if (!ok) break;
        bar.item[m & 1] = it;
        mbar_arrive(&bar.item_full[m & 1]);
        if (it.index < 0) break;
      }
      if (!ok) {  // giving up: no copy may land after the block has gone
        *abort_flag = 1;
        wait(&bar.q_full, (loads - 1) & 1);
        for (int i = max(0, k_tiles - 2); i < k_tiles; ++i) wait(&bar.k_full[i & 1], (i >> 1) & 1);
        for (int i = max(0, tiles - 2); i < tiles; ++i) wait(&bar.v_full[i & 1], (i >> 1) & 1);
        if (asked > 0) wait(&bar.next_full, (asked - 1) & 1);
      }
    }
  } else if (warp == 1) {
    // The whole warp runs the loop, one elected lane issues: descriptors then
    // stay in uniform registers.
    const bool elected = elect_one();
    const uint64_t qd = smem_desc_sw128(smem_u32(sQ));
    const uint64_t kd = smem_desc_sw128(smem_u32(sK)), vd = smem_desc_sw128_mn(smem_u32(sV), SUB);
    int tiles = 0, loads = 0, p_seen[2] = {0, 0}, k_seen = 0;  // key tiles, items and P tiles so far; K waited for
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const Item it = take_item(n);
      if (it.index < 0) break;
      const Tiles w = tiles_of(it);
      if (w.nt == 0) continue;
      ok = warp_wait(&bar.q_full, loads++ & 1);
      auto s_mma = [&](int x, int j) {  // S_X = Q_X K(j)^T
        const int at = tiles + j;
        if (at >= k_seen) {
          k_seen = at + 1;
          ok = ok && warp_wait(&bar.k_full[at & 1], (at >> 1) & 1);
        }
        tc_fence_after();
        const uint64_t a = qd + (x * TILE >> 4), b = kd + ((at & 1) * TILE >> 4);
        const bool last_user = x == 1 || j < w.js[1] || j >= w.je[1];
        if (ok && elected) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = ((kk >> 2) * SUB + (kk & 3) * 32) >> 4;
            umma_f16(tmem + x * 256, a + off, b + off, IDESC_QK, kk != 0);
          }
          umma_commit(&bar.s_full[x]);
          if (last_user) umma_commit(&bar.k_free[at & 1]);
          if (last_user && j == w.nt - 1) umma_commit(&bar.q_free);
        }
        __syncwarp();
      };
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (w.je[x] > 0 && w.js[x] == 0) s_mma(x, 0);
      for (int j = 0; ok && j < w.nt && !__any_sync(0xffffffffu, *abort_flag); ++j) {
        const int at = tiles + j;
        const uint64_t b = vd + ((at & 1) * TILE >> 4);
        ok = warp_wait(&bar.v_full[at & 1], (at >> 1) & 1);
        // rows behind the last sequence may hold anything, their P is 0 and 0
        // has to come out: cleared here, a row being 128 bytes of each sub-tile
        const int live = end - (w.kt0 + j) * BKV;
        if (ok && live < BKV) {
          const uint32_t v = smem_u32(sV + (at & 1) * TILE);
          for (int i = live * 8 + lane; i < BKV * 8; i += 32) {
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(v + i * 16), "r"(0) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(v + SUB + i * 16), "r"(0) : "memory");
          }
          fence_proxy_async();
          __syncwarp();
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (j >= w.js[x] && j < w.je[x]) {
            // O_X += P_X(j) V(j), P_X in tensor memory over the first 64 columns of S_X
            const bool last_user = x == 1 || j < w.js[1] || j >= w.je[1];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && warp_wait(&bar.p_full[x][half], p_seen[x] & 1);
              tc_fence_after();
              if (ok && elected) {
#pragma unroll
                for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                  umma_f16_ts(tmem + x * 256 + 128, tmem + x * 256 + kk * 8, b + kk * 128, IDESC_PV, j != w.js[x] || kk != 0);
                if (half == 1) {
                  umma_commit(&bar.o_done[x]);
                  if (last_user) umma_commit(&bar.v_free[at & 1]);
                }
              }
              __syncwarp();
            }
            ++p_seen[x];
          }
          if (ok && j + 1 >= w.js[x] && j + 1 < w.je[x]) s_mma(x, j + 1);
        }
      }
      tiles += w.nt;
    }
    if (!ok) *abort_flag = 1;
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY_REGS));
    // softmax: tile x, TMEM lane quarter q = warp % 4, a thread per row
    const int x = (warp - 4) >> 2;
    const int q = warp & 3;
    const uint32_t s_col = tmem + ((uint32_t)(q * 32) << 16) + x * 256;  // S_X (P_X over its first 64 columns)
    const uint32_t o_col = s_col + 128;                                   // O_X
    int seen = 0;  // S tiles of the items before
    bool ok = true;
    for (int n = 0; ok; ++n) {
    const Item it = take_item(n);
    if (it.index < 0) break;
    const Tiles w = tiles_of(it);
    const int steps = w.je[x] - w.js[x], h = w.h, kvh = h / group;
    if (steps == 0) continue;
    const int qx0 = w.q0 + x * BQ;
    const int qpos = qx0 + q * 32 + lane;
    const int lo = pk.first_row(qpos);
    const int max_lo = __reduce_max_sync(0xffffffffu, lo), min_lo = __reduce_min_sync(0xffffffffu, lo);
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < steps; ++j) {
      ok = !*abort_flag && wait(&bar.s_full[x], (seen + j) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const int k0 = (w.kt0 + w.js[x] + j) * BKV;
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_col + c * 32, v[c]);
      tmem_ld_wait();
      // warp-uniform: some key lies outside some row's [lo, row]
      const int row0 = qx0 + q * 32;
      const bool masked = k0 + BKV - 1 > row0 || k0 < max_lo;
      uint32_t blank = 0;  // a bit per 32 keys that no row of the warp sees
      if (masked) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int kc = k0 + c * 32, a = lo - kc, b = qpos - kc;
          if (kc > row0 + 31 || kc + 31 < min_lo) {
            blank |= 1u << c;
          } else if (kc + 31 > row0 || kc < max_lo) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < a || i > b) v[c][i] = 0xff800000u;  // -inf
          }
        }
      }
      // row max of the raw scores (the positive scale commutes with max)
      float top[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        top[c] = __uint_as_float(v[c][0]);
#pragma unroll
        for (int i = 1; i + 1 < 32; i += 2)
          top[c] = max3(top[c], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
        top[c] = fmaxf(top[c], __uint_as_float(v[c][31]));
      }
      if (blank) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (blank >> c & 1u) top[c] = -INFINITY;
      }
      const float m_new = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale_log2);
      const bool rescale = m == -INFINITY ? true : (m_new > m + kRescaleThreshold);
      const float m_use = rescale ? m_new : m;
      const float alpha = (rescale && m != -INFINITY) ? ex2(m - m_use) : 1.0f;
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
        // the s_full wait above proves O_X += P_X(j-1) V(j-1) complete
        for (int c = 0; c < 4; ++c) {
          uint32_t ov[32];
          tmem_ld32(o_col + c * 32, ov);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
          tmem_st32(o_col + c * 32, ov);
        }
      }
      // P = exp2(s * scale - m) as one packed fma per pair of scores; a row
      // with no visible score so far uses m = 0 (every exp2 argument is -inf)
      const float nm = m_use == -INFINITY ? 0.0f : -m_use;
      const uint64_t c2 = pack_f32x2(scale_log2, scale_log2), nm2 = pack_f32x2(nm, nm);
      uint64_t sum[2] = {0ull, 0ull};
      auto put_half = [&](int half, auto blanks) {  // without the test where nothing is masked
        uint32_t pk2[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (decltype(blanks)::value && (blank >> (2 * half + c) & 1u)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) pk2[16 * c + i] = 0u;
            continue;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t* s2 = &v[2 * half + c][2 * i];
            const uint64_t t = fma_f32x2(((uint64_t)s2[1] << 32) | s2[0], c2, nm2);
            const uint64_t e = pack_f32x2(ex2(low(t)), ex2(high(t)));
            sum[i & 1] = add_f32x2(sum[i & 1], e);
            pk2[16 * c + i] = pack_bf16x2(low(e), high(e));
          }
        }
        tmem_st32(s_col + half * 32, pk2);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_full[x][half]);
      };
      if (masked) {
        put_half(0, True{});
        put_half(1, True{});
      } else {
        put_half(0, False{});
        put_half(1, False{});
      }
      const uint64_t both = add_f32x2(sum[0], sum[1]);
      l = l * alpha + (low(both) + high(both));
      m = m_use;
    }
    seen += steps;
    if (ok) {
      ok = warp_wait(&bar.o_done[x], (seen - 1) & 1);
      if (ok) {
        tc_fence_after();
        // a row sees itself at least: a sum of 0 means that every visible
        // score is -inf, and 0 / 0 is what the softmax gives then
        const float inv = 1.0f / l;
        const bool mine = qpos >= pk.begin() && qpos < end;
        uint16_t* orow = t.o + (long long)qpos * t.ldo + h * D;
        float worst = 0.0f;  // NaN or 0 * inf = NaN where an output is not finite
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t ov[32];
          tmem_ld32(o_col + c * 32, ov);
          tmem_ld_wait();
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            f[i] = __uint_as_float(ov[i]) * inv;
            worst = fmaf(f[i], 0.0f, worst);
          }
          if (mine) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
              st_global_v4(orow + c * 32 + g * 8, pack_bf16x2(f[8 * g], f[8 * g + 1]),
                           pack_bf16x2(f[8 * g + 2], f[8 * g + 3]), pack_bf16x2(f[8 * g + 4], f[8 * g + 5]),
                           pack_bf16x2(f[8 * g + 6], f[8 * g + 7]));
          }
        }
        // A masked score adds exactly 0 to the sum, so a sum of NaN comes from a
        // visible one: that row is NaN throughout, as it stands (and where the
        // sum is 0).  What is left are values.
        const bool wild = mine && worst != worst && l > 0.0f;
        if (__any_sync(0xffffffffu, wild))
          repair_rows(t, o_col, inv, wild, qpos, lo, (w.kt0 + w.js[x]) * BKV, min(end, qx0 + BQ), h, kvh, scale_log2);
      } else {
        *abort_flag = 1;
      }
    }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Rotate-half RoPE of q and k in place, position = row - first row of its
// sequence.  A block turns 4 rows: an angle a thread, then every thread 8 pairs
// of a head at a time, the first of them loaded before the angles are known.
// Bound: HBM, 16384 rows of 20 heads 37 us of 26; 60 rows add 2.5 us to the
// pass.  (A thread per row and 8 pairs that walked all heads added 10.)
constexpr int kRopeRows = 4, kRopeThreads = 64 * kRopeRows;
__global__ void __launch_bounds__(kRopeThreads)
    rope_packed_kernel(uint16_t* __restrict__ q, long long ld_q, int hq, uint16_t* __restrict__ k, long long ld_k,
                       int hkv, Packing pk, const __grid_constant__ RopeTable table) {
  __shared__ __align__(16) float2 angle[kRopeRows][64];  // (sin, cos)
  launch_dependents();
  const int begin = pk.begin(), r0 = (int)blockIdx.x * kRopeRows, n = min(kRopeRows, pk.end() - r0);
  if (n <= 0 || r0 + n <= begin) return;  // block-uniform
  const int heads = hq + hkv, items = n * 8 * heads;
  struct Item {
    uint16_t* at;  // null: nothing to turn
    int j, k0;
    uint4 a, b;
  };
  auto fetch = [&](int i) {
    Item it{nullptr, (i >> 3) / heads, (i & 7) * 8};
    const int h = (i >> 3) % heads, r = r0 + it.j;
    if (i >= items || r < begin) return it;
    it.at = (h < hq ? q + (long long)r * ld_q + (long long)h * D : k + (long long)r * ld_k + (long long)(h - hq) * D) + it.k0;
    it.a = *reinterpret_cast<const uint4*>(it.at);
    it.b = *reinterpret_cast<const uint4*>(it.at + 64);
    return it;
  };
  Item next = fetch(threadIdx.x);
  {
    const int i = threadIdx.x & 63, j = threadIdx.x >> 6, r = r0 + j;
    if (j < n) rope_sincos(rope_inv(table, i), r - pk.first_row(r), &angle[j][i].x, &angle[j][i].y);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += kRopeThreads) {
    const Item now = next;
    next = fetch(i + kRopeThreads);
    if (!now.at) continue;
    const uint32_t aw[4] = {now.a.x, now.a.y, now.a.z, now.a.w}, bw[4] = {now.b.x, now.b.y, now.b.z, now.b.w};
    uint32_t ya[4], yb[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 turns = *reinterpret_cast<const float4*>(&angle[now.j][now.k0 + 2 * e]);
      float a0 = __uint_as_float(aw[e] << 16), a1 = __uint_as_float(aw[e] & 0xffff0000u);
      float b0 = __uint_as_float(bw[e] << 16), b1 = __uint_as_float(bw[e] & 0xffff0000u);
      rope_turn(a0, b0, turns.x, turns.y);
      rope_turn(a1, b1, turns.z, turns.w);
      ya[e] = pack_bf16x2(a0, a1);
      yb[e] = pack_bf16x2(b0, b1);
    }
    *reinterpret_cast<uint4*>(now.at) = make_uint4(ya[0], ya[1], ya[2], ya[3]);
    *reinterpret_cast<uint4*>(now.at + 64) = make_uint4(yb[0], yb[1], yb[2], yb[3]);
  }
}

SharedMemorySetup g_setup;

}  // namespace
}  // namespace ennx

using namespace ennx;

extern "C" int32_t ennx_b200_gqa_attention_packed(uint16_t* q, int64_t ld_q, uint16_t* k, int64_t ld_k,
                                                  const uint16_t* v, int64_t ld_v, uint16_t* o, int64_t ld_o,
                                                  const int32_t* cu_seqlens, int32_t num_seqs, int64_t rows,
                                                  int32_t hq, int32_t hkv, float rope_theta, void* stream) {
  cudaStream_t s = (cudaStream_t)stream;
  if (!cu_seqlens || num_seqs <= 0) return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_packed: no sequences");
  if (rows < 0 || hq <= 0 || hkv <= 0 || hq % hkv)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_packed: Hq must be a positive multiple of Hkv");
  if (!(rope_theta >= 0.0f) || isinf(rope_theta))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_packed: rope_theta must be finite and not negative");
  if (rows == 0) return ENNX_B200_OK;
  if (!q || !k || !v || !o) return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_packed: null argument");
  if (rope_theta > 0.0f && (q == k || q == v || k == v))
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_packed: q and k are rotated in place and cannot be shared");
  // columns of a row are counted in 32 bits
  if (rows > 0x7fffff00LL || hq > 0x7fffffff / D || (rows + 2 * BQ - 1) / (2 * BQ) * hq > 0x7fffffffLL)
    return set_error(ENNX_B200_UNSUPPORTED, "attention_packed: too many rows or heads");
  if (ld_q < (int64_t)hq * D || ld_o < (int64_t)hq * D || ld_k < (int64_t)hkv * D || ld_v < (int64_t)hkv * D)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_packed: a row stride is shorter than its heads");
  if ((ld_q | ld_k | ld_v | ld_o) % 8 || (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) & 15u))
    return set_error(ENNX_B200_INVALID_ARGUMENT,
                     "attention_packed: operands must be 16-byte aligned with strides of a multiple of 8");
  const auto memory = [&](const uint16_t* p, int64_t ld, int heads) {
    return Memory::rows(p, rows, ld * 2, (int64_t)heads * D * 2);
  };
  const Memory mq = memory(q, ld_q, hq), mk = memory(k, ld_k, hkv), mv = memory(v, ld_v, hkv), mo = memory(o, ld_o, hq);
  const Memory mcu = Memory::bytes(cu_seqlens, ((int64_t)num_seqs + 1) * 4);
  for (const Memory& m : {mq, mk, mv, mcu})
    if (share_bytes(mo, m))
      return set_error(ENNX_B200_INVALID_ARGUMENT, "attention_packed: o must not overlap q, k, v or cu_seqlens");
  if (rope_theta > 0.0f && (share_bytes(mq, mk) || share_bytes(mq, mv) || share_bytes(mk, mv) || share_bytes(mq, mcu) ||
                            share_bytes(mk, mcu)))
    return set_error(ENNX_B200_INVALID_ARGUMENT,
                     "attention_packed: q and k are rotated in place and cannot overlap one another, v or cu_seqlens");
  int dev = 0;
  int* err = nullptr;
  ENNX_TRY(serving_device(&dev, &err));
  ENNX_TRY(allow_shared_memory(g_setup, dev, prompt_attention_kernel, SMEM));
  CUtensorMap tq, tk, tv;
  ENNX_TRY(make_tmap_2d_bf16(&tq, q, (uint64_t)hq * D, (uint64_t)rows, (uint64_t)ld_q, 64, 128, true));
  ENNX_TRY(make_tmap_2d_bf16(&tk, k, (uint64_t)hkv * D, (uint64_t)rows, (uint64_t)ld_k, 64, 128, true));
  ENNX_TRY(make_tmap_2d_bf16(&tv, v, (uint64_t)hkv * D, (uint64_t)rows, (uint64_t)ld_v, 64, 128, true));
  const Packing pk{cu_seqlens, num_seqs, (int)rows};
  if (rope_theta > 0.0f) {
    const RopeTable& table = rope_table(rope_theta);
    rope_packed_kernel<<<(unsigned)((rows + kRopeRows - 1) / kRopeRows), kRopeThreads, 0, s>>>(q, ld_q, hq, k, ld_k, hkv, pk,
                                                                                            table);
    ENNX_LAUNCH_CHECK("rope packed");
  }
  const Operands t{q, k, v, o, ld_q, ld_k, ld_v, ld_o};
  const unsigned grid = (unsigned)((rows + 2 * BQ - 1) / (2 * BQ) * hq);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cudaLaunchAttribute early;  // behind the rotation: the blocks set up while it runs
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = rope_theta > 0.0f ? 1 : 0;
  ENNX_CUDA(cudaLaunchKernelEx(&cfg, prompt_attention_kernel, tq, tk, tv, t, pk, hq, hq / hkv,
                               1.4426950408889634f / sqrtf((float)D), wait_limit_ns(rows), err), "packed attention");
  ENNX_LAUNCH_CHECK("packed attention");
  return ENNX_B200_OK;
}

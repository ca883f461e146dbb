// packed_decode.cu -- packed int4/int8 products for a few tokens (at most 16),
// straight from the codes.
//
//   out[t, r] = sum_groups s[r, G] * (sum_{c in G} code[r, c] x[t, c])
//                        + b[r, G] * (sum_{c in G} x[t, c])
//
// with the codes moved by the packed hash first when the seed is enabled.
// Taking scale and bias out of the sum leaves products of integers below 256
// and bf16 activations, which bf16 tensor products hold exactly; nothing is
// rounded to bf16 but the result, and no dequantised weight exists anywhere.
//
// Bound: HBM, half a byte or a byte per weight and 8 bytes per group.  Weight
// rows are the 16 rows of m16n8k16, tokens the 8 columns.  A warp owns 256
// columns of k: its activations stay in registers for all rows, its codes
// stream through a ring in shared memory; the warps of a row tile are joined through
// shared memory.  Narrow matrices put fewer warps on k and more on rows.  Rows
// may start at any byte: the ring holds the 16-byte granules that cover them
// (each holds at least one byte of the row) and reads are shifted into place.
#include "kernels.cuh"
#include "packed.cuh"
#include "serve.cuh"

namespace ennx {
namespace {

constexpr int kMaxTokens = 16;

struct Product {
  const uint16_t* x;
  const uint8_t* w;   // first code of row 0
  const float *sc, *bi;
  uint16_t* out;
  PackedDesc d;
  ennx_b200_perturb_seed seed;
  int tokens;
};

// The code moved by its step: down where the hash is even, up where it is odd,
// reflected at the ends of the code range (perturb_code, kda_moe.metal:73-90,
// without its branches; a step of 0 leaves the code).  `product` is element *
// 0x9E3779B9, the hash's first multiplication.
__device__ __forceinline__ uint32_t moved_code(uint32_t code, const Product& p, uint32_t product, uint32_t max_code) {
  uint32_t v = p.seed.low ^ product;
  v ^= v >> 16;
  v *= 0x7FEB352Du;
  v ^= v >> 15;
  v *= 0x846CA68Bu;
  v ^= v >> 15;
  v ^= p.seed.high;
  // (v >> 1) < (threshold >> 1) is v < threshold without its last bit
  const uint32_t amount = p.d.whole + (v < (p.d.threshold & ~1u) ? 1u : 0u);
  const uint32_t up = code + amount, down = code - amount;
  const bool room_below = code >= amount;
  const uint32_t when_even = room_below ? down : min(up, max_code);
  const uint32_t when_odd = up <= max_code ? up : room_below ? down : 0u;
  return (v & 1u) ? when_odd : when_even;
}
constexpr uint32_t kHashFactor = 0x9E3779B9u;

// ---------------------------------------------------------------------------
// any group size and width: a warp per row, a lane per column
// ---------------------------------------------------------------------------
template <int kN>
__global__ void __launch_bounds__(256) packed_rows_kernel(const __grid_constant__ Product p) {
  const int lane = threadIdx.x & 31;
  const uint32_t max_code = (1u << p.d.bits) - 1u;
  for (uint64_t row = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < p.d.output_width; row += (uint64_t)gridDim.x * 8) {
    const uint8_t* w = p.w + row * p.d.row_bytes;
    const float *sc = p.sc + row * p.d.groups, *bi = p.bi + row * p.d.groups;
    float acc[kN] = {};
    for (uint32_t c = lane; c < p.d.input_width; c += 32) {
      uint32_t code = p.d.bits == 4 ? (__ldg(w + (c >> 1)) >> ((c & 1) * 4)) & 15u : __ldg(w + c);
      if (p.seed.enabled)
        code = moved_code(code, p, kHashFactor * ((uint32_t)p.d.element_offset + (uint32_t)row * (uint32_t)p.d.input_width + c), max_code);
      const uint32_t group = min(c / p.d.group_size, (uint32_t)p.d.groups - 1u);
      const float v = __fmaf_rn((float)code, __ldg(sc + group), __ldg(bi + group));
#pragma unroll
      for (int t = 0; t < kN; ++t)
        if (t < p.tokens) acc[t] = fmaf(bf16_to_f32(__ldg(p.x + (uint64_t)t * p.d.input_width + c)), v, acc[t]);
    }
#pragma unroll
    for (int t = 0; t < kN; ++t)
      if (t < p.tokens) {
#pragma unroll
        for (int off = 16; off; off >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], off);
        if (lane == 0) p.out[(uint64_t)t * p.d.output_width + row] = f32_to_bf16_rne(acc[t]);
      }
  }
}

// ---------------------------------------------------------------------------
// groups of a multiple of 32 columns: tensor products of codes
// ---------------------------------------------------------------------------
// Columns of k that a warp owns in a pass, and warps of a block.  Moved codes
// cost some 30 integer instructions each and are bound by them: half the
// columns and twice the warps keep twice as many instructions ready.
template <bool kMoved>
struct Shape {
  static constexpr int kChunks = kMoved ? 4 : 8, kSlice = 32 * kChunks, kWarps = kMoved ? 16 : 8, kBlocks = kMoved ? 1 : 2;
};

// How a call is laid out: `along` warps side by side on k, the others on rows.
struct Split {
  int along, row_warps;  // together all warps of a block
  int passes;            // slices per warp on k
  int tiles;             // row tiles of 16
  int* status;
  int shift;   // kWideTiles: a group lasts 1 << shift flushes
};

// How a stage is filled.  kAny: rows at any address, 16-byte granules by cp.async
// and reads shifted into place.  The others want rows that start on 16 bytes.
// kRows: 16-byte pieces by cp.async, without arithmetic per row.  kTiles: a warp's
// codes of a tile come by one TMA copy.  kAllTiles: so do scales and biases
// (kWideTiles: of groups of several flushes), and one more warp copies for the
// block (int4, 4 tokens on 151936 rows, groups of 64: kAny 69 us, kRows 55,
// kAllTiles 51; groups of 128: kRows 55, kWideTiles 51).
enum Fill { kAny, kRows, kTiles, kAllTiles, kWideTiles };

// One stage of a warp's ring: 16 code rows, and their scales and biases.  A
// flush is kFlush products of 16 columns under one scale; lane t of a row takes
// 4 * kFlush consecutive columns of it, one shared-memory read.
template <int kBits, int kFlush, bool kMoved, int kFill>
struct Stage {
  static constexpr int kSlice = Shape<kMoved>::kSlice, kRowBytes = kSlice * kBits / 8;
  static constexpr bool kBoxes = kFill >= kTiles;  // copied by TMA
  // cp.async: rows of a fragment read lie on different banks (an 8-lane phase
  // covers whole rows, each kFlush * 2 * kBits bytes), and a row that starts
  // inside a 16-byte granule still fits.  TMA: 128-byte rows, the 16-byte
  // chunks of row r exchanged by r & 7.
  static constexpr int kPitch = kBoxes ? 128 : kRowBytes + kFlush * 2 * kBits;
  static constexpr int kPieces = kRowBytes / 16 + 1;
  static constexpr int kFlushes = kSlice / 16 / kFlush;
  static constexpr int kCode = 16 * (kBoxes ? kRowBytes : kPitch);
  static constexpr int kScale = 16 * kFlushes * 8;  // (scale, bias) pairs; kAllTiles: scales, then biases
  // from one stage of a warp to the next: cp.async keeps a stage's scales behind
  // its codes, boxes have a ring of their own for them
  static constexpr int kCodeStep = kBoxes ? kCode : kCode + kScale;
  // depth: as many as leave 16 warps on an SM (80 to 100 KB in flight)
  static constexpr int kDepth = kBits == 8 ? 2 : 3;
};
// rings of codes, rings of scales, sums of x, joins
template <int kBits, int kN, int kFlush, bool kMoved, int kFill>
constexpr int smem_bytes() {
  using S = Stage<kBits, kFlush, kMoved, kFill>;
  return (S::kBoxes ? 1024 : 0) +
         Shape<kMoved>::kWarps * (S::kDepth * (S::kCode + S::kScale) + S::kFlushes * 8 * kN * 4 + 2 * kN * 32 * 16);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool ok) {  // zero where !ok
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[N]) {
  static_assert(N == 1 || N == 2 || N == 4, "one shared-memory read");
  if constexpr (N == 1) w[0] = lds32(a);
  else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a) : "memory");
  else asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
}
// 32 bits of a row at any byte address
__device__ __forceinline__ uint32_t word_at(uint32_t a) {
  const uint32_t lo = a & ~3u;
  return __funnelshift_r(lds32(lo), lds32(lo + 4), (a & 3u) * 8);
}
// bf16 pair of two integers below 256, exact: 2^23 + n in fp32, less 2^23
__device__ __forceinline__ uint32_t pair_of(uint32_t lo, uint32_t hi) {
  return pack_bf16x2(__uint_as_float(0x4b000000u | lo) - 8388608.0f, __uint_as_float(0x4b000000u | hi) - 8388608.0f);
}

// box of a tensor map to shared memory, completing on `bar`
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                   dst), "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(x), "r"(y)
               : "memory");
}
// (v & 0x000f000f) | 0x43004300 in one logic instruction: written out, it
// became two, and logic instructions are what the unpacking is made of
__device__ __forceinline__ uint32_t nibbles_under_128(uint32_t v) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(0x000f000fu), "r"(0x43004300u));
  return r;
}
// Eight consecutive codes of a lane as four bf16 pairs, plus kCodeBias.
// 4 bits: pairs (j, j + 4): two nibbles 16 bits apart are or-ed under the
// exponent of 128 (128 + n is exact in bf16) and left there: the 128 x that
// come with the products are taken off once per scale.  8 bits: pairs (0, 1),
// (2, 3), ...  activation_pairs orders x the same way.
template <int kBits>
constexpr float kCodeBias = kBits == 4 ? 128.0f : 0.0f;
template <int kBits, bool kMoved>
__device__ __forceinline__ void code_pairs(const uint32_t* w, uint32_t element, const Product& p, uint32_t (&r)[4]) {
  if constexpr (kMoved) {
    const uint32_t product = element * kHashFactor;
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t code = kBits == 4 ? (w[0] >> (4 * j)) & 15u : (w[j >> 2] >> (8 * (j & 3))) & 255u;
      c[j] = moved_code(code, p, product + (uint32_t)j * kHashFactor, (1u << kBits) - 1u);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      r[j] = kBits == 4 ? (c[j] | c[j + 4] << 16 | 0x43004300u) : pair_of(c[2 * j], c[2 * j + 1]);
  } else if constexpr (kBits == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = nibbles_under_128(w[0] >> (4 * j));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      r[j] = pair_of(__byte_perm(w[j >> 1], 0, 0x4440 + 2 * (j & 1)), __byte_perm(w[j >> 1], 0, 0x4441 + 2 * (j & 1)));
  }
}
template <int kBits>
__device__ __forceinline__ uint4 activation_pairs(uint4 v) {  // columns (0,1) (2,3) (4,5) (6,7)
  if constexpr (kBits == 8) return v;
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                    __byte_perm(v.y, v.w, 0x7632));
}

// Tensor maps of rows of bytes and of floats.  Fills without boxes get none: a
// launch pays for its parameters (three unused maps: 0.15 us).
template <bool kBoxes>
struct Maps {
  CUtensorMap codes, scales, biases;
};
template <>
struct Maps<false> {};

// kAllTiles: one more warp copies for all
template <bool kMoved, int kFill>
constexpr int block_threads() { return 32 * (Shape<kMoved>::kWarps + (kFill >= kAllTiles)); }

// kN: blocks of 8 tokens
template <int kBits, int kN, int kFlush, bool kMoved, int kFill>
__global__ void __launch_bounds__(block_threads<kMoved, kFill>(), Shape<kMoved>::kBlocks)
    packed_tiles_kernel(const __grid_constant__ Product p, const __grid_constant__ Split sp,
                        const __grid_constant__ Maps<(kFill >= kTiles)> maps) {
  using S = Stage<kBits, kFlush, kMoved, kFill>;
  constexpr int kSlice = S::kSlice, kSliceChunks = Shape<kMoved>::kChunks, kWarps = Shape<kMoved>::kWarps;
  constexpr int kFlushes = S::kFlushes, kStages = S::kDepth, kRuns = kFlush / 2;  // runs of 8 columns of a lane in a flush
  extern __shared__ __align__(16) uint8_t raw_smem[];
  uint8_t* smem = raw_smem + (S::kBoxes ? (1024u - (smem_u32(raw_smem) & 1023u)) & 1023u : 0u);
  __shared__ uint64_t bars[kWarps][kStages];  // kAllTiles: of all warps, full in row 0 and free in row 1
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  // A lane's rows of the tile are row_g and row_g + 8.  Of 16 lanes that read 8
  // bytes (or 8 that read 16) in one go the exchanged chunks then differ.
  constexpr int kLane = kRuns * kBits;  // bytes of a lane in a flush
  const int row_g = !S::kBoxes ? g : kLane == 16 ? g >> 1 | (g & 1) << 2 : (g & 3) << 1 | g >> 2;
  const int wk = warp % sp.along, wr = warp / sp.along;
  const int shift = kFill == kWideTiles ? sp.shift : 0;
  const uint32_t base = smem_u32(smem), ring = base + warp * kStages * S::kCodeStep;
  const uint32_t scale_ring = S::kBoxes ? base + kWarps * kStages * S::kCode + warp * kStages * S::kScale : ring + S::kCode;
  uint64_t* full = bars[kFill >= kAllTiles ? 0 : warp];
  uint64_t* free_ = bars[1];
  if constexpr (kFill == kTiles) {
    if (lane < kStages) mbar_init(full + lane, 1);
    fence_barrier_init();
    fence_proxy_async();
    __syncwarp();
  }
  if constexpr (kFill >= kAllTiles) {
    if (threadIdx.x < kStages) {
      mbar_init(full + threadIdx.x, 1);
      mbar_init(free_ + threadIdx.x, kWarps);
      fence_barrier_init();
      fence_proxy_async();
    }
    __syncthreads();
    if (warp == kWarps) {
      // Stages of the whole block: a box of codes per warp, a box of scales and
      // one of biases per row tile.  (Copies by the warps themselves, cp.async
      // or boxes, cost each some 600 of a tile's 2300 clocks.)
      const int item = lane - kWarps;  // of scales and biases
      const int my_wr = lane < kWarps ? lane / sp.along : item >> 1;
      int n = 0;
      bool ok = true;
      for (int tile0 = (int)blockIdx.x * sp.row_warps; ok && tile0 < sp.tiles; tile0 += (int)gridDim.x * sp.row_warps)
        for (int pass = 0; ok && pass < sp.passes; ++pass, ++n) {
          const int at = n % kStages, live = min(sp.row_warps, sp.tiles - tile0);
          ok = __all_sync(0xffffffffu, mbar_wait(free_ + at, ((n / kStages) & 1) ^ 1, sp.status)) != 0;
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(full + at, live * (sp.along * S::kCode + (sp.along * S::kScale >> shift)));
          __syncwarp();
          const int row = (tile0 + my_wr) * 16;
          if (lane < kWarps && my_wr < live) {
            const int first = (pass * sp.along + lane % sp.along) * S::kRowBytes;
#pragma unroll
            for (int i = 0; i < S::kRowBytes / 128; ++i)
              copy_box(base + (at * kWarps + lane) * S::kCode + i * 2048, &maps.codes, full + at, first + 128 * i, row);
          } else if (item >= 0 && item < 2 * live) {
            copy_box(base + kWarps * kStages * S::kCode + at * kWarps * S::kScale + (item & 1) * (kWarps * S::kScale / 2) +
                         (my_wr * sp.along * (S::kScale / 2) >> shift),
                     item & 1 ? &maps.biases : &maps.scales, full + at, pass * sp.along * S::kFlushes >> shift, row);
          }
        }
      // no copy may land behind the block, whose other warps skip their waits once one has given up
      for (int i = max(0, n - kStages); i < n; ++i) mbar_wait(full + i % kStages, (i / kStages) & 1, sp.status);
      return;
    }
  }
  // sums of x over each flush of this warp's slice, per token
  constexpr int kRings = kWarps * kStages * (S::kCode + S::kScale);
  float* xsum = reinterpret_cast<float*>(smem + kRings) + warp * kFlushes * 8 * kN;
  float4* red = reinterpret_cast<float4*>(smem + kRings + kWarps * kFlushes * 8 * kN * 4);
  const uint32_t width = (uint32_t)p.d.input_width, rows = (uint32_t)p.d.output_width, groups = (uint32_t)p.d.groups;
  const uint32_t row_bytes = (uint32_t)p.d.row_bytes;
  const bool wide_x = width % 8 == 0 && ((uintptr_t)p.x & 15u) == 0;

  const int stride = (int)gridDim.x * sp.row_warps;
  int tile = (int)blockIdx.x * sp.row_warps + wr;
  auto slice0 = [&](int pass) { return (uint32_t)(pass * sp.along + wk) * kSlice; };

  // Scale and bias that a lane copies of a tile: at row `scale_row` and every
  // kScaleRows further down.  Offsets run from tile to tile.
  constexpr int kScaleRows = 32 / kFlushes;
  const uint32_t scale_row = lane / kFlushes, scale_col = lane % kFlushes * (kFlush * 16);
  auto group_of = [&](int pass) { return min((slice0(pass) + scale_col) / p.d.group_size, groups - 1u); };
  uint32_t f_group = group_of(0), f_row = (uint32_t)tile * 16;
  uint64_t f_scale = (uint64_t)(f_row + scale_row) * groups;
  const uint64_t scale_step = (uint64_t)(16 * stride) * groups;
  // kRows: a lane's piece of row `code_row` and of every kCopyRows further down
  constexpr int kLanes = S::kRowBytes / 16, kCopyRows = 32 / kLanes;
  const uint32_t code_row = lane / kLanes, code_at = 16 * (lane % kLanes);
  const uint8_t* f_code = p.w + (uint64_t)(f_row + code_row) * row_bytes + code_at;
  const uint64_t code_step = (uint64_t)(16 * stride) * row_bytes;
  int f_tile = tile, f_pass = 0, f_stage = 0, fetched = 0;
  uint32_t f_at = ring;  // without boxes: the stage's address (from the number it takes registers that spill)
  auto fetch = [&] {
    if constexpr (kFill >= kAllTiles) return;
    if (f_tile < sp.tiles) {
      const uint32_t dst = S::kBoxes ? ring + f_stage * S::kCode : f_at, sdst = S::kBoxes ? scale_ring + f_stage * S::kScale : f_at + S::kCode;
      const uint32_t c0 = slice0(f_pass), first = c0 / 8 * kBits;  // c0 * kBits may pass 32 bits
      if constexpr (kFill == kAny) {
        if (c0 < width) {
          // 16-byte granules that hold a byte of the slice, none behind the row's last
          const uint32_t last = min(row_bytes, first + S::kRowBytes);
#pragma unroll
          for (int i = lane; i < 16 * S::kPieces; i += 32) {
            const int r = i / S::kPieces, c = i % S::kPieces;
            const uint32_t row = f_row + r;
            if (row < rows) {
              const uint8_t* start = p.w + (uint64_t)row * row_bytes + first;
              const uint8_t* src = reinterpret_cast<const uint8_t*>((uintptr_t)start & ~(uintptr_t)15) + 16 * c;
              if (src < start + (last - first)) cp_async16(dst + r * S::kPitch + 16 * c, src);
            }
          }
        }
      } else if constexpr (kFill == kRows) {
        if (first + code_at < row_bytes) {
          const uint8_t* src = f_code + first;
          const uint32_t to = dst + code_row * S::kPitch + code_at;
          if (f_row + 16 <= rows) {
#pragma unroll
            for (int i = 0; i < 16 / kCopyRows; ++i)
              cp_async16(to + i * kCopyRows * S::kPitch, src + (uint64_t)(i * kCopyRows) * row_bytes);
          } else {
            for (int i = 0; i < 16 / kCopyRows; ++i)
              if (f_row + code_row + i * kCopyRows < rows)
                cp_async16(to + i * kCopyRows * S::kPitch, src + (uint64_t)(i * kCopyRows) * row_bytes);
          }
        }
      } else if constexpr (kFill == kTiles) {
        if (lane == 0) {  // what lies outside the matrix arrives as zeros
          uint64_t* bar = full + f_stage;
          mbar_arrive_expect_tx(bar, S::kCode);
#pragma unroll
          for (int i = 0; i < S::kRowBytes / 128; ++i) copy_box(dst + i * 2048, &maps.codes, bar, (int)first + 128 * i, (int)f_row);
        }
      }
      if constexpr (kFill < kAllTiles) {
        // scales behind the last column are 0, which takes their columns out
        if (sp.passes > 1) f_group = group_of(f_pass);
        const bool inside = c0 + scale_col < width, whole = f_row + 16 <= rows;
        const float *sc = p.sc + f_scale + f_group, *bi = p.bi + f_scale + f_group;
#pragma unroll
        for (int i = 0; i < 16 / kScaleRows; ++i) {
          const bool ok = inside && (whole || f_row + scale_row + i * kScaleRows < rows);
          const uint64_t down = ok ? (uint64_t)(i * kScaleRows) * groups : 0;
          cp_async4(sdst + lane * 8 + i * 256, ok ? sc + down : p.sc, ok);
          cp_async4(sdst + lane * 8 + i * 256 + 4, ok ? bi + down : p.bi, ok);
        }
      }
      ++fetched;
      if (++f_pass == sp.passes) {
        f_pass = 0;
        f_tile += stride;
        f_row += 16 * stride;
        f_scale += scale_step;
        f_code += code_step;
      }
    }
    f_stage = f_stage + 1 == kStages ? 0 : f_stage + 1;
    f_at = f_at + S::kCodeStep == ring + kStages * S::kCodeStep ? ring : f_at + S::kCodeStep;
    if constexpr (kFill < kAllTiles) cp_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  uint4 xf[kSliceChunks][kN];
  // Activations of the slice, zeros behind the last column or token, and their
  // sums per flush: products with ones, in the order of the codes' products,
  // so that the 128 of a 4-bit code's pair cancels to the last bit.
  auto load_x = [&](int pass) {
    const uint32_t c0 = slice0(pass);
    __syncwarp();
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int tok = n * 8 + g;
      const uint16_t* x = p.x + (uint64_t)(tok < p.tokens ? tok : 0) * width;
#pragma unroll
      for (int j = 0; j < kSliceChunks; ++j) {
        const uint32_t c = c0 + j / kRuns * (16 * kFlush) + t * (8 * kRuns) + j % kRuns * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (tok < p.tokens) {
          if (wide_x) {
            if (c < width) v = __ldg(reinterpret_cast<const uint4*>(x + c));
          } else {
            uint32_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = c + i < width ? __ldg(x + c + i) : 0u;
            v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
          }
        }
        xf[j][n] = activation_pairs<kBits>(v);
      }
    }
    constexpr uint32_t kOnes = 0x3f803f80u;
#pragma unroll
    for (int f = 0; f < kFlushes; ++f)
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        float sum[4] = {};
#pragma unroll
        for (int j = f * kRuns; j < (f + 1) * kRuns; ++j) {
          mma_16x8x16(sum, kOnes, kOnes, kOnes, kOnes, xf[j][n].x, xf[j][n].y);
          mma_16x8x16(sum, kOnes, kOnes, kOnes, kOnes, xf[j][n].z, xf[j][n].w);
        }
        if (g == 0) *reinterpret_cast<float2*>(xsum + (f * kN + n) * 8 + 2 * t) = make_float2(sum[0], sum[1]);
      }
    __syncwarp();
  };
  if (sp.passes == 1) load_x(0);

  int stage = 0, used = 0;
  uint32_t at = ring;  // without boxes: the stage's address
  bool bad = false;  // a wait gave up: later ones are not tried again, the results are void
  for (int done = 0; tile - (kFill >= kAllTiles ? wr : 0) < sp.tiles; ++done) {
    if (kFill >= kAllTiles && tile >= sp.tiles) {  // a stage without a tile for this warp
      for (int pass = 0; pass < sp.passes; ++pass, ++used) {
        if (!bad) bad = !mbar_wait(full + stage, (used / kStages) & 1, sp.status);
        __syncwarp();
        if (lane == 0) mbar_arrive(free_ + stage);
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
      tile += stride;
      continue;
    }
    float out[kN][4] = {};
    for (int pass = 0; pass < sp.passes; ++pass) {
      if (sp.passes > 1) load_x(pass);
      if constexpr (kFill < kAllTiles) cp_wait<kStages - 2>();
      if constexpr (S::kBoxes)
        if (!bad) bad = !mbar_wait(full + stage, (used / kStages) & 1, sp.status);
      ++used;
      __syncwarp();  // the stage is there, and all lanes have read the one before it,
      fetch();       // which is filled again while this one is used
      const uint32_t c0 = slice0(pass);
      {
        // (kAllTiles: rings of the block, scales of the tile's slices side by side)
        const uint32_t st = kFill >= kAllTiles ? base + (stage * kWarps + warp) * S::kCode : S::kBoxes ? ring + stage * S::kCode : at;
        const uint32_t scales = kFill >= kAllTiles ? base + kWarps * kStages * S::kCode + stage * kWarps * S::kScale +
                                                         (wr * sp.along * (S::kScale / 2) >> shift)
                                                   : S::kBoxes ? scale_ring + stage * S::kScale : at + S::kCode;
        uint32_t addr[2], element[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t r = row_g + 8 * h, row = (uint32_t)tile * 16 + r;
          if constexpr (kFill == kAny) {
            const uint32_t skew = (uint32_t)((uintptr_t)(p.w + (uint64_t)row * row_bytes) + c0 / 8 * kBits) & 15u;
            addr[h] = st + r * S::kPitch + skew + t * kLane;
          } else if constexpr (kFill == kRows) {
            addr[h] = st + r * S::kPitch + t * kLane;
          } else {
            addr[h] = st + r * 128 + ((uint32_t)(t * kLane) ^ (r & 7) << 4);
          }
          element[h] = (uint32_t)p.d.element_offset + row * width + c0 + t * (8 * kRuns);
        }
        uint32_t group4[4][4];  // kAllTiles: scales and biases of rows row_g and row_g + 8 in four flushes
#pragma unroll
        for (int f = 0; f < kFlushes; ++f) {
          float acc[kN][4] = {};
          constexpr int kWords = kLane / 4;  // of a lane's columns in a flush
          uint32_t w[2][kWords];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            constexpr int kFlushBytes = 4 * kLane;
            if constexpr (kFill == kAny) {
#pragma unroll
              for (int i = 0; i < kWords; ++i) w[h][i] = word_at(addr[h] + f * kFlushBytes + 4 * i);
            } else if constexpr (kFill == kRows) {
              lds_words<kWords>(addr[h] + f * kFlushBytes, w[h]);
            } else {
              lds_words<kWords>((addr[h] ^ (f * kFlushBytes & 127)) + f * kFlushBytes / 128 * 2048, w[h]);
            }
          }
          if constexpr (kFill >= kAllTiles) {
            const int pitch = kFlushes * sp.along >> shift, group = (wk * kFlushes + f) >> shift;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t from = scales + (i & 1) * (kWarps * S::kScale / 2) + ((row_g + 8 * (i >> 1)) * pitch + group) * 4;
              if constexpr (kFill == kWideTiles) group4[i][f % 4] = lds32(from);
              else if (f % 4 == 0) lds_words<4>(from, group4[i]);
            }
          }
#pragma unroll
          for (int i = 0; i < kRuns; ++i) {
            const int j = f * kRuns + i;
            uint32_t a[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
              code_pairs<kBits, kMoved>(&w[h][i * (kBits / 4)], element[h] + f * (16 * kFlush) + i * 8, p, a[h]);
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              mma_16x8x16(acc[n], a[0][0], a[1][0], a[0][1], a[1][1], xf[j][n].x, xf[j][n].y);
              mma_16x8x16(acc[n], a[0][2], a[1][2], a[0][3], a[1][3], xf[j][n].z, xf[j][n].w);
            }
          }
          {
            uint32_t u[2], v[2];  // (scale, bias) of rows row_g and row_g + 8
            if constexpr (kFill >= kAllTiles) {
#pragma unroll
              for (int i = 0; i < 2; ++i) { u[i] = group4[i][f % 4]; v[i] = group4[2 + i][f % 4]; }
            } else {
              const uint32_t sa = scales + (row_g * kFlushes + f) * 8;
              lds_words<2>(sa, u);
              lds_words<2>(sa + 64 * kFlushes, v);
            }
            const float s0 = __uint_as_float(u[0]), b0 = __uint_as_float(u[1]);
            const float s1 = __uint_as_float(v[0]), b1 = __uint_as_float(v[1]);
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              const float2 xs = *reinterpret_cast<const float2*>(xsum + (f * kN + n) * 8 + 2 * t);
              // exact where all codes are 0: acc is 128 xs then, sum by sum (see load_x)
              constexpr float kBias = kCodeBias<kBits>;
              out[n][0] = fmaf(s0, fmaf(-kBias, xs.x, acc[n][0]), fmaf(b0, xs.x, out[n][0]));
              out[n][1] = fmaf(s0, fmaf(-kBias, xs.y, acc[n][1]), fmaf(b0, xs.y, out[n][1]));
              out[n][2] = fmaf(s1, fmaf(-kBias, xs.x, acc[n][2]), fmaf(b1, xs.x, out[n][2]));
              out[n][3] = fmaf(s1, fmaf(-kBias, xs.y, acc[n][3]), fmaf(b1, xs.y, out[n][3]));
            }
          }
        }
      }
      if constexpr (kFill >= kAllTiles) {
        __syncwarp();
        if (lane == 0) mbar_arrive(free_ + stage);
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
      at = at + S::kCodeStep == ring + kStages * S::kCodeStep ? ring : at + S::kCodeStep;
    }
    if (sp.along > 1) {
      // one barrier a tile: the other buffer is written again only after the
      // next barrier, which every reader of this one reaches first
      float4* buf = red + ((done & 1) * sp.row_warps + wr) * sp.along * kN * 32;
#pragma unroll
      for (int n = 0; n < kN; ++n) buf[(wk * kN + n) * 32 + lane] = make_float4(out[n][0], out[n][1], out[n][2], out[n][3]);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + wr), "r"(32 * sp.along) : "memory");
#pragma unroll
      for (int n = 0; n < kN; ++n)
        if (wk == n) {
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int w = 0; w < sp.along; ++w) {
            const float4 u = buf[(w * kN + n) * 32 + lane];
            v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
          }
          out[n][0] = v.x; out[n][1] = v.y; out[n][2] = v.z; out[n][3] = v.w;
        }
    }
#pragma unroll
    for (int n = 0; n < kN; ++n)
      if (sp.along == 1 || wk == n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t row = (uint32_t)tile * 16 + row_g + 8 * (j >> 1);
          const int tok = n * 8 + 2 * t + (j & 1);
          if (row < rows && tok < p.tokens) p.out[(uint64_t)tok * rows + row] = f32_to_bf16_rne(out[n][j]);
        }
    tile += stride;
  }
  if constexpr (kFill < kAllTiles) cp_wait<0>();
  if (kFill == kTiles && bad)  // no copy may land behind the block
    for (int i = max(0, fetched - kStages); i < fetched; ++i) mbar_wait(full + i % kStages, (i / kStages) & 1, sp.status);
}

template <int kBits, int kN, int kFlush, bool kMoved, int kFill>
int32_t launch_tiles(const Product& p, cudaStream_t s) {
  const auto kernel = packed_tiles_kernel<kBits, kN, kFlush, kMoved, kFill>;
  Split sp{};
  constexpr int kSlice = Shape<kMoved>::kSlice, kWarps = Shape<kMoved>::kWarps;
  const int slices = (int)((p.d.input_width + kSlice - 1) / kSlice);
  sp.along = 1;
  while (sp.along < slices && sp.along < kWarps) sp.along *= 2;
  sp.row_warps = kWarps / sp.along;
  sp.passes = (slices + sp.along - 1) / sp.along;
  sp.tiles = (int)((p.d.output_width + 15) / 16);
  constexpr int smem = smem_bytes<kBits, kN, kFlush, kMoved, kFill>();
  static_assert(Shape<kMoved>::kBlocks * (smem + 2048) <= 228 * 1024 && smem <= 226 * 1024, "blocks of an SM");
  static SharedMemorySetup setup;
  int dev = 0;
  ENNX_TRY(serving_device(&dev, &sp.status));
  ENNX_TRY(allow_shared_memory(setup, dev, kernel, smem));
  Maps<(kFill >= kTiles)> maps{};
  if constexpr (kFill >= kTiles)
    ENNX_TRY(make_tmap_2d(&maps.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, p.d.row_bytes, p.d.output_width, p.d.row_bytes, 128, 16,
                          128));
  if constexpr (kFill >= kAllTiles) {
    constexpr uint32_t kGroups = kSlice / 16 / kFlush;
    while (16u * kFlush << sp.shift < p.d.group_size) ++sp.shift;
    for (int i = 0; i < 2; ++i)
      ENNX_TRY(make_tmap_2d(i ? &maps.biases : &maps.scales, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, i ? p.bi : p.sc, p.d.groups,
                            p.d.output_width, p.d.groups * 4, kGroups * sp.along >> sp.shift, 16, 0));
  }
  const int blocks = (sp.tiles + sp.row_warps - 1) / sp.row_warps, cap = Shape<kMoved>::kBlocks * sm_count();
  kernel<<<(unsigned)(blocks < cap ? blocks : cap), block_threads<kMoved, kFill>(), smem, s>>>(p, sp, maps);
  ENNX_LAUNCH_CHECK("packed tiles");
  return ENNX_B200_OK;
}
template <int kBits, int kN, int kFlush>
int32_t launch_tiles(const Product& p, cudaStream_t s) {
  const auto on_16 = [](const void* base, uint64_t row_bytes) { return ((uintptr_t)base & 15u) == 0 && row_bytes % 16 == 0; };
  // moved codes spend their time on the hash: one variant for any alignment
  if (p.seed.enabled) return launch_tiles<kBits, kN, kFlush, true, kAny>(p, s);
  if (!on_16(p.w, p.d.row_bytes)) return launch_tiles<kBits, kN, kFlush, false, kAny>(p, s);
  // One warp copies for the block up to 8 tokens (figures at kAllTiles).  From 9
  // on a thread holds 64 registers of activations, and with the 96 that the ninth
  // warp leaves it the products spill (16 tokens, by one warp and kRows: int4,
  // groups of 32, 151936 rows 110 and 98 us, 16384 x 4096 64 and 54, 2048 x 2048
  // 9.0 and 7.8; groups of 64 80 and 75, 46 and 42, 7.4 and 5.6).  int8 blocks that
  // have one tile gain nothing from copies ahead: from a block per SM on (4
  // tokens, groups of 64, 2048 columns, by one warp and kRows: 512 rows 3.9 and
  // 3.75 us, 2048 rows 4.7 and 4.6; 4096 rows 6.2 and 6.5, 151936 rows 86 and 89).
  if constexpr (kN == 1) {
    // a power of two of flushes per group, and 16 bytes of a row's scales per copy at least
    const uint32_t flushes = p.d.group_size / (16 * kFlush);
    constexpr uint32_t kSlice = Shape<false>::kSlice, kWarps = Shape<false>::kWarps;
    uint32_t along = 1;
    while (along * kSlice < p.d.input_width && along < kWarps) along *= 2;
    const bool groups_fit = p.d.group_size % (16 * kFlush) == 0 && (flushes & (flushes - 1)) == 0 &&
                            along * kSlice / p.d.group_size % 4 == 0 && along * kSlice >= 4 * p.d.group_size;
    const bool enough = kBits == 4 || p.d.output_width > (uint64_t)sm_count() * (16 * (kWarps / along));
    if (enough && groups_fit && on_16(p.sc, p.d.groups * 4) && on_16(p.bi, p.d.groups * 4))
      return flushes == 1 ? launch_tiles<kBits, kN, kFlush, false, kAllTiles>(p, s)
                          : launch_tiles<kBits, kN, kFlush, false, kWideTiles>(p, s);
  }
  // (16 tokens, groups of 64, boxes of a warp's own and kRows: 151936 rows 117 and
  // 129 us, 16384 x 4096 45.1 and 45.8, 2048 x 2048 6.3 and 6.05; the others spill more)
  if constexpr (kN == 2 && kBits == 8 && kFlush == 4) return launch_tiles<kBits, kN, kFlush, false, kTiles>(p, s);
  else return launch_tiles<kBits, kN, kFlush, false, kRows>(p, s);
}
template <int kBits, int kN>
int32_t launch_tiles(const Product& p, cudaStream_t s) {
  return p.d.group_size % 64 == 0 ? launch_tiles<kBits, kN, 4>(p, s) : launch_tiles<kBits, kN, 2>(p, s);
}

}  // namespace
}  // namespace ennx

using namespace ennx;

extern "C" int32_t ennx_b200_packed_linear_decode(const uint16_t* x, int64_t tokens, const uint8_t* weights,
                                                  const float* scales, const float* biases,
                                                  const ennx_b200_packed_linear* linear, ennx_b200_perturb_seed seed,
                                                  uint16_t* out, void* stream) {
  cudaStream_t s = (cudaStream_t)stream;
  Product p;
  ENNX_TRY(make_desc(linear, &p.d));
  if (tokens < 0) return set_error(ENNX_B200_INVALID_ARGUMENT, "packed linear decode: negative token count");
  if (tokens > kMaxTokens)
    return set_error(ENNX_B200_UNSUPPORTED, "packed linear decode: at most %d tokens", kMaxTokens);
  if (p.d.input_width > 0x7fffff00ull || p.d.output_width > 0x7fffff00ull)
    return set_error(ENNX_B200_UNSUPPORTED, "packed linear decode: widths must be below 2^31");
  if (tokens == 0) return ENNX_B200_OK;
  if (!x || !weights || !scales || !biases || !out)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "packed linear decode: null buffer");
  if (((uintptr_t)x | (uintptr_t)out) & 1u || ((uintptr_t)scales | (uintptr_t)biases) & 3u)
    return set_error(ENNX_B200_INVALID_ARGUMENT, "packed linear decode: misaligned buffer");
  p.x = x;
  p.w = weights + p.d.byte_offset;
  p.sc = scales + p.d.scale_offset;
  p.bi = biases + p.d.bias_offset;
  const Memory written = Memory::bytes(out, tokens * (int64_t)p.d.output_width * 2);
  const int64_t codes = (int64_t)(p.d.output_width * p.d.row_bytes), groups = (int64_t)(p.d.output_width * p.d.groups) * 4;
  for (const Memory& read : {Memory::bytes(x, tokens * (int64_t)p.d.input_width * 2), Memory::bytes(p.w, codes),
                             Memory::bytes(p.sc, groups), Memory::bytes(p.bi, groups)})
    if (share_bytes(written, read))
      return set_error(ENNX_B200_INVALID_ARGUMENT, "packed linear decode: out must not overlap x, the codes, scales or biases");
  p.out = out;
  p.seed = seed;
  p.tokens = (int)tokens;
  // a linear that moves no code needs no hash
  if (p.d.whole == 0 && (p.d.threshold >> 1) == 0) p.seed.enabled = 0;
  // one group over the whole row: any size that covers it says the same
  if (p.d.groups == 1) p.d.group_size = (uint32_t)((p.d.input_width + 63) / 64 * 64);
  if (p.d.group_size % 32 == 0) {
    if (p.d.bits == 4) return tokens <= 8 ? launch_tiles<4, 1>(p, s) : launch_tiles<4, 2>(p, s);
    return tokens <= 8 ? launch_tiles<8, 1>(p, s) : launch_tiles<8, 2>(p, s);
  }
  const uint64_t blocks = (p.d.output_width + 7) / 8, cap = (uint64_t)sm_count() * 16;
  const unsigned grid = (unsigned)(blocks < cap ? blocks : cap);
  if (tokens == 1) packed_rows_kernel<1><<<grid, 256, 0, s>>>(p);
  else if (tokens <= 4) packed_rows_kernel<4><<<grid, 256, 0, s>>>(p);
  else packed_rows_kernel<kMaxTokens><<<grid, 256, 0, s>>>(p);
  ENNX_LAUNCH_CHECK("packed linear decode");
  return ENNX_B200_OK;
}

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
// stream through a cp.async ring; the warps of a row tile are joined through
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
};

// One stage of a warp's ring: 16 code rows, then (scale, bias) pairs.  A flush
// is kFlush products of 16 columns under one scale; lane t of a row takes
// 4 * kFlush consecutive columns of it, one shared-memory read.
template <int kBits, int kFlush, bool kMoved>
struct Stage {
  static constexpr int kSlice = Shape<kMoved>::kSlice, kRowBytes = kSlice * kBits / 8;
  // rows of a fragment read lie on different banks (an 8-lane phase covers
  // whole rows, each kFlush * 2 * kBits bytes), and a row that starts inside
  // a 16-byte granule still fits
  static constexpr int kPitch = kRowBytes + kFlush * 2 * kBits;
  static constexpr int kPieces = kRowBytes / 16 + 1;
  static constexpr int kFlushes = kSlice / 16 / kFlush;
  static constexpr int kBytes = 16 * kPitch + 16 * kFlushes * 8;
  // depth: as many as leave 16 warps on an SM (80 to 100 KB in flight)
  static constexpr int kDepth = kBits == 8 ? 2 : 3;
};
// ring, then sums of x, then the joins
template <int kBits, int kN, int kFlush, bool kMoved>
constexpr int smem_bytes() {
  using S = Stage<kBits, kFlush, kMoved>;
  return Shape<kMoved>::kWarps * (S::kDepth * S::kBytes + S::kFlushes * 8 * kN * 4 + 2 * kN * 32 * 16);
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

// kN: blocks of 8 tokens.  kAligned: rows start on 16 bytes and the slice ends
// on a granule, so copies need no per-row arithmetic and reads no shifting.
template <int kBits, int kN, int kFlush, bool kMoved, bool kAligned>
__global__ void __launch_bounds__(32 * Shape<kMoved>::kWarps, Shape<kMoved>::kBlocks)
    packed_tiles_kernel(const __grid_constant__ Product p, const __grid_constant__ Split sp) {
  using S = Stage<kBits, kFlush, kMoved>;
  constexpr int kSlice = S::kSlice, kSliceChunks = Shape<kMoved>::kChunks, kWarps = Shape<kMoved>::kWarps;
  constexpr int kFlushes = S::kFlushes, kStages = S::kDepth, kRuns = kFlush / 2;  // runs of 8 columns of a lane in a flush
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int wk = warp % sp.along, wr = warp / sp.along;
  const uint32_t base = smem_u32(smem), ring = base + warp * kStages * S::kBytes;
  // sums of x over each flush of this warp's slice, per token
  float* xsum = reinterpret_cast<float*>(smem + kWarps * kStages * S::kBytes) + warp * kFlushes * 8 * kN;
  float4* red = reinterpret_cast<float4*>(smem + kWarps * (kStages * S::kBytes + kFlushes * 8 * kN * 4));
  const uint32_t width = (uint32_t)p.d.input_width, rows = (uint32_t)p.d.output_width, groups = (uint32_t)p.d.groups;
  const uint32_t row_bytes = (uint32_t)p.d.row_bytes;
  const bool wide_x = width % 8 == 0 && ((uintptr_t)p.x & 15u) == 0;

  const int stride = (int)gridDim.x * sp.row_warps;
  int tile = (int)blockIdx.x * sp.row_warps + wr;
  auto slice0 = [&](int pass) { return (uint32_t)(pass * sp.along + wk) * kSlice; };

  // What a lane copies of a tile: codes at row `code_row` (aligned rows: every
  // kCopyRows further down), scale and bias of row `scale_row` and every
  // kScaleRows further down.  Pointers run from tile to tile.
  constexpr int kLanes = S::kRowBytes / 16, kCopyRows = 32 / kLanes, kScaleRows = 32 / kFlushes;
  const uint32_t code_row = lane / kLanes, scale_row = lane / kFlushes, scale_col = lane % kFlushes * (kFlush * 16);
  auto group_of = [&](int pass) { return min((slice0(pass) + scale_col) / p.d.group_size, groups - 1u); };
  uint32_t f_group = group_of(0), f_row = (uint32_t)tile * 16;
  const uint8_t* f_code = p.w + (uint64_t)(f_row + code_row) * row_bytes + 16 * (lane % kLanes);
  uint64_t f_scale = (uint64_t)(f_row + scale_row) * groups;
  const uint64_t code_step = (uint64_t)(16 * stride) * row_bytes, scale_step = (uint64_t)(16 * stride) * groups;
  int f_tile = tile, f_pass = 0;
  uint32_t f_stage = ring;
  auto fetch = [&] {
    if (f_tile < sp.tiles) {
      const uint32_t dst = f_stage, c0 = slice0(f_pass), first = c0 * kBits / 8;
      const bool whole = f_row + 16 <= rows;
      if constexpr (kAligned) {
        if (first + 16 * (lane % kLanes) < row_bytes) {
          const uint8_t* src = f_code + first;
          const uint32_t to = dst + code_row * S::kPitch + 16 * (lane % kLanes);
          if (whole) {
#pragma unroll
            for (int i = 0; i < 16 / kCopyRows; ++i)
              cp_async16(to + i * kCopyRows * S::kPitch, src + (uint64_t)(i * kCopyRows) * row_bytes);
          } else {
            for (int i = 0; i < 16 / kCopyRows; ++i)
              if (f_row + code_row + i * kCopyRows < rows)
                cp_async16(to + i * kCopyRows * S::kPitch, src + (uint64_t)(i * kCopyRows) * row_bytes);
          }
        }
      } else if (c0 < width) {
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
      // scales behind the last column are 0, which takes their columns out
      if (sp.passes > 1) f_group = group_of(f_pass);
      const bool inside = c0 + scale_col < width;
      const float *sc = p.sc + f_scale + f_group, *bi = p.bi + f_scale + f_group;
      const uint32_t sdst = dst + 16 * S::kPitch + lane * 8;
#pragma unroll
      for (int i = 0; i < 16 / kScaleRows; ++i) {
        const bool ok = inside && (whole || f_row + scale_row + i * kScaleRows < rows);
        const uint64_t down = ok ? (uint64_t)(i * kScaleRows) * groups : 0;
        cp_async4(sdst + i * 256, ok ? sc + down : p.sc, ok);
        cp_async4(sdst + i * 256 + 4, ok ? bi + down : p.bi, ok);
      }
      if (++f_pass == sp.passes) {
        f_pass = 0;
        f_tile += stride;
        f_row += 16 * stride;
        f_code += code_step;
        f_scale += scale_step;
      }
    }
    f_stage = f_stage + S::kBytes == ring + kStages * S::kBytes ? ring : f_stage + S::kBytes;
    cp_commit();
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

  uint32_t st = ring;
  for (int done = 0; tile < sp.tiles; ++done) {
    float out[kN][4] = {};
    for (int pass = 0; pass < sp.passes; ++pass) {
      if (sp.passes > 1) load_x(pass);
      cp_wait<kStages - 2>();
      __syncwarp();  // the stage is there, and all lanes have read the one before it,
      fetch();       // which is filled again while this one is used
      const uint32_t c0 = slice0(pass);
      {
        uint32_t addr[2], element[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t row = (uint32_t)tile * 16 + g + 8 * h;
          const uint32_t skew =
              kAligned ? 0u : (uint32_t)((uintptr_t)(p.w + (uint64_t)row * row_bytes) + c0 * kBits / 8) & 15u;
          addr[h] = st + (g + 8 * h) * S::kPitch + skew + t * (kRuns * kBits);
          element[h] = (uint32_t)p.d.element_offset + row * width + c0 + t * (8 * kRuns);
        }
#pragma unroll
        for (int f = 0; f < kFlushes; ++f) {
          float acc[kN][4] = {};
          constexpr int kWords = kRuns * kBits / 4;  // of a lane's columns in a flush
          uint32_t w[2][kWords];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t at = addr[h] + f * (4 * kRuns * kBits);
            if constexpr (kAligned) {
              lds_words<kWords>(at, w[h]);
            } else {
#pragma unroll
              for (int i = 0; i < kWords; ++i) w[h][i] = word_at(at + 4 * i);
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
            const uint32_t sa = st + 16 * S::kPitch + (g * kFlushes + f) * 8;
            uint32_t u[2], v[2];  // (scale, bias) of rows g and g + 8
            lds_words<2>(sa, u);
            lds_words<2>(sa + 64 * kFlushes, v);
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
      st = st + S::kBytes == ring + kStages * S::kBytes ? ring : st + S::kBytes;
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
          const uint32_t row = (uint32_t)tile * 16 + g + 8 * (j >> 1);
          const int tok = n * 8 + 2 * t + (j & 1);
          if (row < rows && tok < p.tokens) p.out[(uint64_t)tok * rows + row] = f32_to_bf16_rne(out[n][j]);
        }
    tile += stride;
  }
  cp_wait<0>();
}

template <int kBits, int kN, int kFlush, bool kMoved, bool kAligned>
int32_t launch_tiles(const Product& p, cudaStream_t s) {
  const auto kernel = packed_tiles_kernel<kBits, kN, kFlush, kMoved, kAligned>;
  Split sp;
  constexpr int kSlice = Shape<kMoved>::kSlice, kWarps = Shape<kMoved>::kWarps;
  const int slices = (int)((p.d.input_width + kSlice - 1) / kSlice);
  sp.along = 1;
  while (sp.along < slices && sp.along < kWarps) sp.along *= 2;
  sp.row_warps = kWarps / sp.along;
  sp.passes = (slices + sp.along - 1) / sp.along;
  sp.tiles = (int)((p.d.output_width + 15) / 16);
  constexpr int smem = smem_bytes<kBits, kN, kFlush, kMoved>();
  static_assert(Shape<kMoved>::kBlocks * (smem + 1024) <= 228 * 1024 && smem <= 227 * 1024, "blocks of an SM");
  static SharedMemorySetup setup;
  int dev = 0;
  int* status = nullptr;
  ENNX_TRY(serving_device(&dev, &status));
  ENNX_TRY(allow_shared_memory(setup, dev, kernel, smem));
  const int blocks = (sp.tiles + sp.row_warps - 1) / sp.row_warps, cap = Shape<kMoved>::kBlocks * sm_count();
  kernel<<<(unsigned)(blocks < cap ? blocks : cap), 32 * kWarps, smem, s>>>(p, sp);
  ENNX_LAUNCH_CHECK("packed tiles");
  return ENNX_B200_OK;
}
template <int kBits, int kN, int kFlush>
int32_t launch_tiles(const Product& p, cudaStream_t s) {
  // moved codes spend their time on the hash: one variant for any alignment
  if (p.seed.enabled) return launch_tiles<kBits, kN, kFlush, true, false>(p, s);
  if (p.d.row_bytes % 16 == 0 && ((uintptr_t)p.w & 15u) == 0) return launch_tiles<kBits, kN, kFlush, false, true>(p, s);
  return launch_tiles<kBits, kN, kFlush, false, false>(p, s);
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

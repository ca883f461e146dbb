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
// shared memory.  Narrow matrices put fewer warps on k and more on rows.
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

__device__ __forceinline__ uint32_t moved_code(uint32_t code, const Product& p, uint32_t element, uint32_t max_code) {
  const uint32_t random = packed_hash(p.seed.low, p.seed.high, element);
  const uint32_t amount = p.d.whole + (uint32_t)((random >> 1) < (p.d.threshold >> 1));
  if (amount == 0u) return code;
  if ((random & 1u) == 0u) return code >= amount ? code - amount : min(code + amount, max_code);
  return code + amount <= max_code ? code + amount : code >= amount ? code - amount : 0u;
}

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
        code = moved_code(code, p, (uint32_t)p.d.element_offset + (uint32_t)row * (uint32_t)p.d.input_width + c, max_code);
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
  const uint64_t blocks = (p.d.output_width + 7) / 8, cap = (uint64_t)sm_count() * 16;
  const unsigned grid = (unsigned)(blocks < cap ? blocks : cap);
  if (tokens == 1) packed_rows_kernel<1><<<grid, 256, 0, s>>>(p);
  else if (tokens <= 4) packed_rows_kernel<4><<<grid, 256, 0, s>>>(p);
  else packed_rows_kernel<kMaxTokens><<<grid, 256, 0, s>>>(p);
  ENNX_LAUNCH_CHECK("packed linear decode");
  return ENNX_B200_OK;
}

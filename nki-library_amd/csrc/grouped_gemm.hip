// Products of the rows of every expert with its weights, with their gradients, and products in 8-bit integers: the C entries and
// the bounds of the experts' rows.  The tiles are in grouped_tile.hip.
//
//   forward   out[s, n]   = sum over k of x[s, k] w[e(s), k, n]
//   backward  dx[s, k]    = sum over n of dout[s, n] w[e(s), k, n]
//             dw[e, k, n] = sum over the rows s of e of x[s, k] dout[s, n]
//   int8      out[s, n]   = xs[s] ws[e(s), n] sum over k of x[s, k] w[e(s), n, k]  (+ bias[n])
//
// Rows row_offsets[e] .. row_offsets[e + 1] are expert e's; rows of no expert come out as zeros, weights of an expert without rows get
// a gradient of zeros.  Sums are taken in 32 bits (int8: whole numbers, exact) and rounded once.
#include "grouped_gemm.hpp"

namespace moe {

// Block i is expert b2e[i]'s, experts ascending: expert e's rows begin with the first block of e or of a later one.  Every block that
// begins an expert writes the bounds that it settles; blocks of no expert stand behind all others.
__global__ __launch_bounds__(256) void expert_row_offsets_kernel(const int32_t* __restrict__ b2e, int64_t N, int64_t B, int E,
                                                                 int32_t* __restrict__ offsets) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i > N) return;
  auto at = [&](int64_t j) {
    const int e = b2e[j];
    return e < 0 || e > E ? E : e;
  };
  const int prev = i == 0 ? -1 : at(i - 1), cur = i == N ? E : at(i);
  for (int e = prev + 1; e <= cur; ++e) offsets[e] = (int32_t)(i * B);
}

}  // namespace moe

using namespace moe;

static constexpr int64_t MAX_COLS = (int64_t)1 << 20;  // of a row: offsets inside a tile stay below 2^31 bytes

static int check_groups(const int32_t* offsets, int64_t S, int64_t K, int64_t N, int64_t E) {
  if (!offsets || S < 0) return MOE_E_BAD_ARG;
  if (K < 1 || N < 1 || K > MAX_COLS || N > MAX_COLS || S >= ((int64_t)1 << 31) - 1024 || E < 1 || E > GG_MAX_GROUPS)
    return MOE_E_BAD_SHAPE;
  return MOE_OK;
}

extern "C" int moe_expert_row_offsets(const int32_t* block_to_expert, int64_t N, int64_t B, int64_t E, int32_t* row_offsets,
                                      void* stream) {
  if ((!block_to_expert && N > 0) || !row_offsets || N < 0) return MOE_E_BAD_ARG;
  if (B < 1 || E < 1 || E > GG_MAX_GROUPS || N >= (int64_t)1 << 31 || B >= (int64_t)1 << 31 || N * B >= (int64_t)1 << 31)
    return MOE_E_BAD_SHAPE;
  hipLaunchKernelGGL(expert_row_offsets_kernel, dim3((unsigned)(N / 256 + 1)), dim3(256), 0, (hipStream_t)stream, block_to_expert, N, B,
                     (int)E, row_offsets);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

extern "C" int moe_grouped_matmul(const void* x, const void* weight, int dtype, const int32_t* row_offsets, int64_t S, int64_t K,
                                  int64_t N, int64_t E, void* out, void* stream) {
  if (!x || !weight || !out || (dtype != MOE_DT_BF16 && dtype != MOE_DT_FP16)) return MOE_E_BAD_ARG;
  const int rc = check_groups(row_offsets, S, K, N, E);
  if (rc != MOE_OK || S == 0) return rc;
  GroupedArgs p{};
  p.a = (const uint8_t*)x, p.b = (const uint8_t*)weight, p.out = (uint8_t*)out, p.offsets = row_offsets;
  p.S = S, p.K = K, p.N = N, p.E = (int)E;
  p.a_pitch = 2 * K, p.b_pitch = 2 * N, p.b_group = 2 * K * N, p.out_pitch = 2 * N;
  p.out_dtype = dtype;
  return dtype == MOE_DT_BF16 ? launch_grouped_bf16(p, (hipStream_t)stream) : launch_grouped_fp16(p, (hipStream_t)stream);
}

extern "C" int moe_grouped_matmul_bwd(const void* d_out, const void* x, const void* weight, int dtype, const int32_t* row_offsets,
                                      int64_t S, int64_t K, int64_t N, int64_t E, void* d_x, void* d_weight, int d_weight_dtype,
                                      void* stream) {
  if (!d_out || (d_x && !weight) || (d_weight && !x) || (!d_x && !d_weight) || (dtype != MOE_DT_BF16 && dtype != MOE_DT_FP16))
    return MOE_E_BAD_ARG;
  if (d_weight && d_weight_dtype != dtype && d_weight_dtype != MOE_DT_FP32) return MOE_E_BAD_ARG;
  const int rc = check_groups(row_offsets, S, K, N, E);
  if (rc != MOE_OK) return rc;
  GroupedArgs px{}, pw{};
  px.offsets = pw.offsets = row_offsets, px.S = pw.S = S, px.E = pw.E = (int)E;
  px.a = (const uint8_t*)d_out, px.b = (const uint8_t*)weight, px.out = (uint8_t*)d_x;
  px.K = N, px.N = K;
  px.a_pitch = px.b_pitch = 2 * N, px.b_group = 2 * K * N, px.out_pitch = 2 * K;
  px.out_dtype = dtype;
  pw.a = (const uint8_t*)x, pw.b = (const uint8_t*)d_out, pw.out = (uint8_t*)d_weight;
  pw.K = K, pw.N = N;
  pw.a_pitch = 2 * K, pw.b_pitch = 2 * N, pw.out_pitch = (d_weight_dtype == MOE_DT_FP32 ? 4 : 2) * N;
  pw.out_dtype = d_weight_dtype;
  const auto launch = dtype == MOE_DT_BF16 ? launch_grouped_bwd_bf16 : launch_grouped_bwd_fp16;
  return launch(d_x ? &px : nullptr, d_weight ? &pw : nullptr, (hipStream_t)stream);
}

extern "C" int moe_int8_matmul(const int8_t* x, const float* x_scales, const int8_t* weight, const float* weight_scales,
                               const void* bias, const int32_t* row_offsets, int64_t S, int64_t K, int64_t N, int64_t E, void* out,
                               int out_dtype, void* stream) {
  if (!x || !x_scales || !weight || !weight_scales || !out || out_dtype < MOE_DT_BF16 || out_dtype > MOE_DT_FP32) return MOE_E_BAD_ARG;
  if (!row_offsets && E != 1) return MOE_E_BAD_ARG;  // (without bounds all rows are one matrix's)
  if (row_offsets && bias) return MOE_E_UNSUPPORTED;
  const int rc = check_groups(row_offsets ? row_offsets : (const int32_t*)x, S, K, N, E);
  if (rc != MOE_OK) return rc;
  if (K >= (int64_t)1 << 17) return MOE_E_BAD_SHAPE;  // (2^14 per product: sums of fewer than 2^17 stay inside 32 bits)
  if (S == 0) return MOE_OK;
  GroupedArgs p{};
  p.a = (const uint8_t*)x, p.b = (const uint8_t*)weight, p.out = (uint8_t*)out, p.offsets = row_offsets;
  p.a_scale = x_scales, p.b_scale = weight_scales, p.bias = bias;
  p.S = S, p.K = K, p.N = N, p.E = (int)E;
  p.a_pitch = K, p.b_pitch = K, p.b_group = K * N, p.out_pitch = (out_dtype == MOE_DT_FP32 ? 4 : 2) * N;
  p.out_dtype = out_dtype;
  return launch_grouped_int8(p, (hipStream_t)stream);
}

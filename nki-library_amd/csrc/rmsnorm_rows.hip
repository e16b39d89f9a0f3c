// Root-mean-square norm with the residual's addition and an output in 8 bits with one scale per row, its gradient, and such rows
// as the values they stand for.
//
//   s = x + r rounded to x's type        (the new residual stream; without a residual s = x)
//   y = s / sqrt(mean of s^2 + eps) * gamma
//   scale = max(max |y|, 2^-100) / M,  code = y * (M / max(max |y|, 2^-100)) rounded to nearest    M = 127 (int8) or 448 (e4m3)
//
//   d_y -> dn = d_y gamma, n = s inv:  d_s = inv (dn - n mean(dn n)) + d_residual,  d_gamma = sum over rows of d_y n
//
// A row is read once and kept in registers; what bounds it is memory.  Sums over a row are taken in 64 bits (they cost a tenth of the
// time that the row's bytes take) and 1 / sqrt is rounded to fp32 once; every other operation is one fp32 operation (no contraction), so
// that a code depends on its row alone, not on the launch.  A row whose y is not finite has the scale NaN and codes 0.
#include "rows.hpp"

#pragma clang fp contract(off)

namespace moe {
namespace {

constexpr int NORM_MAX_H = 16384;
constexpr float LEAST = 7.888609052210118e-31f;  // 2^-100: a row's largest value counts as no less, so that its inverse stays finite

// Rows are dealt to groups of TPR threads (a wave or a workgroup); a thread holds P pieces of N neighbours, piece p from column
// (p * TPR + lane) * N on.
template <int DT>
constexpr int NV = Elem<DT>::N;

template <int DT>
__device__ __forceinline__ u32x4 load_part(const uint8_t* row, int col, int H) {  // piece from col on, zeros behind the row's end
  if (col + NV<DT> <= H) return load_piece<DT>(row + (int64_t)col * Elem<DT>::SIZE);
  u32x4 d = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NV<DT>; ++i)
    if (col + i < H) {
      const uint32_t e = ((const typename Elem<DT>::raw*)row)[col + i];
      if constexpr (Elem<DT>::SIZE == 4) d[i] = e;
      else d[i / 2] |= e << (16 * (i & 1));
    }
  return d;
}
template <int DT>
__device__ __forceinline__ void store_part(uint8_t* row, int col, int H, const u32x4& d) {
  if (col + NV<DT> <= H) {
    store_piece<DT>(row + (int64_t)col * Elem<DT>::SIZE, d);
    return;
  }
#pragma unroll
  for (int i = 0; i < NV<DT>; ++i)
    if (col + i < H) ((typename Elem<DT>::raw*)row)[col + i] = (typename Elem<DT>::raw)(Elem<DT>::SIZE == 4 ? d[i % 4] : d[i / 2] >> (16 * (i & 1)));
}

// gamma of a piece; ones without one (zeros behind the row's end)
template <int DT>
__device__ __forceinline__ void load_gamma(const void* gamma, int dtype, int col, int H, float (&g)[NV<DT>]) {
  if (gamma && dtype == DT && col + NV<DT> <= H) {
    unpack<DT>(load_piece_kept<DT>((const uint8_t*)gamma + (int64_t)col * Elem<DT>::SIZE), g);
    return;
  }
#pragma unroll
  for (int i = 0; i < NV<DT>; ++i) g[i] = col + i < H ? (gamma ? load_as_f32(gamma, dtype, col + i) : 1.f) : 0.f;
}

template <int TPR>
__device__ __forceinline__ double row_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (TPR == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < TPR / 64; ++i) t += red[i];
  return t;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t u = __shfl_xor(v, o, 64);
    v = u > v ? u : v;
  }
  if constexpr (TPR == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t t = red[0];
#pragma unroll
  for (int i = 1; i < TPR / 64; ++i) t = red[i] > t ? red[i] : t;
  return t;
}

struct NormArgs {
  const uint8_t* x;
  const uint8_t* residual;
  const void* gamma;
  uint8_t* codes;
  float* scales;
  uint8_t* out_residual;
  int64_t rows;
  double eps;
  int H, gamma_dtype, do_norm;
};

template <int DT, int TPR, int P, bool E4M3>
__global__ __launch_bounds__(256) void norm_quant_kernel(const NormArgs a) {
  constexpr int N = NV<DT>;
  __shared__ double red_sum[4];
  __shared__ uint32_t red_max[4];
  const int lane = threadIdx.x % TPR, H = a.H;
  const int64_t row_bytes = (int64_t)H * Elem<DT>::SIZE;
  for (int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR; r < a.rows; r += (int64_t)gridDim.x * (256 / TPR)) {
    const uint8_t* x = a.x + r * row_bytes;
    float v[P][N];
    u32x4 d[P], e[P];
#pragma unroll
    for (int p = 0; p < P; ++p) d[p] = load_part<DT>(x, (p * TPR + lane) * N, H);
    if (a.residual) {
#pragma unroll
      for (int p = 0; p < P; ++p) e[p] = load_part<DT>(a.residual + r * row_bytes, (p * TPR + lane) * N, H);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      unpack<DT>(d[p], v[p]);
      if (a.residual) {
        float w[N];
        unpack<DT>(e[p], w);
#pragma unroll
        for (int i = 0; i < N; ++i) v[p][i] = v[p][i] + w[i];
        const u32x4 s = pack<DT>(v[p]);
        store_part<DT>(a.out_residual + r * row_bytes, (p * TPR + lane) * N, H, s);
        unpack<DT>(s, v[p]);
      }
    }
    if (a.do_norm) {
      double sum = 0.0;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < N; ++i) sum = __builtin_fma((double)v[p][i], (double)v[p][i], sum);
      sum = row_sum<TPR>(sum, red_sum);
      const float inv = (float)(1.0 / sqrt(sum / H + a.eps));
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float g[N];
        load_gamma<DT>(a.gamma, a.gamma_dtype, (p * TPR + lane) * N, H, g);
#pragma unroll
        for (int i = 0; i < N; ++i) v[p][i] = v[p][i] * inv * g[i];
      }
    }
    uint32_t most = 0;  // (magnitudes in the order of their bits: infinities and NaN above all numbers)
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t b = (p * TPR + lane) * N + i < H ? __float_as_uint(v[p][i]) & 0x7fffffffu : 0u;
        most = b > most ? b : most;
      }
    most = row_max<TPR>(most, red_max);
    const bool finite = most < 0x7f800000u;
    const float largest = fmaxf(__uint_as_float(most), LEAST);
    constexpr float M = E4M3 ? 448.0f : 127.0f;
    const float q = M / largest;
    if (lane == 0) a.scales[r] = finite ? largest / M : __uint_as_float(0x7fc00000u);
    uint8_t* codes = a.codes + r * H;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      uint32_t c[N / 4];
#pragma unroll
      for (int w = 0; w < N / 4; ++w) {
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = finite ? v[p][4 * w + i] * q : 0.f;
        if constexpr (E4M3) {
          c[w] = pack4_e4m3(clip448(t[0]), clip448(t[1]), clip448(t[2]), clip448(t[3]));
        } else {
          c[w] = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) c[w] |= ((uint32_t)(int)rintf(t[i]) & 0xffu) << (8 * i);
        }
      }
      const int col = (p * TPR + lane) * N;
      if (col + N <= H) {
        typedef uint32_t part_t __attribute__((ext_vector_type(N / 4), aligned(1)));
        part_t o;
        if constexpr (N == 4) o = c[0];
        else o = part_t{c[0], c[1]};
        __builtin_nontemporal_store(o, (part_t*)(codes + col));
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (col + i < H) codes[col + i] = (uint8_t)(c[i / 4] >> (8 * (i & 3)));
      }
    }
  }
}

struct NormBwdArgs {
  const uint8_t* d_y;
  const uint8_t* x;
  const void* gamma;
  const uint8_t* d_residual;
  uint8_t* d_x;
  float* parts;  // [gridDim.x][H]
  int64_t rows;
  double eps;
  int H, gamma_dtype;
};
// A workgroup takes every gridDim.x-th row; a thread has the same columns in all of them and adds up their d_gamma in registers.
template <int DT, int P>
__global__ __launch_bounds__(256) void norm_bwd_kernel(const NormBwdArgs a) {
  constexpr int N = NV<DT>;
  __shared__ double red[8];
  const int H = a.H, tid = threadIdx.x;
  const int64_t row_bytes = (int64_t)H * Elem<DT>::SIZE;
  float dg[P][N], gm[P][N];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    load_gamma<DT>(a.gamma, a.gamma_dtype, (p * 256 + tid) * N, H, gm[p]);
#pragma unroll
    for (int i = 0; i < N; ++i) dg[p][i] = 0.f;
  }
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    u32x4 xs[P], ds[P], rs[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      xs[p] = load_part<DT>(a.x + r * row_bytes, (p * 256 + tid) * N, H);
      ds[p] = load_part<DT>(a.d_y + r * row_bytes, (p * 256 + tid) * N, H);
    }
    if (a.d_residual) {
#pragma unroll
      for (int p = 0; p < P; ++p) rs[p] = load_part<DT>(a.d_residual + r * row_bytes, (p * 256 + tid) * N, H);
    }
    double sx = 0.0, sd = 0.0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float x[N], d[N];
      unpack<DT>(xs[p], x);
      unpack<DT>(ds[p], d);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        sx = __builtin_fma((double)x[i], (double)x[i], sx);
        sd = __builtin_fma((double)x[i], (double)(d[i] * gm[p][i]), sd);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      sx += __shfl_xor(sx, o, 64);
      sd += __shfl_xor(sd, o, 64);
    }
    __syncthreads();
    if ((tid & 63) == 0) {
      red[tid >> 6] = sx;
      red[4 + (tid >> 6)] = sd;
    }
    __syncthreads();
    sx = (red[0] + red[1]) + (red[2] + red[3]);
    sd = (red[4] + red[5]) + (red[6] + red[7]);
    const double inv64 = 1.0 / sqrt(sx / H + a.eps);
    const float inv = (float)inv64, mean = (float)(sd * inv64 / H);  // mean of dn n
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float x[N], d[N], o[N];
      unpack<DT>(xs[p], x);
      unpack<DT>(ds[p], d);
      if (a.d_residual) unpack<DT>(rs[p], o);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float n = x[i] * inv;
        dg[p][i] += d[i] * n;
        const float s = (d[i] * gm[p][i] - n * mean) * inv;
        o[i] = a.d_residual ? s + o[i] : s;
      }
      store_part<DT>(a.d_x + r * row_bytes, (p * 256 + tid) * N, H, pack<DT>(o));
    }
  }
  if (!a.parts) return;
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int col = (p * 256 + tid) * N + i;
      if (col < H) a.parts[(int64_t)blockIdx.x * H + col] = dg[p][i];
    }
}
// d_gamma: 64 columns a workgroup, the parts' sums in 64 bits.
template <int DT>
__global__ __launch_bounds__(1024) void norm_parts_kernel(const float* __restrict__ parts, int n, int H, uint8_t* __restrict__ d_gamma) {
  __shared__ double s[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  double t = 0.0;
  if (col < H)
    for (int i = w; i < n; i += 16) t += parts[(int64_t)i * H + col];
  s[w][threadIdx.x & 63] = t;
  __syncthreads();
  if (w == 0 && col < H) {
#pragma unroll
    for (int i = 1; i < 16; ++i) t += s[i][threadIdx.x];
    ((typename Elem<DT>::raw*)d_gamma)[col] = f32_to_elem<DT>((float)t);
  }
}

// 16 codes a thread.
template <int DT, bool E4M3>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, int64_t rows,
                                                              int H, uint8_t* __restrict__ out) {
  typedef uint32_t bytes16 __attribute__((ext_vector_type(4), aligned(1)));
  const int col = (blockIdx.y * 256 + threadIdx.x) * 16;
  if (col >= H) return;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float s = scales[r];
    const uint8_t* src = codes + r * H + col;
    uint32_t c[4] = {0, 0, 0, 0};
    const int left = H - col;
    if (left >= 16) {
      const bytes16 d = __builtin_nontemporal_load((const bytes16*)src);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = d[i];
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < left) c[i / 4] |= (uint32_t)src[i] << (8 * (i & 3));
    }
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t b = (c[i / 4] >> (8 * (i & 3))) & 0xffu;
      if constexpr (E4M3) v[i] = ((b & 0x7f) == 0x7f ? __uint_as_float(0x7fc00000u) : e4m3_to_f32(b)) * s;
      else v[i] = (float)(int)(int8_t)b * s;
    }
    uint8_t* row = out + r * H * Elem<DT>::SIZE;
    constexpr int N = NV<DT>;
#pragma unroll
    for (int p = 0; p < 16 / N; ++p) {
      float w[N];
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = v[p * N + i];
      store_part<DT>(row, col + p * N, H, pack<DT>(w));
    }
  }
}

template <int DT, bool E4M3>
void launch_norm(const NormArgs& a, hipStream_t s) {
  constexpr int N = NV<DT>;
  // a wave per row where that leaves a thread at most 4 pieces and the rows fill the chip, else a workgroup
  const bool wave = a.H <= 64 * N * 4 && a.rows >= 2048;
  const int64_t groups = wave ? (a.rows + 3) / 4 : a.rows;
  const dim3 grid((unsigned)(groups < 1 << 20 ? groups : 1 << 20));
  const int per = wave ? 64 * N : 256 * N, pieces = (a.H + per - 1) / per;
#define MOE_NORM(TPR, P) hipLaunchKernelGGL((norm_quant_kernel<DT, TPR, P, E4M3>), grid, dim3(256), 0, s, a)
  if (wave) {
    if (pieces <= 1) MOE_NORM(64, 1);
    else if (pieces <= 2) MOE_NORM(64, 2);
    else MOE_NORM(64, 4);
  } else {
    if (pieces <= 1) MOE_NORM(256, 1);
    else if (pieces <= 2) MOE_NORM(256, 2);
    else if (pieces <= 4) MOE_NORM(256, 4);
    else if (pieces <= 8) MOE_NORM(256, 8);
    else if constexpr (N == 4) MOE_NORM(256, 16);
  }
#undef MOE_NORM
}
template <int DT>
void launch_norm_bwd(const NormBwdArgs& a, int groups, hipStream_t s) {
  const int per = 256 * NV<DT>, pieces = (a.H + per - 1) / per;
#define MOE_NORM(P) hipLaunchKernelGGL((norm_bwd_kernel<DT, P>), dim3(groups), dim3(256), 0, s, a)
  if (pieces <= 1) MOE_NORM(1);
  else if (pieces <= 2) MOE_NORM(2);
  else if (pieces <= 4) MOE_NORM(4);
  else if (pieces <= 8) MOE_NORM(8);
  else if constexpr (NV<DT> == 4) MOE_NORM(16);
#undef MOE_NORM
}
// Workgroups of the gradient: as many as run at once, and no more parts of d_gamma than that.
int bwd_groups(int64_t rows) { return (int)(rows < 1024 ? rows : 1024); }

bool row_dtype(int d) { return d == MOE_DT_BF16 || d == MOE_DT_FP16 || d == MOE_DT_FP32; }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_rmsnorm_quant_rows(const void* x, int dtype, const void* residual, const void* gamma, int gamma_dtype, int do_norm,
                                      double eps, int64_t rows, int64_t H, int code_dtype, void* codes, float* scales,
                                      void* out_residual, void* stream) {
  if (!x || !codes || !scales || rows < 0 || !row_dtype(dtype) || (gamma && !row_dtype(gamma_dtype)) || !(eps >= 0)) return MOE_E_BAD_ARG;
  if ((residual != nullptr) != (out_residual != nullptr) || (code_dtype != MOE_DT_INT8 && code_dtype != MOE_DT_FP8_E4M3)) return MOE_E_BAD_ARG;
  if (H < 1 || H > NORM_MAX_H || rows >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  if (rows == 0) return MOE_OK;
  const NormArgs a{(const uint8_t*)x, (const uint8_t*)residual, gamma, (uint8_t*)codes, scales, (uint8_t*)out_residual, rows, eps, (int)H,
                   gamma_dtype, do_norm};
  const hipStream_t s = (hipStream_t)stream;
#define MOE_NORM(DT)                                            \
  if (code_dtype == MOE_DT_INT8) launch_norm<DT, false>(a, s);  \
  else launch_norm<DT, true>(a, s)
  if (dtype == MOE_DT_BF16) {
    MOE_NORM(MOE_DT_BF16);
  } else if (dtype == MOE_DT_FP16) {
    MOE_NORM(MOE_DT_FP16);
  } else {
    MOE_NORM(MOE_DT_FP32);
  }
#undef MOE_NORM
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

extern "C" size_t moe_rmsnorm_quant_rows_bwd_workspace_bytes(int64_t rows, int64_t H) {
  if (rows < 1 || H < 1 || H > NORM_MAX_H || rows >= (int64_t)1 << 31) return 0;
  return (size_t)bwd_groups(rows) * H * sizeof(float);
}

extern "C" int moe_rmsnorm_quant_rows_bwd(const void* d_y, const void* x, int dtype, const void* gamma, int gamma_dtype,
                                          const void* d_residual, double eps, int64_t rows, int64_t H, void* d_x, void* d_gamma,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!d_y || !x || !d_x || rows < 0 || !row_dtype(dtype) || (gamma && !row_dtype(gamma_dtype)) || !(eps >= 0)) return MOE_E_BAD_ARG;
  if (d_gamma && !gamma) return MOE_E_BAD_ARG;
  if (H < 1 || H > NORM_MAX_H || rows < 1 || rows >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  if (d_gamma && (!workspace || workspace_bytes < moe_rmsnorm_quant_rows_bwd_workspace_bytes(rows, H))) return MOE_E_WORKSPACE;
  if (d_gamma && ((uintptr_t)workspace & 3)) return MOE_E_BAD_ARG;
  const int groups = bwd_groups(rows);
  const NormBwdArgs a{(const uint8_t*)d_y, (const uint8_t*)x, gamma, (const uint8_t*)d_residual, (uint8_t*)d_x,
                      d_gamma ? (float*)workspace : nullptr, rows, eps, (int)H, gamma_dtype};
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == MOE_DT_BF16) launch_norm_bwd<MOE_DT_BF16>(a, groups, s);
  else if (dtype == MOE_DT_FP16) launch_norm_bwd<MOE_DT_FP16>(a, groups, s);
  else launch_norm_bwd<MOE_DT_FP32>(a, groups, s);
  MOE_CHECK_LAUNCH();
  if (!d_gamma) return MOE_OK;
  const dim3 grid((unsigned)((H + 63) / 64));
  if (gamma_dtype == MOE_DT_BF16)
    hipLaunchKernelGGL(norm_parts_kernel<MOE_DT_BF16>, grid, dim3(1024), 0, s, a.parts, groups, (int)H, (uint8_t*)d_gamma);
  else if (gamma_dtype == MOE_DT_FP16)
    hipLaunchKernelGGL(norm_parts_kernel<MOE_DT_FP16>, grid, dim3(1024), 0, s, a.parts, groups, (int)H, (uint8_t*)d_gamma);
  else
    hipLaunchKernelGGL(norm_parts_kernel<MOE_DT_FP32>, grid, dim3(1024), 0, s, a.parts, groups, (int)H, (uint8_t*)d_gamma);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

extern "C" int moe_dequantize_rows(const void* codes, int code_dtype, const float* scales, int64_t rows, int64_t H, void* out, int dtype,
                                   void* stream) {
  if (!codes || !scales || !out || rows < 0 || !row_dtype(dtype) || (code_dtype != MOE_DT_INT8 && code_dtype != MOE_DT_FP8_E4M3))
    return MOE_E_BAD_ARG;
  if (H < 1 || H >= (int64_t)1 << 24 || rows >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  if (rows == 0) return MOE_OK;
  const dim3 grid((unsigned)(rows < 1 << 20 ? rows : 1 << 20), (unsigned)((H + 4095) / 4096));
  const hipStream_t s = (hipStream_t)stream;
#define MOE_DEQ(DT)                                                                                                               \
  do {                                                                                                                            \
    if (code_dtype == MOE_DT_INT8)                                                                                                \
      hipLaunchKernelGGL((dequantize_rows_kernel<DT, false>), grid, dim3(256), 0, s, (const uint8_t*)codes, scales, rows, (int)H, \
                         (uint8_t*)out);                                                                                          \
    else                                                                                                                          \
      hipLaunchKernelGGL((dequantize_rows_kernel<DT, true>), grid, dim3(256), 0, s, (const uint8_t*)codes, scales, rows, (int)H,  \
                         (uint8_t*)out);                                                                                          \
  } while (0)
  if (dtype == MOE_DT_BF16) MOE_DEQ(MOE_DT_BF16);
  else if (dtype == MOE_DT_FP16) MOE_DEQ(MOE_DT_FP16);
  else MOE_DEQ(MOE_DT_FP32);
#undef MOE_DEQ
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

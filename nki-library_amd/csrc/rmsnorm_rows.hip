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
// time that the row's bytes take), in an order that is the row's (row_sum), and 1 / sqrt is rounded to fp32 once; every other operation
// is one fp32 operation (no contraction), so that a code depends on its row alone, not on the launch.  A row whose y is not finite has
// the scale NaN and codes 0.
#include <type_traits>

#include "rows.hpp"

#pragma clang fp contract(off)

namespace moe {
namespace {

constexpr int NORM_MAX_H = 16384;
constexpr float LEAST = 7.888609052210118e-31f;  // 2^-100: a row's largest value counts as no less, so that its inverse stays finite

// Rows are dealt to groups of TPR threads (a wave or a workgroup); a thread holds P pieces of N neighbours, piece p from column
// (p * TPR + lane) * N on.  WHOLE: rows are whole pieces; a thread beyond the last one loads that and takes zeros.
template <int DT>
constexpr int NV = Elem<DT>::N;

template <int DT, bool WHOLE>
__device__ __forceinline__ u32x4 load_part(const uint8_t* row, int col, int H) {  // piece from col on, zeros behind the row's end
  if constexpr (WHOLE) {
    const u32x4 d = load_piece<DT>(row + (int64_t)(col < H ? col : H - NV<DT>) * Elem<DT>::SIZE);
    const uint32_t keep = col < H ? ~0u : 0u;
    return u32x4{d[0] & keep, d[1] & keep, d[2] & keep, d[3] & keep};
  }
  if (H >= NV<DT>) {  // a piece that passes the row's end: the row's last one, moved down
    const int from = col <= H - NV<DT> ? col : H - NV<DT>, gone = 8 * Elem<DT>::SIZE * (col - from);
    const u32x4 d = load_piece<DT>(row + (int64_t)from * Elem<DT>::SIZE);
    uint64_t lo = (uint64_t)d[1] << 32 | d[0], hi = (uint64_t)d[3] << 32 | d[2];
    if (gone >= 64) {
      lo = gone < 128 ? hi >> (gone - 64) : 0;
      hi = 0;
    } else if (gone > 0) {
      lo = lo >> gone | hi << (64 - gone);
      hi >>= gone;
    }
    return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
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
template <int DT, bool WHOLE>
__device__ __forceinline__ void store_part(uint8_t* row, int col, int H, const u32x4& d) {
  if (col + NV<DT> <= H) {
    store_piece<DT>(row + (int64_t)col * Elem<DT>::SIZE, d);
    return;
  }
  if constexpr (!WHOLE) {
#pragma unroll
    for (int i = 0; i < NV<DT>; ++i)
      if (col + i < H)
        ((typename Elem<DT>::raw*)row)[col + i] = (typename Elem<DT>::raw)(Elem<DT>::SIZE == 4 ? d[i % 4] : d[i / 2] >> (16 * (i & 1)));
  }
}

// gamma of a piece; ones without one (zeros behind the row's end)
template <int DT, bool WHOLE>
__device__ __forceinline__ void load_gamma(const void* gamma, int dtype, int col, int H, float (&g)[NV<DT>]) {
  if (gamma && dtype == DT && (WHOLE || col + NV<DT> <= H)) {
    unpack<DT>(load_piece_kept<DT>((const uint8_t*)gamma + (int64_t)(col < H ? col : 0) * Elem<DT>::SIZE), g);
    return;
  }
#pragma unroll
  for (int i = 0; i < NV<DT>; ++i) g[i] = col + i < H ? (gamma ? load_as_f32(gamma, dtype, col + i) : 1.f) : 0.f;
}

// Sum and maximum over a wave, the same bits in all lanes: sixteen lanes by rotations (every lane adds the same pairs), then the four
// sixteens through scalar registers.  (Shuffles go through LDS, six of them in a row were a third of a short row's time.)
template <int N>
__device__ __forceinline__ uint32_t turned(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, true);  // row_ror:N
}
template <int N>
__device__ __forceinline__ double turned(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)turned<N>((uint32_t)(b >> 32)) << 32 | turned<N>((uint32_t)b));
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double sum_of_wave(double v) {
  v += turned<8>(v);
  v += turned<4>(v);
  v += turned<2>(v);
  v += turned<1>(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
__device__ __forceinline__ uint32_t max_of_wave(uint32_t v) {
  auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  v = larger(v, turned<8>(v));
  v = larger(v, turned<4>(v));
  v = larger(v, turned<2>(v));
  v = larger(v, turned<1>(v));
  const uint32_t a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = __builtin_amdgcn_readlane((int)v, 32), d = __builtin_amdgcn_readlane((int)v, 48);
  return larger(larger(a, b), larger(c, d));
}
// Sum over a row of what its threads have of its pieces, P each.  A row of up to 256 pieces may be a wave's (up to four pieces a thread) or
// a workgroup's (one): wave w's threads then have what the wave's have as piece w.  Either adds the four numbers of a lane first and the
// lanes then, so that the sum is the row's alone.  (A wave's sum of every piece by itself cost 7 % with the residual, 16384 rows of 2048 bf16.)
// One barrier here and in the maximum: `red` is a place of its own for every reduction between two others.
template <int TPR, int P>
__device__ __forceinline__ double row_sum(const double (&v)[P], double* red) {
  double t = v[0];
  if constexpr (TPR == 256 && P == 1) {
    red[threadIdx.x] = t;
    __syncthreads();
    t = red[threadIdx.x & 63];
#pragma unroll
    for (int i = 1; i < 4; ++i) t += red[64 * i + (threadIdx.x & 63)];
    return sum_of_wave(t);
  }
#pragma unroll
  for (int p = 1; p < P; ++p) t += v[p];
  t = sum_of_wave(t);
  if constexpr (TPR == 64) return t;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
  __syncthreads();
  return ((red[0] + red[1]) + red[2]) + red[3];
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* red) {
  v = max_of_wave(v);
  if constexpr (TPR == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t t = red[0];
#pragma unroll
  for (int i = 1; i < TPR / 64; ++i) t = red[i] > t ? red[i] : t;
  return t;
}

// 1 / sqrt(mean + eps), rounded once, is no normal float where a row's values are denormal (it passes the largest float) or near the
// largest (it is denormal itself).  Then: the power of two that brings it back among the normal ones, by which it is divided and the
// row's values are multiplied, which is exact for all that are of weight.  (fp16 does not reach either end.)  A branch of its own, which
// hardly a row takes: with a product by 1 in the others 16384 rows of 7168 fp32 take 171 us instead of 137, the gradient of 65536 rows of
// 1024 bf16 147 instead of 141.
__device__ __forceinline__ float far_factor(double inv, float& inv32) {
  const float far = inv > 1.0 ? 0x1p64f : inv <= 1.0 ? 0x1p-64f : 1.f;
  inv32 = (float)(inv / far);
  return far;
}
template <int DT>
__device__ __forceinline__ bool is_far(float inv) {
  return DT != MOE_DT_FP16 && !__builtin_isnormal(inv);
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

template <int DT, int TPR, int P, bool WHOLE, bool E4M3>
__global__ __launch_bounds__(256) void norm_quant_kernel(const NormArgs a) {
  constexpr int N = NV<DT>;
  __shared__ double red_sum[P == 1 ? 256 : 4];
  __shared__ uint32_t red_max[2][4];
  int turn = 0;
  const int lane = threadIdx.x % TPR, H = a.H;
  const int64_t row_bytes = (int64_t)H * Elem<DT>::SIZE;
  for (int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR; r < a.rows; r += (int64_t)gridDim.x * (256 / TPR)) {
    const uint8_t* x = a.x + r * row_bytes;
    float v[P][N];
    u32x4 d[P], e[P];
#pragma unroll
    for (int p = 0; p < P; ++p) d[p] = load_part<DT, WHOLE>(x, (p * TPR + lane) * N, H);
    if (a.residual) {
#pragma unroll
      for (int p = 0; p < P; ++p) e[p] = load_part<DT, WHOLE>(a.residual + r * row_bytes, (p * TPR + lane) * N, H);
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
        store_part<DT, WHOLE>(a.out_residual + r * row_bytes, (p * TPR + lane) * N, H, s);
        unpack<DT>(s, v[p]);
      }
    }
    if (a.do_norm) {
      double part[P];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        part[p] = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) part[p] = __builtin_fma((double)v[p][i], (double)v[p][i], part[p]);
      }
      const double sum = row_sum<TPR, P>(part, red_sum);
      const double inv64 = 1.0 / sqrt(sum / H + a.eps);
      float inv = (float)inv64;
      if (is_far<DT>(inv)) [[unlikely]] {
        const float far = far_factor(inv64, inv);
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < N; ++i) v[p][i] = v[p][i] * far;
      }
      // (The lane is taken anew: the addresses of gamma's elements would otherwise be worked out ahead of the first row and kept.  16384 rows
      // of 7168 bf16: 256 registers and 136 us, or 120 and 92.)
      int at = lane;
      asm volatile("" : "+v"(at));
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float g[N];
        load_gamma<DT, WHOLE>(a.gamma, a.gamma_dtype, (p * TPR + at) * N, H, g);
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
    most = row_max<TPR>(most, red_max[turn]);
    turn ^= 1;  // (without the norm the next barrier is the next row's maximum)
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
      } else if constexpr (!WHOLE) {
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
// A workgroup has SUB rows at a time, 256 threads each; a thread has the same columns in all of its rows and adds up their d_gamma in
// registers.  The SUB sums are added in LDS, so that there are few parts to be read again.
template <int DT, int P, int SUB, bool WHOLE>
__global__ __launch_bounds__(SUB * 256) void norm_bwd_kernel(const NormBwdArgs a) {
  constexpr int N = NV<DT>;
  __shared__ double red[2][2][4 * SUB];
  extern __shared__ float s_dg[];  // [H]; with SUB > 1
  const int H = a.H, sub = threadIdx.x / 256, tid = threadIdx.x % 256;
  const int64_t row_bytes = (int64_t)H * Elem<DT>::SIZE;
  float dg[P][N], gm[P][N];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    load_gamma<DT, WHOLE>(a.gamma, a.gamma_dtype, (p * 256 + tid) * N, H, gm[p]);
#pragma unroll
    for (int i = 0; i < N; ++i) dg[p][i] = 0.f;
  }
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * SUB; r0 < a.rows; r0 += (int64_t)gridDim.x * SUB) {
    const bool on = r0 + sub < a.rows;  // (the last round's threads beyond work on the last row and write nothing)
    const int64_t r = on ? r0 + sub : a.rows - 1;
    u32x4 xs[P], ds[P], rs[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      xs[p] = load_part<DT, WHOLE>(a.x + r * row_bytes, (p * 256 + tid) * N, H);
      ds[p] = load_part<DT, WHOLE>(a.d_y + r * row_bytes, (p * 256 + tid) * N, H);
    }
    if (a.d_residual) {
#pragma unroll
      for (int p = 0; p < P; ++p) rs[p] = load_part<DT, WHOLE>(a.d_residual + r * row_bytes, (p * 256 + tid) * N, H);
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
    sx = sum_of_wave(sx);
    sd = sum_of_wave(sd);
    if ((tid & 63) == 0) {
      red[turn][0][threadIdx.x >> 6] = sx;
      red[turn][1][threadIdx.x >> 6] = sd;
    }
    __syncthreads();
    const double* const rx = red[turn][0] + 4 * sub;
    const double* const rd = red[turn][1] + 4 * sub;
    turn ^= 1;
    sx = (rx[0] + rx[1]) + (rx[2] + rx[3]);
    sd = (rd[0] + rd[1]) + (rd[2] + rd[3]);
    const double inv64 = 1.0 / sqrt(sx / H + a.eps);
    const float mean = (float)(sd * inv64 / H);  // mean of dn n
    auto finish = [&](float inv, float far, auto use_far) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float x[N], d[N], o[N];
        unpack<DT>(xs[p], x);
        unpack<DT>(ds[p], d);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (use_far) x[i] = x[i] * far;
          const float n = x[i] * inv;
          dg[p][i] += d[i] * n;
          o[i] = (d[i] * gm[p][i] - n * mean) * inv;
          if (use_far) o[i] = o[i] * far;
        }
        if (a.d_residual) {
          float r[N];
          unpack<DT>(rs[p], r);
#pragma unroll
          for (int i = 0; i < N; ++i) o[i] = o[i] + r[i];
        }
        store_part<DT, WHOLE>(a.d_x + r * row_bytes, (p * 256 + tid) * N, H, pack<DT>(o));
      }
    };
    if (on) {
      float inv = (float)inv64;
      if (is_far<DT>(inv)) [[unlikely]] {
        const float far = far_factor(inv64, inv);
        finish(inv, far, std::true_type{});
      } else {
        finish(inv, 1.f, std::false_type{});
      }
    }
  }
  if (!a.parts) return;
  for (int part = 0; part < SUB; ++part) {
    if (sub == part) {
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int col = (p * 256 + tid) * N + i;
          if (col < H) {
            const float t = part == 0 ? dg[p][i] : s_dg[col] + dg[p][i];
            if (part + 1 < SUB) s_dg[col] = t;
            else a.parts[(int64_t)blockIdx.x * H + col] = t;
          }
        }
    }
    if constexpr (SUB > 1) __syncthreads();
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

// A piece of the result, from 8 or 4 codes, of four rows a thread and round.  (8192 x 7168 int8 to bf16 in us: 33; 16 codes a thread,
// whose two stores fill every other 16 bytes of a line each, 65.)
template <int DT, bool E4M3>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, int64_t rows,
                                                              int H, uint8_t* __restrict__ out) {
  constexpr int U = 4, N = NV<DT>;
  typedef uint32_t part_t __attribute__((ext_vector_type(N / 4), aligned(1)));
  const int col = (blockIdx.y * 256 + threadIdx.x) * N, left = H - col;
  if (left <= 0) return;
  for (int64_t r0 = (int64_t)blockIdx.x * U; r0 < rows; r0 += (int64_t)gridDim.x * U) {
    uint64_t c[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u < rows ? r0 + u : rows - 1;
      const uint8_t* src = codes + r * H + col;
      s[u] = scales[r];
      c[u] = 0;
      if (H >= N) {  // (the last piece of a row that is not whole: the row's last codes, moved down)
        const int gone = left < N ? N - left : 0;
        const part_t d = __builtin_nontemporal_load((const part_t*)(src - gone));
        if constexpr (N == 8) c[u] = ((uint64_t)d[1] << 32 | d[0]) >> (8 * gone);
        else c[u] = d[0] >> (8 * gone);
      } else {
        for (int i = 0; i < left; ++i) c[u] |= (uint64_t)src[i] << (8 * i);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u >= rows) break;
      float w[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t b = (uint32_t)(c[u] >> (8 * i)) & 0xffu;
        if constexpr (E4M3) w[i] = ((b & 0x7f) == 0x7f ? __uint_as_float(0x7fc00000u) : e4m3_to_f32(b)) * s[u];
        else w[i] = (float)(int)(int8_t)b * s[u];
      }
      store_part<DT, false>(out + (r0 + u) * H * Elem<DT>::SIZE, col, H, pack<DT>(w));
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
  const bool whole = a.H % N == 0;
#define MOE_NORM(TPR, P)                                                                                            \
  do {                                                                                                              \
    if (whole) hipLaunchKernelGGL((norm_quant_kernel<DT, TPR, P, true, E4M3>), grid, dim3(256), 0, s, a);           \
    else hipLaunchKernelGGL((norm_quant_kernel<DT, TPR, P, false, E4M3>), grid, dim3(256), 0, s, a);                \
  } while (0)
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
// Rows that a workgroup of the gradient has at a time: what a thread holds of each has to fit its registers (128 with four rows, 256 with
// two).
constexpr int bwd_sub(int pieces) { return pieces <= 2 ? 4 : pieces <= 4 ? 2 : 1; }
int bwd_sub_of(int dtype, int64_t H) {
  const int n = dtype == MOE_DT_FP32 ? 4 : 8;
  return bwd_sub((int)((H + 256 * n - 1) / (256 * n)));
}
// ... and workgroups: two per CU, one of four rows; a part of d_gamma each.
int bwd_groups(int64_t rows, int sub) {
  const int64_t n = (rows + sub - 1) / sub, most = sub == 4 ? 256 : 512;
  return (int)(n < most ? n : most);
}
template <int DT, bool WHOLE>
void launch_norm_bwd(const NormBwdArgs& a, hipStream_t s) {
  const int per = 256 * NV<DT>, pieces = (a.H + per - 1) / per, sub = bwd_sub(pieces), groups = bwd_groups(a.rows, sub);
#define MOE_NORM(P)                                                                                                          \
  hipLaunchKernelGGL((norm_bwd_kernel<DT, P, bwd_sub(P), WHOLE>), dim3(groups), dim3(sub * 256),                         \
                     bwd_sub(P) > 1 && a.parts ? a.H * sizeof(float) : 0, s, a)
  if (pieces <= 1) MOE_NORM(1);
  else if (pieces <= 2) MOE_NORM(2);
  else if (pieces <= 4) MOE_NORM(4);
  else if (pieces <= 8) MOE_NORM(8);
  else if constexpr (NV<DT> == 4) MOE_NORM(16);
#undef MOE_NORM
}

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
  return (size_t)bwd_groups(rows, 1) * H * sizeof(float);  // (512 parts at most, whatever the type)
}

extern "C" int moe_rmsnorm_quant_rows_bwd(const void* d_y, const void* x, int dtype, const void* gamma, int gamma_dtype,
                                          const void* d_residual, double eps, int64_t rows, int64_t H, void* d_x, void* d_gamma,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!d_y || !x || !d_x || rows < 0 || !row_dtype(dtype) || (gamma && !row_dtype(gamma_dtype)) || !(eps >= 0)) return MOE_E_BAD_ARG;
  if (d_gamma && !gamma) return MOE_E_BAD_ARG;
  if (H < 1 || H > NORM_MAX_H || rows < 1 || rows >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  if (d_gamma && (!workspace || workspace_bytes < moe_rmsnorm_quant_rows_bwd_workspace_bytes(rows, H))) return MOE_E_WORKSPACE;
  if (d_gamma && ((uintptr_t)workspace & 3)) return MOE_E_BAD_ARG;
  const int groups = bwd_groups(rows, bwd_sub_of(dtype, H));
  const NormBwdArgs a{(const uint8_t*)d_y, (const uint8_t*)x, gamma, (const uint8_t*)d_residual, (uint8_t*)d_x,
                      d_gamma ? (float*)workspace : nullptr, rows, eps, (int)H, gamma_dtype};
  const hipStream_t s = (hipStream_t)stream;
#define MOE_NORM(DT)                                                   \
  if (H % NV<DT> == 0) launch_norm_bwd<DT, true>(a, s);                \
  else launch_norm_bwd<DT, false>(a, s)
  if (dtype == MOE_DT_BF16) {
    MOE_NORM(MOE_DT_BF16);
  } else if (dtype == MOE_DT_FP16) {
    MOE_NORM(MOE_DT_FP16);
  } else {
    MOE_NORM(MOE_DT_FP32);
  }
#undef MOE_NORM
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
  const int64_t fours = (rows + 3) / 4;
  const int per = 256 * (dtype == MOE_DT_FP32 ? 4 : 8);  // columns of a workgroup
  const dim3 grid((unsigned)(fours < 1 << 20 ? fours : 1 << 20), (unsigned)((H + per - 1) / per));
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

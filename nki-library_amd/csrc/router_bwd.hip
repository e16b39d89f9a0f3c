// Gradient of the router (router_topk.hip): from the gradient g of the affinities to those of the logits, the hidden states, the
// weights and the bias.
//
//   softmax over the chosen (also: over all, divided by the chosen's sum, which is the same)   dl_j = a_j (g_j - sum g a)
//   softmax over all                                                                          dl_e = p_e (g_e - sum g p)
//   sigmoid                                                                                   dl_j = g_j s_j (1 - s_j)
//   sigmoid, divided by the chosen's sum S        dl_j = (g_j - sum g a) / S  s_j (1 - s_j),  a_j = s_j / S
//   dx = dl w^T    dw = x^T dl    db = sum over the tokens of dl
//
// Everything up to dl is fp32.  The two products run on bf16 MFMAs with dl as the sum of two bf16 (hi + lo, 2^-17 of the value): a
// softmax's dl sum to zero over the experts, and a single bf16 (2^-8) would leave that much of every term where the terms
// cancel.  x and w are bf16 as they are.  Sums are fp32; splits of the token axis are added in a fixed order.
//
// Three launches:
//   1. router_dlogits_kernel  a workgroup takes 32 tokens: dl in LDS, then hi / lo fragments of 16 bytes per lane in the order
//                             in which either product reads them, and the tokens' part of db; further workgroups bring w into
//                             fragment order (w is a few MB, any E, padded with zeros to the K of an MFMA);
//   2. router_grad_kernel     jobs of dw, then jobs of dx, in one launch: the one reads the tokens and the other writes
//                             their gradients, and neither waits for the other;
//   3. router_reduce_kernel   adds up the parts of dw and of db.
#include <type_traits>

#include "common.hpp"

namespace moe {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

struct RouterBwdArgs {
  const void* d_aff;
  const uint16_t *x, *w;
  const void* logits;
  const int32_t* ids;
  int aff_dtype, logits_dtype;
  int64_t T, H, E, k;
  int softmax, chosen, norm, full;  // chosen: activation of the chosen logits only; full: affinities of all experts were handed out
  u32x4* dlx;   // [tokens / 16][KS][2][64]   K = experts, for dx
  u32x4* dlw;   // [tokens / 32][2 KS][2][64] K = tokens, for dw
  u32x4* wp;    // [H / 64][4][KS][64]
  float* dbp;   // [tokens / 32][E]
  uint16_t *dx, *dw;
  float* dwp;   // [splits][H][E]
  void* db;
  int db_dtype;
  int64_t steps, splits;  // steps of 32 tokens; parts of them for dw
  int64_t n_dw, mt, hb_per;  // jobs of dw; 16-token tiles and 64-column blocks of a job of dx
};

__device__ __forceinline__ uint32_t hi_lo(float a, float b, uint32_t& lo) {
  const uint32_t h = pack2_bf16(a, b);
  lo = pack2_bf16(a - bf16_lo(h), b - bf16_hi(h));
  return h;
}

// sum / max over the eight lanes that share a token
__device__ __forceinline__ float sum8(float v) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float max8(float v) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

template <int KS>
__global__ __launch_bounds__(256) void router_dlogits_kernel(const RouterBwdArgs a) {
  constexpr int EP = 32 * KS, PITCH = EP + 4;
  extern __shared__ __attribute__((aligned(16))) float s_dl[];  // [32][PITCH]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x >= a.steps) {  // w: 64 rows into fragment order; lane (r, g) of tile m holds row 16 (r / 4) + 4 m + r % 4, so that a
    const int64_t hb = blockIdx.x - a.steps;  // lane's results are 16 neighbours
    for (int i = tid; i < 4 * KS * 64; i += 256) {
      const int l = i & 63, ks = (i >> 6) % KS, m = (i >> 6) / KS, r = l & 15;
      const int64_t h = hb * 64 + 16 * (r >> 2) + 4 * m + (r & 3), e = 32 * ks + 8 * (l >> 4);
      const uint16_t* src = a.w + h * a.E + e;
      u32x4 v = {0, 0, 0, 0};
      if (e + 8 <= a.E) {
        const u32x4_any d = *(const u32x4_any*)src;
        v = u32x4{d[0], d[1], d[2], d[3]};
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (e + q < a.E) v[q / 2] |= (uint32_t)src[q] << (16 * (q % 2));
      }
      a.wp[hb * (4 * KS * 64) + i] = v;
    }
    return;
  }
  const int64_t t0 = (int64_t)blockIdx.x * 32;
  for (int i = tid; i < 32 * PITCH; i += 256) s_dl[i] = 0.f;
  __syncthreads();
  {
    // eight lanes per token, one per chosen expert
    const int tl = wave * 8 + (lane >> 3), j = lane & 7;
    const int64_t t = t0 + tl;
    int id = t < a.T && j < a.k ? a.ids[t * a.k + j] : -1;
    bool on = id >= 0 && id < a.E;
#pragma unroll
    for (int o = 1; o < 8; ++o) {  // an expert named twice counts once
      const int other = __shfl(id, (lane & 56) | ((j - o) & 7), 64);
      on = on && !(o <= j && other == id);
    }
    const float l = on ? load_as_f32(a.logits, a.logits_dtype, t * a.E + id) : -__builtin_inff();
    const float g = on ? load_as_f32(a.d_aff, a.aff_dtype, t * a.E + id) : 0.f;
    if (a.softmax && !(a.chosen || a.norm)) {
      if (on) s_dl[tl * PITCH + id] = g;  // below
    } else if (a.softmax) {
      const float p = on ? expf(l - max8(on ? l : -__builtin_inff())) : 0.f;
      const float q = p / sum8(p);
      const float mean = sum8(on ? g * q : 0.f);
      if (on) s_dl[tl * PITCH + id] = q * (g - mean);
    } else {
      const float e = expf(-fabsf(l)), r = 1.f / (1.f + e);  // sigmoid(|l|); sigmoid(l) = r or e r
      const float s = on ? (l >= 0.f ? r : e * r) : 0.f, slope = e * r * r;
      float gg = g;
      if (a.norm && !a.chosen) {
        const float total = sum8(s);
        const float mean = sum8(on ? g * s : 0.f) / total;
        gg = (g - mean) / total;
      }
      if (on) s_dl[tl * PITCH + id] = gg * slope;
    }
  }
  if (a.full || (a.softmax && !(a.chosen || a.norm))) {
    // every expert has a part: the lanes of a wave share a token's row
    __syncthreads();
    constexpr int NE = (EP + 63) / 64;
    for (int i = 0; i < 8; ++i) {
      const int tl = wave * 8 + i;
      const int64_t t = t0 + tl;
      if (t >= a.T) break;
      float l[NE], g[NE], mx = -__builtin_inff();
#pragma unroll
      for (int n = 0; n < NE; ++n) {
        const int e = n * 64 + lane;
        l[n] = e < a.E ? load_as_f32(a.logits, a.logits_dtype, t * a.E + e) : -__builtin_inff();
        g[n] = 0.f;
        if (e < a.E) g[n] = a.full ? load_as_f32(a.d_aff, a.aff_dtype, t * a.E + e) : s_dl[tl * PITCH + e];
        mx = fmaxf(mx, l[n]);
      }
      if (a.softmax) {
        mx = wave_max(mx);
        float sum = 0.f, mean = 0.f;
#pragma unroll
        for (int n = 0; n < NE; ++n) {
          l[n] = n * 64 + lane < a.E ? expf(l[n] - mx) : 0.f;
          sum += l[n];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int n = 0; n < NE; ++n) {
          l[n] /= sum;
          mean += g[n] * l[n];
        }
        mean = wave_sum(mean);
#pragma unroll
        for (int n = 0; n < NE; ++n)
          if (n * 64 + lane < a.E) s_dl[tl * PITCH + n * 64 + lane] = l[n] * (g[n] - mean);
      } else {
#pragma unroll
        for (int n = 0; n < NE; ++n)
          if (n * 64 + lane < a.E) {
            const float e = expf(-fabsf(l[n])), r = 1.f / (1.f + e);
            s_dl[tl * PITCH + n * 64 + lane] = g[n] * e * r * r;
          }
      }
    }
  }
  __syncthreads();
  for (int64_t e = tid; e < a.E; e += 256) {
    float v = 0.f;
    for (int t = 0; t < 32; ++t) v += s_dl[t * PITCH + e];
    a.dbp[blockIdx.x * a.E + e] = v;
  }
  const int c = lane & 15, g = lane >> 4;
  for (int i = wave; i < 2 * KS; i += 4) {  // dx: token tile i / KS, 32 experts i % KS
    const float* row = s_dl + (16 * (i / KS) + c) * PITCH + 32 * (i % KS) + 8 * g;
    u32x4 h, lo;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t l;
      h[q] = hi_lo(row[2 * q], row[2 * q + 1], l);
      lo[q] = l;
    }
    u32x4* dst = a.dlx + ((2 * (int64_t)blockIdx.x * KS + i) * 2) * 64 + lane;
    dst[0] = h;
    dst[64] = lo;
  }
  for (int i = wave; i < 2 * KS; i += 4) {  // dw: 16 experts i
    const float* col = s_dl + 8 * g * PITCH + 16 * i + c;
    u32x4 h, lo;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t l;
      h[q] = hi_lo(col[2 * q * PITCH], col[(2 * q + 1) * PITCH], l);
      lo[q] = l;
    }
    u32x4* dst = a.dlw + (((int64_t)blockIdx.x * 2 * KS + i) * 2) * 64 + lane;
    dst[0] = h;
    dst[64] = lo;
  }
}

__device__ __forceinline__ v4f mfma(const u32x4& x, const u32x4& y, const v4f& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x), __builtin_bit_cast(v8bf, y), c, 0, 0, 0);
}

constexpr int GRAD_THREADS = 512;
constexpr int GRAD_LDS = 128 * 1024;

// dw: 128 columns of x by up to 256 experts over a part of the tokens.  Waves 0 .. 3 and 4 .. 7 take alternate steps of 32 tokens;
// within either four, a wave has a quarter of the experts.  x is read in rows (16 bytes of 8 columns per lane) and turned in
// registers: lane (r, g) holds 8 tokens x 8 columns, i.e. the fragments of eight row tiles whose row r is column 8 r + j.
template <int KS>
__device__ __forceinline__ void grad_w(const RouterBwdArgs& a, int64_t job, uint8_t* smem) {
  constexpr int NQ = KS > 8 ? KS / 8 : 1;          // column blocks of 256 experts
  constexpr int NT = KS > 8 ? 4 : KS / 2;          // 16-expert tiles per wave
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4, kg = wave >> 2, nq = wave & 3;
  const int64_t nb = job % NQ, hb = job / NQ % (a.H / 128), sp = job / NQ / (a.H / 128);
  const int64_t s0 = a.steps * sp / a.splits, s1 = a.steps * (sp + 1) / a.splits;
  const int n0 = (int)nb * 16 + nq * NT;  // first of the wave's 16-expert tiles
  v4f acc[8][NT];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[j][n] = (v4f){0.f, 0.f, 0.f, 0.f};
  const uint16_t* xc = a.x + hb * 128 + 8 * r;
  for (int64_t s = s0 + kg; s < s1; s += 2) {
    u32x4 x[8], b[NT], bl[NT];
    const int64_t t = s * 32 + 8 * g;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = u32x4{0, 0, 0, 0};
      if (t + j < a.T) {
        const u32x4_any d = *(const u32x4_any*)(xc + (t + j) * a.H);
        x[j] = u32x4{d[0], d[1], d[2], d[3]};
      }
    }
    const u32x4* src = a.dlw + ((s * 2 * KS + n0) * 2) * 64 + lane;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      b[n] = src[n * 128];
      bl[n] = src[n * 128 + 64];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u32x4 f;
#pragma unroll
      for (int q = 0; q < 4; ++q)  // tokens 2 q and 2 q + 1 of column j
        f[q] = __builtin_amdgcn_perm(x[2 * q + 1][j / 2], x[2 * q][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[j][n] = mfma(f, b[n], acc[j][n]);
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[j][n] = mfma(f, bl[n], acc[j][n]);
    }
  }
  v4f* s_acc = (v4f*)smem + (int64_t)nq * (8 * NT * 64) + lane;
  if (kg == 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int n = 0; n < NT; ++n) s_acc[(j * NT + n) * 64] = acc[j][n];
  }
  __syncthreads();
  if (kg == 1) return;
  const bool whole = a.splits == 1;
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const v4f v = acc[j][n] + s_acc[(j * NT + n) * 64];
      const int64_t e = (n0 + n) * 16 + r;
      if (e < a.E) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t at = (hb * 128 + 8 * (4 * g + i) + j) * a.E + e;
          if (whole) a.dw[at] = f32_to_bf16_bits(v[i]);
          else a.dwp[sp * a.H * a.E + at] = v[i];
        }
      }
    }
}

// dx: up to 128 tokens, whose dl lie in LDS, by some blocks of 64 columns, each wave a block at a time with the block's w in
// registers.
template <int KS>
__device__ __forceinline__ void grad_x(const RouterBwdArgs& a, int64_t job, uint8_t* smem) {
  constexpr int NM = KS > 8 ? 2 : 4;  // row tiles whose w is held at a time
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t parts = (a.H / 64 + a.hb_per - 1) / a.hb_per, tg = job / parts, hp = job % parts;
  const int64_t tile0 = tg * a.mt, tiles = a.steps * 2;
  const int mt = (int)(tiles - tile0 < a.mt ? tiles - tile0 : a.mt);
  u32x4* s_dl = (u32x4*)smem;
  const u32x4* src = a.dlx + tile0 * (KS * 128);
  for (int i = threadIdx.x; i < mt * KS * 128; i += GRAD_THREADS) s_dl[i] = src[i];
  __syncthreads();
  const int64_t hb1 = (hp + 1) * a.hb_per < a.H / 64 ? (hp + 1) * a.hb_per : a.H / 64;
  for (int64_t hb = hp * a.hb_per + wave; hb < hb1; hb += GRAD_THREADS / 64) {
#pragma unroll 1
    for (int m0 = 0; m0 < 4; m0 += NM) {
      u32x4 w[NM][KS];
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) w[m][ks] = a.wp[((hb * 4 + m0 + m) * KS + ks) * 64 + lane];
#pragma unroll 1
      for (int i = 0; i < mt; ++i) {
        v4f acc[NM];
#pragma unroll
        for (int m = 0; m < NM; ++m) acc[m] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 h = s_dl[(i * KS + ks) * 128 + lane], lo = s_dl[(i * KS + ks) * 128 + 64 + lane];
#pragma unroll
          for (int m = 0; m < NM; ++m) acc[m] = mfma(w[m][ks], h, acc[m]);
#pragma unroll
          for (int m = 0; m < NM; ++m) acc[m] = mfma(w[m][ks], lo, acc[m]);
        }
        const int64_t t = (tile0 + i) * 16 + c;
        if (t < a.T) {
          uint16_t* dst = a.dx + t * a.H + hb * 64 + 16 * g + 4 * m0;
#pragma unroll
          for (int m = 0; m < NM; m += 2) {
            const u32x4_any v = {pack2_bf16(acc[m][0], acc[m][1]), pack2_bf16(acc[m][2], acc[m][3]),
                                 pack2_bf16(acc[m + 1][0], acc[m + 1][1]), pack2_bf16(acc[m + 1][2], acc[m + 1][3])};
            *(u32x4_any*)(dst + 4 * m) = v;
          }
        }
      }
    }
  }
}

template <int KS>
__global__ __launch_bounds__(GRAD_THREADS) void router_grad_kernel(const RouterBwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int64_t job = blockIdx.x;
  if (job < a.n_dw) grad_w<KS>(a, job, smem);
  else grad_x<KS>(a, job - a.n_dw, smem);
}

__global__ __launch_bounds__(256) void router_reduce_kernel(const RouterBwdArgs a, int64_t n_w) {
  if (blockIdx.x < n_w) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = a.H * a.E;
    if (i >= n) return;
    float v = 0.f;
    for (int64_t s = 0; s < a.splits; ++s) v += a.dwp[s * n + i];
    a.dw[i] = f32_to_bf16_bits(v);
    return;
  }
  const int64_t e = (int64_t)(blockIdx.x - n_w) * 4 + (threadIdx.x >> 6);
  if (e >= a.E) return;
  float v = 0.f;
  for (int64_t s = threadIdx.x & 63; s < a.steps; s += 64) v += a.dbp[s * a.E + e];
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) {
    if (a.db_dtype == MOE_DT_FP32) ((float*)a.db)[e] = v;
    else ((uint16_t*)a.db)[e] = f32_to_bf16_bits(v);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

struct RouterBwdPlan {
  int ks;
  int64_t steps, splits, mt, hb_per, n_dw, n_dx;
  size_t dlx, dlw, wp, dbp, dwp, total;
};
static RouterBwdPlan router_bwd_plan(int64_t T, int64_t H, int64_t E) {
  RouterBwdPlan p;
  p.ks = E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 16;
  p.steps = (T + 31) / 32;
  const int64_t nq = p.ks > 8 ? p.ks / 8 : 1, tiles = H / 128 * nq;
  // dw: a workgroup per CU where the tokens allow parts of eight steps, four per half of a workgroup
  p.splits = 256 / tiles;
  if (p.splits > p.steps / 8) p.splits = p.steps / 8;
  if (p.splits < 1) p.splits = 1;
  p.n_dw = tiles * p.splits;
  // dx: as many tokens as LDS holds, fewer where that leaves CUs without a job; two blocks of 64 columns per wave, or one
  const int64_t most = GRAD_LDS / (p.ks * 2048);
  p.hb_per = 16;
  p.mt = p.steps * 2 * ((H / 64 + p.hb_per - 1) / p.hb_per) / 256;
  if (p.mt < 1) {
    p.hb_per = 8;
    p.mt = 1;
  }
  if (p.mt > (most < 8 ? most : 8)) p.mt = most < 8 ? most : 8;
  p.n_dx = (p.steps * 2 + p.mt - 1) / p.mt * ((H / 64 + p.hb_per - 1) / p.hb_per);
  auto al = [](size_t v) { return (v + 255) & ~(size_t)255; };
  size_t off = 0;
  p.dlx = off; off += al((size_t)p.steps * 2 * p.ks * 2048);
  p.dlw = off; off += al((size_t)p.steps * 2 * p.ks * 2048);
  p.wp = off; off += al((size_t)H / 64 * 4 * p.ks * 1024);
  p.dbp = off; off += al((size_t)p.steps * E * 4);
  p.dwp = off; off += p.splits > 1 ? al((size_t)p.splits * H * E * 4) : 0;
  p.total = off;
  return p;
}

template <int KS>
static int launch_router_bwd(const RouterBwdArgs& a, const RouterBwdPlan& p, hipStream_t s) {
  constexpr int LDS1 = 32 * (32 * KS + 4) * 4;
  if (allow_lds<router_dlogits_kernel<KS>>(LDS1) != hipSuccess) return MOE_E_LAUNCH;
  if (allow_lds<router_grad_kernel<KS>>(GRAD_LDS) != hipSuccess) return MOE_E_LAUNCH;
  hipLaunchKernelGGL(router_dlogits_kernel<KS>, dim3((unsigned)(p.steps + a.H / 64)), dim3(256), LDS1, s, a);
  MOE_CHECK_LAUNCH();
  const int lds_w = 4 * 8 * (KS > 8 ? 4 : KS / 2) * 64 * 16, lds_x = (int)p.mt * KS * 2048;
  hipLaunchKernelGGL(router_grad_kernel<KS>, dim3((unsigned)(p.n_dw + p.n_dx)), dim3(GRAD_THREADS), lds_w > lds_x ? lds_w : lds_x, s,
                     a);
  MOE_CHECK_LAUNCH();
  const int64_t n_w = p.splits > 1 ? (a.H * a.E + 255) / 256 : 0, n_b = a.db ? (a.E + 3) / 4 : 0;
  if (n_w + n_b > 0) {
    hipLaunchKernelGGL(router_reduce_kernel, dim3((unsigned)(n_w + n_b)), dim3(256), 0, s, a, n_w);
    MOE_CHECK_LAUNCH();
  }
  return MOE_OK;
}

static int router_bwd_shape(int64_t T, int64_t H, int64_t E) {
  if (T < 1 || H < 1 || E < 1) return MOE_E_BAD_ARG;
  // (a launch holds fewer than 2^32 threads)
  if (E > 512 || H % 128 != 0 || H > (int64_t)1 << 20 || T > (int64_t)1 << 26) return MOE_E_BAD_SHAPE;
  const RouterBwdPlan p = router_bwd_plan(T, H, E);
  if ((p.n_dw + p.n_dx) * GRAD_THREADS >= (int64_t)1 << 32 || (p.steps + H / 64) * 256 >= (int64_t)1 << 32) return MOE_E_BAD_SHAPE;
  return MOE_OK;
}

}  // namespace moe

using namespace moe;

extern "C" size_t moe_router_topk_bwd_workspace_bytes(int64_t T, int64_t H, int64_t E) {
  return router_bwd_shape(T, H, E) == MOE_OK ? router_bwd_plan(T, H, E).total : 0;
}

extern "C" int moe_router_topk_bwd(const void* d_affinities, int aff_dtype, const void* x, const void* w, const void* router_logits,
                                   int logits_dtype, const int32_t* expert_index, int64_t T, int64_t H, int64_t E, int k, int act_fn,
                                   int router_pre_norm, int norm_topk_prob, int mask_to_topk, void* d_x, void* d_w, void* d_bias,
                                   int bias_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d_affinities || !x || !w || !router_logits || !expert_index || !d_x || !d_w) return MOE_E_BAD_ARG;
  if (aff_dtype != MOE_DT_BF16 && aff_dtype != MOE_DT_FP32) return MOE_E_BAD_ARG;
  if (logits_dtype != MOE_DT_BF16 && logits_dtype != MOE_DT_FP32) return MOE_E_BAD_ARG;
  if (d_bias && bias_dtype != MOE_DT_BF16 && bias_dtype != MOE_DT_FP32) return MOE_E_BAD_ARG;
  if (act_fn < 0 || act_fn > 1) return MOE_E_BAD_ARG;
  const int rc = router_bwd_shape(T, H, E);
  if (rc != MOE_OK) return rc;
  if (k < 1 || k > 8 || k > E) return MOE_E_BAD_SHAPE;
  const RouterBwdPlan p = router_bwd_plan(T, H, E);
  if (!workspace || workspace_bytes < p.total) return MOE_E_WORKSPACE;
  if (((uintptr_t)workspace & 15) != 0) return MOE_E_BAD_ARG;
  uint8_t* ws = (uint8_t*)workspace;
  RouterBwdArgs a;
  a.d_aff = d_affinities;
  a.x = (const uint16_t*)x;
  a.w = (const uint16_t*)w;
  a.logits = router_logits;
  a.ids = expert_index;
  a.aff_dtype = aff_dtype;
  a.logits_dtype = logits_dtype;
  a.T = T; a.H = H; a.E = E; a.k = k;
  a.softmax = act_fn == 1;
  a.chosen = !router_pre_norm;
  a.norm = router_pre_norm && norm_topk_prob;
  a.full = router_pre_norm && !norm_topk_prob && !mask_to_topk;
  a.dlx = (u32x4*)(ws + p.dlx);
  a.dlw = (u32x4*)(ws + p.dlw);
  a.wp = (u32x4*)(ws + p.wp);
  a.dbp = (float*)(ws + p.dbp);
  a.dx = (uint16_t*)d_x;
  a.dw = (uint16_t*)d_w;
  a.dwp = (float*)(ws + p.dwp);
  a.db = d_bias;
  a.db_dtype = bias_dtype;
  a.steps = p.steps; a.splits = p.splits; a.n_dw = p.n_dw; a.mt = p.mt; a.hb_per = p.hb_per;
  const hipStream_t s = (hipStream_t)stream;
  switch (p.ks) {
    case 2: return launch_router_bwd<2>(a, p, s);
    case 4: return launch_router_bwd<4>(a, p, s);
    case 8: return launch_router_bwd<8>(a, p, s);
    default: return launch_router_bwd<16>(a, p, s);
  }
}

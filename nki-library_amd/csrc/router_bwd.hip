// Gradient of the router (router_topk.hip): from the gradient g of the affinities to those of the logits, the hidden states, the
// weights and the bias.
//
//   softmax over the chosen (also: over all, divided by the chosen's sum, which is the same)   dl_j = a_j (g_j - sum g a)
//   softmax over all                                                                          dl_e = p_e (g_e - sum g p)
//   sigmoid                                                                                   dl_j = g_j s_j (1 - s_j)
//   sigmoid, divided by the chosen's sum S        dl_j = (g_j - sum g a) / S  s_j (1 - s_j),  a_j = s_j / S
//   dx = dl w^T    dw = x^T dl    db = sum over the tokens of dl
//
// Everything up to dl is fp32.  A token has k of them at most, but for the softmax over all experts ("dense").  dw runs on bf16
// MFMAs with dl as the sum of two bf16 (hi + lo, 2^-17 of the value): a single bf16 (2^-8) would double the error of a result
// that is rounded to bf16 itself, and leave more than that where terms cancel over the tokens.  dx of k experts is k
// multiply-adds per value, in fp32 from a slice of w in LDS; dense, it runs on MFMAs like dw (there a single bf16 would leave
// 2^-8 of every term of sums that vanish by construction: dl add up to zero over the experts).  x and w are bf16 as they are.
// Sums are fp32; parts of the token axis are added in a fixed order.
//
// Three launches:
//   1. router_dlogits_kernel   a workgroup takes 32 tokens: dl in LDS, then hi / lo fragments of 16 bytes per lane in the order in
//                              which the products read them, each token's list of (expert, dl), and the tokens' part of db;
//                              further workgroups transpose w (dense: bring it into fragment order);
//   2. router_grad_kernel      dw and dx (large calls: router_dw_kernel, bound by the matrix pipes at the 1.64 GHz of 2.4 that their
//                              power leaves, and router_dx_list_kernel, by the vector ALU: 75 instructions a token and 256
//                              columns, half of them to unpack w);
//   3. router_reduce_kernel    the sums of the parts of dw and of db (large calls: the workgroups of dx, when done).
// T = 8192, H = 7168, E = 256, top-8: 9 + 57 + 50 us; 52 for its bytes at the rate of a copy and 50 for 2 x 30 GFLOP, the products of
// dw and of dx, at that of a large product.  (dw alone, with hi and lo, is as much.)
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
  int softmax, norm, full;          // full: affinities of all experts were handed out
  int dense, kp;                    // dense: every expert has a part in dl; kp: k rounded up to a power of two
  u32x4* dlx;   // [tokens / 16][KS][2][64]   K = experts, for dx
  u32x4* dlw;   // [tokens / 32][2 KS][2][64] K = tokens, for dw
  u32x4* wp;    // [H / 64][4][KS][64], for dense dx
  uint16_t* wt; // [E][H], for sparse dx
  uint2* list;  // [T][KP] expert and dl, k of them and zeros of the first expert behind them, for sparse dx
  float* dbp;   // [tokens / 32][E]
  uint16_t *dx, *dw;
  float* dwp;   // [splits][H][E]
  void* db;
  int db_dtype;
  int64_t steps, splits;  // steps of 32 tokens; parts of them for dw
  int64_t n_dw, x_splits;    // jobs of dw; parts of the tokens for dx
};

// (An infinite value is its own hi part, with nothing behind it: inf - inf would make a NaN of what a sum in fp32 leaves infinite.  A
// finite dl is at most half of the largest fp32, whose bf16 is finite too.)
__device__ __forceinline__ uint32_t hi_lo(float a, float b, uint32_t& lo) {
  const uint32_t h = pack2_bf16(a, b);
  const float ra = fabsf(a) < __builtin_inff() ? a - bf16_lo(h) : 0.f, rb = fabsf(b) < __builtin_inff() ? b - bf16_hi(h) : 0.f;
  lo = pack2_bf16(ra, rb);
  return h;
}

// sum / max over the eight lanes that share a token, all of which have to be there: a lane that a branch leaves out hands over anything
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
struct GradW {
  static constexpr int NQ = KS > 8 ? KS / 8 : 1;  // column blocks of 256 experts
  static constexpr int NT = KS > 8 ? 4 : KS / 2;  // 16-expert tiles per wave
};

template <int KS>
__global__ __launch_bounds__(256) void router_dlogits_kernel(const RouterBwdArgs a) {
  constexpr int EP = 32 * KS, PITCH = EP + 4;
  extern __shared__ __attribute__((aligned(16))) float s_dl[];  // [32][PITCH]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x >= a.steps) {  // 64 rows of w
    const int64_t hb = blockIdx.x - a.steps;
    if (!a.dense) {
      uint16_t* s_w = (uint16_t*)s_dl;  // [64][E]
      const uint16_t* src = a.w + hb * 64 * a.E;
      for (int i = tid; i < 8 * (int)a.E; i += 256) {
        const u32x4_any d = *(const u32x4_any*)(src + 8 * i);
        *(u32x4*)(s_w + 8 * i) = u32x4{d[0], d[1], d[2], d[3]};
      }
      __syncthreads();
      for (int i = tid; i < 8 * (int)a.E; i += 256) {
        const int e = i >> 3, p = i & 7;
        u32x4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          v[q] = (uint32_t)s_w[(8 * p + 2 * q) * (int)a.E + e] | (uint32_t)s_w[(8 * p + 2 * q + 1) * (int)a.E + e] << 16;
        *(u32x4*)(a.wt + e * a.H + hb * 64 + 8 * p) = v;
      }
      return;
    }
    // fragments: lane (r, g) of tile m holds row 16 (r / 4) + 4 m + r % 4, so that a lane's results are 16 neighbours
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
    float dl = 0.f;
    if (a.dense) {
      dl = g;  // below
    } else if (a.softmax) {
      const float mx = max8(l);  // (all eight lanes take part; l of one that is off is -inf)
      const float p = on ? expf(l - mx) : 0.f;
      const float q = p / sum8(p);
      const float mean = sum8(on ? g * q : 0.f);
      dl = q * (g - mean);
    } else {
      const float e = expf(-fabsf(l)), r = 1.f / (1.f + e);  // sigmoid(|l|); sigmoid(l) = r or e r
      const float s = on ? (l >= 0.f ? r : e * r) : 0.f, slope = e * r * r;
      dl = g * slope;
      if (a.norm) {
        const float total = sum8(s);
        const float mean = sum8(on ? g * s : 0.f) / total;
        dl = (g - mean) * (slope / total);  // (a_j (1 - s_j), at most one: scores near zero do not overflow on the way)
      }
    }
    if (on) s_dl[tl * PITCH + id] = dl;
    if (!a.dense && t < a.T && j < a.kp) {
      const uint64_t who = __ballot(on) >> (lane & 56) & 0xff;
      const int first = __shfl(id, (lane & 56) | (who ? __builtin_ctzll(who) : 0), 64);
      a.list[t * a.kp + j] = on ? make_uint2((uint32_t)id, __float_as_uint(dl)) : make_uint2(who ? (uint32_t)first : 0u, 0u);
    }
  }
  if (a.dense) {
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
  for (int i = a.dense ? wave : 2 * KS; i < 2 * KS; i += 4) {  // dx: token tile i / KS, 32 experts i % KS
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
  for (int i = wave; i < 2 * KS; i += 4) {  // dw: tile i % NT of a wave's NT; its column c is expert NT c + i % NT of theirs
    constexpr int NT = GradW<KS>::NT;
    const float* col = s_dl + 8 * g * PITCH + i / NT * (16 * NT) + NT * c + i % NT;
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

constexpr int GRAD_THREADS = 512, DX_THREADS = 1024;

// Rows [t0, t0 + 32) of x or dx, as a buffer: what lies behind the last token reads as zeros and is not written.  No branch
// stands around a load or store then, and the waits count the operations that are really out.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t token_rows(const uint16_t* base, int64_t t0, int64_t t1, int64_t H, int rows) {
  const int64_t left = t1 - t0 < rows ? t1 - t0 : rows;
  return __builtin_amdgcn_make_buffer_rsrc((void*)(base + t0 * H), 0, left > 0 ? (int)(left * H * 2) : 0, 0x00020000);
}

// dw: 128 columns of x by up to 256 experts over a part of the tokens.  Waves 0 .. 3 and 4 .. 7 take alternate steps of 32 tokens
// (two waves per SIMD: the one multiplies while the other waits), a quarter of the experts per wave.  A step's rows (256 bytes
// each) go through LDS.  Lane (r, g) reads 8 tokens x 8 columns of them and turns them in registers: they are the fragments of
// eight row tiles whose row r is column 8 r + j.  A step goes over them twice, for dl's hi and for its lo parts, so that the
// fragments of either part arrive in registers that the other half step has no use for; the rows are asked for two steps ahead.
constexpr int DW_LDS = 32768;
template <int KS>
__device__ __forceinline__ void grad_w(const RouterBwdArgs& a, int64_t job, uint8_t* smem) {
  constexpr int NQ = GradW<KS>::NQ, NT = GradW<KS>::NT;
  u32x4(*s_x)[2][512] = (u32x4(*)[2][512])smem;  // [group][buffer][32 tokens][16]; at the end the sums of a quarter
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tid = threadIdx.x & 255, kg = wave >> 2, nq = wave & 3, r = lane & 15, g = lane >> 4;
  const int64_t nb = job % NQ, hb = job / NQ % (a.H / 128), sp = job / NQ / (a.H / 128);
  const int64_t s0 = a.steps * sp / a.splits, s1 = a.steps * (sp + 1) / a.splits;
  const int n0 = (int)nb * 16 + nq * NT;  // first of the wave's 16-expert tiles
  v4f acc[8][NT];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[j][n] = (v4f){0.f, 0.f, 0.f, 0.f};
  const int off = (int)(((tid >> 4) * a.H + hb * 128 + 8 * (tid & 15)) * 2), half = (int)(16 * a.H * 2);
  u32x4 in[2], b[NT], bl[NT];
  auto fetch_x = [&](int64_t s) {
    const __amdgpu_buffer_rsrc_t rows = token_rows(a.x, s * 32, s < s1 ? a.T : 0, a.H, 32);
    in[0] = __builtin_amdgcn_raw_buffer_load_b128(rows, off, 0, 0);
    in[1] = __builtin_amdgcn_raw_buffer_load_b128(rows, off + half, 0, 0);
  };
  auto store_x = [&](u32x4* buf) {
    buf[tid] = in[0];
    buf[256 + tid] = in[1];
  };
  auto fetch_dl = [&](int64_t s, int part, u32x4(&d)[NT]) {  // (as a buffer too: zeros behind the last step)
    const __amdgpu_buffer_rsrc_t step =
        __builtin_amdgcn_make_buffer_rsrc((void*)(a.dlw + s * (2 * KS * 128)), 0, s < s1 ? 2 * KS * 2048 : 0, 0x00020000);
    const int at = ((n0 * 2 + part) * 64 + lane) * 16;
#pragma unroll
    for (int n = 0; n < NT; ++n) d[n] = __builtin_amdgcn_raw_buffer_load_b128(step, at + n * 2048, 0, 0);
  };
  auto multiply = [&](const u32x4* buf, const u32x4(&d)[NT]) {
    u32x4 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = buf[(8 * g + j) * 16 + r];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u32x4 f;
#pragma unroll
      for (int q = 0; q < 4; ++q)  // tokens 2 q and 2 q + 1 of column j
        f[q] = __builtin_amdgcn_perm(x[2 * q + 1][j / 2], x[2 * q][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[j][n] = mfma(f, d[n], acc[j][n]);
    }
  };
  // both groups take as many turns: in one without a step the rows and dl are zeros (another step's dl would do, were it finite)
  const int64_t turns = (s1 - s0 + 1) / 2;
  fetch_x(s0 + kg);
  store_x(s_x[kg][0]);
  fetch_x(s0 + kg + 2);
  fetch_dl(s0 + kg, 0, b);
  __syncthreads();
  for (int64_t i = 0; i < turns; ++i) {
    const int64_t s = s0 + 2 * i + kg;
    const u32x4* buf = s_x[kg][i & 1];
    fetch_dl(s, 1, bl);
    __builtin_amdgcn_sched_barrier(0);
    multiply(buf, b);
    __builtin_amdgcn_sched_barrier(0);
    store_x(s_x[kg][(i + 1) & 1]);
    fetch_dl(s + 2, 0, b);
    fetch_x(s + 4);
    __builtin_amdgcn_sched_barrier(0);
    multiply(buf, bl);
    __syncthreads();
  }
  // both groups' sums by way of LDS, JC of the eight columns of a lane's 8 r + j at a time, and from there to memory in pieces of
  // four experts: in a loop, since code that runs once is fetched cold (written out as stores of accumulators, this launch took
  // 11.3 us for 128 tokens, now 8.2)
  constexpr int JC = 8 / NT;
  float* s_sum = (float*)smem;  // [4 waves][JC][NT][64 lanes][4]
  v4f* s_acc = (v4f*)smem + nq * (JC * NT * 64) + lane;
  const bool whole = a.splits == 1;
  const int64_t e_base = nb * 256;
#pragma unroll
  for (int j0 = 0; j0 < 8; j0 += JC) {
    if (kg == 1) {
#pragma unroll
      for (int j = 0; j < JC; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) s_acc[(j * NT + n) * 64] = acc[j0 + j][n];
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int j = 0; j < JC; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) s_acc[(j * NT + n) * 64] += acc[j0 + j][n];
    }
    __syncthreads();
    // piece p: row p / (16 NT) of 16 JC, experts 4 (p % (16 NT)) ..
#pragma unroll 1
    for (int p = threadIdx.x; p < 2048; p += GRAD_THREADS) {
      const int row = p / (16 * NT), e4 = 4 * (p % (16 * NT)), j = row % JC, gi = row / JC;  // gi = 4 g + i of the accumulators
      const int64_t e = e_base + e4, at = (hb * 128 + 8 * gi + j0 + j) * a.E + e;
      v4f v;
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // expert (wave, NT r + n)
        const int ee = e4 + q, wv = ee / (16 * NT), in = ee % (16 * NT), r2 = in / NT, n = in % NT;
        v[q] = s_sum[(((wv * JC + j) * NT + n) * 64 + 16 * (gi >> 2) + r2) * 4 + (gi & 3)];
      }
      if (e + 4 <= a.E) {
        typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
        typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
        if (whole) *(u32x2_any*)(a.dw + at) = u32x2_any{pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3])};
        else *(v4f_any*)(a.dwp + sp * a.H * a.E + at) = v4f_any{v[0], v[1], v[2], v[3]};
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (e + q < a.E) {
            if (whole) a.dw[at + q] = f32_to_bf16_bits(v[q]);
            else a.dwp[sp * a.H * a.E + at + q] = v[q];
          }
      }
    }
    __syncthreads();
  }
}

// dx of k experts per token: a workgroup keeps the slice of w of 64 * CPL columns in LDS, a wave takes two tokens at a time, CPL
// columns per lane: k reads of LDS and k multiply-adds per value, expert and dl in scalar registers.
template <int CPL, int KP, int THREADS>
__device__ __forceinline__ void grad_x_list(const RouterBwdArgs& a, int64_t job, uint8_t* smem) {
  constexpr int COLS = 64 * CPL, W = CPL / 2;  // words of a lane
  uint32_t* s_w = (uint32_t*)smem;             // [E][COLS / 2]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t slices = (a.H + COLS - 1) / COLS, c0 = job % slices * COLS, sp = job / slices;
  const int cols = (int)(a.H - c0 < COLS ? a.H - c0 : COLS);  // (H is a multiple of 128)
  const int pieces = cols / 8;
  for (int i = threadIdx.x; i < (int)a.E * pieces; i += THREADS) {
    const int e = i / pieces, p = i - e * pieces;
    *(u32x4*)(s_w + e * (COLS / 2) + 4 * p) = *(const u32x4*)(a.wt + e * a.H + c0 + 8 * p);
  }
  __syncthreads();
  const int64_t t0 = a.T * sp / a.x_splits, t1 = a.T * (sp + 1) / a.x_splits;
  const bool mine = lane * CPL < cols;
  // (address space 4: read-only for the launch, uniform over the wave.  The lists come by scalar loads, which no store is waited
  // for ahead of, a turn early)
  typedef const __attribute__((address_space(4))) uint32_t* list_ptr;
  auto fetch = [&](int64_t t, uint32_t(&l)[2 * KP]) {
    const list_ptr src = (list_ptr)(uintptr_t)(a.list + (t < t1 ? t : t1 - 1) * KP);
#pragma unroll
    for (int i = 0; i < 2 * KP; ++i) l[i] = src[i];
  };
  constexpr int STEP = 2 * THREADS / 64;
  uint32_t now[2][2 * KP], next[2][2 * KP];
  int64_t t = t0 + 2 * wave;
  if (t < t1) {
    fetch(t, now[0]);
    fetch(t + 1, now[1]);
  }
  for (; t < t1; t += STEP) {
    fetch(t + STEP, next[0]);
    fetch(t + STEP + 1, next[1]);
    uint32_t v[2][KP][W];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < KP; ++j)
#pragma unroll
        for (int q = 0; q < W; ++q) v[u][j][q] = s_w[now[u][2 * j] * (COLS / 2) + lane * W + q];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float acc[CPL];
#pragma unroll
      for (int i = 0; i < CPL; ++i) acc[i] = 0.f;
#pragma unroll
      for (int j = 0; j < KP; ++j) {
        const float dl = __uint_as_float(now[u][2 * j + 1]);
#pragma unroll
        for (int q = 0; q < W; ++q) {
          acc[2 * q] = fmaf(dl, bf16_lo(v[u][j][q]), acc[2 * q]);
          acc[2 * q + 1] = fmaf(dl, bf16_hi(v[u][j][q]), acc[2 * q + 1]);
        }
      }
      if (mine && t + u < t1) {
        uint32_t* dst = (uint32_t*)(a.dx + (t + u) * a.H + c0) + lane * W;
        if constexpr (W == 2) {
          typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
          __builtin_nontemporal_store((u32x2{pack2_bf16(acc[0], acc[1]), pack2_bf16(acc[2], acc[3])}), (u32x2*)dst);
        } else {
          __builtin_nontemporal_store(pack2_bf16(acc[0], acc[1]), dst);
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * KP; ++i) now[u][i] = next[u][i];
    }
  }
}

// Dense dx: each wave keeps the w of 64 columns (32 beyond 256 experts) in registers and multiplies 16 tokens after 16 tokens of a
// part of them, whose dl go through LDS, the next ones' while these are multiplied.
template <int KS>
struct GradX {
  static constexpr int NM = KS > 8 ? 2 : 4;         // row tiles of 16 columns per wave
  static constexpr int COLS = NM * 16 * 8;          // columns of a workgroup
};
template <int KS>
__device__ __forceinline__ void grad_x(const RouterBwdArgs& a, int64_t job, uint8_t* smem) {
  u32x4* s_dl = (u32x4*)smem;  // [2][KS][2][64]
  constexpr int NM = GradX<KS>::NM, PIECES = KS * 128 / GRAD_THREADS > 0 ? KS * 128 / GRAD_THREADS : 1;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t groups = (a.H + GradX<KS>::COLS - 1) / GradX<KS>::COLS, hg = job % groups, sp = job / groups;
  const int64_t tiles = (a.T + 15) / 16, i0 = tiles * sp / a.x_splits, i1 = tiles * (sp + 1) / a.x_splits;
  const int64_t unit = hg * 8 + wave;  // of 16 NM columns
  const bool mine = unit * NM / 4 < a.H / 64;  // (the others multiply the last block once more and keep nothing)
  const int64_t hb = mine ? unit * NM / 4 : a.H / 64 - 1, m0 = unit * NM % 4;
  u32x4 w[NM][KS];
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) w[m][ks] = a.wp[((hb * 4 + m0 + m) * KS + ks) * 64 + lane];
  u32x4 in[PIECES];
  auto fetch = [&](int64_t i) {
    const u32x4* src = a.dlx + (i < i1 ? i : i1 - 1) * (KS * 128) + tid;
#pragma unroll
    for (int q = 0; q < PIECES; ++q)
      if (q * GRAD_THREADS + tid < KS * 128) in[q] = src[q * GRAD_THREADS];
  };
  auto store = [&](u32x4* buf) {
#pragma unroll
    for (int q = 0; q < PIECES; ++q)
      if (q * GRAD_THREADS + tid < KS * 128) buf[q * GRAD_THREADS + tid] = in[q];
  };
  fetch(i0);
  store(s_dl);
  fetch(i0 + 1);
  __syncthreads();
  const int off = (int)((c * a.H + hb * 64 + 16 * g + 4 * m0) * 2);
  for (int64_t i = i0; i < i1; ++i) {
    const u32x4* buf = s_dl + ((i - i0) & 1) * (KS * 128);
    v4f acc[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) acc[m] = (v4f){0.f, 0.f, 0.f, 0.f};
    // the next 32 experts' dl are read from LDS while these are multiplied
    u32x4 h[2], lo[2];
    h[0] = buf[lane];
    lo[0] = buf[64 + lane];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + 1 < KS) {
        h[(ks + 1) & 1] = buf[(ks + 1) * 128 + lane];
        lo[(ks + 1) & 1] = buf[(ks + 1) * 128 + 64 + lane];
      }
      if (ks == KS / 2) {
        store(s_dl + ((i + 1 - i0) & 1) * (KS * 128));
        fetch(i + 2);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < NM; ++m) acc[m] = mfma(w[m][ks], h[ks & 1], acc[m]);
#pragma unroll
      for (int m = 0; m < NM; ++m) acc[m] = mfma(w[m][ks], lo[ks & 1], acc[m]);
    }
    const __amdgpu_buffer_rsrc_t rows = token_rows(a.dx, i * 16, mine ? a.T : 0, a.H, 16);
#pragma unroll
    for (int m = 0; m < NM; m += 2) {
      const u32x4 v = {pack2_bf16(acc[m][0], acc[m][1]), pack2_bf16(acc[m][2], acc[m][3]),
                       pack2_bf16(acc[m + 1][0], acc[m + 1][1]), pack2_bf16(acc[m + 1][2], acc[m + 1][3])};
      __builtin_amdgcn_raw_buffer_store_b128(v, rows, off + 8 * m, 0, 0);
    }
    __syncthreads();
  }
}

// The parts of dw and db added up, by all workgroups of a launch.
__device__ __forceinline__ void reduce_parts(const RouterBwdArgs& a, int threads) {
  const int64_t first = (int64_t)blockIdx.x * threads + threadIdx.x, step = (int64_t)gridDim.x * threads;
  if (a.splits > 1) {
    const int64_t n = a.H * a.E;  // (H is a multiple of 128: whole pieces of four)
    for (int64_t i = first; i < n / 4; i += step) {
      v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
      for (int64_t s = 0; s < a.splits; ++s) v += ((const v4f*)(a.dwp + s * n))[i];
      typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
      *(u32x2_any*)(a.dw + 4 * i) = u32x2_any{pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3])};
    }
  }
  if (a.db)
    for (int64_t e = first >> 6; e < a.E; e += step >> 6) {
      float v = 0.f;
      for (int64_t s = threadIdx.x & 63; s < a.steps; s += 64) v += a.dbp[s * a.E + e];
      v = wave_sum(v);
      if ((threadIdx.x & 63) == 0) {
        if (a.db_dtype == MOE_DT_FP32) ((float*)a.db)[e] = v;
        else ((uint16_t*)a.db)[e] = f32_to_bf16_bits(v);
      }
    }
}

// dw and dx in one launch, then the sums: jobs of dw, then jobs of dx, which need nothing of each other.  KP: the places of a token's
// list; 0: dense.  (Slices of 256 columns of w in LDS, of 128 beyond 256 experts.)
template <int KS, int KP>
__global__ __launch_bounds__(GRAD_THREADS) void router_grad_kernel(const RouterBwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int64_t job = blockIdx.x;
  if (job < a.n_dw) grad_w<KS>(a, job, smem);
  else if constexpr (KP == 0) grad_x<KS>(a, job - a.n_dw, smem);
  else grad_x_list<(KS > 8 ? 2 : 4), KP, GRAD_THREADS>(a, job - a.n_dw, smem);
}
__global__ __launch_bounds__(256) void router_reduce_kernel(const RouterBwdArgs a) { reduce_parts(a, 256); }

// Or dw, and then dx with the sums behind it: dx by lists needs a quarter of dw's registers, so that a CU has 16 waves of it instead
// of 8, and gains by it the earlier the more dw there is beside a token, which goes by the experts (k changes little).  In one
// launch | two, us of a call by values of x (2^20): top-4 of 60 experts 8: 24.5 | 27.4, 16: 29.9 | 31.7, 32: 43.3 | 43.8; top-8 of 64 8:
// 27.1 | 28.3, 16: 35.4 | 35.6, 32: 54.3 | 52.0; top-2 of 8 32: 38.3 | 39.6; top-8 of 128 4: 28.1 | 29.3, 8: 37.0 | 34.5, 16: 47.5 | 44.2;
// top-2 of 128 4: 24.6 | 26.9, 8: 32.6 | 31.2; top-8 of 256 3.5: 35.7 | 37.6, 7: 42.1 | 38.5, 28: 75.7 | 64.5; of 512 4: 45.3 | 40.8.
static int64_t one_launch_values(int64_t E) { return E <= 64 ? (int64_t)16 << 20 : (int64_t)6 << 20; }
template <int KS>
__global__ __launch_bounds__(GRAD_THREADS) void router_dw_kernel(const RouterBwdArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[DW_LDS];
  grad_w<KS>(a, blockIdx.x, smem);
}
template <int CPL, int KP>
__global__ __launch_bounds__(DX_THREADS) void router_dx_list_kernel(const RouterBwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  grad_x_list<CPL, KP, DX_THREADS>(a, blockIdx.x, smem);
  reduce_parts(a, DX_THREADS);
}

// ---- host ---------------------------------------------------------------------------------------------------------

struct RouterBwdPlan {
  int ks;
  int64_t steps, splits, n_dw;
  size_t dlx, dlw, w, list, dbp, dwp, total;
};
static RouterBwdPlan router_bwd_plan(int64_t T, int64_t H, int64_t E) {
  RouterBwdPlan p;
  p.ks = E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 16;
  p.steps = (T + 31) / 32;
  // a workgroup of dw per CU where the tokens allow parts of eight steps: every part is written and read again
  const int64_t tiles = H / 128 * (p.ks > 8 ? p.ks / 8 : 1);
  p.splits = 256 / tiles;
  if (p.splits > p.steps / 8) p.splits = p.steps / 8;
  if (p.splits < 1) p.splits = 1;
  p.n_dw = tiles * p.splits;
  auto al = [](size_t v) { return (v + 255) & ~(size_t)255; };
  size_t off = 0;
  p.dlx = off; off += al((size_t)p.steps * 2 * p.ks * 2048);
  p.dlw = off; off += al((size_t)p.steps * 2 * p.ks * 2048);
  p.w = off; off += al((size_t)H / 64 * 4 * p.ks * 1024);  // (fragments, or [E][H])
  p.list = off; off += al((size_t)T * 8 * 8);
  p.dbp = off; off += al((size_t)p.steps * E * 4);
  p.dwp = off; off += p.splits > 1 ? al((size_t)p.splits * H * E * 4) : 0;
  p.total = off;
  return p;
}

constexpr int GRAD_LDS = 128 * 1024;  // 256 experts by 256 columns of w, or 512 by 128
template <int KS, int KP>
static int launch_grad(RouterBwdArgs& a, hipStream_t s) {
  const int64_t cols = KP == 0 ? GradX<KS>::COLS : KS > 8 ? 128 : 256, groups = (a.H + cols - 1) / cols;
  // dx: a job per CU, of 16 tokens at least
  a.x_splits = 256 / groups;
  if (a.x_splits > (a.T + 15) / 16) a.x_splits = (a.T + 15) / 16;
  if (a.x_splits < 1) a.x_splits = 1;
  const int64_t n_dx = groups * a.x_splits;
  if constexpr (KP > 0) {
    if (a.T * a.H > one_launch_values(a.E)) {
      constexpr int CPL = KS > 8 ? 2 : 4;
      if (allow_lds<router_dx_list_kernel<CPL, KP>>(GRAD_LDS) != hipSuccess) return MOE_E_LAUNCH;
      hipLaunchKernelGGL(router_dw_kernel<KS>, dim3((unsigned)a.n_dw), dim3(GRAD_THREADS), 0, s, a);
      MOE_CHECK_LAUNCH();
      hipLaunchKernelGGL((router_dx_list_kernel<CPL, KP>), dim3((unsigned)n_dx), dim3(DX_THREADS), (size_t)(a.E * cols * 2), s, a);
      MOE_CHECK_LAUNCH();
      return MOE_OK;
    }
  }
  const int dx = KP == 0 ? 2 * KS * 2048 : (int)(a.E * cols * 2);
  if (allow_lds<router_grad_kernel<KS, KP>>(GRAD_LDS) != hipSuccess) return MOE_E_LAUNCH;
  hipLaunchKernelGGL((router_grad_kernel<KS, KP>), dim3((unsigned)(a.n_dw + n_dx)), dim3(GRAD_THREADS), dx > DW_LDS ? dx : DW_LDS, s, a);
  MOE_CHECK_LAUNCH();
  if (a.splits > 1 || a.db) {
    const int64_t wgs = a.splits > 1 ? a.H * a.E / 1024 : 0, least = a.db ? (a.E + 3) / 4 : 1;
    hipLaunchKernelGGL(router_reduce_kernel, dim3((unsigned)(wgs > least ? wgs : least)), dim3(256), 0, s, a);
    MOE_CHECK_LAUNCH();
  }
  return MOE_OK;
}
template <int KS>
static int launch_router_bwd(RouterBwdArgs& a, const RouterBwdPlan& p, hipStream_t s) {
  constexpr int LDS = 32 * (32 * KS + 4) * 4;
  if (allow_lds<router_dlogits_kernel<KS>>(LDS) != hipSuccess) return MOE_E_LAUNCH;
  hipLaunchKernelGGL(router_dlogits_kernel<KS>, dim3((unsigned)(p.steps + a.H / 64)), dim3(256), LDS, s, a);
  MOE_CHECK_LAUNCH();
  return a.dense ? launch_grad<KS, 0>(a, s) : a.kp == 2 ? launch_grad<KS, 2>(a, s) : a.kp == 4 ? launch_grad<KS, 4>(a, s) : launch_grad<KS, 8>(a, s);
}

static int router_bwd_shape(int64_t T, int64_t H, int64_t E) {
  if (T < 1 || H < 1 || E < 1) return MOE_E_BAD_ARG;
  // (every launch stays below 2^32 threads: at these limits 2^21 + 2^14 workgroups of 256, 2^14 + 2^13 of 512)
  if (E > 512 || H % 128 != 0 || H > (int64_t)1 << 20 || T > (int64_t)1 << 26) return MOE_E_BAD_SHAPE;
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
  if ((((uintptr_t)workspace | (uintptr_t)x | (uintptr_t)d_x) & 15) != 0) return MOE_E_BAD_ARG;
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
  a.norm = router_pre_norm && norm_topk_prob;
  a.full = router_pre_norm && !norm_topk_prob && !mask_to_topk;
  a.dense = a.full || (a.softmax && router_pre_norm && !a.norm);
  a.kp = k > 4 ? 8 : k > 2 ? 4 : 2;
  a.dlx = (u32x4*)(ws + p.dlx);
  a.dlw = (u32x4*)(ws + p.dlw);
  a.wp = (u32x4*)(ws + p.w);
  a.wt = (uint16_t*)(ws + p.w);
  a.list = (uint2*)(ws + p.list);
  a.dbp = (float*)(ws + p.dbp);
  a.dx = (uint16_t*)d_x;
  a.dw = (uint16_t*)d_w;
  a.dwp = (float*)(ws + p.dwp);
  a.db = d_bias;
  a.db_dtype = bias_dtype;
  a.steps = p.steps; a.splits = p.splits; a.n_dw = p.n_dw;
  const hipStream_t s = (hipStream_t)stream;
  switch (p.ks) {
    case 2: return launch_router_bwd<2>(a, p, s);
    case 4: return launch_router_bwd<4>(a, p, s);
    case 8: return launch_router_bwd<8>(a, p, s);
    default: return launch_router_bwd<16>(a, p, s);
  }
}

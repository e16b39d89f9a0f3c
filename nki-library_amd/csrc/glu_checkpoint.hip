// The gated activation h = act(g) u with its inputs kept in 8 bits for the backward pass, and that backward pass.
//
// A record of R rows: e4m3 codes [R][2][I] (gate, then up) and one E8M0 scale byte per 32 neighbours of I, [R][2][ceil(I/32)].
// A value is code * 2^(byte - 127).  The scale is the smallest power of two that brings the group's largest finite magnitude to
// 448 or less: nothing saturates (the layer's own MX rule, which keeps the exponent of the largest value alone, clips what
// lies above 448/512 of the next power of two: up to an eighth of the values that matter most).  Dividing by it is exact, so each
// value is rounded once, by half a step of e4m3 (2^-4 of the value at most, 2^-10 of the scale where it is subnormal).
// Infinities and NaN become NaN codes and have no part in the scale: their neighbours keep their values.
//
//   forward    g, u -> h and the record of (g, u) as clamped
//   pack       the same record from moe_cte's checkpoint [N][2][I][B]
//   backward   record, dh -> du = dh act(g), dg = dh u act'(g) (0 at and beyond a clamp), and h again for the down weights'
//              gradient
//
// A clamped value is recorded as its limit rounded to e4m3 (7.2 as 7.0), so a record's value is at its clamp where it reaches
// what the record makes of the limit in its group, not the limit itself.  Values that were not clamped but round to the same
// code, up to half a step inside, cannot be told from those and count as clamped, unless the forward pass also keeps a bit per
// value (`clamped`, an eighth of a record's bytes, one for the eight values of a lane) and the backward pass goes by those.
//
// act(x) = x s(x) for every kind: SiLU and Swish s = sigmoid(a x); GELU s = Phi(x); its tanh form 0.5 (1 + tanh z) = sigmoid(2 z).
// All of it moves bytes: a pair of values costs 4 + 2 + 2 + 1/16 bytes forward in bf16, 2 + 1/16 + 2 + 4 + 2 backward.  Four lanes
// share a group of 32, eight values each (16 bytes of bf16), so that a group's maximum is two exchanges between neighbours.
// Rows of padding slots have no part in a result and zero outputs: the forward pass works them out as zeros, the backward pass
// leaves them out, neither reads them; the pack reads what lies in a tile beside a token's row.
// Measured: forward, fp16, 9088 rows (8192 of tokens) of I = 14336 174 us = 5.7 TB/s; backward, bf16, 98048 rows (65536) of 2048
// 282 us = 6.2 TB/s, 296 with stores that stay in the caches, 286 with such loads; pack of 1408 rows (512) of 1024 8.7 us, of
// which the bytes are 2 (with 2-byte loads and a lookup of the row's id for each 14).  A copy moves 4.9 TB/s, a fill 6.9.
// 98048 rows (65536) of 2048, forward | backward, us: bf16 SiLU 230 | 278, Swish with clamps 263 | 288, with their bits 302 |
// 286, GELU (erfc: arithmetic) 372 | 355; fp32 456 | 680.
#include <type_traits>

#include "rows.hpp"

namespace moe {

struct GluArgs {
  const int32_t* tp2id;  // [R] or null: every row counts
  int64_t n_tokens, R;
  int64_t I, V;          // V: pieces of eight values per row of I, a multiple of four (those past I are empty)
  uint32_t v_magic;      // ceil(2^32 / V)
  int clamp_mask;
  float clamp[4];        // gate upper, gate lower, up upper, up lower
  float clamp16[4];      // the same as bf16 holds them: what the layer's checkpoint has of a clamped value
  uint8_t* clamped;      // [R][2][ceil(I/8)] or null: bit i of byte v for value 8 v + i
};

// s(x) and x s'(x).  EXACT (fp32 rows): the exponent's rounding is made good; it costs up to |z| / 2 units of the last place, which
// rows of 16 bits do not see.
template <int ACT, bool EXACT>
__device__ __forceinline__ void act_parts(float x, float& s, float& xds) {
  if constexpr (ACT == MOE_ACT_GELU) {
    s = 0.5f * erfcf(x * -0.70710678118654752440f);
    const float d = __builtin_amdgcn_exp2f(-0.72134752044448170368f * x * x) * 0.39894228040143267794f;
    xds = d == 0.f ? 0.f : x * d;
  } else {
    float z = x, dz = 1.f;
    if constexpr (ACT == MOE_ACT_SWISH) {
      z = 1.702f * x;
      dz = 1.702f;
    }
    if constexpr (ACT == MOE_ACT_GELU_TANH) {
      z = 1.59576912160573071176f * (x + 0.044715f * x * x * x);
      dz = 1.59576912160573071176f * (1.f + 0.134145f * x * x);
    }
    const float t = z * -1.44269504088896340736f;
    float e = __builtin_amdgcn_exp2f(t);
    if constexpr (EXACT) {
      const float lost = fmaf(z, -1.44269504088896340736f, -t) + z * -1.925963e-8f;  // log2 e = 1.4426950216.. + 1.9e-8
      if (fabsf(t) < 128.f) e = fmaf(e, lost * 0.69314718055994530942f, e);
    }
    s = __builtin_amdgcn_rcpf(1.f + e);
    // 1 - s = e s, which loses nothing where s is near one; where e overflows, s is zero and the product would be NaN
    const float both = s * (e > 1e30f ? 1.f : e * s);
    xds = both == 0.f ? 0.f : x * dz * both;  // (an infinite x, or dz, beside a slope of zero)
  }
}

__device__ __forceinline__ float clamp_value(float x, int mask, int hi_bit, int lo_bit, float hi, float lo) {
  // (comparisons that a NaN fails: it stays)
  if ((mask & hi_bit) && x > hi) x = hi;
  if ((mask & lo_bit) && x < lo) x = lo;
  return x;
}

// (NaN is at no limit)
__device__ __forceinline__ bool at_limit(float x, int mask, int hi_bit, int lo_bit, float hi, float lo) {
  return ((mask & hi_bit) && x >= hi) || ((mask & lo_bit) && x <= lo);
}

__device__ __forceinline__ uint32_t max_finite(uint32_t m, float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u && b > m ? b : m;
}
// Bits of the largest finite magnitude -> scale byte.
__device__ __forceinline__ uint32_t scale_of(uint32_t m) {
  const int s = (int)(m >> 23) - 8 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return (uint32_t)(s < 0 ? 0 : s);
}
// The scale byte of a group that four neighbouring lanes hold.
__device__ __forceinline__ uint32_t group_scale(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max_finite(m, v[i]);
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, true);  // lanes 1 0 3 2 of each four
  m = o > m ? o : m;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, true);  // 2 3 0 1
  return scale_of(o > m ? o : m);
}
// Eight values -> eight codes.  (The values are at most 448 by then; infinities and NaN are written as such.)
__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t scale) {
  const float inv = mx_inv_scale(scale);
  uint32_t out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    out[h] = pack4_e4m3(v[4 * h] * inv, v[4 * h + 1] * inv, v[4 * h + 2] * inv, v[4 * h + 3] * inv);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((__float_as_uint(v[4 * h + i]) & 0x7f800000u) == 0x7f800000u) out[h] |= 0x7fu << (8 * i);
  }
  return make_uint2(out[0], out[1]);
}
__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 0x00400000u); }
__device__ __forceinline__ void decode8(const uint2& c, uint32_t byte, float (&v)[8]) {
  const float s = scale_value(byte);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = (int)(h ? c.y : c.x);
    const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    v[4 * h] = a[0] * s;
    v[4 * h + 1] = a[1] * s;
    v[4 * h + 2] = b[0] * s;
    v[4 * h + 3] = b[1] * s;
  }
}
// The limits of a gate or up group as its record holds them.  The value recorded is the limit itself or, by way of moe_cte's
// checkpoint, its bf16, which may round to another code (7.2503 to 7.5, its bf16 7.25 to 7.0): the one further inside.  A limit
// above 448 times the scale is above every value of the group and stays what it is.
__device__ __forceinline__ void recorded_limits(const GluArgs& a, int upper, uint32_t byte, float& hi, float& lo) {
  const float inv = mx_inv_scale(byte), s = scale_value(byte);
  const float v[4] = {a.clamp[upper], a.clamp16[upper], a.clamp[upper + 1], a.clamp16[upper + 1]};
  const int w = (int)pack4_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  const v2f h = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), l = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  const float r[4] = {h[0] * s, h[1] * s, l[0] * s, l[1] * s};
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = fabsf(v[i] * inv) <= 448.f ? r[i] : v[i];
  hi = fminf(q[0], q[1]);
  lo = fmaxf(q[2], q[3]);
}

// n of eight values of a row at p (n = 8 except at the end of a row whose length is no multiple of eight)
template <int DT>
__device__ __forceinline__ void load8(const uint8_t* p, int n, float (&v)[8]) {
  typedef Elem<DT> EL;
  if (n == 8) {
#pragma unroll
    for (int q = 0; q < 8 / EL::N; ++q) {
      float part[EL::N];
      unpack<DT>(load_piece<DT>(p + 16 * q), part);
#pragma unroll
      for (int i = 0; i < EL::N; ++i) v[q * EL::N + i] = part[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? elem_to_f32<DT>(((const typename EL::raw*)p)[i]) : 0.f;
  }
}
template <int DT>
__device__ __forceinline__ void store8(uint8_t* p, int n, const float (&v)[8]) {
  typedef Elem<DT> EL;
  if (n == 8) {
#pragma unroll
    for (int q = 0; q < 8 / EL::N; ++q) {
      float part[EL::N];
#pragma unroll
      for (int i = 0; i < EL::N; ++i) part[i] = v[q * EL::N + i];
      store_piece<DT>(p + 16 * q, pack<DT>(part));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) ((typename EL::raw*)p)[i] = f32_to_elem<DT>(v[i]);
  }
}
typedef uint32_t codes8 __attribute__((ext_vector_type(2), aligned(1)));
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int n) {
  if (n == 8) {
    const codes8 c = __builtin_nontemporal_load((const codes8*)p);
    return make_uint2(c[0], c[1]);
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i / 4] |= (uint32_t)p[i] << (8 * (i % 4));
  return make_uint2(w[0], w[1]);
}
template <bool PAST = true>
__device__ __forceinline__ void store_codes(uint8_t* p, int n, const uint2& c) {
  if (n == 8) {
    if (PAST) __builtin_nontemporal_store((codes8{c.x, c.y}), (codes8*)p);
    else *(codes8*)p = codes8{c.x, c.y};
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i % 4)));
}

// The pieces of all rows, one after the other, are dealt to the threads: no lane is left over at the end of a row.
// Piece -> row and place in it: the workgroup's first piece by a division, the others from there by multiplication.
struct Place {
  int64_t row;
  int v, n;  // piece of the row, values in it
  bool in, on;  // a row; one that is not padding
};
__device__ __forceinline__ Place place_of(const GluArgs& a) {
  // (a launch has fewer than 2^32 pieces: 32 bits, a division in 64 would take longer than the rest of a piece's arithmetic)
  const uint32_t V = (uint32_t)a.V, base = blockIdx.x * 256u, row0 = base / V;
  Place p;
  const uint32_t j = base - row0 * V + threadIdx.x, dr = __umulhi(j, a.v_magic);
  p.row = (int64_t)row0 + dr;
  p.v = (int)(j - dr * V);
  p.in = p.row < a.R;
  p.on = p.in;
  if (p.in && a.tp2id) {
    const int id = a.tp2id[p.row];
    p.on = id >= 0 && id < a.n_tokens;
  }
  const int64_t left = a.I - 8 * (int64_t)p.v;
  p.n = left >= 8 ? 8 : left > 0 ? (int)left : 0;
  return p;
}

template <int DT, int ACT>
__global__ __launch_bounds__(256) void glu_checkpoint_kernel(const GluArgs a, const uint8_t* __restrict__ gate_up,
                                                             uint8_t* __restrict__ h, uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
  constexpr int ES = Elem<DT>::SIZE;
  const Place p = place_of(a);
  if (!p.in) return;  // (whole groups of four lanes: V is a multiple of four)
  const int64_t G = a.V / 4, off = p.row * 2 * a.I + 8 * p.v;
  float g[8], u[8], r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = u[i] = r[i] = 0.f;
  if (p.on && p.n > 0) {
    load8<DT>(gate_up + off * ES, p.n, g);
    load8<DT>(gate_up + (off + a.I) * ES, p.n, u);
  }
  if (a.clamped && p.n > 0) {
    uint32_t at_g = 0, at_u = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool real = p.on && i < p.n;
      if (real && at_limit(g[i], a.clamp_mask, MOE_CLAMP_GATE_HI, MOE_CLAMP_GATE_LO, a.clamp[0], a.clamp[1])) at_g |= 1u << i;
      if (real && at_limit(u[i], a.clamp_mask, MOE_CLAMP_UP_HI, MOE_CLAMP_UP_LO, a.clamp[2], a.clamp[3])) at_u |= 1u << i;
    }
    const int64_t G8 = (a.I + 7) / 8;
    a.clamped[p.row * 2 * G8 + p.v] = (uint8_t)at_g;
    a.clamped[p.row * 2 * G8 + G8 + p.v] = (uint8_t)at_u;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (a.clamp_mask) {
      g[i] = clamp_value(g[i], a.clamp_mask, MOE_CLAMP_GATE_HI, MOE_CLAMP_GATE_LO, a.clamp[0], a.clamp[1]);
      u[i] = clamp_value(u[i], a.clamp_mask, MOE_CLAMP_UP_HI, MOE_CLAMP_UP_LO, a.clamp[2], a.clamp[3]);
      if (!p.on || i >= p.n) g[i] = u[i] = 0.f;
    }
    float s, xds;
    act_parts<ACT, DT == MOE_DT_FP32>(g[i], s, xds);
    r[i] = g[i] * s * u[i];
  }
  const uint32_t sg = group_scale(g), su = group_scale(u);
  if (p.n > 0) {
    store8<DT>(h + (p.row * a.I + 8 * p.v) * ES, p.n, r);
    store_codes(codes + off, p.n, encode8(g, sg));
    store_codes(codes + off + a.I, p.n, encode8(u, su));
  }
  if ((p.v & 3) == 0) {
    scales[p.row * 2 * G + p.v / 4] = (uint8_t)sg;
    scales[p.row * 2 * G + G + p.v / 4] = (uint8_t)su;
  }
}

// Waves per SIMD: four at most for fp32 rows, eight for rows of 16 bits; 98048 rows (65536) of 2048 take, us, with four and with
// eight: fp32 680 and 720, bf16 299 and 278.
template <int DT, int ACT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, DT == MOE_DT_FP32 ? 4 : 8)))
void glu_checkpoint_bwd_kernel(const GluArgs a, const uint8_t* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales,
                                                                 const uint8_t* __restrict__ dh, uint8_t* __restrict__ d_gate_up,
                                                                 uint8_t* __restrict__ h) {
  constexpr int ES = Elem<DT>::SIZE;
  const Place p = place_of(a);
  if (!p.in || p.n == 0) return;
  const int64_t G = a.V / 4, off = p.row * 2 * a.I + 8 * p.v;
  float dg[8], du[8], r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dg[i] = du[i] = r[i] = 0.f;
  if (p.on) {
    float g[8], u[8], d[8];
    const uint2 cg = load_codes(codes + off, p.n), cu = load_codes(codes + off + a.I, p.n);
    const uint32_t sg = scales[p.row * 2 * G + p.v / 4], su = scales[p.row * 2 * G + G + p.v / 4];
    load8<DT>(dh + (p.row * a.I + 8 * p.v) * ES, p.n, d);
    decode8(cg, sg, g);
    decode8(cu, su, u);
    float g_hi = 0.f, g_lo = 0.f, u_hi = 0.f, u_lo = 0.f;
    uint32_t at_g = 0, at_u = 0;
    if (a.clamped) {
      const int64_t G8 = (a.I + 7) / 8;
      at_g = a.clamped[p.row * 2 * G8 + p.v];
      at_u = a.clamped[p.row * 2 * G8 + G8 + p.v];
    } else if (a.clamp_mask) {
      recorded_limits(a, 0, sg, g_hi, g_lo);
      recorded_limits(a, 2, su, u_hi, u_lo);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bool in_g = !(at_g >> i & 1), in_u = !(at_u >> i & 1);
      if (a.clamp_mask) {
        const float g0 = g[i], u0 = u[i];
        g[i] = clamp_value(g0, a.clamp_mask, MOE_CLAMP_GATE_HI, MOE_CLAMP_GATE_LO, a.clamp[0], a.clamp[1]);
        u[i] = clamp_value(u0, a.clamp_mask, MOE_CLAMP_UP_HI, MOE_CLAMP_UP_LO, a.clamp[2], a.clamp[3]);
        if (!a.clamped) {
          in_g = !at_limit(g0, a.clamp_mask, MOE_CLAMP_GATE_HI, MOE_CLAMP_GATE_LO, g_hi, g_lo);
          in_u = !at_limit(u0, a.clamp_mask, MOE_CLAMP_UP_HI, MOE_CLAMP_UP_LO, u_hi, u_lo);
        }
      }
      float s, xds;
      act_parts<ACT, DT == MOE_DT_FP32>(g[i], s, xds);
      const float act = g[i] * s;
      r[i] = act * u[i];
      du[i] = in_u ? d[i] * act : 0.f;
      dg[i] = in_g ? d[i] * u[i] * (s + xds) : 0.f;
    }
  }
  store8<DT>(d_gate_up + off * ES, p.n, dg);
  store8<DT>(d_gate_up + (off + a.I) * ES, p.n, du);
  if (h) store8<DT>(h + (p.row * a.I + 8 * p.v) * ES, p.n, r);
}

// codes and scales -> values.  (The values of one row and half behind one another: rows of I, scales of G.)
template <int DT>
__global__ __launch_bounds__(256) void dequantize_checkpoint_kernel(const GluArgs a, const uint8_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ scales, uint8_t* __restrict__ out) {
  const Place p = place_of(a);
  if (!p.in || p.n == 0) return;
  const int64_t off = p.row * a.I + 8 * p.v;
  float v[8];
  decode8(load_codes(codes + off, p.n), scales[p.row * (a.V / 4) + p.v / 4], v);
  store8<DT>(out + off * Elem<DT>::SIZE, p.n, v);
}

// ---- pack ---------------------------------------------------------------------------------------------------------

// The checkpoint of moe_cte has a block's rows side by side: [N][2 I][B].  A workgroup takes a tile of tb rows x tc columns (tb a
// power of two up to 64, tb * tc = PACK_TILE, tc a multiple of 32) through LDS: read in pieces of eight neighbours, 16 bytes, then
// a row and a group of 32 columns per thread.  Two bytes per value from LDS: neighbouring lanes hold neighbouring rows.
// (Groups lie max(8, tb) values apart beyond their length, so that lanes of several groups do not meet in a bank.)
constexpr int PACK_TILE = 8192;
// The limits of gate and of up as the checkpoint holds them (bf16; NaN, which nothing reaches, where there is none), for `out`:
// which values lie there.
struct PackClamps {
  float hi[2], lo[2];
  uint8_t* out;  // [N B][2][ceil(I/8)] or null
};
__global__ __launch_bounds__(256) void pack_checkpoint_kernel(const uint16_t* __restrict__ x, const int32_t* __restrict__ tp2id,
                                                              int64_t n_tokens, int64_t I, int64_t B, int ltb, const PackClamps at,
                                                              uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  __shared__ __attribute__((aligned(16))) uint16_t s_x[PACK_TILE + PACK_TILE / 32 * 8];
  const int tid = threadIdx.x, tb = 1 << ltb, tc = PACK_TILE >> ltb, pad = tb > 8 ? tb : 8;
  const int64_t G = (I + 31) / 32, tiles_c = (I + tc - 1) / tc, tiles_b = (B + tb - 1) / tb;
  uint32_t i = blockIdx.x;  // (divided in 32 bits: the tiles of one block are fewer than 2^24)
  const int64_t ci = i % (uint32_t)tiles_c;
  i /= (uint32_t)tiles_c;
  const int64_t z = i % 2;
  i /= 2;
  const int64_t bi = i % (uint32_t)tiles_b, blk = i / (uint32_t)tiles_b;
  const int64_t c0 = ci * tc, r0 = bi * tb;
  const int nc = (int)(I - c0 < tc ? I - c0 : tc), nr = (int)(B - r0 < tb ? B - r0 : tb);
  // the thread's row and group; a tile of padding alone is not read
  const int r = tid & (tb - 1), cg = tid >> ltb;
  bool on = r < nr;
  if (tp2id && on) {
    const int id = tp2id[blk * B + r0 + r];
    on = id >= 0 && id < n_tokens;
  }
  const bool any = __syncthreads_or(on);
  const uint16_t* src = x + ((blk * 2 + z) * I + c0) * B + r0;
  auto place = [&](int c, int row) { return c / 32 * (32 * tb + pad) + (c % 32) * tb + row; };
  if (any) {
    if (((B % 8 == 0 && tb >= 8) || B == tb) && ((uintptr_t)src & 15) == 0 && nc * tb % 8 == 0) {
      u32x4 d[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int e = 8 * (tid + 256 * q), c = e >> ltb, row = e & (tb - 1);
        d[q] = u32x4{0, 0, 0, 0};
        if (c < nc && row < nr) d[q] = __builtin_nontemporal_load((const u32x4*)(src + (int64_t)c * B + row));
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int e = 8 * (tid + 256 * q);
        *(u32x4*)(s_x + place(e >> ltb, e & (tb - 1))) = d[q];
      }
    } else {
      for (int e = tid; e < PACK_TILE; e += 256) {
        const int c = e >> ltb, row = e & (tb - 1);
        s_x[place(c, row)] = c < nc && row < nr ? src[(int64_t)c * B + row] : (uint16_t)0;
      }
    }
  }
  __syncthreads();
  const int left = nc - 32 * cg;
  if (r >= nr || left <= 0) return;
  float v[32];
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    v[c] = on && c < left ? bf16_bits_to_f32(s_x[cg * (32 * tb + pad) + c * tb + r]) : 0.f;
    m = max_finite(m, v[c]);
  }
  const uint32_t s = scale_of(m);
  const int64_t row = (blk * B + r0 + r) * 2 + z;
  uint8_t* dst = codes + row * I + c0 + 32 * cg;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float part[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) part[e] = v[8 * q + e];
    const int n = left - 8 * q;
    // (not past the caches: a row's 128 bytes come from several waves)
    if (n > 0) store_codes<false>(dst + 8 * q, n > 8 ? 8 : n, encode8(part, s));
  }
  scales[row * G + c0 / 32 + cg] = (uint8_t)s;
  if (at.out) {
    const float hi = z ? at.hi[1] : at.hi[0], lo = z ? at.lo[1] : at.lo[0];
    uint8_t* bytes = at.out + row * ((I + 7) / 8) + c0 / 8 + 4 * cg;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (on && 8 * q + e < left && (v[8 * q + e] >= hi || v[8 * q + e] <= lo)) m |= 1u << e;
      if (8 * q < left) bytes[q] = (uint8_t)m;
    }
  }
}

}  // namespace moe

using namespace moe;

// bf16 of a value, rounded to the nearest even.
static float as_bf16(float f) {
  uint32_t u;
  __builtin_memcpy(&u, &f, 4);
  if ((u & 0x7fffffffu) < 0x7f800000u) u += 0x7fffu + ((u >> 16) & 1u);
  u &= 0xffff0000u;
  __builtin_memcpy(&f, &u, 4);
  return f;
}
static int glu_args(GluArgs& a, int64_t R, int64_t I, int act_fn, int clamp_mask, const float* clamps, const int32_t* tp2id,
                    int64_t n_tokens, int64_t rows = (int64_t)1 << 31) {
  if (R < 0 || I < 1 || n_tokens < 0) return MOE_E_BAD_ARG;
  if (act_fn < MOE_ACT_SILU || act_fn > MOE_ACT_SWISH || (clamp_mask & ~15) || (clamp_mask && !clamps)) return MOE_E_BAD_ARG;
  // (the place of a piece within its workgroup's rows is found by a 32-bit multiplication, exact up to here)
  if (I > 1 << 17 || R >= rows) return MOE_E_BAD_SHAPE;
  a.tp2id = tp2id;
  a.n_tokens = n_tokens;
  a.R = R;
  a.I = I;
  a.V = (I + 31) / 32 * 4;
  a.v_magic = (uint32_t)((((uint64_t)1 << 32) + a.V - 1) / a.V);
  a.clamp_mask = clamp_mask;
  a.clamped = nullptr;
  for (int i = 0; i < 4; ++i) {
    a.clamp[i] = clamp_mask ? clamps[i] : 0.f;
    a.clamp16[i] = as_bf16(a.clamp[i]);
  }
  return MOE_OK;
}
// Rows per launch: fewer than 2^32 threads, and at least one row.
static int64_t rows_per_launch(const GluArgs& a) { return (((int64_t)1 << 32) - 256) / a.V; }

template <class F>
static int by_act(int act, F&& f) {
  switch (act) {
    case MOE_ACT_SILU: return f(std::integral_constant<int, MOE_ACT_SILU>{});
    case MOE_ACT_GELU: return f(std::integral_constant<int, MOE_ACT_GELU>{});
    case MOE_ACT_GELU_TANH: return f(std::integral_constant<int, MOE_ACT_GELU_TANH>{});
    default: return f(std::integral_constant<int, MOE_ACT_SWISH>{});
  }
}
template <class F>
static int by_dtype(int dtype, F&& f) {
  switch (dtype) {
    case MOE_DT_BF16: return f(std::integral_constant<int, MOE_DT_BF16>{});
    case MOE_DT_FP16: return f(std::integral_constant<int, MOE_DT_FP16>{});
    case MOE_DT_FP32: return f(std::integral_constant<int, MOE_DT_FP32>{});
    default: return MOE_E_BAD_ARG;
  }
}

extern "C" int moe_glu_checkpoint_clamped(const void* gate_up, int dtype, int64_t R, int64_t I, int act_fn, int clamp_mask,
                                          const float* clamps, const int32_t* token_position_to_id, int64_t n_tokens,
                                          void* intermediate, uint8_t* codes, uint8_t* scales, uint8_t* clamped, void* stream) {
  if (!gate_up || !intermediate || !codes || !scales) return MOE_E_BAD_ARG;
  GluArgs a;
  const int rc = glu_args(a, R, I, act_fn, clamp_mask, clamps, token_position_to_id, n_tokens);
  if (rc != MOE_OK) return rc;
  return by_dtype(dtype, [&](auto dt) {
    return by_act(act_fn, [&](auto act) {
      constexpr int DT = decltype(dt)::value, ES = Elem<DT>::SIZE;
      const int64_t per = rows_per_launch(a);
      for (int64_t r0 = 0; r0 < R; r0 += per) {
        GluArgs p = a;
        p.R = R - r0 < per ? R - r0 : per;
        if (p.tp2id) p.tp2id += r0;
        if (clamped) p.clamped = clamped + r0 * 2 * ((I + 7) / 8);
        hipLaunchKernelGGL((glu_checkpoint_kernel<DT, decltype(act)::value>), dim3((unsigned)((p.R * p.V + 255) / 256)), dim3(256),
                           0, (hipStream_t)stream, p, (const uint8_t*)gate_up + r0 * 2 * I * ES,
                           (uint8_t*)intermediate + r0 * I * ES, codes + r0 * 2 * I, scales + r0 * (p.V / 2));
        MOE_CHECK_LAUNCH();
      }
      return MOE_OK;
    });
  });
}

extern "C" int moe_glu_checkpoint(const void* gate_up, int dtype, int64_t R, int64_t I, int act_fn, int clamp_mask,
                                  const float* clamps, const int32_t* token_position_to_id, int64_t n_tokens,
                                  void* intermediate, uint8_t* codes, uint8_t* scales, void* stream) {
  return moe_glu_checkpoint_clamped(gate_up, dtype, R, I, act_fn, clamp_mask, clamps, token_position_to_id, n_tokens, intermediate,
                                    codes, scales, nullptr, stream);
}

extern "C" int moe_glu_checkpoint_bwd_clamped(const uint8_t* codes, const uint8_t* scales, const uint8_t* clamped,
                                              const void* d_intermediate, int dtype, int64_t R, int64_t I, int act_fn,
                                              int clamp_mask, const float* clamps, const int32_t* token_position_to_id,
                                              int64_t n_tokens, void* d_gate_up, void* intermediate, void* stream) {
  if (!codes || !scales || !d_intermediate || !d_gate_up) return MOE_E_BAD_ARG;
  GluArgs a;
  const int rc = glu_args(a, R, I, act_fn, clamp_mask, clamps, token_position_to_id, n_tokens);
  if (rc != MOE_OK) return rc;
  return by_dtype(dtype, [&](auto dt) {
    return by_act(act_fn, [&](auto act) {
      constexpr int DT = decltype(dt)::value, ES = Elem<DT>::SIZE;
      const int64_t per = rows_per_launch(a);
      for (int64_t r0 = 0; r0 < R; r0 += per) {
        GluArgs p = a;
        p.R = R - r0 < per ? R - r0 : per;
        if (p.tp2id) p.tp2id += r0;
        if (clamped) p.clamped = const_cast<uint8_t*>(clamped) + r0 * 2 * ((I + 7) / 8);
        hipLaunchKernelGGL((glu_checkpoint_bwd_kernel<DT, decltype(act)::value>), dim3((unsigned)((p.R * p.V + 255) / 256)),
                           dim3(256), 0, (hipStream_t)stream, p, codes + r0 * 2 * I, scales + r0 * (p.V / 2),
                           (const uint8_t*)d_intermediate + r0 * I * ES, (uint8_t*)d_gate_up + r0 * 2 * I * ES,
                           intermediate ? (uint8_t*)intermediate + r0 * I * ES : nullptr);
        MOE_CHECK_LAUNCH();
      }
      return MOE_OK;
    });
  });
}

extern "C" int moe_glu_checkpoint_bwd(const uint8_t* codes, const uint8_t* scales, const void* d_intermediate, int dtype, int64_t R,
                                      int64_t I, int act_fn, int clamp_mask, const float* clamps,
                                      const int32_t* token_position_to_id, int64_t n_tokens, void* d_gate_up,
                                      void* intermediate, void* stream) {
  return moe_glu_checkpoint_bwd_clamped(codes, scales, nullptr, d_intermediate, dtype, R, I, act_fn, clamp_mask, clamps,
                                        token_position_to_id, n_tokens, d_gate_up, intermediate, stream);
}

extern "C" int moe_dequantize_checkpoint(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t I, void* out, int dtype,
                                         void* stream) {
  if (!codes || !scales || !out) return MOE_E_BAD_ARG;
  GluArgs a;
  // (a record of R rows has 2 R here)
  const int rc = glu_args(a, rows, I, MOE_ACT_SILU, 0, nullptr, nullptr, 0, (int64_t)1 << 32);
  if (rc != MOE_OK) return rc;
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const int64_t per = rows_per_launch(a);
    for (int64_t r0 = 0; r0 < rows; r0 += per) {
      GluArgs p = a;
      p.R = rows - r0 < per ? rows - r0 : per;
      hipLaunchKernelGGL(dequantize_checkpoint_kernel<DT>, dim3((unsigned)((p.R * p.V + 255) / 256)), dim3(256), 0,
                         (hipStream_t)stream, p, codes + r0 * I, scales + r0 * (p.V / 4), (uint8_t*)out + r0 * I * Elem<DT>::SIZE);
      MOE_CHECK_LAUNCH();
    }
    return MOE_OK;
  });
}

extern "C" int moe_pack_gate_up_checkpoint_clamped(const void* gate_up_activations_T, int64_t N, int64_t I, int64_t B, int clamp_mask,
                                                   const float* clamps, const int32_t* token_position_to_id, int64_t n_tokens,
                                                   uint8_t* codes, uint8_t* scales, uint8_t* clamped, void* stream) {
  if (!gate_up_activations_T || !codes || !scales || N < 0 || I < 1 || B < 1 || n_tokens < 0) return MOE_E_BAD_ARG;
  if ((clamp_mask & ~15) || (clamp_mask && !clamps)) return MOE_E_BAD_ARG;
  if (I > 1 << 17 || N >= (int64_t)1 << 31 || B >= (int64_t)1 << 31 || N * B >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  int ltb = 0;
  while (ltb < 6 && (1 << ltb) < B) ++ltb;
  const int tb = 1 << ltb, tc = PACK_TILE >> ltb;
  const int64_t per_block = (I + tc - 1) / tc * 2 * ((B + tb - 1) / tb);
  const int64_t blocks = (((int64_t)1 << 24) - 1) / per_block;  // (of a launch: fewer than 2^32 threads)
  if (blocks < 1) return MOE_E_BAD_SHAPE;
  const int64_t G = (I + 31) / 32;
  constexpr int HI[2] = {MOE_CLAMP_GATE_HI, MOE_CLAMP_UP_HI}, LO[2] = {MOE_CLAMP_GATE_LO, MOE_CLAMP_UP_LO};
  PackClamps at;
  for (int z = 0; z < 2; ++z) {
    at.hi[z] = clamp_mask & HI[z] ? as_bf16(clamps[2 * z]) : __builtin_nanf("");
    at.lo[z] = clamp_mask & LO[z] ? as_bf16(clamps[2 * z + 1]) : __builtin_nanf("");
  }
  for (int64_t n0 = 0; n0 < N; n0 += blocks) {
    const int64_t n = N - n0 < blocks ? N - n0 : blocks;
    at.out = clamped ? clamped + n0 * B * 2 * ((I + 7) / 8) : nullptr;
    hipLaunchKernelGGL(pack_checkpoint_kernel, dim3((unsigned)(n * per_block)), dim3(256), 0, (hipStream_t)stream,
                       (const uint16_t*)gate_up_activations_T + n0 * 2 * I * B,
                       token_position_to_id ? token_position_to_id + n0 * B : nullptr, n_tokens, I, B, ltb, at,
                       codes + n0 * B * 2 * I, scales + n0 * B * 2 * G);
    MOE_CHECK_LAUNCH();
  }
  return MOE_OK;
}

extern "C" int moe_pack_gate_up_checkpoint(const void* gate_up_activations_T, int64_t N, int64_t I, int64_t B,
                                           const int32_t* token_position_to_id, int64_t n_tokens, uint8_t* codes, uint8_t* scales,
                                           void* stream) {
  return moe_pack_gate_up_checkpoint_clamped(gate_up_activations_T, N, I, B, 0, nullptr, token_position_to_id, n_tokens, codes, scales,
                                             nullptr, stream);
}

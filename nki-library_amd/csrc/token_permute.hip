// Tokens into the order of the block table and back, with their gradients.
//
//   permute           out[s] = x[id(s)]                           0 where slot s holds padding
//   permute, backward dx[t]  = sum over the slots s of t of d[s]
//   combine           out[t] = sum over the slots s of t of a[t, e(s)] y[s]
//   combine, backward dy[s]  = a[t, e(s)] dout[t],  da[t, e] = sum over t's slots s of e of <dout[t], y[s]>
//
// id(s) = token_position_to_id[s], padding where it is no token; e(s) = block_to_expert[s / B].  All four move rows and
// hardly compute: their bound is memory.  Sums run over the slots in ascending order in 32 bits and are rounded once, so
// that a result depends on its inputs alone.  (The layer's own combine, combine.hip, adds in bf16 as the reference does.)
//
// T = 8192 tokens of 14 KB in 8 of 98048 slots: combine 202 us with its list (5.2 TB/s), its backward pass 500 (4.9; 5.3 without
// list and launches); T = 8192, 4 KB, 8 of 81792 52 us = 5.8 TB/s.  A copy moves 4.9.
//
// All but permute work by token: a token's row is read or written once whatever k is.  They go by a list of every token's slots,
// which token_slots_kernel inverts the table into.
#include <type_traits>

#include "rows.hpp"

namespace moe {

constexpr int SLOTS_MAX_K = 64;        // most slots a list holds per token
constexpr int SLOTS_LDS_WORDS = 12288;  // 48 KB of lists per workgroup
// Entries that the workgroups of token_slots_kernel read in all, at most: as many as slots times workgroups, which grow with the tokens
// from 256 * SLOTS_LDS_WORDS / (1 + k) on.  The whole table in every workgroup | global counters, us: 8192 tokens in 8 of 98 k slots
// 8.0 | 10.9 (2^24.6 entries), 262 k in 8 of 2.1 M 85 | 68 (2^29), 131 k in 16 of 2.2 M 92 | 122 (2^29.1), 400 k in 8 of 3.3 M
// 244 | 151 (2^29.9), 131 k in 32 of 4.3 M 323 | 365, 262 k in 16 of 4.3 M 313 | 254 (2^30.5 both), 80 k in 64 of 5.2 M 393 | 377 (2^31).
constexpr int64_t LISTS_WHOLE_TABLE = (int64_t)1 << 30;

// lists [T][1 + k]: how many slots the token has (more than k: the list is cut), its slots ascending, -1 behind them.
// The lists of nt tokens from t0 on, whose slots were taken in any order into s_list: each goes to the place that its rank names.
__device__ __forceinline__ void write_ranked(const int* s_list, int nt, int64_t t0, int k, int32_t* __restrict__ lists) {
  const int w = 1 + k;
  for (int i = threadIdx.x; i < nt * w; i += 1024) {
    const int t = i / w, j = i - t * w, n = s_list[t * w], held = n < k ? n : k;
    int32_t* out = lists + (t0 + t) * w;
    if (j == 0) {
      out[0] = n;
    } else if (j > held) {
      out[j] = -1;
    } else {
      const int mine = s_list[t * w + j];
      int rank = 1;
      for (int o = 1; o <= held; ++o) rank += s_list[t * w + o] < mine;
      out[rank] = mine;
    }
  }
}
// A workgroup owns `range` tokens and reads the whole table, which the L2 hands out: a table of 98 k slots is 0.4 MB, and
// one launch without global atomics or cleared counters is shorter than the two that those would take.
__global__ __launch_bounds__(1024) void token_slots_kernel(const int32_t* __restrict__ tp2id, int64_t S, int64_t T, int k,
                                                           int range, int32_t* __restrict__ lists) {
  __shared__ int s_list[SLOTS_LDS_WORDS];
  const int64_t t0 = (int64_t)blockIdx.x * range;
  const int nt = (int)(T - t0 < range ? T - t0 : range), w = 1 + k;
  for (int i = threadIdx.x; i < nt; i += 1024) s_list[i * w] = 0;
  __syncthreads();
  // (unsigned: whatever lies outside of the range, negative ids too, is far above it)
  auto mine = [&](int id) { return (uint32_t)id - (uint32_t)t0 < (uint32_t)nt; };
  auto take = [&](int64_t s, int id) {
    if (mine(id)) {
      const int t = (int)((uint32_t)id - (uint32_t)t0), p = atomicAdd(&s_list[t * w], 1);
      if (p < k) s_list[t * w + 1 + p] = (int)s;
    }
  };
  const int64_t n4 = ((uintptr_t)tp2id & 15) == 0 ? S / 4 : 0;
  constexpr int U = 8;
  for (int64_t i0 = threadIdx.x; i0 < n4; i0 += 1024 * U) {
    int4 d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      d[u] = make_int4(-1, -1, -1, -1);
      if (i0 + 1024 * u < n4) d[u] = ((const int4*)tp2id)[i0 + 1024 * u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = 4 * (i0 + 1024 * u);
      if (mine(d[u].x) | mine(d[u].y) | mine(d[u].z) | mine(d[u].w)) {
        take(i, d[u].x);
        take(i + 1, d[u].y);
        take(i + 2, d[u].z);
        take(i + 3, d[u].w);
      }
    }
  }
  for (int64_t s = 4 * n4 + threadIdx.x; s < S; s += 1024) take(s, tp2id[s]);
  __syncthreads();
  write_ranked(s_list, nt, t0, k, lists);
}

// Long tables (every workgroup's reading of the whole would grow with their square): counts cleared, each slot put behind its token's
// others by a global counter, the lists ranked by way of LDS.  Which slots of a token with more than k are kept is left open.
__global__ __launch_bounds__(256) void clear_counts_kernel(int64_t T, int w, int32_t* __restrict__ lists) {
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < T; t += (int64_t)gridDim.x * 256) lists[t * w] = 0;
}
__global__ __launch_bounds__(256) void place_slots_kernel(const int32_t* __restrict__ tp2id, int64_t S, int64_t T, int k,
                                                          int32_t* __restrict__ lists) {
  constexpr int U = 4;
  const int64_t threads = (int64_t)gridDim.x * 256;
  for (int64_t s0 = (int64_t)blockIdx.x * 256 + threadIdx.x; s0 < S; s0 += threads * U) {
    int id[U], p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = s0 + u * threads < S ? tp2id[s0 + u * threads] : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) p[u] = id[u] >= 0 && id[u] < T ? atomicAdd(&lists[(int64_t)id[u] * (1 + k)], 1) : k;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p[u] < k) lists[(int64_t)id[u] * (1 + k) + 1 + p[u]] = (int)(s0 + u * threads);
  }
}
__global__ __launch_bounds__(1024) void rank_slots_kernel(int64_t T, int k, int range, int32_t* __restrict__ lists) {
  __shared__ int s_list[SLOTS_LDS_WORDS];
  for (int64_t t0 = (int64_t)blockIdx.x * range; t0 < T; t0 += (int64_t)gridDim.x * range) {
    const int nt = (int)(T - t0 < range ? T - t0 : range);
    __syncthreads();  // (the lists of the round before have been read)
    for (int i = threadIdx.x; i < nt * (1 + k); i += 1024) s_list[i] = lists[t0 * (1 + k) + i];
    __syncthreads();
    write_ranked(s_list, nt, t0, k, lists);
  }
}

// ---- permute ----------------------------------------------------------------------------------------------------

typedef uint32_t bytes16 __attribute__((ext_vector_type(4), aligned(1)));

constexpr int64_t SHORT_ROW = 4096;           // bytes of a row that is a wave's work
constexpr int64_t SHORT_WEIGHTED_ROW = 5120;  // with weights, in the combine
// TPR threads per row or part of a row (a whole number of waves, so that everything about a row is uniform).
template <int TPR>
__device__ __forceinline__ int64_t row_of_group() {
  return (int64_t)blockIdx.x * (256 / TPR) + __builtin_amdgcn_readfirstlane((int)(threadIdx.x / TPR));
}
// Up to four pieces of 16 bytes per thread are asked for before the first is written, and written past the caches: the x rows come
// as often as they have slots, from the Infinity Cache if the output leaves them there.  T = 8192 tokens of 14 KB in 8 of 98048
// slots, x in no cache, us: 306; a piece at a time 319, with ordinary stores 359, a workgroup per 512 pieces 361; token by token,
// each row read once and written to 8 places, 301 with the list of the slots that this takes.  The writes alone, in order: 205.
// A wave or a workgroup per row, us: 8192 tokens of 1 KB 29 and 49, 3 KB 67 and 82, 5.6 KB 129 and 127, 8 KB 180 and 172; 1024 of
// 3 KB 18 and 24, 5.6 KB 32 and 32.
template <int TPR>
__global__ __launch_bounds__(256) void permute_kernel(const uint8_t* __restrict__ x, const int32_t* __restrict__ tp2id, int64_t S,
                                                      int64_t T, int64_t row_bytes, uint8_t* __restrict__ out) {
  constexpr int U = 4;
  const int lane = threadIdx.x % TPR;
  const int64_t whole = row_bytes / 16;
  for (int64_t s = row_of_group<TPR>(); s < S; s += (int64_t)gridDim.x * (256 / TPR)) {
    const int64_t id = tp2id[s];
    const bool token = id >= 0 && id < T;
    const uint8_t* src = x + (token ? id : 0) * row_bytes;
    uint8_t* dst = out + s * row_bytes;
    for (int64_t c0 = lane; c0 < whole; c0 += TPR * U) {
      bytes16 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u] = bytes16{0, 0, 0, 0};
        if (token && c0 + TPR * u < whole) v[u] = *(const bytes16*)(src + 16 * (c0 + TPR * u));
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + TPR * u < whole) __builtin_nontemporal_store(v[u], (bytes16*)(dst + 16 * (c0 + TPR * u)));
    }
    for (int64_t b = 16 * whole + lane; b < row_bytes; b += TPR) dst[b] = token ? src[b] : (uint8_t)0;
  }
}

// ---- combine, and the backward pass of permute --------------------------------------------------------------------

struct SlotTables {
  const int32_t* lists;  // [T][1 + k]
  const int32_t* b2e;    // null: every weight is one
  const void* aff;       // [>= T][E]
  int aff_dtype, k;
  uint32_t B, N;
  int64_t E, S;          // S: rows of y
};
// Eight neighbours of a token's list: rows (-1: none; one outside of y, of a list made of another table, is none either), weights.
// A slot of a block without an expert counts for nothing: `on` is false, its weight 0.  Its row is asked for all the same: the
// rows of y do not wait for the chain of expert and affinity.
struct SlotGroup {
  int64_t row[8];
  float w[8];
  int e[8];
  bool on[8];
};
template <class SLOT>
__device__ __forceinline__ void load_rows(const SlotTables& a, SLOT&& slot, int j0, int n, SlotGroup& g) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    g.row[j] = j0 + j < n ? slot(j0 + j) : -1;
    if (g.row[j] >= a.S) g.row[j] = -1;
  }
}
__device__ __forceinline__ void load_weights(const SlotTables& a, int64_t t, SlotGroup& g) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    g.w[j] = 1.f;
    g.e[j] = 0;
    g.on[j] = g.row[j] >= 0;
    if (a.b2e && g.on[j]) {
      const uint32_t b = (uint32_t)g.row[j] / a.B;
      g.e[j] = b < a.N ? a.b2e[b] : -1;
    }
  }
  if (!a.b2e) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (g.on[j]) {
      g.on[j] = g.e[j] >= 0 && g.e[j] < a.E;
      g.w[j] = g.on[j] ? load_as_f32(a.aff, a.aff_dtype, t * a.E + g.e[j]) : 0.f;
    }
}

// TPR threads per token; where the tokens are few, gridDim.y groups of them side by side along the row.  SCAN: every group looks
// its token up in the table itself, of at most COMBINE_SCAN_SLOTS slots, for tokens of a single round of the launch: a launch
// less, which at such sizes takes as long as the sums (8 tokens, 64 slots of 14 KB: kernels 6.1 + 3.0 us by the list, 6.8 so; a
// call 17.6 and 13.0).
constexpr int64_t COMBINE_SCAN_SLOTS = 2048;
template <int DT, int TPR, bool SCAN>
__global__ __launch_bounds__(256) void combine_tokens_kernel(const uint8_t* __restrict__ y, const SlotTables a,
                                                             const int32_t* __restrict__ tp2id, int64_t T, int64_t H,
                                                             uint8_t* __restrict__ out) {
  typedef Elem<DT> EL;
  typedef typename EL::raw raw;
  constexpr int N = EL::N;
  static_assert(TPR == 256 || !SCAN, "the scan is the workgroup's");
  __shared__ int found[SCAN ? 1 + SLOTS_MAX_K : 1], sorted[SCAN ? SLOTS_MAX_K : 1];
  const int lane = blockIdx.y * TPR + threadIdx.x % TPR, step = gridDim.y * TPR;
  if constexpr (SCAN) {
    const int i0 = threadIdx.x, S = (int)a.S;
    const int t = (int)row_of_group<TPR>();
    if (i0 == 0) found[0] = 0;
    __syncthreads();
    for (int s0 = i0; s0 < S; s0 += 8 * TPR) {
      int id[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) id[u] = s0 + TPR * u < S ? tp2id[s0 + TPR * u] : -1;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (id[u] == t) {
          const int p = atomicAdd(&found[0], 1);
          if (p < a.k) found[1 + p] = s0 + TPR * u;
        }
    }
    __syncthreads();
    const int held = found[0] < a.k ? found[0] : a.k;
    for (int i = i0; i < held; i += TPR) {
      int rank = 0;
      for (int o = 0; o < held; ++o) rank += found[1 + o] < found[1 + i];
      sorted[rank] = found[1 + i];
    }
    __syncthreads();
  }
  for (int64_t t = row_of_group<TPR>(); t < T; t += (int64_t)gridDim.x * (256 / TPR)) {
    const int32_t* list = SCAN ? nullptr : a.lists + t * (1 + a.k);
    auto slot = [&](int j) {
      if constexpr (SCAN) return __builtin_amdgcn_readfirstlane(sorted[j]);
      else return list[1 + j];
    };
    const int count = SCAN ? __builtin_amdgcn_readfirstlane(found[0]) : list[0];
    const bool cut = count > a.k;  // the table lists the token more often than its caller said: no sum of a part
    const int n = cut ? 0 : count;
    const float start = cut ? __builtin_nanf("") : 0.f;
    SlotGroup g;
    load_rows(a, slot, 0, n, g);
    bool weighted = false;  // (the first eight's weights, once; more than eight slots: each time)
    // (the last piece of a row that is no whole number of them begins early and writes what its neighbour writes)
    for (int64_t c0 = (int64_t)lane * N; c0 < H && H >= N; c0 += (int64_t)step * N) {
      const int64_t c = c0 < H - N ? c0 : H - N;
      float acc[N];
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = start;
      for (int j0 = 0; j0 < n; j0 += 8) {
        if (n > 8) load_rows(a, slot, j0, n, g);
        u32x4 d[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g.row[j] >= 0) d[j] = load_piece<DT>(y + (g.row[j] * H + c) * EL::SIZE);
        if (n > 8 || !weighted) load_weights(a, t, g);
        weighted = true;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g.on[j]) {
            float v[N];
            unpack<DT>(d[j], v);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] = fmaf(g.w[j], v[i], acc[i]);
          }
      }
      store_piece<DT>(out + (t * H + c) * EL::SIZE, pack<DT>(acc));
    }
    for (int64_t c = lane; c < H && H < N; c += step) {
      float acc = start;
      for (int j0 = 0; j0 < n; j0 += 8) {
        load_rows(a, slot, j0, n, g);
        load_weights(a, t, g);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g.on[j]) acc = fmaf(g.w[j], elem_to_f32<DT>(((const raw*)y)[g.row[j] * H + c]), acc);
      }
      ((raw*)out)[t * H + c] = f32_to_elem<DT>(acc);
    }
  }
}

// ---- combine, backward --------------------------------------------------------------------------------------------

// Jobs [0, T) take a token each: its row of dout is read once per eight slots, eight rows of y and dy beside it.  The next
// ceil(S / PAD_SLOTS) write the rows of slots that no token's list holds (few slots each: padding comes in runs, at an expert's
// end; with 64 the kernel took 480 us instead of 465 at T = 8192, 98048 slots of 14 KB), the last one the rows of da behind T.
// A job has TPR threads: a workgroup, or a wave where rows are short, which shares nothing with the others of its workgroup.
// The kernel with workgroups and with waves, us: 3855 tokens in 3 slots of 130 bytes 48 and 16, 8192 in 8 of 1.5 KB 160 and 60,
// 3 KB 175 and 100, 5.6 KB 222 and 180, 8 KB 262 and 263, 14 KB 467 and 482.  (Calls for 1024 tokens: 3 KB 43 and 35, 5.6 KB 54
// and 54; for 128: 20 and 21, 23 and 27.)
constexpr int PAD_SLOTS = 8;
template <int DT, int TPR>
__global__ __launch_bounds__(256) void combine_tokens_bwd_kernel(const uint8_t* __restrict__ dout, const uint8_t* __restrict__ y,
                                                                 const SlotTables a, const int32_t* __restrict__ tp2id,
                                                                 int64_t S, int64_t T, int64_t T1, int64_t H,
                                                                 uint8_t* __restrict__ dy, float* __restrict__ daff) {
  typedef Elem<DT> EL;
  typedef typename EL::raw raw;
  constexpr int N = EL::N;
  constexpr bool WAVE_JOB = TPR == 64;
  static_assert(TPR == 64 || TPR == 256, "a wave or the workgroup");
  __shared__ float s_part[4][8], s_dot[SLOTS_MAX_K];
  __shared__ int s_e[SLOTS_MAX_K];
  const int tid = threadIdx.x % TPR;
  const int64_t whole = H / N * N, n_pad = (S + PAD_SLOTS - 1) / PAD_SLOTS;
  for (int64_t job = row_of_group<TPR>(); job < T + n_pad + 1; job += (int64_t)gridDim.x * (256 / TPR)) {
    if (job == T + n_pad) {
      for (int64_t i = T * a.E + tid; i < T1 * a.E; i += TPR) daff[i] = 0.f;
      continue;
    }
    if (job >= T) {
      const int64_t s0 = (job - T) * PAD_SLOTS, mine = s0 + (tid & 63);
      const bool in = mine < S && mine < s0 + PAD_SLOTS;
      const int64_t id = in ? tp2id[mine] : 0;
      const int e = in ? a.b2e[(uint32_t)mine / a.B] : 0;
      const bool token = id >= 0 && id < T && e >= 0 && e < a.E;
      const bool cut = in && token && a.lists[id * (1 + a.k)] > a.k;
      const uint64_t nans = __ballot(cut);
      for (uint64_t left = __ballot(in && (!token || cut)); left; left &= left - 1) {
        const int i = __builtin_ctzll(left);
        const int64_t s = s0 + i;
        float v[N];
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = (nans >> i) & 1 ? __builtin_nanf("") : 0.f;
        for (int64_t c = (int64_t)tid * N; c < whole; c += TPR * N) store_piece<DT>(dy + (s * H + c) * EL::SIZE, pack<DT>(v));
        for (int64_t c = whole + tid; c < H; c += TPR) ((raw*)dy)[s * H + c] = f32_to_elem<DT>(v[0]);
      }
      continue;
    }
    const int64_t t = job;
    const int32_t* list = a.lists + t * (1 + a.k);
    const int n = list[0];
    float* drow = daff + t * a.E;
    if (n > a.k) {
      for (int64_t e = tid; e < a.E; e += TPR) drow[e] = __builtin_nanf("");
      continue;
    }
    if (WAVE_JOB && n <= 0)
      for (int64_t e = tid; e < a.E; e += TPR) drow[e] = 0.f;
    for (int j0 = 0; j0 < n; j0 += 8) {
      SlotGroup g;
      load_rows(a, [&](int j) { return list[1 + j]; }, j0, n, g);
      load_weights(a, t, g);
      float dot[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) dot[j] = 0.f;
      for (int64_t c = (int64_t)tid * N; c < whole; c += TPR * N) {
        u32x4 d[8];
        const u32x4 dg = load_piece_kept<DT>(dout + (t * H + c) * EL::SIZE);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g.on[j]) d[j] = load_piece<DT>(y + (g.row[j] * H + c) * EL::SIZE);
        float gv[N];
        unpack<DT>(dg, gv);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g.on[j]) {
            float v[N];
            unpack<DT>(d[j], v);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              dot[j] = fmaf(gv[i], v[i], dot[j]);
              v[i] = g.w[j] * gv[i];
            }
            store_piece<DT>(dy + (g.row[j] * H + c) * EL::SIZE, pack<DT>(v));
          }
      }
      for (int64_t c = whole + tid; c < H; c += TPR) {
        const float gv = elem_to_f32<DT>(((const raw*)dout)[t * H + c]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g.on[j]) {
            dot[j] = fmaf(gv, elem_to_f32<DT>(((const raw*)y)[g.row[j] * H + c]), dot[j]);
            ((raw*)dy)[g.row[j] * H + c] = f32_to_elem<DT>(g.w[j] * gv);
          }
      }
      if constexpr (WAVE_JOB) {
        // every lane has the sums: each adds up the entries of da that are its own, group by group
#pragma unroll
        for (int j = 0; j < 8; ++j) dot[j] = wave_sum(dot[j]);
        for (int64_t e = tid; e < a.E; e += TPR) {
          float v = j0 ? drow[e] : 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (g.on[j] && g.e[j] == e) v += dot[j];
          drow[e] = v;
        }
      } else {
        __syncthreads();  // (the sums of the group before, and of the token before, have been read)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = wave_sum(dot[j]);
          if ((tid & 63) == 0) s_part[tid >> 6][j] = v;
          if (tid == 0 && j0 + j < n) s_e[j0 + j] = g.on[j] ? g.e[j] : -1;
        }
        __syncthreads();
        if (tid < 8 && j0 + tid < n) s_dot[j0 + tid] = (s_part[0][tid] + s_part[1][tid]) + (s_part[2][tid] + s_part[3][tid]);
      }
    }
    if constexpr (!WAVE_JOB) {
      __syncthreads();
      for (int64_t e = tid; e < a.E; e += TPR) {
        float v = 0.f;
        for (int j = 0; j < n; ++j)
          if (s_e[j] == e) v += s_dot[j];
        drow[e] = v;
      }
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

// (a launch holds fewer than 2^32 threads; what lies beyond a million workgroups is a second round of the same ones)
static unsigned grid_of(int64_t jobs) { return (unsigned)(jobs < ((int64_t)1 << 20) ? jobs : (int64_t)1 << 20); }

}  // namespace moe

using namespace moe;

static int launch_token_slots(const int32_t* tp2id, int64_t S, int64_t T, int k, int32_t* lists, hipStream_t s) {
  if (T == 0) return MOE_OK;
  int64_t range = (T + 255) / 256;  // a workgroup per CU
  if (range > SLOTS_LDS_WORDS / (1 + k)) range = SLOTS_LDS_WORDS / (1 + k);
  const int64_t groups = (T + range - 1) / range;
  if (groups * S <= LISTS_WHOLE_TABLE) {
    hipLaunchKernelGGL(token_slots_kernel, dim3((unsigned)groups), dim3(1024), 0, s, tp2id, S, T, k, (int)range, lists);
    MOE_CHECK_LAUNCH();
    return MOE_OK;
  }
  hipLaunchKernelGGL(clear_counts_kernel, dim3(grid_of((T + 255) / 256)), dim3(256), 0, s, T, 1 + k, lists);
  MOE_CHECK_LAUNCH();
  hipLaunchKernelGGL(place_slots_kernel, dim3(grid_of((S + 1023) / 1024)), dim3(256), 0, s, tp2id, S, T, k, lists);
  MOE_CHECK_LAUNCH();
  hipLaunchKernelGGL(rank_slots_kernel, dim3(grid_of(groups)), dim3(1024), 0, s, T, k, (int)range, lists);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

extern "C" int moe_token_slots(const int32_t* token_position_to_id, int64_t S, int64_t T, int top_k, int32_t* token_slots,
                               void* stream) {
  if ((!token_position_to_id && S > 0) || !token_slots || S < 0 || T < 0) return MOE_E_BAD_ARG;
  if (top_k < 1 || top_k > SLOTS_MAX_K || S >= (int64_t)1 << 31 || T >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  return launch_token_slots(token_position_to_id, S, T, top_k, token_slots, (hipStream_t)stream);
}

extern "C" int moe_permute_tokens(const void* x, const int32_t* token_position_to_id, int64_t S, int64_t T, int64_t row_bytes,
                                  void* out, void* stream) {
  if (!x || !token_position_to_id || !out || S < 0 || T < 0 || row_bytes < 0) return MOE_E_BAD_ARG;
  if (S >= (int64_t)1 << 31 || T >= (int64_t)1 << 31 || row_bytes >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  if (S == 0 || row_bytes == 0) return MOE_OK;
  const hipStream_t s = (hipStream_t)stream;
  if (row_bytes > SHORT_ROW)
    hipLaunchKernelGGL(permute_kernel<256>, dim3(grid_of(S)), dim3(256), 0, s, (const uint8_t*)x, token_position_to_id, S, T,
                       row_bytes, (uint8_t*)out);
  else
    hipLaunchKernelGGL(permute_kernel<64>, dim3(grid_of((S + 3) / 4)), dim3(256), 0, s, (const uint8_t*)x,
                       token_position_to_id, S, T, row_bytes, (uint8_t*)out);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

// tp2id: for the scan, else null
template <int DT>
static void launch_combine_tokens(const void* y, const SlotTables& a, const int32_t* tp2id, int64_t T, int64_t H, void* out,
                                  hipStream_t s) {
  // a workgroup per token, or a wave where rows are short and tokens many: weighted, each of a workgroup's four waves works out the
  // weights, so that a wave alone pays up to longer rows (us a call with lists made before, bf16, wave | workgroup: 8192 tokens in 8
  // slots of 2.0 KB 29.9 | 36.4, 3.9 KB 56.2 | 63.0, 4.0 KB 60.8 | 63.7, 4.5 KB 66.6 | 69.9, 5.5 KB 81.0 | 78.7, in 2 of 4.5 KB 26.2 |
  // 32.0, 5.5 KB 31.0 | 34.7; unweighted in 8 of 1.0 KB 15.2 | 15.9, 2.0 KB 28.3 | 27.7, 3.9 KB 54.8 | 50.6, 4.0 KB 58.3 | 53.1, in 2 of
  // 2.0 KB 12.0 | 16.8, 3.9 KB 20.9 | 22.3, 4.0 KB 22.5 | 22.3, 5.5 KB 29.6 | 28.8; 20000 tokens alike); few tokens (decode): several
  // workgroups per token, a piece per thread
  const bool wide = H * Elem<DT>::SIZE >= (a.b2e ? SHORT_WEIGHTED_ROW : SHORT_ROW) || T < 2048;
  const int64_t groups = wide ? T : (T + 3) / 4;
  int64_t parts = 1;
  if (wide && groups < 512) {
    parts = (H + 256 * Elem<DT>::N - 1) / (256 * Elem<DT>::N);
    if (parts > 512 / groups) parts = 512 / groups;
  }
  const dim3 grid(grid_of(groups), (unsigned)parts);
#define MOE_COMBINE(TPR, SCAN)                                                                                                  \
  hipLaunchKernelGGL((combine_tokens_kernel<DT, TPR, SCAN>), grid, dim3(256), 0, s, (const uint8_t*)y, a, tp2id, T, H, (uint8_t*)out)
  if (wide && tp2id) MOE_COMBINE(256, true);
  else if (wide) MOE_COMBINE(256, false);
  else MOE_COMBINE(64, false);
#undef MOE_COMBINE
}
// (every group of threads reads the table: for few tokens and slots that costs less than the launch it saves)
static bool combine_scans(int64_t S, int64_t T) { return S <= COMBINE_SCAN_SLOTS && T <= 512; }

// What the calls that go by lists check alike, and the list itself where it is asked for.
static int begin_by_list(const SlotTables& a, int64_t T, int64_t T1, const int32_t* tp2id, int build, bool launch, hipStream_t s) {
  if (!a.lists || a.S < 0 || T < 0 || (build && !tp2id && a.S > 0)) return MOE_E_BAD_ARG;
  if (a.k < 1 || a.k > SLOTS_MAX_K || T >= (int64_t)1 << 31 || a.S >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  if (a.b2e) {
    if (!a.aff || (a.aff_dtype != MOE_DT_BF16 && a.aff_dtype != MOE_DT_FP32)) return MOE_E_BAD_ARG;
    if (a.E <= 0 || a.E >= (int64_t)1 << 31 || T1 < T) return MOE_E_BAD_SHAPE;
  }
  return build && launch ? launch_token_slots(tp2id, a.S, T, a.k, (int32_t*)a.lists, s) : MOE_OK;
}

extern "C" int moe_combine_tokens(const void* y, int dtype, const void* expert_affinities, int aff_dtype, int64_t T1, int64_t E,
                                  const int32_t* token_position_to_id, const int32_t* block_to_expert, int64_t B, int64_t N,
                                  int32_t* token_slots, int top_k, int build_token_slots, int64_t S, int64_t T, int64_t H, void* out,
                                  void* stream) {
  if (!y || !out || H < 0 || dtype < MOE_DT_BF16 || dtype > MOE_DT_FP32) return MOE_E_BAD_ARG;
  if ((expert_affinities != nullptr) != (block_to_expert != nullptr)) return MOE_E_BAD_ARG;
  if (block_to_expert && (B <= 0 || N < 0 || B >= (int64_t)1 << 31 || N >= (int64_t)1 << 31 || S != B * N)) return MOE_E_BAD_SHAPE;
  const SlotTables a{token_slots, block_to_expert, expert_affinities, aff_dtype, top_k, (uint32_t)B, (uint32_t)N, E, S};
  const hipStream_t s = (hipStream_t)stream;
  const bool scan = build_token_slots && token_position_to_id && combine_scans(S, T);  // (no table, no slots: the list of none)
  const int rc = begin_by_list(a, T, T1, token_position_to_id, build_token_slots, !scan, s);
  if (rc != MOE_OK) return rc;
  if (T == 0 || H == 0) return MOE_OK;
  const int32_t* table = scan ? token_position_to_id : nullptr;
  switch (dtype) {
    case MOE_DT_BF16: launch_combine_tokens<MOE_DT_BF16>(y, a, table, T, H, out, s); break;
    case MOE_DT_FP16: launch_combine_tokens<MOE_DT_FP16>(y, a, table, T, H, out, s); break;
    default: launch_combine_tokens<MOE_DT_FP32>(y, a, table, T, H, out, s); break;
  }
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

extern "C" int moe_combine_tokens_bwd(const void* d_out, const void* y, int dtype, const void* expert_affinities, int aff_dtype,
                                      int64_t T1, int64_t E, const int32_t* token_position_to_id, const int32_t* block_to_expert,
                                      int64_t B, int64_t N, int32_t* token_slots, int top_k, int build_token_slots, int64_t T,
                                      int64_t H, void* d_y, float* d_affinities, void* stream) {
  if (!d_out || !y || !expert_affinities || !token_position_to_id || !block_to_expert || !d_y || !d_affinities || H < 0 || N < 0 ||
      dtype < MOE_DT_BF16 || dtype > MOE_DT_FP32)
    return MOE_E_BAD_ARG;
  if (B <= 0 || B >= (int64_t)1 << 31 || N >= (int64_t)1 << 31) return MOE_E_BAD_SHAPE;
  const int64_t S = B * N;
  const SlotTables a{token_slots, block_to_expert, expert_affinities, aff_dtype, top_k, (uint32_t)B, (uint32_t)N, E, S};
  const hipStream_t s = (hipStream_t)stream;
  const int rc = begin_by_list(a, T, T1, token_position_to_id, build_token_slots, true, s);
  if (rc != MOE_OK) return rc;
  const int64_t jobs = T + (S + PAD_SLOTS - 1) / PAD_SLOTS + 1;
  const int64_t row_bytes = H * (dtype == MOE_DT_FP32 ? 4 : 2);
#define MOE_BWD(DT)                                                                                                             \
  do {                                                                                                                          \
    if (row_bytes > SHORT_ROW)                                                                                                  \
      hipLaunchKernelGGL((combine_tokens_bwd_kernel<DT, 256>), dim3(grid_of(jobs)), dim3(256), 0, s, (const uint8_t*)d_out,     \
                         (const uint8_t*)y, a, token_position_to_id, S, T, T1, H, (uint8_t*)d_y, d_affinities);                 \
    else                                                                                                                        \
      hipLaunchKernelGGL((combine_tokens_bwd_kernel<DT, 64>), dim3(grid_of((jobs + 3) / 4)), dim3(256), 0, s,                   \
                         (const uint8_t*)d_out, (const uint8_t*)y, a, token_position_to_id, S, T, T1, H, (uint8_t*)d_y,         \
                         d_affinities);                                                                                         \
  } while (0)
  switch (dtype) {
    case MOE_DT_BF16: MOE_BWD(MOE_DT_BF16); break;
    case MOE_DT_FP16: MOE_BWD(MOE_DT_FP16); break;
    default: MOE_BWD(MOE_DT_FP32); break;
  }
#undef MOE_BWD
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

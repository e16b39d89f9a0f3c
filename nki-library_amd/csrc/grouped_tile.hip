// Tiles of products of ragged groups of rows, for one element type per translation unit (GG_TYPE: GG_BF16, GG_FP16, GG_INT8).
//
// A workgroup walks over tiles of BM x BN of the result.  A step takes 128 bytes along the terms from both operands: 64 terms of 16
// bits or 128 of 8, two MFMAs deep.  Either operand lies in memory along its terms ("rows": a piece of 16 bytes is a lane's
// operand as it is) or across them ("columns": a piece is 8 neighbouring columns of one term), and stays so in LDS, where the
// transposing read (ds_read_b64_tr_b16) hands a lane the terms of its column.  So weights [E, K, N] are multiplied as they are, and
// their gradient, whose terms are rows, takes both operands across.
//   rows:    LDS row of 128 bytes per row; piece j of row r in place j ^ (r & 7)
//   columns: LDS row of BN columns per term; piece j of term k in place j ^ f(k), f(k) = 2 (k & 3) + 8 ((k >> 3) & 1): the 16 lanes of
//            a transposing read fetch 32 bytes from each of 4 terms, two such groups at a time terms 8 apart, all in other banks.
// DMA: operands go global -> LDS without a register (rows that begin at 4 bytes; at 16 they come faster, 8192 rows of 4160 x 4160 bf16 348
// | 408 us); otherwise through registers, where a piece that passes a row's end is the row's last one moved down (641 us).  Two stages; a
// step's second half of fragments is read under the MFMAs of its first, the next step's first half under those of its second; the one
// barrier of a step stands between them: all have read the step's stage, which then takes the step after the next, and the next step's
// has landed.  The loads go out one per row tile of the second half: all at once they hold up the waves' issue (8192^3 bf16 895 | 857 us).
// What bounds it: 70 % of the cycles the matrix pipes work (2950 cycles for a step of 256 x 256, MFMAs alone 2048), the rest is the barrier
// and what stands around it, and a tile's edges (see STORES); after some milliseconds power leaves a clock of 1.5 GHz.  8192^3, us:
// bf16 weights across 806 (1.36 PFLOP/s), along 793, their gradient 808, int8 500 (2.2 POP/s).
// The matrix is the MFMA's first operand, so that a lane holds four neighbouring columns of one row; rows go out through LDS in whole
// 128-byte lines.
#include <type_traits>

#include "grouped_gemm.hpp"

namespace moe {
namespace {

constexpr int TYPE = GG_TYPE;
constexpr int ES = TYPE == GG_INT8 ? 1 : 2;
constexpr int STEP = 128 / ES;  // terms of a step

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t bytes16 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t words4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_byte;
using acc_t = std::conditional_t<TYPE == GG_INT8, v4i, v4f>;

__device__ __forceinline__ acc_t mfma(const v4i& w, const v4i& x, const acc_t& c) {
  if constexpr (TYPE == GG_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, x), c, 0, 0, 0);
  else if constexpr (TYPE == GG_FP16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, x), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
}

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Raw buffer over `bytes` (any number; offsets of a step stay below 2^31) from p on: what lies outside reads as zeros.
__device__ __forceinline__ v4i buffer_of(const uint8_t* p, int64_t bytes) {
  const uint64_t addr = (uint64_t)p;
  const int64_t least = bytes > 0 ? bytes : 0;
  const uint32_t n = least > 0x7ffffff0 ? 0x7ffffff0u : (uint32_t)least;
  v4i d;
  d[0] = uni((int)(uint32_t)addr);
  d[1] = uni((int)(uint32_t)(addr >> 32)) & 0xffff;
  d[2] = uni((int)n);
  d[3] = 0x00020000;
  return d;
}
constexpr uint32_t NOWHERE = 0x80000000u;  // an offset outside of every buffer, as are those of the rows behind it (all below 2^31 apart)
// 16 bytes per lane to lds + 16 * lane.  (The wait states: a scalar operand may have been written by a vector instruction just before,
// which the compiler does not see here.  It keeps nothing in M0 between instructions of its own.)
__device__ __forceinline__ void load_to_lds(uint32_t lds, uint32_t off, const v4i& buf) {
  asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               : : "s"(lds), "v"(off), "s"(buf) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ int spread(int k) { return 2 * (k & 3) + 8 * ((k >> 3) & 1); }

struct Tile {
  const uint8_t* a;
  const uint8_t* b;
  int64_t a_bytes, b_bytes;  // from there to the end of what may be read
  uint8_t* out;
  int steps, rows, cols;  // rows and columns of the result that the tile holds
  int64_t row0;           // GG_ROWS: first row
  int64_t n0;
  int expert;
};

// One operand's way into LDS.  ROWS_: lies along its terms.  BR: rows (columns) of a tile.
template <bool ROWS_, int BR, int THREADS, bool DMA>
struct Feed {
  static constexpr int BYTES = BR * 128;
  static constexpr int PITCH = ROWS_ ? 128 : BR * ES;  // of an LDS row
  static constexpr int PPR = PITCH / 16;               // pieces of one
  static constexpr int N = BYTES / 16 / THREADS;       // pieces of a thread
  static constexpr int RPT = THREADS / PPR;            // rows between two pieces of a thread
  static_assert(THREADS % PPR == 0 && RPT % 16 == 0, "a thread's pieces lie alike in all of its rows");
  uint32_t off;  // of the thread's first piece; piece i lies i * RPT rows behind it
  words4 held[DMA ? 1 : N];

  static __device__ __forceinline__ int row() { return threadIdx.x / PPR; }
  static __device__ __forceinline__ int place() { return threadIdx.x % PPR; }
  static __device__ __forceinline__ int swizzled() { return place() ^ (ROWS_ ? row() & 7 : spread(row())); }
  __device__ __forceinline__ void begin(int pitch) { off = (uint32_t)(row() * pitch + (DMA ? swizzled() : place()) * 16); }
  // DMA: what the loads of a step need, and the loads one by one, into the stage at lds.  left: bytes of a row's terms from this step
  // on (ROWS_).
  struct Step {
    v4i buf;
    uint32_t o, leap, lds;
  };
  __device__ __forceinline__ Step step_of(uint32_t lds, const uint8_t* p, int64_t bytes, int pitch, int step, int left) const {
    const int64_t skip = ROWS_ ? (int64_t)step * 128 : (int64_t)step * STEP * pitch;
    Step q;
    q.buf = buffer_of(p + skip, bytes - skip);
    q.o = ROWS_ && swizzled() * 16 >= left ? NOWHERE : off;
    q.leap = (uint32_t)(RPT * pitch);
    q.lds = uni(lds + (threadIdx.x & ~63) * 16);
    return q;
  }
  static __device__ __forceinline__ void load(const Step& q, int i) { load_to_lds(q.lds + i * THREADS * 16, q.o + i * q.leap, q.buf); }
  // Through registers: rows r < rows_left are read, terms_left bytes (ROWS_) or terms from this step on, cols_left bytes of a row.  Where
  // rows, terms or columns end inside the tile (all steps of a group's last row tile) the pieces are waited for one or two at a time.
  __device__ __forceinline__ void fetch(const uint8_t* p, int pitch, int step, int rows_left, int terms_left, int cols_left) {
    const int c = place() * 16;
    if (ROWS_ ? rows_left >= BR && terms_left >= 128 : terms_left >= STEP && cols_left >= BR * ES) {  // (nothing ends inside)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint8_t* src = p + (ROWS_ ? (int64_t)step * 128 : (int64_t)step * STEP * pitch) + (int64_t)i * RPT * pitch;
        const bytes16 d = *(const bytes16*)(src + (int)off);
        held[i] = words4{d[0], d[1], d[2], d[3]};
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = row() + i * RPT;
      const uint8_t* src = p + (ROWS_ ? (int64_t)step * 128 : (int64_t)step * STEP * pitch) + (int64_t)i * RPT * pitch;
      const int left = ROWS_ ? (r < rows_left ? terms_left - c : 0) : (r < terms_left ? cols_left - c : 0);
      uint64_t lo = 0, hi = 0;
      if (left > 0) {
        // a piece that passes the row's end: the row's last 16 bytes, moved down (rows of fewer: element by element)
        const int gone = left >= 16 ? 0 : 16 - left;
        if (pitch >= 16) {
          const bytes16 d = *(const bytes16*)(src + ((int)off - gone));  // (may lie ahead of src: the step before)
          lo = (uint64_t)d[1] << 32 | d[0];
          hi = (uint64_t)d[3] << 32 | d[2];
          if (gone >= 8) {
            lo = hi >> (8 * (gone - 8));
            hi = 0;
          } else if (gone > 0) {
            lo = lo >> (8 * gone) | hi << (64 - 8 * gone);
            hi >>= 8 * gone;
          }
        } else {
#pragma unroll 1
          for (int b = 0; b < left; b += ES) {
            const uint64_t x = ES == 2 ? (uint64_t)*(const uint16_t*)(src + off + b) : (uint64_t)src[off + b];
            if (b < 8) lo |= x << (8 * b);
            else hi |= x << (8 * (b - 8));
          }
        }
      }
      // (One value of 128 bits from here on.  Kept as 32-bit parts that meet behind the branches, as a struct of four is, AMD clang 22 (ROCm 7.2)
      // takes two of a piece's four registers for free in the gradient of the weights while the piece waits to be put, and writes addresses
      // in its place.  Seen in an emulation of the compiled code, in which every load was waited for; with the compiler's instruction
      // scheduler off the same source came out right, so the fault is behind its intermediate code.  build.py looks for such a write.)
      words4 v = {(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      asm volatile("" : "+v"(v));
      held[i] = v;
    }
  }
  __device__ __forceinline__ void put(uint8_t* lds) {
#pragma unroll
    for (int i = 0; i < N; ++i) *(words4*)(lds + (row() + i * RPT) * PITCH + swizzled() * 16) = held[i];
  }
};
// ... and a wave's fragments out of it: tiles of 16 rows (columns), the first and every LEAP-th behind it.
template <bool ROWS_, int BR, int TILES, int LEAP>
struct Frags {
  static constexpr int PITCH = ROWS_ ? 128 : BR * ES;
  uint32_t at[ROWS_ ? 2 : TILES];
  __device__ __forceinline__ void begin(int first) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    if constexpr (ROWS_) {
      at[0] = (first * 16 + c) * 128 + ((g ^ (c & 7)) * 16);
      at[1] = at[0] ^ 64;
    } else {
      const int k = 8 * g + (c >> 2);
#pragma unroll
      for (int j = 0; j < TILES; ++j)
        at[j] = k * PITCH + (((2 * (first + j * LEAP) + ((c & 3) >> 1)) ^ spread(k)) * 16) + (c & 1) * 8;
    }
  }
  template <int HALF>
  __device__ __forceinline__ v4i read(const lds_byte* stage, int j) const {
    if constexpr (ROWS_) {
      return *(const __attribute__((address_space(3))) v4i*)(stage + at[HALF] + j * LEAP * 2048);
    } else {
      const lds_byte* p = stage + at[j] + HALF * 32 * PITCH;
      typedef __attribute__((address_space(3))) v4s* lds_v4s;
      union { v4s s[2]; v4i v; } u;
      u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)p);
      u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(p + 4 * PITCH));
      return u.v;
    }
  }
};

// WHOLE: rows of all operands are multiples of 16 bytes and begin at such.
template <int BM_, int BN_, int WM_, int WN_, bool DMA_, bool WHOLE_, int PER_CU_>
struct Cfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, THREADS = WM * WN * 64;
  static constexpr bool DMA = DMA_, WHOLE = WHOLE_;
  static constexpr int PER_CU = PER_CU_;  // workgroups of a CU
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  static constexpr int STAGE = (BM + BN) * 128;
  static constexpr int EXCHANGE = 2048;  // per wave
  static constexpr int LDS = 2 * STAGE + WM * WN * EXCHANGE;
  static_assert(NT % 4 == 0, "64 columns make lines of 128 bytes");
};

// The tiles t, t + workgroups and so on of a product; the first such number behind them is the result, counted from the last tile on.
// (The groups' table stands behind C::LDS.)
template <class C, int MODE, bool B_ROWS>
__device__ __forceinline__ int64_t tiles_of(const GroupedArgs& p, uint8_t* const smem, int64_t t) {
  constexpr bool A_ROWS = MODE == GG_ROWS;
  const int tid = threadIdx.x, wave = uni(tid >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  lds_byte* const lds = (lds_byte*)smem;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  uint8_t* const exchange = smem + 2 * C::STAGE + wave * C::EXCHANGE;
  int* const bound = (int*)(smem + C::LDS);
  int* const cum = bound + p.E + 3;
  // blocks of up to four row tiles of a group by all columns, row tiles fastest
  const int ntn = (int)((p.N + C::BN - 1) / C::BN), ntm = (int)((p.K + C::BM - 1) / C::BM);
  const int64_t total = MODE == GG_ROWS ? (int64_t)uni(cum[p.E + 2]) * ntn : (int64_t)p.E * ntm * ntn;

  auto find = [&](int64_t t) {
    Tile q;
    int64_t local;
    int rt, tiles;
    int j;
    if (MODE == GG_ROWS) {
      j = group_of_tile(cum, p.E, (int)(t / ntn));
      const int c0 = uni(cum[j]);
      tiles = uni(cum[j + 1]) - c0;
      local = t - (int64_t)c0 * ntn;
    } else {
      j = (int)(t / ((int64_t)ntm * ntn)) + 1;
      tiles = ntm;
      local = t - (int64_t)(j - 1) * ntm * ntn;
    }
    const int blk = (int)(local / (4 * ntn)), in = (int)(local - (int64_t)blk * 4 * ntn);
    const int h = tiles - blk * 4 < 4 ? tiles - blk * 4 : 4;
    const int ct = in / h;
    rt = blk * 4 + in - ct * h;
    const int begin = uni(bound[j]), rows = uni(bound[j + 1]) - begin;
    q.expert = j - 1;
    q.n0 = (int64_t)ct * C::BN;
    q.cols = (int)(p.N - q.n0 < C::BN ? p.N - q.n0 : C::BN);
    const int64_t m0 = (int64_t)rt * C::BM;
    if (MODE == GG_ROWS) {
      q.row0 = begin + m0;
      q.rows = (int)(rows - m0 < C::BM ? rows - m0 : C::BM);
      const bool zero = j == 0 || j == p.E + 1;
      q.steps = zero ? 0 : (int)((p.K * ES + 127) / 128);
      q.a = p.a + q.row0 * p.a_pitch;
      q.a_bytes = (p.S - q.row0) * p.a_pitch;
      const uint8_t* b = p.b + (zero ? 0 : q.expert) * p.b_group;
      q.b = b + (B_ROWS ? q.n0 * p.b_pitch : q.n0 * ES);
      q.b_bytes = (B_ROWS ? (p.N - q.n0) * p.b_pitch : p.K * p.b_pitch - q.n0 * ES);
      q.out = p.out + q.row0 * p.out_pitch;
    } else {
      q.row0 = m0;
      q.rows = (int)(p.K - m0 < C::BM ? p.K - m0 : C::BM);
      q.steps = (rows + STEP - 1) / STEP;
      q.a = p.a + begin * p.a_pitch + m0 * ES;
      q.a_bytes = rows * p.a_pitch - m0 * ES;
      q.b = p.b + begin * p.b_pitch + q.n0 * ES;
      q.b_bytes = rows * p.b_pitch - q.n0 * ES;
      q.out = p.out + ((int64_t)q.expert * p.K + m0) * p.out_pitch;
    }
    return q;
  };

  Feed<A_ROWS, C::BM, C::THREADS, C::DMA> fa;
  Feed<B_ROWS, C::BN, C::THREADS, C::DMA> fb;
  Frags<A_ROWS, C::BM, C::MT, C::WM> ra;
  Frags<B_ROWS, C::BN, C::NT, 1> rb;
  fa.begin((int)p.a_pitch);
  fb.begin((int)p.b_pitch);
  ra.begin(wm);
  rb.begin(wn * C::NT);
  constexpr int SA = C::BM * 128;

  const int pa = (int)p.a_pitch, pb = (int)p.b_pitch;
  // terms of a tile (DMA, GG_CONTRACT: the group's rows end the buffers)
  auto terms_of = [&](const Tile& q) { return MODE == GG_ROWS ? (int)p.K : uni(bound[q.expert + 2]) - uni(bound[q.expert + 1]); };
  // DMA: the loads of a step, A's and B's; beyond the last step they bring zeros
  typename decltype(fa)::Step sa;
  typename decltype(fb)::Step sb;
  auto prepare = [&](const Tile& q, int terms, int step) {
    const uint32_t st = lds0 + (step & 1) * C::STAGE;
    const bool in = step < q.steps;
    const int left = (terms - step * STEP) * ES;
    sa = fa.step_of(st, q.a, in ? q.a_bytes : 0, pa, step, left);
    sb = fb.step_of(st + SA, q.b, in ? q.b_bytes : 0, pb, step, left);
  };
  constexpr int LA = decltype(fa)::N, LB = decltype(fb)::N, LOADS = LA + LB;
  // (rows of A, RPT of them a load: those that a tile does not have are not loaded; what stands in their place has no part in its rows)
  auto load = [&](int i, int a_loads) {
    if (i < a_loads) fa.load(sa, i);
    else fb.load(sb, i - a_loads);
  };
  auto load_two = [&](const Tile& q) {
    if (q.steps == 0) return;
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      prepare(q, terms_of(q), step);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) load(i, LA);
    }
  };

  // otherwise: a step into registers (nothing from the last one on), and from there into its stage
  auto fetch = [&](const Tile& q, int terms, int step) {
    const int left = terms - step * STEP;
    fa.fetch(q.a, pa, step, q.rows, A_ROWS ? left * ES : left, q.rows * ES);
    fb.fetch(q.b, pb, step, q.cols, B_ROWS ? left * ES : left, q.cols * ES);
  };
  auto put = [&](int step) {
    uint8_t* st = smem + (step & 1) * C::STAGE;
    fa.put(st);
    fb.put(st + SA);
  };
  // DMA: a row's end inside a piece leaves the next row's first terms behind it in the last step's stage: zeros in their place
  const int last_bytes = MODE == GG_ROWS ? (int)((p.K * ES - 1) % 128 + 1) : 128;
  auto cut = [&](int step) {
    uint8_t* const st = smem + (step & 1) * C::STAGE;
    const int piece = last_bytes / 16;
    if constexpr (A_ROWS)
      for (int r = tid; r < C::BM; r += C::THREADS)
        for (int w = last_bytes & 15; w < 16; w += 4) *(uint32_t*)(st + r * 128 + ((piece ^ (r & 7)) * 16) + w) = 0;
    if constexpr (B_ROWS)
      for (int r = tid; r < C::BN; r += C::THREADS)
        for (int w = last_bytes & 15; w < 16; w += 4) *(uint32_t*)(st + SA + r * 128 + ((piece ^ (r & 7)) * 16) + w) = 0;
    barrier();
  };
  const bool cuts = C::DMA && !C::WHOLE && last_bytes % 16 != 0;
  auto begin = [&](const Tile& q) {
    if constexpr (C::DMA) load_two(q);
    else if (q.steps > 0) fetch(q, terms_of(q), 0);
  };

  // A tile's first two steps (without DMA: the first) are requested ahead of the results of the tile before, whose stores may then drain
  // under its first steps: at least STORES of them stand behind the loads in the order in which these are waited for (stored), or nothing
  // is counted on.  (In the tiles of 128 x 128 they do.  Those of 256 x 256 have 3 to 15 of their registers in scratch memory, offsets of the
  // loads mostly: a reload waits for all that is under way, and some stand between these requests, ahead of the results and between the
  // loads of the first step.  So there both steps have landed before the first result leaves, and the stores have drained by the
  // tile's first loads.)
  constexpr int STORES = 2 * C::MT;
  bool stored = false;
  if (t >= total) return t - total;
  Tile q = find(t);
  begin(q);
  for (;;) {
    const int terms = terms_of(q);
    acc_t acc[C::MT][C::NT];
#pragma unroll
    for (int m = 0; m < C::MT; ++m)
#pragma unroll
      for (int n = 0; n < C::NT; ++n) acc[m][n] = acc_t{0, 0, 0, 0};

    // The steps of a tile of which a wave has V row tiles.
    auto multiply = [&](auto row_tiles) {
      constexpr int V = decltype(row_tiles)::value;
      constexpr int A_LOADS = A_ROWS ? V * C::WM * 16 / decltype(fa)::RPT : LA;
      static_assert(!A_ROWS || V * C::WM * 16 % decltype(fa)::RPT == 0, "whole loads");
      if constexpr (C::DMA) {
        if (stored) wait_loads<LOADS + STORES>();
        else wait_loads<LOADS>();
      } else {
        put(0);
        fetch(q, terms, 1);
      }
      barrier();
      if (cuts && q.steps == 1) cut(0);
      // Half a step: its MFMAs, and under those of its first rows the fragments of the next half and what `more` does.  (The order is
      // pinned: left to itself the compiler moves every read to where its value is used and waits for it there.)
      auto half = [&](auto next_half, const lds_byte* st, v4i (&a)[V], v4i (&b)[C::NT], v4i (&an)[V], v4i (&bn)[C::NT], auto&& more) {
        constexpr int H = decltype(next_half)::value, R = V / 2;  // R: row tiles under which the fragments are read
#pragma unroll
        for (int m = 0; m < V; ++m) {
          if (m < R) {
#pragma unroll
            for (int n = m * C::NT / R; n < (m + 1) * C::NT / R; ++n) bn[n] = rb.template read<H>(st + SA, n);
            an[2 * m] = ra.template read<H>(st, 2 * m);
            an[2 * m + 1] = ra.template read<H>(st, 2 * m + 1);
          }
          more(m);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int n = 0; n < C::NT; ++n) acc[m][n] = mfma(b[n], a[m], acc[m][n]);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      v4i a0[V], b0[C::NT], a1[V], b1[C::NT];
#pragma unroll
      for (int n = 0; n < C::NT; ++n) b0[n] = rb.template read<0>(lds + SA, n);
#pragma unroll
      for (int m = 0; m < V; ++m) a0[m] = ra.template read<0>(lds, m);
      for (int ks = 0; ks < q.steps; ++ks) {
        if constexpr (C::DMA) prepare(q, terms, ks + 2);
        half(std::integral_constant<int, 1>{}, lds + (ks & 1) * C::STAGE, a0, b0, a1, b1, [](int) {});
        if constexpr (C::DMA) {
          if (ks == 0 && stored) wait_loads<STORES>();
          else wait_loads<0>();
        } else {
          put(ks + 1);  // (its stage was last read ahead of the barrier before)
        }
        barrier();
        if (cuts && ks + 2 == q.steps) cut(ks + 1);
        if constexpr (!C::DMA) fetch(q, terms, ks + 2);
        half(std::integral_constant<int, 0>{}, lds + ((ks + 1) & 1) * C::STAGE, a1, b1, a0, b0, [&](int m) {
          if constexpr (C::DMA) {
#pragma unroll
            for (int i = m * (A_LOADS + LB) / V; i < (m + 1) * (A_LOADS + LB) / V; ++i) load(i, A_LOADS);
          }
        });
      }
      if constexpr (C::DMA) wait_loads<0>();
      barrier();
    };
    if (q.steps > 0) {
      const int v = (q.rows + 16 * C::WM - 1) / (16 * C::WM);
      if (C::MT > 6 && v > 6) multiply(std::integral_constant<int, (C::MT > 6 ? 8 : 2)>{});
      else if (C::MT > 4 && v > 4) multiply(std::integral_constant<int, (C::MT > 4 ? 6 : 2)>{});
      else if (v > 2) multiply(std::integral_constant<int, 4>{});
      else multiply(std::integral_constant<int, 2>{});
    }
    const bool last = t + gridDim.x >= total;
    Tile following = q;
    if (!last) {
      t += gridDim.x;
      following = find(t);
      begin(following);
    }

    // ---- results: 16 rows of a wave at a time, by way of its 2 KB of LDS
    // (The lane is taken anew: what follows from it would otherwise be worked out ahead of the first tile and kept, for want of
    // registers, in memory, whose loads wait for all that is under way.  Offsets of the loads still are, see above.)
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int c = lane & 15, g = lane >> 4;
    const int oes = p.out_dtype == MOE_DT_FP32 ? 4 : 2;
#pragma unroll
    for (int n4 = 0; n4 < C::NT; n4 += 4) {
      const int64_t col0 = q.n0 + (wn * C::NT + n4) * 16;  // of these 64 columns, in the matrix
      const int cols = q.cols - (wn * C::NT + n4) * 16;    // that there are
      // (int8: what the scales and the bias bring waits for the stores ahead of them, a row tile's scale for those of the row tile before; with
      // a bias each of its 16 columns is waited for by itself.)
      v4f ws[4], bs[4];
      if constexpr (TYPE == GG_INT8) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int cc = n * 16 + 4 * g + i;
            const bool on = cc < cols && q.steps > 0;
            ws[n][i] = on ? p.b_scale[(int64_t)q.expert * p.N + col0 + cc] : 0.f;
            bs[n][i] = on && p.bias ? load_as_f32(p.bias, p.out_dtype, col0 + cc) : 0.f;
          }
      }
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        const int r0 = (m * C::WM + wm) * 16;  // of these 16 rows, in the tile
        if (r0 >= q.rows || cols <= 0) continue;
        v4f v[4];
        if constexpr (TYPE == GG_INT8) {
          const float xs = r0 + c < q.rows && q.steps > 0 ? p.a_scale[q.row0 + r0 + c] : 0.f;
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[n][i] = (float)acc[m][n4 + n][i] * xs * ws[n][i] + bs[n][i];
        } else {
#pragma unroll
          for (int n = 0; n < 4; ++n) v[n] = acc[m][n4 + n];
        }
        auto out_rows = [&](int first_col, int per_piece) {  // 8 pieces of 16 bytes a row
          asm volatile("" ::: "memory");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = h * 8 + (lane >> 3), piece = (lane & 7) ^ (r & 7), col = first_col + piece * per_piece;
            const uint4 d = *(const uint4*)(exchange + r * 128 + (lane & 7) * 16);
            if (r0 + r < q.rows && col < cols) {
              uint8_t* o = q.out + (int64_t)(r0 + r) * p.out_pitch + (col0 + col) * oes;
              if (C::WHOLE || col + per_piece <= cols) {
                *(bytes16*)o = bytes16{d.x, d.y, d.z, d.w};
              } else {
                const uint32_t w[4] = {d.x, d.y, d.z, d.w};
                if (oes == 2) {
                  for (int i = 0; i < cols - col; ++i) ((uint16_t*)o)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
                } else {
                  for (int i = 0; i < cols - col; ++i) ((uint32_t*)o)[i] = w[i];
                }
              }
            }
          }
          asm volatile("" ::: "memory");
          __builtin_amdgcn_wave_barrier();
        };
        if (p.out_dtype == MOE_DT_FP32) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int n = 0; n < 2; ++n) *(v4f*)(exchange + c * 128 + (((n * 4 + g) ^ (c & 7)) * 16)) = v[2 * h + n];
            out_rows(h * 32, 4);
          }
        } else {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            uint2 d;
            if (p.out_dtype == MOE_DT_BF16) {
              d = make_uint2(pack2_bf16(v[n][0], v[n][1]), pack2_bf16(v[n][2], v[n][3]));
            } else {
              typedef _Float16 v4h __attribute__((ext_vector_type(4)));
              const v4h h = __builtin_convertvector(v[n], v4h);
              d = __builtin_bit_cast(uint2, h);
            }
            *(uint2*)(exchange + c * 128 + (((n * 2 + (g >> 1)) ^ (c & 7)) * 16) + (g & 1) * 8) = d;
          }
          out_rows(0, 8);
        }
      }
    }
    if (last) return t + gridDim.x - total;
    stored = C::NT == 4 && q.rows == C::BM && q.cols == C::BN;
    q = following;
  }
}

// Tiles go out in rounds, in each of them a run of neighbours to every XCD (workgroup b is on XCD b % 8), so that what tiles share is
// in one L2 and all XCDs work at the same group.  (A run for all rounds gave one of 8 experts to each XCD: the gradient of their
// weights took 227 us for 8192 rows of 4096 x 2048, popular and unpopular, instead of 164.)
__device__ __forceinline__ int64_t first_tile() { return (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3); }
#define GG_KERNEL                                          \
  __global__ __launch_bounds__(C::THREADS) __attribute__(( \
      amdgpu_waves_per_eu(C::PER_CU * C::THREADS / 256, C::PER_CU * C::THREADS / 256)))

template <class C, int MODE, bool B_ROWS>
GG_KERNEL void grouped_kernel(const GroupedArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int* const bound = (int*)(smem + C::LDS);
  build_group_table(p.offsets, p.E, (int)p.S, C::BM, bound, bound + p.E + 3);
  tiles_of<C, MODE, B_ROWS>(p, smem, first_tile());
}
// Both gradients, of the rows and then of the weights (the same groups): the workgroups that the last round of the first leaves idle begin
// with the second.  (8192 rows of 4096 x 2048 bf16 in 8 groups: 2.25 and 4 rounds, 303 us; one after the other 322.)
template <class C>
GG_KERNEL void grouped_bwd_kernel(const GroupedArgs px, const GroupedArgs pw) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int* const bound = (int*)(smem + C::LDS);
  build_group_table(px.offsets, px.E, (int)px.S, C::BM, bound, bound + px.E + 3);
  const int64_t t = tiles_of<C, GG_ROWS, true>(px, smem, first_tile());
  __syncthreads();
  tiles_of<C, GG_CONTRACT, false>(pw, smem, t);
}

template <class C, int MODE>
int64_t most_tiles(const GroupedArgs& p) {  // (groups without rows have none)
  const int64_t ntn = (p.N + C::BN - 1) / C::BN, ntm = (p.K + C::BM - 1) / C::BM;
  return MODE == GG_ROWS ? ((p.S + C::BM - 1) / C::BM + (p.S < p.E + 1 ? p.S : p.E + 1)) * ntn : p.E * ntm * ntn;
}
template <class C>
unsigned workgroups(int64_t tiles) {  // no more than run at once
  const int cus = device_cus();
  const int64_t at_once = (int64_t)(cus > 0 ? cus : 256) * C::PER_CU;
  return (unsigned)((tiles < at_once ? tiles + 7 : at_once) / 8 * 8);
}
template <class C, int MODE, bool B_ROWS>
int launch(const GroupedArgs& p, hipStream_t s) {
  constexpr auto kernel = grouped_kernel<C, MODE, B_ROWS>;
  if (allow_lds<kernel>(160 * 1024) != hipSuccess) return MOE_E_LAUNCH;
  hipLaunchKernelGGL(kernel, dim3(workgroups<C>(most_tiles<C, MODE>(p))), dim3(C::THREADS), C::LDS + (p.E + 3) * 8, s, p);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}
template <class C>
int launch_bwd(const GroupedArgs& px, const GroupedArgs& pw, hipStream_t s) {
  constexpr auto kernel = grouped_bwd_kernel<C>;
  if (allow_lds<kernel>(160 * 1024) != hipSuccess) return MOE_E_LAUNCH;
  const int64_t tiles = most_tiles<C, GG_ROWS>(px) + most_tiles<C, GG_CONTRACT>(pw);
  hipLaunchKernelGGL(kernel, dim3(workgroups<C>(tiles)), dim3(C::THREADS), C::LDS + (px.E + 3) * 8, s, px, pw);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

#include "grouped_few.hpp"

typedef Cfg<256, 256, 2, 4, true, true, 1> Large;
typedef Cfg<128, 128, 2, 2, true, true, 2> Small;
typedef Cfg<256, 256, 2, 4, true, false, 1> LargeCut;
typedef Cfg<128, 128, 2, 2, true, false, 2> SmallCut;
typedef Cfg<128, 128, 2, 2, false, false, 2> Any;

// Which kernel: the one whose time per step of 64 terms (128 bytes), as it was measured, is the least, in ns; n: its tiles over the 256
// CUs of the chip.  A launch of few tiles takes the time of one tile's steps, one of many grows with them:
//   256 x 256  1250, from n = 0.86 on 1460 n   (8192 rows of 4096 x 1024 | 2048 bf16: 90 | 103 us)
//   128 x 128   600, from n = 1.25 on  480 n   (the same 68 | 129 us; 1 row of 7168 x 4096 int8 33, 2048 rows 75)
//   any address 1150, from there on 1200 n     (1999 rows of 1030 x 515 int8 22 us)
//   few rows, weights along their terms: 16 rows at a time 82, from n = 0.78 on 105 n; 32 rows 100, from n = 0.65 on 154 n
//     (7168 x 4096 int8, 1 | 16 | 32 | 64 rows: 10.5 | 10.6 | 13.6 | 22.4 us; tiles of 128 x 128 33 | 32 | 32 | 35)
//   few rows, weights across them: 282 | 358 for every round of the chip
//     (64 rows of 128 bf16 experts of 2048 x 1536: 61 us, tiles of 128 x 128 75; 2048 rows 166 and 161)
// Rows of a group are not known here: they are taken as spread over as many groups as there may be, half a tile of each filled up.  Where
// few of many groups have all the rows there are fewer tiles than that; what another kernel would then take has not been measured.
struct Estimate {
  int64_t S, groups, cols;
  int64_t tiles(int bm, int bn) const {
    const int64_t t = groups > 1 ? S / bm + groups / 2 : (S + bm - 1) / bm;
    return (t > groups ? t : groups) * ((cols + bn - 1) / bn);
  }
};
enum Kind { ANY, SMALL, LARGE, FEW1, FEW2 };
bool rows_at(const GroupedArgs& p, int bytes) {
  const uintptr_t at = (uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.a_pitch | (uintptr_t)p.b_pitch;
  return (at & (bytes - 1)) == 0;
}
bool whole_rows(const GroupedArgs& p) { return rows_at(p, 16) && (((uintptr_t)p.out | (uintptr_t)p.out_pitch) & 15) == 0; }
template <int MODE, bool B_ROWS>
Kind choose(const GroupedArgs& p) {
  const bool aligned = rows_at(p, 4);
  const int64_t groups = p.offsets ? (p.S < p.E ? p.S : p.E) : 1;
  const Estimate e = MODE == GG_ROWS ? Estimate{p.S, groups, p.N} : Estimate{p.K, 1, p.N};
  const int64_t each = MODE == GG_ROWS ? 1 : p.E;  // (a result per group)
  auto larger = [](int64_t a, int64_t b) { return a > b ? a : b; };
  const int64_t large = larger(1250, 1460 * each * e.tiles(256, 256) / 256), small = larger(600, 480 * each * e.tiles(128, 128) / 256);
  const int64_t any = larger(1150, 1200 * each * e.tiles(128, 128) / 256);
  const int64_t tile = !aligned ? any : large < small ? large : small;
  if constexpr (MODE == GG_ROWS) {
    constexpr int COLS = B_ROWS ? 16 : 128;
    const int64_t n1 = e.tiles(16, COLS), n2 = e.tiles(32, COLS);
    const int64_t few1 = B_ROWS ? larger(82, 105 * n1 / 256) : 282 * ((n1 + 255) / 256);
    const int64_t few2 = B_ROWS ? larger(100, 154 * n2 / 256) : 358 * ((n2 + 255) / 256);
    const int64_t few = few1 < few2 ? few1 : few2;
    // (a launch has fewer than 2^16 workgroups along the rows)
    if (few < tile && p.K * ES >= 16 && p.N >= 8 && p.S < (1 << 19)) return few1 <= few2 ? FEW1 : FEW2;
  }
  return !aligned ? ANY : large < small ? LARGE : SMALL;
}
template <int MODE, bool B_ROWS>
int run(const GroupedArgs& p, hipStream_t s) {
  const Kind kind = choose<MODE, B_ROWS>(p);
  if constexpr (MODE == GG_ROWS) {
    if (kind == FEW1) return launch_few<B_ROWS, 1>(p, p.a_pitch % 16 == 0, s);
    if (kind == FEW2) return launch_few<B_ROWS, 2>(p, p.a_pitch % 16 == 0, s);
  }
  if (kind == ANY) return launch<Any, MODE, B_ROWS>(p, s);
  if (whole_rows(p)) return kind == LARGE ? launch<Large, MODE, B_ROWS>(p, s) : launch<Small, MODE, B_ROWS>(p, s);
  return kind == LARGE ? launch<LargeCut, MODE, B_ROWS>(p, s) : launch<SmallCut, MODE, B_ROWS>(p, s);
}

}  // namespace

#if GG_TYPE == 2
int launch_grouped_int8(const GroupedArgs& p, hipStream_t s) { return run<GG_ROWS, true>(p, s); }
#else
#if GG_TYPE == 0
#define GG_NAME(WHAT) WHAT##_bf16
#else
#define GG_NAME(WHAT) WHAT##_fp16
#endif
int GG_NAME(launch_grouped)(const GroupedArgs& p, hipStream_t s) { return run<GG_ROWS, false>(p, s); }
int GG_NAME(launch_grouped_bwd)(const GroupedArgs* px, const GroupedArgs* pw, hipStream_t s) {
  if (px && pw && px->S > 0 && choose<GG_ROWS, true>(*px) == LARGE && choose<GG_CONTRACT, false>(*pw) == LARGE && whole_rows(*px) &&
      whole_rows(*pw))
    return launch_bwd<Large>(*px, *pw, s);
  if (px && px->S > 0) {
    const int rc = run<GG_ROWS, true>(*px, s);
    if (rc != MOE_OK) return rc;
  }
  return pw ? run<GG_CONTRACT, false>(*pw, s) : MOE_OK;
}
#endif

}  // namespace moe

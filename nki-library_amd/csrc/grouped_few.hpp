// Products by expert where there are too few tiles to fill the chip: few rows (decode), or small matrices.  Included by grouped_tile.hip.
//
// What bounds them is the stream of weights, or the chain of a single tile's steps.  So a workgroup takes few columns and its eight
// waves share the terms, chunk by chunk in turns; fragments come from memory straight into registers (nothing is used twice inside a
// workgroup but rows of x, which the caches hand out), the next chunk under the MFMAs of this one; the waves' sums meet in LDS, in
// the order of the waves.  16 MT rows of a group at a time.
//   weights along their terms ([E, N, K]): 16 columns a workgroup; a chunk is a line of 128 bytes of each row, two MFMAs deep
//   across them ([E, K, N]): 128 columns; a chunk is 32 terms.  A lane loads 8 columns of 8 terms, and 32 byte permutations make
//   operands of them: MFMA j takes column 8 c + j of lane c.  A lane whose columns pass the end takes the last 8 instead, which come
//   out twice alike.
#pragma once

constexpr int FEW_WAVES = 8;

// 16 bytes at `off` of a row of n >= 16, zeros behind its end.
template <bool WHOLE>
__device__ __forceinline__ v4i piece_of(const uint8_t* row, int off, int n) {
  const int from = off <= n - 16 ? off : n - 16;
  const bytes16 d = *(const bytes16*)(row + from);
  if constexpr (WHOLE) {
    const int keep = off < n ? ~0 : 0;
    return v4i{(int)d[0] & keep, (int)d[1] & keep, (int)d[2] & keep, (int)d[3] & keep};
  }
  const int gone = 8 * (off - from);
  uint64_t lo = (uint64_t)d[1] << 32 | d[0], hi = (uint64_t)d[3] << 32 | d[2];
  if (gone >= 64) {
    lo = gone < 128 ? hi >> (gone - 64) : 0;
    hi = 0;
  } else if (gone > 0) {
    lo = lo >> gone | hi << (64 - gone);
    hi >>= gone;
  }
  return v4i{(int)(uint32_t)lo, (int)(uint32_t)(lo >> 32), (int)(uint32_t)hi, (int)(uint32_t)(hi >> 32)};
}

__device__ __forceinline__ void store_value(uint8_t* row, int64_t col, int dtype, float v) {
  if (dtype == MOE_DT_FP32) ((float*)row)[col] = v;
  else if (dtype == MOE_DT_BF16) ((uint16_t*)row)[col] = (uint16_t)pack2_bf16(v, v);
  else ((_Float16*)row)[col] = (_Float16)v;
}

// WHOLE: rows are multiples of 16 bytes.
template <bool B_ROWS, int MT, bool WHOLE>
__global__ __launch_bounds__(FEW_WAVES * 64) void few_kernel(const GroupedArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int NT = B_ROWS ? 1 : 8, COLS = NT * 16, CHUNK = B_ROWS ? 128 : 64;  // CHUNK: bytes along the terms
  constexpr int STEPS = CHUNK / 64;                                              // MFMAs deep
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), c = lane & 15, g = lane >> 4;

  // the group and rows of this workgroup
  int expert = 0, begin = 0, rows = (int)p.S, tile = blockIdx.y;
  bool zero = false;
  if (p.offsets) {
    int* const bound = (int*)smem;
    int* const cum = bound + p.E + 3;
    build_group_table(p.offsets, p.E, (int)p.S, 16 * MT, bound, cum);
    if (tile >= uni(cum[p.E + 2])) return;
    const int j = group_of_tile(cum, p.E, tile);
    tile -= uni(cum[j]);
    begin = uni(bound[j]);
    rows = uni(bound[j + 1]) - begin;
    zero = j == 0 || j == p.E + 1;
    expert = zero ? 0 : j - 1;
    __syncthreads();  // (the sums use the table's place)
  }
  const int64_t row0 = begin + (int64_t)tile * 16 * MT;
  const int left = (int)(rows - (int64_t)tile * 16 * MT), have = left < 16 * MT ? left : 16 * MT;
  const int64_t n0 = (int64_t)blockIdx.x * COLS;
  const int kbytes = (int)p.K * ES;

  acc_t acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = acc_t{0, 0, 0, 0};
  // lane's column(s): rows of the matrix, or 8 neighbours
  const int64_t col = B_ROWS ? (n0 + c < p.N ? n0 + c : p.N - 1) : (n0 + 8 * c <= p.N - 8 ? n0 + 8 * c : p.N - 8);
  const uint8_t* const w = p.b + (int64_t)expert * p.b_group + (B_ROWS ? col * p.b_pitch : col * ES);
  const uint8_t* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = p.a + (row0 + (16 * m + c < have ? 16 * m + c : have - 1)) * p.a_pitch;

  struct Chunk {
    v4i x[MT][STEPS];
    v4i w[B_ROWS ? STEPS : 8];
  };
  const int chunks = zero ? 0 : (kbytes + CHUNK - 1) / CHUNK;
  auto load = [&](Chunk& q, int i) {
    if (i >= chunks) return;
    const int k = i * CHUNK;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
      for (int m = 0; m < MT; ++m) q.x[m][s] = piece_of<WHOLE>(xr[m], k + s * 64 + g * 16, kbytes);
      if constexpr (B_ROWS) q.w[s] = piece_of<WHOLE>(w, k + s * 64 + g * 16, kbytes);
    }
    if constexpr (!B_ROWS) {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int term = i * 32 + 8 * g + t;
        const bytes16 d = *(const bytes16*)(w + (int64_t)(term < p.K ? term : p.K - 1) * p.b_pitch);
        q.w[t] = v4i{(int)d[0], (int)d[1], (int)d[2], (int)d[3]};
      }
      if (i == chunks - 1) {  // (terms behind the last are zeros on both sides: what stands there may be no number)
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const int keep = i * 32 + 8 * g + t < p.K ? ~0 : 0;
          q.w[t] = v4i{q.w[t][0] & keep, q.w[t][1] & keep, q.w[t][2] & keep, q.w[t][3] & keep};
        }
      }
    }
  };
  auto multiply = [&](const Chunk& q) {
    if constexpr (B_ROWS) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][0] = mfma(q.x[m][s], q.w[s], acc[m][0]);
    } else {
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        v4i f;
#pragma unroll
        for (int t = 0; t < 4; ++t)  // column n of terms 2 t and 2 t + 1
          f[t] = (int)__builtin_amdgcn_perm((uint32_t)q.w[2 * t + 1][n / 2], (uint32_t)q.w[2 * t][n / 2], n & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][n] = mfma(q.x[m][0], f, acc[m][n]);
      }
    }
  };
  Chunk q0, q1;
  load(q0, wave);
  for (int i = wave; i < chunks; i += 2 * FEW_WAVES) {
    load(q1, i + FEW_WAVES);
    multiply(q0);
    if (i + FEW_WAVES >= chunks) break;
    load(q0, i + 2 * FEW_WAVES);
    multiply(q1);
  }

  // ---- the waves' sums, 16 rows at a time; lane (c, g) holds rows 4 g + i of column c (columns 8 c + n)
  typedef typename std::conditional<TYPE == GG_INT8, int, float>::type sum_t;
  typedef sum_t sum4 __attribute__((ext_vector_type(4)));
  sum_t* const part = (sum_t*)smem;  // [wave][16][COLS]
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (16 * m >= have) break;
    if (m > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum_t* const row = part + (wave * 16 + 4 * g + i) * COLS;
      if constexpr (B_ROWS) {
        row[c] = acc[m][0][i];
      } else {
        *(sum4*)(row + 8 * c) = sum4{acc[m][0][i], acc[m][1][i], acc[m][2][i], acc[m][3][i]};
        *(sum4*)(row + 8 * c + 4) = sum4{acc[m][4][i], acc[m][5][i], acc[m][6][i], acc[m][7][i]};
      }
    }
    __syncthreads();
    constexpr int PER = B_ROWS ? 1 : 4;  // columns of a thread
    if (tid < 16 * COLS / PER) {
      const int r = tid / (COLS / PER), cc = tid % (COLS / PER) * PER;
      sum_t s[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) s[i] = part[r * COLS + cc + i];
#pragma unroll
      for (int v = 1; v < FEW_WAVES; ++v)
#pragma unroll
        for (int i = 0; i < PER; ++i) s[i] += part[(v * 16 + r) * COLS + cc + i];
      if (16 * m + r < have && n0 + (B_ROWS ? cc : cc & ~7) < p.N) {
        const int64_t row = row0 + 16 * m + r;
        const int64_t first = B_ROWS ? n0 + cc : (n0 + (cc & ~7) <= p.N - 8 ? n0 + (cc & ~7) : p.N - 8) + (cc & 4);
        uint8_t* const out = p.out + row * p.out_pitch;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          float v = (float)s[i];
          if constexpr (TYPE == GG_INT8) {
            v = zero ? 0.f : v * p.a_scale[row] * p.b_scale[(int64_t)expert * p.N + first + i];
            if (p.bias) v += load_as_f32(p.bias, p.out_dtype, first + i);
          }
          store_value(out, first + i, p.out_dtype, v);
        }
      }
    }
  }
}

template <bool B_ROWS, int MT>
int launch_few(const GroupedArgs& p, bool whole, hipStream_t s) {
  constexpr int COLS = B_ROWS ? 16 : 128;
  const int sums = FEW_WAVES * 16 * COLS * 4, table = p.offsets ? (p.E + 3) * 8 : 0, lds = sums > table ? sums : table;
  const int64_t tiles = p.offsets ? p.S / (16 * MT) + (p.S < p.E + 2 ? p.S : p.E + 2) : (p.S + 16 * MT - 1) / (16 * MT);
  const dim3 grid((unsigned)((p.N + COLS - 1) / COLS), (unsigned)tiles);
  if (whole) {
    constexpr auto kernel = few_kernel<B_ROWS, MT, true>;
    if (allow_lds<kernel>(64 * 1024) != hipSuccess) return MOE_E_LAUNCH;
    hipLaunchKernelGGL(kernel, grid, dim3(FEW_WAVES * 64), lds, s, p);
  } else {
    constexpr auto kernel = few_kernel<B_ROWS, MT, false>;
    if (allow_lds<kernel>(64 * 1024) != hipSuccess) return MOE_E_LAUNCH;
    hipLaunchKernelGGL(kernel, grid, dim3(FEW_WAVES * 64), lds, s, p);
  }
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

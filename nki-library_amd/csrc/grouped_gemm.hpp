// Products of ragged groups of rows with a matrix per group (grouped_gemm.hip, grouped_tile.hip, grouped_few.hpp).
#pragma once

#include "common.hpp"

namespace moe {

// What is multiplied: rows of a with the group's matrix, out[s, n] = sum over k of a[s, k] b[e(s), k, n] (GG_ROWS), or, group by
// group, the rows of a with the rows of b, out[e, m, n] = sum over the rows s of e of a[s, m] b[s, n] (GG_CONTRACT).
enum { GG_ROWS = 0, GG_CONTRACT = 1 };
enum { GG_BF16 = 0, GG_FP16 = 1, GG_INT8 = 2 };  // element of both operands

constexpr int GG_MAX_GROUPS = 1024;

struct GroupedArgs {
  const uint8_t* a;
  const uint8_t* b;
  uint8_t* out;
  const int32_t* offsets;  // [E + 1] rows at which the groups begin and end; null: one group of all rows
  const float* a_scale;    // int8: per row, per group and column
  const float* b_scale;
  const void* bias;        // int8, dense: per column, of the output's type
  int64_t S, K, N;         // rows in all; GG_ROWS: length of a row, GG_CONTRACT: its columns, the rows of a result; columns of a result
  int64_t a_pitch, b_pitch, b_group, out_pitch;  // bytes from row to row, from matrix to matrix
  int E;
  int out_dtype;  // MOE_DT_*
};

// The groups' bounds as a workgroup keeps them: group j of E + 2 holds rows [bound[j], bound[j + 1]) and tiles [cum[j], cum[j + 1])
// of `bm` rows each.  Groups 0 and E + 1 are the rows ahead of the first expert's and behind the last one's, which get zeros;
// group j is expert j - 1.  Offsets are taken into [0, S] and never fall, so that whatever they are every row has one group.
__device__ __forceinline__ int wave_excl_max(int v) {
  const int lane = threadIdx.x & 63;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(inc, o, 64);
    if (lane >= o && u > inc) inc = u;
  }
  const int e = __shfl_up(inc, 1, 64);
  return lane == 0 ? 0 : e;
}
__device__ __forceinline__ int wave_excl_sum(int v) {
  const int lane = threadIdx.x & 63;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(inc, o, 64);
    if (lane >= o) inc += u;
  }
  return inc - v;
}
// (ends with a barrier)
__device__ __forceinline__ void build_group_table(const int32_t* __restrict__ offsets, int E, int S, int bm, int* bound, int* cum) {
  const int n = E + 3;  // bounds 0, offsets[0 .. E], S
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    int v = j == 0 ? 0 : S;
    if (j >= 1 && j <= E + 1) {
      v = offsets ? offsets[j - 1] : j == 1 ? 0 : S;
      v = v < 0 ? 0 : v > S ? S : v;
    }
    bound[j] = v;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int per = (n + 63) / 64, j0 = threadIdx.x * per, j1 = j0 + per < n ? j0 + per : n;
    int m = 0;
    for (int j = j0; j < j1; ++j) m = bound[j] > m ? bound[j] : m;
    m = wave_excl_max(m);
    for (int j = j0; j < j1; ++j) {
      m = bound[j] > m ? bound[j] : m;
      bound[j] = m;
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int per = (n + 63) / 64, j0 = threadIdx.x * per, j1 = j0 + per < n ? j0 + per : n;
    auto tiles = [&](int j) { return j + 1 < n ? (bound[j + 1] - bound[j] + bm - 1) / bm : 0; };
    int t = 0;
    for (int j = j0; j < j1; ++j) t += tiles(j);
    t = wave_excl_sum(t);
    for (int j = j0; j < j1; ++j) {
      cum[j] = t;
      t += tiles(j);
    }
  }
  __syncthreads();
}
// The group whose tiles hold tile r (r < cum[E + 2]).
__device__ __forceinline__ int group_of_tile(const int* cum, int E, int r) {
  int lo = 0, hi = E + 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid + 1] <= r) lo = mid + 1;
    else hi = mid;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// A product, and its gradients (either may be null).
int launch_grouped_bf16(const GroupedArgs& p, hipStream_t s);
int launch_grouped_fp16(const GroupedArgs& p, hipStream_t s);
int launch_grouped_bwd_bf16(const GroupedArgs* px, const GroupedArgs* pw, hipStream_t s);
int launch_grouped_bwd_fp16(const GroupedArgs* px, const GroupedArgs* pw, hipStream_t s);
int launch_grouped_int8(const GroupedArgs& p, hipStream_t s);

}  // namespace moe

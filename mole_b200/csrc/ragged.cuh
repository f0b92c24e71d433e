// Products over rows packed by expert: interface between the C entries (ragged.cu) and the kernels.
//
// Expert e owns the rows [offsets[e], offsets[e + 1]) of the packed matrices; the offsets live on
// the device and are never read by the host.  Rows before offsets[0] and from offsets[E] on belong
// to nobody: products write zeros there.  Offsets are clamped on the device to 0 <= o[0] <= ... <= R,
// so a bad array costs a wrong result and never an access out of range.
#pragma once
#include "common.cuh"

namespace mole {

struct RaggedRows {         // out[r, n] = sum_k x[r, k] w_e(n, k)
  const void* x;            // [R, K]
  const void* w;            // [E, N, K] (kn = 0) or [E, K, N] (kn = 1)
  const int32_t* offsets;   // [E + 1], or null: one expert, all rows
  const float* x_scale;     // 8-bit integers: scale of row r,
  const float* w_scale;     //                 scale of channel (e, n)
  void* out;                // [R, N]
  int64_t R;
  int N, K, E, kn;
  int ldx, ldw;             // elements between rows of x, and of w's inner matrices
  float* part;              // fp32: room for `split` partial results [R, N] (split > 1)
  int split;
};
struct RaggedWgrad {        // out[e, p, q] = sum over the rows r of e of a[r, p] b[r, q]
  const void* a;            // [R, P]
  const void* b;            // [R, Q]
  const int32_t* offsets;
  void* out;                // [E, P, Q]
  int64_t R;
  int P, Q, E;
  int lda, ldb;
  float* part;              // room for `split` partial results [E, P, Q] (split > 1)
  int split;
};

int ragged_rows_simt(const RaggedRows& a, cudaStream_t st);          // fp32
int ragged_wgrad_simt(const RaggedWgrad& a, cudaStream_t st);
// Into how many parts the reduction is cut where there are too few tiles for the SMs; partial results
// are added in their order by ragged_join.
int ragged_rows_simt_split(const RaggedRows& a);
int ragged_wgrad_split(bool tensor, const RaggedWgrad& a);
int ragged_join(int out_dtype, const float* part, int split, int64_t n, void* out, cudaStream_t st);
// up to 16 rows, every type (ldx = K, ldw dense)
bool ragged_rows_few_takes(const RaggedRows& a);
int ragged_rows_few(int dtype, const RaggedRows& a, cudaStream_t st);
int ragged_rows_few_i8(int out_dtype, const RaggedRows& a, cudaStream_t st);
// tensor cores; elem 2 = bf16, 1 = 8-bit integers.  Rows of every operand start on 16 bytes (base and ld).
int ragged_rows_tc(int elem, int out_dtype, const RaggedRows& a, cudaStream_t st);
int ragged_wgrad_tc(const RaggedWgrad& a, cudaStream_t st);

constexpr int kMaxRaggedExperts = 256;
// Spans of rows: 0 = the rows before the first expert, 1 .. E = the experts, E + 1 = the rows behind
// the last.  row0[i] .. row0[i + 1] is span i, tile0[i] the tiles before it (of 2^shift rows).
struct RaggedSpans {
  int row0[kMaxRaggedExperts + 3];
  int tile0[kMaxRaggedExperts + 3];
};

// By one whole warp; the caller synchronises the block afterwards.
__device__ __forceinline__ void load_spans(RaggedSpans& s, const int32_t* offsets, int E, int R, int shift) {
  const int lane = threadIdx.x & 31, unit1 = (1 << shift) - 1;
  int row = 0, tiles = 0;                            // where the spans so far end
#pragma unroll 1
  for (int j0 = 0; j0 < E + 2; j0 += 32) {           // a span per lane
    const int j = j0 + lane;
    int end = R;
    if (j <= E) end = offsets ? min(max(offsets[j], 0), R) : j == 0 ? 0 : R;
    if (lane == 0) end = max(end, row);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {               // never before the end of an earlier one
      const int v = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end = max(end, v);
    }
    int first = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) first = row;
    int sum = (end - first + unit1) >> shift;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    sum += tiles;
    if (j < E + 2) { s.row0[j + 1] = end; s.tile0[j + 1] = sum; }
    row = __shfl_sync(0xffffffffu, end, 31);
    tiles = __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) { s.row0[0] = 0; s.tile0[0] = 0; }
}
// the span that holds tile t (t < tile0[E + 2]): the last one that starts at or before it
__device__ __forceinline__ int span_of(const RaggedSpans& s, int E, int t) {
  int lo = 0, hi = E + 2;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.tile0[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

}  // namespace mole

// Products over rows packed by expert on the CUDA cores: every size, alignment and type.  fp32 runs
// here (its products have to be exact to 2^-24, which the tensor cores' input types are not), and so
// do the widths whose rows a TMA load cannot address.
#include "ragged.cuh"

namespace mole {

constexpr int kST = 64;      // tile of rows and of columns
constexpr int kSK = 16;      // reduction per step

template <typename T> struct SimtIn {
  using Acc = float;
  __device__ static __forceinline__ float get(T v) { return Elem<T>::to_f(v); }
};
template <> struct SimtIn<int8_t> {
  using Acc = int;
  __device__ static __forceinline__ int get(int8_t v) { return v; }
};

// acc[4][4] += A (64 x 16, row ty * 4 + i) * B (16 x 64, column tx * 4 + j)
template <typename Acc>
__device__ __forceinline__ void simt_step(const Acc (&as)[kSK][kST + 4], const Acc (&bs)[kSK][kST + 4], Acc (&acc)[4][4],
                                          int ty, int tx) {
#pragma unroll
  for (int k = 0; k < kSK; ++k) {
    Acc a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = as[k][ty * 4 + i]; b[i] = bs[k][tx * 4 + i]; }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += a[i] * b[j];
  }
}

template <typename TI, typename TO, bool KN>
__global__ void __launch_bounds__(256)
ragged_rows_kernel(const RaggedRows a) {
  using Acc = typename SimtIn<TI>::Acc;
  constexpr bool I8 = sizeof(TI) == 1;
  __shared__ RaggedSpans sp;
  __shared__ Acc as[kSK][kST + 4], bs[kSK][kST + 4];
  const int t = threadIdx.x;
  if (t < 32) load_spans(sp, a.offsets, a.E, (int)a.R, kST);
  __syncthreads();
  const int tile = blockIdx.x;
  if (tile >= sp.tile0[a.E + 2]) return;
  const int span = span_of(sp, a.E, tile);
  const int r0 = sp.row0[span] + (tile - sp.tile0[span]) * kST, rend = sp.row0[span + 1];
  const int n0 = blockIdx.y * kST;
  const int ty = t >> 4, tx = t & 15;
  TO* out = static_cast<TO*>(a.out);
  const int e = span - 1;
  const bool owned = e >= 0 && e < a.E;
  Acc acc[4][4] = {};
  if (owned) {
    const TI* x = static_cast<const TI*>(a.x);
    const TI* w = static_cast<const TI*>(a.w) + (int64_t)e * a.N * a.K;
    for (int k0 = 0; k0 < a.K; k0 += kSK) {
      {
        const int r = r0 + (t >> 2), k = k0 + (t & 3) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          as[(t & 3) * 4 + i][t >> 2] =
              (r < rend && k + i < a.K) ? SimtIn<TI>::get(x[(int64_t)r * a.K + k + i]) : Acc(0);
      }
      if (KN) {
        const int k = k0 + (t >> 4), n = n0 + (t & 15) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          bs[t >> 4][(t & 15) * 4 + i] =
              (k < a.K && n + i < a.N) ? SimtIn<TI>::get(w[(int64_t)k * a.N + n + i]) : Acc(0);
      } else {
        const int n = n0 + (t >> 2), k = k0 + (t & 3) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          bs[(t & 3) * 4 + i][t >> 2] =
              (n < a.N && k + i < a.K) ? SimtIn<TI>::get(w[(int64_t)n * a.K + k + i]) : Acc(0);
      }
      __syncthreads();
      simt_step(as, bs, acc, ty, tx);
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + ty * 4 + i;
    if (r >= rend) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n >= a.N) continue;
      float v = (float)acc[i][j];
      // the token's scale, then the channel's
      if (I8 && owned) v = __fmul_rn(__fmul_rn(v, a.x_scale[r]), a.w_scale[(int64_t)e * a.N + n]);
      out[(int64_t)r * a.N + n] = Elem<TO>::from_f(v);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
ragged_wgrad_kernel(const RaggedWgrad a) {
  __shared__ RaggedSpans sp;
  __shared__ float as[kSK][kST + 4], bs[kSK][kST + 4];
  const int t = threadIdx.x;
  if (t < 32) load_spans(sp, a.offsets, a.E, (int)a.R, kST);
  __syncthreads();
  const int e = blockIdx.z, q0 = blockIdx.x * kST, p0 = blockIdx.y * kST;
  const int r0 = sp.row0[e + 1], rend = sp.row0[e + 2];
  const int ty = t >> 4, tx = t & 15;
  const T* A = static_cast<const T*>(a.a);
  const T* B = static_cast<const T*>(a.b);
  float acc[4][4] = {};
  for (int r1 = r0; r1 < rend; r1 += kSK) {
    const int r = r1 + (t >> 4), c = (t & 15) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      as[t >> 4][c + i] = (r < rend && p0 + c + i < a.P) ? Elem<T>::to_f(A[(int64_t)r * a.P + p0 + c + i]) : 0.f;
      bs[t >> 4][c + i] = (r < rend && q0 + c + i < a.Q) ? Elem<T>::to_f(B[(int64_t)r * a.Q + q0 + c + i]) : 0.f;
    }
    __syncthreads();
    simt_step(as, bs, acc, ty, tx);
    __syncthreads();
  }
  T* out = static_cast<T*>(a.out) + (int64_t)e * a.P * a.Q;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + ty * 4 + i, q = q0 + tx * 4 + j;
      if (p < a.P && q < a.Q) out[(int64_t)p * a.Q + q] = Elem<T>::from_f(acc[i][j]);
    }
}

// every span may end in a partial tile
static dim3 rows_grid(const RaggedRows& a) {
  return dim3((unsigned)(a.R / kST + a.E + 2), (unsigned)((a.N + kST - 1) / kST));
}

int ragged_rows_simt(int dtype, const RaggedRows& a, cudaStream_t st) {
  const dim3 grid = rows_grid(a);
  if (dtype == MOLE_F32) {
    if (a.kn) ragged_rows_kernel<float, float, true><<<grid, 256, 0, st>>>(a);
    else ragged_rows_kernel<float, float, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (a.kn) ragged_rows_kernel<__nv_bfloat16, __nv_bfloat16, true><<<grid, 256, 0, st>>>(a);
    else ragged_rows_kernel<__nv_bfloat16, __nv_bfloat16, false><<<grid, 256, 0, st>>>(a);
  }
  MOLE_LAUNCH_OK();
  return MOLE_OK;
}
int ragged_rows_simt_i8(int out_dtype, const RaggedRows& a, cudaStream_t st) {
  const dim3 grid = rows_grid(a);
  if (out_dtype == MOLE_F32) ragged_rows_kernel<int8_t, float, false><<<grid, 256, 0, st>>>(a);
  else ragged_rows_kernel<int8_t, __nv_bfloat16, false><<<grid, 256, 0, st>>>(a);
  MOLE_LAUNCH_OK();
  return MOLE_OK;
}
int ragged_wgrad_simt(int dtype, const RaggedWgrad& a, cudaStream_t st) {
  const dim3 grid((unsigned)((a.Q + kST - 1) / kST), (unsigned)((a.P + kST - 1) / kST), (unsigned)a.E);
  if (dtype == MOLE_F32) ragged_wgrad_kernel<float><<<grid, 256, 0, st>>>(a);
  else ragged_wgrad_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  MOLE_LAUNCH_OK();
  return MOLE_OK;
}

}  // namespace mole

// Products over rows packed by expert on the CUDA cores: every size, alignment and type.  fp32 runs
// here (its products have to be exact to 2^-24, which the tensor cores' input types are not), and so
// do the widths whose rows a TMA load cannot address.
//
// A thread block takes a tile of T x T outputs, a thread (T / 16)^2 of them in registers; tiles of both
// operands, 16 deep in the reduction, go through shared memory, the next ones on their way in
// registers meanwhile.  With T = 128 a thread makes 64 multiply-adds per step on four 16-byte reads:
// bound by the fp32 pipes (8192 x 512 x 2048 over 8 experts in REPLACE_FP32).  T = 64 where experts have few
// rows.  Sums run over the reduction in its order, one fused multiply-add after the other.
#include <type_traits>

#include "ragged.cuh"

namespace mole {

constexpr int kSK = 16;      // reduction per step

template <typename T> struct SimtIn {
  using Acc = float;
  __device__ static __forceinline__ float get(T v) { return Elem<T>::to_f(v); }
};
template <> struct SimtIn<int8_t> {
  using Acc = int;
  __device__ static __forceinline__ int get(int8_t v) { return v; }
};
__device__ __forceinline__ void mad(float& c, float a, float b) { c = fmaf(a, b, c); }
__device__ __forceinline__ void mad(int& c, int a, int b) { c += a * b; }

// Eight neighbouring elements, those from `n` on as zeros
template <typename TI, bool WIDE, typename Acc>
__device__ __forceinline__ void load8(const TI* p, int n, Acc (&v)[8]) {
  if (WIDE && n >= 8) {
    if constexpr (sizeof(TI) == 1) {
      const uint2 t = *reinterpret_cast<const uint2*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (Acc)(int8_t)((i < 4 ? t.x : t.y) >> (8 * (i & 3)));
    } else {
      constexpr int V = Vec16<TI>::N;
#pragma unroll
      for (int i = 0; i < 8 / V; ++i) {
        float t[V];
        Vec16<TI>::load(p + i * V, t);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i * V + j] = t[j];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? SimtIn<TI>::get(p[i]) : Acc(0);
  }
}

// One operand's tile: `mn` runs over T rows (or columns) of the output, k over the reduction.  KMAJOR:
// element (mn, k) at p + mn * ld + k, else at p + k * ld + mn.
template <typename TI, int T, bool KMAJOR, bool WIDE>
struct Operand {
  using Acc = typename SimtIn<TI>::Acc;
  static constexpr int kThreads = KMAJOR ? 2 * T : 2 * T;        // that load: T * 16 elements, eight each
  Acc v[8];
  // `mn_left`, `k_left`: what exists from this tile's first element on
  __device__ __forceinline__ void fetch(const TI* p, int64_t ld, int mn_left, int k_left) {
    const int t = threadIdx.x;
    if (t >= kThreads) return;
    if (KMAJOR) {
      const int mn = t % T, k = t / T * 8;
      load8<TI, WIDE>(p + (int64_t)mn * ld + k, mn < mn_left ? k_left - k : 0, v);
    } else {
      const int k = t / (T / 8), mn = t % (T / 8) * 8;
      load8<TI, WIDE>(p + (int64_t)k * ld + mn, k < k_left ? mn_left - mn : 0, v);
    }
  }
  __device__ __forceinline__ void put(Acc (&s)[kSK][T + 4]) const {
    const int t = threadIdx.x;
    if (t >= kThreads) return;
    if (KMAJOR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[t / T * 8 + i][t % T] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[t / (T / 8)][t % (T / 8) * 8 + i] = v[i];
    }
  }
};

// acc = A (T x K) B (K x T); pa and pb point to the tile's first elements at k = 0.  Output (i, j) of a
// thread is row row_of(i), column col_of(j) of the tile.
template <int T>
__device__ __forceinline__ int tile_index(int t16, int i) { return (i >> 2) * 64 + t16 * 4 + (i & 3); }
template <typename TI, int T, bool A_K, bool B_K, bool WIDE>
__device__ __forceinline__ void tile_product(const TI* pa, int64_t lda, int m_left, const TI* pb, int64_t ldb, int n_left,
                                             int K, typename SimtIn<TI>::Acc (&acc)[T / 16][T / 16]) {
  using Acc = typename SimtIn<TI>::Acc;
  constexpr int M = T / 16;
  __shared__ __align__(16) Acc as[2][kSK][T + 4], bs[2][kSK][T + 4];
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  Operand<TI, T, A_K, WIDE> a;
  Operand<TI, T, B_K, WIDE> b;
  a.fetch(pa, lda, m_left, K);
  b.fetch(pb, ldb, n_left, K);
  a.put(as[0]);
  b.put(bs[0]);
  __syncthreads();
  for (int k0 = 0, buf = 0; k0 < K; k0 += kSK, buf ^= 1) {
    const bool more = k0 + kSK < K;
    if (more) {
      const int k1 = k0 + kSK;
      a.fetch(A_K ? pa + k1 : pa + (int64_t)k1 * lda, lda, m_left, K - k1);
      b.fetch(B_K ? pb + k1 : pb + (int64_t)k1 * ldb, ldb, n_left, K - k1);
    }
#pragma unroll
    for (int k = 0; k < kSK; ++k) {
      Acc x[M], y[M];
#pragma unroll
      for (int i = 0; i < M; ++i) { x[i] = as[buf][k][tile_index<T>(ty, i)]; y[i] = bs[buf][k][tile_index<T>(tx, i)]; }
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int j = 0; j < M; ++j) mad(acc[i][j], x[i], y[j]);
    }
    if (more) {
      a.put(as[buf ^ 1]);
      b.put(bs[buf ^ 1]);
      __syncthreads();
    }
  }
}

template <typename TI, typename TO, int T, bool KN, bool WIDE>
__global__ void __launch_bounds__(256, T == 128 ? 2 : 4)
ragged_rows_kernel(const RaggedRows a) {
  using Acc = typename SimtIn<TI>::Acc;
  constexpr bool I8 = sizeof(TI) == 1;
  constexpr int M = T / 16;
  __shared__ RaggedSpans sp;
  if (threadIdx.x < 32) load_spans(sp, a.offsets, a.E, (int)a.R, T);
  __syncthreads();
  const int tile = blockIdx.x;
  if (tile >= sp.tile0[a.E + 2]) return;
  const int span = span_of(sp, a.E, tile);
  const int r0 = sp.row0[span] + (tile - sp.tile0[span]) * T, rend = sp.row0[span + 1];
  const int n0 = blockIdx.y * T;
  TO* out = static_cast<TO*>(a.out);
  const int e = span - 1;
  const bool owned = e >= 0 && e < a.E;
  Acc acc[M][M] = {};
  if (owned) {
    const TI* x = static_cast<const TI*>(a.x) + (int64_t)r0 * a.K;
    const TI* w = static_cast<const TI*>(a.w) + (int64_t)e * a.N * a.K;
    tile_product<TI, T, true, !KN, WIDE>(x, a.K, rend - r0, KN ? w + n0 : w + (int64_t)n0 * a.K, KN ? a.N : a.K, a.N - n0,
                                         a.K, acc);
  }
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int r = r0 + tile_index<T>(ty, i);
    if (r >= rend) continue;
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const int n = n0 + tile_index<T>(tx, j);
      if (n >= a.N) continue;
      float v = (float)acc[i][j];
      // the token's scale, then the channel's
      if (I8 && owned) v = __fmul_rn(__fmul_rn(v, a.x_scale[r]), a.w_scale[(int64_t)e * a.N + n]);
      out[(int64_t)r * a.N + n] = Elem<TO>::from_f(v);
    }
  }
}

template <typename TI, int T, bool WIDE>
__global__ void __launch_bounds__(256, T == 128 ? 2 : 4)
ragged_wgrad_kernel(const RaggedWgrad a) {
  constexpr int M = T / 16;
  __shared__ RaggedSpans sp;
  if (threadIdx.x < 32) load_spans(sp, a.offsets, a.E, (int)a.R, T);
  __syncthreads();
  const int e = blockIdx.z, q0 = blockIdx.x * T, p0 = blockIdx.y * T;
  const int r0 = sp.row0[e + 1], rows = sp.row0[e + 2] - r0;
  float acc[M][M] = {};
  if (rows > 0)
    tile_product<TI, T, false, false, WIDE>(static_cast<const TI*>(a.a) + (int64_t)r0 * a.P + p0, a.P, a.P - p0,
                                            static_cast<const TI*>(a.b) + (int64_t)r0 * a.Q + q0, a.Q, a.Q - q0, rows, acc);
  TI* out = static_cast<TI*>(a.out) + (int64_t)e * a.P * a.Q;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const int p = p0 + tile_index<T>(ty, i), q = q0 + tile_index<T>(tx, j);
      if (p < a.P && q < a.Q) out[(int64_t)p * a.Q + q] = Elem<TI>::from_f(acc[i][j]);
    }
}

// eight elements from a multiple of eight on can be loaded in 16-byte pieces (8 bytes of integers)
static bool wide_rows(const void* p, int64_t ld, int elem) {
  const uintptr_t unit = elem == 1 ? 8 : 16;
  return (ld * elem) % unit == 0 && (reinterpret_cast<uintptr_t>(p) & (unit - 1)) == 0;
}

template <typename TI, typename TO, bool KN>
static int launch_rows(const RaggedRows& a, cudaStream_t st) {
  const bool wide = wide_rows(a.x, a.K, sizeof(TI)) && wide_rows(a.w, KN ? a.N : a.K, sizeof(TI));
  // 128-row tiles once experts have about as many rows on average: half a tile per expert is idle
  const bool large = a.R >= 128ll * a.E && a.N > 64;
  auto grid = [&](int T) {
    return dim3((unsigned)(a.R / T + a.E + 2), (unsigned)((a.N + T - 1) / T));     // every span may end in a partial tile
  };
  if (large && wide) ragged_rows_kernel<TI, TO, 128, KN, true><<<grid(128), 256, 0, st>>>(a);
  else if (large) ragged_rows_kernel<TI, TO, 128, KN, false><<<grid(128), 256, 0, st>>>(a);
  else if (wide) ragged_rows_kernel<TI, TO, 64, KN, true><<<grid(64), 256, 0, st>>>(a);
  else ragged_rows_kernel<TI, TO, 64, KN, false><<<grid(64), 256, 0, st>>>(a);
  MOLE_LAUNCH_OK();
  return MOLE_OK;
}
template <typename TI>
static int launch_wgrad(const RaggedWgrad& a, cudaStream_t st) {
  const bool wide = wide_rows(a.a, a.P, sizeof(TI)) && wide_rows(a.b, a.Q, sizeof(TI));
  // 128 x 128 tiles where they fill the SMs
  auto grid = [&](int T) { return dim3((unsigned)((a.Q + T - 1) / T), (unsigned)((a.P + T - 1) / T), (unsigned)a.E); };
  const dim3 g = grid(128);
  const bool large = (int64_t)g.x * g.y * g.z >= 2 * sm_count();
  if (large && wide) ragged_wgrad_kernel<TI, 128, true><<<g, 256, 0, st>>>(a);
  else if (large) ragged_wgrad_kernel<TI, 128, false><<<g, 256, 0, st>>>(a);
  else if (wide) ragged_wgrad_kernel<TI, 64, true><<<grid(64), 256, 0, st>>>(a);
  else ragged_wgrad_kernel<TI, 64, false><<<grid(64), 256, 0, st>>>(a);
  MOLE_LAUNCH_OK();
  return MOLE_OK;
}

int ragged_rows_simt(int dtype, const RaggedRows& a, cudaStream_t st) {
  if (dtype == MOLE_F32) return a.kn ? launch_rows<float, float, true>(a, st) : launch_rows<float, float, false>(a, st);
  return a.kn ? launch_rows<__nv_bfloat16, __nv_bfloat16, true>(a, st) : launch_rows<__nv_bfloat16, __nv_bfloat16, false>(a, st);
}
int ragged_rows_simt_i8(int out_dtype, const RaggedRows& a, cudaStream_t st) {
  return out_dtype == MOLE_F32 ? launch_rows<int8_t, float, false>(a, st) : launch_rows<int8_t, __nv_bfloat16, false>(a, st);
}
int ragged_wgrad_simt(int dtype, const RaggedWgrad& a, cudaStream_t st) {
  return dtype == MOLE_F32 ? launch_wgrad<float>(a, st) : launch_wgrad<__nv_bfloat16>(a, st);
}

}  // namespace mole

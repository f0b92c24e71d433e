// fp32 products over rows packed by expert, on the CUDA cores: they have to be exact to 2^-24, which the
// tensor cores' input types are not.  Every size and alignment.
//
// A thread block takes a tile of T x T outputs, a thread (T / 16)^2 of them in registers; tiles of both
// operands, 16 deep in the reduction, go through shared memory, the next ones on their way in
// registers meanwhile.  With T = 128 a thread makes 64 multiply-adds per step on four 16-byte reads.
// T = 64 where experts have few rows.  Sums run over the reduction in its order, one fused
// multiply-add after the other.  Bound by the fp32 pipes: 8192 rows, 8 experts of 512 x 2048 in 0.45 ms
// each way, 38 to 41 TFLOP/s, which is what a plain loop of library products reaches; pairs on the
// packed instructions (0.52 ms), fragments read one step ahead and one block of twice the registers
// per SM (0.45 to 0.5) are no faster.
#include "ragged.cuh"

namespace mole {

constexpr int kSK = 16;      // reduction per step

// Eight neighbouring elements, those from `n` on as zeros
template <bool WIDE>
__device__ __forceinline__ void load8(const float* p, int n, float (&v)[8]) {
  if (WIDE && n >= 8) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}

// One operand's tile: `mn` runs over T rows (or columns) of the output, k over the reduction.  KMAJOR:
// element (mn, k) at p + mn * ld + k, else at p + k * ld + mn.
template <int T, bool KMAJOR, bool WIDE>
struct Operand {
  static constexpr int kThreads = 2 * T;         // that load: T * 16 elements, eight each
  float v[8];
  // `mn_left`, `k_left`: what exists from this tile's first element on
  __device__ __forceinline__ void fetch(const float* p, int64_t ld, int mn_left, int k_left) {
    const int t = threadIdx.x;
    if (t >= kThreads) return;
    if (KMAJOR) {
      const int mn = t % T, k = t / T * 8;
      load8<WIDE>(p + (int64_t)mn * ld + k, mn < mn_left ? k_left - k : 0, v);
    } else {
      const int k = t / (T / 8), mn = t % (T / 8) * 8;
      load8<WIDE>(p + (int64_t)k * ld + mn, k < k_left ? mn_left - mn : 0, v);
    }
  }
  __device__ __forceinline__ void put(float (&s)[kSK][T + 4]) const {
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
template <int T, bool A_K, bool B_K, bool WIDE>
__device__ __forceinline__ void tile_product(const float* pa, int64_t lda, int m_left, const float* pb, int64_t ldb,
                                             int n_left, int K, float (&acc)[T / 16][T / 16]) {
  constexpr int M = T / 16;
  __shared__ __align__(16) float as[2][kSK][T + 4], bs[2][kSK][T + 4];
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  Operand<T, A_K, WIDE> a;
  Operand<T, B_K, WIDE> b;
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
      float x[M], y[M];
#pragma unroll
      for (int i = 0; i < M; ++i) { x[i] = as[buf][k][tile_index<T>(ty, i)]; y[i] = bs[buf][k][tile_index<T>(tx, i)]; }
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int j = 0; j < M; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
    }
    if (more) {
      a.put(as[buf ^ 1]);
      b.put(bs[buf ^ 1]);
      __syncthreads();
    }
  }
}

template <int T, bool KN, bool WIDE>
__global__ void __launch_bounds__(256, T == 128 ? 2 : 4)
ragged_rows_kernel(const RaggedRows a) {
  constexpr int M = T / 16;
  __shared__ RaggedSpans sp;
  if (threadIdx.x < 32) load_spans(sp, a.offsets, a.E, (int)a.R, T);
  __syncthreads();
  const int tile = blockIdx.x;
  if (tile >= sp.tile0[a.E + 2]) return;
  const int span = span_of(sp, a.E, tile);
  const int r0 = sp.row0[span] + (tile - sp.tile0[span]) * T, rend = sp.row0[span + 1];
  const int n0 = blockIdx.y * T;
  float* out = static_cast<float*>(a.out);
  const int e = span - 1;
  const bool owned = e >= 0 && e < a.E;
  float acc[M][M] = {};
  if (owned) {
    const float* x = static_cast<const float*>(a.x) + (int64_t)r0 * a.K;
    const float* w = static_cast<const float*>(a.w) + (int64_t)e * a.N * a.K;
    tile_product<T, true, !KN, WIDE>(x, a.K, rend - r0, KN ? w + n0 : w + (int64_t)n0 * a.K, KN ? a.N : a.K, a.N - n0,
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
      if (n < a.N) out[(int64_t)r * a.N + n] = acc[i][j];
    }
  }
}

template <int T, bool WIDE>
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
    tile_product<T, false, false, WIDE>(static_cast<const float*>(a.a) + (int64_t)r0 * a.P + p0, a.P, a.P - p0,
                                            static_cast<const float*>(a.b) + (int64_t)r0 * a.Q + q0, a.Q, a.Q - q0, rows, acc);
  float* out = static_cast<float*>(a.out) + (int64_t)e * a.P * a.Q;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const int p = p0 + tile_index<T>(ty, i), q = q0 + tile_index<T>(tx, j);
      if (p < a.P && q < a.Q) out[(int64_t)p * a.Q + q] = acc[i][j];
    }
}

// rows that start on 16 bytes
static bool wide_rows(const void* p, int64_t ld) { return ld % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <bool KN>
static int launch_rows(const RaggedRows& a, cudaStream_t st) {
  const bool wide = wide_rows(a.x, a.K) && wide_rows(a.w, KN ? a.N : a.K);
  // 128-row tiles once experts have about as many rows on average: half a tile per expert is idle
  const bool large = a.R >= 128ll * a.E && a.N > 64;
  auto grid = [&](int T) {
    return dim3((unsigned)(a.R / T + a.E + 2), (unsigned)((a.N + T - 1) / T));     // every span may end in a partial tile
  };
  if (large && wide) ragged_rows_kernel<128, KN, true><<<grid(128), 256, 0, st>>>(a);
  else if (large) ragged_rows_kernel<128, KN, false><<<grid(128), 256, 0, st>>>(a);
  else if (wide) ragged_rows_kernel<64, KN, true><<<grid(64), 256, 0, st>>>(a);
  else ragged_rows_kernel<64, KN, false><<<grid(64), 256, 0, st>>>(a);
  MOLE_LAUNCH_OK();
  return MOLE_OK;
}

int ragged_rows_simt(const RaggedRows& a, cudaStream_t st) {
  return a.kn ? launch_rows<true>(a, st) : launch_rows<false>(a, st);
}
int ragged_wgrad_simt(const RaggedWgrad& a, cudaStream_t st) {
  const bool wide = wide_rows(a.a, a.P) && wide_rows(a.b, a.Q);
  // 128 x 128 tiles where they fill the SMs
  auto grid = [&](int T) { return dim3((unsigned)((a.Q + T - 1) / T), (unsigned)((a.P + T - 1) / T), (unsigned)a.E); };
  const dim3 g = grid(128);
  const bool large = (int64_t)g.x * g.y * g.z >= 2 * sm_count();
  if (large && wide) ragged_wgrad_kernel<128, true><<<g, 256, 0, st>>>(a);
  else if (large) ragged_wgrad_kernel<128, false><<<g, 256, 0, st>>>(a);
  else if (wide) ragged_wgrad_kernel<64, true><<<grid(64), 256, 0, st>>>(a);
  else ragged_wgrad_kernel<64, false><<<grid(64), 256, 0, st>>>(a);
  MOLE_LAUNCH_OK();
  return MOLE_OK;
}

}  // namespace mole

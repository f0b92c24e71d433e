// fp32 products over rows packed by expert, on the CUDA cores: operands of 24 bits, which one term of bf16
// does not hold (three would; products of split operands on the tensor cores are not tried here).  Every size
// and alignment.
//
// A thread block takes a tile of T x T outputs, a thread 16 x 8 of them in registers (4 x 4 for T = 64);
// tiles of both operands, 16 deep in the reduction, go through shared memory, the next ones on their way
// in registers meanwhile.  Rows come in pairs on the packed multiply-add, the column's value twice in
// a pair of registers: 64 instructions per step on six 16-byte reads, which shared memory serves in 24
// cycles a warp, the multiply-adds in 32 (of four warps at a time).  With 8 x 8 it is 32 on four, both
// take the same time, and the kernel a tenth longer; with pairs along the reduction in 8 x 4 (no value
// twice, but six reads for 32) a fifth longer still.
// T = 64 where experts have few rows, and 16 rows for a tile that holds no more.  Sums run over the
// reduction in its order, one fused multiply-add after the other; where there are too few tiles for
// the SMs the reduction is cut into parts, joined in their order by a second kernel.  Bound by the
// fp32 pipes: 8192 rows over 8 experts of 512 x 2048 in 0.35 ms, dx in 0.37 and dw in 0.35 (46 to 49
// TFLOP/s; 56 where the tiles fill the SMs evenly, a library product of the same size 55).
#include "f32x2.cuh"
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

// Four neighbouring elements, those from `n` on as zeros
template <bool WIDE>
__device__ __forceinline__ void load4(const float* p, int n, float (&v)[4]) {
  if (WIDE && n >= 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}

// Tiles of T x T outputs: `kThreads` threads, kRows x kCols outputs each
template <int T>
struct Tile {
  static constexpr int kThreads = T == 128 ? 128 : 256;
  static constexpr int kRows = T == 128 ? 16 : 4, kCols = T * T / kThreads / kRows;
  static constexpr int kRowStep = kThreads / 16 * 4;       // rows of a thread come in fours, so far apart
  __device__ static __forceinline__ int row(int i) { return (i >> 2) * kRowStep + (threadIdx.x >> 4) * 4 + (i & 3); }
  __device__ static __forceinline__ int col(int j) { return (j >> 2) * 64 + (threadIdx.x & 15) * 4 + (j & 3); }
};

// One operand's tile: `mn` runs over T rows (or columns) of the output, k over the reduction.  KMAJOR:
// element (mn, k) at p + mn * ld + k, else at p + k * ld + mn.
template <int T, bool KMAJOR, bool WIDE>
struct Operand {
  static constexpr int kThreads = Tile<T>::kThreads;
  static constexpr int kPer = T * kSK / 4 / kThreads;      // pieces of four that a thread loads
  float v[kPer][4];
  __device__ __forceinline__ int mn_of(int h) const { return KMAJOR ? (threadIdx.x >> 2) + kThreads / 4 * h : threadIdx.x % (T / 4) * 4; }
  __device__ __forceinline__ int k_of(int h) const { return KMAJOR ? (threadIdx.x & 3) * 4 : threadIdx.x / (T / 4) + kThreads / (T / 4) * h; }
  // `mn_left`, `k_left`: what exists from this tile's first element on
  __device__ __forceinline__ void fetch(const float* p, int64_t ld, int mn_left, int k_left) {
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      const int mn = mn_of(h), k = k_of(h);
      if (KMAJOR) load4<WIDE>(p + (int64_t)mn * ld + k, mn < mn_left ? k_left - k : 0, v[h]);
      else load4<WIDE>(p + (int64_t)k * ld + mn, k < k_left ? mn_left - mn : 0, v[h]);
    }
  }
  __device__ __forceinline__ void put(float (&s)[kSK][T + 4]) const {
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      if (KMAJOR) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[k_of(h) + i][mn_of(h)] = v[h][i];
      } else {
        *reinterpret_cast<float4*>(&s[k_of(h)][mn_of(h)]) = make_float4(v[h][0], v[h][1], v[h][2], v[h][3]);
      }
    }
  }
};

// acc = A (T x K) B (K x T); pa and pb point to the tile's first elements at k = 0.  Output (i, j) of a
// thread is row Tile<T>::row(i), column Tile<T>::col(j) of the tile.
template <int T, bool A_K, bool B_K, bool WIDE>
__device__ __forceinline__ void tile_product(const float* pa, int64_t lda, int m_left, const float* pb, int64_t ldb,
                                             int n_left, int K, float (&acc)[Tile<T>::kRows][Tile<T>::kCols]) {
  constexpr int M = Tile<T>::kRows, N = Tile<T>::kCols;
  __shared__ __align__(16) float as[2][kSK][T + 4], bs[2][kSK][T + 4];
  uint64_t acc2[M / 2][N] = {};                            // of two neighbouring rows
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
      uint64_t x[M / 2];
      float y[N];
#pragma unroll
      for (int i = 0; i < M; i += 4) {
        const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(&as[buf][k][Tile<T>::row(i)]);
        x[i / 2] = t.x; x[i / 2 + 1] = t.y;
      }
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const float4 t = *reinterpret_cast<const float4*>(&bs[buf][k][Tile<T>::col(j)]);
        y[j] = t.x; y[j + 1] = t.y; y[j + 2] = t.z; y[j + 3] = t.w;
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint64_t yy = f2_dup(y[j]);
#pragma unroll
        for (int i = 0; i < M / 2; ++i) acc2[i][j] = f2_fma(x[i], yy, acc2[i][j]);
      }
    }
    if (more) {
      a.put(as[buf ^ 1]);
      b.put(bs[buf ^ 1]);
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < M / 2; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) f2_unpack(acc2[i][j], acc[2 * i][j], acc[2 * i + 1][j]);
}

// The same for a tile of at most 16 rows and 64 columns: four groups of 64 threads take a quarter of every
// 64 elements of the reduction each (so that nothing is multiplied for rows that are not there) and
// are added in their order.
template <bool A_K, bool B_K, bool WIDE>
__device__ __forceinline__ void few_rows_product(const float* pa, int64_t lda, int m_left, const float* pb, int64_t ldb,
                                                 int n_left, int K, float (&acc)[4][4]) {
  constexpr int D = 64;
  __shared__ __align__(16) float as[D][16 + 4], bs[D][64 + 4];
  const int t = threadIdx.x, g = t >> 6, ty = (t >> 4) & 3, tx = t & 15;
  static_assert(A_K, "rows are read along the reduction");
  for (int k0 = 0; k0 < K; k0 += D) {
    __syncthreads();
    {
      const int m = t >> 4, k = (t & 15) * 4;                     // 16 rows x 64, four each
#pragma unroll
      for (int i = 0; i < 4; ++i) as[k + i][m] = m < m_left && k0 + k + i < K ? pa[(int64_t)m * lda + k0 + k + i] : 0.f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {                                 // 64 x 64, twice eight each
      float v[8];
      if (B_K) {
        const int n = t & 63, k = (t >> 6) * 8 + 32 * h;
        load8<WIDE>(pb + (int64_t)n * ldb + k0 + k, n < n_left ? K - k0 - k : 0, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) bs[k + i][n] = v[i];
      } else {
        const int k = (t >> 3) + 32 * h, n = (t & 7) * 8;
        load8<WIDE>(pb + (int64_t)(k0 + k) * ldb + n, k0 + k < K ? n_left - n : 0, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) bs[k][n + i] = v[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[i] = as[16 * g + k][4 * ty + i]; y[i] = bs[16 * g + k][4 * tx + i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
    }
  }
  __syncthreads();
  float (*sums)[16][64 + 4] = reinterpret_cast<float (*)[16][64 + 4]>(&bs[0][0]);       // [4], as large as bs
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[g][4 * ty + i][4 * tx + j] = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[i][j] = 0.f;
      if (g == 0)
        for (int q = 0; q < 4; ++q) acc[i][j] += sums[q][4 * ty + i][4 * tx + j];
    }
}

// Four neighbouring columns of a row; `left` of them exist.  `vec`: rows of out start on 16 bytes.
__device__ __forceinline__ void put4(float* d, const float* v, int left, bool vec) {
  if (vec && left >= 4) {
    *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) d[j] = v[j];
  }
}

// The tile's outputs; `m_left`, `n_left` of its rows and columns exist
template <int T>
__device__ __forceinline__ void put_tile(float* out, int64_t ld, int m_left, int n_left,
                                         const float (&acc)[Tile<T>::kRows][Tile<T>::kCols], bool vec) {
#pragma unroll
  for (int i = 0; i < Tile<T>::kRows; ++i) {
    const int r = Tile<T>::row(i);
    if (r >= m_left) continue;
#pragma unroll
    for (int j = 0; j < Tile<T>::kCols; j += 4) put4(out + r * ld + Tile<T>::col(j), &acc[i][j], n_left - Tile<T>::col(j), vec);
  }
}

template <int T, bool KN, bool WIDE>
__global__ void __launch_bounds__(Tile<T>::kThreads, T == 128 ? 2 : 4)
ragged_rows_kernel(const RaggedRows a) {
  __shared__ RaggedSpans sp;
  after_previous();
  if (threadIdx.x < 32) load_spans(sp, a.offsets, a.E, (int)a.R, T == 128 ? 7 : 6);
  __syncthreads();
  const int tile = blockIdx.x;
  if (tile >= sp.tile0[a.E + 2]) return;
  const int span = span_of(sp, a.E, tile);
  const int r0 = sp.row0[span] + (tile - sp.tile0[span]) * T, rend = sp.row0[span + 1];
  const int n0 = blockIdx.y * T;
  // part z of the reduction
  const int share = (a.K + a.split * kSK - 1) / (a.split * kSK) * kSK;
  const int k0 = blockIdx.z * share, len = min(a.K - k0, share);          // len <= 0: nothing left for this part
  float* out = a.split > 1 ? a.part + (int64_t)blockIdx.z * a.R * a.N : static_cast<float*>(a.out);
  const bool vec = a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const int e = span - 1;
  const bool owned = e >= 0 && e < a.E;
  float acc[Tile<T>::kRows][Tile<T>::kCols] = {};
  if (owned) {
    const float* x = static_cast<const float*>(a.x) + (int64_t)r0 * a.K + k0;
    const float* w = static_cast<const float*>(a.w) + (int64_t)e * a.N * a.K + (KN ? (int64_t)k0 * a.N : (int64_t)k0);
    const float* wt = KN ? w + n0 : w + (int64_t)n0 * a.K;
    const int64_t ldw = KN ? a.N : a.K;
    if constexpr (T == 64) {
      if (rend - r0 <= 16) {
        few_rows_product<true, !KN, WIDE>(x, a.K, rend - r0, wt, ldw, a.N - n0, len, acc);
        const int t = threadIdx.x, ty = (t >> 4) & 3, tx = t & 15;
        if (t < 64)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (r0 + 4 * ty + i < rend)
              put4(out + (int64_t)(r0 + 4 * ty + i) * a.N + n0 + 4 * tx, acc[i], a.N - n0 - 4 * tx, vec);
        return;
      }
    }
    if (len > 0) tile_product<T, true, !KN, WIDE>(x, a.K, rend - r0, wt, ldw, a.N - n0, len, acc);
  }
  put_tile<T>(out + (int64_t)r0 * a.N + n0, a.N, rend - r0, a.N - n0, acc, vec);
}

// Rows of one expert, by a whole block: the running maximum over the offsets before it only where they do
// not rise by themselves
__device__ __forceinline__ void expert_rows(const int32_t* offsets, int E, int R, int e, int& first, int& end) {
  auto at = [&](int i) { return min(max(offsets[i], 0), R); };
  first = at(e);
  end = at(e + 1);
  bool falls = false;
  for (int i = threadIdx.x; i < E; i += blockDim.x) falls |= offsets[i + 1] < offsets[i];
  if (__syncthreads_or(falls)) {
    for (int i = 0; i < e; ++i) first = max(first, at(i));
    end = max(first, end);
  }
}

template <int T, bool WIDE>
__global__ void __launch_bounds__(Tile<T>::kThreads, T == 128 ? 2 : 4)
ragged_wgrad_kernel(const RaggedWgrad a) {
  const int e = blockIdx.z / a.split, part = blockIdx.z % a.split, q0 = blockIdx.x * T, p0 = blockIdx.y * T;
  after_previous();
  int first, end;
  expert_rows(a.offsets, a.E, (int)a.R, e, first, end);
  const int all = end - first;
  const int share = (all + a.split * kSK - 1) / (a.split * kSK) * kSK;    // of an expert's rows per part
  const int r0 = first + part * share, rows = min(share, all - part * share);
  float acc[Tile<T>::kRows][Tile<T>::kCols] = {};
  if (rows > 0)
    tile_product<T, false, false, WIDE>(static_cast<const float*>(a.a) + (int64_t)r0 * a.P + p0, a.P, a.P - p0,
                                            static_cast<const float*>(a.b) + (int64_t)r0 * a.Q + q0, a.Q, a.Q - q0, rows, acc);
  float* out = (a.split > 1 ? a.part + (int64_t)part * a.E * a.P * a.Q : static_cast<float*>(a.out)) + (int64_t)e * a.P * a.Q;
  const bool vec = a.Q % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  put_tile<T>(out + (int64_t)p0 * a.Q + q0, a.Q, a.P - p0, a.Q - q0, acc, vec);
}

// rows that start on 16 bytes
static bool wide_rows(const void* p, int64_t ld) { return ld % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// 128-row tiles once experts have about as many rows on average: half a tile per expert is idle
static int rows_tile(const RaggedRows& a) { return a.R >= 128ll * a.E && a.N > 64 ? 128 : 64; }
// Into how many parts to cut the reduction: the number that costs least, by this account.  `slots` tiles run
// at a time, and together they do `rate` operations a second, so cutting pays where the tiles fill the
// last round (or the only one) badly; partial results are written and read once, at 5 TB/s.
static int parts_for(int64_t tiles, int tile, int64_t reduction, int64_t outputs, int slots, double rate) {
  if (tiles < 1) return 1;
  const double whole = 2.0 * tile * tile * (double)reduction / (rate / slots);        // one tile's time
  int best = 1;
  double least = (double)((tiles + slots - 1) / slots) * whole;
  for (int s = 2; s <= 32 && reduction / s >= 128; ++s) {
    const double t = (double)((tiles * s + slots - 1) / slots) * whole / s + s * (double)outputs * 8 / 5e12 + 3e-6;
    if (t < 0.95 * least) { least = t; best = s; }
  }
  return best;
}
int ragged_rows_simt_split(const RaggedRows& a) {
  const int T = rows_tile(a);
  const int64_t live = a.E < a.R ? a.E : a.R;
  const int64_t tiles = (a.R / T + (live + 1) / 2) * ((a.N + T - 1) / T);     // (half of the experts end in a tile of their own)
  return parts_for(tiles, T, a.K, a.R * a.N, sm_count() * (T == 128 ? 2 : 4), 4e13);
}
static int64_t wgrad_tiles(const RaggedWgrad& a, int T) {
  return (int64_t)a.E * ((a.P + T - 1) / T) * ((a.Q + T - 1) / T);
}
static int wgrad_tile(const RaggedWgrad& a) { return wgrad_tiles(a, 128) >= sm_count() ? 128 : 64; }
int ragged_wgrad_split(bool tensor, const RaggedWgrad& a) {
  const int T = tensor ? 256 : wgrad_tile(a);          // on the tensor cores a pair of SMs per tile
  const int slots = tensor ? sm_count() / 2 : sm_count() * (T == 128 ? 2 : 4);
  return parts_for(wgrad_tiles(a, T), T, a.R / a.E, (int64_t)a.E * a.P * a.Q, slots, tensor ? 1e15 : 4e13);
}

// out[i] = part[0][i] + part[1][i] + ...
template <typename TO>
__global__ void __launch_bounds__(256) join_kernel(const float* part, int split, int64_t n, TO* __restrict__ out) {
  after_previous();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float v = part[i];
    for (int s = 1; s < split; ++s) v += part[(int64_t)s * n + i];
    out[i] = Elem<TO>::from_f(v);
  }
}
int ragged_join(int out_dtype, const float* part, int split, int64_t n, void* out, cudaStream_t st) {
  int64_t blocks = (n + 255) / 256;
  if (blocks > (int64_t)sm_count() * 8) blocks = (int64_t)sm_count() * 8;
  const dim3 grid((unsigned)blocks);
  if (out_dtype == MOLE_F32) return launch_early(join_kernel<float>, grid, 256, 0, st, part, split, n, static_cast<float*>(out));
  return launch_early(join_kernel<__nv_bfloat16>, grid, 256, 0, st, part, split, n, static_cast<__nv_bfloat16*>(out));
}

template <bool KN>
static int launch_rows(const RaggedRows& a, cudaStream_t st) {
  const bool wide = wide_rows(a.x, a.K) && wide_rows(a.w, KN ? a.N : a.K);
  const bool large = rows_tile(a) == 128;
  auto grid = [&](int T) {                                                   // every span may end in a partial tile
    return dim3((unsigned)(a.R / T + a.E + 2), (unsigned)((a.N + T - 1) / T), (unsigned)a.split);
  };
  if (large) return launch_early(wide ? ragged_rows_kernel<128, KN, true> : ragged_rows_kernel<128, KN, false>, grid(128),
                                 Tile<128>::kThreads, 0, st, a);
  return launch_early(wide ? ragged_rows_kernel<64, KN, true> : ragged_rows_kernel<64, KN, false>, grid(64),
                      Tile<64>::kThreads, 0, st, a);
}

int ragged_rows_simt(const RaggedRows& a, cudaStream_t st) {
  if (int rc = a.kn ? launch_rows<true>(a, st) : launch_rows<false>(a, st)) return rc;
  return a.split > 1 ? ragged_join(MOLE_F32, a.part, a.split, a.R * a.N, a.out, st) : MOLE_OK;
}
int ragged_wgrad_simt(const RaggedWgrad& a, cudaStream_t st) {
  const bool wide = wide_rows(a.a, a.P) && wide_rows(a.b, a.Q);
  auto grid = [&](int T) { return dim3((unsigned)((a.Q + T - 1) / T), (unsigned)((a.P + T - 1) / T), (unsigned)(a.E * a.split)); };
  const bool large = wgrad_tile(a) == 128;
  if (int rc = large ? launch_early(wide ? ragged_wgrad_kernel<128, true> : ragged_wgrad_kernel<128, false>, grid(128),
                                    Tile<128>::kThreads, 0, st, a)
                     : launch_early(wide ? ragged_wgrad_kernel<64, true> : ragged_wgrad_kernel<64, false>, grid(64),
                                    Tile<64>::kThreads, 0, st, a))
    return rc;
  return a.split > 1 ? ragged_join(MOLE_F32, a.part, a.split, (int64_t)a.E * a.P * a.Q, a.out, st) : MOLE_OK;
}

}  // namespace mole

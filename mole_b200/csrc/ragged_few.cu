// Products over few rows packed by expert (up to 16 in all: decode steps), every type and layout.
//
// With that few rows a product is a reading of the weights of the experts that have rows: 2 N K
// bytes of bf16 per expert, a row's worth of multiply-adds on each, which the CUDA cores keep up with for
// up to four rows of an expert; every four more read its weights once more.
// What counts is loads in flight.  The tensor-core kernel gives a decode step one pair of SMs per
// 256 features (64 pairs at best, and a pipeline to fill); here every warp of every SM streams weights:
// one token with two of 64 experts of 2048 x 8192 takes 15 us (67 MB at 4.5 TB/s), there 22.
//
// K-major weights (few_nk): a warp takes four features, its lanes run along the reduction with 16-byte
// loads; up to eight warps share the reduction of the same features when there are few of them.
// N-major weights (few_kn): a lane takes neighbouring features, warps and the eight thread blocks of a
// cluster share the reduction; partial sums meet in shared memory, then across the cluster.  All
// sums are joined in a fixed order.
#include <type_traits>

#include "ragged.cuh"

namespace mole {

constexpr int kFewWarps = 8;
constexpr int kFewChunk = 4;       // rows that share one pass over the weights

template <typename T> struct FewIn;
template <> struct FewIn<float> {
  using Acc = float;
  static constexpr int V = 4;
  __device__ static __forceinline__ float get(float v) { return v; }
};
template <> struct FewIn<__nv_bfloat16> {
  using Acc = float;
  static constexpr int V = 8;
  __device__ static __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <> struct FewIn<int8_t> {
  using Acc = int;
  static constexpr int V = 16;
  __device__ static __forceinline__ int get(int8_t v) { return v; }
};

__device__ __forceinline__ uint4 load_stream(const void* p) {      // weights: read once, not kept in L1
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// acc += sum over 16 bytes of a and of b
__device__ __forceinline__ void dot16(float& acc, const uint4& a, const uint4& b, const float*) {
  const float* x = reinterpret_cast<const float*>(&a);
  const float* y = reinterpret_cast<const float*>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = fmaf(x[i], y[i], acc);
}
__device__ __forceinline__ void dot16(float& acc, const uint4& a, const uint4& b, const __nv_bfloat16*) {
  const uint32_t* x = reinterpret_cast<const uint32_t*>(&a);
  const uint32_t* y = reinterpret_cast<const uint32_t*>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), acc);
    acc = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), acc);
  }
}
__device__ __forceinline__ void dot16(int& acc, const uint4& a, const uint4& b, const int8_t*) {
  const int* x = reinterpret_cast<const int*>(&a);
  const int* y = reinterpret_cast<const int*>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __dp4a(x[i], y[i], acc);
}

// Offsets (clamped as everywhere) in shared memory and the `which`-th expert that has rows; -1: there are
// not that many.  By the whole block of 256 threads: a decode step waits for this before its first
// weight, so every thread looks at one expert, and the running maximum is taken only where the
// offsets do not rise by themselves.
struct FewSpans {
  int o[kMaxRaggedExperts + 1];
  int live[kFewWarps];
  int e;
};
static_assert(kMaxRaggedExperts == 32 * kFewWarps, "one thread per expert");
__device__ __forceinline__ int find_expert(FewSpans& s, const RaggedRows& a, int which) {
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, R = (int)a.R;
  auto clamped = [&](int i) { return a.offsets ? min(max(a.offsets[i], 0), R) : (i == 0 ? 0 : R); };
  if (t <= a.E) s.o[t] = clamped(t);
  if (t == 0 && a.E == kMaxRaggedExperts) s.o[a.E] = clamped(a.E);
  if (t == 0) s.e = -1;
  __syncthreads();
  if (__syncthreads_or(t < a.E && s.o[t + 1] < s.o[t])) {
    if (t == 0)
      for (int i = 1; i <= a.E; ++i) s.o[i] = max(s.o[i], s.o[i - 1]);
    __syncthreads();
  }
  const bool live = t < a.E && s.o[t + 1] > s.o[t];
  const unsigned mask = __ballot_sync(0xffffffffu, live);
  if (lane == 0) s.live[warp] = __popc(mask);
  __syncthreads();
  if (live) {
    int rank = __popc(mask & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) rank += s.live[w];
    if (rank == which) s.e = t;
  }
  __syncthreads();
  return s.e;
}

// Zeros into features [f0, f1) of the rows that belong to nobody
template <typename TO>
__device__ __forceinline__ void zero_nobody(const FewSpans& s, const RaggedRows& a, int f0, int f1) {
  f1 = min(f1, a.N);
  TO* out = static_cast<TO*>(a.out);
  for (int r = 0; r < (int)a.R; ++r) {
    if (r >= s.o[0] && r < s.o[a.E]) continue;
    for (int f = f0 + threadIdx.x; f < f1; f += blockDim.x) out[(int64_t)r * a.N + f] = Elem<TO>::from_f(0.f);
  }
}
template <typename TO, typename Acc>
__device__ __forceinline__ void put(const RaggedRows& a, int e, int r, int f, Acc acc) {
  float v = (float)acc;
  if (a.w_scale != nullptr) v = __fmul_rn(__fmul_rn(v, a.x_scale[r]), a.w_scale[(int64_t)e * a.N + f]);
  static_cast<TO*>(a.out)[(int64_t)r * a.N + f] = Elem<TO>::from_f(v);
}

// grid (feature groups, experts with rows); `split` warps share the reduction of four features.
// WIDE: 16-byte loads along the reduction.
template <typename T, typename TO, bool WIDE>
__global__ void __launch_bounds__(32 * kFewWarps, 4)
few_nk_kernel(const RaggedRows a, const int split) {
  using Acc = typename FewIn<T>::Acc;
  constexpr int V = WIDE ? FewIn<T>::V : 1;
  __shared__ FewSpans sp;
  __shared__ Acc part[kFewWarps][4 * kFewChunk];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  after_previous();
  const int e = find_expert(sp, a, blockIdx.y);
  const int groups = kFewWarps / split;
  const int fb = blockIdx.x * groups * 4;
  if (blockIdx.y == 0) zero_nobody<TO>(sp, a, fb, fb + groups * 4);
  if (e < 0) return;
  const int f0 = fb + (warp / split) * 4, p = warp % split;
  const T* w = static_cast<const T*>(a.w) + ((int64_t)e * a.N + f0) * a.K;
  const int nf = min(4, a.N - f0);                   // may be <= 0: the warp only takes part in the joins
  for (int r0 = sp.o[e]; r0 < sp.o[e + 1]; r0 += kFewChunk) {
    const int nr = min(kFewChunk, sp.o[e + 1] - r0);
    const T* x = static_cast<const T*>(a.x) + (int64_t)r0 * a.K;
    Acc acc[4][kFewChunk] = {};
    auto pass = [&](auto rows) {
      constexpr int C = decltype(rows)::value;
#pragma unroll (C > 2 ? 1 : 2)
      for (int k = (p * 32 + lane) * V; k < a.K; k += split * 32 * V) {
        if constexpr (WIDE) {
          uint4 wv[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) wv[i] = i < nf ? load_stream(w + (int64_t)i * a.K + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < C; ++j) {
            const uint4 xv = *reinterpret_cast<const uint4*>(x + (int64_t)min(j, nr - 1) * a.K + k);
#pragma unroll
            for (int i = 0; i < 4; ++i) dot16(acc[i][j], wv[i], xv, static_cast<const T*>(nullptr));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const Acc wv = i < nf ? FewIn<T>::get(w[(int64_t)i * a.K + k]) : Acc(0);
#pragma unroll
            for (int j = 0; j < C; ++j) acc[i][j] += wv * FewIn<T>::get(x[(int64_t)min(j, nr - 1) * a.K + k]);
          }
        }
      }
    };
    if (nr == 1) pass(std::integral_constant<int, 1>());
    else if (nr == 2) pass(std::integral_constant<int, 2>());
    else pass(std::integral_constant<int, 4>());
    // 16 sums over the lanes; lane 4 i + j ends up with feature i, row j
    Acc mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kFewChunk; ++j) {
        if (j >= nr) continue;
        Acc v = acc[i][j];
#pragma unroll
        for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == 4 * i + j) mine = v;
      }
    if (split > 1) {
      if (lane < 16) part[warp][lane] = mine;
      __syncthreads();
      if (p == 0 && lane < 16)
        for (int q = 1; q < split; ++q) mine += part[warp + q][lane];
      __syncthreads();
    }
    if (p == 0 && lane < 16 && (lane >> 2) < nf && (lane & 3) < nr) put<TO>(a, e, r0 + (lane & 3), f0 + (lane >> 2), mine);
  }
}

// grid (8 x feature tiles, experts with rows), clusters of 8 along the first: thread block q of a
// cluster takes the q-th eighth of the reduction, its warps an eighth of that each.  A lane owns V features.
constexpr int kFewCluster = 8;
template <typename T, int V>
__global__ void __cluster_dims__(kFewCluster, 1, 1) __launch_bounds__(32 * kFewWarps)
few_kn_kernel(const RaggedRows a) {
  constexpr int TILE = 32 * V;
  __shared__ FewSpans sp;
  __shared__ float part[kFewWarps][kFewChunk][TILE];
  __shared__ float sum[kFewChunk][TILE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  after_previous();
  const int e = find_expert(sp, a, blockIdx.y);
  const int q = blockIdx.x % kFewCluster, fb = blockIdx.x / kFewCluster * TILE;
  if (blockIdx.y == 0 && q == 0) zero_nobody<T>(sp, a, fb, fb + TILE);
  if (e < 0) return;                                 // the whole cluster
  const int f0 = fb + lane * V;
  const int share = (a.K + kFewCluster * kFewWarps - 1) / (kFewCluster * kFewWarps);
  const int k0 = min(a.K, (q * kFewWarps + warp) * share), k1 = min(a.K, k0 + share);
  const T* w = static_cast<const T*>(a.w) + (int64_t)e * a.K * a.N + f0;
  for (int r0 = sp.o[e]; r0 < sp.o[e + 1]; r0 += kFewChunk) {
    const int nr = min(kFewChunk, sp.o[e + 1] - r0);
    const T* x = static_cast<const T*>(a.x) + (int64_t)r0 * a.K;
    float acc[kFewChunk][V] = {};
    if (f0 < a.N) {                                  // V > 1 only where N is a multiple of V
#pragma unroll 8
      for (int k = k0; k < k1; ++k) {
        float wv[V];
        if constexpr (V == 1) {
          wv[0] = FewIn<T>::get(w[(int64_t)k * a.N]);
        } else if constexpr (sizeof(T) == 4) {
          const uint4 t = load_stream(w + (int64_t)k * a.N);
          wv[0] = __uint_as_float(t.x); wv[1] = __uint_as_float(t.y); wv[2] = __uint_as_float(t.z); wv[3] = __uint_as_float(t.w);
        } else {
          const uint2 t = *reinterpret_cast<const uint2*>(w + (int64_t)k * a.N);
          wv[0] = __uint_as_float(t.x << 16); wv[1] = __uint_as_float(t.x & 0xffff0000u);
          wv[2] = __uint_as_float(t.y << 16); wv[3] = __uint_as_float(t.y & 0xffff0000u);
        }
#pragma unroll
        for (int j = 0; j < kFewChunk; ++j) {
          if (j >= nr) break;
          const float xv = FewIn<T>::get(x[(int64_t)j * a.K + k]);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[j][i] = fmaf(xv, wv[i], acc[j][i]);
        }
      }
    }
    for (int j = 0; j < nr; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) part[warp][j][lane * V + i] = acc[j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < nr * TILE; i += 32 * kFewWarps) {
      float v = 0.f;
#pragma unroll
      for (int u = 0; u < kFewWarps; ++u) v += part[u][i / TILE][i % TILE];
      sum[i / TILE][i % TILE] = v;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    // an eighth of the tile's sums each, over the cluster's thread blocks in their order
    for (int i = q * (kFewChunk * TILE / kFewCluster) + threadIdx.x; i < (q + 1) * (kFewChunk * TILE / kFewCluster);
         i += 32 * kFewWarps) {
      const int j = i / TILE, f = i % TILE;
      if (j >= nr || fb + f >= a.N) continue;
      const uint32_t local = static_cast<uint32_t>(__cvta_generic_to_shared(&sum[j][f]));
      float v = 0.f;
#pragma unroll
      for (int u = 0; u < kFewCluster; ++u) {
        uint32_t addr;
        float t;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(local), "r"(u));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(t) : "r"(addr) : "memory");
        v += t;
      }
      put<T>(a, e, r0 + j, fb + f, v);
    }
    // nobody's sums are overwritten, and nobody leaves, while another block may read them
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// By all rows together: the host does not know how they fall to the experts.  Measured against the forms
// for more rows (tensor cores, for fp32 the tiles), in us, three sets of weights in turn; 17 rows take those:
//   rows                                1         4         8        16       17
//   bf16, 64 experts of 2048 x 2048   5.3/16   9.8/17    15/18    27/32      31
//   bf16, the same N-major            8.0/16    16/17    32/17    63/32      31
//   8 bits, 64 of 2048 x 2048         4.1/11   6.4/11   8.6/12    15/20      20
//   fp32, 64 of 2048 x 2048           6.6/83   15/81     27/117   47/191    174
//   bf16, one expert of 8192 x 8192    27/46    39/46    74/46   142/46      46
//   bf16, the same N-major             54/46    66/46   129/46   257/46      46
//   8 bits, one of 8192 x 8192         13/25    16/25    28/25    52/25      25
//   fp32, one of 8192 x 8192          45/155   49/156   95/158  192/162     251
//   fp32, the same N-major            69/119    82/120  162/122   323/126     230
// So the rule is right where rows fall to many experts, but for bf16 and N-major weights from five rows on;
// for one expert it is right up to four rows (not for bf16 and N-major weights) and wrong from eight on (fp32
// and K-major weights: from sixteen).
bool ragged_rows_few_takes(const RaggedRows& a) { return a.R <= 16; }

template <typename T, typename TO>
static int launch_few(const RaggedRows& a, cudaStream_t st) {
  const unsigned experts = (unsigned)(a.E < a.R ? a.E : a.R);      // with rows, at most
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w);
  if constexpr (sizeof(T) > 1) {
    if (a.kn) {
      const bool wide = a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.w) & (4 * sizeof(T) - 1)) == 0;
      const int tile = 32 * (wide ? 4 : 1);
      const dim3 grid((unsigned)((a.N + tile - 1) / tile * kFewCluster), experts);
      return launch_early(wide ? few_kn_kernel<T, 4> : few_kn_kernel<T, 1>, grid, 32 * kFewWarps, 0, st, a);
    }
  }
  const bool wide = (size_t)a.K * sizeof(T) % 16 == 0 && (bases & 15) == 0;
  // warps for about 24 per SM, as long as each has a few loads to make
  int split = 1;
  while (split < kFewWarps && (int64_t)experts * a.N / 4 * split < (int64_t)sm_count() * 24 &&
         a.K >= 2 * split * 32 * (wide ? FewIn<T>::V : 1))
    split *= 2;
  const int per = kFewWarps / split * 4;
  const dim3 grid((unsigned)((a.N + per - 1) / per), experts);
  return launch_early(wide ? few_nk_kernel<T, TO, true> : few_nk_kernel<T, TO, false>, grid, 32 * kFewWarps, 0, st, a, split);
}

int ragged_rows_few(int dtype, const RaggedRows& a, cudaStream_t st) {
  return dtype == MOLE_F32 ? launch_few<float, float>(a, st) : launch_few<__nv_bfloat16, __nv_bfloat16>(a, st);
}
int ragged_rows_few_i8(int out_dtype, const RaggedRows& a, cudaStream_t st) {
  return out_dtype == MOLE_F32 ? launch_few<int8_t, float>(a, st) : launch_few<int8_t, __nv_bfloat16>(a, st);
}

}  // namespace mole

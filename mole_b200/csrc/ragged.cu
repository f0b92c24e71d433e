// C entries of the products over rows packed by expert, and the quantisation of rows to 8-bit
// integers that the integer product takes.
#include <cstring>

#include "ragged.cuh"

namespace mole {

// ---- rows to 8-bit integers ------------------------------------------------------------------
// scale = max |x| / 127 rounded to fp32; q = the integer nearest to x / scale, ties to even.  The
// quotient t is taken as x * (1 / scale), which is off by less than 2^-23 of 127; where that leaves
// doubt about the nearest integer (1 value in 10^4), the sign of x - (n + 1/2) scale decides, which
// one fused multiply-add gives exactly.  (A call: inlined 64 times, the kernel misses in the instruction
// cache.)  Bound by instructions, not by HBM's 3 bytes an element: 32768 x 2048 of bf16 in 47 us (4.3 TB/s;
// half as much again with a division each).
__device__ __noinline__ int quantize_one(float x, float scale, float inv) {
  const float t = x * inv;
  float r = rintf(t);
  if (fabsf(fabsf(t - r) - 0.5f) < 6e-5f) {
    const float half = floorf(t) + 0.5f;
    const float d = fmaf(-half, scale, x);
    r = d > 0.f ? half + 0.5f : d < 0.f ? half - 0.5f : rintf(half);
  }
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}

// One row per group of G threads (a warp or a block).  HELD: the row fits the group's registers (eight
// 16-byte vectors a thread), is read once and waits there for its scale; otherwise it is read twice.
// V = 1: rows that 16-byte loads cannot address.  Four blocks an SM (64 registers): 32768 x 2048 in 47 us; with
// three, as many as registers allow unasked, 53; with five, which spill, 52.
template <typename T, int V, int G, bool HELD>
__global__ void __launch_bounds__(256, HELD ? 4 : 1)
quantize_rows_kernel(const T* x, int64_t R, int K, int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int kHeld = 8;
  __shared__ uint32_t tops[8];
  after_previous();
  const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (row >= R) return;                                      // a whole warp, or the whole block
  const int t = threadIdx.x % G;
  const T* xr = x + row * K;
  auto load = [&](int k, float (&v)[V]) {
    if constexpr (V > 1) Vec16<T>::load(xr + k, v);
    else v[0] = Elem<T>::to_f(xr[k]);
  };
  uint4 held[kHeld];
  uint32_t top = 0;                                          // of the magnitudes' bits: NaN above infinity above all
  auto see = [&](const float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  };
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int k = (j * G + t) * V;
      held[j] = k < K ? *reinterpret_cast<const uint4*>(xr + k) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      float v[V];
      Vec16<T>::load(reinterpret_cast<const T*>(&held[j]), v);
      see(v);
    }
  } else {
    for (int k = t * V; k < K; k += G * V) {
      float v[V];
      load(k, v);
      see(v);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < G / 32; ++w) top = max(top, tops[w]);
  }
  const float s = __fdiv_rn(__uint_as_float(top), 127.f);
  if (t == 0) scale[row] = s;
  const bool zero = !(s > 0.f && s < __int_as_float(0x7f800000));    // all zero, or not finite: the scale says it
  // rows of tiny values: both sides times 2^100, so that neither 1 / scale overflows nor the
  // difference in quantize_one leaves the range of fp32
  const float up = s < 0x1p-100f ? 0x1p100f : 1.f;
  const bool odd = zero || s < 0x1p-100f;
  const float su = s * up, inv = zero ? 0.f : __fdiv_rn(1.f, su);
  auto store = [&](int k, const float (&v)[V]) {
    uint32_t w[V];
    float off[V], doubt = 0.f;
    // the nearest integer sits in the low bits of t + 3 2^22 (|t| rounds to 127 at most); a quotient in
    // doubt is nearly half a unit off it.  bf16 rows are full of true ties (both x and the top have 8 bits):
    // one element in some hundred, looked at one by one.
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float t = v[i] * inv, r = t + 12582912.f;
      w[i] = __float_as_uint(r);
      off[i] = fabsf(t - (r - 12582912.f));
      doubt = fmaxf(doubt, off[i]);
    }
    if (doubt > 0.5f - 6e-5f || odd) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (off[i] > 0.5f - 6e-5f || odd) w[i] = zero ? 0u : (uint32_t)quantize_one(v[i] * up, su, inv);
    }
    int8_t* d = q + row * K + k;
    auto pack = [](uint32_t a, uint32_t b, uint32_t c, uint32_t e) {
      return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, e, 0x0040), 0x5410);
    };
    if constexpr (V == 8) *reinterpret_cast<uint2*>(d) = make_uint2(pack(w[0], w[1], w[2], w[3]), pack(w[4], w[5], w[6], w[7]));
    else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(d) = pack(w[0], w[1], w[2], w[3]);
    else *d = (int8_t)w[0];
  };
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int k = (j * G + t) * V;
      float v[V];
      Vec16<T>::load(reinterpret_cast<const T*>(&held[j]), v);
      if (k < K) store(k, v);
    }
  } else {
    for (int k = t * V; k < K; k += G * V) {
      float v[V];
      load(k, v);
      store(k, v);
    }
  }
}

template <typename T>
static int launch_quantize(const void* x, int64_t R, int K, void* q, float* scale, cudaStream_t st) {
  constexpr int V = Vec16<T>::N;
  const bool wide = K % V == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & (V - 1)) == 0;
  const T* xp = static_cast<const T*>(x);
  int8_t* qp = static_cast<int8_t*>(q);
  // a warp a row while rows are short and fill the SMs, else a block a row
  const bool block = K > 32 * V * 8 || R < (int64_t)sm_count() * 16;
  const unsigned grid = (unsigned)(block ? R : (R + 7) / 8);
  auto kern = wide && block && K <= 256 * V * 8 ? quantize_rows_kernel<T, V, 256, true>
              : wide && block                   ? quantize_rows_kernel<T, V, 256, false>
              : wide                            ? quantize_rows_kernel<T, V, 32, true>
              : block                           ? quantize_rows_kernel<T, 1, 256, false>
                                                : quantize_rows_kernel<T, 1, 32, false>;
  return launch_early(kern, dim3(grid), 256, 0, st, xp, R, K, qp, scale);
}

// ---- operands that the tensor cores cannot address, partial results ---------------------------
// TMA wants rows that start on 16 bytes.  Operands of other widths or at other addresses are copied to
// rows that do, in the caller's workspace; the copy costs a pass of HBM over the operand (weights:
// only those of experts that have rows), the products on the CUDA cores an order of magnitude.
// A thread makes 16 bytes of the copy from two aligned pieces.  Matrix m of `rows` rows belongs to expert
// m; a single matrix belongs to all.  (1237 rows of 13 experts, 1001 x 328: dx 105 -> 14 us, dw 83 -> 16.)
__global__ void __launch_bounds__(256)
align_rows_kernel(const uint8_t* src, int64_t rows, int row_bytes, int ld_bytes, uint8_t* dst, const int32_t* offsets) {
  after_previous();
  if (offsets != nullptr && offsets[blockIdx.y + 1] <= offsets[blockIdx.y]) return;
  const int per_row = ld_bytes / 16;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * per_row) return;
  const int64_t r = i / per_row;
  const int c = (int)(i - r * per_row) * 16;
  const int64_t matrix = rows * row_bytes;
  const uint8_t* first = src, *last = src + (int64_t)gridDim.y * matrix;         // what may be read
  const uint8_t* s = src + (int64_t)blockIdx.y * matrix + r * row_bytes + c;
  const uint8_t* at = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(s) & ~static_cast<uintptr_t>(15));
  uint32_t o[4];
  if (at >= first && at + 32 <= last) {
    // the two aligned pieces that hold the sixteen bytes, moved down by the distance in words and bytes
    const uint4 a = *reinterpret_cast<const uint4*>(at), b = *reinterpret_cast<const uint4*>(at + 16);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const int off = (int)(s - at);
    if (off & 8) {
#pragma unroll
      for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
    }
    if (off & 4) {
#pragma unroll
      for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = __funnelshift_r(w[j], w[j + 1], 8 * (off & 3));
    const int left = row_bytes - c;                  // bytes behind the row's end are zeros
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = left - 4 * j;
      if (n < 4) o[j] = n > 0 ? o[j] & ((1u << (8 * n)) - 1u) : 0u;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j] = 0;
      for (int k = 0; k < 4; ++k)
        if (c + 4 * j + k < row_bytes) o[j] |= (uint32_t)s[4 * j + k] << (8 * k);
    }
  }
  *reinterpret_cast<uint4*>(dst + ((int64_t)blockIdx.y * rows + r) * ld_bytes + c) = make_uint4(o[0], o[1], o[2], o[3]);
}

static bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
struct Aligner {            // deals out the workspace, or only counts
  uint8_t* at;
  int64_t left, used;
  bool count_only;
};
// *p: the operand, [matrices, rows, cols] elements of `elem` bytes; on return it and *ld can be addressed
static int align_operand(Aligner& ws, const void** p, int64_t matrices, int64_t rows, int cols, int elem, int* ld,
                         const int32_t* offsets, cudaStream_t st) {
  const int unit = 16 / elem;
  *ld = cols;
  if (cols % unit == 0 && aligned_to(*p, 16)) return MOLE_OK;
  *ld = (cols + unit - 1) / unit * unit;
  const int64_t bytes = (matrices * rows * *ld * elem + 255) / 256 * 256;
  ws.used += bytes;
  if (ws.count_only) return MOLE_OK;
  MOLE_REQUIRE(ws.at != nullptr && ws.used <= ws.left && aligned_to(ws.at, 16),
               "workspace of %lld bytes, %lld needed (mole_grouped_mm_workspace_bytes)", (long long)ws.left, (long long)ws.used);
  void* dst = ws.at + ws.used - bytes;
  const dim3 grid((unsigned)((rows * (*ld / unit) + 255) / 256), (unsigned)matrices);
  if (int rc = launch_early(align_rows_kernel, grid, 256, 0, st, static_cast<const uint8_t*>(*p), rows, cols * elem,
                            *ld * elem, static_cast<uint8_t*>(dst), offsets))
    return rc;
  *p = dst;
  return MOLE_OK;
}
// room for the partial results of a cut reduction
static int take_parts(Aligner& ws, int split, int64_t n, float** part) {
  if (split <= 1) return MOLE_OK;
  const int64_t bytes = ((int64_t)split * n * 4 + 255) / 256 * 256;
  ws.used += bytes;
  if (ws.count_only) return MOLE_OK;
  MOLE_REQUIRE(ws.at != nullptr && ws.used <= ws.left && aligned_to(ws.at, 16),
               "workspace of %lld bytes, %lld needed (mole_grouped_mm_workspace_bytes)", (long long)ws.left, (long long)ws.used);
  *part = reinterpret_cast<float*>(ws.at + ws.used - bytes);
  return MOLE_OK;
}
static int align_rows(RaggedRows& a, int elem, Aligner ws, int64_t* used, cudaStream_t st) {
  if (int rc = align_operand(ws, &a.x, 1, a.R, a.K, elem, &a.ldx, nullptr, st)) return rc;
  if (int rc = align_operand(ws, &a.w, a.E, a.kn ? a.K : a.N, a.kn ? a.N : a.K, elem, &a.ldw, a.offsets, st)) return rc;
  if (used) *used = ws.used;
  return MOLE_OK;
}

static int check_sizes(int64_t R, int a, int b, int E) {
  MOLE_REQUIRE(R >= 0 && R < (1ll << 31) - 65536, "rows=%lld", (long long)R);
  MOLE_REQUIRE(a >= 1 && b >= 1 && a <= (1 << 21) && b <= (1 << 21), "widths %d, %d", a, b);
  MOLE_REQUIRE(E >= 1 && E <= kMaxRaggedExperts, "E=%d (1..%d)", E, kMaxRaggedExperts);
  return MOLE_OK;
}

}  // namespace mole

using namespace mole;

extern "C" int mole_grouped_mm(const void* x, const void* w, const int32_t* offsets, int64_t R,
                               int32_t N, int32_t K, int32_t E, int32_t w_kn, int32_t dtype,
                               void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_sizes(R, N, K, E)) return rc;
  MOLE_REQUIRE(dtype == MOLE_F32 || dtype == MOLE_BF16, "dtype %d", dtype);
  if (R == 0) return MOLE_OK;
  MOLE_REQUIRE(x && w && offsets && out, "null pointer argument");
  const size_t size = dtype == MOLE_F32 ? 4 : 2;
  MOLE_REQUIRE(aligned_to(x, size) && aligned_to(w, size) && aligned_to(out, size) && aligned_to(offsets, 4), "a pointer is not aligned to its element");
  RaggedRows a{};
  a.x = x; a.w = w; a.offsets = offsets; a.out = out;
  a.R = R; a.N = N; a.K = K; a.E = E; a.kn = w_kn != 0;
  if (int rc = check_no_fault()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (ragged_rows_few_takes(a)) return ragged_rows_few(dtype, a, st);
  Aligner ws{static_cast<uint8_t*>(workspace), workspace_bytes, 0, false};
  if (dtype == MOLE_F32) {
    a.split = ragged_rows_simt_split(a);
    if (int rc = take_parts(ws, a.split, R * N, &a.part)) return rc;
    return ragged_rows_simt(a, st);
  }
  if (int rc = align_rows(a, 2, ws, nullptr, st)) return rc;
  return ragged_rows_tc(2, dtype, a, st);
}

extern "C" int mole_grouped_mm_workspace_bytes(const void* x, const void* w, int64_t R, int32_t N, int32_t K, int32_t E,
                                               int32_t w_kn, int32_t elem_bytes, int64_t* bytes) {
  if (int rc = check_sizes(R, N, K, E)) return rc;
  MOLE_REQUIRE(bytes != nullptr && (elem_bytes == 1 || elem_bytes == 2 || elem_bytes == 4), "bad argument");
  RaggedRows a{};
  a.x = x; a.w = w;
  a.R = R; a.N = N; a.K = K; a.E = E; a.kn = w_kn != 0;
  *bytes = 0;
  if (R == 0 || ragged_rows_few_takes(a)) return MOLE_OK;
  if (elem_bytes == 4) {
    Aligner ws{nullptr, 0, 0, true};
    if (int rc = take_parts(ws, ragged_rows_simt_split(a), R * N, nullptr)) return rc;
    *bytes = ws.used;
    return MOLE_OK;
  }
  return align_rows(a, elem_bytes, Aligner{nullptr, 0, 0, true}, bytes, nullptr);
}

extern "C" int mole_grouped_mm_wgrad(const void* a, const void* b, const int32_t* offsets, int64_t R,
                                     int32_t P, int32_t Q, int32_t E, int32_t dtype, void* out,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_sizes(R, P, Q, E)) return rc;
  MOLE_REQUIRE(dtype == MOLE_F32 || dtype == MOLE_BF16, "dtype %d", dtype);
  MOLE_REQUIRE((a && b) || R == 0, "null pointer argument");
  MOLE_REQUIRE(offsets && out, "null pointer argument");
  const size_t size = dtype == MOLE_F32 ? 4 : 2;
  MOLE_REQUIRE(aligned_to(a, size) && aligned_to(b, size) && aligned_to(out, size) && aligned_to(offsets, 4), "a pointer is not aligned to its element");
  RaggedWgrad g{};
  g.a = a; g.b = b; g.offsets = offsets; g.out = out;
  g.R = R; g.P = P; g.Q = Q; g.E = E;
  if (int rc = check_no_fault()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Aligner ws{static_cast<uint8_t*>(workspace), workspace_bytes, 0, false};
  g.split = ragged_wgrad_split(dtype == MOLE_BF16, g);
  if (int rc = take_parts(ws, g.split, (int64_t)E * P * Q, &g.part)) return rc;
  if (dtype == MOLE_F32) return ragged_wgrad_simt(g, st);
  if (R == 0) {
    MOLE_CUDA_OK(cudaMemsetAsync(out, 0, (size_t)E * P * Q * size, st));
    return MOLE_OK;
  }
  if (int rc = align_operand(ws, &g.a, 1, R, P, 2, &g.lda, nullptr, st)) return rc;
  if (int rc = align_operand(ws, &g.b, 1, R, Q, 2, &g.ldb, nullptr, st)) return rc;
  return ragged_wgrad_tc(g, st);
}

extern "C" int mole_grouped_mm_wgrad_workspace_bytes(const void* a, const void* b, int64_t R, int32_t P, int32_t Q,
                                                     int32_t E, int32_t dtype, int64_t* bytes) {
  if (int rc = check_sizes(R, P, Q, E)) return rc;
  MOLE_REQUIRE(bytes != nullptr && (dtype == MOLE_F32 || dtype == MOLE_BF16), "bad argument");
  *bytes = 0;
  if (R == 0) return MOLE_OK;
  Aligner ws{nullptr, 0, 0, true};
  int ld = 0;
  RaggedWgrad g{};
  g.R = R; g.P = P; g.Q = Q; g.E = E;
  if (int rc = take_parts(ws, ragged_wgrad_split(dtype == MOLE_BF16, g), (int64_t)E * P * Q, nullptr)) return rc;
  *bytes = ws.used;
  if (dtype == MOLE_F32) return MOLE_OK;
  if (int rc = align_operand(ws, &a, 1, R, P, 2, &ld, nullptr, nullptr)) return rc;
  if (int rc = align_operand(ws, &b, 1, R, Q, 2, &ld, nullptr, nullptr)) return rc;
  *bytes = ws.used;
  return MOLE_OK;
}

extern "C" int mole_quantize_rows(const void* x, int64_t R, int32_t K, int32_t dtype, void* q,
                                  float* scale, void* stream) {
  MOLE_REQUIRE(R >= 0 && R < (1ll << 31), "rows=%lld", (long long)R);
  MOLE_REQUIRE(K >= 1 && K <= (1 << 21), "K=%d", K);
  MOLE_REQUIRE(dtype == MOLE_F32 || dtype == MOLE_BF16, "dtype %d", dtype);
  if (R == 0) return MOLE_OK;
  MOLE_REQUIRE(x && q && scale, "null pointer argument");
  MOLE_REQUIRE(aligned_to(x, dtype == MOLE_F32 ? 4 : 2) && aligned_to(scale, 4), "a pointer is not aligned to its element");
  if (int rc = check_no_fault()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MOLE_F32 ? launch_quantize<float>(x, R, K, q, scale, st)
                           : launch_quantize<__nv_bfloat16>(x, R, K, q, scale, st);
}

extern "C" int mole_grouped_mm_i8(const void* q, const float* q_scale, const void* w, const float* w_scale,
                                  const int32_t* offsets, int64_t R, int32_t N, int32_t K, int32_t E,
                                  int32_t out_dtype, void* out, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  if (int rc = check_sizes(R, N, K, E)) return rc;
  MOLE_REQUIRE(out_dtype == MOLE_F32 || out_dtype == MOLE_BF16, "dtype %d", out_dtype);
  // |q w| <= 2^14: more terms could leave 32 bits
  MOLE_REQUIRE(K < (1 << 17), "K=%d: sums of 2^17 and more products may leave 32 bits", K);
  MOLE_REQUIRE(offsets || E == 1, "offsets may be null for one expert only");
  if (R == 0) return MOLE_OK;
  MOLE_REQUIRE(q && q_scale && w && w_scale && out, "null pointer argument");
  MOLE_REQUIRE(aligned_to(out, out_dtype == MOLE_F32 ? 4 : 2) && aligned_to(q_scale, 4) && aligned_to(w_scale, 4) && aligned_to(offsets, 4), "a pointer is not aligned to its element");
  RaggedRows a{};
  a.x = q; a.w = w; a.offsets = offsets; a.x_scale = q_scale; a.w_scale = w_scale; a.out = out;
  a.R = R; a.N = N; a.K = K; a.E = E;
  if (int rc = check_no_fault()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (ragged_rows_few_takes(a)) return ragged_rows_few_i8(out_dtype, a, st);
  if (int rc = align_rows(a, 1, Aligner{static_cast<uint8_t*>(workspace), workspace_bytes, 0, false}, nullptr, st)) return rc;
  return ragged_rows_tc(1, out_dtype, a, st);
}

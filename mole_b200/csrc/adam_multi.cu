// One Adam step over many tensors, with the two moments in 32 or in 8 bits.
//
//   adamw: p *= 1 - lr lam;   else: g += lam p
//   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2;   p -= lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// 8-bit states.  256 consecutive elements share one fp32 scale per moment (their largest magnitude
// over 448).  m is held as e4m3 times its scale; of v its square root is held, which halves the
// range of exponents that a code has to cover: a block may span 2^17 in gradient size.  Both are
// rounded up or down at random with the probability of the distance (to nearest, v would never
// move: with beta2 = 0.999 a step changes it by 0.1 %, and half a code is 3 to 6 %).  The random
// bits are a function of (seed, t, place of the tensor in the list, element), so a step can be
// repeated bit for bit.  p is updated from the moments before they are rounded.
//
// Bound by HBM: p, m, v read and written, g read, 8 bytes an element for bf16 with 8-bit states.
// A warp owns the 256 elements of a block, eight per lane, so that a scale costs one warp maximum.
// The tensors' table travels in the launch's parameters: no copy to the device, nothing to keep
// alive, and the launch can be issued on any stream.
//
// Every product, sum, quotient and root is rounded by itself (no fused multiply-add): whether a
// state's code is the one above or below must not depend on how the compiler contracts.
#include <cuda_fp8.h>

#include <cmath>

#include "common.cuh"

namespace mole {

constexpr int kAdamBlock = 256;                  // elements per scale; a warp's share
constexpr int kAdamChunk = 8 * kAdamBlock * 4;   // elements per thread block: 8 warps, 4 blocks each

struct AdamEntry {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* ms;
  float* vs;
  int64_t n;
  int32_t first_chunk;     // chunks of the launch before this tensor's
  int32_t wide;            // pointers aligned for the wide accesses
};
// kernel parameters may take 32,764 bytes: up to 500 entries a launch; a few tensors take a small
// table (fewer bytes to hand over per launch)
template <int CAP>
struct AdamTable {
  AdamEntry e[CAP];
};
struct AdamMulti {
  float decay, lam, b1, c1, b2, c2, step, r2, eps;
  int adamw;
  uint32_t key;            // of (seed, t)
  int n_entries;
  int place0;              // index of entry 0 in the caller's list
};

__host__ __device__ __forceinline__ uint32_t adam_mix(uint32_t h) {
  h *= 0x9E3779B1u;
  h = (h ^ (h >> 15)) * 0x85157AF5u;
  return h ^ (h >> 13);
}

// e4m3 by the 16 random bits u, as an fp32 value on the code grid (before the clamp to 448): codes
// of normal values keep 3 of 23 fraction bits; below 2^-6 they are 2^-9 apart, the spacing of
// [2^-6, 2^-5), so such values are lifted there and back.  A NaN is brought to 0x7fc00000 first: the
// sum of its bits and u would run over.
__device__ __forceinline__ float e4m3_random(float a, uint32_t u) {
  const float lift = a < 0.015625f ? 0.015625f : 0.f;
  const uint32_t bits = (min(__float_as_uint(__fadd_rn(a, lift)), 0x7fc00000u) + (u << 4)) & 0xFFF00000u;
  return __fsub_rn(__uint_as_float(bits), lift);
}

template <typename T>
__device__ __forceinline__ void adam_load8(const T* q, int n, bool wide, float (&v)[8]) {
  if (wide && n >= 8) {
    constexpr int V = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) {
      float t[V];
      Vec16<T>::load(q + i * V, t);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = t[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? Elem<T>::to_f(q[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void adam_store8(T* q, int n, bool wide, const float (&v)[8]) {
  if (wide && n >= 8) {
    constexpr int V = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) {
      float t[V];
#pragma unroll
      for (int j = 0; j < V; ++j) t[j] = v[i * V + j];
      Vec16<T>::store(q + i * V, t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) q[i] = Elem<T>::from_f(v[i]);
  }
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* q, int n, bool wide) {
  if (wide && n >= 8) return *reinterpret_cast<const uint2*>(q);
  uint32_t w[2] = {0, 0};
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i >> 2] |= (uint32_t)q[i] << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(uint8_t* q, int n, bool wide, uint2 c) {
  if (wide && n >= 8) {
    *reinterpret_cast<uint2*>(q) = c;
  } else {
    for (int i = 0; i < 8; ++i)
      if (i < n) q[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
  }
}
__device__ __forceinline__ void decode8(uint2 c, float (&v)[8]) {
  const uint32_t w[4] = {c.x & 0xffffu, c.x >> 16, c.y & 0xffffu, c.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w[i], __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint2 encode8(const float (&v)[8]) {    // values on the grid: exact; above 448: 448
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}
// Largest finite magnitude of the warp's 256 values (non-negative floats order as their bits).  A
// value that is not finite counts for nothing: it must not spoil its neighbours' scale.
__device__ __forceinline__ float block_top(const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if (top >= 0x7f800000u) {
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
      if (b < 0x7f800000u) top = max(top, b);
    }
    top = __reduce_max_sync(0xffffffffu, top);
  }
  return __uint_as_float(top);
}

// 256 elements of one tensor, from element `at` on; `left` of them exist (at least one)
template <typename T, int BITS>
__device__ __forceinline__ void adam_block(const AdamEntry& e, const AdamMulti& a, uint32_t key, int64_t at,
                                           int64_t left, int lane) {
  const int64_t i0 = at + lane * 8;
  const int n = (int)max((int64_t)0, min((int64_t)8, left - lane * 8));
  const bool wide = e.wide != 0;
  T* pp = static_cast<T*>(e.p) + i0;
  float p[8], g[8], m[8], v[8];
  adam_load8(pp, n, wide, p);
  adam_load8(static_cast<const T*>(e.g) + i0, n, wide, g);
  if (BITS == 32) {
    adam_load8(static_cast<const float*>(e.m) + i0, n, wide, m);
    adam_load8(static_cast<const float*>(e.v) + i0, n, wide, v);
  } else {
    const uint2 mc = load_codes(static_cast<const uint8_t*>(e.m) + i0, n, wide);
    const uint2 vc = load_codes(static_cast<const uint8_t*>(e.v) + i0, n, wide);
    const float sm = e.ms[at / kAdamBlock], sv = e.vs[at / kAdamBlock];
    decode8(mc, m);
    decode8(vc, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = __fmul_rn(m[i], sm);
      v[i] = __fmul_rn(v[i], sv);
      v[i] = __fmul_rn(v[i], v[i]);
    }
  }
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!a.adamw) g[i] = __fadd_rn(g[i], __fmul_rn(a.lam, p[i]));
    m[i] = __fadd_rn(__fmul_rn(a.b1, m[i]), __fmul_rn(a.c1, g[i]));
    v[i] = __fadd_rn(__fmul_rn(a.b2, v[i]), __fmul_rn(__fmul_rn(a.c2, g[i]), g[i]));
    s[i] = __fsqrt_rn(v[i]);
    if (a.adamw) p[i] = __fmul_rn(p[i], a.decay);
    p[i] = __fsub_rn(p[i], __fdiv_rn(__fmul_rn(a.step, m[i]), __fadd_rn(__fmul_rn(s[i], a.r2), a.eps)));
  }
  adam_store8(pp, n, wide, p);
  if (BITS == 32) {
    adam_store8(static_cast<float*>(e.m) + i0, n, wide, m);
    adam_store8(static_cast<float*>(e.v) + i0, n, wide, v);
    return;
  }
  // lanes behind the tensor's end hold zeros
  if (n < 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= n) m[i] = s[i] = 0.f;
  }
  const float mt = block_top(m), st = block_top(s);
  // a block whose largest value is below 2^-100 is held as zeros: 448 / top would overflow
  const bool ml = mt >= 0x1p-100f, sl = st >= 0x1p-100f;
  const float mi = ml ? __fdiv_rn(448.f, mt) : 0.f, si = sl ? __fdiv_rn(448.f, st) : 0.f;
  uint32_t r = adam_mix((uint32_t)(i0 >> 3) + key);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r = r * 1664525u + 1013904223u;
    const float y = __fmul_rn(m[i], mi);
    m[i] = __uint_as_float(__float_as_uint(e4m3_random(fabsf(y), r >> 16)) | (__float_as_uint(y) & 0x80000000u));
    // a second moment that is not zero is never held as zero: the step divides by it
    const float q = e4m3_random(__fmul_rn(s[i], si), r & 0xffffu);
    s[i] = (q < 0.001953125f && s[i] > 0.f && sl) ? 0.001953125f : q;
  }
  store_codes(static_cast<uint8_t*>(e.m) + i0, n, wide, encode8(m));
  store_codes(static_cast<uint8_t*>(e.v) + i0, n, wide, encode8(s));
  if (lane == 0) {
    e.ms[at / kAdamBlock] = ml ? __fmul_rn(mt, 1.f / 448.f) : 0.f;
    e.vs[at / kAdamBlock] = sl ? __fmul_rn(st, 1.f / 448.f) : 0.f;
  }
}

template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(256)
adam_multi_kernel(const __grid_constant__ AdamTable<CAP> table, const __grid_constant__ AdamMulti a) {
  const int chunk = blockIdx.x;
  int lo = 0, hi = a.n_entries;                     // last entry whose first chunk is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table.e[mid].first_chunk <= chunk) lo = mid; else hi = mid;
  }
  const AdamEntry& e = table.e[lo];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t key = adam_mix(a.key + (uint32_t)(a.place0 + lo));
  const int64_t base = (int64_t)(chunk - e.first_chunk) * kAdamChunk;
  for (int i = 0; i < 4; ++i) {
    const int64_t at = base + (int64_t)(i * 8 + warp) * kAdamBlock;
    if (at < e.n) adam_block<T, BITS>(e, a, key, at, e.n - at, lane);
  }
}

template <typename T, int BITS, int CAP>
static int adam_launch(const mole_adam_tensor* t, int from, int to, AdamMulti a, cudaStream_t st) {
  static_assert(sizeof(AdamTable<CAP>) + sizeof(AdamMulti) <= 32764, "kernel parameters");
  AdamTable<CAP> table;
  int64_t chunks = 0;
  a.n_entries = 0;
  a.place0 = from;
  for (int i = from; i < to; ++i) {
    // empty tensors keep their place (an entry with no chunk is never picked: the search takes the last)
    AdamEntry& e = table.e[a.n_entries++];
    e.p = t[i].p; e.g = t[i].g; e.m = t[i].m; e.v = t[i].v;
    e.ms = t[i].m_scale; e.vs = t[i].v_scale;
    e.n = t[i].n;
    e.first_chunk = (int32_t)chunks;
    const uintptr_t pg = reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.g);
    const uintptr_t mv = reinterpret_cast<uintptr_t>(e.m) | reinterpret_cast<uintptr_t>(e.v);
    e.wide = (pg & 15) == 0 && (mv & (BITS == 32 ? 15 : 7)) == 0;
    chunks += (e.n + kAdamChunk - 1) / kAdamChunk;
    MOLE_REQUIRE(chunks <= 0x7fffffff, "too many elements for one call");
  }
  if (chunks == 0) return MOLE_OK;
  adam_multi_kernel<T, BITS, CAP><<<(unsigned)chunks, 256, 0, st>>>(table, a);
  MOLE_LAUNCH_OK();
  return MOLE_OK;
}

template <typename T, int BITS>
static int adam_all(const mole_adam_tensor* t, int n, const AdamMulti& a, cudaStream_t st) {
  if (n <= 16) return adam_launch<T, BITS, 16>(t, 0, n, a, st);
  for (int from = 0; from < n; from += 500)
    if (int rc = adam_launch<T, BITS, 500>(t, from, from + 500 < n ? from + 500 : n, a, st)) return rc;
  return MOLE_OK;
}

}  // namespace mole

using namespace mole;

extern "C" int mole_adam_multi(const mole_adam_tensor* tensors, int32_t n_tensors, int32_t dtype,
                               int32_t state_bits, double beta1, double beta2, int32_t t, double lr,
                               double lam, double eps, int32_t adamw, uint32_t seed, void* stream) {
  MOLE_REQUIRE(n_tensors >= 0 && (tensors || n_tensors == 0), "bad tensor list");
  MOLE_REQUIRE(t >= 1, "step count t=%d must be at least 1 (the count after this step)", t);
  MOLE_REQUIRE(dtype == MOLE_F32 || dtype == MOLE_BF16, "dtype %d", dtype);
  MOLE_REQUIRE(state_bits == 32 || state_bits == 8, "state_bits=%d: the moments are held in 32 or 8 bits", state_bits);
  MOLE_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "beta1=%g beta2=%g", beta1, beta2);
  MOLE_REQUIRE(eps >= 0.0 && std::isfinite(lr) && std::isfinite(lam), "lr=%g lam=%g eps=%g", lr, lam, eps);
  for (int i = 0; i < n_tensors; ++i) {
    const mole_adam_tensor& x = tensors[i];
    MOLE_REQUIRE(x.n >= 0 && x.n < (1ll << 34), "tensor %d: n=%lld", i, (long long)x.n);
    MOLE_REQUIRE(x.n == 0 || (x.p && x.g && x.m && x.v), "tensor %d: null pointer", i);
    MOLE_REQUIRE(x.n == 0 || state_bits == 32 || (x.m_scale && x.v_scale), "tensor %d: 8-bit states need their scales", i);
    const uintptr_t el = dtype == MOLE_F32 ? 3 : 1, mv = state_bits == 32 ? 3 : 0;
    MOLE_REQUIRE(((reinterpret_cast<uintptr_t>(x.p) | reinterpret_cast<uintptr_t>(x.g)) & el) == 0 &&
                     ((reinterpret_cast<uintptr_t>(x.m) | reinterpret_cast<uintptr_t>(x.v)) & mv) == 0 &&
                     ((reinterpret_cast<uintptr_t>(x.m_scale) | reinterpret_cast<uintptr_t>(x.v_scale)) & 3) == 0,
                 "tensor %d: a pointer is not aligned to its element", i);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  MOLE_CUDA_OK(cudaStreamIsCapturing(st, &cap));
  if (cap != cudaStreamCaptureStatusNone)
    return fail(MOLE_ERR_STATE, "t and lr are taken by value: a captured step would repeat one step count for ever");
  AdamMulti a{};
  a.decay = (float)(1.0 - lr * lam);
  a.lam = (float)lam;
  a.b1 = (float)beta1; a.c1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2; a.c2 = (float)(1.0 - beta2);
  a.step = (float)(lr / (1.0 - std::pow(beta1, (double)t)));
  a.r2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)t)));
  a.eps = (float)eps;
  a.adamw = adamw;
  a.key = adam_mix(adam_mix(seed) + (uint32_t)t);
  if (dtype == MOLE_F32)
    return state_bits == 32 ? adam_all<float, 32>(tensors, n_tensors, a, st) : adam_all<float, 8>(tensors, n_tensors, a, st);
  return state_bits == 32 ? adam_all<__nv_bfloat16, 32>(tensors, n_tensors, a, st)
                          : adam_all<__nv_bfloat16, 8>(tensors, n_tensors, a, st);
}

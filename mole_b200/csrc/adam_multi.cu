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
// Bytes: p, m, v read and written, g read, 8 an element for bf16 with 8-bit states.  537M such elements
// take 1.05 ms (4.1 TB/s; the bytes alone 0.82), 1.17 ms when the power limit holds the clock: bound by
// instructions, 53 an element, since every rounding is by itself.  32-bit states are bound by HBM: 60M
// bf16 elements in 400 tensors in 0.25 ms (41 us of it the host's, floor 0.20).
// A warp takes the 256 elements of a block, eight per lane, so that a scale costs one warp maximum.
// The tensors' table travels in the launch's parameters: no copy to the device, nothing to keep
// alive, and the launch can be issued on any stream.
//
// Every product, sum, quotient and root is an operation of its own, in both forms of the arithmetic below,
// rounded correctly but for about one root or quotient in 2^20 of the whole blocks' form: whether a state's
// code is the one above or below must not depend on how a compiler contracts.
//
// The rounding of sqrt(v) has mean zero; its square has not: v is held 4 % too large on average where
// gradients vary (beta2 = 0.999 or 0.99; 2.5 % at 0.95; gradients of equal size: 0.3 %), a simulation of
// 3000 steps against the recursion in 64 bits.  sqrt(v), which the step divides by, is 1 % too large.
#include <cuda_fp8.h>

#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "f32x2.cuh"
#include "tc_ptx.cuh"

namespace mole {

constexpr int kAdamBlock = 256;                  // elements per scale; what a warp takes at a time
constexpr int kAdamWarps = 8;                    // of a thread block that compute; one more moves data
constexpr int kAdamThreads = 32 * (kAdamWarps + 1);

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
  float decay, lam;        // AdamW: decay = 1 - lr lam, lam = 0; Adam: decay = 1, lam
  float b1, c1, b2, c2, step, r2, eps;
  float one;               // 1, which the compiler must not know
  uint32_t key;            // of (seed, t)
  int chunks;              // of all entries; a thread block walks every gridDim.x-th
  int n_entries;
  int32_t* fault;
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

// Rounds the warp's 256 values of both moments (m and the root s of v; zeros where lanes have no element)
// to codes and stores them with their scales: any values.
__device__ __forceinline__ void adam_round(const AdamEntry& e, const AdamMulti& a, uint32_t key, int64_t at, int64_t i0, int n,
                                        int lane, float (&m)[8], float (&s)[8]) {
  const bool wide = e.wide != 0;
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

// 256 elements of one tensor, from element `at` on; `left` of them exist (at least one): any values, any
// alignment.  The common case is adam_block_full below.
template <typename T, int BITS>
__device__ __noinline__ void adam_block(const AdamEntry& e, const AdamMulti& a, uint32_t key, int64_t at,
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
    if (a.lam != 0.f) g[i] = __fadd_rn(g[i], __fmul_rn(a.lam, p[i]));
    m[i] = __fadd_rn(__fmul_rn(a.b1, m[i]), __fmul_rn(a.c1, g[i]));
    v[i] = __fadd_rn(__fmul_rn(a.b2, v[i]), __fmul_rn(__fmul_rn(a.c2, g[i]), g[i]));
    s[i] = __fsqrt_rn(v[i]);
    p[i] = __fsub_rn(__fmul_rn(p[i], a.decay), __fdiv_rn(__fmul_rn(a.step, m[i]), __fadd_rn(__fmul_rn(s[i], a.r2), a.eps)));
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
  adam_round(e, a, key, at, i0, n, lane, m, s);
}

// ---- a whole block of ordinary values ---------------------------------------------------------------
// At 44 instructions an element the issue slots are full by the time HBM has moved 8 bytes; this form,
// with everything around it, gets by with 53 (32-bit states: 37), by
//   * pairs of values on the packed instructions, but for the root and the quotient, whose scalars would
//     have to be moved into pairs;
//   * root and quotient from the hardware's approximation with one Newton step whose residual is a
//     fused multiply-add (Markstein 1990): the correctly rounded result but for about one value in
//     2^20, without the handling of special ranges;
//   * codes made in the integer domain: a value times 2^-120 has, as an fp32 number, e4m3's exponent
//     field and its gradual underflow, 20 fraction bits further down; adding the random bits there and
//     cutting rounds normal and subnormal codes alike.
// Whatever does not fit (zeros and tiny values in v, values that are not finite, a top outside
// [2^-100, 2^13], beyond which 448 / top 2^-120 is no normal number) shows as a quotient that is not
// finite or in the tops, and the block is redone by the general form; nothing has been stored by then.
// That is dear: 180 instructions an element in all (130 for 32-bit states).  The ordinary case among them is
// an expert that has had no rows yet, gradient and state zero: 268M bf16 elements with 8-bit states take
// 0.56 ms, with a quarter, half and all of them so 0.97, 1.40 and 2.23; 67M with 32-bit states 0.24, 0.34,
// 0.44 and 0.66.  Tensors that do not start on 16 bytes take the general form throughout: 1.98 and 0.67 ms.
__device__ __forceinline__ float rsqrt_hw(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_hw(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float root(float x) {
  const float y = rsqrt_hw(x), r = __fmul_rn(x, y);                          // off by 2^-22
  return __fmaf_rn(__fmaf_rn(-r, r, x), __fmul_rn(0.5f, y), r);
}
__device__ __forceinline__ float minus_quotient(float num, float den) {
  const float nr = rcp_hw(-den), q = __fmul_rn(num, nr);
  return __fmaf_rn(__fmaf_rn(den, q, num), nr, q);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float quotient_448(float top) {
  const float r = rcp_hw(top), q = 448.f * r;
  return fmaf(fmaf(-top, q, 448.f), r, q);
}

template <typename T> struct AdamLane;               // eight values of a type, in shared and global memory
template <> struct AdamLane<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void read(const void* q) { w = *static_cast<const uint4*>(q); }
  __device__ __forceinline__ uint64_t pair(int i) const {
    const uint32_t x = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
    return f2_pack(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
  __device__ static __forceinline__ void store(void* q, const uint64_t (&v)[4]) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      f2_unpack(v[i], lo, hi);
      const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
      o[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *static_cast<uint4*>(q) = make_uint4(o[0], o[1], o[2], o[3]);
  }
};
template <> struct AdamLane<float> {
  float4 a, b;
  __device__ __forceinline__ void read(const void* q) {
    a = static_cast<const float4*>(q)[0];
    b = static_cast<const float4*>(q)[1];
  }
  __device__ __forceinline__ uint64_t pair(int i) const {
    return i == 0 ? f2_pack(a.x, a.y) : i == 1 ? f2_pack(a.z, a.w) : i == 2 ? f2_pack(b.x, b.y) : f2_pack(b.z, b.w);
  }
  __device__ static __forceinline__ void store(void* q, const uint64_t (&v)[4]) {
    float4 x, y;
    f2_unpack(v[0], x.x, x.y); f2_unpack(v[1], x.z, x.w);
    f2_unpack(v[2], y.x, y.y); f2_unpack(v[3], y.z, y.w);
    static_cast<float4*>(q)[0] = x;
    static_cast<float4*>(q)[1] = y;
  }
};
struct e4m3_code {};
template <> struct AdamLane<e4m3_code> {
  uint2 w;
  __device__ __forceinline__ void read(const void* q) { w = *static_cast<const uint2*>(q); }
  __device__ __forceinline__ uint64_t pair(int i) const {
    const uint32_t x = i < 2 ? w.x : w.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((i & 1) ? x >> 16 : x & 0xffffu), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    return f2_pack(f.x, f.y);
  }
};
// A chunk of one tensor in shared memory: p, g, m, v as they lie in global memory, updated in place
template <typename T, int BITS>
struct AdamStage {
  using M = typename std::conditional<BITS == 8, AdamLane<e4m3_code>, AdamLane<float>>::type;
  using P = AdamLane<T>;
  static constexpr int kElems = BITS == 8 && sizeof(T) == 2 ? 4096 : 2048;
  static constexpr int kBlocks = kElems / kAdamBlock;
  static constexpr int kP = kElems * (int)sizeof(T), kM = kElems * (BITS / 8);
  static constexpr int kBytes = 2 * kP + 2 * kM;                     // 20 to 32 KB
  static constexpr int kResident = 228 * 1024 / (3 * kBytes + 3328);   // thread blocks per SM
};
// top bytes of four words
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

// The scalars of the whole blocks' form, twice each where pairs take them
struct AdamConsts {
  uint64_t lam2, b12, c12, b22, c22, decay2, one2;
  float step, r2, eps;
  bool l2;
  __device__ __forceinline__ void init(const AdamMulti& a) {
    lam2 = f2_dup(a.lam);
    l2 = a.lam != 0.f;
    b12 = f2_dup(a.b1); c12 = f2_dup(a.c1); b22 = f2_dup(a.b2); c22 = f2_dup(a.c2); decay2 = f2_dup(a.decay); one2 = f2_dup(a.one);
    step = a.step; r2 = a.r2; eps = a.eps;
  }
};

// Block b of a stage, in place; `scale` in: of m and v, out: the new ones.  false: nothing changed, the
// block needs the general form.
template <typename T, int BITS>
__device__ __forceinline__ bool adam_block_full(uint8_t* stage, int b, float2& scale, const AdamConsts& a, uint32_t hash_at,
                                                int lane) {
  using S = AdamStage<T, BITS>;
  const int i0 = b * kAdamBlock + lane * 8;
  uint8_t* ap = stage + i0 * (int)sizeof(T);
  uint8_t* am = stage + 2 * S::kP + i0 * (BITS / 8);
  uint8_t* av = am + S::kM;
  typename S::P rp, rg;
  typename S::M rm, rv;
  rp.read(ap);
  rg.read(ap + S::kP);
  rm.read(am);
  rv.read(av);
  uint64_t p[4], m[4], v[4], s[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint64_t g = rg.pair(i);
    p[i] = rp.pair(i);
    m[i] = rm.pair(i);
    v[i] = rv.pair(i);
    if (BITS == 8) {
      m[i] = f2_mul(m[i], f2_dup(scale.x));
      v[i] = f2_mul(v[i], f2_dup(scale.y));
      v[i] = f2_mul(v[i], v[i]);
    }
    // x + y as x * one + y: the compiler contracts packed products into packed sums that follow them
    if (a.l2) g = f2_fma(f2_mul(a.lam2, p[i]), a.one2, g);
    m[i] = f2_fma(f2_mul(a.b12, m[i]), a.one2, f2_mul(a.c12, g));
    v[i] = f2_fma(f2_mul(a.b22, v[i]), a.one2, f2_mul(f2_mul(a.c22, g), g));
    float v0, v1, m0, m1;
    f2_unpack(v[i], v0, v1);
    f2_unpack(m[i], m0, m1);
    const float s0 = root(v0), s1 = root(v1);
    s[i] = f2_pack(s0, s1);
    const uint64_t q = f2_pack(minus_quotient(__fmul_rn(a.step, m0), __fadd_rn(__fmul_rn(s0, a.r2), a.eps)),
                               minus_quotient(__fmul_rn(a.step, m1), __fadd_rn(__fmul_rn(s1, a.r2), a.eps)));
    sum = i == 0 ? q : f2_add(sum, q);
    p[i] = f2_fma(f2_mul(p[i], a.decay2), a.one2, q);
  }
  float lo, hi;
  f2_unpack(sum, lo, hi);
  bool odd = !(fabsf(lo + hi) < __int_as_float(0x7f800000));
  if (BITS == 32) {
    if (__any_sync(0xffffffffu, odd)) return false;
    AdamLane<T>::store(ap, p);
    AdamLane<float>::store(am, m);
    AdamLane<float>::store(av, v);
    return true;
  }
  float mt = 0.f, st = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f2_unpack(m[i], lo, hi);
    mt = max3(mt, fabsf(lo), fabsf(hi));
    f2_unpack(s[i], lo, hi);
    st = max3(st, lo, hi);
  }
  mt = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mt)));
  st = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(st)));
  odd = odd || !(mt >= 0x1p-100f && mt <= 8192.f && st >= 0x1p-100f && st <= 8192.f);
  if (__any_sync(0xffffffffu, odd)) return false;
  AdamLane<T>::store(ap, p);
  const uint64_t mi = f2_dup(quotient_448(mt) * 0x1p-120f), si = f2_dup(quotient_448(st) * 0x1p-120f);
  uint32_t r = adam_mix(hash_at);
  uint32_t mw[8], sw[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[2], z[2];
    f2_unpack(f2_mul(m[i], mi), y[0], y[1]);
    f2_unpack(f2_mul(s[i], si), z[0], z[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      r = r * 1664525u + 1013904223u;
      // bits of a value: sign, four zeros, the code's seven bits, 20 bits below them, to which the random
      // 16 are added at their top.  Moved up by four, the code is the top byte.  The top is 448 and at
      // most some units, so the sum stays below the code of NaN.
      const uint32_t b = __float_as_uint(y[j]);
      mw[2 * i + j] = ((b << 4) + __byte_perm(r, 0, 0x4324)) | (b & 0x80000000u);
      // a second moment that is not zero is never held as zero
      sw[2 * i + j] = max((__float_as_uint(z[j]) << 4) + __byte_perm(r, 0, 0x4104), 1u << 24);
    }
  }
  *reinterpret_cast<uint2*>(am) =
      make_uint2(top_bytes(mw[0], mw[1], mw[2], mw[3]), top_bytes(mw[4], mw[5], mw[6], mw[7]));
  *reinterpret_cast<uint2*>(av) =
      make_uint2(top_bytes(sw[0], sw[1], sw[2], sw[3]), top_bytes(sw[4], sw[5], sw[6], sw[7]));
  scale = make_float2(__fmul_rn(mt, 1.f / 448.f), __fmul_rn(st, 1.f / 448.f));
  return true;
}

// Chunks come and go by bulk copies of 4 to 16 KB, three stages deep, and are updated in place in
// shared memory; one warp moves data, eight compute and meet only at the stages' barriers.  Copies
// that large, by neighbouring thread blocks at the same time, keep DRAM pages open: the same bytes read
// and written by every warp in pieces of 256 to 512 bytes took 1.14 ms for 537M bf16 elements with 8-bit
// states without any arithmetic, longer than this whole kernel (1.05 ms; its copies alone 0.79).
constexpr int kAdamStages = 3;
constexpr int kAdamWalk = 32;                    // chunks of a thread block at most: the scheduler evens out the SMs

template <int CAP>
__device__ __forceinline__ int entry_of(const AdamTable<CAP>& table, int n, int chunk) {
  int lo = 0, hi = n;                               // last entry whose first chunk is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table.e[mid].first_chunk <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kAdamThreads, AdamStage<T, BITS>::kResident)
adam_multi_kernel(const __grid_constant__ AdamTable<CAP> table, const __grid_constant__ AdamMulti a) {
  using S = AdamStage<T, BITS>;
  extern __shared__ __align__(128) uint8_t ring[];  // [kAdamStages][S::kBytes]
  __shared__ __align__(8) uint64_t bars[2 * kAdamStages];
  __shared__ uint32_t odd_s[kAdamWalk];             // bit b: block b of that chunk goes to the general form
  __shared__ int abort_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full0 = smem_u32(bars), done0 = smem_u32(bars + kAdamStages), ring0 = smem_u32(ring);
  if (threadIdx.x < kAdamWalk) odd_s[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int i = 0; i < kAdamStages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(done0 + 8 * i, kAdamWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  after_previous();
  const int steps = (a.chunks - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;

  struct Place { int entry, end; };                 // entry of a chunk, first chunk behind that entry
  auto place_of = [&](int chunk, Place& w) {
    if (chunk < w.end) return;
    w.entry = entry_of(table, a.n_entries, chunk);
    w.end = w.entry + 1 < a.n_entries ? table.e[w.entry + 1].first_chunk : a.chunks;
  };
  auto whole_blocks = [&](const AdamEntry& e, int chunk) {
    const int64_t left = e.n - (int64_t)(chunk - e.first_chunk) * S::kElems;
    return e.wide ? (left >= S::kElems ? S::kBlocks : (int)left / kAdamBlock) : 0;
  };
  Place here = {0, 0};
  if (warp == kAdamWarps) {
    if (lane == 0) {
      Place ahead = {0, 0};
      auto fetch = [&](int i) {
        const int chunk = blockIdx.x + i * gridDim.x;
        place_of(chunk, ahead);
        const AdamEntry& e = table.e[ahead.entry];
        const int n = whole_blocks(e, chunk) * kAdamBlock;
        if (n == 0) return;
        const int64_t at = (int64_t)(chunk - e.first_chunk) * S::kElems;
        const uint32_t dst = ring0 + (i % kAdamStages) * S::kBytes, bar = full0 + 8 * (i % kAdamStages);
        const uint32_t pb = n * (uint32_t)sizeof(T), mb = n * (BITS / 8);
        mbar_expect_tx(bar, 2 * pb + 2 * mb);
        bulk_load(dst, static_cast<const T*>(e.p) + at, pb, bar);
        bulk_load(dst + S::kP, static_cast<const T*>(e.g) + at, pb, bar);
        bulk_load(dst + 2 * S::kP, static_cast<const uint8_t*>(e.m) + at * (BITS / 8), mb, bar);
        bulk_load(dst + 2 * S::kP + S::kM, static_cast<const uint8_t*>(e.v) + at * (BITS / 8), mb, bar);
      };
      for (int i = 0; i < kAdamStages - 1 && i < steps; ++i) fetch(i);
      uint32_t uses = 0;                            // bit s: parity of the uses of stage s so far
      for (int i = 0; i < steps; ++i) {
        const int chunk = blockIdx.x + i * gridDim.x, st = i % kAdamStages;
        place_of(chunk, here);
        const AdamEntry& e = table.e[here.entry];
        const int whole = whole_blocks(e, chunk);
        if (whole > 0) {
          if (!mbar_wait(done0 + 8 * st, (uses >> st) & 1u, &abort_s, a.fault, 82)) break;
          uses ^= 1u << st;
          const int64_t at = (int64_t)(chunk - e.first_chunk) * S::kElems;
          const uint32_t src = ring0 + st * S::kBytes;
          const uint32_t pb = whole * kAdamBlock * (uint32_t)sizeof(T), mb = whole * kAdamBlock * (BITS / 8);
          bulk_store(static_cast<T*>(e.p) + at, src, pb);
          bulk_store(static_cast<uint8_t*>(e.m) + at * (BITS / 8), src + 2 * S::kP, mb);
          bulk_store(static_cast<uint8_t*>(e.v) + at * (BITS / 8), src + 2 * S::kP + S::kM, mb);
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        // the rest of the chunk: a partial block, or all of it where the tensor is not wide
        const int64_t left = e.n - (int64_t)(chunk - e.first_chunk) * S::kElems;
        const int blocks = left >= S::kElems ? S::kBlocks : ((int)left + kAdamBlock - 1) / kAdamBlock;
        if (blocks > whole) atomicOr(&odd_s[i], ((1u << blocks) - 1u) & ~((1u << whole) - 1u));
        // the stage of the step before is free once its stores have read it
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        if (i + kAdamStages - 1 < steps) fetch(i + kAdamStages - 1);
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  } else {
    AdamConsts c;
    c.init(a);
    constexpr int kPer = S::kBlocks / kAdamWarps;
    // While the chunks stay inside the whole chunks of one tensor (before `end`) a step costs no more
    // than advancing these: the scales of this warp's first block, the hash's argument.
    float* ms = nullptr;
    float* vs = nullptr;
    uint32_t hash0 = 0, uses = 0;
    int end = 0, st = 0, chunk = blockIdx.x;
    const int stride = (int)gridDim.x * S::kBlocks;
#pragma unroll 1
    for (int i = 0; i < steps; ++i, chunk += gridDim.x) {
      int whole = S::kBlocks;
      if (chunk < end) {
        if (BITS == 8) { ms += stride; vs += stride; }
        hash0 += (uint32_t)stride * (kAdamBlock / 8);
      } else {
        place_of(chunk, here);
        const AdamEntry& e = table.e[here.entry];
        whole = whole_blocks(e, chunk);
        const int blk0 = (chunk - e.first_chunk) * S::kBlocks + warp;
        if (BITS == 8) { ms = e.ms + blk0; vs = e.vs + blk0; }
        hash0 = adam_mix(a.key + (uint32_t)(a.place0 + here.entry)) + (uint32_t)blk0 * (kAdamBlock / 8) + lane;
        end = whole == S::kBlocks ? e.first_chunk + (int)(e.n / S::kElems) : 0;
      }
      if (whole > 0) {
        float2 scale[kPer];
        if (BITS == 8) {
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (warp + kAdamWarps * j < whole) scale[j] = make_float2(ms[kAdamWarps * j], vs[kAdamWarps * j]);
        }
        if (!__all_sync(0xffffffffu, mbar_wait(full0 + 8 * st, (uses >> st) & 1u, &abort_s, a.fault, 81))) break;
        uses ^= 1u << st;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int b = warp + kAdamWarps * j;
          if (b >= whole) break;
          if (adam_block_full<T, BITS>(ring + st * S::kBytes, b, scale[j], c, hash0 + j * kAdamWarps * (kAdamBlock / 8), lane)) {
            if (BITS == 8 && lane < 2) (lane ? vs : ms)[kAdamWarps * j] = lane ? scale[j].y : scale[j].x;
          } else if (lane == 0) {
            atomicOr(&odd_s[i], 1u << b);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the bulk stores read what was written here
        __syncwarp();
        if (lane == 0) mbar_arrive(done0 + 8 * st);
      }
      if (++st == kAdamStages) st = 0;
    }
  }
  __syncthreads();
  if (abort_s) {                                    // loads under way get time to land
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 20000000ull) __nanosleep(1000);
    if (threadIdx.x == 0) report_fault(a.fault);
    return;
  }
  // what the whole blocks' form left over, now that its stores are done
  if (warp == kAdamWarps) return;
  for (int i = 0; i < steps; ++i) {
    const uint32_t odd = odd_s[i];
    if (odd == 0) continue;
    const int chunk = blockIdx.x + i * gridDim.x;
    const int en = entry_of(table, a.n_entries, chunk);
    const AdamEntry& e = table.e[en];
    for (int b = warp; b < S::kBlocks; b += kAdamWarps) {
      if (!((odd >> b) & 1u)) continue;
      const int64_t first = (int64_t)(chunk - e.first_chunk) * S::kElems + b * kAdamBlock;
      adam_block<T, BITS>(e, a, adam_mix(a.key + (uint32_t)(a.place0 + en)), first, e.n - first, lane);
    }
  }
}

template <typename T, int BITS, int CAP>
static int adam_launch(const mole_adam_tensor* t, int from, int to, AdamMulti a, cudaStream_t st) {
  using S = AdamStage<T, BITS>;
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
    e.wide = ((pg | mv) & 15) == 0;
    chunks += (e.n + S::kElems - 1) / S::kElems;
    MOLE_REQUIRE(chunks <= 0x3fffffff, "too many elements for one call");
  }
  if (chunks == 0) return MOLE_OK;
  a.chunks = (int)chunks;
  auto kern = adam_multi_kernel<T, BITS, CAP>;
  constexpr int smem = kAdamStages * S::kBytes;
  static PerDeviceInt configured;
  const int dev = current_device();
  if (!configured.get(dev)) {
    MOLE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    configured.set(dev, 1);
  }
  int64_t grid = (int64_t)sm_count() * S::kResident;
  if (grid < (chunks + kAdamWalk - 1) / kAdamWalk) grid = (chunks + kAdamWalk - 1) / kAdamWalk;
  if (grid > chunks) grid = chunks;
  return launch_early(kern, dim3((unsigned)grid), kAdamThreads, smem, st, table, a);
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
  if (int rc = check_no_fault()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  MOLE_CUDA_OK(cudaStreamIsCapturing(st, &cap));
  if (cap != cudaStreamCaptureStatusNone)
    return fail(MOLE_ERR_STATE, "t and lr are taken by value: a captured step would repeat one step count for ever");
  AdamMulti a{};
  a.fault = device_fault_word();
  MOLE_REQUIRE(a.fault != nullptr, "fault word not allocated");
  a.decay = adamw ? (float)(1.0 - lr * lam) : 1.f;
  a.lam = adamw ? 0.f : (float)lam;
  a.b1 = (float)beta1; a.c1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2; a.c2 = (float)(1.0 - beta2);
  a.step = (float)(lr / (1.0 - std::pow(beta1, (double)t)));
  a.r2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)t)));
  a.eps = (float)eps;
  a.one = 1.f;
  a.key = adam_mix(adam_mix(seed) + (uint32_t)t);
  if (dtype == MOLE_F32)
    return state_bits == 32 ? adam_all<float, 32>(tensors, n_tensors, a, st) : adam_all<float, 8>(tensors, n_tensors, a, st);
  return state_bits == 32 ? adam_all<__nv_bfloat16, 32>(tensors, n_tensors, a, st)
                          : adam_all<__nv_bfloat16, 8>(tensors, n_tensors, a, st);
}

// Products over rows packed by expert on the sm_100a tensor cores: bf16 with fp32 sums and 8-bit
// integers with 32-bit sums (tcgen05.mma, cta_group::2, accumulators in TMEM, operands by TMA).
//
// Rows product.  The weights are the M side: a pair of CTAs takes 512 output features of one expert, 2 x
// 128 each (256 where there are few items), and a panel of up to 256 of its rows as the N side, in steps
// of 16 (32 for integers), so that ragged row counts cost their own size and not the next multiple of
// 128 or 256.  A stage of the ring is 128 bytes of the reduction: this CTA's features (16 KB per 128)
// and its half of the panel's rows.  The two blocks of 256 features have an accumulator each, and the
// MMAs alternate between them: back to back into one, each takes 43 cycles more than its N / 2, and a
// byte of rows staged serves both.  TMEM holds two accumulators of 256 columns.  Panels of up to 128
// rows use one half of it, so that their epilogue runs under the next item's main loop; larger ones
// need both halves, and the next item starts on the first while the second is still being drained.
// Neighbouring rows that a panel's last step reads belong to other experts: each row is a column of
// the accumulator of its own, and such columns are not stored.
//
// Weight gradient.  out_e = a_e^T b_e: 256 x 256 of an expert's matrix per pair, the reduction runs
// over its rows, 64 per stage.  The last 16-row step of an expert may reach into rows of others,
// which must not enter the sum, not even as 0 times NaN: a warp per CTA (the "fixer") writes zeros
// over them in shared memory, in both operands, before that stage is handed to the tensor cores.
// There are no padding rows in memory to do without it, and 16 rows are all that is wasted.
//
// What bounds them: in a single launch the waits for the ring and, in the weight gradient, for accumulators; in
// a long run the board's power as well (the clock falls to 1.0 to 1.5 GHz of 1.97).  64 experts of 256 rows,
// 8192 -> 2048, N-major: 0.45, 0.44 and 0.57 ms for the three products in single launches (1.2, 1.2 and
// 1.0 PFLOP/s; memory 5.5, 5.6 and 4.4 TB/s), 0.58, 0.58 and 0.71 back to back for seconds; a batched library
// product of the same equal batches 0.54 (forward) and 0.59 (dw), 0.63 and 0.71.  12 experts of 340 rows,
// 2048 -> 8192: 0.14, 0.16 and 0.17 ms, the library's 0.12 and 0.15.  Integers, 32768 rows of 128 experts,
// 2048 -> 8192: 0.49 ms in a single launch, 0.63 back to back (2.3 and 1.75 POP/s).
//
// Every wait is bounded: a wait that runs out leaves a code in the fault word, the CTA's other roles
// stop at their next wait, copies in flight get time to land, the host is told, the TMEM is freed.
#include <type_traits>

#include "ragged.cuh"
#include "tc_ptx.cuh"

namespace mole {

constexpr int kREpiWarps = 16;
constexpr int kRThreads = 32 * (4 + kREpiWarps);         // producer, issuer, fixer, spare, epilogue
constexpr uint32_t kRABytes = 128 * 128;                 // 128 features x 128 bytes of the reduction
constexpr int kRMaxStages = 12;
constexpr uint32_t kRStripBytes = 1024;                  // per epilogue warp

struct RowsMaps {
  CUtensorMap w;        // K-major: 128 B x 128 features; N-major: 64 features x 64 of the reduction
  CUtensorMap x[4];     // 128 B x {64, 32, 16, 8} rows
};
struct RowsParams {
  const int32_t* offsets;
  const float* x_scale;
  const float* w_scale;
  void* out;
  int32_t* fault;
  int R, N, E;
  int nkb;              // stages of the reduction
  int panel_shift;      // a panel has at most 2^panel_shift rows
  int sorted;           // experts in the order of their row counts (more items than pairs of CTAs)
  int wide;             // rows of out are multiples of 16 bytes, its base too
  int stages;
  uint32_t stage_bytes;
};

// The experts, where there are more items than pairs in the order of falling row counts: the round-robin
// deal of the items gives every pair its share of large and of small ones.
struct RowsOrder {
  int row0[kMaxRaggedExperts + 3];       // as RaggedSpans
  int tile0[kMaxRaggedExperts + 3];
  int start[kMaxRaggedExperts + 1];      // panels before the i-th expert of the order
  uint8_t order[kMaxRaggedExperts];
};
struct RowsItem {
  int valid;
  int e, f0;             // expert, first of the pair's 256 or 512 features
  int row0, rows, n;     // panel: first row, rows, columns of the accumulator
};

template <int STEP, int FB>
__device__ __forceinline__ RowsItem rows_item(const RowsOrder& o, int E, int nb, int item) {
  RowsItem w;
  w.valid = 0;
  if (item >= o.start[E] * nb) return w;
  int lo = 0, hi = E;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (o.start[mid] * nb <= item) lo = mid; else hi = mid;
  }
  const unsigned np = o.start[lo + 1] - o.start[lo], local = item - o.start[lo] * nb;
  const unsigned blk = local / np;         // panels of a feature block are neighbours: they share weights through L2
  const int pan = local - blk * np;
  const int e = o.order[lo];
  const int b = o.row0[e + 1], cnt = o.row0[e + 2] - b;
  const int per = ((cnt + np - 1) / np + STEP - 1) / STEP * STEP;
  w.valid = 1;
  w.e = e;
  w.f0 = blk * FB;
  w.row0 = b + pan * per;
  w.rows = min(per, cnt - pan * per);      // may be <= 0 for a last panel: nothing to do
  w.n = (max(w.rows, 0) + STEP - 1) / STEP * STEP;
  return w;
}

__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\n"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                                  int32_t* fault, int code) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  if (!mbar_wait(bar, parity, abort_flag, fault, code)) return false;
  return mbar_try_wait_cluster(bar, parity) || true;      // completed: this one orders what the peer wrote
}
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ bool warp_all_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* fault, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, fault, code));
}
// after an abort: loads already issued take microseconds to land; they get 20 ms
__device__ __forceinline__ void settle() {
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 20000000ull) __nanosleep(1000);
}
__device__ __forceinline__ void tcgen05_mma2_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                                uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// Zeros into the rows that belong to nobody, by the epilogue warps of all CTAs
template <typename TO>
__device__ __forceinline__ void zero_rows(TO* out, int r0, int r1, int N, int worker, int workers, int lane) {
  for (int r = r0 + worker; r < r1; r += workers)
    for (int n = lane; n < N; n += 32) out[(int64_t)r * N + n] = Elem<TO>::from_f(0.f);
}

// One chunk of 16 rows x 32 features of a warp, bf16: turned round through a 1 KB strip so that a
// lane stores eight neighbouring features of two rows.  Word (rp, l) of the strip holds rows 2 rp
// and 2 rp + 1 of feature l, at rp * 32 + (l ^ 4 (rp & 1)): no bank conflicts on either side.
__device__ __forceinline__ void store_chunk(__nv_bfloat16* out, const float (&v)[16], uint32_t* strip, int row, int rows_left,
                                            int f_warp, int N, int lane) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) strip[32 * i + (lane ^ ((i & 1) << 2))] = two_bf16(v[2 * i], v[2 * i + 1]);
  __syncwarp();
  const int rp = lane >> 2, g = lane & 3;
  const uint4* s4 = reinterpret_cast<const uint4*>(strip);
  const uint4 lo = s4[rp * 8 + 2 * g + (rp & 1)], hi = s4[rp * 8 + 2 * g + 1 - (rp & 1)];
  const int f = f_warp + 8 * g;
  if (f < N) {
    __nv_bfloat16* d = out + (int64_t)(row + 2 * rp) * N + f;
    if (2 * rp < rows_left)
      *reinterpret_cast<uint4*>(d) = make_uint4(__byte_perm(lo.x, lo.y, 0x5410), __byte_perm(lo.z, lo.w, 0x5410),
                                                __byte_perm(hi.x, hi.y, 0x5410), __byte_perm(hi.z, hi.w, 0x5410));
    if (2 * rp + 1 < rows_left)
      *reinterpret_cast<uint4*>(d + N) = make_uint4(__byte_perm(lo.x, lo.y, 0x7632), __byte_perm(lo.z, lo.w, 0x7632),
                                                    __byte_perm(hi.x, hi.y, 0x7632), __byte_perm(hi.z, hi.w, 0x7632));
  }
}

template <bool I8, bool KN, bool DUAL, typename TO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kRThreads, 1)
ragged_rows_tc_kernel(const __grid_constant__ RowsMaps maps, const __grid_constant__ RowsParams p) {
  static_assert(!(I8 && KN), "integers are read K-major");
  constexpr int STEP = I8 ? 32 : 16;             // columns of the accumulator come in these steps
  constexpr int KB = I8 ? 128 : 64;              // elements of the reduction per stage
  constexpr int NA = DUAL ? 2 : 1;               // blocks of 256 features per item
  constexpr int FB = 256 * NA;
  constexpr uint32_t kABytes = NA * kRABytes;
  constexpr uint32_t kIdesc = ((I8 ? 2u : 1u) << 4) | (1u << 7) | (1u << 10) | ((KN ? 1u : 0u) << 15) |
                              ((uint32_t)(256 >> 4) << 24);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ __align__(8) uint64_t bars[2 * kRMaxStages + 5];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_flag_s;
  __shared__ RowsOrder ord;
  __shared__ __align__(16) uint32_t strips[kREpiWarps][kRStripBytes / 4];
  __shared__ __align__(16) float scales[I8 ? kREpiWarps : 1][64];       // of the rows a warp stores
  volatile int* abort_flag = &abort_flag_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[kRMaxStages]);
  const uint32_t tfull0 = smem_u32(&bars[2 * kRMaxStages]), tempty0 = smem_u32(&bars[2 * kRMaxStages + 2]);
  const uint32_t drain0 = smem_u32(&bars[2 * kRMaxStages + 4]);
  const uint32_t smem_base = smem_u32(smem);
  const int cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;
  const int E = p.E, nb = (p.N + FB - 1) / FB;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_s)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 64) {
    abort_flag_s = 0;
    mbar_init(drain0, 1);
    for (int s = 0; s < kRMaxStages; ++s) {
      mbar_init(full0 + 8 * s, 1);                  // the even CTA's arrive.expect_tx
      mbar_init(empty0 + 8 * s, 1);                 // a commit that arrives in both CTAs
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull0 + 8 * a, 1);
      mbar_init(tempty0 + 8 * a, 2 * kREpiWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  after_previous();
  if (warp == 0) load_spans(*reinterpret_cast<RaggedSpans*>(&ord), p.offsets, E, p.R, p.panel_shift);
  if (p.sorted) {
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRThreads) {
      const int mine = ord.row0[e + 2] - ord.row0[e + 1];
      int rk = 0;
      for (int o = 0; o < E; ++o) {
        const int other = ord.row0[o + 2] - ord.row0[o + 1];
        rk += (other > mine) || (other == mine && o < e);
      }
      ord.order[rk] = (uint8_t)e;
    }
    __syncthreads();
    if (warp == 0) {                                  // panels before the i-th expert of the order
      int base = 0;
      for (int i0 = 0; i0 < E; i0 += 32) {
        const int i = i0 + lane;
        int v = 0;
        if (i < E) { const int e = ord.order[i]; v = ord.tile0[e + 2] - ord.tile0[e + 1]; }
        int incl = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, incl, d);
          if (lane >= d) incl += u;
        }
        if (i < E) ord.start[i] = base + incl - v;
        base += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) ord.start[E] = base;
    }
  } else if (warp == 0) {
    __syncwarp();
    for (int i = lane; i <= E; i += 32) {
      ord.start[i] = ord.tile0[i + 1] - ord.tile0[1];
      if (i < E) ord.order[i] = (uint8_t)i;
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_arrive_all();
  const RowsItem first = rows_item<STEP, FB>(ord, E, nb, cluster_id);
  cluster_wait_all();                               // barriers initialised, TMEM addresses there, in both CTAs
  tcgen05_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  if (warp == 0) {
    // ---- TMA producer (both CTAs; every box has its own lane) ----
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    RowsItem w = first;
    for (int item = cluster_id; ok && w.valid; w = rows_item<STEP, FB>(ord, E, nb, item += n_clusters)) {
      if (w.n == 0) continue;
      const int h = w.n >> 1;                       // rows that this CTA stages
      const uint32_t tx = 2u * (kABytes + (uint32_t)h * 128u);
      const int f0 = w.f0 + 128 * (int)rank;
      const int wbox = lane < 2 ? lane : lane < 7 ? 99 : lane - 5;        // lanes 0, 1, 7, 8: boxes of the weights
      int kind = -1, off = 0;                       // lanes 2..6: the panel's rows in boxes of 64, 64, 32, 16, 8
      {
        const int n64 = h >> 6, rem = h & 63;
        if (lane == 2 || lane == 3) { if (lane - 2 < n64) { kind = 0; off = 64 * (lane - 2); } }
        else if (lane == 4) { if (rem & 32) { kind = 1; off = 64 * n64; } }
        else if (lane == 5) { if (rem & 16) { kind = 2; off = 64 * n64 + (rem & 32); } }
        else if (lane == 6) { if (rem & 8) { kind = 3; off = 64 * n64 + (rem & 48); } }
      }
      const int srow = w.row0 + h * (int)rank + off;
      for (int kb = 0; kb < p.nkb; ++kb) {
        ok = warp_all_wait(empty0 + 8 * stage, phase ^ 1, abort_flag, p.fault, 61);
        if (!ok) break;
        const uint32_t bar = (full0 + 8 * stage) & kPeerMask;      // the even CTA's
        const uint32_t sa = smem_base + stage * p.stage_bytes, sb = sa + kABytes;
        if (rank == 0 && lane == 0) mbar_expect_tx(full0 + 8 * stage, tx);
        if (KN) {
          if (wbox < 2 * NA)
            tma2_load_3d(sa + wbox * (kRABytes / 2), &maps.w, bar, f0 + 64 * (wbox & 1) + 256 * (wbox >> 1), kb * KB, w.e);
        } else {
          if (wbox < NA) tma2_load_3d(sa + wbox * kRABytes, &maps.w, bar, kb * KB, f0 + 256 * wbox, w.e);
        }
        if (kind >= 0) tma2_load_2d(sb + off * 128, &maps.x[kind], bar, kb * KB, srow);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer (even CTA) ----
    if (lane == 0 && rank == 0) {
      int stage = 0, half = 0;
      uint32_t phase = 0, hph = 0;                  // hph: bit h = parity of the uses of TMEM half h so far
      bool ok = true;
      RowsItem w = first;
      for (int item = cluster_id; ok && w.valid; w = rows_item<STEP, FB>(ord, E, nb, item += n_clusters)) {
        if (w.n == 0) continue;
        const bool both = DUAL && w.n > 128;
        const int h0 = both ? 0 : half;
        if (!(ok = mbar_wait(tempty0 + 8 * h0, ((hph >> h0) & 1u) ^ 1u, abort_flag, p.fault, 62))) break;
        tcgen05_fence_after();
        const uint32_t d0 = tmem_base + 256 * h0, d1 = d0 + (both ? 256 : 128);
        const uint32_t idesc = kIdesc | ((uint32_t)(w.n >> 3) << 17);
        auto mma = [&](int at_stage, int ks, int blk, int kb) {      // 32 bytes of the reduction
          const uint32_t sa = smem_base + at_stage * p.stage_bytes, at = sa + blk * kRABytes;
          const uint64_t ad = KN ? make_desc(at + ks * (16 * 128), kRABytes / 2, 1024) : make_desc(at + ks * 32, 16, 1024);
          const uint64_t bd = make_desc(sa + kABytes + ks * 32, 16, 1024);
          if (I8) tcgen05_mma2_i8(blk ? d1 : d0, ad, bd, idesc, (kb | ks) ? 1u : 0u);
          else tcgen05_mma2_bf16(blk ? d1 : d0, ad, bd, idesc, (kb | ks) ? 1u : 0u);
        };
        int kb = 0;
        if (both) {
          // The epilogue of the item before drains the first accumulator, then the second: until that
          // is free, the ring's stages go into the first one only, and into the second afterwards.
          const int ahead = min(p.stages, p.nkb);
          int st = stage;
          uint32_t ph = phase;
          for (int i = 0; ok && i < ahead; ++i) {
            if (!(ok = mbar_wait(full0 + 8 * st, ph, abort_flag, p.fault, 63))) break;
            tcgen05_fence_after();
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) mma(st, ks, 0, i);
            if (++st == p.stages) { st = 0; ph ^= 1; }
          }
          if (!ok || !(ok = mbar_wait(tempty0 + 8, ((hph >> 1) & 1u) ^ 1u, abort_flag, p.fault, 62))) break;
          tcgen05_fence_after();
          for (; kb < ahead; ++kb) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) mma(stage, ks, 1, kb);
            tcgen05_commit2(empty0 + 8 * stage);
            if (++stage == p.stages) { stage = 0; phase ^= 1; }
          }
        }
        for (; kb < p.nkb; ++kb) {
          if (!(ok = mbar_wait(full0 + 8 * stage, phase, abort_flag, p.fault, 63))) break;
          tcgen05_fence_after();
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int blk = 0; blk < NA; ++blk) mma(stage, ks, blk, kb);
          tcgen05_commit2(empty0 + 8 * stage);
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tcgen05_commit2(tfull0 + 8 * h0);
        if (both) tcgen05_commit2(tfull0 + 8);
        hph ^= both ? 3u : 1u << h0;
        if (!both) half ^= 1;
      }
      if (*abort_flag) {
        tcgen05_commit2(drain0);
        mbar_drain(drain0, 0, globaltimer_ns() + 200000000ull);
      }
    }
  } else if (warp >= 4) {
    // ---- epilogue (both CTAs): warp -> 32 features (the TMEM lanes it may read), every fourth chunk of 16 rows ----
    const int quarter = warp & 3, grp = (warp - 4) >> 2;
    uint32_t* strip = strips[warp - 4];
    TO* out = static_cast<TO*>(p.out);
    {
      const int worker = blockIdx.x * kREpiWarps + warp - 4, workers = gridDim.x * kREpiWarps;
      zero_rows(out, 0, ord.row0[1], p.N, worker, workers, lane);
      zero_rows(out, ord.row0[E + 1], p.R, p.N, worker, workers, lane);
    }
    int half = 0;
    uint32_t hph = 0;
    RowsItem w = first;
    for (int item = cluster_id; w.valid; w = rows_item<STEP, FB>(ord, E, nb, item += n_clusters)) {
      if (w.n == 0) continue;
      const bool both = DUAL && w.n > 128;
      const int h0 = both ? 0 : half;
      if (I8) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 2; ++j) {               // entry 16 q + i: row 64 q + 16 grp + i of the panel
          const int at = 32 * j + lane, row = (at >> 4) * 64 + grp * 16 + (at & 15);
          scales[warp - 4][at] = row < w.rows ? p.x_scale[w.row0 + row] : 0.f;
        }
        __syncwarp();
      }
      bool ok = true;
#pragma unroll 1
      for (int blk = 0; blk < NA; ++blk) {
        const int h = both ? blk : h0;
        const int f_warp = w.f0 + 256 * blk + 128 * (int)rank + 32 * quarter, f = f_warp + lane;
        float ws = 0.f;
        if (I8 && f < p.N) ws = p.w_scale[(int64_t)w.e * p.N + f];
        if (both || blk == 0) {
          if (!(ok = warp_all_wait(tfull0 + 8 * h, (hph >> h) & 1u, abort_flag, p.fault, 64))) break;
          tcgen05_fence_after();
        }
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + 256 * h + (both ? 0 : 128 * blk);
        for (int c = grp * 16; c < w.rows; c += 64) {
          uint32_t r[16];
          tmem_ld16(taddr + c, r);
          tmem_ld_wait();
          const int left = w.rows - c;              // rows of the chunk that exist: 1 .. 16 and more
          float v[16];
          if (I8) {
            const float4* sc = reinterpret_cast<const float4*>(&scales[warp - 4][(c >> 6) * 16]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 x = sc[i];
              v[4 * i] = __fmul_rn(__fmul_rn((float)(int)r[4 * i], x.x), ws);
              v[4 * i + 1] = __fmul_rn(__fmul_rn((float)(int)r[4 * i + 1], x.y), ws);
              v[4 * i + 2] = __fmul_rn(__fmul_rn((float)(int)r[4 * i + 2], x.z), ws);
              v[4 * i + 3] = __fmul_rn(__fmul_rn((float)(int)r[4 * i + 3], x.w), ws);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
          }
          if constexpr (sizeof(TO) == 2) {
            if (p.wide) {
              store_chunk(out, v, strip, w.row0 + c, left, f_warp, p.N, lane);
              continue;
            }
          }
          if (f < p.N) {
            TO* d = out + (int64_t)(w.row0 + c) * p.N + f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (i < left) d[(int64_t)i * p.N] = Elem<TO>::from_f(v[i]);
          }
        }
        if (both || blk == NA - 1) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster((tempty0 + 8 * h) & kPeerMask);
        }
      }
      if (!ok) break;
      hph ^= both ? 3u : 1u << h0;
      if (!both) half ^= 1;
    }
  }

  __syncwarp();
  if (*abort_flag) settle();
  __syncwarp();
  tcgen05_fence_before();
  cluster_meet();              // nobody leaves while the peer may still touch its shared memory
  if (threadIdx.x == 0 && *abort_flag) report_fault(p.fault);      // whichever warp's wait it was
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ---- weight gradient ---------------------------------------------------------------------------------
constexpr int kWStages = 6;
constexpr uint32_t kWHalfBytes = 128 * 128;              // 128 columns x 64 rows of one operand, two boxes
constexpr uint32_t kWStageBytes = 2 * kWHalfBytes;
constexpr uint32_t kWBoxBytes = 64 * 128;                // 64 columns x 64 rows
constexpr uint32_t kWStripBytes = 32 * 64;               // per epilogue warp: 32 rows x 32 columns on their way out

struct WgradParams {
  const int32_t* offsets;
  __nv_bfloat16* out;
  int32_t* fault;
  int R, P, Q, E;
  int wide;             // rows of out are multiples of 16 bytes, its base too
  int sorted;           // experts in the order of their row counts
  int split;            // an expert's rows are cut into so many parts,
  float* part;          // with a result [E, P, Q] each (split > 1)
};
struct WgradOrder {
  int row0[kMaxRaggedExperts + 3];
  uint8_t order[kMaxRaggedExperts];      // experts, by falling row counts where there are more items than pairs
};
struct WgradItem {
  int valid, e, p0, q0, row0, rows, part;
};
__device__ __forceinline__ WgradItem wgrad_item(const WgradOrder& o, const WgradParams& p, int item) {
  WgradItem w;
  const unsigned qb = (p.Q + 255) / 256, per = (p.P + 255) / 256 * qb * p.split;
  w.valid = item < p.E * (int)per;
  if (!w.valid) return w;
  const unsigned i = item / per, r = item - i * per, tile = r / p.split, pb = tile / qb;
  w.e = o.order[i];
  w.part = r - tile * p.split;
  w.p0 = pb * 256;
  w.q0 = (tile - pb * qb) * 256;
  w.row0 = o.row0[w.e + 1];
  w.rows = o.row0[w.e + 2] - w.row0;
  if (p.split > 1) {
    const int share = (w.rows + p.split * 64 - 1) / (p.split * 64) * 64;
    w.row0 += w.part * share;
    w.rows = max(0, min(share, w.rows - w.part * share));
  }
  return w;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kRThreads, 1)
ragged_wgrad_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                       const __grid_constant__ CUtensorMap map_out, const __grid_constant__ WgradParams p) {
  constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) |
                              ((uint32_t)(256 >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ __align__(8) uint64_t bars[3 * kWStages + 5];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_flag_s;
  __shared__ WgradOrder ord;
  volatile int* abort_flag = &abort_flag_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[kWStages]), part0 = smem_u32(&bars[2 * kWStages]);
  const uint32_t tfull0 = smem_u32(&bars[3 * kWStages]), tempty0 = smem_u32(&bars[3 * kWStages + 2]);
  const uint32_t drain0 = smem_u32(&bars[3 * kWStages + 4]);
  const uint32_t smem_base = smem_u32(smem);
  const int cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;
  const int E = p.E;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_s)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 64) {
    abort_flag_s = 0;
    mbar_init(drain0, 1);
    for (int s = 0; s < kWStages; ++s) {
      mbar_init(full0 + 8 * s, 2);                  // one arrival of either CTA
      mbar_init(empty0 + 8 * s, 1);
      mbar_init(part0 + 8 * s, 1);                  // this CTA's loads of a stage that the fixer takes
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull0 + 8 * a, 1);
      mbar_init(tempty0 + 8 * a, kREpiWarps);       // eight warps of either CTA
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  after_previous();
  // (the spans' tiles, which this kernel has no use for, lie where the ring will be)
  RaggedSpans& spans = *reinterpret_cast<RaggedSpans*>(smem);
  if (warp == 0) load_spans(spans, p.offsets, E, p.R, 8);
  __syncthreads();
  if (threadIdx.x < E + 3) ord.row0[threadIdx.x] = spans.row0[threadIdx.x];
  for (int e = threadIdx.x; e < E; e += kRThreads) {
    int rk = e;
    if (p.sorted) {
      const int mine = spans.row0[e + 2] - spans.row0[e + 1];
      rk = 0;
      for (int o = 0; o < E; ++o) {
        const int other = spans.row0[o + 2] - spans.row0[o + 1];
        rk += (other > mine) || (other == mine && o < e);
      }
    }
    ord.order[rk] = (uint8_t)e;
  }
  fence_async_proxy();                              // the ring's first loads overwrite the spans
  tcgen05_fence_before();
  __syncthreads();
  cluster_arrive_all();
  const WgradItem first = wgrad_item(ord, p, cluster_id);
  cluster_wait_all();
  tcgen05_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  if (warp == 0) {
    // ---- TMA producer: lanes 0, 1 the boxes of a, lanes 2, 3 those of b ----
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    WgradItem w = first;
    for (int item = cluster_id; ok && w.valid; w = wgrad_item(ord, p, item += n_clusters)) {
      const int c0 = (lane < 2 ? w.p0 : w.q0) + 128 * (int)rank + 64 * (lane & 1);
      for (int r = 0; r < w.rows; r += 64) {
        ok = warp_all_wait(empty0 + 8 * stage, phase ^ 1, abort_flag, p.fault, 71);
        if (!ok) break;
        const uint32_t dst = smem_base + stage * kWStageBytes + lane * kWBoxBytes;
        if (w.rows - r < 64 && (w.rows & 15) != 0) {
          // a stage for the fixer: this CTA's boxes land on its own barrier, the fixer arrives
          if (lane == 0) mbar_expect_tx(part0 + 8 * stage, kWStageBytes);
          __syncwarp();
          if (lane < 4) tma_load_2d(dst, lane < 2 ? &map_a : &map_b, part0 + 8 * stage, c0, w.row0 + r);
        } else {
          const uint32_t bar = (full0 + 8 * stage) & kPeerMask;
          if (lane == 0) {
            if (rank == 0) mbar_expect_tx(full0 + 8 * stage, 2u * kWStageBytes);
            else mbar_arrive_cluster(bar);
          }
          __syncwarp();
          if (lane < 4) tma2_load_2d(dst, lane < 2 ? &map_a : &map_b, bar, c0, w.row0 + r);
        }
        if (++stage == kWStages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer (even CTA) ----
    if (lane == 0 && rank == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      WgradItem w = first;
      for (int item = cluster_id; ok && w.valid; w = wgrad_item(ord, p, item += n_clusters)) {
        if (w.rows == 0) continue;
        if (!(ok = mbar_wait(tempty0 + 8 * acc, acc_phase ^ 1, abort_flag, p.fault, 72))) break;
        tcgen05_fence_after();
        const uint32_t d_tmem = tmem_base + 256 * acc;
        for (int r = 0; r < w.rows; r += 64) {
          if (!(ok = mbar_wait_cluster(full0 + 8 * stage, phase, abort_flag, p.fault, 73))) break;
          tcgen05_fence_after();
          const uint32_t sa = smem_base + stage * kWStageBytes, sb = sa + kWHalfBytes;
          auto mma = [&](int ks) {
            tcgen05_mma2_bf16(d_tmem, make_desc(sa + ks * (16 * 128), kWBoxBytes, 1024),
                              make_desc(sb + ks * (16 * 128), kWBoxBytes, 1024), kIdesc, (r | ks) ? 1u : 0u);
          };
          const int left = w.rows - r;
          if (left >= 64) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) mma(ks);
          } else {
            for (int ks = 0; ks * 16 < left; ++ks) mma(ks);
          }
          tcgen05_commit2(empty0 + 8 * stage);
          if (++stage == kWStages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tcgen05_commit2(tfull0 + 8 * acc);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      if (*abort_flag) {
        tcgen05_commit2(drain0);
        mbar_drain(drain0, 0, globaltimer_ns() + 200000000ull);
      }
    }
  } else if (warp == 2) {
    // ---- fixer (both CTAs): zeros over the rows of others in an expert's last 16-row step ----
    int stage = 0;
    uint32_t seen = 0;                              // bit s: parity of the uses of part0[s] so far
    WgradItem w = first;
    for (int item = cluster_id; w.valid; w = wgrad_item(ord, p, item += n_clusters)) {
      if (w.rows == 0) continue;
      const int n = (w.rows + 63) / 64;
      const int last = (stage + n - 1) % kWStages;
      stage = (stage + n) % kWStages;
      if ((w.rows & 15) == 0) continue;
      if (!warp_all_wait(part0 + 8 * last, (seen >> last) & 1u, abort_flag, p.fault, 74)) break;
      seen ^= 1u << last;
      const int valid = (w.rows - 1) % 64 + 1, end = (valid + 15) & ~15;
      // a box's row is 128 bytes; four boxes; the swizzle moves 16-byte pieces within a row only
      const int pieces = (end - valid) * 8;
      uint8_t* base = smem + last * kWStageBytes + valid * 128;
      for (int i = lane; i < 4 * pieces; i += 32)
        *reinterpret_cast<uint4*>(base + (i / pieces) * kWBoxBytes + (i % pieces) * 16) = make_uint4(0, 0, 0, 0);
      fence_async_proxy();                          // the tensor cores read through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive_release_cluster((full0 + 8 * last) & kPeerMask);
    }
  } else if (warp >= 4) {
    // ---- epilogue (both CTAs): warp -> 32 rows of the gradient and 128 columns of every second item ----
    // (the two accumulators have eight warps each: a warp's way from TMEM to memory takes longer than an
    // item's MMAs, and so two of them are under way)
    const int quarter = warp & 3, grp = ((warp - 4) >> 2) & 1, acc = (warp - 4) >> 3;
    uint8_t* strip = smem + kWStages * kWStageBytes + (warp - 4) * kWStripBytes;
    int turn = 0;
    uint32_t acc_phase = 0;
    WgradItem w = first;
    for (int item = cluster_id; w.valid; w = wgrad_item(ord, p, item += n_clusters)) {
      const bool empty = w.rows == 0;               // no rows: the gradient is zero
      if (empty ? ((item / n_clusters) & 1) != acc : turn != acc) {
        if (!empty) turn ^= 1;
        continue;
      }
      if (!empty) {
        turn ^= 1;
        if (!warp_all_wait(tfull0 + 8 * acc, acc_phase, abort_flag, p.fault, 75)) break;
        tcgen05_fence_after();
        acc_phase ^= 1;
      }
      const int prow = w.p0 + 128 * (int)rank + 32 * quarter;     // of lane 0
#pragma unroll 1
      for (int part = 0; part < 4; ++part) {
        const int col = 128 * grp + 32 * part, qcol = w.q0 + col;
        uint32_t o[16];
        uint32_t r[2][16];
        if (!empty) {
          const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + 256 * acc + col;
          tmem_ld16(taddr, r[0]);
          tmem_ld16(taddr + 16, r[1]);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            o[i] = two_bf16(__uint_as_float(r[i >> 3][2 * (i & 7)]), __uint_as_float(r[i >> 3][2 * (i & 7) + 1]));
          if (part == 3) {
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster((tempty0 + 8 * acc) & kPeerMask);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) r[0][i] = r[1][i] = o[i] = 0u;
        }
        if (p.split > 1) {
          if (prow + lane < p.P) {
            float* d = p.part + (((int64_t)w.part * p.E + w.e) * p.P + prow + lane) * p.Q + qcol;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const uint32_t* v = &r[i >> 4][i & 15];
              if (p.Q % 4 == 0) {                   // (the parts start on 256 bytes)
                if (qcol + i < p.Q) *reinterpret_cast<uint4*>(d + i) = make_uint4(v[0], v[1], v[2], v[3]);
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (qcol + i + j < p.Q) d[i + j] = __uint_as_float(v[j]);
              }
            }
          }
        } else if (p.wide) {
          // 32 rows x 64 bytes, 16-byte pieces swizzled as the map says, and off by one TMA store, which
          // leaves out what lies beyond the expert's matrix
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(strip + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          fence_async_proxy();
          __syncwarp();
          if (lane == 0 && prow < p.P && qcol < p.Q) {
            asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                         ::"l"(&map_out), "r"(smem_u32(strip)), "r"(qcol), "r"(prow), "r"(w.e) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          // rows of the gradient at any address: turned round in the strip, so that a store instruction
          // writes 32 neighbouring columns of one row
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(strip + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          __syncwarp();
          if (qcol + lane < p.Q) {
            __nv_bfloat16* d = p.out + ((int64_t)w.e * p.P + prow) * p.Q + qcol + lane;
            for (int i = 0; i < 32 && prow + i < p.P; ++i)
              d[(int64_t)i * p.Q] = *reinterpret_cast<const __nv_bfloat16*>(
                  strip + i * 64 + (((lane >> 3) ^ ((i >> 1) & 3)) << 4) + 2 * (lane & 7));
          }
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  __syncwarp();
  if (*abort_flag) settle();
  __syncwarp();
  tcgen05_fence_before();
  cluster_meet();
  if (threadIdx.x == 0 && *abort_flag) report_fault(p.fault);      // whichever warp's wait it was
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

constexpr size_t kRBudget = 192 * 1024 + 1024;           // dynamic shared memory, next to the static 22 KB

// ---- host side ---------------------------------------------------------------------------------------
// Pairs of CTAs that are resident at once with the kernel's largest shared memory
template <typename Kern>
static int resident_pairs(Kern kern, size_t smem, PerDeviceInt& cache, int* pairs) {
  const int dev = current_device();
  int n = (int)cache.get(dev);
  if (n == 0) {
    MOLE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (sm_count() / 2));
    cfg.blockDim = dim3(kRThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = sm_count() / 2;
    }
    cache.set(dev, n);
  }
  *pairs = n;
  return MOLE_OK;
}


template <bool I8, bool KN, bool DUAL, typename TO>
static int launch_rows(const RowsMaps& maps, RowsParams p, int n_max, int64_t panels, cudaStream_t st) {
  auto kern = ragged_rows_tc_kernel<I8, KN, DUAL, TO>;
  constexpr int FB = DUAL ? 512 : 256;
  p.stage_bytes = (DUAL ? 2 : 1) * kRABytes + (uint32_t)(n_max / 2) * 128u;
  p.stages = (int)((kRBudget - 1024) / p.stage_bytes);
  if (p.stages > kRMaxStages) p.stages = kRMaxStages;
  const int64_t max_items = panels * ((p.N + FB - 1) / FB);
  static PerDeviceInt cache;
  int pairs = 0;
  if (int rc = resident_pairs(kern, kRBudget, cache, &pairs)) return rc;
  p.sorted = max_items > pairs;
  if (max_items < pairs) pairs = (int)max_items;
  const size_t smem = (size_t)p.stages * p.stage_bytes + 1024;
  return launch_early(kern, dim3(2 * pairs), kRThreads, smem, st, maps, p);
}

int ragged_rows_tc(int elem, int out_dtype, const RaggedRows& a, cudaStream_t st) {
  RowsMaps maps;
  const uint32_t kb = 128 / elem;
  for (int i = 0; i < 4; ++i) {
    const uint64_t dims[2] = {(uint64_t)a.K, (uint64_t)a.R};
    const uint32_t box[2] = {kb, (uint32_t)(64 >> i)};
    if (int rc = encode_map(&maps.x[i], a.x, 2, dims, box, elem, (uint64_t)a.ldx * elem)) return rc;
  }
  const uint64_t dims[3] = {(uint64_t)(a.kn ? a.N : a.K), (uint64_t)(a.kn ? a.K : a.N), (uint64_t)a.E};
  const uint32_t box_k[3] = {kb, 128, 1}, box_n[3] = {64, 64, 1};
  if (int rc = encode_map(&maps.w, a.w, 3, dims, a.kn ? box_n : box_k, elem, (uint64_t)a.ldw * elem)) return rc;
  RowsParams p{};
  p.offsets = a.offsets; p.x_scale = a.x_scale; p.w_scale = a.w_scale; p.out = a.out;
  p.fault = device_fault_word();
  MOLE_REQUIRE(p.fault != nullptr, "fault word not allocated");
  p.R = (int)a.R; p.N = a.N; p.E = a.E;
  p.nkb = (int)((a.K + kb - 1) / kb);
  const size_t osize = out_dtype == MOLE_F32 ? 4 : 2;
  p.wide = a.N * osize % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  // panels of 256 rows, of half as many as long as all items still run at once (1000 rows, 2048 -> 2000 in 8
  // bits: 64 items of 128 rows, 11.1 us; 32 of 256, 11.8)
  const int step = elem == 1 ? 32 : 16;
  auto panels_of = [&](int panel) { return a.R / panel + (a.E < a.R ? a.E : a.R); };  // every expert may end in a partial one
  int panel = 256;
  while (panel > 32 && panels_of(panel / 2) * ((a.N + 255) / 256) <= sm_count() / 2) panel /= 2;
  p.panel_shift = panel == 256 ? 8 : panel == 128 ? 7 : panel == 64 ? 6 : 5;
  const int64_t panels = panels_of(panel);
  // no panel has more rows than there are: few rows leave the shared memory to more stages
  const int n_max = a.R >= panel ? panel : (int)((a.R + step - 1) / step * step);
  // 512 features per item where that still leaves every pair two items or so, and the last block is not
  // mostly empty: 64 experts of 256 rows, 8192 -> 2048: 0.49 ms, with 256 features 0.63; 1000 rows of one
  // expert, 2048 -> 2000 in 8 bits: 20 us, with 256 features 13
  const bool dual = panels * ((a.N + 511) / 512) >= sm_count() && (a.N % 512 == 0 || a.N > 1024);
  auto launch = [&](auto two) {
    constexpr bool D = decltype(two)::value;
    if (elem == 1) {
      if (out_dtype == MOLE_F32) return launch_rows<true, false, D, float>(maps, p, n_max, panels, st);
      return launch_rows<true, false, D, __nv_bfloat16>(maps, p, n_max, panels, st);
    }
    if (a.kn) return launch_rows<false, true, D, __nv_bfloat16>(maps, p, n_max, panels, st);
    return launch_rows<false, false, D, __nv_bfloat16>(maps, p, n_max, panels, st);
  };
  return dual ? launch(std::true_type()) : launch(std::false_type());
}

int ragged_wgrad_tc(const RaggedWgrad& a, cudaStream_t st) {
  CUtensorMap ma, mb;
  const uint32_t box[2] = {64, 64};
  const uint64_t da[2] = {(uint64_t)a.P, (uint64_t)a.R}, db[2] = {(uint64_t)a.Q, (uint64_t)a.R};
  if (int rc = encode_map(&ma, a.a, 2, da, box, 2, (uint64_t)a.lda * 2)) return rc;
  if (int rc = encode_map(&mb, a.b, 2, db, box, 2, (uint64_t)a.ldb * 2)) return rc;
  WgradParams p{};
  p.offsets = a.offsets;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.fault = device_fault_word();
  MOLE_REQUIRE(p.fault != nullptr, "fault word not allocated");
  p.R = (int)a.R; p.P = a.P; p.Q = a.Q; p.E = a.E;
  p.wide = a.Q % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  constexpr size_t smem = (size_t)kWStages * kWStageBytes + kREpiWarps * kWStripBytes + 1024;
  static PerDeviceInt cache;
  int pairs = 0;
  if (int rc = resident_pairs(ragged_wgrad_tc_kernel, smem, cache, &pairs)) return rc;
  p.split = a.split;
  p.part = a.part;
  const int64_t items = (int64_t)a.E * a.split * ((a.P + 255) / 256) * ((a.Q + 255) / 256);
  MOLE_REQUIRE(items < (1ll << 31), "%d experts of %d x %d", a.E, a.P, a.Q);
  p.sorted = items > pairs;
  if (items < pairs) pairs = (int)items;
  CUtensorMap mo = ma;
  if (p.wide) {
    const uint64_t dims[3] = {(uint64_t)a.Q, (uint64_t)a.P, (uint64_t)a.E};
    const uint32_t box_out[3] = {32, 32, 1};
    if (int rc = encode_map(&mo, a.out, 3, dims, box_out, 2)) return rc;
  }
  if (int rc = launch_early(ragged_wgrad_tc_kernel, dim3(2 * pairs), kRThreads, smem, st, ma, mb, mo, p)) return rc;
  return a.split > 1 ? ragged_join(MOLE_BF16, a.part, a.split, (int64_t)a.E * a.P * a.Q, a.out, st) : MOLE_OK;
}

}  // namespace mole

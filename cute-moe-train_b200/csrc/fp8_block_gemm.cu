// Grouped e4m3 GEMM with a scale for each block of 128 (ragged M), three fused epilogues.
//
//   acc[r, c] = sum over blocks b of 128 along k:  sa[r, b] * sb[e, b, c / 128] * (A[r, b] . B[e, b, c])
//   MGF_EPI_BIAS        D = bf16(acc + bias[e])
//   MGF_EPI_SWIGLU      aux = bf16(acc + bias[e]), D2 = clamped SwiGLU(aux)
//   MGF_EPI_SWIGLU_BWD  D = SwiGLU_bwd(acc, aux)
//
// Two forms, chosen on the device by what the scales are (pack_scales_kernel):
//
//   gemm_kernel   any fp32 scales.  They change every 128 elements of k, so the tensor cores cannot keep one accumulator over
//                 the whole contraction: each block's product goes into a TMEM buffer (4 tcgen05.mma of K = 32), and the
//                 epilogue warps add it, scaled, to fp32 accumulators in registers while the next block is multiplied into
//                 another buffer.  A thread owns one row and 128 columns (one scale block) of the 128 x 256 tile, so the
//                 factor sa * sb is one scalar per thread and block and the promotion one FMA per element.  Bound by the
//                 buffers' way round (about 1000 clocks a block against 512 of its MMAs): 1.7 PFLOP/s at 16384 rows in 4
//                 groups, n = 5760, k = 2880.  Few rows: the weights' bytes.
//   mx_kernel     powers of two.  The tensor cores apply the scales and the accumulator stays in TMEM: 2.3 PFLOP/s at the
//                 same sizes, bound by the products' issue and shared-memory traffic (operands written and read) and,
//                 sustained, by the power cap: 98304 x 2880 x 5760 with SwiGLU over 32 experts 1480 us in short bursts,
//                 1680-1740 back to back (1.9 PFLOP/s), as long as with one scale per row in the same run.  128 rows over
//                 256 experts, n = 4096, k = 7168: 250 us, 5.9 TB/s of weights.
//
// B is read as stored, [E, k, n] with unit stride along n (the weights' own layout: MN-major operand) or along
// k (the transposed view, the input gradient), so one set of codes serves both.  Warp roles, CTA pairs,
// tile order, bounded waits and the handling of malformed offs are those of moe_gemm_sm100.cu.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <mutex>

#include "drain.cuh"
#include "epilogue.cuh"
#include "host.h"
#include "moe_gemm.h"
#include "ptx.cuh"

namespace mgf {
namespace block_gemm {

constexpr int BM = 128;             // rows of A per CTA
constexpr int BK = 128;             // elements (= bytes) of k per stage = one scale block
constexpr int kMaxGroups = 1024;
constexpr int kNumEpiWarps = 8;     // two warpgroups, each half of the tile's columns
constexpr int kThreads = 64 + 32 * kNumEpiWarps;
constexpr uint64_t kWaitLimitNs = 1500ull * 1000ull * 1000ull;  // 1.5 s per pipeline wait

template <int BN, int CG>
struct Cfg {
  static constexpr int A_BYTES = BM * BK;
  static constexpr int BNC = BN / CG;  // columns of B held by this CTA
  static constexpr int B_BYTES = BNC * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int BAR_BYTES = 512;
  static constexpr int SCHED_BYTES = 3 * 4 * (kMaxGroups + 1);
  static constexpr int TAIL_BYTES = (BAR_BYTES + SCHED_BYTES + 1023) / 1024 * 1024;
  static constexpr int BUDGET = 227 * 1024 - 1024 - TAIL_BYTES;
  static constexpr int STAGES = BUDGET / STAGE_BYTES > 8 ? 8 : BUDGET / STAGE_BYTES;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + TAIL_BYTES;
  // TMEM buffers: a buffer is away for about 1300 clocks around its products (commit, wake-up, drain, arrive,
  // wake-up), which two buffers of 256 columns hide half of and four of 128 columns all of.
  static constexpr int TMEM_COLS = 512;
  static constexpr int BUFS = TMEM_COLS / BN;
  static_assert(STAGES >= 3 && (2 * STAGES + 2 * BUFS + 1) * 8 + 16 <= BAR_BYTES && SMEM_BYTES <= 227 * 1024, "shared memory");
};

struct Params {
  int E, n, k, n_tiles;
  int64_t total_rows;
  const int32_t* offs;
  const float* scale_a;
  int64_t lds_a;
  const float* scale_b;
  int64_t sb_e, sb_k, sb_n;
  const __nv_bfloat16* bias;
  int64_t bias_stride;
  __nv_bfloat16* d;
  int64_t ldd;
  __nv_bfloat16* d2;
  int64_t ldd2;
  const __nv_bfloat16* aux;
  int64_t ld_aux;
  float alpha, limit;
  int aux_v8, d_v8, d2_v8;  // base 32-byte aligned and row pitch a multiple of 32 bytes
  int stall_test;           // test hook: 1: no tile is loaded, 2: none is multiplied; every wait behind that runs out
  unsigned int* status;
  // The form with the scales in the tensor cores (below) runs where every scale is a power of two, the form with
  // the promotion in registers where one is not: pack_scales_kernel leaves one word per block, not 0 where it
  // found another number, and each form returns at once where the words call for the other.  nullptr: no choice.
  const int32_t* other_scales;
  int num_words;
  // packed scales: byte j of a word is the exponent of block 4 * w + j; [w][row] and [e][w][n block]
  const uint32_t* packed_a;
  const uint32_t* packed_b;
  int64_t packed_rows;  // row pitch of packed_a: rows past the last one that a tile reads included
};

// Whether some scale is no power of two; one barrier, all threads of the CTA.
__device__ __forceinline__ bool any_other_scale(const Params& p) {
  int found = 0;
  for (int i = threadIdx.x; i < p.num_words; i += blockDim.x) found |= __ldg(p.other_scales + i);
  return __syncthreads_or(found) != 0;
}

struct Tile {
  int e, n0, row0, row_end;
};

// Arrive without release semantics, on this CTA's barrier or (shared::cluster address) the other CTA's.  The
// barriers that hand TMEM buffers back guard no memory of the generic proxy: tcgen05.wait::ld has completed
// the reads and tcgen05.fence orders them.  A release at cluster scope, once per block of k, costs a
// memory barrier that waits for the tile's output stores (measured: 2.2x the time of a pair launch).
__device__ __forceinline__ void arrive_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_relaxed_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Wait for phase `parity` of an mbarrier for at most kWaitLimitNs.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                             unsigned int* status) {
  // The waits come once per block of k, so the common case reads no timer (a %globaltimer read costs far
  // more than the wait): the limit counts from the 64th failed try.
  uint64_t t0 = 0;
  for (uint32_t it = 1; !ptx::mbar_try_wait(bar, parity); ++it) {
    if ((it & 63u) != 0) continue;
    if (*abort_flag) return false;
    const uint64_t now = ptx::globaltimer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      atomicOr(status, MGF_DEV_WAIT_TIMEOUT);
      return false;
    }
  }
  return true;
}

// The same for the barrier that the scales of both CTAs of a pair arrive on: acquired at cluster scope.
template <int CG>
__device__ __forceinline__ bool wait_scales_bounded(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                                    unsigned int* status) {
  if constexpr (CG == 1) return wait_bounded(bar, parity, abort_flag, status);
  if (!wait_bounded(bar, parity, abort_flag, status)) return false;
  return ptx::mbar_try_wait_cluster(bar, parity);  // the phase is complete: this only acquires
}

// Group bounds clamped into [0, total_rows] and the prefix of their tile counts; one warp.
template <int TM>
__device__ void build_schedule(const Params& p, int* prefix, int* seg_start, int* seg_end, int lane) {
  int running = 0;
  bool bad = false;
  const long long tr = p.total_rows;
  for (int base = 0; base < p.E; base += 32) {
    const int e = base + lane;
    int cnt = 0;
    if (e < p.E) {
      const long long raw_prev = e == 0 ? 0 : (long long)__ldg(p.offs + e - 1);
      const long long raw_end = (long long)__ldg(p.offs + e);
      if (raw_end < raw_prev || raw_end > tr || raw_prev < 0) bad = true;
      const long long sp = raw_prev < 0 ? 0 : (raw_prev > tr ? tr : raw_prev);
      const long long ep = raw_end < sp ? sp : (raw_end > tr ? tr : raw_end);
      seg_start[e] = (int)sp;
      seg_end[e] = (int)ep;
      cnt = (int)((ep - sp + TM - 1) / TM) * p.n_tiles;
    }
    int inc = cnt;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += o;
    }
    if (e < p.E) prefix[e + 1] = running + inc;
    running += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) prefix[0] = 0;
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(p.status, MGF_DEV_BAD_OFFS);
}

// Tile t: n fastest, so the CTAs at work share a few row blocks and the expert's weight slab.
template <int TM, int BN>
__device__ __forceinline__ Tile decode_tile(int t, const Params& p, const int* prefix, const int* seg_start,
                                            const int* seg_end) {
  int lo = 0, hi = p.E;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= t) lo = mid; else hi = mid;
  }
  const int local = t - prefix[lo], m_blk = local / p.n_tiles;
  return Tile{lo, (local - m_blk * p.n_tiles) * BN, seg_start[lo] + m_blk * TM, seg_end[lo]};
}

// 16 consecutive fp32 columns of this thread's TMEM lane; no wait.
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Sigmoid from the exponential (relative error a few 2^-23): the tanh form's absolute error of about 2^-12
// would be a relative error of tens of percent at gates of -4.  neg_alpha_log2e = -alpha * log2(e).
__device__ __forceinline__ float sigmoid(float gate, float neg_alpha_log2e) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(gate * neg_alpha_log2e));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float swiglu(float g, float u, float neg_alpha_log2e, float limit) {
  const float gc = min_nan(g, limit), uc = max_nan(min_nan(u, limit), -limit);
  return gc * sigmoid(gc, neg_alpha_log2e) * (uc + 1.0f);
}
// d_gate = gs (uc + 1) sig (1 + alpha gc (1 - sig)), d_up = gs gc sig, each 0 where its own input is clamped or NaN (the
// clamp's derivative is 1 in its range only); a NaN of the other input or of gs stays one.
__device__ __forceinline__ uint32_t swiglu_bwd(float gs, uint32_t aux_word, float alpha, float neg_alpha_log2e, float limit) {
  const float g = bf16_lo(aux_word), u = bf16_hi(aux_word);
  const float gc = min_nan(g, limit), uc = max_nan(min_nan(u, limit), -limit);
  const float sig = sigmoid(gc, neg_alpha_log2e), t = gs * sig;
  const float d_gate = g <= limit ? t * (uc + 1.0f) * fmaf(alpha * gc, 1.0f - sig, 1.0f) : 0.0f;
  const float d_up = fabsf(u) <= limit ? t * gc : 0.0f;
  return pack_bf16x2(d_gate, d_up);
}

// Epilogue of one row's COLS columns from column c0 on.  AHEAD (SWIGLU_BWD): aw holds the first 32 columns' aux words
// and every chunk's are loaded one chunk ahead (two ahead: no gain); otherwise they are loaded where they are used
// (fewer registers).
template <int EPI, int COLS, bool AHEAD>
__device__ __forceinline__ void write_columns(const Params& p, const float (&acc)[COLS], int e, int grow, int c0,
                                              uint4 (&aw)[8]) {
  const float nal = -p.alpha * kLog2e;
  // 32 columns at a time; n is a multiple of 8 (SWIGLU: 16), so units of 8 columns are whole
#pragma unroll
  for (int c = 0; c < COLS / 32; ++c) {
    const int col0 = c0 + c * 32;
    if (col0 >= p.n) break;
    if constexpr (EPI == MGF_EPI_SWIGLU_BWD) {
      uint4 cur[8];
      if constexpr (AHEAD) {
#pragma unroll
        for (int g = 0; g < 8; ++g) cur[g] = aw[g];
        if (c + 1 < COLS / 32 && col0 + 32 < p.n)
          load_aux_chunk(p.aux + (int64_t)grow * p.ld_aux, col0 + 32, p.n, true, p.aux_v8, aw);
      } else {
        load_aux_chunk(p.aux + (int64_t)grow * p.ld_aux, col0, p.n, true, p.aux_v8, cur);
      }
      uint4* gp = reinterpret_cast<uint4*>(p.d + (int64_t)grow * p.ldd + 2 * col0);
      const int nvalid = (p.n - col0) >> 2;
#pragma unroll
      for (int g = 0; g < 8; g += 2) {
        if (g < nvalid) {
          uint4 o[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float* f = acc + c * 32 + 4 * (g + h);
            o[h].x = swiglu_bwd(f[0], cur[g + h].x, p.alpha, nal, p.limit);
            o[h].y = swiglu_bwd(f[1], cur[g + h].y, p.alpha, nal, p.limit);
            o[h].z = swiglu_bwd(f[2], cur[g + h].z, p.alpha, nal, p.limit);
            o[h].w = swiglu_bwd(f[3], cur[g + h].w, p.alpha, nal, p.limit);
          }
          if (p.d_v8) ptx::st_v8(gp + g, o[0], o[1]);
          else {
            gp[g] = o[0];
            gp[g + 1] = o[1];
          }
        }
      }
    } else {
      uint32_t packed[16];
      const uint4* bp = reinterpret_cast<const uint4*>(p.bias + (int64_t)e * p.bias_stride + col0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint4 b = make_uint4(0, 0, 0, 0);
        if (p.bias != nullptr && col0 + 8 * g < p.n) b = __ldg(bp + g);
        const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const float* f = acc + c * 32 + 8 * g + 2 * h;
          packed[4 * g + h] = pack_bf16x2(f[0] + bf16_lo(w[h]), f[1] + bf16_hi(w[h]));
        }
      }
      uint4 u[4];
#pragma unroll
      for (int g = 0; g < 4; ++g)
        u[g] = make_uint4(packed[4 * g], packed[4 * g + 1], packed[4 * g + 2], packed[4 * g + 3]);
      store_units<4>(p.d + (int64_t)grow * p.ldd + col0, u, (p.n - col0) >> 3, p.d_v8);
      if constexpr (EPI == MGF_EPI_SWIGLU) {
        uint32_t so[8];
#pragma unroll
        for (int h = 0; h < 8; ++h)
          so[h] = pack_bf16x2(
              swiglu(bf16_lo(packed[2 * h]), bf16_hi(packed[2 * h]), nal, p.limit),
              swiglu(bf16_lo(packed[2 * h + 1]), bf16_hi(packed[2 * h + 1]), nal, p.limit));
        const uint4 us[2] = {make_uint4(so[0], so[1], so[2], so[3]), make_uint4(so[4], so[5], so[6], so[7])};
        store_units<2>(p.d2 + (int64_t)grow * p.ldd2 + (col0 >> 1), us, (p.n - col0) >> 4, p.d2_v8);
      }
    }
  }
}

template <int BN, int EPI, bool B_MN, int CG>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA32,
                const __grid_constant__ CUtensorMap tmB, const Params p) {
  using C = Cfg<BN, CG>;
  constexpr int BUFS = C::BUFS;
  if (p.other_scales != nullptr && !any_other_scale(p)) return;
  constexpr int STAGES = C::STAGES;
  constexpr int TM = BM * CG;       // rows of a tile
  constexpr int COLS = BN / 2;      // columns of a tile that one epilogue thread owns
  constexpr int kMmas = BK / 32;
  static_assert(COLS == 128 || (COLS == 64 && CG == 1), "a thread's columns lie in one scale block");

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE_BYTES);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + STAGES;
  uint64_t* tfull_bar = bars + 2 * STAGES;
  uint64_t* tempty_bar = bars + 2 * STAGES + BUFS;
  uint64_t* drain_bar = bars + 2 * STAGES + 2 * BUFS;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  drain::Copies* loads = reinterpret_cast<drain::Copies*>(tmem_holder + 2);  // the producer's, when it has stopped
  int* prefix = reinterpret_cast<int*>(smem + STAGES * C::STAGE_BYTES + C::BAR_BYTES);
  int* seg_start = prefix + (kMaxGroups + 1);
  int* seg_end = seg_start + (kMaxGroups + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = CG == 2 ? ptx::cluster_ctarank() : 0u;
  const bool leader = crank == 0;
  const int unit = CG == 2 ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int num_units = CG == 2 ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
    }
    for (int b = 0; b < BUFS; ++b) {
      ptx::mbar_init(ptx::smem_u32(&tfull_bar[b]), 1);
      ptx::mbar_init(ptx::smem_u32(&tempty_bar[b]), kNumEpiWarps * CG);
    }
    ptx::mbar_init(ptx::smem_u32(drain_bar), 1);
    *abort_flag = 0;
    *loads = drain::Copies();
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmA);
    ptx::prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      ptx::tmem_alloc_pair(ptx::smem_u32(tmem_holder), C::TMEM_COLS);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(ptx::smem_u32(tmem_holder), C::TMEM_COLS);
      ptx::tmem_relinquish();
    }
  }
  if (warp == 2) build_schedule<TM>(p, prefix, seg_start, seg_end, lane);
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) ptx::cluster_sync();  // barriers of both CTAs initialised before any remote use
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int total_tiles = prefix[p.E];
  const int nk = (p.k + BK - 1) / BK;

  auto leader_addr = [&](const void* ptr) -> uint32_t {
    const uint32_t a = ptx::smem_u32(ptr);
    if constexpr (CG == 2) return ptx::mapa_shared(a, 0);
    return a;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (ptx::elect_one()) {
      uint32_t stage = 0, phase = 0;
      drain::Copies armed;
      bool ok = true;
      for (int t = unit; ok && t < total_tiles && p.stall_test != 1; t += num_units) {
        const Tile ti = decode_tile<TM, BN>(t, p, prefix, seg_start, seg_end);
        const int nb0 = ti.n0 + static_cast<int>(crank) * C::BNC;
        // a tile of up to 32 rows loads 32 rows of A; the products of the stage's other rows are never read
        const bool few_rows = CG == 1 && ti.row_end - ti.row0 <= 32;
        for (int kb = 0; kb < nk; ++kb) {
          if (!wait_bounded(ptx::smem_u32(&empty_bar[stage]), phase ^ 1, abort_flag, p.status)) { ok = false; break; }
          uint32_t fb = ptx::smem_u32(&full_bar[stage]);
          if constexpr (CG == 2) {  // both CTAs' bytes count on the even CTA's barrier
            if (leader) ptx::mbar_arrive_expect_tx(fb, 2 * C::STAGE_BYTES);
            else fb = leader_addr(&full_bar[stage]);
          } else {
            ptx::mbar_arrive_expect_tx(fb, few_rows ? 32 * BK + C::B_BYTES : C::STAGE_BYTES);
          }
          const uint32_t sA = ptx::smem_u32(smem + stage * C::STAGE_BYTES), sB = sA + C::A_BYTES;
          const int row = ti.row0 + static_cast<int>(crank) * BM;
          if constexpr (CG == 2) {
            ptx::tma_load_2d_pair(sA, &tmA, fb, kb * BK, row);
            if constexpr (B_MN) ptx::tma_load_3d_pair(sB, &tmB, fb, nb0, kb * BK, ti.e);
            else ptx::tma_load_3d_pair(sB, &tmB, fb, kb * BK, nb0, ti.e);
          } else {
            ptx::tma_load_2d(sA, few_rows ? &tmA32 : &tmA, fb, kb * BK, row);
            if constexpr (B_MN) {
#pragma unroll
              for (int c = 0; c < C::BNC / 128; ++c)
                ptx::tma_load_3d(sB + c * 16384, &tmB, fb, nb0 + 128 * c, kb * BK, ti.e);
            } else {
              ptx::tma_load_3d(sB, &tmB, fb, kb * BK, nb0, ti.e);
            }
          }
          if (leader) armed.arm(stage, phase);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      *loads = armed;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ UMMA issuer (one elected thread of the even CTA)
    constexpr uint32_t idesc = ptx::make_idesc_e4m3(BM * CG, BN, false, B_MN);
    // MN-major B: 128-column chunks of 128 k rows, 16 KB apart, 32 k rows of 128 bytes per instruction;
    // K-major: 32 bytes of every 128-byte row per instruction
    constexpr uint32_t b_lbo = B_MN ? 16384u : 16u;
    constexpr uint32_t b_kstep = B_MN ? (32u * 128u) >> 4 : 32u >> 4;
    constexpr uint32_t a_kstep = 32u >> 4;
    uint32_t stage = 0, phase = 0, part = 0;  // part: k blocks multiplied so far, the TMEM buffers in turn
    bool ok = p.stall_test != 2;
    if (leader && ptx::elect_one()) {
      for (int t = unit; ok && t < total_tiles; t += num_units) {
        for (int kb = 0; kb < nk; ++kb, ++part) {
          const uint32_t buf = part % BUFS, bph = (part / BUFS) & 1;
          ok = wait_bounded(ptx::smem_u32(&tempty_bar[buf]), bph ^ 1, abort_flag, p.status);
          if (!ok) break;
          ok = wait_bounded(ptx::smem_u32(&full_bar[stage]), phase, abort_flag, p.status);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t sA = ptx::smem_u32(smem + stage * C::STAGE_BYTES);
          const uint64_t adesc = ptx::make_smem_desc_sw128(sA, 16, 1024);
          const uint64_t bdesc = ptx::make_smem_desc_sw128(sA + C::A_BYTES, b_lbo, 1024);
          const uint32_t d_tmem = tmem_base + buf * BN;
#pragma unroll
          for (int kk = 0; kk < kMmas; ++kk) {
            if constexpr (CG == 2) ptx::umma_f8_pair(d_tmem, adesc + kk * a_kstep, bdesc + kk * b_kstep, idesc, kk != 0);
            else ptx::umma_f8(d_tmem, adesc + kk * a_kstep, bdesc + kk * b_kstep, idesc, kk != 0);
          }
          // the epilogue's signal first: the buffer's way round is the critical path
          if constexpr (CG == 2) {
            ptx::umma_commit_pair(ptx::smem_u32(&tfull_bar[buf]), 0x3);
            ptx::umma_commit_pair(ptx::smem_u32(&empty_bar[stage]), 0x3);
          } else {
            ptx::umma_commit(ptx::smem_u32(&tfull_bar[buf]));
            ptx::umma_commit(ptx::smem_u32(&empty_bar[stage]));
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ promotion and epilogue
    const int q = warp & 3, wg = (warp - 2) >> 2;
    const int r = q * 32 + lane;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + wg * COLS;
    const uint32_t tempty_leader = leader_addr(tempty_bar);
    uint32_t part = 0;
    bool ok = true;
    for (int t = unit; ok && t < total_tiles; t += num_units) {
      const Tile ti = decode_tile<TM, BN>(t, p, prefix, seg_start, seg_end);
      const int c0 = ti.n0 + wg * COLS;                            // this thread's first column
      const int crow0 = ti.row0 + static_cast<int>(crank) * BM;    // first row of this CTA's half
      const int grow = crow0 + r;
      const bool active = crow0 + q * 32 < ti.row_end && c0 < p.n;  // warp-uniform
      const bool valid = grow < ti.row_end;
      float acc[COLS];
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[j] = 0.0f;
      // scales: this row's, one block ahead; the tile column block's, one block ahead
      const float* sa_row = p.scale_a + (valid ? grow : ti.row0) * p.lds_a;
      const float* sb_col = p.scale_b + ti.e * p.sb_e + (c0 / BK) * p.sb_n;
      float sa = active ? __ldg(sa_row) : 0.0f, sb = active ? __ldg(sb_col) : 0.0f;
      for (int kb = 0; kb < nk; ++kb, ++part) {
        const uint32_t buf = part % BUFS, bph = (part / BUFS) & 1;
        const float s = sa * sb;
        if (active && kb + 1 < nk) {
          sa = __ldg(sa_row + kb + 1);
          sb = __ldg(sb_col + (kb + 1) * p.sb_k);
        }
        ok = __all_sync(0xffffffffu, wait_bounded(ptx::smem_u32(&tfull_bar[buf]), bph, abort_flag, p.status));
        if (!ok) break;
        ptx::tc_fence_after();
        if (active) {
          const uint32_t tb = lane_base + buf * BN;
          uint32_t v[2][16];
          tmem_ld_x16(tb, v[0]);
#pragma unroll
          for (int c = 0; c < COLS / 16; ++c) {
            ptx::tmem_ld_wait();
            if (c + 1 < COLS / 16) tmem_ld_x16(tb + (c + 1) * 16, v[(c + 1) & 1]);
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[c * 16 + j] = fmaf(s, __uint_as_float(v[c & 1][j]), acc[c * 16 + j]);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) arrive_relaxed_cluster(tempty_leader + 8 * buf);
          else arrive_relaxed(ptx::smem_u32(&tempty_bar[buf]));
        }
      }
      if (!ok) break;
      if (!valid || !active) continue;
      uint4 aw[8];
      write_columns<EPI, COLS, false>(p, acc, ti.e, grow, c0, aw);
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // stopped early: the same for all threads, every role has ended
    if (warp == 0 && ptx::elect_one()) drain::copies<CG>(*loads, full_bar, p.status);
    if (warp == 1 && leader && ptx::elect_one()) drain::products<CG>(drain_bar, p.status);
    __syncthreads();
  }
  // A pair leaves together: the peer may still signal this CTA's barriers until both are done.
  if constexpr (CG == 2) ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    if constexpr (CG == 2) ptx::tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
    else ptx::tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------- scales in the tensor cores
// Where all scales are powers of two (what the quantisers make), the tensor cores apply them: kind::mxf8f6f4 takes a
// power-of-two scale per row of A and column of B for every 32 elements of k, here the same one four times.
// The accumulator then stays in TMEM over the whole contraction and no promotion is needed.

// Scales as bytes, and whether there is one that is no power of two.  A: rows of groups only (those behind the
// last group have no result, and moe_permute_fp8 gives them zeros).  One thread per row, four blocks at a time.
__global__ void __launch_bounds__(256) pack_scales_kernel(const Params p, uint32_t* __restrict__ pa,
                                                          uint32_t* __restrict__ pb, int32_t* __restrict__ words) {
  const int nk = (p.k + BK - 1) / BK, nkw = (nk + 3) / 4, nnb = (p.n + BK - 1) / BK;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t nt = static_cast<int64_t>(gridDim.x) * blockDim.x;
  bool other = false;
  auto byte_of = [&](float s) -> uint32_t {
    const uint32_t b = __float_as_uint(s), e = b >> 23;
    other |= (b & 0x807FFFFFu) != 0u || e == 0u || e == 255u;
    return e & 0xffu;
  };
  // the largest end, not the last one: decreasing offs are clamped by the products, whose rows need their scales too
  __shared__ int last_row;
  if (threadIdx.x == 0) last_row = 0;
  __syncthreads();
  int most = 0;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) most = max(most, __ldg(p.offs + e));
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) atomicMax(&last_row, most);
  __syncthreads();
  const int64_t rows = last_row < p.total_rows ? last_row : p.total_rows;
  const bool vec = (reinterpret_cast<uintptr_t>(p.scale_a) & 15u) == 0 && p.lds_a % 4 == 0;
  for (int64_t r = t0; r < rows; r += nt) {
    const float* s = p.scale_a + r * p.lds_a;
    for (int w = 0; w < nkw; ++w) {
      uint32_t v = 0;
      if (vec && 4 * w + 4 <= nk) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(s + 4 * w));
        v = byte_of(f.x) | (byte_of(f.y) << 8) | (byte_of(f.z) << 16) | (byte_of(f.w) << 24);
      } else {
        for (int j = 0; j < 4; ++j)
          if (4 * w + j < nk) v |= byte_of(__ldg(s + 4 * w + j)) << (8 * j);
      }
      pa[w * p.packed_rows + r] = v;
    }
  }
  const int64_t nb = static_cast<int64_t>(p.E) * nkw * nnb;
  for (int64_t i = t0; i < nb; i += nt) {
    const int64_t c = i % nnb, w = i / nnb % nkw, e = i / nnb / nkw;
    uint32_t v = 0;
    for (int j = 0; j < 4; ++j)
      if (4 * w + j < nk) v |= byte_of(__ldg(p.scale_b + e * p.sb_e + (4 * w + j) * p.sb_k + c * p.sb_n)) << (8 * j);
    pb[i] = v;
  }
  const int found = __syncthreads_or(other ? 1 : 0);
  if (threadIdx.x == 0) words[blockIdx.x] = found;
}

// TMEM: the accumulator's 256 columns, then kSlots scale slots of 4 columns (A: one word per row of 32 x 4) and of 8
// (B: one word per column of 32 x 8).  One accumulator: the epilogue takes it into registers and hands it back before
// it converts and stores, so that the next tile's products run under the stores.
template <int CG>
struct MxCfg {
  static constexpr int BN = 256;
  static constexpr int BNC = BN / CG;  // columns of B held by this CTA
  static constexpr int STAGE_BYTES = BM * BK + BNC * BK;
  static constexpr int STAGES = CG == 2 ? 6 : 4;
  static constexpr int kSlots = 4;               // each holds the scales of four blocks of k
  static constexpr int SLOT_BYTES = 512 + 1024;  // 128 rows of A, 256 columns of B
  static constexpr int BAR_BYTES = 512;
  static constexpr int SCHED_BYTES = 3 * 4 * (kMaxGroups + 1);
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + kSlots * SLOT_BYTES + BAR_BYTES + SCHED_BYTES;
  static constexpr int TMEM_COLS = 512, SFA_COL = BN, SFB_COL = BN + 4 * kSlots;
  static constexpr int kThreads = 384;  // producer, issuer, scales, schedule; 8 epilogue warps
  // __launch_bounds__(384) gives the block 168 x 384 = 64512 registers; the first warpgroup hands back what it does
  // not need: 72 x 128 + 216 x 256 = 64512.  The epilogue holds 128 accumulators and the aux words ahead.
  static constexpr int kSetupRegs = 72, kEpiRegs = 216;
  static_assert(kSetupRegs * 128 + kEpiRegs * 256 <= 168 * kThreads, "register split");
  static_assert(SMEM_BYTES <= 227 * 1024 && SFB_COL + 8 * kSlots <= TMEM_COLS, "shared and tensor memory");
};

// CG = 2: a pair of CTAs on a 256 x 256 tile; each loads its 128 rows of A and 128 columns of B and holds the scales of its
// rows and of all columns, the even CTA issues.
template <int EPI, bool B_MN, int CG>
__global__ void __launch_bounds__(MxCfg<CG>::kThreads, 1)
    mx_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA32,
              const __grid_constant__ CUtensorMap tmA64, const __grid_constant__ CUtensorMap tmB, const Params p) {
  using C = MxCfg<CG>;
  constexpr int TM = BM * CG;
  constexpr int STAGES = C::STAGES, BN = C::BN, COLS = BN / 2, kSlots = C::kSlots;
  if (any_other_scale(p)) return;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slots = smem + STAGES * C::STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(slots + kSlots * C::SLOT_BYTES);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + STAGES;
  uint64_t* sf_full = bars + 2 * STAGES;
  uint64_t* sf_empty = bars + 2 * STAGES + kSlots;
  uint64_t* tfull_bar = bars + 2 * STAGES + 2 * kSlots;
  uint64_t* tempty_bar = tfull_bar + 1;
  uint64_t* drain_bar = tfull_bar + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tfull_bar + 3);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  drain::Copies* loads = reinterpret_cast<drain::Copies*>(tmem_holder + 2);  // the producer's, when it has stopped
  int* prefix = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + C::BAR_BYTES);
  int* seg_start = prefix + (kMaxGroups + 1);
  int* seg_end = seg_start + (kMaxGroups + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = CG == 2 ? ptx::cluster_ctarank() : 0u;
  const bool leader = crank == 0;
  const int unit = CG == 2 ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int num_units = CG == 2 ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  auto leader_addr = [&](const void* ptr) -> uint32_t {
    const uint32_t a = ptx::smem_u32(ptr);
    if constexpr (CG == 2) return ptx::mapa_shared(a, 0);
    return a;
  };
  auto commit = [&](const void* bar) {  // on this CTA's barrier, or the same one of both CTAs of a pair
    if constexpr (CG == 2) ptx::umma_commit_pair(ptx::smem_u32(bar), 0x3);
    else ptx::umma_commit(ptx::smem_u32(bar));
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      ptx::mbar_init(ptx::smem_u32(&sf_full[s]), CG);
      ptx::mbar_init(ptx::smem_u32(&sf_empty[s]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(tfull_bar), 1);
    ptx::mbar_init(ptx::smem_u32(tempty_bar), kNumEpiWarps * CG);
    ptx::mbar_init(ptx::smem_u32(drain_bar), 1);
    *abort_flag = 0;
    *loads = drain::Copies();
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmA);
    ptx::prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      ptx::tmem_alloc_pair(ptx::smem_u32(tmem_holder), C::TMEM_COLS);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(ptx::smem_u32(tmem_holder), C::TMEM_COLS);
      ptx::tmem_relinquish();
    }
  }
  if (warp == 3) build_schedule<TM>(p, prefix, seg_start, seg_end, lane);
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) ptx::cluster_sync();  // barriers of both CTAs initialised before any remote use
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int total_tiles = prefix[p.E];
  const int nk = (p.k + BK - 1) / BK, nkw = (nk + 3) / 4, nnb = (p.n + BK - 1) / BK;

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kSetupRegs));
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (ptx::elect_one()) {
      uint32_t stage = 0, phase = 0;
      drain::Copies armed;
      bool ok = true;
      for (int t = unit; ok && t < total_tiles && p.stall_test != 1; t += num_units) {
        const Tile ti = decode_tile<TM, BN>(t, p, prefix, seg_start, seg_end);
        // a tile of few rows loads 32 or 64 rows of A; the products of the stage's other rows are never read
        const int rows = CG == 2 || ti.row_end - ti.row0 > 64 ? BM : ti.row_end - ti.row0 > 32 ? 64 : 32;
        const CUtensorMap* map_a = rows == BM ? &tmA : rows == 64 ? &tmA64 : &tmA32;
        for (int kb = 0; kb < nk; ++kb) {
          if (!wait_bounded(ptx::smem_u32(&empty_bar[stage]), phase ^ 1, abort_flag, p.status)) { ok = false; break; }
          uint32_t fb = ptx::smem_u32(&full_bar[stage]);
          if constexpr (CG == 2) {  // both CTAs' bytes count on the even CTA's barrier
            if (leader) ptx::mbar_arrive_expect_tx(fb, 2 * C::STAGE_BYTES);
            else fb = leader_addr(&full_bar[stage]);
          } else {
            ptx::mbar_arrive_expect_tx(fb, rows * BK + C::BNC * BK);
          }
          const uint32_t sA = ptx::smem_u32(smem + stage * C::STAGE_BYTES), sB = sA + BM * BK;
          const int row = ti.row0 + static_cast<int>(crank) * BM, col = ti.n0 + static_cast<int>(crank) * C::BNC;
          if constexpr (CG == 2) {
            ptx::tma_load_2d_pair(sA, &tmA, fb, kb * BK, row);
            if constexpr (B_MN) ptx::tma_load_3d_pair(sB, &tmB, fb, col, kb * BK, ti.e);
            else ptx::tma_load_3d_pair(sB, &tmB, fb, kb * BK, col, ti.e);
          } else {
            ptx::tma_load_2d(sA, map_a, fb, kb * BK, row);
            if constexpr (B_MN) {
              ptx::tma_load_3d(sB, &tmB, fb, col, kb * BK, ti.e);
              ptx::tma_load_3d(sB + 16384, &tmB, fb, col + 128, kb * BK, ti.e);
            } else {
              ptx::tma_load_3d(sB, &tmB, fb, kb * BK, col, ti.e);
            }
          }
          if (leader) armed.arm(stage, phase);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      *loads = armed;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ UMMA issuer (one elected thread of the even CTA)
    if (leader && ptx::elect_one()) {
      constexpr uint32_t b_lbo = B_MN ? 16384u : 16u;
      constexpr uint32_t b_kstep = B_MN ? (32u * 128u) >> 4 : 32u >> 4;
      constexpr uint32_t a_kstep = 32u >> 4;
      uint32_t stage = 0, phase = 0, slot = 0, sphase = 0, tphase = 0;
      bool ok = p.stall_test != 2;
      for (int t = unit; ok && t < total_tiles; t += num_units, tphase ^= 1) {
        ok = wait_bounded(ptx::smem_u32(tempty_bar), tphase ^ 1, abort_flag, p.status);
        if (!ok) break;
        ptx::tc_fence_after();
        uint32_t sfa = 0, sfb = 0;
        for (int kb = 0; kb < nk; ++kb) {
          if ((kb & 3) == 0) {  // the scales of the next four blocks
            ok = wait_scales_bounded<CG>(ptx::smem_u32(&sf_full[slot]), sphase, abort_flag, p.status);
            if (!ok) break;
            const uint32_t src = ptx::smem_u32(slots + slot * C::SLOT_BYTES);
            sfa = tmem_base + C::SFA_COL + 4 * slot;
            sfb = tmem_base + C::SFB_COL + 8 * slot;
#pragma unroll
            for (int j = 0; j < 3; ++j) {  // 128 rows of A, 2 x 128 columns of B
              const uint32_t dst = j == 0 ? sfa : sfb + 4 * (j - 1);
              const uint64_t desc = ptx::make_smem_desc_plain(src + 512 * j, 16, 128);
              if constexpr (CG == 2) ptx::tmem_cp_32x128b_x4_pair(dst, desc);
              else ptx::tmem_cp_32x128b_x4(dst, desc);
            }
          }
          ok = wait_bounded(ptx::smem_u32(&full_bar[stage]), phase, abort_flag, p.status);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t sA = ptx::smem_u32(smem + stage * C::STAGE_BYTES);
          const uint64_t adesc = ptx::make_smem_desc_sw128(sA, 16, 1024);
          const uint64_t bdesc = ptx::make_smem_desc_sw128(sA + BM * BK, b_lbo, 1024);
          const uint32_t idesc = ptx::make_idesc_mxf8(TM, BN, false, B_MN, kb & 3);
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk) {
            if constexpr (CG == 2)
              ptx::umma_mxf8_pair(tmem_base, adesc + kk * a_kstep, bdesc + kk * b_kstep, idesc, sfa, sfb, (kb | kk) != 0);
            else
              ptx::umma_mxf8(tmem_base, adesc + kk * a_kstep, bdesc + kk * b_kstep, idesc, sfa, sfb, (kb | kk) != 0);
          }
          commit(&empty_bar[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
          if ((kb & 3) == 3 || kb == nk - 1) {
            commit(&sf_empty[slot]);
            if (++slot == kSlots) { slot = 0; sphase ^= 1; }
          }
        }
        if (!ok) break;
        commit(tfull_bar);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------ scales to shared memory, four blocks of k at a time
    // tcgen05.cp takes 32 rows of 16 bytes: lane i's are the words of rows i, i + 32, i + 64 and i + 96 (of the
    // columns for B, which within one block of 128 are all the same word).
    uint32_t slot = 0, sphase = 0;
    bool ok = true;
    for (int t = unit; ok && t < total_tiles && p.stall_test != 1; t += num_units) {
      const Tile ti = decode_tile<TM, BN>(t, p, prefix, seg_start, seg_end);
      const uint32_t* pa = p.packed_a + ti.row0 + static_cast<int>(crank) * BM + lane;
      const int c0 = ti.n0 / BK, c1 = c0 + 1 < nnb ? c0 + 1 : c0;
      const uint32_t* pb = p.packed_b + static_cast<int64_t>(ti.e) * nkw * nnb;
      for (int w = 0; w < nkw; ++w) {
        const uint4 a = make_uint4(__ldg(pa + w * p.packed_rows), __ldg(pa + w * p.packed_rows + 32),
                                   __ldg(pa + w * p.packed_rows + 64), __ldg(pa + w * p.packed_rows + 96));
        const uint32_t b0 = __ldg(pb + w * nnb + c0), b1 = __ldg(pb + w * nnb + c1);
        ok = __all_sync(0xffffffffu, wait_bounded(ptx::smem_u32(&sf_empty[slot]), sphase ^ 1, abort_flag, p.status));
        if (!ok) break;
        uint4* dst = reinterpret_cast<uint4*>(slots + slot * C::SLOT_BYTES) + lane;
        dst[0] = a;
        dst[32] = make_uint4(b0, b0, b0, b0);
        dst[64] = make_uint4(b1, b1, b1, b1);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {  // the even CTA issues the copies of both
          if constexpr (CG == 2) ptx::mbar_arrive_cluster(leader_addr(&sf_full[slot]));
          else ptx::mbar_arrive(ptx::smem_u32(&sf_full[slot]));
        }
        if (++slot == kSlots) { slot = 0; sphase ^= 1; }
      }
    }
  }
  } else {
    // ------------------------------------------------------------ epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kEpiRegs));
    const int q = warp & 3, wg = (warp - 4) >> 2;
    uint32_t tphase = 0;
    for (int t = unit; t < total_tiles; t += num_units, tphase ^= 1) {
      const Tile ti = decode_tile<TM, BN>(t, p, prefix, seg_start, seg_end);
      const int crow0 = ti.row0 + static_cast<int>(crank) * BM;  // first row of this CTA's half
      const int c0 = ti.n0 + wg * COLS, grow = crow0 + q * 32 + lane;
      const bool active = crow0 + q * 32 < ti.row_end && c0 < p.n;  // warp-uniform
      uint4 aw[8];
      if (EPI == MGF_EPI_SWIGLU_BWD && active && grow < ti.row_end)  // does not depend on the accumulator
        load_aux_chunk(p.aux + (int64_t)grow * p.ld_aux, c0, p.n, true, p.aux_v8, aw);
      if (!__all_sync(0xffffffffu, wait_bounded(ptx::smem_u32(tfull_bar), tphase, abort_flag, p.status))) break;
      ptx::tc_fence_after();
      float acc[COLS];
      if (active) {
        const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + wg * COLS;
#pragma unroll
        for (int c = 0; c < COLS / 32; ++c)
          ptx::tmem_ld_32x32b_x32(tb + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&acc[c * 32]));
        ptx::tmem_ld_wait();
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) arrive_relaxed_cluster(leader_addr(tempty_bar));
        else arrive_relaxed(ptx::smem_u32(tempty_bar));
      }
      if (active && grow < ti.row_end) write_columns<EPI, COLS, true>(p, acc, ti.e, grow, c0, aw);
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // stopped early: the same for all threads, every role has ended
    if (warp == 0 && ptx::elect_one()) drain::copies<CG>(*loads, full_bar, p.status);
    if (warp == 1 && leader && ptx::elect_one()) drain::products<CG>(drain_bar, p.status);
    __syncthreads();
  }
  // A pair leaves together: the peer may still signal this CTA's barriers until both are done.
  if constexpr (CG == 2) ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    if constexpr (CG == 2) ptx::tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
    else ptx::tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// Launch of a persistent kernel with at most one CTA (or pair of CTAs) per SM (or pair of SMs).  A template on the
// kernel itself: what it remembers per device belongs to that kernel.
template <auto KERN, int CG, typename... Args>
int launch_persistent(int threads, int smem, const char* form, int epi, bool b_mn, const Params& p, int64_t tiles, int sms,
                      cudaStream_t st, const Args&... args) {
  static std::mutex mu;
  static bool attr_done[64] = {};
  static int max_units[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MGF_ERR_CUDA;
  int units = sms / CG;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>(units * CG));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  {
    std::lock_guard<std::mutex> g(mu);
    if (!attr_done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) {
        record_error("cudaFuncSetAttribute", e);
        return MGF_ERR_CUDA;
      }
      max_units[dev] = 1 << 30;
      if (CG == 2) {  // never more persistent pairs than can be resident at once
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, KERN, &cfg) == cudaSuccess && n > 0) max_units[dev] = n;
        cudaGetLastError();
      }
      attr_done[dev] = true;
    }
  }
  if (units > max_units[dev]) units = max_units[dev];
  if (tiles < units) units = static_cast<int>(tiles);
  cfg.gridDim = dim3(static_cast<unsigned>(units * CG));
  forget_cuda_error();
  cudaError_t e = cudaLaunchKernelEx(&cfg, KERN, args...);
  if (e == cudaSuccess && debug_sync()) {
    e = cudaStreamSynchronize(st);
    fprintf(stderr, "[mgf] block-scaled form=%s CG=%d epi=%d b_mn=%d units=%d E=%d rows=%lld n=%d k=%d -> %s\n", form, CG, epi,
            int(b_mn), units, p.E, (long long)p.total_rows, p.n, p.k, cudaGetErrorString(e));
  }
  if (e != cudaSuccess) {
    record_error("kernel launch", e);
    return MGF_ERR_CUDA;
  }
  return MGF_OK;
}

template <int EPI, bool B_MN, int CG>
int launch_mx(const CUtensorMap& tA, const CUtensorMap& tA32, const CUtensorMap& tA64, const CUtensorMap& tB, const Params& p, int64_t tiles, int sms, cudaStream_t st) {
  return launch_persistent<mx_kernel<EPI, B_MN, CG>, CG>(MxCfg<CG>::kThreads, MxCfg<CG>::SMEM_BYTES, "mx", EPI, B_MN, p,
                               tiles, sms, st, tA, tA32, tA64, tB, p);
}

template <int BN, int EPI, bool B_MN, int CG>
int launch(const CUtensorMap& tA, const CUtensorMap& tA32, const CUtensorMap& tB, const Params& p, int64_t tiles, int sms,
           cudaStream_t st) {
  return launch_persistent<gemm_kernel<BN, EPI, B_MN, CG>, CG>(kThreads, Cfg<BN, CG>::SMEM_BYTES, BN == 128 ? "128" : "256",
                               EPI, B_MN, p, tiles, sms, st, tA, tA32, tB, p);
}

template <int BN, int CG>
int dispatch(int epi, bool b_mn, const CUtensorMap& tA, const CUtensorMap& tA32, const CUtensorMap& tB, const Params& p, int64_t tiles, int sms,
             cudaStream_t st) {
  switch (epi) {
    case MGF_EPI_BIAS:
      return b_mn ? launch<BN, MGF_EPI_BIAS, true, CG>(tA, tA32, tB, p, tiles, sms, st)
                  : launch<BN, MGF_EPI_BIAS, false, CG>(tA, tA32, tB, p, tiles, sms, st);
    case MGF_EPI_SWIGLU:
      return b_mn ? launch<BN, MGF_EPI_SWIGLU, true, CG>(tA, tA32, tB, p, tiles, sms, st)
                  : launch<BN, MGF_EPI_SWIGLU, false, CG>(tA, tA32, tB, p, tiles, sms, st);
    default:
      return b_mn ? launch<BN, MGF_EPI_SWIGLU_BWD, true, CG>(tA, tA32, tB, p, tiles, sms, st)
                  : launch<BN, MGF_EPI_SWIGLU_BWD, false, CG>(tA, tA32, tB, p, tiles, sms, st);
  }
}

template <int CG>
int dispatch_mx(int epi, bool b_mn, const CUtensorMap& tA, const CUtensorMap& tA32, const CUtensorMap& tA64,
                const CUtensorMap& tB, const Params& p, int64_t tiles, int sms,
                cudaStream_t st) {
  switch (epi) {
    case MGF_EPI_BIAS:
      return b_mn ? launch_mx<MGF_EPI_BIAS, true, CG>(tA, tA32, tA64, tB, p, tiles, sms, st)
                  : launch_mx<MGF_EPI_BIAS, false, CG>(tA, tA32, tA64, tB, p, tiles, sms, st);
    case MGF_EPI_SWIGLU:
      return b_mn ? launch_mx<MGF_EPI_SWIGLU, true, CG>(tA, tA32, tA64, tB, p, tiles, sms, st)
                  : launch_mx<MGF_EPI_SWIGLU, false, CG>(tA, tA32, tA64, tB, p, tiles, sms, st);
    default:
      return b_mn ? launch_mx<MGF_EPI_SWIGLU_BWD, true, CG>(tA, tA32, tA64, tB, p, tiles, sms, st)
                  : launch_mx<MGF_EPI_SWIGLU_BWD, false, CG>(tA, tA32, tA64, tB, p, tiles, sms, st);
  }
}

// Workspace of the form with the scales in the tensor cores: packed scales of A (256 rows past the end: a tile reads
// whole 128- or 256-row blocks), of B, and a word per block of the packing kernel.
constexpr int kPackBlocks = 296;
struct MxSpace {
  int64_t rows, a_words, b_words;
  int64_t bytes() const { return 4 * (a_words + b_words + kPackBlocks); }
};
MxSpace mx_space(const mgf_block_gemm_desc& g) {
  const int64_t nkw = ((g.k + BK - 1) / BK + 3) / 4, nnb = (g.n + BK - 1) / BK;
  MxSpace s;
  s.rows = (g.total_rows + 2 * BM + 3) / 4 * 4;
  s.a_words = nkw * s.rows;
  s.b_words = g.num_groups * nkw * nnb;
  return s;
}

// Tiles of 128 x 256, at most.
int64_t wide_tiles(const mgf_block_gemm_desc& g) {
  return (std::min<int64_t>(g.total_rows, g.num_groups) + g.total_rows / BM) * ((g.n + 255) / 256);
}

// The tensor cores' scales save the promotion but cost two small launches (packing 3-5 us, the form that returns at once
// 2.5), so they have to be earned in blocks of k per SM: from 24 on with many rows, where the promotion is what a block
// waits for (8 groups, k = n = 2048: 25 against 19 us at 1024 rows and 14 blocks, 33 against 43 at 4096 rows and 35);
// from 120 on with few, where both forms wait for the weights and this one keeps more of them under way (128 rows,
// k = 2880, n = 5760: 32 groups and 118 blocks 82 against 81, 128 groups and 460 blocks 126 against 137; 256 groups,
// k = 2048, n = 7168: 127 against 136).  Rows behind the last group count as rows: how many they are is known on the device only.
// MGF_BLOCK_MX=0|1 forces a choice.
bool use_mx(const mgf_block_gemm_desc& g, int sms) {
  if (const char* env = getenv("MGF_BLOCK_MX"); env != nullptr && (env[0] == '0' || env[0] == '1')) return env[0] == '1';
  const int64_t blocks = wide_tiles(g) * ((g.k + BK - 1) / BK);
  return g.n > 128 && blocks >= (g.total_rows >= 1024 ? 24ll : 120ll) * sms;
}

bool aligned(const void* ptr, unsigned n) { return (reinterpret_cast<uintptr_t>(ptr) & (n - 1u)) == 0; }

}  // namespace block_gemm
}  // namespace mgf

extern "C" size_t mgf_block_gemm_desc_size(void) { return sizeof(mgf_block_gemm_desc); }

extern "C" int64_t mgf_block_gemm_workspace_bytes(const mgf_block_gemm_desc* desc) {
  using namespace mgf::block_gemm;
  if (desc == nullptr || desc->num_groups < 1 || desc->total_rows <= 0 || desc->n <= 0 || desc->k <= 0) return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  return use_mx(*desc, mgf::device_info(dev).sms) ? mx_space(*desc).bytes() : 0;
}

extern "C" int mgf_block_gemm_launch(const mgf_block_gemm_desc* desc, void* stream) {
  using namespace mgf;
  using namespace mgf::block_gemm;
  if (desc == nullptr) return MGF_ERR_INVALID_ARGUMENT;
  const mgf_block_gemm_desc& g = *desc;
  if (g.num_groups < 1 || g.num_groups > kMaxGroups) return MGF_ERR_TOO_MANY_GROUPS;
  if (g.epilogue < MGF_EPI_BIAS || g.epilogue > MGF_EPI_SWIGLU_BWD) return MGF_ERR_INVALID_ARGUMENT;
  if (g.total_rows < 0 || g.total_rows > kMaxRows) return MGF_ERR_INVALID_ARGUMENT;
  if (g.n <= 0 || g.k <= 0 || g.n > INT32_MAX / 2 || g.k > INT32_MAX / 2 || g.n % 8 != 0) return MGF_ERR_INVALID_ARGUMENT;
  if (g.epilogue == MGF_EPI_SWIGLU && g.n % 16 != 0) return MGF_ERR_INVALID_ARGUMENT;
  if (g.total_rows == 0) return MGF_OK;  // nothing to write; the tensors of an empty batch have no address
  if (g.epilogue == MGF_EPI_SWIGLU && (g.d2 == nullptr || g.bias == nullptr)) return MGF_ERR_INVALID_ARGUMENT;
  if (g.epilogue == MGF_EPI_SWIGLU_BWD && g.aux == nullptr) return MGF_ERR_INVALID_ARGUMENT;
  if (g.a == nullptr || g.b == nullptr || g.offs == nullptr || g.scale_a == nullptr || g.scale_b == nullptr ||
      g.d == nullptr)
    return MGF_ERR_INVALID_ARGUMENT;
  auto out_ok = [](const void* ptr, int64_t ld) { return aligned(ptr, 16) && ld > 0 && ld % 8 == 0; };
  if (!aligned(g.a, 16) || !aligned(g.b, 16) || g.lda <= 0 || g.lda % 16 != 0 || g.ldb <= 0 || g.ldb % 16 != 0 ||
      g.ldb_batch < 0 || g.ldb_batch % 16 != 0 || (g.num_groups > 1 && g.ldb_batch == 0) || !out_ok(g.d, g.ldd))
    return MGF_ERR_ALIGNMENT;
  if (g.epilogue == MGF_EPI_SWIGLU && !out_ok(g.d2, g.ldd2)) return MGF_ERR_ALIGNMENT;
  if (g.epilogue == MGF_EPI_SWIGLU_BWD && !out_ok(g.aux, g.ld_aux)) return MGF_ERR_ALIGNMENT;
  if (g.bias != nullptr && (!aligned(g.bias, 16) || g.bias_stride % 8 != 0)) return MGF_ERR_ALIGNMENT;

  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MGF_ERR_CUDA;
  clear_error();
  if (!bind_device(dev)) return MGF_ERR_CUDA;
  const DeviceInfo di = device_info(dev);
  if (di.major != 10) return MGF_ERR_NO_DEVICE_SUPPORT;

  auto v8 = [](const void* ptr, int64_t ld) { return ptr != nullptr && aligned(ptr, 32) && ld % 16 == 0 ? 1 : 0; };
  Params p{};
  p.E = g.num_groups;
  p.n = static_cast<int>(g.n);
  p.k = static_cast<int>(g.k);
  p.total_rows = g.total_rows;
  p.offs = g.offs;
  p.scale_a = g.scale_a;
  p.lds_a = g.scale_a_stride;
  p.scale_b = g.scale_b;
  p.sb_e = g.scale_b_stride_e;
  p.sb_k = g.scale_b_stride_k;
  p.sb_n = g.scale_b_stride_n;
  p.bias = g.epilogue == MGF_EPI_SWIGLU_BWD ? nullptr : static_cast<const __nv_bfloat16*>(g.bias);
  p.bias_stride = g.bias_stride;
  p.d = static_cast<__nv_bfloat16*>(g.d);
  p.ldd = g.ldd;
  p.d2 = static_cast<__nv_bfloat16*>(g.d2);
  p.ldd2 = g.ldd2;
  p.aux = static_cast<const __nv_bfloat16*>(g.aux);
  p.ld_aux = g.ld_aux;
  p.alpha = g.swiglu_alpha;
  p.limit = g.swiglu_limit;
  p.d_v8 = v8(g.d, g.ldd);
  p.d2_v8 = v8(g.d2, g.ldd2);
  p.aux_v8 = v8(g.aux, g.ld_aux);
  p.status = status_word_address();
  if (p.status == nullptr) return MGF_ERR_CUDA;
  {
    const char* env = getenv("MGF_TEST_STALL_PRODUCER");  // see moe_gemm_sm100.cu
    p.stall_test = env != nullptr && (env[0] == '1' || env[0] == '2') ? env[0] - '0' : 0;
  }

  // Pairs (256-row tiles, half the B bytes per SM) for groups of 2048 rows and more on average (32 groups, k = 2880,
  // n = 5760, SwiGLU: 32768 rows 692 single against 739 us in pairs, 98304 rows 2103 against 2034);
  // MGF_CTA_GROUP=1|2 forces.  128-column tiles where one covers n, and where 256-column tiles would leave SMs
  // without one (4 rows, n = 5760, k = 2880: 12.4 against 16 us); with more tiles the wide ones read fewer bytes of A
  // per product (256 rows: 97.5 against 107 us).  MGF_BN=128|256 forces.
  const bool b_mn = g.b_mn_major != 0;
  int cg = g.total_rows / g.num_groups >= 2048 ? 2 : 1;
  if (const char* env = getenv("MGF_CTA_GROUP"); env != nullptr && (env[0] == '1' || env[0] == '2')) cg = env[0] - '0';
  int bn = g.n <= 128 || wide_tiles(g) < di.sms ? 128 : 256;
  if (const char* env = getenv("MGF_BN"); env != nullptr && (atoi(env) == 128 || atoi(env) == 256)) bn = atoi(env);
  // tensor-core scales: pairs from 1024 rows on (SwiGLU, 32 groups, k = 2880, n = 5760: 512 rows each 306 us
  // single against 323 in pairs, 2048 rows each 1122 against 1015)
  const int mx_cg = getenv("MGF_CTA_GROUP") != nullptr ? cg : (g.total_rows / g.num_groups >= 1024 ? 2 : 1);
  if (bn == 128) cg = 1;
  p.n_tiles = static_cast<int>((g.n + bn - 1) / bn);

  CUtensorMap tA, tA32, tB;
  const uint64_t dA[2] = {static_cast<uint64_t>(g.k), static_cast<uint64_t>(g.total_rows)};
  const uint64_t sA[1] = {static_cast<uint64_t>(g.lda)};
  const uint32_t bA[2] = {BK, BM}, bA32[2] = {BK, 32};
  const uint64_t batch = g.num_groups > 1 ? static_cast<uint64_t>(g.ldb_batch) : 16;
  const uint64_t sB[2] = {static_cast<uint64_t>(g.ldb), batch};
  const uint64_t dB_mn[3] = {static_cast<uint64_t>(g.n), static_cast<uint64_t>(g.k), static_cast<uint64_t>(g.num_groups)};
  const uint64_t dB_k[3] = {static_cast<uint64_t>(g.k), static_cast<uint64_t>(g.n), static_cast<uint64_t>(g.num_groups)};
  const uint32_t bB_mn[3] = {128, BK, 1};
  const uint32_t bB_k[3] = {BK, static_cast<uint32_t>(bn / cg), 1};
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  if (!encode_bf16(&tA, g.a, 2, dA, sA, bA, CU_TENSOR_MAP_SWIZZLE_128B, u8) ||
      !encode_bf16(&tA32, g.a, 2, dA, sA, bA32, CU_TENSOR_MAP_SWIZZLE_128B, u8) ||
      !encode_bf16(&tB, g.b, 3, b_mn ? dB_mn : dB_k, sB, b_mn ? bB_mn : bB_k, CU_TENSOR_MAP_SWIZZLE_128B, u8))
    return MGF_ERR_CUDA;

  const int64_t tiles = (g.total_rows / (BM * cg) + g.num_groups) * static_cast<int64_t>(p.n_tiles);  // upper bound
  if (tiles > INT32_MAX) return MGF_ERR_INVALID_ARGUMENT;
  int sms = di.sms - (g.sm_carveout > 0 ? g.sm_carveout : 0);
  if (sms < cg) sms = cg;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (use_mx(g, di.sms) && g.workspace != nullptr) {
    if (!aligned(g.workspace, 16)) return MGF_ERR_ALIGNMENT;
    const MxSpace sp = mx_space(g);
    uint32_t* ws = static_cast<uint32_t*>(g.workspace);
    int32_t* words = reinterpret_cast<int32_t*>(ws + sp.a_words + sp.b_words);
    p.packed_a = ws;
    p.packed_b = ws + sp.a_words;
    p.packed_rows = sp.rows;
    p.other_scales = words;
    p.num_words = kPackBlocks;
    forget_cuda_error();
    pack_scales_kernel<<<kPackBlocks, 256, 0, st>>>(p, ws, ws + sp.a_words, words);
    if (cudaGetLastError() != cudaSuccess) return MGF_ERR_CUDA;
    Params pm = p;
    constexpr int kBN = MxCfg<1>::BN;
    pm.n_tiles = static_cast<int>((g.n + kBN - 1) / kBN);
    CUtensorMap tA64, tBm;
    const uint32_t bA64[2] = {BK, 64};
    const uint32_t bBm[3] = {BK, static_cast<uint32_t>(kBN / mx_cg), 1};
    if (!encode_bf16(&tA64, g.a, 2, dA, sA, bA64, CU_TENSOR_MAP_SWIZZLE_128B, u8) ||
        !encode_bf16(&tBm, g.b, 3, b_mn ? dB_mn : dB_k, sB, b_mn ? bB_mn : bBm, CU_TENSOR_MAP_SWIZZLE_128B, u8))
      return MGF_ERR_CUDA;
    const int64_t mx_tiles = (g.total_rows / (BM * mx_cg) + g.num_groups) * static_cast<int64_t>(pm.n_tiles);
    if (mx_tiles > INT32_MAX) return MGF_ERR_INVALID_ARGUMENT;
    const int mx_sms = std::max(sms, mx_cg);  // a pair needs two
    const int rc = mx_cg == 2 ? dispatch_mx<2>(g.epilogue, b_mn, tA, tA32, tA64, tBm, pm, mx_tiles, mx_sms, st)
                              : dispatch_mx<1>(g.epilogue, b_mn, tA, tA32, tA64, tBm, pm, mx_tiles, mx_sms, st);
    if (rc != MGF_OK) return rc;
  }
  if (bn == 128) return dispatch<128, 1>(g.epilogue, b_mn, tA, tA32, tB, p, tiles, sms, st);
  if (cg == 2) return dispatch<256, 2>(g.epilogue, b_mn, tA, tA32, tB, p, tiles, sms, st);
  return dispatch<256, 1>(g.epilogue, b_mn, tA, tA32, tB, p, tiles, sms, st);
}

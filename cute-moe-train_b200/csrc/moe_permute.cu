// Tokens sorted by expert and back (one GPU): the plan, the copies, the weighted sums and the gradients.
//
//   sort       stable counting sort of the n = tokens * topk routed copies (copy c = token * topk + slot) by
//              expert; an id of -1 drops its copy.  offs[e] = end of expert e's rows, row_of_copy[c] = the
//              copy's row or -1, copy_of_row[r] = the row's copy or -1 behind the last row.
//   permute    rows[row_of_copy[c]] = x[c / topk]; rows behind the last one are zeros
//   unpermute  out[t] = sum_j w[t, j] * rows[row_of_copy[t, j]]       (fp32 sum, one rounding; w absent: 1)
//   gradients  of permute: unpermute without weights.  Of unpermute: drows[r] = w[c] * g[t] and
//              dw[c] = <rows[r], g[t]> in one pass over the rows.
//
// Everything but the sort moves rows once and is bound by HBM: 16-byte accesses, each token's row is read
// once and written to its topk rows (not gathered once per row), several accesses in flight per thread.
// No atomics: every sum has a fixed order, so results repeat bit for bit.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

#include "host.h"
#include "moe_gemm.h"

namespace mgf {

unsigned int* status_word_address();

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 8;  // warps per block of the row kernels

// ---------------------------------------------------------------- sort
constexpr int kFewCopies = 1024;  // up to here sort and permute are one launch
constexpr int kSortBatch = 8;  // ids a lane loads together (and keeps from pass 1 to pass 2)

// The copies are split into contiguous ranges, one per warp, and every warp keeps its own histogram in
// shared memory.  Pass 1 counts (shared-memory atomics: a count has no order), the histograms are
// prefix-summed over the warps of a CTA, over the CTAs and over the experts, pass 2 walks the same ranges
// again 32 copies at a time, ranks them within the warp and writes, so the order within an expert is the
// copies' order.  Up to 8192 copies one CTA does it all in one launch (3 us for 32 copies); above, a first
// launch leaves every CTA's counts in the workspace.  (One launch of a cluster of 8 CTAs, counts exchanged in
// distributed shared memory, took 17 us for 98304 copies: 8 SMs are too few for their scattered writes.)
__device__ __forceinline__ void load_ids(const int64_t* ids, int64_t first, int64_t end, int E, int lane,
                                         int (&id)[kSortBatch], bool& bad) {
  int64_t v[kSortBatch];
#pragma unroll
  for (int b = 0; b < kSortBatch; ++b) v[b] = first + 32 * b + lane < end ? __ldg(ids + first + 32 * b + lane) : -1;
#pragma unroll
  for (int b = 0; b < kSortBatch; ++b) {
    const bool ok = v[b] >= -1 && v[b] < E;
    bad |= !ok;
    id[b] = ok ? static_cast<int>(v[b]) : -1;
  }
}

// Lanes whose id equals this lane's (ids in [-1, 2^bits - 1)): one ballot per bit of id + 1.  A match.any gives
// the same in one instruction, but its cost grows with the number of distinct ids in the warp: 98304
// copies over 128 experts took 24 us with it, 18 with ballots and the rest unchanged.
__device__ __forceinline__ unsigned same_id(int id, int bits) {
  unsigned same = kFull;
  const unsigned v = static_cast<unsigned>(id + 1);
  for (int b = 0; b < bits; ++b) {
    const bool bit = (v >> b) & 1u;
    const unsigned set = __ballot_sync(kFull, bit);
    same &= bit ? set : ~set;
  }
  return same;
}

// Copies of CTA c of `ctas`: [c * per, (c + 1) * per).
__device__ __host__ __forceinline__ int64_t copies_per_cta(int64_t n, int ctas) {
  return ((n + ctas - 1) / ctas + 31) / 32 * 32;
}

// counts[cta][e] of every CTA's copies.
__global__ void __launch_bounds__(256) count_kernel(const int64_t* __restrict__ ids, int64_t n, int E,
                                                    int32_t* __restrict__ counts) {
  extern __shared__ __align__(16) int32_t smem[];
  for (int e = threadIdx.x; e < E; e += blockDim.x) smem[e] = 0;
  __syncthreads();
  const int64_t per = copies_per_cta(n, gridDim.x), begin = blockIdx.x * per;
  const int64_t end = begin + per < n ? begin + per : n;
  for (int64_t i = begin + threadIdx.x; i < end; i += blockDim.x) {
    const int64_t v = __ldg(ids + i);
    if (v >= 0 && v < E) atomicAdd(smem + v, 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) counts[static_cast<int64_t>(blockIdx.x) * E + e] = smem[e];
}

// Sort of CTA `rank` of `ctas`.  blockDim.x: a multiple of 256, at least E, at most 1024.  smem: (warps + 2) * E words.
// counts: of all CTAs, nullptr for one CTA.  WRITE: the plan goes to global memory; local_rows (or nullptr): the
// rows of the copies, [n].  Returns the number of rows.
template <bool WRITE>
__device__ __forceinline__ int32_t sort_copies(int32_t* smem, int rank, int ctas, const int64_t* __restrict__ ids, int64_t n,
                                               int E, const int32_t* __restrict__ counts, int32_t* __restrict__ offs,
                                               int32_t* __restrict__ row_of_copy, int32_t* __restrict__ copy_of_row,
                                               int32_t* local_rows, unsigned int* __restrict__ status) {
  const int threads = blockDim.x, warps = threads >> 5;
  int32_t* hist = smem;                // [warps][E]
  int32_t* total = smem + warps * E;   // [E] this CTA's counts
  int32_t* base = total + E;           // [E] first row of this CTA's copies of each expert
  __shared__ int32_t warp_sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t per_cta = copies_per_cta(n, ctas), per = ((per_cta + warps - 1) / warps + 31) / 32 * 32;
  const int64_t first_copy = rank * per_cta < n ? rank * per_cta : n;
  const int64_t last_copy = first_copy + per_cta < n ? first_copy + per_cta : n;
  const int64_t begin = first_copy + warp * per < last_copy ? first_copy + warp * per : last_copy;
  const int64_t end = begin + per < last_copy ? begin + per : last_copy;
  const int bits = 32 - __clz(E);  // of the largest id + 1
  bool bad = false;
  int id[kSortBatch];
  load_ids(ids, begin, end, E, lane, id, bad);
  for (int i = threadIdx.x; i < warps * E; i += threads) hist[i] = 0;
  if (threadIdx.x < 32) warp_sums[threadIdx.x] = 0;
  __syncthreads();
  int32_t* mine = hist + warp * E;
  for (int64_t i = begin;;) {
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b)
      if (id[b] >= 0) atomicAdd(mine + id[b], 1);
    i += 32 * kSortBatch;
    if (i >= end) break;
    load_ids(ids, i, end, E, lane, id, bad);
  }
  if (__any_sync(kFull, bad) && lane == 0) atomicOr(status, MGF_DEV_ROW_OUT_OF_RANGE);
  __syncthreads();
  if (threadIdx.x < E) {
    const int e = threadIdx.x;
    int32_t run = 0;
    for (int w0 = 0; w0 < warps; w0 += 8) {  // warps is 8, 16, 24 or 32
      int32_t c[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) c[w] = hist[(w0 + w) * E + e];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        hist[(w0 + w) * E + e] = run;
        run += c[w];
      }
    }
    total[e] = run;
  }
  __syncthreads();
  // one expert per thread: counts of all CTAs and of those before this one
  int32_t all = 0, before = 0;
  if (threadIdx.x < E) {
    if (counts != nullptr) {
      for (int c0 = 0; c0 < ctas; c0 += 16) {
        int32_t v[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = c0 + c < ctas ? __ldg(counts + static_cast<int64_t>(c0 + c) * E + threadIdx.x) : 0;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          all += v[c];
          before += c0 + c < rank ? v[c] : 0;
        }
      }
    } else {
      all = total[threadIdx.x];
    }
  }
  int32_t incl = all;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int32_t o = __shfl_up_sync(kFull, incl, off);
    if (lane >= off) incl += o;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int32_t s = warp_sums[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int32_t o = __shfl_up_sync(kFull, s, off);
      if (lane >= off) s += o;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  const int32_t first = incl - all + (warp > 0 ? warp_sums[warp - 1] : 0);
  if (threadIdx.x < E) {
    base[threadIdx.x] = first + before;
    if (WRITE && rank == 0) offs[threadIdx.x] = first + all;
  }
  const int32_t kept = warp_sums[31];
  __syncthreads();
  if (end - begin > 32 * kSortBatch) load_ids(ids, begin, end, E, lane, id, bad);  // else the registers still hold them
  for (int64_t i = begin; i < end;) {
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      if (i + 32 * b >= end) break;  // the same for all lanes
      const int64_t c = i + 32 * b + lane;
      const unsigned same = same_id(id[b], bits);
      int32_t row = -1;
      if (id[b] >= 0) row = base[id[b]] + mine[id[b]] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (id[b] >= 0 && lane == __ffs(same) - 1) mine[id[b]] += __popc(same);
      __syncwarp();
      if (c < end) {
        if (WRITE) {
          row_of_copy[c] = row;
          if (row >= 0) copy_of_row[row] = static_cast<int32_t>(c);
        }
        if (local_rows != nullptr) local_rows[c] = row;
      }
    }
    i += 32 * kSortBatch;
    if (i < end) load_ids(ids, i, end, E, lane, id, bad);
  }
  if (WRITE)
    for (int64_t r = kept + static_cast<int64_t>(rank) * threads + threadIdx.x; r < n;
         r += static_cast<int64_t>(ctas) * threads)
      copy_of_row[r] = -1;
  return kept;
}

__global__ void __launch_bounds__(1024) sort_kernel(const int64_t* __restrict__ ids, int64_t n, int E,
                                                    const int32_t* __restrict__ counts, int32_t* __restrict__ offs,
                                                    int32_t* __restrict__ row_of_copy,
                                                    int32_t* __restrict__ copy_of_row,
                                                    unsigned int* __restrict__ status) {
  extern __shared__ __align__(16) int32_t smem[];
  sort_copies<true>(smem, blockIdx.x, gridDim.x, ids, n, E, counts, offs, row_of_copy, copy_of_row, nullptr, status);
}

// ---------------------------------------------------------------- row access
// 16 bytes (VEC) or one element at a time where a base, a pitch or the width is not a multiple of 16 bytes.
// The raw words stay packed until they are added: unpacked early, the loads in flight would double the
// registers and halve the warps that hide their latency.
template <typename T, bool VEC>
struct Access {
  static constexpr int N = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  using Raw = typename std::conditional<VEC, uint4, T>::type;
  static __device__ __forceinline__ Raw load(const T* p) { return __ldg(reinterpret_cast<const Raw*>(p)); }
  static __device__ __forceinline__ void store(T* p, const Raw& r) { *reinterpret_cast<Raw*>(p) = r; }
  static __device__ __forceinline__ Raw zero() {
    if constexpr (VEC) return make_uint4(0, 0, 0, 0);
    else return T(0.0f);
  }
  // f[] = the elements of r in fp32
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[N]) {
    if constexpr (!VEC) {
      f[0] = static_cast<float>(r);
    } else {
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, float>::value) {
          f[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          f[2 * i] = v.x;
          f[2 * i + 1] = v.y;
        } else {
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
      }
    }
  }
  // one rounding of every element
  static __device__ __forceinline__ Raw pack(const float (&f)[N]) {
    if constexpr (!VEC) {
      return static_cast<T>(f[0]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, float>::value) {
          w[i] = __float_as_uint(f[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// Rows of up to B copies of one token (-1: dropped, or outside the rows -- a wrong plan, which is reported
// and touched nowhere).  All indices are loaded before the first is looked at: a check in between would
// make every load wait for the one before it.
template <int B>
__device__ __forceinline__ void load_rows(const int32_t* row_of_copy, int count, int64_t n_rows, unsigned int* status,
                                          int32_t (&row)[B]) {
#pragma unroll
  for (int b = 0; b < B; ++b) row[b] = b < count ? __ldg(row_of_copy + b) : -1;
  bool bad = false;
#pragma unroll
  for (int b = 0; b < B; ++b) {
    if (row[b] >= n_rows) {
      bad = true;
      row[b] = -1;
    }
  }
  if (bad) atomicOr(status, MGF_DEV_ROW_OUT_OF_RANGE);
}

// Zeros into the rows behind the last one, offs_end[0] .. n_rows, shared out over the whole grid.
template <typename T, bool VEC>
__device__ __forceinline__ void zero_tail(T* rows, int64_t ld, int64_t n_rows, int64_t nv, const int32_t* offs_end) {
  int64_t kept = __ldg(offs_end);
  if (kept < 0) kept = 0;
  if (kept >= n_rows) return;
  using A = Access<T, VEC>;
  const typename A::Raw z = A::zero();
  const int64_t w0 = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int64_t nw = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  for (int64_t r = kept + w0; r < n_rows; r += nw)
    for (int64_t v = threadIdx.x & 31; v < nv; v += 32) A::store(rows + r * ld + v * A::N, z);
}

// ---------------------------------------------------------------- permute
// A token's row is read once and written to its topk rows.  24576 tokens of 5760 bytes, top 4: 110 us, 6.4 TB/s.
constexpr int kPermuteVecs = 4;  // vectors per lane and work unit: a warp moves 2 KB of one token

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps)
    permute_kernel(const T* __restrict__ x, int64_t ldx, int64_t tokens, int topk, int64_t nv, int64_t chunks,
                   const int32_t* __restrict__ row_of_copy, const int32_t* __restrict__ offs_end, int64_t n_rows,
                   T* __restrict__ rows, int64_t ldr, unsigned int* __restrict__ status) {
  using A = Access<T, VEC>;
  const int lane = threadIdx.x & 31;
  const int64_t u = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (u < tokens * chunks) {
    const int64_t t = u / chunks;
    const int64_t v0 = (u - t * chunks) * (32 * kPermuteVecs) + lane;
    typename A::Raw r[kPermuteVecs];
#pragma unroll
    for (int i = 0; i < kPermuteVecs; ++i)
      if (v0 + 32 * i < nv) r[i] = A::load(x + t * ldx + (v0 + 32 * i) * A::N);
    for (int j0 = 0; j0 < topk; j0 += 4) {
      int32_t row[4];
      load_rows(row_of_copy + t * topk + j0, topk - j0, n_rows, status, row);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (row[b] < 0) continue;
        T* d = rows + static_cast<int64_t>(row[b]) * ldr;
#pragma unroll
        for (int i = 0; i < kPermuteVecs; ++i)
          if (v0 + 32 * i < nv) A::store(d + (v0 + 32 * i) * A::N, r[i]);
      }
    }
  }
  zero_tail<T, VEC>(rows, ldr, n_rows, nv, offs_end);
}

// Sort of up to 256 copies by counting: a copy's row is the number of copies with a smaller id or with its own id and
// before it, a thread per copy; offs[e] is the number with an id up to e, a thread per expert.  No histogram, no scan and
// one barrier (decode permutation, 32 copies: 3.8 us against 4.7).  ids_s: shared memory, a multiple of 4 words.
constexpr int kCountedCopies = 256;

template <bool WRITE>
__device__ __forceinline__ int32_t count_copies(int32_t* ids_s, const int64_t* __restrict__ ids, int n, int E,
                                                int32_t* __restrict__ offs, int32_t* __restrict__ row_of_copy,
                                                int32_t* __restrict__ copy_of_row, int32_t* local_rows,
                                                unsigned int* __restrict__ status) {
  const int c = threadIdx.x, n4 = (n + 3) / 4 * 4;
  int mine = E;  // dropped copies sort behind all experts
  if (c < n) {
    const int64_t v = __ldg(ids + c);
    if (v >= 0 && v < E) mine = static_cast<int>(v);
    else if (v != -1) atomicOr(status, MGF_DEV_ROW_OUT_OF_RANGE);
  }
  if (c < n4) ids_s[c] = mine;
  const int32_t kept = __syncthreads_count(mine < E);
  const int4* all = reinterpret_cast<const int4*>(ids_s);
  if (c < n) {
    int row = 0;
    for (int i = 0; i < n4 / 4; ++i) {
      const int4 v = all[i];
      row += (v.x < mine || (v.x == mine && 4 * i < c)) + (v.y < mine || (v.y == mine && 4 * i + 1 < c)) +
             (v.z < mine || (v.z == mine && 4 * i + 2 < c)) + (v.w < mine || (v.w == mine && 4 * i + 3 < c));
    }
    if (mine == E) row = -1;
    local_rows[c] = row;
    if (WRITE) {
      row_of_copy[c] = row;
      if (row >= 0) copy_of_row[row] = c;
      if (c >= kept) copy_of_row[c] = -1;
    }
  }
  if (WRITE)
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
      int end = 0;
      for (int i = 0; i < n4 / 4; ++i) {
        const int4 v = all[i];
        end += (v.x <= e) + (v.y <= e) + (v.z <= e) + (v.w <= e);
      }
      offs[e] = end;
    }
  return kept;
}

// Sort and permute of few copies in one launch: every CTA sorts them all for itself (the first one writes the plan),
// then the CTAs share out the rows.  One launch less on a path that is nothing but launches.
template <typename T, bool VEC>
__global__ void __launch_bounds__(1024)
    sort_permute_kernel(const int64_t* __restrict__ ids, int E, const T* __restrict__ x, int64_t ldx, int64_t tokens, int topk,
                        int64_t nv, int64_t chunks, int32_t* __restrict__ offs, int32_t* __restrict__ row_of_copy,
                        int32_t* __restrict__ copy_of_row, T* __restrict__ rows, int64_t ldr,
                        unsigned int* __restrict__ status) {
  using A = Access<T, VEC>;
  extern __shared__ __align__(16) int32_t smem[];
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int64_t n = tokens * topk;
  int32_t* row_of = smem + (n <= kCountedCopies ? kCountedCopies : (warps + 2) * E);
  int32_t kept;
  if (n <= kCountedCopies)
    kept = blockIdx.x == 0 ? count_copies<true>(smem, ids, n, E, offs, row_of_copy, copy_of_row, row_of, status)
                           : count_copies<false>(smem, ids, n, E, offs, row_of_copy, copy_of_row, row_of, status);
  else
    kept = blockIdx.x == 0
               ? sort_copies<true>(smem, 0, 1, ids, n, E, nullptr, offs, row_of_copy, copy_of_row, row_of, status)
               : sort_copies<false>(smem, 0, 1, ids, n, E, nullptr, offs, row_of_copy, copy_of_row, row_of, status);
  __syncthreads();
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * warps + (threadIdx.x >> 5), nw = static_cast<int64_t>(gridDim.x) * warps;
  for (int64_t u = w0; u < tokens * chunks; u += nw) {
    const int64_t t = u / chunks;
    const int64_t v0 = (u - t * chunks) * (32 * kPermuteVecs) + lane;
    typename A::Raw r[kPermuteVecs];
#pragma unroll
    for (int i = 0; i < kPermuteVecs; ++i)
      if (v0 + 32 * i < nv) r[i] = A::load(x + t * ldx + (v0 + 32 * i) * A::N);
    for (int j = 0; j < topk; ++j) {
      const int32_t row = row_of[t * topk + j];
      if (row < 0) continue;
#pragma unroll
      for (int i = 0; i < kPermuteVecs; ++i)
        if (v0 + 32 * i < nv) A::store(rows + static_cast<int64_t>(row) * ldr + (v0 + 32 * i) * A::N, r[i]);
    }
  }
  const typename A::Raw z = A::zero();
  for (int64_t r = kept + w0; r < n; r += nw)
    for (int64_t v = lane; v < nv; v += 32) A::store(rows + r * ldr + v * A::N, z);
}

// ---------------------------------------------------------------- unpermute
constexpr int kSumBatch = 4;  // copies whose loads are in flight together

// One vector per lane: 4 loads in flight and few registers, so that many warps are resident.  A warp walks
// `vecs` / 32 chunks of its token: four where that leaves work for every SM, so that blocks live longer than it takes to
// start them (24576 tokens of 5760 bytes, 4 copies: 124 us against 133 with one), one chunk for few tokens.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps)
    unpermute_kernel(const T* __restrict__ rows, int64_t ldr, int64_t n_rows, int64_t tokens, int topk, int64_t nv,
                     int64_t chunks, int vecs, const int32_t* __restrict__ row_of_copy, const float* __restrict__ weights,
                     T* __restrict__ out, int64_t ldo, unsigned int* __restrict__ status) {
  using A = Access<T, VEC>;
  const int lane = threadIdx.x & 31;
  const int64_t u = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (u >= tokens * chunks) return;
  const int64_t t = u / chunks;
  const int64_t v_begin = (u - t * chunks) * vecs;
  const int64_t v_end = v_begin + vecs < nv ? v_begin + vecs : nv;
#pragma unroll 1
  for (int64_t v = v_begin + lane; v < v_end; v += 32) {
    float acc[A::N];
#pragma unroll
    for (int c = 0; c < A::N; ++c) acc[c] = 0.0f;
    for (int j0 = 0; j0 < topk; j0 += kSumBatch) {
      int32_t row[kSumBatch];
      float w[kSumBatch];
      typename A::Raw r[kSumBatch];
#pragma unroll
      for (int b = 0; b < kSumBatch; ++b)
        w[b] = weights != nullptr && j0 + b < topk ? __ldg(weights + t * topk + j0 + b) : 1.0f;
      load_rows(row_of_copy + t * topk + j0, topk - j0, n_rows, status, row);
#pragma unroll
      for (int b = 0; b < kSumBatch; ++b)
        if (row[b] >= 0) r[b] = A::load(rows + static_cast<int64_t>(row[b]) * ldr + v * A::N);
#pragma unroll
      for (int b = 0; b < kSumBatch; ++b) {
        if (row[b] < 0) continue;
        float f[A::N];
        A::unpack(r[b], f);
#pragma unroll
        for (int c = 0; c < A::N; ++c) acc[c] = fmaf(w[b], f[c], acc[c]);
      }
    }
    A::store(out + t * ldo + v * A::N, A::pack(acc));
  }
}

// ---------------------------------------------------------------- unpermute, backward
constexpr int kBwdBatch = 4;  // copies handled per walk over the token's row

// WPT warps per token (1: many tokens, 8: few).  Each lane keeps the partial dot products of up to
// kBwdBatch copies; they are summed over the lanes by shuffles and over the warps in a fixed order.  16384 tokens of
// 14 KB, top 8: 575 us, 6.6 TB/s (rows and output gradient in, rows' gradient out).
template <typename T, bool VEC, int WPT>
__global__ void __launch_bounds__(32 * kWarps)
    unpermute_bwd_kernel(const T* __restrict__ g, int64_t ldg, const T* __restrict__ rows, int64_t ldr, int64_t n_rows,
                         int64_t tokens, int topk, int64_t nv, const int32_t* __restrict__ row_of_copy,
                         const int32_t* __restrict__ offs_end, const float* __restrict__ weights,
                         T* __restrict__ grad_rows, int64_t ldgr, float* __restrict__ grad_weights,
                         unsigned int* __restrict__ status) {
  using A = Access<T, VEC>;
  __shared__ float part[kWarps][kBwdBatch];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) / WPT;  // uniform over a block for WPT = kWarps
  const int sub = warp % WPT;
  if (t < tokens) {
    for (int j0 = 0; j0 < topk; j0 += kBwdBatch) {
      int32_t row[kBwdBatch];
      float w[kBwdBatch], dot[kBwdBatch];
#pragma unroll
      for (int b = 0; b < kBwdBatch; ++b) {
        w[b] = weights != nullptr && j0 + b < topk ? __ldg(weights + t * topk + j0 + b) : 1.0f;
        dot[b] = 0.0f;
      }
      load_rows(row_of_copy + t * topk + j0, topk - j0, n_rows, status, row);
      for (int64_t v = sub * 32 + lane; v < nv; v += 32 * WPT) {
        float gf[A::N];
        A::unpack(A::load(g + t * ldg + v * A::N), gf);
        typename A::Raw rv[kBwdBatch];
        if (grad_weights != nullptr) {
#pragma unroll
          for (int b = 0; b < kBwdBatch; ++b)
            if (row[b] >= 0) rv[b] = A::load(rows + static_cast<int64_t>(row[b]) * ldr + v * A::N);
        }
#pragma unroll
        for (int b = 0; b < kBwdBatch; ++b) {
          if (row[b] < 0) continue;
          float f[A::N];
          if (grad_weights != nullptr) {
            A::unpack(rv[b], f);
#pragma unroll
            for (int c = 0; c < A::N; ++c) dot[b] = fmaf(f[c], gf[c], dot[b]);
          }
          if (grad_rows != nullptr) {
#pragma unroll
            for (int c = 0; c < A::N; ++c) f[c] = w[b] * gf[c];
            A::store(grad_rows + static_cast<int64_t>(row[b]) * ldgr + v * A::N, A::pack(f));
          }
        }
      }
      if (grad_weights == nullptr) continue;
#pragma unroll
      for (int b = 0; b < kBwdBatch; ++b) {
#pragma unroll
        for (int off = 16; off; off >>= 1) dot[b] += __shfl_xor_sync(kFull, dot[b], off);
      }
      if constexpr (WPT == 1) {
        if (lane < kBwdBatch && j0 + lane < topk) {
          float d = dot[0];
#pragma unroll
          for (int b = 1; b < kBwdBatch; ++b) d = lane == b ? dot[b] : d;
          grad_weights[t * topk + j0 + lane] = d;
        }
      } else {
        static_assert(WPT == kWarps, "one token per block");
        if (lane == 0) {
#pragma unroll
          for (int b = 0; b < kBwdBatch; ++b) part[warp][b] = dot[b];
        }
        __syncthreads();
        if (warp == 0 && lane < kBwdBatch && j0 + lane < topk) {
          float d = 0.0f;
          for (int i = 0; i < kWarps; ++i) d += part[i][lane];
          grad_weights[t * topk + j0 + lane] = d;
        }
        __syncthreads();
      }
    }
  }
  if (grad_rows != nullptr) zero_tail<T, VEC>(grad_rows, ldgr, n_rows, nv, offs_end);
}

// ---------------------------------------------------------------- host
int elem_size(int32_t dtype) { return dtype == MGF_DT_F32 ? 4 : 2; }

bool vec_ok(const void* p, int64_t ld, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * size) % 16 == 0;
}

// Calls f(element, VEC) for the element type and whether all rows can be accessed 16 bytes at a time.
template <typename F>
int for_type(int32_t dtype, bool vec, F&& f) {
  switch (dtype) {
    case MGF_DT_BF16:
      return vec ? f(__nv_bfloat16{}, std::true_type{}) : f(__nv_bfloat16{}, std::false_type{});
    case MGF_DT_F16:
      return vec ? f(__half{}, std::true_type{}) : f(__half{}, std::false_type{});
    default:
      return vec ? f(float{}, std::true_type{}) : f(float{}, std::false_type{});
  }
}

bool row_args_ok(int32_t dtype, int64_t tokens, int32_t topk, int64_t hidden, int64_t n_rows) {
  return dtype >= MGF_DT_BF16 && dtype <= MGF_DT_F32 && tokens >= 0 && topk >= 1 && hidden >= 0 && n_rows >= 0 &&
         n_rows <= INT32_MAX && tokens <= INT32_MAX / topk;
}

int launched() { return cudaGetLastError() == cudaSuccess ? MGF_OK : MGF_ERR_CUDA; }

// Blocks for `units` warps of work; false where a one-dimensional grid cannot hold them.
bool grid_of(int64_t units, unsigned& grid) {
  const int64_t b = (units + kWarps - 1) / kWarps;
  if (b > INT32_MAX) return false;
  grid = static_cast<unsigned>(b > 0 ? b : 1);
  return true;
}

}  // namespace
}  // namespace mgf

// CTAs of a sort in two launches: 2048 copies each up to one wave of them.
static int sort_ctas(int64_t n) {
  if (n <= 8192) return 1;
  const int64_t c = (n + 2047) / 2048;
  return static_cast<int>(c < 148 ? c : 148);
}

extern "C" int64_t mgf_moe_sort_workspace_words(int64_t n, int32_t num_experts) {
  const int ctas = sort_ctas(n);
  return ctas > 1 ? static_cast<int64_t>(ctas) * num_experts : 0;
}

extern "C" int mgf_moe_sort(const int64_t* expert_idx, int64_t n, int32_t num_experts, int32_t* offs,
                            int32_t* row_of_copy, int32_t* copy_of_row, int32_t* workspace, void* stream) {
  using namespace mgf;
  forget_cuda_error();
  if (n < 0 || n > INT32_MAX || num_experts < 1 || num_experts > 1024 || offs == nullptr)
    return MGF_ERR_INVALID_ARGUMENT;
  if (n > 0 && (expert_idx == nullptr || row_of_copy == nullptr || copy_of_row == nullptr))
    return MGF_ERR_INVALID_ARGUMENT;
  const int ctas = sort_ctas(n);
  if (ctas > 1 && workspace == nullptr) return MGF_ERR_INVALID_ARGUMENT;
  unsigned int* status = status_word_address();
  if (status == nullptr) return MGF_ERR_CUDA;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MGF_ERR_CUDA;
  static std::atomic<bool> attr_done[64];
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(34 * 1024 * sizeof(int32_t))) != cudaSuccess)
      return MGF_ERR_CUDA;
    attr_done[dev] = true;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (ctas > 1) {
    count_kernel<<<ctas, 256, num_experts * sizeof(int32_t), st>>>(expert_idx, n, num_experts, workspace);
    if (launched() != MGF_OK) return MGF_ERR_CUDA;
  }
  // 8 warps, or as many as E needs threads; all 32 where one CTA has many copies
  const unsigned least = (static_cast<unsigned>(num_experts) + 255u) / 256u * 256u;
  const unsigned threads = ctas == 1 && n > 1024 ? 1024u : least;
  const size_t smem = static_cast<size_t>(threads / 32 + 2) * num_experts * sizeof(int32_t);
  sort_kernel<<<ctas, threads, smem, st>>>(expert_idx, n, num_experts, ctas > 1 ? workspace : nullptr, offs, row_of_copy,
                                           copy_of_row, status);
  return launched();
}

extern "C" int mgf_moe_sort_permute(const int64_t* expert_idx, int32_t num_experts, const void* x, int32_t dtype,
                                    int64_t ldx, int64_t tokens, int32_t topk, int64_t hidden, int32_t* offs,
                                    int32_t* row_of_copy, int32_t* copy_of_row, void* rows, int64_t ldr,
                                    int32_t* workspace, void* stream) {
  using namespace mgf;
  forget_cuda_error();
  if (topk < 1 || tokens < 0 || tokens > INT32_MAX / topk) return MGF_ERR_INVALID_ARGUMENT;
  const int64_t n = tokens * topk;
  if (n == 0 || hidden == 0 || n > kFewCopies) {
    const int rc = mgf_moe_sort(expert_idx, n, num_experts, offs, row_of_copy, copy_of_row, workspace, stream);
    if (rc != MGF_OK) return rc;
    return mgf_moe_permute(x, dtype, ldx, tokens, topk, hidden, row_of_copy, offs + num_experts - 1, rows, ldr, n, stream);
  }
  if (!row_args_ok(dtype, tokens, topk, hidden, n) || num_experts < 1 || num_experts > 1024 || expert_idx == nullptr ||
      x == nullptr || offs == nullptr || row_of_copy == nullptr || copy_of_row == nullptr || rows == nullptr)
    return MGF_ERR_INVALID_ARGUMENT;
  unsigned int* status = status_word_address();
  if (status == nullptr) return MGF_ERR_CUDA;
  const int es = elem_size(dtype);
  const bool vec = (hidden * es) % 16 == 0 && vec_ok(x, ldx, es) && vec_ok(rows, ldr, es);
  return for_type(dtype, vec, [&](auto e, auto v) {
    using T = decltype(e);
    constexpr bool VEC = decltype(v)::value;
    auto kern = sort_permute_kernel<T, VEC>;
    const int smem_most = static_cast<int>((34 * 1024 + kFewCopies) * sizeof(int32_t));
    static std::atomic<bool> attr_done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return static_cast<int>(MGF_ERR_CUDA);
    if (!attr_done[dev]) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_most) != cudaSuccess)
        return static_cast<int>(MGF_ERR_CUDA);
      attr_done[dev] = true;
    }
    const unsigned threads = n <= kCountedCopies ? 256u : (static_cast<unsigned>(num_experts) + 255u) / 256u * 256u;
    const int64_t nv = hidden / Access<T, VEC>::N, chunks = (nv + 32 * kPermuteVecs - 1) / (32 * kPermuteVecs);
    const int64_t blocks = (tokens * chunks * 32 + threads - 1) / threads;
    const unsigned grid = static_cast<unsigned>(blocks < 296 ? blocks : 296);
    const size_t plan_words = n <= kCountedCopies ? kCountedCopies : (threads / 32 + 2) * static_cast<size_t>(num_experts);
    const size_t smem = (plan_words + n) * sizeof(int32_t);
    kern<<<grid, threads, smem, static_cast<cudaStream_t>(stream)>>>(
        expert_idx, num_experts, static_cast<const T*>(x), ldx, tokens, topk, nv, chunks, offs, row_of_copy, copy_of_row,
        static_cast<T*>(rows), ldr, status);
    return launched();
  });
}

extern "C" int mgf_moe_permute(const void* x, int32_t dtype, int64_t ldx, int64_t tokens, int32_t topk, int64_t hidden,
                               const int32_t* row_of_copy, const int32_t* offs_end, void* rows, int64_t ldr,
                               int64_t n_rows, void* stream) {
  using namespace mgf;
  forget_cuda_error();
  if (!row_args_ok(dtype, tokens, topk, hidden, n_rows)) return MGF_ERR_INVALID_ARGUMENT;
  if (n_rows == 0 || hidden == 0) return MGF_OK;
  if (offs_end == nullptr || rows == nullptr || (tokens > 0 && (x == nullptr || row_of_copy == nullptr)))
    return MGF_ERR_INVALID_ARGUMENT;
  unsigned int* status = status_word_address();
  if (status == nullptr) return MGF_ERR_CUDA;
  const int es = elem_size(dtype);
  const bool vec = (hidden * es) % 16 == 0 && vec_ok(x, ldx, es) && vec_ok(rows, ldr, es);
  return for_type(dtype, vec, [&](auto e, auto v) {
    using T = decltype(e);
    constexpr bool VEC = decltype(v)::value;
    const int64_t nv = hidden / Access<T, VEC>::N, chunks = (nv + 32 * kPermuteVecs - 1) / (32 * kPermuteVecs);
    unsigned grid;
    if (!grid_of(tokens * chunks, grid)) return static_cast<int>(MGF_ERR_INVALID_ARGUMENT);
    permute_kernel<T, VEC><<<grid, 32 * kWarps, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(x), ldx, tokens, topk, nv, chunks, row_of_copy, offs_end, n_rows, static_cast<T*>(rows),
        ldr, status);
    return launched();
  });
}

extern "C" int mgf_moe_unpermute(const void* rows, int32_t dtype, int64_t ldr, int64_t n_rows, int64_t tokens,
                                 int32_t topk, int64_t hidden, const int32_t* row_of_copy, const float* weights,
                                 void* out, int64_t ldo, void* stream) {
  using namespace mgf;
  forget_cuda_error();
  if (!row_args_ok(dtype, tokens, topk, hidden, n_rows)) return MGF_ERR_INVALID_ARGUMENT;
  if (tokens == 0 || hidden == 0) return MGF_OK;
  if (out == nullptr || row_of_copy == nullptr || (n_rows > 0 && rows == nullptr)) return MGF_ERR_INVALID_ARGUMENT;
  unsigned int* status = status_word_address();
  if (status == nullptr) return MGF_ERR_CUDA;
  const int es = elem_size(dtype);
  const bool vec = (hidden * es) % 16 == 0 && vec_ok(rows, ldr, es) && vec_ok(out, ldo, es);
  return for_type(dtype, vec, [&](auto e, auto v) {
    using T = decltype(e);
    constexpr bool VEC = decltype(v)::value;
    const int64_t nv = hidden / Access<T, VEC>::N;
    const int vecs = tokens * ((nv + 31) / 32) >= 8 * 148 * 64 ? 128 : 32;
    const int64_t chunks = (nv + vecs - 1) / vecs;
    unsigned grid;
    if (!grid_of(tokens * chunks, grid)) return static_cast<int>(MGF_ERR_INVALID_ARGUMENT);
    unpermute_kernel<T, VEC><<<grid, 32 * kWarps, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(rows), ldr, n_rows, tokens, topk, nv, chunks, vecs, row_of_copy, weights, static_cast<T*>(out),
        ldo, status);
    return launched();
  });
}

extern "C" int mgf_moe_unpermute_bwd(const void* grad_out, int64_t ldg, const void* rows, int64_t ldr, int32_t dtype,
                                     int64_t n_rows, int64_t tokens, int32_t topk, int64_t hidden,
                                     const int32_t* row_of_copy, const int32_t* offs_end, const float* weights,
                                     void* grad_rows, int64_t ldgr, float* grad_weights, void* stream) {
  using namespace mgf;
  forget_cuda_error();
  if (!row_args_ok(dtype, tokens, topk, hidden, n_rows)) return MGF_ERR_INVALID_ARGUMENT;
  if (grad_rows == nullptr && grad_weights == nullptr) return MGF_OK;
  if (tokens > 0 && (grad_out == nullptr || row_of_copy == nullptr)) return MGF_ERR_INVALID_ARGUMENT;
  if (offs_end == nullptr || (n_rows > 0 && grad_weights != nullptr && rows == nullptr))
    return MGF_ERR_INVALID_ARGUMENT;
  if (tokens == 0 && n_rows == 0) return MGF_OK;
  unsigned int* status = status_word_address();
  if (status == nullptr) return MGF_ERR_CUDA;
  const int es = elem_size(dtype);
  const bool vec = (hidden * es) % 16 == 0 && vec_ok(grad_out, ldg, es) &&
                   (grad_weights == nullptr || vec_ok(rows, ldr, es)) &&
                   (grad_rows == nullptr || vec_ok(grad_rows, ldgr, es));
  return for_type(dtype, vec, [&](auto e, auto v) {
    using T = decltype(e);
    constexpr bool VEC = decltype(v)::value;
    const int64_t nv = hidden / Access<T, VEC>::N;
    auto run = [&](auto wpt) {
      constexpr int WPT = decltype(wpt)::value;
      unsigned grid;
      if (!grid_of(tokens * WPT, grid)) return static_cast<int>(MGF_ERR_INVALID_ARGUMENT);
      unpermute_bwd_kernel<T, VEC, WPT><<<grid, 32 * kWarps, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(grad_out), ldg, static_cast<const T*>(rows), ldr, n_rows, tokens, topk, nv, row_of_copy,
          offs_end, weights, static_cast<T*>(grad_rows), ldgr, grad_weights, status);
      return launched();
    };
    // one warp per token as soon as that fills the 148 SMs' 64 warps twice
    if (tokens >= 2 * 148 * 64) return run(std::integral_constant<int, 1>{});
    return run(std::integral_constant<int, kWarps>{});
  });
}

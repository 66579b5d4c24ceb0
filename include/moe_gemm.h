/*
 * moe_gemm.h -- C ABI of the B200 (sm_100a) MoE FFN grouped-GEMM library (libmoe_gemm.so).
 *
 * One launcher runs every GEMM of the MoE FFN forward and backward.  A call describes one
 * grouped GEMM over E experts whose token rows are delimited by `offs` (int32 cumulative
 * end offsets, on the device) and picks one of four fused epilogues.  All pointers are
 * device pointers; nothing here allocates, synchronises the host or reads `offs` on the host.
 *
 * Reference interfaces this ABI replaces (Butterfingrz/CuTe-MoE-Train,
 * paths relative to cutlass_op/bf16_grouped_mm/):
 *   MGF_EPI_BIAS            <- csrc/binding.cu:13-34  `_grouped_mm_cuda` (ragged-M, bias optional)
 *                              and csrc/grouped_mm_kernel.cuh:478 `bf16bf16_grouped_mm`
 *   MGF_EPI_SWIGLU          <- csrc/binding.cu:39-64  `_grouped_mm_swiglu_cuda`
 *                              and csrc/grouped_mm_kernel.cuh:1365 `bf16bf16_grouped_mm_swiglu`
 *   MGF_EPI_SWIGLU_BWD      <- csrc/binding.cu:68-118 `_grouped_mm_swiglu_bwd_cuda`
 *                              and csrc/grouped_mm_kernel.cuh:854 `bf16bf16_grouped_mm_swiglu_bwd`
 *   MGF_EPI_WGRAD           <- the ragged-K (2D x 2D) branch of `_grouped_mm_cuda`
 *                              (csrc/grouped_mm_kernel.cuh:224-226, csrc/grouped_mm_common.cuh:120-133)
 *                              fused with custom_op.py:79-101 `_segment_sum_rows` (bias gradient)
 *
 * Error behaviour: host-side argument errors return a negative MGF_ERR_* code and launch
 * nothing (the torch layer turns them into RuntimeError, like the reference's TORCH_CHECKs).
 * Device-side problems (malformed offs, a pipeline wait that ran out) never trap: the kernel
 * records a bit in a device status word that mgf_device_status() reads.
 */
#ifndef MOE_GEMM_H_
#define MOE_GEMM_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Epilogue selector. */
enum mgf_epilogue {
  MGF_EPI_BIAS = 0,       /* D = bf16(A*B[e] + bias[e])           (bias may be NULL)          */
  MGF_EPI_SWIGLU = 1,     /* aux = bf16(A*B[e] + bias[e]); D2 = swiglu(aux) (gate/up interleaved) */
  MGF_EPI_SWIGLU_BWD = 2, /* D = swiglu_bwd(A*B[e], aux): interleaved (d_gate, d_up) pairs     */
  MGF_EPI_WGRAD = 3       /* ragged-K: D[e] = A[g]^T-view * B[g]; D2[e] = column sums of B[g]  */
};

/* Status codes returned by the host entry points. */
enum mgf_status {
  MGF_OK = 0,
  MGF_ERR_INVALID_ARGUMENT = -1,
  MGF_ERR_UNSUPPORTED_LAYOUT = -2,
  MGF_ERR_ALIGNMENT = -3,
  MGF_ERR_TOO_MANY_GROUPS = -4,
  MGF_ERR_CUDA = -5,
  MGF_ERR_NO_DEVICE_SUPPORT = -6
};

/* Device status bits recorded by the kernels (read with mgf_device_status). */
#define MGF_DEV_WAIT_TIMEOUT 0x1u  /* a pipeline wait ran out; the kernel stopped early        */
#define MGF_DEV_DRAIN_TIMEOUT 0x8u /* after that, its own copies or products in flight did not end in time either */
#define MGF_DEV_BAD_OFFS 0x2u      /* offs not non-decreasing or beyond the row extent; clamped */
#define MGF_DEV_ROW_OUT_OF_RANGE 0x4u /* a row index of gather/combine/push/permute fell outside its buffer (or an expert id its range);
                                         that row was skipped (left unwritten)                    */

/*
 * One grouped GEMM.  Matrix layouts are given as element strides of bf16 tensors.
 *
 * Ragged-M epilogues (BIAS, SWIGLU, SWIGLU_BWD):
 *   A    : [total_rows, k] row-major (stride lda, unit stride along k); rows of group e are
 *          offs[e-1]..offs[e]-1.
 *   B    : [E, k, n] with batch stride ldb_batch; b_mn_major=1 means unit stride along n
 *          (row stride ldb), b_mn_major=0 means unit stride along k (column stride ldb).
 *   D    : [total_rows, n_out] row-major, stride ldd (n_out = n, or the aux tensor for SWIGLU).
 *   D2   : SWIGLU only: swiglu_out [total_rows, n/2], stride ldd2.
 *   aux  : SWIGLU_BWD only: [total_rows, 2n] interleaved (gate, up), stride ld_aux; D is then
 *          grad_aux [total_rows, 2n] with stride ldd.
 * Ragged-K epilogue (WGRAD):
 *   A    : [total_rows, m] row-major (stride lda): the GEMM uses its transpose per group.
 *   B    : [total_rows, n] row-major (stride ldb).
 *   D    : [E, m, n] bf16, row stride ldd, batch stride ldd_batch.  Empty groups get zeros.
 *   D2   : optional [E, n] bf16 bias gradient (stride ldd2 between groups): column sums of B.
 * Extents: n a multiple of 8 (whole 16-byte output units); k (ragged-M) and m (ragged-K) any
 * positive value.  Every base pointer 16-byte aligned and every row / batch stride a multiple of
 * 8 elements (the TMA rule); reads past k, m, n or total_rows return zeros.
 */
typedef struct mgf_gemm_desc {
  int32_t epilogue;      /* enum mgf_epilogue */
  int32_t num_groups;    /* E (1..1024) */
  int64_t total_rows;    /* extent of the ragged dimension (tokens), at most 2^31 - 257 */
  int64_t m, n, k;       /* fixed GEMM extents (m unused for ragged-M, k unused for ragged-K) */
  const void* a;
  int64_t lda;
  const void* b;
  int64_t ldb;
  int64_t ldb_batch;
  int32_t b_mn_major;
  const int32_t* offs;   /* device int32 [E] cumulative end offsets */
  const void* bias;      /* device bf16 [E, n] or NULL */
  int64_t bias_stride;
  void* d;
  int64_t ldd;
  int64_t ldd_batch;
  void* d2;
  int64_t ldd2;
  const void* aux;
  int64_t ld_aux;
  float swiglu_alpha;
  float swiglu_limit;
  int32_t store_aux;     /* SWIGLU: 1 = also write aux (D) */
  int32_t sm_carveout;   /* SMs left free for concurrent work (collectives); 0 = use all */
  int32_t* workspace;    /* WGRAD: device int32[1], zero-filled before the call: the dynamic tile
                            counter (tiles of a ragged-K launch cost in proportion to their group's
                            size; handing them out in order keeps the CTAs on neighbouring tiles).
                            NULL = static tile striding.  One workspace per launch in flight. */
  int32_t bias_per_row;  /* BIAS, ragged-M only: 0 = bias[e, col] added to every row (the MoE case);
                            1 = bias[e, row - group start] added to every column of a row (the
                            transposed form of the reference's ragged-N bias, csrc/grouped_mm_common.cuh:107-118) */
  int32_t ab_type;       /* enum mgf_ab_type: element type of A and B.  MGF_AB_E4M3 (8-bit float).
                            Ragged-M (BIAS, SWIGLU, SWIGLU_BWD; B with unit stride along k): the
                            accumulator is scaled by scale_a[row] * scale_b[e * scale_b_stride + col]
                            before the bias / SwiGLU / SwiGLU backward.  Ragged-K (WGRAD): A and B are
                            the same row-major token layouts as for bf16, with per-feature scales:
                            D[e][i][j] = acc * scale_a[i] * scale_b[j], the bias gradient acc * scale_b[j]
                            (scale_b_stride unused).  lda / ldb / ldb_batch then count bytes
                            (multiples of 16). */
  const float* scale_a;  /* E4M3: device fp32 [total_rows] (ragged-M) or [m] (ragged-K) */
  const float* scale_b;  /* E4M3: device fp32 [E, n] (ragged-M) or [n] (ragged-K) */
  int64_t scale_b_stride;
  const int64_t* d_row_ptrs; /* BIAS (bf16) only, NULL = off.  Scatter mode: output row r is written
                            at the address d_row_ptrs[r] (device int64 [total_rows]; any address this
                            device can store to, e.g. a peer GPU's IPC-mapped buffer; 0 = row not
                            written; 16-byte aligned, 32-byte aligned for whole-sector stores)
                            instead of d + r * ldd (d and ldd are then unused).  The expert-parallel
                            combine writes each expert output straight into its source rank's buffer
                            this way, fusing the transfer into the GEMM epilogue. */
  int32_t group_begin;   /* groups 0 .. group_begin-1 are skipped (no tile computed, nothing written --
                            for WGRAD not even the zeros of empty groups); 0 = all.  Lets a caller run a grouped GEMM in two launches
                            over the expert ranges [0, g) and [g, E) of one offs array, e.g. while the
                            rows of the second range are still arriving. */
} mgf_gemm_desc;

enum mgf_ab_type { MGF_AB_BF16 = 0, MGF_AB_E4M3 = 1 };

/* Launch one grouped GEMM on `stream` (a cudaStream_t; NULL = legacy default stream).
 * Replaces: csrc/binding.cu:13-148 (the three pybind entry points) + the dispatch in
 * csrc/grouped_mm_kernel.cuh:390-486, 760-864, 1267-1390. */
int mgf_grouped_gemm_launch(const mgf_gemm_desc* desc, void* stream);

/* Allocation-free variant of the ragged-K weight-gradient launch (MGF_EPI_WGRAD only).
 * No counterpart in the reference.  For callers that cannot allocate device memory when they
 * launch (a runtime with a fixed, up-front memory plan; a host program that binds this ABI and
 * only holds the buffers it was given): the zero-filled tile counter normally passed as
 * desc->workspace comes instead from a 256-byte static device array inside the library (64 int32
 * words, 1 used per call; held by every GPU that loads the library until exit).  desc->workspace
 * must be NULL.  The call clears the word it uses on `stream` before the kernel; all calls share
 * the array, so calls that overlap on the GPU race and must not be issued.  Each call looks up
 * the array's address on the calling device (so it stays right after a device reset); the first
 * call on a device should come before any stream capture.  Allocates
 * nothing (no cudaMalloc/cudaFree).  Same return codes as mgf_grouped_gemm_launch. */
int mgf_grouped_gemm_launch_noalloc(const mgf_gemm_desc* desc, void* stream);

/* Expert-parallel row movement (no counterpart in the reference, which has no distributed code).
 * bf16 rows of row_elems elements (a multiple of 8), row strides ld_* in elements (multiples of 8),
 * 16-byte aligned bases, int64 device index arrays, optional fp32 device scales (NULL = 1).
 *   mgf_gather_rows:  dst[i] = scale[i] * src[idx[i]],                     i < n_rows
 *   mgf_combine_rows: out[t] = sum_{j<k} weights[t*k+j] * rows[pos[t*k+j]], t < n_out (fp32 sum)
 * n_src / n_rows is the row count of src / rows: an index outside [0, n_src) leaves its output
 * row unwritten (combine: any of the token's k indices) and sets MGF_DEV_ROW_OUT_OF_RANGE.
 * Dispatch gathers token copies into expert order; combine sums each token's k expert outputs;
 * each is the other's backward. */
int mgf_gather_rows(const void* src, int64_t ld_src, int64_t n_src, const int64_t* idx, const float* scale,
                    int64_t n_rows, int64_t row_elems, void* dst, int64_t ld_dst, void* stream);
int mgf_combine_rows(const void* rows, int64_t ld_rows, int64_t n_rows, const int64_t* pos, const float* weights,
                     int64_t n_out, int32_t k, int64_t row_elems, void* out, int64_t ld_out, void* stream);

/* Expert-parallel push over NVLink peer memory (no counterpart in the reference): for i < n rows
 * (n = n_max, or *n_dev when n_dev is non-NULL -- a device-side count), write
 * scale[i] * src[src_idx[i]] (src_idx NULL = i, scale NULL = 1) to row dst_row[i] of the buffer at
 * peer_bases[dst_rank[i]] (device array of `world` base addresses, one per rank, from CUDA IPC
 * mappings; each buffer dst_rows rows of stride ld_dst).  Rows whose rank or destination row falls
 * outside [0, world) x [0, dst_rows), or whose source row falls outside [0, n_src), are skipped and
 * set MGF_DEV_ROW_OUT_OF_RANGE.  Plain peer stores, no multicast.
 * Completion signal (flag_bases non-NULL): when all of the launch's stores are visible, `seq` is
 * written (release, system scope) into slot `rank` of every rank's flag array (flag_bases: device
 * array of `world` addresses of uint64 [world] flag arrays, IPC-mapped); `counter` is a zeroed
 * device uint64 of this rank that the launch uses and leaves at zero.  Readers then call
 * mgf_wait_flags on their own flag array instead of a collective barrier.
 * rotate (optional device int64): entries are visited starting at index *rotate (mod n), so that ranks
 * whose entries are sorted by destination do not all write to the same rank at the same time. */
int mgf_push_rows(const void* src, int64_t ld_src, int64_t n_src, const int64_t* src_idx, const float* scale,
                  int64_t n_max, const int32_t* n_dev, const int64_t* dst_rank, const int64_t* dst_row,
                  const unsigned long long* peer_bases, int64_t world, int64_t dst_rows, int64_t ld_dst,
                  int64_t row_elems, const unsigned long long* flag_bases, unsigned long long* counter,
                  unsigned long long seq, int64_t rank, const int64_t* rotate, void* stream);

/* Wait on `stream` until flags[s] >= seq for every s < world (every rank's push with sequence
 * number seq has landed here), at most timeout_ns; a wait that runs out records
 * MGF_DEV_WAIT_TIMEOUT in the device status word and returns.  One small kernel, no host sync
 * (no counterpart in the reference). */
int mgf_wait_flags(const unsigned long long* flags, int64_t world, unsigned long long seq, int64_t timeout_ns,
                   void* stream);

/* Signal on `stream`: after every earlier operation of the stream (e.g. a scatter-epilogue GEMM
 * that stored rows into peers' buffers), write seq into slot `rank` of every rank's flag array
 * (flag_bases as for mgf_push_rows).  Readers use mgf_wait_flags.  No counterpart in the reference. */
int mgf_signal_flags(const unsigned long long* flag_bases, int64_t world, int64_t rank, unsigned long long seq,
                     void* stream);

/* Device-side plan of the expert-parallel peer transport (no counterpart in the reference; no host
 * synchronisation).  mgf_ep_sort: stable counting sort of n routed copies (expert_ids int64 [n], copy
 * i = token i / topk) by expert: order[p] (copy at sorted position p), inv_order[copy], copy_token[p],
 * e_sorted[p], counts[E] (int64); workspace: int32 [mgf_ep_sort_workspace_words(n, E)] device scratch.
 * Out-of-range ids are clamped and set MGF_DEV_ROW_OUT_OF_RANGE.
 * mgf_ep_routes: from the all-gathered count matrix c_all [world, E] (int64) and this rank's e_sorted:
 * dst_rank / dst_row [n] (owner rank and row of each sorted copy in the owner's receive buffer: local
 * expert-major, then source rank, then sorted order), src_rank / src_pos [cap] (source rank and its
 * sorted position of each receive row; -1 past the received rows), optional ptr_ret / ptr_gret [cap]
 * (ret_bases[src] + src_pos * row_bytes and the same in gret_bases; 0 past the received rows: the row
 * addresses of the scatter epilogues), offs [E / world] (int32) and n_recv [1] (int32).  workspace:
 * int32 [mgf_ep_routes_workspace_words(world, E)] device scratch. */
int64_t mgf_ep_sort_workspace_words(int64_t n, int32_t num_experts);
int mgf_ep_sort(const int64_t* expert_ids, int64_t n, int32_t num_experts, int32_t topk, int32_t* workspace,
                int64_t* order, int64_t* inv_order, int64_t* copy_token, int64_t* e_sorted, int64_t* counts,
                void* stream);
int64_t mgf_ep_routes_workspace_words(int32_t world, int32_t num_experts);
int mgf_ep_routes(const int64_t* c_all, int32_t world, int32_t num_experts, const int64_t* e_sorted, int64_t n,
                  int32_t rank, int64_t cap, const unsigned long long* ret_bases,
                  const unsigned long long* gret_bases, int64_t row_bytes, int32_t* workspace, int64_t* dst_rank,
                  int64_t* dst_row, int64_t* src_rank, int64_t* src_pos, int64_t* ptr_ret, int64_t* ptr_gret,
                  int32_t* offs, int32_t* n_recv, void* stream);

/* e4m3 quantisers of the FP8 path (no counterpart in the reference, which has no FP8): bf16 in,
 * float8_e4m3fn out, fp32 scales = max(amax, 1e-12) / 448, q = saturate(x / scale), round to nearest.
 *   rows:    x [rows, cols] (row stride ldx) -> q [rows, cols] (row stride ldq), scale [rows];
 *   cols:    the same with one scale per column, scale [cols];
 *   weights: w [E, K, N] with element strides s_e, s_k, s_n (s_n == 1 or s_k == 1 read coalesced)
 *            -> q [E, N, K] with K contiguous (row stride ldq >= K), scale [E, N].
 * cols, ldx and ldq multiples of 8, x 16-byte aligned.  Each a few kernels on `stream`, no host sync. */
int mgf_fp8_quantize_rows(const void* x, int64_t rows, int64_t cols, int64_t ldx, void* q, int64_t ldq, float* scale,
                          void* stream);
int mgf_fp8_quantize_cols(const void* x, int64_t rows, int64_t cols, int64_t ldx, void* q, int64_t ldq, float* scale,
                          void* stream);
/* Both scalings of one [rows, cols] activation in two passes: (q_r, s_r) as mgf_fp8_quantize_rows and
 * (q_c, s_c) as mgf_fp8_quantize_cols give, bit-identical (no counterpart in the reference). */
int mgf_fp8_quantize_rows_cols(const void* x, int64_t rows, int64_t cols, int64_t ldx, void* q_r, int64_t ldq_r,
                               float* s_r, void* q_c, int64_t ldq_c, float* s_c, void* stream);
int mgf_fp8_quantize_weights(const void* w, int64_t E, int64_t K, int64_t N, int64_t s_e, int64_t s_k, int64_t s_n,
                             void* q, int64_t ldq, float* scale, void* stream);
/* Both axes of one weight [E, K, N] (unit stride along n, n % 8 == 0, 16-byte aligned strides and
 * bases) in two passes: qa [E, N, ldqa] / sa [E, N] as mgf_fp8_quantize_weights gives for w, and
 * qb [E, K, ldqb] / sb [E, K] as it gives for w^T (codes n-contiguous, one scale per (e, k));
 * bit-identical to the two calls (no counterpart in the reference). */
int mgf_fp8_quantize_weights_both(const void* w, int64_t E, int64_t K, int64_t N, int64_t s_e, int64_t s_k, void* qa,
                                  int64_t ldqa, float* sa, void* qb, int64_t ldqb, float* sb, void* stream);

/* ------------------------------------------------------------------ the MoE block around the products
 * (no counterpart in the reference, whose path starts from rows already in expert order). */
enum mgf_dtype { MGF_DT_BF16 = 0, MGF_DT_F16 = 1, MGF_DT_F32 = 2 };
enum mgf_route_score { MGF_ROUTE_SOFTMAX = 0, MGF_ROUTE_SIGMOID = 1 };
#define MGF_ROUTE_BIAS_ON_SCORE 0x100 /* or'ed to a score: the bias is added to the score, not to the logit */

/* Router.  logits [tokens, E] (E <= 1024, topk <= min(E, 32), row stride ld): the topk experts with the
 * largest logit + bias (bias fp32 [E] or NULL, selection only), largest first, ties to the lowest expert.  With
 * MGF_ROUTE_BIAS_ON_SCORE it is the largest score + bias instead, the score being the sigmoid or the softmax over
 * all experts in fp32 (the order differs: neither is linear); without a bias the flag changes nothing.
 * weights fp32 [tokens, topk]: scale * softmax (over the chosen experts if renormalize, else over all) or
 * scale * sigmoid (divided by the chosen experts' sum if renormalize) of the logits without bias.
 * expert_idx int64 [tokens, topk].  A logit of -inf is never chosen, nor is a sum with the bias of -inf: slots left over, and
 * all slots of tokens whose token_mask (bytes, or NULL) is 0, get id -1 and weight 0.
 * mgf_moe_route_bwd: grad_logits [tokens, E] (row stride ldg, every element written) from the gradient of
 * the weights; the chosen experts are those of expert_idx. */
int mgf_moe_route(const void* logits, int32_t dtype, int64_t ld, int64_t tokens, int32_t num_experts, int32_t topk,
                  int32_t score, int32_t renormalize, float scale, const float* bias, const uint8_t* token_mask,
                  float* weights, int64_t* expert_idx, void* stream);
int mgf_moe_route_bwd(const void* logits, int32_t dtype, int64_t ld, int64_t tokens, int32_t num_experts, int32_t topk,
                      int32_t score, int32_t renormalize, float scale, const int64_t* expert_idx,
                      const float* grad_weights, void* grad_logits, int64_t ldg, void* stream);

/* Plan of the permutation: stable counting sort of n routed copies (expert_idx int64 [n], copy c = token
 * c / topk) by expert, E <= 1024.  offs int32 [E] (cumulative row ends, what the grouped products take),
 * row_of_copy int32 [n] (-1 for a copy whose id is -1), copy_of_row int32 [n] (-1 behind offs[E-1]).  Ids
 * outside [-1, E) drop their copy too and set MGF_DEV_ROW_OUT_OF_RANGE.  workspace: int32
 * [mgf_moe_sort_workspace_words(n, E)] device scratch of this call (may be NULL where that is 0). */
int64_t mgf_moe_sort_workspace_words(int64_t n, int32_t num_experts);
int mgf_moe_sort(const int64_t* expert_idx, int64_t n, int32_t num_experts, int32_t* offs, int32_t* row_of_copy,
                 int32_t* copy_of_row, int32_t* workspace, void* stream);

/* Rows by a plan (any hidden size; strides in elements; 16-byte accesses where every base and pitch and the
 * width allow).  offs_end points at offs[E-1].  A row index >= n_rows is skipped and sets
 * MGF_DEV_ROW_OUT_OF_RANGE.
 *   permute:       rows[row_of_copy[t*topk+j]] = x[t]; rows from *offs_end to n_rows become zeros
 *   sort_permute:  mgf_moe_sort and permute (n_rows = tokens * topk) in one call; one launch for few copies
 *   unpermute:     out[t] = sum_j weights[t*topk+j] * rows[row_of_copy[t*topk+j]]  (fp32 sum; NULL weights: 1)
 *   unpermute_bwd: grad_rows[row] = weight * grad_out[t] (rows behind *offs_end: zeros) and
 *                  grad_weights[t*topk+j] = <rows[row], grad_out[t]> (0 for a dropped copy); either may be NULL. */
int mgf_moe_permute(const void* x, int32_t dtype, int64_t ldx, int64_t tokens, int32_t topk, int64_t hidden,
                    const int32_t* row_of_copy, const int32_t* offs_end, void* rows, int64_t ldr, int64_t n_rows,
                    void* stream);
int mgf_moe_sort_permute(const int64_t* expert_idx, int32_t num_experts, const void* x, int32_t dtype, int64_t ldx,
                         int64_t tokens, int32_t topk, int64_t hidden, int32_t* offs, int32_t* row_of_copy,
                         int32_t* copy_of_row, void* rows, int64_t ldr, int32_t* workspace, void* stream);
int mgf_moe_unpermute(const void* rows, int32_t dtype, int64_t ldr, int64_t n_rows, int64_t tokens, int32_t topk,
                      int64_t hidden, const int32_t* row_of_copy, const float* weights, void* out, int64_t ldo,
                      void* stream);
int mgf_moe_unpermute_bwd(const void* grad_out, int64_t ldg, const void* rows, int64_t ldr, int32_t dtype,
                          int64_t n_rows, int64_t tokens, int32_t topk, int64_t hidden, const int32_t* row_of_copy,
                          const int32_t* offs_end, const float* weights, void* grad_rows, int64_t ldgr,
                          float* grad_weights, void* stream);

/* e4m3 quantisers with a scale per block of 128: bf16 in, float8_e4m3fn codes and fp32 scales out; the scale
 * is the smallest power of two with amax / scale <= 448 (1 for a block of zeros, never subnormal), amax over
 * the block's finite elements; non-finite elements become NaN codes.
 *   rows:    x [tokens, cols] -> q (row stride ldq, a multiple of 16), scale [.., ceil(cols / 128)] (row
 *            stride lds).  row_of_copy NULL: row t of q is token t (topk 1, n_rows = tokens).  Else the
 *            token's codes go to its topk rows, and rows from *offs_end to n_rows get zero codes and scales.
 *   weights: w [E, R, C] with unit stride along C -> q in the same layout (strides q_e, q_r multiples of 8)
 *            and scale [E, ceil(R / 128), ceil(C / 128)] with any strides. */
int mgf_fp8_block_quantize_rows(const void* x, int64_t ldx, int64_t tokens, int64_t cols, int32_t topk,
                                const int32_t* row_of_copy, const int32_t* offs_end, void* q, int64_t ldq,
                                float* scale, int64_t lds, int64_t n_rows, void* stream);
int mgf_fp8_block_quantize_weights(const void* w, int64_t E, int64_t R, int64_t C, int64_t s_e, int64_t s_r, void* q,
                                   int64_t q_e, int64_t q_r, float* scale, int64_t ss_e, int64_t ss_r, int64_t ss_c,
                                   void* stream);

/* Grouped GEMM of e4m3 operands with a scale per block of 128 (ragged M; epilogues BIAS, SWIGLU and
 * SWIGLU_BWD, the fields that mgf_gemm_desc has too as there):
 *   acc[r, c] = sum_b scale_a[r, b] * scale_b[e, b, c / 128] * sum_{k in block b} a[r, k] * b[e, k, c]
 * with fp32 accumulation of every block and of their sum.  Any fp32 scales, not only powers of two, whose products
 * scale_a * scale_b are 0 or normal fp32 numbers.  NaN is kept, in the clamps of the SwiGLU too.
 *   a       e4m3 [total_rows, k], unit stride along k, row stride lda (bytes, a multiple of 16)
 *   b       e4m3 [E, k, n]: b_mn_major 1: unit stride along n, ldb between k rows; 0: unit stride along k, ldb
 *           between columns (bytes, multiples of 16; ldb_batch between groups likewise)
 *   scale_a fp32 [total_rows, ceil(k / 128)], unit stride along the blocks, row stride scale_a_stride
 *   scale_b fp32 [E, ceil(k / 128), ceil(n / 128)] with any strides
 *   n a multiple of 8 (SWIGLU: 16), k any; outputs as for mgf_gemm_desc (16-byte rules).  Rows behind
 *   offs[E-1] are not written. */
typedef struct mgf_block_gemm_desc {
  int32_t epilogue;
  int32_t num_groups;
  int64_t total_rows, n, k; /* total_rows at most 2^31 - 257 */
  const void* a;
  int64_t lda;
  const void* b;
  int64_t ldb, ldb_batch;
  int32_t b_mn_major;
  int32_t sm_carveout;
  const int32_t* offs;
  const float* scale_a;
  int64_t scale_a_stride;
  const float* scale_b;
  int64_t scale_b_stride_e, scale_b_stride_k, scale_b_stride_n;
  const void* bias;
  int64_t bias_stride;
  void* d;
  int64_t ldd;
  void* d2;
  int64_t ldd2;
  const void* aux;
  int64_t ld_aux;
  float swiglu_alpha;
  float swiglu_limit;
  void* workspace;       /* device scratch of mgf_block_gemm_workspace_bytes(), 16-byte aligned, for this launch
                            alone while it runs; NULL = the form that needs none */
} mgf_block_gemm_desc;

/* Two forms.  Where the workspace is given and every scale of a row in a group and of B turns out (on the device) to be
 * a power of two in the normal range, the tensor cores apply the scales; otherwise every block's product is scaled
 * and added in registers.  workspace_bytes: 0 where the first form would not pay. */
int64_t mgf_block_gemm_workspace_bytes(const mgf_block_gemm_desc* desc);
int mgf_block_gemm_launch(const mgf_block_gemm_desc* desc, void* stream);
size_t mgf_block_gemm_desc_size(void);

/* Map a peer process's device allocation (its 64-byte cudaIpcMemHandle_t) into the context of
 * the calling thread's current device, peer access enabled, for mgf_push_rows destinations
 * (no counterpart in the reference).  mgf_ipc_close unmaps it. */
int mgf_ipc_open(const void* handle, void** base_out);
/* The 64-byte IPC handle of the allocation containing device pointer `ptr`, and ptr's byte offset
 * in it (what a peer passes to mgf_ipc_open, then adds the offset). */
int mgf_ipc_get_handle(const void* ptr, void* handle_out, int64_t* offset_out);
int mgf_ipc_close(void* base);

/* Read (and optionally clear) the device status word of `device`.  Synchronises that
 * device; meant for tests and debugging, never called on the hot path. */
int mgf_device_status(int device, uint32_t* status_out, int clear);

/* Human-readable text for a mgf_status code. */
const char* mgf_status_string(int status);

/* Text of the last CUDA / driver error seen by mgf_grouped_gemm_launch on this host thread
 * ("" when the last call succeeded). */
const char* mgf_last_error_detail(void);

/* Library ABI version (major * 100 + minor). */
int mgf_version(void);

/* sizeof(mgf_gemm_desc) as compiled into the library, for bindings that declare the struct
 * themselves (ctypes, cffi) to check their layout against. */
size_t mgf_gemm_desc_size(void);

#ifdef __cplusplus
}
#endif

#endif /* MOE_GEMM_H_ */

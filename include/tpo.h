/*
 * tpo.h -- C ABI of libtpo_hip.so, the MI355X (gfx950) kernels behind the
 * torch_point_ops operators chamfer / knn / fps / gather_points / emd and the
 * transformer operators layer norm / packed attention / gated projection /
 * rotary positions / 8-bit cache.
 *
 * Conventions for every entry point:
 *   - all pointers are device pointers (hipMalloc / torch CUDA-device tensors)
 *     to contiguous row-major arrays; `stream` is a hipStream_t (or NULL for
 *     the default stream) and every call is asynchronous on it;
 *   - no entry point allocates, frees or synchronises; buffers that need
 *     scratch take a caller-provided workspace sized by a *_workspace_size()
 *     query;
 *   - outputs are written completely (no pre-zeroing needed);
 *   - return 0 on success or a negative TPO_ERR_* code; tpo_last_error()
 *     returns a thread-local description of the last failure;
 *   - dtype is one of TPO_F32, TPO_F64, TPO_F16 (IEEE binary16), TPO_BF16
 *     (only where stated).
 * The functions keep no global mutable state (apart from
 * tpo_chamfer_fwd_noalloc's static device scratch and its per-device address
 * cache) and may be called from any thread.
 */
#ifndef TPO_H
#define TPO_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  TPO_F32 = 0,
  TPO_F64 = 1,
  TPO_F16 = 2,
  TPO_BF16 = 3,
  TPO_I64 = 4 /* of places (tpo_rotary, tpo_cache_append) only */
};

enum {
  TPO_OK = 0,
  TPO_ERR_ARG = -1,       /* bad size / argument */
  TPO_ERR_DTYPE = -2,     /* dtype not supported by this entry point */
  TPO_ERR_LAUNCH = -3,    /* HIP launch error (message from hipGetLastError) */
  TPO_ERR_WORKSPACE = -4  /* workspace missing or too small */
};

/* Thread-local message for the last non-zero return on this thread. */
const char* tpo_last_error(void);

/* ABI version of this header (major << 16 | minor). */
int tpo_abi_version(void);

/*
 * Chamfer forward.  Replaces chamfer_cuda_forward
 * (torch_point_ops/chamfer/csrc/cuda/chamfer.cu:169-198), the CUDA-key body
 * of torch_point_ops_chamfer::chamfer_forward (chamfer.cpp:35-36).
 *   xyz1 (B,N,3), xyz2 (B,M,3) of `dtype` (F32/F64/F16)
 *   dist1 (B,N), dist2 (B,M) of `dtype`: squared distance to the nearest
 *   point of the other cloud; idx1 (B,N), idx2 (B,M) int32: the FIRST index
 *   attaining it.  An empty other cloud gives dist 0, idx 0.
 *   workspace (optional, tpo_chamfer_workspace_size() bytes, 256-byte
 *   aligned; size 0 means none is used): with it, float and half clouds of
 *   at least 2048 points each are searched with exact spatial pruning, which
 *   is much faster on clustered or spread-out data; results are identical
 *   with or without it.
 */
int64_t tpo_chamfer_workspace_size(int dtype, int64_t B, int64_t N, int64_t M);
int tpo_chamfer_fwd(int dtype, const void* xyz1, const void* xyz2,
                    int64_t B, int64_t N, int64_t M,
                    void* dist1, void* dist2, int32_t* idx1, int32_t* idx2,
                    void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Chamfer forward that allocates nothing.  No counterpart in the reference:
 * it is for callers that cannot allocate device memory or pass a workspace
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  Same arguments and results as tpo_chamfer_fwd, bit for bit;
 * the grid-search workspace is a static device array of
 * tpo_chamfer_noalloc_max_workspace() bytes (32 MiB) that every GPU the
 * library runs on holds until the process ends.  Sizes whose workspace
 * (tpo_chamfer_workspace_size) exceeds it are rejected with
 * TPO_ERR_WORKSPACE (B=32, N=M=8192 needs about 19 MB).  All calls on one
 * device share that array: calls that overlap on one GPU (other streams or
 * threads) race; calls ordered on one stream do not.
 */
int64_t tpo_chamfer_noalloc_max_workspace(void);
int tpo_chamfer_fwd_noalloc(int dtype, const void* xyz1, const void* xyz2,
                            int64_t B, int64_t N, int64_t M,
                            void* dist1, void* dist2, int32_t* idx1, int32_t* idx2,
                            void* stream);

/*
 * Diagnostic, no counterpart in the reference: after a tpo_chamfer_fwd call
 * that used the workspace (same dtype and sizes), writes to the device
 * int64 `pairs` the number of (query, reference) pairs the pruned search
 * evaluated (a brute-force search evaluates 2*B*N*M).  Asynchronous on
 * `stream`.
 */
int tpo_chamfer_pairs_evaluated(int dtype, const void* workspace, int64_t B,
                                int64_t N, int64_t M, int64_t* pairs, void* stream);

/*
 * Chamfer backward.  Replaces chamfer_cuda_backward (chamfer.cu:236-271),
 * torch_point_ops_chamfer::chamfer_backward (chamfer.cpp:37-38).
 *   grad_dist1 (B,N), grad_dist2 (B,M) of `dtype`
 *   grad_xyz1 (B,N,3), grad_xyz2 (B,M,3) of `dtype`:
 *     grad_xyz1[i] =  2 g1[i] (x1_i - x2_idx1[i]) - sum_{j: idx2[j]=i} 2 g2[j] (x2_j - x1_i)
 *   (and symmetrically), the scatter summed by atomics in unspecified order.
 */
int tpo_chamfer_bwd(int dtype, const void* xyz1, const void* xyz2,
                    const int32_t* idx1, const int32_t* idx2,
                    const void* grad_dist1, const void* grad_dist2,
                    int64_t B, int64_t N, int64_t M,
                    void* grad_xyz1, void* grad_xyz2, void* stream);

/*
 * Chamfer loss: ChamferDistance(reduction="mean" / "sum")
 * (torch_point_ops/chamfer/chamfer.py:18-24) in one forward and one
 * backward call.  No single counterpart in the reference, which reduces
 * chamfer_forward's distances with torch.mean / torch.sum; these entry points
 * fuse that reduction into the forward and the reduction's gradient into the
 * backward.
 *   loss (one element of `dtype`): mean != 0: mean(dist1) + mean(dist2)
 *     (NaN when a cloud is empty, like torch.mean); mean == 0: sum + sum.
 *     The sums are taken in a fixed order, so the loss is deterministic; it
 *     matches torch's reduction of tpo_chamfer_fwd's distances to rounding.
 *   idx1, idx2 as tpo_chamfer_fwd (the backward needs them); the distances
 *   themselves are not stored.
 *   workspace (required): tpo_chamfer_loss_workspace_size() bytes, 256-byte
 *   aligned, contents need not be initialised.
 * tpo_chamfer_loss_bwd: grad_loss is ONE device element of `dtype`; the
 *   gradients equal tpo_chamfer_bwd's with grad_dist = grad_loss / numel
 *   (mean, multiplied by the reciprocal as torch's MeanBackward does) or
 *   grad_loss (sum) for every point.
 */
int64_t tpo_chamfer_loss_workspace_size(int dtype, int64_t B, int64_t N, int64_t M);
int tpo_chamfer_loss_fwd(int dtype, const void* xyz1, const void* xyz2,
                         int64_t B, int64_t N, int64_t M, int mean, void* loss,
                         int32_t* idx1, int32_t* idx2,
                         void* workspace, int64_t workspace_bytes, void* stream);
int tpo_chamfer_loss_bwd(int dtype, const void* xyz1, const void* xyz2,
                         const int32_t* idx1, const int32_t* idx2,
                         const void* grad_loss, int mean,
                         int64_t B, int64_t N, int64_t M,
                         void* grad_xyz1, void* grad_xyz2, void* stream);

/*
 * KNN forward.  Replaces knn_cuda_forward
 * (torch_point_ops/knn/csrc/cuda/knn.cu:295-398),
 * torch_point_ops_knn::knn_forward (knn.cpp:168-169).
 *   p1 (N,P1,D), p2 (N,P2,D) of `dtype`; lengths1/lengths2 (N) int64
 *   (clamped to [0,P1] / [0,P2]); norm 1 or 2; K >= 1; version -1 for
 *   automatic, 0..3 to force one of the reference's kernel semantics (an
 *   invalid choice falls back to automatic, as the reference does).
 *   F32/F64/F16: idxs (N,P1,K) int64 and dists (N,P1,K) `dtype`, unsorted,
 *   laid out exactly as the reference's MinK slots, including its padding
 *   rules: rows >= lengths1 are (0,0); slots >= lengths2 are (0,0) for
 *   versions 2/3 and (-1,+inf) for versions 0/1.  workspace is optional
 *   (tpo_knn_workspace_size bytes): with it the queries are processed in
 *   spatial order, which is faster; results are identical.
 *   BF16 (no reference kernel; the reference raises): norm 2, D % 8 == 0,
 *   8 <= D <= 128, K <= 32, points 16-byte aligned, workspace required.
 *   Squared distances |q|^2 + |r|^2 - 2 q.r in float, summed on the matrix
 *   cores (the norms, float sums of the bf16 squares, enter as exact
 *   three-piece bf16 splits), clamped at 0; each row's K nearest sorted by
 *   (distance, index), dists rounded to bfloat16; rows >= lengths1 and
 *   slots >= lengths2 are (0,0).  version is ignored and version_out
 *   receives -1.  For P2 >= max(4096, 1536 K) the workspace also holds a
 *   per-query bound sampled from 64 tiles of 32 references, the candidates
 *   at or below it (up to 128 per query and reference slice) and a list of
 *   the rows that overflowed or fell short (and every row of a cloud whose
 *   lengths2 is below that size), which are recomputed without it; results
 *   do not depend on it.
 *   If version_out is not NULL it receives the version that ran.
 */
int64_t tpo_knn_workspace_size(int dtype, int64_t N, int64_t P1, int64_t P2,
                               int64_t D, int64_t K, int norm);
int tpo_knn_fwd(int dtype, const void* p1, const void* p2,
                const int64_t* lengths1, const int64_t* lengths2,
                int64_t N, int64_t P1, int64_t P2, int64_t D, int64_t K,
                int norm, int version, int64_t* idxs, void* dists,
                int* version_out, void* workspace, int64_t workspace_bytes,
                void* stream);

/*
 * KNN forward with the rows sorted the way knn_points(return_sorted=True)
 * returns them (torch_point_ops/knn/__init__.py:111-131: torch's sort of
 * each row after the forward, slots past lengths2 keyed +inf, then zeroed).
 * No single counterpart in the reference: the forward and the module's sort
 * in one launch.  F32/F64/F16 with 2 <= K <= 32 only; arguments and padding
 * as tpo_knn_fwd.  Each row is sorted by replaying torch's 32-wide bitonic
 * network, so equal distances come out in the same order as torch.sort
 * puts them.
 */
int tpo_knn_fwd_sorted(int dtype, const void* p1, const void* p2,
                       const int64_t* lengths1, const int64_t* lengths2,
                       int64_t N, int64_t P1, int64_t P2, int64_t D, int64_t K,
                       int norm, int version, int64_t* idxs, void* dists,
                       int* version_out, void* workspace, int64_t workspace_bytes,
                       void* stream);

/*
 * Sorts the rows (N,P1,K) of a BF16 tpo_knn_fwd in place, K <= 32, as
 * tpo_knn_fwd_sorted sorts the other types' rows.
 */
int tpo_knn_sort_rows(int dtype, const int64_t* lengths2, int64_t N, int64_t P1, int64_t K,
                      int64_t* idxs, void* dists, void* stream);

/*
 * Bytes of workspace with which tpo_knn_fwd_sorted, and tpo_knn_fwd with
 * K = 1, select rows by distance (float: cell grid for D = 3, matrix cores for
 * D = 4 .. 128 with norm 2).  At least tpo_knn_workspace_size, with which the
 * same rows come from the insertion-order kernels.
 */
int64_t tpo_knn_rows_workspace_size(int dtype, int64_t N, int64_t P1, int64_t P2, int64_t D,
                                    int64_t K, int norm);

/*
 * knn_gather forward.  Replaces the expand + gather + mask of
 * knn_gather (torch_point_ops/knn/__init__.py:136-183), which the reference
 * runs as torch ops.
 *   x (N,M,U), idx (N,L,K) int64, lengths (N) int64 valid counts of x;
 *   out (N,L,K,U) of `dtype` (F32/F64/F16/BF16): out[n,l,k] = x[n, idx[n,l,k]]
 *   for k < lengths[n], else 0 (and 0 for an index outside [0, M)).
 */
int tpo_knn_gather(int dtype, const void* x, const int64_t* idx,
                   const int64_t* lengths, int64_t N, int64_t M, int64_t L, int64_t K,
                   int64_t U, void* out, void* stream);

/*
 * knn_gather backward: grad_x (N,M,U) = the sum of grad_out (N,L,K,U) over the
 * entries (l, k), k < lengths[n], by row idx[n,l,k] (clamped to [0, M)); every
 * row is written.  F32/F64/F16; half sums are taken in float and rounded once.
 * The workspace size is 0 where the call does not apply (U > 7, very long
 * clouds, no entries) and the call then returns TPO_ERR_ARG.
 */
int64_t tpo_knn_gather_bwd_workspace_size(int dtype, int64_t N, int64_t M, int64_t L, int64_t K,
                                          int64_t U);
int tpo_knn_gather_bwd(int dtype, const void* grad_out, const int64_t* idx,
                       const int64_t* lengths, int64_t N, int64_t M, int64_t L, int64_t K,
                       int64_t U, void* grad_x, void* workspace, int64_t workspace_bytes,
                       void* stream);

/*
 * KNN backward.  Replaces knn_cuda_backward (knn.cu:469-534),
 * torch_point_ops_knn::knn_backward (knn.cpp:170-171).
 *   idxs / grad_dists (N,P1,K); grad_p1 (N,P1,D), grad_p2 (N,P2,D) `dtype`.
 *   Rows >= lengths1 and slots with idx == -1 contribute nothing; L2:
 *   diff = (2 g)(p1 - p2); L1: diff = g sign(p1 - p2) with sign(0) = 0;
 *   grad_p1 += diff, grad_p2[idx] -= diff.
 */
int tpo_knn_bwd(int dtype, const void* p1, const void* p2,
                const int64_t* lengths1, const int64_t* lengths2,
                const int64_t* idxs, int norm, const void* grad_dists,
                int64_t N, int64_t P1, int64_t P2, int64_t D, int64_t K,
                void* grad_p1, void* grad_p2, void* stream);

/*
 * tpo_knn_bwd with a workspace (the same reference function,
 * knn_cuda_backward, knn.cu:469-534).  With workspace_bytes >=
 * tpo_knn_bwd_workspace_size() (non-zero for D <= 7, K <= 256 and
 * reference clouds up to ~750 K points) grad_p2 is accumulated without
 * global atomics: the terms are grouped by reference rows in the workspace
 * and each group is summed in LDS.  A smaller or NULL workspace runs the
 * atomic scatter of tpo_knn_bwd.  workspace: 256-byte aligned.
 */
int64_t tpo_knn_bwd_workspace_size(int dtype, int64_t N, int64_t P1, int64_t P2, int64_t D,
                                   int64_t K);
int tpo_knn_bwd_ws(int dtype, const void* p1, const void* p2,
                   const int64_t* lengths1, const int64_t* lengths2,
                   const int64_t* idxs, int norm, const void* grad_dists,
                   int64_t N, int64_t P1, int64_t P2, int64_t D, int64_t K,
                   void* grad_p1, void* grad_p2, void* workspace, int64_t workspace_bytes,
                   void* stream);

/*
 * Furthest point sampling.  Replaces fps_cuda_forward
 * (torch_point_ops/fps/csrc/cuda/fps.cu:273-315),
 * torch_point_ops_fps::fps_forward (fps.cpp:159).
 *   points (B,N,3) `dtype` (F32/F64/F16), 1 <= nsamples <= N;
 *   idx (B,nsamples) int64, identical to the reference kernel including its
 *   skip rule (|p|^2 <= 1e-3 never selected), start index 0 and tie order.
 *   workspace: tpo_fps_workspace_size(dtype, B, N) bytes, 256-byte aligned.
 */
int64_t tpo_fps_workspace_size(int dtype, int64_t B, int64_t N);
int tpo_fps_fwd(int dtype, const void* points, int64_t B, int64_t N,
                int64_t nsamples, int64_t* idx,
                void* workspace, int64_t workspace_bytes, void* stream);

/*
 * gather_points forward.  Replaces gather_points_cuda_forward
 * (fps.cu:318-357), torch_point_ops_fps::gather_points_forward (fps.cpp:160).
 *   points (B,C,N), idx (B,M) int64 in [0,N), out (B,C,M).  F32/F64/F16.
 */
int tpo_gather_fwd(int dtype, const void* points, const int64_t* idx,
                   int64_t B, int64_t C, int64_t N, int64_t M, void* out,
                   void* stream);

/*
 * gather_points backward.  Replaces gather_points_cuda_backward
 * (fps.cu:360-404), torch_point_ops_fps::gather_points_backward
 * (fps.cpp:161).
 *   grad_out (B,C,M), idx (B,M) int64, grad_points (B,C,N):
 *   zeros + scatter-add of grad_out at idx (duplicates sum).
 *   workspace: tpo_gather_bwd_workspace_size(B, N) bytes.
 */
int64_t tpo_gather_bwd_workspace_size(int64_t B, int64_t N);
int tpo_gather_bwd(int dtype, const void* grad_out, const int64_t* idx,
                   int64_t B, int64_t C, int64_t N, int64_t M,
                   void* grad_points, void* workspace, int64_t workspace_bytes,
                   void* stream);

/*
 * Earth mover's distance (approximate matching).
 *
 * tpo_emd_fwd replaces emd_cuda_forward (emd.cu:305-347: approxmatch
 * emd.cu:18-183 + matchcost emd.cu:187-230), the CUDA kernel of
 * torch_point_ops_emd::emd_forward (emd.cpp:32).
 *   xyz1 (B,n,3), xyz2 (B,m,3) -> cost (B) (the matching cost before the
 *   Python wrapper's division by n) and match (B,m,n).  F32/F64/F16.
 *   n == 0 or m == 0: cost = 0 and match is empty (emd.cu:313-318).
 *   Deterministic; within a tolerance of the reference (its exponential is
 *   CUDA's, this one is ROCm's, and the sums run in another order).
 * tpo_emd_bwd replaces emd_cuda_backward (emd.cu:349-389: matchcostgrad1
 * emd.cu:234-257 + matchcostgrad2 emd.cu:261-303), the kernel of
 * torch_point_ops_emd::emd_backward (emd.cpp:33).
 *   grad_cost (B), match (B,m,n) -> grad_xyz1 (B,n,3), grad_xyz2 (B,m,3).
 * Both take a workspace of tpo_emd_workspace_size(dtype, B, n, m) bytes,
 * 256-byte aligned (0 bytes when B, n or m is 0).  B < 2^31; n, m < 2^30.
 */
int64_t tpo_emd_workspace_size(int dtype, int64_t B, int64_t n, int64_t m);
int tpo_emd_fwd(int dtype, const void* xyz1, const void* xyz2, int64_t B,
                int64_t n, int64_t m, void* cost, void* match,
                void* workspace, int64_t workspace_bytes, void* stream);
int tpo_emd_bwd(int dtype, const void* grad_cost, const void* xyz1,
                const void* xyz2, const void* match, int64_t B, int64_t n,
                int64_t m, void* grad_xyz1, void* grad_xyz2,
                void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Transformer operators.  No counterpart in the reference: what a model over
 * point patches runs between the grouping above and a loss on clouds.
 * F32/F16/BF16; sums are taken in float and outputs rounded once.
 *
 * Layer norm over the last axis of x (rows, width):
 *   y = (x - mean) rstd weight + bias, rstd = 1 / sqrt(var + eps), var the
 *   mean square about the mean.
 *   weight, bias (width) of `wdtype` (x's dtype or F32); NULL for 1 and 0.
 *   mean, rstd (rows) float: what the backward needs; both NULL to leave out.
 *   1 <= width <= 2^20, rows < 2^31.
 * tpo_layer_norm_bwd: grad_x (rows, width) of `dtype`, grad_weight and
 *   grad_bias (width) of `wdtype`; each may be NULL and is then left out.
 *   The sums over rows run in a fixed order.  The workspace is needed where
 *   grad_weight or grad_bias is asked for.
 */
int tpo_layer_norm_fwd(int dtype, int wdtype, const void* x, const void* weight,
                       const void* bias, int64_t rows, int64_t width, double eps,
                       void* y, float* mean, float* rstd, void* stream);
int64_t tpo_layer_norm_bwd_workspace_size(int64_t rows, int64_t width);
int tpo_layer_norm_bwd(int dtype, int wdtype, const void* grad_y, const void* x,
                       const void* weight, const float* mean, const float* rstd,
                       int64_t rows, int64_t width, double eps, void* grad_x,
                       void* grad_weight, void* grad_bias, void* workspace,
                       int64_t workspace_bytes, void* stream);

/*
 * Softmax attention over packed sequences, with grouped heads.
 *   q (Tq,Hq,D), k and v (Tk,Hk,D), Hq a multiple of Hk (query head h reads
 *   key head h / (Hq / Hk)), 1 <= D <= 128.  These three may be strided:
 *   *_row and *_head are the strides, in elements, of a row and of a head;
 *   the D values of a head are contiguous.
 *   offsets_q, offsets_k (B + 1) int64, not decreasing: sequence b has the
 *   rows offsets[b] .. offsets[b + 1].  lengths_q, lengths_k (B) int64 or
 *   NULL: how many of these rows, from the first, are in use (the others are
 *   not read: a cache with room to grow).  Bounds are clamped to the arrays.
 *   causal: row i of a sequence sees key j where j <= i + (keys - rows): the
 *   last row sees every key.
 *   out (Tq,Hq,D) contiguous; rows not in use, and rows that see no key, are 0.
 *   lse (Hq,Tq) float: log of the sum of exponentials of each row (-inf for
 *   a row that sees no key), what the backward needs; NULL to leave out.
 *   rest (as out) or NULL: what rounding to the type took from out, for a
 *   more exact backward; of no use with F32.
 *   Pointers, heads (D values) and strides are multiples of 16 bytes, a row's
 *   stride is 16 to 2^25 bytes.
 *   B <= 2^24, Hq <= 1024, Tq Hq and Tk Hk < 2^31.
 *   A NaN or an infinity in v reaches the rows that see it and, by 0 times it,
 *   earlier rows of the sequence that share a tile of 64 keys with it; it
 *   reaches no row of another sequence, and rows not in use are not read.  In
 *   the backward one in q, k or grad_out likewise reaches gradients of keys and
 *   rows of its tile that do not see each other.
 * tpo_attention_bwd: grad_out, out, rest and the gradients are contiguous.  Every
 *   row of grad_q, grad_k, grad_v is written, rows not in use with 0; sums
 *   run in a fixed order.  grad_q, or grad_k and grad_v together, may be NULL and
 *   are left out; without grad_k and grad_v no workspace is needed.
 * Workspaces are 256-byte aligned; size 0 means none is used.
 * tpo_attention_fwd_rows is a diagnostic: the query rows (tokens times the heads
 *   of a group) that a workgroup of the forward takes for these sizes, 128 where
 *   it loads its keys once for all of them, 32 where waves share the keys.
 */
int tpo_attention_fwd_rows(int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq,
                           int64_t Hk, int64_t D);
int64_t tpo_attention_fwd_workspace_size(int dtype, int64_t B, int64_t Tq, int64_t Tk,
                                         int64_t Hq, int64_t Hk, int64_t D);
int tpo_attention_fwd(int dtype, const void* q, const void* k, const void* v,
                      const int64_t* offsets_q, const int64_t* offsets_k,
                      const int64_t* lengths_q, const int64_t* lengths_k, int64_t B,
                      int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                      int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                      int64_t v_row, int64_t v_head, int causal, double scale,
                      void* out, float* lse, void* rest, void* workspace,
                      int64_t workspace_bytes, void* stream);
int64_t tpo_attention_bwd_workspace_size(int dtype, int64_t B, int64_t Tq, int64_t Tk,
                                         int64_t Hq, int64_t Hk, int64_t D);
int tpo_attention_bwd(int dtype, const void* grad_out, const void* q, const void* k,
                      const void* v, const void* out, const void* rest,
                      const float* lse,
                      const int64_t* offsets_q, const int64_t* offsets_k,
                      const int64_t* lengths_q, const int64_t* lengths_k, int64_t B,
                      int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                      int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                      int64_t v_row, int64_t v_head, int causal, double scale,
                      void* grad_q, void* grad_k, void* grad_v, void* workspace,
                      int64_t workspace_bytes, void* stream);

/*
 * Gated projection: h = act(x w_gate^T) * (x w_up^T).
 *   x (M,K), w_gate and w_up (F,K), h (M,F), M <= 2^22, 1 <= K <= 2^20,
 *   F <= 2^20; activation is a TPO_ACT_* code (GELU is x times the normal
 *   distribution function, by erf).
 * tpo_gated_bwd: grad_h (M,F) -> grad_x (M,K), grad_w_gate and grad_w_up
 *   (F,K).  The gradients at the projections are rounded to `dtype` between
 *   the products.  grad_x, or the two weights' gradients together, may be NULL
 *   and are left out.
 *   keep (M,2F), F32 only, or NULL: the forward's projections, which the
 *   backward then takes as kept; with NULL it computes them again (as it
 *   always does for the half types, whose products take less time than
 *   unrounded projections take through memory).
 * x, the weights and the workspace are 16-byte aligned.
 * Workspaces are 256-byte aligned; size 0 means none is used.
 */
enum {
  TPO_ACT_SILU = 0,
  TPO_ACT_GELU = 1,
  TPO_ACT_RELU = 2,
  TPO_ACT_SIGMOID = 3
};
int64_t tpo_gated_fwd_workspace_size(int dtype, int64_t M, int64_t K, int64_t F);
int tpo_gated_fwd(int dtype, const void* x, const void* w_gate, const void* w_up,
                  int64_t M, int64_t K, int64_t F, int activation, void* h,
                  void* keep, void* workspace, int64_t workspace_bytes, void* stream);
int64_t tpo_gated_bwd_workspace_size(int dtype, int64_t M, int64_t K, int64_t F);
int tpo_gated_bwd(int dtype, const void* grad_h, const void* x, const void* w_gate,
                  const void* w_up, const void* kept, int64_t M, int64_t K, int64_t F,
                  int activation, void* grad_x, void* grad_w_gate, void* grad_w_up, void* workspace,
                  int64_t workspace_bytes, void* stream);

/*
 * Rotary positions: pairs of a head's values turned by angles that grow with a
 * token's place.
 *   y1 = m (x1 cos a - x2 sin a), y2 = m (x2 cos a + x1 sin a), a = place f_j,
 *   pair j being values j and j + pairs of a head (interleaved: 2 j and
 *   2 j + 1), m the amplitude; the D - 2 pairs values behind stay as they are.
 *   x (tokens,heads,D) strided: x_row and x_head are the strides, in elements,
 *   of a token and of a head; the D values of a head are contiguous.  y
 *   contiguous, not x.  Any alignment.  1 <= D <= 512, heads <= 2^16.
 *   places (tokens,axes) of places_dtype (I64 or F32), frequencies (pairs)
 *   double: pair j goes by axis j / (pairs / axes).  Angles are taken in 64 bits;
 *   those beyond 2^45 give NaN.
 *   back: the angles' signs turned, which makes it the gradient.
 */
int tpo_rotary(int dtype, const void* x, int64_t tokens, int64_t heads, int64_t D,
               int64_t x_row, int64_t x_head, const void* places, int places_dtype,
               int64_t axes, const double* frequencies, int64_t pairs, int interleaved,
               double amplitude, int back, void* y, void* stream);

/*
 * A cache of keys and values in pages of 8-bit codes (e4m3: 448 the largest, no
 * infinities), Dr being D rounded up to 16:
 *   keys (pages,Hk,page/32,Dr/16,32,16), values (pages,Hk,page/32,Dr,32),
 *   key_scales and value_scales (pages,Hk) float, positive: a value is its code
 *   times the scale of its page and head; 16-byte aligned.
 *   table (B,M) int32: the pages of each sequence in order.  An entry outside of
 *   [0, pages) is a page that is not there: nothing is written to it, and its
 *   places are not seen.  lengths (B) int64: the tokens of each sequence, those
 *   that a call brings included, clamped to M page.
 *   page is 32 to 256 in steps of 32, 1 <= D <= 128, M page <= 2^30.
 * The rows of a call (T) belong to the sequences as those of the packed
 * attention do: offsets (B + 1) int64, lengths_new or lengths_q (B) int64 or
 * NULL.  The n rows of a sequence that are in use are its last n tokens.
 *
 * tpo_cache_append puts k and v (T,Hk,D) into the pages, k turned by its places
 *   as tpo_rotary turns (pairs = 0: as it is) in 64 bits and rounded once.  places
 *   (T,axes) or NULL for the tokens' own places in their sequences.  Scales are
 *   powers of two, 2^-40 to 2^40, the smallest with every value of the page at
 *   most 448 times it: a page whose first token is new gets its own, one that
 *   holds older tokens keeps its scale or, where a new token needs it, grows, and
 *   its older codes are rounded to the new one.  What is not finite becomes the
 *   code for NaN, what is beyond 448 2^40 that value.  No two sequences of a call
 *   may write to one page.  Nothing but the new tokens' codes, the codes before
 *   them in a page whose scale grows, and the scales of these pages is written.
 *   q (T,Hq,D) or NULL: turned likewise into q_out (T,Hq,D) contiguous, of
 *   k's type; rows not in use are 0.
 * tpo_cache_attention: softmax(scale q k^T) v over the cache, into out (T,Hq,D)
 *   contiguous.  Causal: row i of a sequence's n sees place j where
 *   j <= i + length - n.  Rows not in use, and rows that see no key, are 0.
 *   What lies behind a sequence's last token is read but never counts, whatever
 *   it holds.  q as the packed attention takes it.
 * Workspaces are 256-byte aligned; size 0 means none is used.
 * tpo_cache_attention_rows is a diagnostic, as tpo_attention_fwd_rows: 128 where a
 *   workgroup converts its codes once for as many rows, else 32.
 */
int tpo_cache_append(int dtype, const void* k, const void* v, const void* q,
                     const int64_t* offsets, const int64_t* lengths_new, int64_t B,
                     int64_t T, int64_t Hq, int64_t D, int64_t k_row, int64_t k_head,
                     int64_t v_row, int64_t v_head, int64_t q_row, int64_t q_head,
                     const void* places, int places_dtype, int64_t axes,
                     const double* frequencies, int64_t pairs, int interleaved,
                     double amplitude, void* keys, void* values, float* key_scales,
                     float* value_scales, const int32_t* table, const int64_t* lengths,
                     int64_t pages, int64_t Hk, int64_t page, int64_t Dr, int64_t M,
                     void* q_out, void* stream);
int64_t tpo_cache_attention_workspace_size(int dtype, int64_t B, int64_t T, int64_t Hq,
                                           int64_t Hk, int64_t D, int64_t page, int64_t M);
int tpo_cache_attention_rows(int dtype, int64_t B, int64_t T, int64_t Hq, int64_t Hk,
                             int64_t D, int64_t page, int64_t M);
int tpo_cache_attention(int dtype, const void* q, const int64_t* offsets,
                        const int64_t* lengths_q, int64_t B, int64_t T, int64_t Hq,
                        int64_t D, int64_t q_row, int64_t q_head, const void* keys,
                        const void* values, const float* key_scales,
                        const float* value_scales, const int32_t* table,
                        const int64_t* lengths, int64_t pages, int64_t Hk, int64_t page,
                        int64_t Dr, int64_t M, int causal, double scale, void* out,
                        void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TPO_H */

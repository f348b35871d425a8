/*
 * alsmi — MI355X (gfx950) kernels for the ALS / IMC / DirtyIMC update loop.
 *
 * C ABI of libalsmi.so.  The upstream project (GrierPhillips/Recommendation-Models)
 * is pure Python and has no FFI of its own; each entry point below replaces the
 * numpy/scipy arithmetic of the cited reference lines and is bound from Python
 * with ctypes (recommendation-models_amd/alsmi/_lib.py is that binding).
 *
 * Conventions
 *  - every function returns 0 on success and a negative ALSMI_E* code on failure;
 *    alsmi_last_error() gives the message of the calling thread's last failure.
 *    No C++ exception crosses the boundary.
 *  - pointers named *_host are host memory, everything else is DEVICE memory on
 *    the current HIP device, owned by the caller, and only used during the call
 *    (kernels are enqueued on `stream`; the call does not synchronise unless it
 *    says so).
 *  - `dtype` is ALSMI_F32 or ALSMI_F64 and fixes the element type of every
 *    `void*` factor / rating / attribute buffer of that call.
 *  - factor tables are ROW-major [n x ld] with ld = alsmi_padded_rank(rank)
 *    (16, 32, 64 or 128); columns rank..ld-1 must be zero.  The reference keeps
 *    (rank, n) C-order arrays (src/als.py:149-151); the host binding transposes.
 *  - sparse structure: `indptr` int64 [n_rows+1], `indices` int32 [nnz] sorted
 *    inside a row, `vals` [nnz] of dtype.  For the item side pass the CSC arrays.
 *  - calls that share a plan or a workspace must not overlap in time.
 */
#ifndef ALSMI_H
#define ALSMI_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ALSMI_F32 0
#define ALSMI_F64 1
/* taken by the ranking operators (alsmi_mx4_*, alsmi_adjust_scores, alsmi_topk_rows) only */
#define ALSMI_F16 2
#define ALSMI_BF16 3
#define ALSMI_MX4 4 /* alsmi_mx4_scores: activations as codes and scales */

#define ALSMI_OK 0
#define ALSMI_EINVAL (-1)   /* bad argument (shape, dtype, rank, null pointer) */
#define ALSMI_EHIP (-2)     /* a HIP runtime call failed */
#define ALSMI_ENOMEM (-3)   /* allocation failed */

typedef struct alsmi_plan alsmi_plan;

/* Library version (major*10000 + minor*100 + patch). */
int alsmi_version(void);

/* Message of the last error raised on the calling thread ("" if none). */
const char *alsmi_last_error(void);

/* Row stride (in elements) of a factor table for `rank`: the next of
 * 16/32/64/128 that is >= rank; 0 if rank is < 1 or > 128. */
int alsmi_padded_rank(int rank);

/* ---- ALS half-sweep: src/als.py:173-300 (_update_parallel,
 * _thread_update_features, _update_one, make_item_submats, make_user_submats) --
 *
 * A plan is the schedule of one side's half-sweep over rows
 * [row_begin, row_end) of a structure with n_rows_total rows: rows ordered by
 * degree, rows longer than `chunk` entries cut into chunks whose partial normal
 * equations are combined in a fixed order.  It replaces the reference's
 * np.array_split chunking (src/als.py:155-159).  It owns a little device memory
 * (work lists and the partial-sum workspace) allocated at creation on the
 * current device; no call on the plan allocates afterwards.
 * `chunk` = 0 picks the default.  Synchronous. */
int alsmi_plan_create(alsmi_plan **out, const int64_t *indptr_host,
                      int64_t n_rows_total, int64_t row_begin, int64_t row_end,
                      int rank, int dtype, int chunk);
int alsmi_plan_destroy(alsmi_plan *plan);
/* Any out pointer may be NULL. */
int alsmi_plan_info(const alsmi_plan *plan, int64_t *n_rows, int64_t *n_heavy_rows,
                    int64_t *n_chunks, int64_t *workspace_bytes);

/* For every row r of the plan:
 *   A = sum_t f_t f_t^T + alpha*n_r*I,  b = sum_t vals_t f_t,  dst[r] = A^-1 b
 * with f_t = src_factors[indices[t]] over the row's n_r stored entries
 * (src/als.py:243-247); an empty row or a matrix that is not positive definite
 * gives a zero vector (the reference's LinAlgError branch, src/als.py:248-249).
 * Rows outside the plan's range are not touched.
 * ALSMI_F32: the products f f^T are formed on the fp16 matrix cores
 * from values scaled by a power of two taken from the largest |element| of the
 * source table (read once per call); the result has fp32 accuracy for
 * 2^-40 <= max|src| <= 2^40, elements below max|src| * 2^-16 lose precision
 * relative to themselves only.  An fp32 source table above 4 GiB is accepted
 * at padded rank 128 (64-bit gather addresses are switched in) and rejected
 * with ALSMI_EINVAL at padded rank <= 64 (more than 16.7 M rows).  At padded
 * rank 64 / 128 rows of at most 48 / 64 stored entries — and never more than
 * `rank` of them — are solved in the equivalent n x n form
 * x = F^T (F F^T + alpha n I)^-1 vals; with alpha = 0
 * such a row gets the minimum-norm least-squares solution where the rank x rank
 * matrix of the reference is singular.  Results are bit-reproducible from run
 * to run. */
int alsmi_half_sweep(alsmi_plan *plan, const int64_t *indptr, const int32_t *indices,
                     const void *vals, const void *src_factors, int64_t n_src,
                     void *dst_factors, double alpha, void *stream);

/* The same half-sweep, which also returns the squared training error of the factors it
 * REPLACES: sse_out[0] (one double, device) = sum over the stored entries t of the plan's
 * rows of (vals_t - <cur_factors[r], f_t>)^2, the quantity the reference computes in a
 * separate pass after every sweep (src/als.py:161-165).  The kernels read every f_t anyway,
 * so the error of sweep s comes for free with the user half of sweep s+1.  cur_factors is
 * indexed like dst_factors and may be the same table (a row is read before it is
 * written).  Partial sums are combined in a fixed order. */
int alsmi_half_sweep_err(alsmi_plan *plan, const int64_t *indptr, const int32_t *indices,
                         const void *vals, const void *src_factors, int64_t n_src,
                         const void *cur_factors, void *dst_factors, double alpha,
                         double *sse_out, void *stream);

/* Debug / test aid: the assembled normal equations of the plan's rows before the
 * solve.  A_out [n_rows x ld x ld], b_out [n_rows x ld], both indexed by
 * (row - row_begin), natural (unpermuted) order, ridge included. */
int alsmi_normal_equations(alsmi_plan *plan, const int64_t *indptr, const int32_t *indices,
                           const void *vals, const void *src_factors, int64_t n_src,
                           void *A_out, void *b_out, double alpha, void *stream);

/* ---- pair predictions and squared error: src/als.py:161-165 (train RMSE),
 * :316-321 (_predict), :383-388 (score) ------------------------------------
 *
 * pred_p = <row_factors[users[p]], col_factors[items[p]]> for p < n_pairs.
 * pred_out (dtype, [n_pairs]) may be NULL.  If vals is not NULL, sse_out[0]
 * (one double) receives sum_p (vals[p]-pred_p)^2 accumulated in fp64 in a fixed
 * order.  workspace: at least alsmi_sddmm_workspace_bytes() bytes. */
size_t alsmi_sddmm_workspace_bytes(void);
int alsmi_sddmm(int dtype, int rank, int64_t n_pairs, const int32_t *users,
                const int32_t *items, const void *row_factors, const void *col_factors,
                const void *vals, void *pred_out, double *sse_out, void *workspace,
                void *stream);

/* alsmi_sddmm for callers that cannot allocate or hand over a workspace (code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc).  It has no
 * counterpart in the reference.  Same arguments and results as alsmi_sddmm without the
 * workspace: the per-block partial sums live in a 16 KiB device array that is part of the
 * library image (one copy per GPU, held until the process ends), and the call performs no
 * hipMalloc / hipFree.  At most ALSMI_SDDMM_NOALLOC_MAX_PAIRS pairs per call (more is
 * ALSMI_EINVAL).  All calls on one GPU share that array: calls that overlap in time on one
 * GPU (different streams or threads) race on sse_out; pred_out is unaffected.
 * The FIRST call on a device looks the array's address up (hipGetSymbolAddress, which makes
 * the runtime load the library's code object there and may allocate inside the runtime):
 * make one warm-up call per device outside any stream capture; every later call on that
 * device only enqueues kernels. */
#define ALSMI_SDDMM_NOALLOC_MAX_PAIRS ((int64_t)1 << 28)
int alsmi_sddmm_noalloc(int dtype, int rank, int64_t n_pairs, const int32_t *users,
                        const int32_t *items, const void *row_factors, const void *col_factors,
                        const void *vals, void *pred_out, double *sse_out, void *stream);

/* ---- the k best items of a batch of users: src/als.py:347-364 (predict_all returns one
 * user's score for every item and leaves the ranking to the caller) -----------------
 *
 * For every p < n_sel: the k items i with the largest <user_factors[users[p]],
 * item_factors[i]>, best first, ties broken by the smaller item id; items_out [n_sel x k]
 * int32, scores_out [n_sel x k] of dtype.  1 <= k <= min(1024, n_items), n_items <= 16 776 960.
 * workspace: at least
 * alsmi_topk_workspace_bytes(dtype, n_sel, n_items) bytes (room for the dense n_sel x n_items
 * score block: batch the users accordingly).  From 8192 items on and for small k (about
 * k <= n_items / 170) the block is not written: a strided sample of the item tiles gives every
 * user a lower bound of its k-th best score, a pass over all items keeps only the scores at
 * or above it, and those candidates are sorted; a user with more candidates than there are
 * slots (many equal scores) switches the whole call back to the dense block, on the device,
 * with the same result.  ALSMI_F32 scores are formed on the fp16 matrix cores from a scaled
 * two-way fp16 split of both tables (scales from the largest |factor| of the selected users
 * and of the items): fp32 accuracy, the same bits for the same pair of vectors within a
 * call.  ALSMI_F64 in that form: the candidates come from the fp32 pass on the tables rounded
 * to fp32, with every user's threshold lowered by twice a bound of the fp32 scores' error
 * (2^-13 |u| max_i |v_i|), and those within that distance of the user's k-th best fp32 score
 * are scored again in fp64 from the fp64 tables and ranked by those scores — the lists are
 * those of fp64 scores of all items; the last bits of a score may differ from the dense block's
 * (another summation order), i.e. between calls that batch the users differently.
 * ALSMI_TOPK_F64_PREFILTER=0: fp64 scores of all items on the fp64 matrix pipe instead.
 * Deterministic.  Scores are ranked by their bit
 * pattern in the total order of IEEE 754: -0.0 ranks below +0.0 (they do not tie), and a NaN
 * score with a clear sign bit ranks above +infinity, i.e. first (one with the sign bit set
 * below -infinity, last); finite factor tables never produce one. */
size_t alsmi_topk_workspace_bytes(int dtype, int64_t n_sel, int64_t n_items);
int alsmi_topk_items(int dtype, int rank, int64_t n_sel, const int32_t *users,
                     const void *user_factors, const void *item_factors, int64_t n_items, int k,
                     int32_t *items_out, void *scores_out, void *workspace, void *stream);

/* The dense score block that alsmi_topk_items ranks: out [n_sel x n_items] of dtype,
 * out[p, i] = <user_factors[users[p]], item_factors[i]>, by the same kernels (ALSMI_F32: scaled fp16
 * split, fp32 accuracy).  For callers that change the scores before they select from them.
 * alsmi_score_rows takes the number of rows of user_factors: an id outside 0 .. n_users-1 gives a row
 * of NaN.  alsmi_score_items leaves it to its caller that users[] are rows of user_factors.
 * workspace: 16 bytes, aligned to 4. */
int alsmi_score_rows(int dtype, int rank, int64_t n_sel, const int32_t *users, int64_t n_users,
                     const void *user_factors, const void *item_factors, int64_t n_items,
                     void *scores_out, void *workspace, void *stream);
int alsmi_score_items(int dtype, int rank, int64_t n_sel, const int32_t *users,
                      const void *user_factors, const void *item_factors, int64_t n_items,
                      void *scores_out, void *workspace, void *stream);

/* ---- ranking operators: a catalogue in 4 bits, scores changed before the selection, the
 * selection itself.  The reference stops at predict_all (src/als.py:347-364): no counterparts.
 * They take fp32, fp64, fp16 and bf16 elements (ALSMI_F32 .. ALSMI_BF16) unless said otherwise, any
 * row strides (in elements, >= the row's length) and any element alignment; no call allocates,
 * synchronises or records a memset, so all of them can be captured into a graph.  Calls that are
 * in flight together need output and workspace memory of their own. -----------------------------
 *
 * 4-bit microscaled tables: a row of `width` elements is cut into nb = ceil(width / 32) blocks of 32
 * (the last one padded by zeros); codes [n_rows x 16 nb] hold two four-bit codes per byte (the
 * element of even index in the low half), scales [n_rows x nb] one byte per block.  A code is a
 * sign bit and one of 0, 1/2, 1, 3/2, 2, 3, 4, 6; byte b scales by 2^(b - 127).
 * alsmi_mx4_quantize: b - 127 = floor(log2 max|x|) - 2, held to -127 .. 127 (-127 for a block of
 * zeros); the code nearest to |x| / 2^(b-127), ties to the even code, above 6 as 6.  A block with an
 * infinity or a NaN gets byte 255 and codes 0.  1 <= width <= 2^20, codes aligned to 4 bytes.
 * alsmi_mx4_dequantize: out row i = row rows[i] of the table (row i where rows is NULL); byte 255
 * reads as NaN, and so does a row id outside 0 .. n_rows-1.  Exact in fp64; in fp32 and bf16 up to byte
 * 252 (4 x 2^126 of byte 253, which only fp64 elements are quantised to, is past their range and
 * becomes an infinity); fp16 rounds and overflows to infinity. */
int alsmi_mx4_quantize(int dtype, int64_t n_rows, int64_t width, const void *x, int64_t ld_x,
                       uint8_t *codes, uint8_t *scales, void *stream);
int alsmi_mx4_dequantize(int dtype, int64_t n_sel, const int32_t *rows, int64_t n_rows,
                         int64_t width, const uint8_t *codes, const uint8_t *scales, void *out,
                         int64_t ld_out, void *stream);

/* out[i, j] = sum_k a[i, k] table[j, k] for i < n_sel, j < n_items; out [n_sel x n_items] of
 * out_dtype (ALSMI_F32, F16 or BF16).  `a` has n_rows rows of `width` elements of dtype ALSMI_F32,
 * F16 or BF16, or with ALSMI_MX4 is a table's codes and a_scales its scales (a_scales is ignored
 * otherwise).  Products are exact and sums fp32.  Two ranges are left out of that: bits below 2^-133 of
 * an ALSMI_F32 activation (which those of 2^-110 and more do not have) are cut off, and beside float
 * activations a table element past bf16's range (from byte 253 on, as above) counts as an infinity.  rows as in alsmi_mx4_dequantize: a row of NaN where
 * there is no such row.  workspace: alsmi_mx4_scores_workspace_bytes() bytes, aligned to 16 (large
 * products of float activations split them there first, 256 MiB at a time or 128 rows); may be
 * NULL where that is 0; what is enough for some rows, items and width is for fewer. */
size_t alsmi_mx4_scores_workspace_bytes(int dtype, int64_t n_sel, int64_t n_items, int64_t width);
int alsmi_mx4_scores(int dtype, int64_t n_sel, const int32_t *rows, int64_t n_rows, const void *a,
                     int64_t ld_a, const uint8_t *a_scales, int64_t n_items, int64_t width,
                     const uint8_t *codes, const uint8_t *scales, int out_dtype, void *out,
                     int64_t ld_out, void *workspace, void *stream);

/* Penalties, exclusion, biases and masks of score rows.  For row r and item i, with c = the
 * occurrences of i in the row's history:
 *   c > 0:  x = s > 0 ? s / repetition : s * repetition, then x -= frequency * c + presence
 *   c == 0: x = s
 *   x += item_bias[i];  x += the value of the last entry of i in the row's bias list
 *   x = -inf where the row's mask has no bit i (bit i % 32 of word i / 32 set: i is on offer), or
 *   where c > 0 if `exclude`
 * worked in fp32 (fp64 for ALSMI_F64), rounded once.  `out` may be `scores` itself.
 * Any pointer may be NULL: no history / bias list / item bias / mask.  repetition, frequency and
 * presence are [n_rows] fp32 arrays, or NULL for the *_value fields.  The history of row r is list
 * history_rows[r] of the n_history_rows lists (list r where history_rows is NULL; none where it is
 * outside), the mask of row r row mask_rows[r] (where mask_rows is NULL row r, or the only one; a
 * negative id: no mask; one past the masks: nothing is on offer).  List r is entries [ptr[r],
 * ptr[r+1]) of the ids; ids outside 0 .. n_items-1 are skipped, so lists may be padded.  Lists need
 * no order and may repeat an id.  repetition > 0. */
typedef struct alsmi_adjust {
    int64_t n_rows, n_items, ld_scores, ld_out;
    const int64_t *history_ptr;
    const int32_t *history_ids;
    int64_t n_history; /* entries of history_ids */
    const int32_t *history_rows;
    int64_t n_history_rows;
    const float *repetition, *frequency, *presence;
    double repetition_value, frequency_value, presence_value;
    const void *item_bias; /* [n_items] of item_bias_dtype */
    const int64_t *bias_ptr; /* [n_rows + 1] */
    const int32_t *bias_ids;
    const float *bias_values;
    int64_t n_bias; /* entries of bias_ids */
    const uint32_t *mask; /* [n_masks x ceil(n_items / 32)] */
    int64_t n_masks;
    const int32_t *mask_rows;
    int exclude;
    int item_bias_dtype; /* ALSMI_F32, or ALSMI_F64 for fp64 scores */
} alsmi_adjust;
int alsmi_adjust_scores(int dtype, const alsmi_adjust *args, const void *scores, void *out,
                        void *stream);

/* The k largest scores of every row, best first, ties by the smaller index: items_out [n_rows x k]
 * int32, scores_out [n_rows x k] of dtype.  1 <= k <= min(1024, n_items); the order of scores is that
 * of alsmi_topk_items.  workspace: alsmi_topk_rows_workspace_bytes() bytes, aligned to 16; what is
 * enough for some rows, items and k is for fewer. */
size_t alsmi_topk_rows_workspace_bytes(int dtype, int64_t n_rows, int64_t n_items, int k);
int alsmi_topk_rows(int dtype, int64_t n_rows, int64_t n_items, const void *scores,
                    int64_t ld_scores, int k, int32_t *items_out, void *scores_out, void *workspace,
                    void *stream);

/* Row index of every stored entry of rows [row_begin,row_end) (the `users`
 * array of data.nonzero(), src/als.py:161), written to rows_out[0 .. nnz_local). */
int alsmi_expand_rows(const int64_t *indptr, int64_t row_begin, int64_t row_end,
                      int32_t *rows_out, void *stream);

/* ---- sparse structure on the device: src/als.py:137-140 (triplets -> lil -> CSR)
 * and src/als.py:268-280 (scipy's csr_tocsc, which the reference re-runs per item) --
 *
 * alsmi_build_csr: n_in triplets (users, items int32; vals always fp64, the
 * reference's y) of an n_rows x n_cols matrix.  Same result as the reference's
 * element-by-element fill: a position written more than once keeps the LAST
 * value, a final value of exactly 0 is not stored, column indices inside a row
 * are sorted.  Outputs: indptr [n_rows+1], indices and vals_out (dtype) with
 * room for n_in entries, nnz_out[0] (device) = number stored.
 * alsmi_csr_to_csc: entries ordered by column, row ids ascending inside a
 * column (bit-identical to scipy's csr_tocsc); cptr [n_cols+1], cidx/cvals [nnz].
 * workspace: alsmi_sparse_workspace_bytes(number of input entries) bytes
 * (0 is returned when no HIP device is present to size it). */
size_t alsmi_sparse_workspace_bytes(int64_t n_entries);
int alsmi_build_csr(int dtype, int64_t n_rows, int64_t n_cols, int64_t n_in,
                    const int32_t *users, const int32_t *items, const double *vals,
                    int64_t *indptr, int32_t *indices, void *vals_out, int64_t *nnz_out,
                    void *workspace, void *stream);
int alsmi_csr_to_csc(int dtype, int64_t n_rows, int64_t n_cols, int64_t nnz,
                     const int64_t *indptr, const int32_t *indices, const void *vals,
                     int64_t *cptr, int32_t *cidx, void *cvals, void *workspace, void *stream);

/* ---- IMC objective pieces: src/imc.py:43-48 (_cost), :65-71 (_cost_prime),
 * :91-96 (_cost_hess), :157 (initial Z) ------------------------------------
 *
 * The reference works on one dense feature row per SAMPLE.  Here the samples
 * are index pairs grouped by user: `indptr` [n_users+1] and `items` [n_s] are
 * the CSR structure of the ratings, `ratings` [n_s] their values in that order;
 * X [n_users x p] and M [p x q] are plain row-major; Y is [n_items x ldy] with
 * ldy = alsmi_imc_padded_width(q) and zero pad columns.  With A = X M and
 * d_e = <A[u_e], Y[i_e]>:
 *   mode 0: out = X^T diag-weighted-sum (d_e - r_e) Y[i_e]   (the data part of the
 *           gradient), sse_out[0] = sum_e (r_e - d_e)^2       (the data part of the cost)
 *   mode 1: out = X^T sum d_e Y[i_e]                          (the data part of H*M)
 * `out` [p x q] row-major, `pred_out` [n_s] (the d_e, in the order of `items`) and
 * `sse_out` may each be NULL when not wanted.  The caller
 * adds the reference's regulariser terms, which are O(p q): 0.5*n_s*lam*||Z||^2 to
 * the cost (the reference counts it once per sample), lam*Z to the gradient and
 * the scalar lam to every entry of the Hessian-vector product.
 * Calling mode 0 with M = 0 and negated ratings gives X^T diag(r) Y of
 * src/imc.py:157.  1 <= q <= 256.  n_samples = indptr[n_users] (the host needs it to size
 * the launch: the pass cuts the ENTRIES, not the users, into equal chunks, so its time does not
 * depend on how unevenly the entries are spread over the users; every sum has a fixed order).
 * The workspace layout depends on all of n_users, n_samples, p and q (chunk length and the
 * number of partial results follow from them): size it with exactly the values of the call. */
int alsmi_imc_padded_width(int q);
size_t alsmi_imc_workspace_bytes(int dtype, int64_t n_users, int64_t n_samples, int p, int q);
int alsmi_imc_eval(int dtype, int mode, int64_t n_users, int64_t n_samples, int p, int q,
                   const int64_t *indptr, const int32_t *items, const void *ratings, const void *X,
                   const void *Y, const void *M, void *out, void *pred_out, double *sse_out,
                   void *workspace, void *stream);

/* table_out [n_rows x alsmi_imc_padded_width(q)] = X [n_rows x p] M [p x q], pad columns zero:
 * the projected attribute table of the rank-constrained IMC form (Z = U V^T: the rows of Y V
 * take the place of the item attributes and U that of Z, so the pass over the samples is
 * n_components wide instead of q wide).  No reference counterpart: the reference validates
 * n_components and then ignores it (src/imc.py:148-154). */
int alsmi_imc_project(int dtype, int64_t n_rows, int p, int q, const void *X, const void *M,
                      void *table_out, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ALSMI_H */

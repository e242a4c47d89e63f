/*
 * C ABI of the expert layers and 4-bit products of libh2o4gpu_kmeans_hip.so.
 *
 * What a language model does with clusters of its tokens: every token goes to the models
 * ("experts") of its best centroids, their results come back and are joined by weight; and the
 * 16 values that k-means finds in a weight matrix serve as that matrix's 4-bit codebook. The
 * reference has no counterpart of any of these functions.
 *
 * Every pointer named d_* is device memory of the CURRENT device. Work is queued on `stream` (a
 * hipStream_t, NULL = the default stream) and the call returns without waiting; no function
 * allocates, copies to the host or keeps data or a workspace between calls, so all of them can be
 * recorded into a graph. What stays is a kernel's limit of shared memory on a device: a call that
 * needs more than 64 KB and more than any before it raises it, and is to be outside a capture, so
 * make one of the same type and sizes before recording. That may be route (distances), sort, both
 * products with codebooks, the experts' own products, their gradients and the microscaled products. Strides count elements. A call that returns an error has queued nothing, but for
 * H2O4GPU_KMEANS_EDEVICE. Sizes of 0 rows are a success that queues nothing (but for the offsets
 * of experts_sort). Same inputs give the same bits in every call.
 * Status codes are those of h2o4gpu_kmeans.h.
 */
#ifndef H2O4GPU_EXPERTS_H
#define H2O4GPU_EXPERTS_H

#include <stddef.h>

#include "h2o4gpu_kmeans.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of `dtype` and `scale_dtype` */
#define H2O4GPU_EXPERTS_FLOAT32 0
#define H2O4GPU_EXPERTS_BFLOAT16 1
#define H2O4GPU_EXPERTS_FLOAT16 2

#define H2O4GPU_EXPERTS_MAX_EXPERTS 16384
#define H2O4GPU_EXPERTS_MAX_TOP_K 64
#define H2O4GPU_CODEBOOK4_MAX_GROUP (1 << 30)
#define H2O4GPU_EXPERTS_MAX_SIDE (1 << 20)

/* The top_k best experts of every row and their weights.
 * d_scores: rows x experts of `dtype`; element (t, e) lies at t * row_stride + e * expert_stride,
 * so both a model's scores [rows][experts] and the distances [experts][rows] of
 * h2o4gpu_kmeans_transform_resident are taken as they are. largest != 0: the largest score is the
 * best (scores), 0: the smallest (distances). Equal scores go to the lowest index. A NaN and the
 * worst infinity (-inf, +inf for largest == 0) mark an expert that is not available.
 * d_experts [rows][top_k]: best first; -1 where no expert is left.
 * d_weights [rows][top_k] (float): softmax of scale * score (scale * -score for largest == 0;
 * scale >= 0, finite) over the chosen experts, or over all available ones where over_all != 0; 0
 * beside a -1. Scores of the best infinity share the whole weight equally. */
int h2o4gpu_experts_route(int dtype, size_t rows, int experts, int top_k, int largest, int over_all, float scale,
                          const void *d_scores, ptrdiff_t row_stride, ptrdiff_t expert_stride, int *d_experts,
                          float *d_weights, void *stream);

/* d_dscores (same type and shape as the scores, strides of its own, every element written):
 * gradient of sum(d_dweights * weights) with respect to the scores, the choice held fixed.
 * d_scores, d_experts and d_weights are those of the forward call; d_dweights [rows][top_k] float. */
int h2o4gpu_experts_route_backward(int dtype, size_t rows, int experts, int top_k, int largest, int over_all,
                                   float scale, const void *d_scores, ptrdiff_t row_stride,
                                   ptrdiff_t expert_stride, const int *d_experts, const float *d_weights,
                                   const float *d_dweights, void *d_dscores, ptrdiff_t drow_stride,
                                   ptrdiff_t dexpert_stride, void *stream);

/* Slots ordered by expert: a slot is one entry of d_experts (token t's j-th choice is slot
 * t * top_k + j). d_order [slots]: the slots of expert 0 in ascending order, then those of expert
 * 1, ..., then those whose value is none of 0 .. experts-1. d_offsets [experts + 1]: where each
 * expert's rows begin, and last how many slots have an expert. d_position [slots]: a slot's place
 * in d_order, as ~place (a negative number) where it has no expert.
 * d_workspace: h2o4gpu_experts_sort_workspace() bytes, 4-byte aligned (NULL where that is 0). */
size_t h2o4gpu_experts_sort_workspace(size_t slots, int experts);
int h2o4gpu_experts_sort(size_t slots, int experts, const int *d_experts, int *d_order, int *d_position,
                         int *d_offsets, void *d_workspace, size_t workspace_bytes, void *stream);

/* Rows in expert order. dispatch: d_rows[position(t, j)] = d_x[t] for every slot with an expert,
 * zeros for the others' places. dispatch_backward: d_dx[t] = sum over j of d_drows[position(t, j)]
 * over the slots with an expert, summed in float, j ascending.
 * x: [tokens][cols], rows: [tokens * top_k][cols], rows x_stride and rows_stride elements apart. */
int h2o4gpu_experts_dispatch(int dtype, size_t tokens, int top_k, size_t cols, const void *d_x, size_t x_stride,
                             const int *d_position, void *d_rows, size_t rows_stride, void *stream);
int h2o4gpu_experts_dispatch_backward(int dtype, size_t tokens, int top_k, size_t cols, const void *d_drows,
                                      size_t rows_stride, const int *d_position, void *d_dx, size_t x_stride,
                                      void *stream);

/* The experts' results joined: d_out[t] = sum over j of d_weights[t][j] * d_rows[position(t, j)]
 * over the slots with an expert (what lies in other places is not read), in float, j ascending.
 * combine_backward: d_drows[position(t, j)] = d_weights[t][j] * d_dout[t] (zeros in the places of
 * slots without an expert), d_dweights[t][j] = <d_dout[t], d_rows[position(t, j)]> (0 likewise). */
int h2o4gpu_experts_combine(int dtype, size_t tokens, int top_k, size_t cols, const void *d_rows,
                            size_t rows_stride, const float *d_weights, const int *d_position, void *d_out,
                            size_t out_stride, void *stream);
int h2o4gpu_experts_combine_backward(int dtype, size_t tokens, int top_k, size_t cols, const void *d_dout,
                                     size_t dout_stride, const void *d_rows, size_t rows_stride,
                                     const float *d_weights, const int *d_position, void *d_drows,
                                     size_t drows_stride, float *d_dweights, void *stream);

/* A 4-bit matrix [out][cols]: codes are 4 bits each, the even column in a byte's low half, rows
 * codes_pitch bytes apart (at least cols / 2, rounded up); scales [out][ceil(cols / group)] of
 * `scale_dtype`, group a multiple of 32 (up to MAX_GROUP); codebook: 16 finite values of `dtype`. Element (n, k) is
 * codebook[code(n, k)] * scales[n][k / group].
 *
 * quantize: codes and scales of a matrix d_w of `dtype`. A group's scale is its largest magnitude
 * over `top` (> 0: the codebook's value that this magnitude stands for), rounded to scale_dtype (1
 * where that gives 0 or no finite number); an element's code is the entry nearest to element / scale,
 * ties to the lowest (0 for a NaN and an infinity). A row's bytes behind column cols are written as 0. */
int h2o4gpu_codebook4_quantize(int dtype, size_t out, size_t cols, int group, float top, const void *d_w,
                               size_t w_stride, const void *d_codebook, void *d_codes, size_t codes_pitch,
                               int scale_dtype, void *d_scales, void *stream);
/* The order in which the products read a matrix, or `experts` matrices one behind another (codes
 * [experts][out][codes_pitch], scales [experts][out][groups]): made once from codes and scales, which are not
 * needed any more. d_laid_codes: codes_bytes() bytes, d_laid_scales: scales_bytes() bytes, both 16-byte
 * aligned. A tile of 16 rows and 128 columns is 1024 bytes of codes: 64 times 16 bytes, number 16 q + r
 * of which holds in its word i the columns 32 i + 8 q .. + 7 of row r; tiles of a row of tiles follow
 * each other. Its scales are 16, one a row, or, where group is no multiple of 128, 16 x 2 (a multiple of
 * 64) or 16 x 4. Behind the matrix's last row and column lie zeros. The byte counts are 0 for bad arguments. */
size_t h2o4gpu_codebook4_codes_bytes(size_t experts, size_t out, size_t cols);
size_t h2o4gpu_codebook4_scales_bytes(size_t experts, size_t out, size_t cols, int group, int scale_dtype);
int h2o4gpu_codebook4_layout(size_t experts, size_t out, size_t cols, int group, const void *d_codes,
                             size_t codes_pitch, int scale_dtype, const void *d_scales, void *d_laid_codes,
                             void *d_laid_scales, void *stream);
/* d_y [rows][out] = d_x [rows][cols] times the matrix's transpose; products and sums in float, one
 * rounding at the end. */
int h2o4gpu_codebook4_product(int dtype, size_t rows, size_t out, size_t cols, int group, const void *d_x,
                              size_t x_stride, const void *d_laid_codes, int scale_dtype, const void *d_laid_scales,
                              const void *d_codebook, void *d_y, size_t y_stride, void *stream);
/* The same with a matrix per expert, rows in expert order (experts_sort on [tokens][top_k] choices):
 * d_y[p] = d_x[d_order[p] / top_k] times the transpose of the matrix whose rows p is among; zeros
 * for the rows behind d_offsets[experts]. Codebook of expert e at d_codebook + e * codebook_stride (0:
 * one for all). */
int h2o4gpu_codebook4_experts_product(int dtype, size_t tokens, int top_k, int experts, size_t out, size_t cols,
                                      int group, const void *d_x, size_t x_stride, const void *d_laid_codes,
                                      int scale_dtype, const void *d_laid_scales, const void *d_codebook,
                                      size_t codebook_stride, const int *d_order, const int *d_offsets, void *d_y,
                                      size_t y_stride, void *stream);

/* The experts' own products, rows in expert order: d_y[p] = W_e d_rows[p] for the rows p in
 * [d_offsets[e], d_offsets[e + 1]) of each expert e, zeros for those behind d_offsets[experts] (what
 * lies there is not read). d_offsets [experts + 1] as experts_sort writes it: from 0, ascending, at
 * most rows. W_e: [out][cols], rows w_stride (at most 2^23) elements apart, at d_weights + e * expert_stride (0: one
 * matrix for all). Sums in float, one rounding at the end.
 * product_drows: d_drows[p] = W_e^T d_dy[p], zeros likewise. product_dweights: d_dweights
 * [experts][out][cols], W_e's is the sum over its rows of d_dy[p] d_rows[p]^T (zeros for none), out, cols
 * and both strides at most MAX_SIDE;
 * d_workspace: product_dweights_workspace() bytes, 16-byte aligned (NULL where that is 0): sums of parts of the
 * rows, where few matrices of few tiles of 128 x 128 have many rows. Which kernel adds up depends on sizes, strides
 * and addresses, and with it the last bit of a result. */
int h2o4gpu_experts_product(int dtype, size_t rows, int experts, size_t out, size_t cols, const void *d_rows,
                            size_t rows_stride, const void *d_weights, size_t expert_stride, size_t w_stride,
                            const int *d_offsets, void *d_y, size_t y_stride, void *stream);
int h2o4gpu_experts_product_drows(int dtype, size_t rows, int experts, size_t out, size_t cols, const void *d_dy,
                                  size_t dy_stride, const void *d_weights, size_t expert_stride, size_t w_stride,
                                  const int *d_offsets, void *d_drows, size_t drows_stride, void *stream);
size_t h2o4gpu_experts_product_dweights_workspace(int dtype, size_t rows, int experts, size_t out, size_t cols);
int h2o4gpu_experts_product_dweights(int dtype, size_t rows, int experts, size_t out, size_t cols, const void *d_dy,
                                     size_t dy_stride, const void *d_rows, size_t rows_stride, const int *d_offsets,
                                     void *d_dweights, void *d_workspace, size_t workspace_bytes, void *stream);

/* Rows of `matrices` matrices [rows][cols], the matrices matrix_stride elements apart, to rows that begin at
 * multiples of 16 bytes, as short as they can be, one matrix behind another; zeros behind column cols. The
 * products above are faster where strides and addresses of both operands are multiples of 4 bytes, most so
 * those of 16-bit elements and many rows: 1.5 us and more for 10^9 operations, beside 1 us for 1.8 MB copied. */
int h2o4gpu_experts_align_rows(int dtype, size_t matrices, size_t rows, size_t cols, const void *d_in,
                               size_t matrix_stride, size_t stride, void *d_out, void *stream);

/* Microscaled 4-bit matrices: every 32 columns of a row share a power of two, 2^(byte - 127), and an
 * element is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (codes 0 .. 7, the sign is 8) times it. A
 * scale byte of 255 is not a number, and neither is its block.
 * In memory: rows of codes_pitch(cols) bytes, two codes a byte, the even column in the low half; rows of
 * scales_pitch(cols) bytes of scales, block b of every 16 at byte 4 * (b % 4) + b / 4. Both start at a
 * multiple of 16 bytes; behind a row's last column lie zeros. Pitches are 0 for bad arguments.
 *
 * quantize: the scale of a block is 2^(floor(log2(largest magnitude)) - 2), at least 2^-127; elements
 * are rounded to the nearest, a tie to the even code, those beyond 6 are 6. A block with a NaN or an
 * infinity is not a number; a block of zeros has scale byte 0. dequantize: the reverse, rounded to dtype.
 * layout: from codes in rows codes_stride bytes apart and scales [rows][ceil(cols / 32)]. */
size_t h2o4gpu_microscale4_codes_pitch(size_t cols);
size_t h2o4gpu_microscale4_scales_pitch(size_t cols);
int h2o4gpu_microscale4_quantize(int dtype, size_t rows, size_t cols, const void *d_x, size_t x_stride, void *d_codes,
                                 void *d_scales, void *stream);
int h2o4gpu_microscale4_dequantize(int dtype, size_t rows, size_t cols, const void *d_codes, const void *d_scales,
                                   void *d_out, size_t out_stride, void *stream);
int h2o4gpu_microscale4_layout(size_t rows, size_t cols, const void *d_codes, size_t codes_stride,
                               const void *d_scales, void *d_laid_codes, void *d_laid_scales, void *stream);
/* d_y [rows][out] of dtype = x [rows][cols] times the transpose of w [out][cols], both microscaled;
 * sums in float, one rounding at the end. experts_product: w [experts][out][cols], rows in expert
 * order: row p of d_y is x's row d_order[p] / top_k (d_order NULL: x's row p, x then has
 * tokens * top_k rows) times the matrix of the expert whose rows p is among; zeros for the rows
 * behind d_offsets[experts]. */
int h2o4gpu_microscale4_product(int dtype, size_t rows, size_t out, size_t cols, const void *d_x, const void *d_x_scales,
                                const void *d_w, const void *d_w_scales, void *d_y, size_t y_stride, void *stream);
int h2o4gpu_microscale4_experts_product(int dtype, size_t tokens, int top_k, int experts, size_t out, size_t cols,
                                        const void *d_x, const void *d_x_scales, const void *d_w,
                                        const void *d_w_scales, const int *d_order, const int *d_offsets, void *d_y,
                                        size_t y_stride, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* H2O4GPU_EXPERTS_H */

/*
 * b200sp_rows.h -- rows of tokens in the order of the experts that they are routed to, and back; products in 8-bit integers
 * with a scale for each row and each channel.
 *
 * They stand beside b200sp_tokens.h and share its objects and its common rules: handle, stream, pointer mode, row-major
 * operands of any ld and alignment, alpha and beta (NULL: 1 and 0; beta = 0 never reads the output), sums in a fixed order,
 * values that f16 cannot hold become infinite, calls that enqueue, wait for nothing and allocate nothing, and may be captured.
 * An output overlaps no input.
 *
 * A layer of experts in 8 bits, R as b200spRoute left it:
 *   b200spExpertsPreprocess(R), b200spExpertsQuantise(X -> Q in the order of the experts), b200spExpertsScaledMM(Q -> Y),
 *   (the layer's activation on Y), b200spQuantiseRows(Y -> P), b200spExpertsScaledMM(P -> Z), b200spExpertsCombine(Z -> out).
 * Trained in 16 or 32 bits: b200spExpertsDispatch, the caller's products of every expert's rows, b200spExpertsCombine; back
 * b200spExpertsCombineGrad, the products' gradients, and b200spExpertsCombine without weights, which is Dispatch's gradient.
 */
#ifndef B200SP_ROWS_H_
#define B200SP_ROWS_H_

#include <stddef.h>
#include <stdint.h>

#include "b200sp_tokens.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Rows in the order of the experts ----
 * R: any CSR matrix of tokens x experts (1024 at most).  b200spExpertsPreprocess orders its entries: all of the first expert, in
 * R's order, then the second's, ..., at last those whose column is no expert.  place(i) is where entry i comes in it.  `buffer` is one
 * that b200spExpertsPreprocess has written for this R, under the rules that the experts' products have for it; as large as this says: */
aclsparseStatus_t b200spExpertsOrderBufferSize(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matR, size_t *bufferSize);

/* S[place(i)] = alpha * X[token of entry i] + beta * S[place(i)]: S has a row for every entry, X for every token; those of no expert
 * become beta * S.  X: f32, f16 or bf16; S: the same, or f32.  offsets: NULL, or a dense vector of ACL_INT32 that takes, for
 * each expert, the first of its rows of S, and at last the end of the last one's: experts + 1 numbers. */
aclsparseStatus_t b200spExpertsDispatch(aclsparseHandle_t handle, const void *alpha, aclsparseConstSpMatDescr_t matR,
                                        aclsparseConstDnMatDescr_t matX, const void *beta, aclsparseDnMatDescr_t matS,
                                        aclsparseDnVecDescr_t offsets, const void *buffer);

typedef enum b200spExpertWeights_t {
    B200SP_WEIGHTS_NONE = 0, /* rows are summed as they are */
    B200SP_WEIGHTS_OF_R      /* times R's values: f32, f16 or bf16 */
} b200spExpertWeights_t;

/* out[t] = alpha * (sum of w_i * S[place(i)] over the entries i of token t, in R's order) + beta * out[t].  Entries of no expert
 * take no part; one of weight 0 does.  S and out: f32, f16 or bf16, two unlike types of 16 bits excepted. */
aclsparseStatus_t b200spExpertsCombine(aclsparseHandle_t handle, b200spExpertWeights_t weights, const void *alpha,
                                       aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matS, const void *beta,
                                       aclsparseDnMatDescr_t matOut, const void *buffer);

/* The gradient of the weighted sum: dS[place(i)] = alpha * w_i * dOut[t] + beta * dS[place(i)], and
 * dValues[i] = alpha * <dOut[t], S[place(i)]> + beta * dValues[i]; for entries of no expert the first terms are 0.  dOut, S: as out and S
 * above; dS of S's type, dValues f32, f16 or bf16.  S and dValues may both be NULL: no gradient of the weights.  dS may be S. */
aclsparseStatus_t b200spExpertsCombineGrad(aclsparseHandle_t handle, const void *alpha, aclsparseConstSpMatDescr_t matR,
                                           aclsparseConstDnMatDescr_t dOut, aclsparseConstDnMatDescr_t matS, const void *beta,
                                           aclsparseDnMatDescr_t dS, aclsparseDnVecDescr_t dValues, const void *buffer);

/* ---- Rows in 8 bits ----
 * Q[r][c] = 127 * X[r][c] / m rounded to the nearest whole number, m the row's largest absolute value; scales[r] = m / 127 in f32.  The
 * number that is rounded is the quotient itself, not one of rounded arithmetic, and a half goes to the even number: Q is unique.  A row
 * of zeros has scale 0.  One with an infinity or a NaN has scale NaN and zeros: a product shows it.  X: f32, f16 or bf16; Q: ACL_INT8;
 * scales: ACL_FLOAT, one for every row of Q.  A matrix of weights has a row for each of its channels. */
aclsparseStatus_t b200spQuantiseRows(aclsparseHandle_t handle, aclsparseConstDnMatDescr_t matX, aclsparseDnMatDescr_t matQ,
                                     aclsparseDnVecDescr_t scales);

/* The same of every token's row, into the rows of its entries in the order of the experts; those of no expert become zeros of scale 0.
 * offsets, buffer: as b200spExpertsDispatch takes them. */
aclsparseStatus_t b200spExpertsQuantise(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matX,
                                        aclsparseDnMatDescr_t matQ, aclsparseDnVecDescr_t scales, aclsparseDnVecDescr_t offsets,
                                        const void *buffer);

/* ---- Products in 8 bits ----
 * Y[i][j] = alpha * scalesX[i] * scalesW[j] * (sum of X[i][c] * W[j][c]) + beta * Y[i][j].  X, W: ACL_INT8, of the same columns, 131,071 at
 * most: the sums are exact.  scalesX, scalesW: ACL_FLOAT, one for every row.  Y: f32, f16 or bf16.  Fastest where the rows of X and W
 * start on 16 bytes; others are copied into the buffer in every call, weights, too (one row of 4096 by 4096 13 us, where 6.6).  buffer: of the size
 * that this says (0: it may be NULL) for one call at a time. */
aclsparseStatus_t b200spScaledMMBufferSize(aclsparseHandle_t handle, aclsparseConstDnMatDescr_t matX,
                                           aclsparseConstDnMatDescr_t matW, aclsparseConstDnMatDescr_t matY, size_t *bufferSize);
aclsparseStatus_t b200spScaledMM(aclsparseHandle_t handle, const void *alpha, aclsparseConstDnMatDescr_t matX,
                                 aclsparseConstDnVecDescr_t scalesX, aclsparseConstDnMatDescr_t matW,
                                 aclsparseConstDnVecDescr_t scalesW, const void *beta, aclsparseDnMatDescr_t matY, void *buffer);

/* The same with every expert's rows of X, in the order of the experts, and its own matrix.  W: the experts' matrices one below
 * the other, experts x (n rows); X and Y have a row for every entry of R.  Rows of no expert become beta * Y.  buffer: what
 * b200spExpertsPreprocess wrote for R, with as many bytes as this says; room for copies of operands is counted and asked for as
 * b200spExpertsMM has it. */
aclsparseStatus_t b200spExpertsScaledMMBufferSize(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matR,
                                                  aclsparseConstDnMatDescr_t matX, aclsparseConstDnMatDescr_t matW,
                                                  aclsparseConstDnMatDescr_t matY, size_t *bufferSize);
aclsparseStatus_t b200spExpertsScaledMM(aclsparseHandle_t handle, const void *alpha, aclsparseConstSpMatDescr_t matR,
                                        aclsparseConstDnMatDescr_t matX, aclsparseConstDnVecDescr_t scalesX,
                                        aclsparseConstDnMatDescr_t matW, aclsparseConstDnVecDescr_t scalesW, const void *beta,
                                        aclsparseDnMatDescr_t matY, void *buffer);

/* What went wrong in a product in 8 bits since the flag was cleared, as b200sp_experts_error says it of the others: 1: a bounded wait ran out,
 * rows of the output are unwritten; 2: its buffer held no order.  (The other calls of this header that follow an order raise 2 in
 * b200sp_experts_error.)  Both are for the current device and synchronise it. */
int b200sp_scaled_error(void);
int b200sp_scaled_error_clear(void);
/* For tests of that path, as b200sp_experts_wait_test. */
void b200sp_scaled_wait_test(long long wait_cycles, unsigned extra_tx);

#ifdef __cplusplus
}
#endif

#endif /* B200SP_ROWS_H_ */

/*
 * b200sp_tokens.h -- operators of token models: products whose sparse matrix the model makes itself, one entry a row
 * (a token's row of a table) or a few entries a row (a token's experts).
 *
 * They stand beside SpMM, SDDMM and the converters and share their objects: the handle with its stream and pointer
 * mode, dense descriptors (row-major here), and a CSR matrix R (tokens x experts) that b200spRoute fills.  R is an
 * ordinary matrix: aclsparseSpMM with R's values sums the experts' rows of every token, aclsparseSDDMM gives the
 * gradient of the values, aclsparseCsr2cscEx2 the tokens of every expert.
 *
 * Common rules.  alpha / beta are float, on the host or, with ACL_SPARSE_POINTER_MODE_DEVICE, on the device; NULL means
 * 1 and 0.  beta = 0 never reads the output.  Dense operands are row-major with any ld and alignment (fastest where rows
 * start on 16-byte boundaries); f32, f16 and bf16 unless said otherwise.  Sums are in f32 in a fixed order and
 * rounded once: the same inputs give the same bits.  Values that f16 cannot hold become infinite (SpMM clamps them; a
 * gradient has to show that it overflowed).  Calls enqueue on the handle's stream, wait for nothing, allocate nothing,
 * and may be captured.  A handle is used on the device that it was created on, whatever device is current.
 * (A call on no tokens can not be described: aclsparseCreateDnMat refuses a matrix of no rows.)
 * An output overlaps no input, unless it says so.  At most 2^31 - 2^20 tokens, columns or entries of R, and tables of 2^31 - 2 rows.
 * Column-major operands, index bases of one and 64-bit CSR indices are ACL_SPARSE_STATUS_NOT_SUPPORTED.
 */
#ifndef B200SP_TOKENS_H_
#define B200SP_TOKENS_H_

#include <stddef.h>
#include <stdint.h>

#include "cann_ops_sparse.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Embedding: out[i] = alpha * table[tokens[i]] + beta * out[i] ----
 * tokens: a dense vector of ACL_INT32 or ACL_INT64.  A token outside [0, rows of table) stands for no row (padding): its row
 * of the table is taken as zeros. */
aclsparseStatus_t b200spEmbedding(aclsparseHandle_t handle, const void *alpha, aclsparseConstDnMatDescr_t table,
                                  aclsparseConstDnVecDescr_t tokens, const void *beta, aclsparseDnMatDescr_t out);

/* Gradient of the table: dTable[v] = alpha * (sum of grad[i] over the i with tokens[i] = v) + beta * dTable[v], all rows
 * of dTable.  Tokens outside the table are left out.  The tokens are sorted in the call; grad's rows of one token are
 * summed in the order of their positions, in pieces.  dTable must not overlap grad.  beta = 1 reads and writes the rows of
 * the tokens only.  A buffer serves one call at a time; what it holds need not be kept. */
aclsparseStatus_t b200spEmbeddingGradBufferSize(aclsparseHandle_t handle, aclsparseConstDnMatDescr_t grad,
                                                aclsparseConstDnVecDescr_t tokens, aclsparseConstDnMatDescr_t dTable,
                                                size_t *bufferSize);
aclsparseStatus_t b200spEmbeddingGrad(aclsparseHandle_t handle, const void *alpha, aclsparseConstDnMatDescr_t grad,
                                      aclsparseConstDnVecDescr_t tokens, const void *beta, aclsparseDnMatDescr_t dTable,
                                      void *buffer);

/* ---- Routing: a CSR matrix with the k best experts of every token ---- */
typedef enum b200spRouteScore_t {
    B200SP_ROUTE_SOFTMAX = 0, /* over all experts of the token */
    B200SP_ROUTE_SIGMOID
} b200spRouteScore_t;
typedef enum b200spGroupScore_t {
    B200SP_GROUP_MAX = 0, /* the best selection value of the group */
    B200SP_GROUP_TOP2     /* the sum of its two best (of p + bias) */
} b200spGroupScore_t;

typedef struct b200spRouteRule {
    int32_t score;       /* b200spRouteScore_t */
    int32_t groups;      /* of neighbouring experts, all equally large; 1: none */
    int32_t groupsKept;  /* experts of other groups are not chosen */
    int32_t groupScore;  /* b200spGroupScore_t */
    int32_t renormalise; /* 1: the weights of a token are divided by their sum */
    float scale;         /* the weights are multiplied by it */
} b200spRouteRule;

/* Writes R's row offsets (k * row), its columns (ascending in every row) and its values.  k is R's entries over its rows; R's
 * value type is that of the weights.  logits: tokens x experts, f32, f16 or bf16; bias: f32 per expert, or NULL.
 *
 * An expert's selection value is p + bias with a bias, where p is its score, and without one the logit itself: both
 * scores ascend with it.  The groupsKept groups of the highest group score are kept, then the k experts of the
 * highest selection value taken; what is equal goes to the lower index.  The order is that of f64 arithmetic: values
 * that f32 might not tell apart are compared in f64.  An expert with a logit or bias of -infinity or NaN is masked: no score,
 * and taken only where fewer than k others are left in the kept groups, the lowest index first; experts of groups that are
 * not kept are treated alike.  Such entries have weight 0.  The other weights are p, over their sum if renormalise,
 * times scale; the bias is in none of them.
 * (A masked bias leaves the softmax of the others as it is.)  At most 1024 experts, 32 entries a row and 32 groups. */
aclsparseStatus_t b200spRoute(aclsparseHandle_t handle, const b200spRouteRule *rule, aclsparseConstDnMatDescr_t logits,
                              aclsparseConstDnVecDescr_t bias, aclsparseSpMatDescr_t matR);

/* Gradient of the logits (whole, zeros included) from that of R's values (dValues: f32, f16 or bf16, one per entry).  R has k
 * entries in every row, as b200spRoute left it; entries whose value is 0 are taken as masked.  The choice of the experts has no
 * gradient.  dLogits may be logits. */
aclsparseStatus_t b200spRouteGrad(aclsparseHandle_t handle, const b200spRouteRule *rule, aclsparseConstDnMatDescr_t logits,
                                  aclsparseConstSpMatDescr_t matR, aclsparseConstDnVecDescr_t dValues,
                                  aclsparseDnMatDescr_t dLogits);

/* ---- Experts' products over R ----
 * R: any CSR matrix of tokens x experts (1024 at most); its values are not read.  An entry i of R lies in the row token(i) and the
 * column expert(i).  Entries whose column is no expert take part in nothing (their rows of Y are beta * Y).
 * W: the experts' matrices one below the other, experts x (n rows of d columns); X, Y, W, dY, dW all f16 or all bf16, and Y
 * and dW also f32. */
typedef enum b200spExpertRows_t {
    B200SP_ROWS_OF_TOKENS = 0, /* X has a row for every token */
    B200SP_ROWS_OF_ENTRIES     /* X has a row for every entry of R */
} b200spExpertRows_t;

/* Orders the entries of R by expert in `buffer`; wanted again when R's offsets or columns change, or when the buffer has been
 * written.  After a b200spRoute into R products are refused (ACL_SPARSE_STATUS_INVALID_VALUE) until it has been called again.
 * Nothing is waited for: it may be captured with the products that follow. */
aclsparseStatus_t b200spExpertsPreprocess(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matR, void *buffer);

/* Operands of the products whose rows do not start on 16 bytes are copied into the buffer first, in every call: the BufferSize calls count
 * the room for the operands they are given.  A product that copies is refused (ACL_SPARSE_STATUS_INVALID_VALUE) unless so much has been
 * asked for through R's own descriptor; that a buffer has the size that was asked for is the caller's to see to, for every buffer.
 *
 * Y[i] = alpha * X[row of entry i] * op(W of its expert) + beta * Y[i], a row of Y for every entry of R.
 * opW = T: X has d columns, Y n (a layer whose weights lie as n x d); opW = N: X has n columns, Y d (the
 * gradient of that layer's input rows).  `buffer`: what b200spExpertsPreprocess wrote, with as many bytes as
 * the BufferSize call says; one buffer serves several products with the same R, one at a time, with the largest size. */
aclsparseStatus_t b200spExpertsMMBufferSize(aclsparseHandle_t handle, aclsparseOperation_t opW, b200spExpertRows_t rowsOfX,
                                            aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matX,
                                            aclsparseConstDnMatDescr_t matW, aclsparseConstDnMatDescr_t matY,
                                            size_t *bufferSize);
aclsparseStatus_t b200spExpertsMM(aclsparseHandle_t handle, aclsparseOperation_t opW, b200spExpertRows_t rowsOfX,
                                  const void *alpha, aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matX,
                                  aclsparseConstDnMatDescr_t matW, const void *beta, aclsparseDnMatDescr_t matY, void *buffer);

/* dW_e = alpha * (sum over the entries i of expert e of dY[i]^T X[row of entry i]) + beta * dW_e, for every expert (one
 * without entries gets beta * dW_e).  dY: a row of n columns for every entry; X: d columns. */
aclsparseStatus_t b200spExpertsGradBufferSize(aclsparseHandle_t handle, b200spExpertRows_t rowsOfX,
                                              aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t dY,
                                              aclsparseConstDnMatDescr_t matX, aclsparseConstDnMatDescr_t dW,
                                              size_t *bufferSize);
aclsparseStatus_t b200spExpertsGrad(aclsparseHandle_t handle, b200spExpertRows_t rowsOfX, const void *alpha,
                                    aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t dY,
                                    aclsparseConstDnMatDescr_t matX, const void *beta, aclsparseDnMatDescr_t dW,
                                    void *buffer);

/* What went wrong in an experts' product since the flag was cleared.  1: a bounded wait ran out (never observed outside the test that
 * provokes it), rows of the output are unwritten; 2: its buffer held no order, or one of earlier columns, because the b200spExpertsPreprocess
 * that belongs to it was captured and not replayed yet, and the output is untouched.  Both calls are for the current device, which has to be
 * that of the product's handle, and synchronise it (not during a capture); b200sp_experts_error is -1 if that fails. */
int b200sp_experts_error(void);
int b200sp_experts_error_clear(void);
/* For tests of that path: later products wait at most wait_cycles SM clocks (0 = the default, about two seconds; for a tile's results 4096 more
 * for each of its steps of 64 terms) and expect extra_tx bytes more than they copy on every barrier, so that with extra_tx > 0 every wait runs out. */
void b200sp_experts_wait_test(long long wait_cycles, unsigned extra_tx);

#ifdef __cplusplus
}
#endif

#endif /* B200SP_TOKENS_H_ */

/*
 * theseus_vocab.h -- C ABI of the vocabulary operators in libtheseus_wkv7.so (gfx950):
 * what a model's head is trained on and answers with, for M tokens of width D and a
 * vocabulary of V.
 *
 *   theseus_vocab_loss   softmax cross entropy, or the divergence from a teacher's top
 *                        logits, of z = hidden weight^T without keeping z, with the
 *                        gradients of hidden and weight
 *   theseus_vocab_top    the k largest logits of each row, their indices, and the row's
 *                        log-sum-exp
 *
 * With sparse targets q_ik at indices j_ik, Q_i = sum_k q_ik, T the temperature,
 * z_iv = hidden_i . weight_v / T and p_iv = exp(z_iv) / sum_v exp(z_iv):
 *
 *   L_i = T^2 [ sum_k q_ik log q_ik + sum_k q_ik (lse_i - z_{i j_ik}) ],  lse_i = log sum_v exp(z_iv)
 *   G_iv = T c_i [ Q_i p_iv - sum_k q_ik 1(j_ik = v) ]
 *   dhidden = G weight,  dweight = G^T hidden
 *
 * Pointers are device memory on the current device; hidden, weight and their gradients are
 * bfloat16, all sums float32 or wider.  Nothing is allocated or synchronised.  Results are
 * deterministic: sums run in a fixed order, and only counts and places in lists whose order changes
 * nothing come from (LDS) atomics.  Status codes are those of theseus_wkv7.h: sizes out of range
 * THESEUS_WKV7_ERR_SHAPE, an unknown type _ERR_DTYPE, an unknown kind or reduction _ERR_FLAGS.
 */
#ifndef THESEUS_VOCAB_H
#define THESEUS_VOCAB_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* hipStream_t;

enum theseus_vocab_dtype { THESEUS_VOCAB_BF16 = 0, THESEUS_VOCAB_FP32 = 1 };
enum theseus_vocab_reduction { THESEUS_VOCAB_NONE = 0, THESEUS_VOCAB_SUM = 1, THESEUS_VOCAB_MEAN = 2 };

/* targets of one token, k of theseus_vocab_top */
#define THESEUS_VOCAB_MAX_TOP 256

typedef struct theseus_vocab_loss_args {
    long long rows;          /* M >= 0 (0: the reduced loss and dweight are 0)                 */
    long long vocab;         /* V in 1 .. 2^22                                                 */
    int width;               /* D in 1 .. 2^17                                                 */
    int targets;             /* K in 1 .. THESEUS_VOCAB_MAX_TOP (labels: 1)                    */
    const void* hidden;      /* bfloat16 [M][D], hidden_stride elements from row to row        */
    const void* weight;      /* bfloat16 [V][D], weight_stride elements from row to row        */
    long long hidden_stride, weight_stride; /* at least D (of one row: not used); weight_stride up to 2^21.
                                Rows that are not 16-byte aligned, not whole multiples of 64 wide or (hidden)
                                more than 2^21 elements apart are copied in the workspace            */
    const int64_t* index;    /* [M][K]: the labels, or the teacher's top indices               */
    const void* top_values;  /* [M][K] the teacher's logits; NULL: index holds labels (K = 1,
                                q = 1, rows with ignore_index left out)                        */
    int top_dtype;           /* theseus_vocab_dtype of top_values                              */
    int reduction;           /* theseus_vocab_reduction                                        */
    const float* teacher_lse;/* [M] log sum exp(teacher's logits / T): q = exp(t / T - lse);
                                NULL: q = exp(t / T) over its sum over the K                   */
    const float* row_weight; /* [M] factor of each token's loss, NULL: 1                       */
    long long ignore_index;
    float temperature;       /* T > 0                                                          */
    float* loss;             /* reduction NONE: [M], row_weight_i L_i; SUM: their sum; MEAN:
                                the sum over the sum of the weights (labels: over the labels
                                that count), 0 where that is 0.  May be NULL                   */
    const float* row_grad;   /* [M] upstream gradient of each token's loss, NULL: 1            */
    void* dhidden;           /* bfloat16 [M][D], or NULL                                       */
    void* dweight;           /* bfloat16 [V][D], or NULL                                       */
    long long piece_rows;    /* tokens whose probabilities (V 16-bit values each) are in the
                                workspace at a time, 0: as many as 2 GiB hold.  Rounded up to
                                a multiple of 256                                              */
    void* kept;              /* theseus_vocab_loss_kept_size bytes: what the forward of a call with
                                reduction NONE leaves for its gradients                        */
    int phase;               /* theseus_vocab_phase                                            */
} theseus_vocab_loss_args;

/* ALL: the losses and, where asked for, the gradients.  With kept of the size given, reduction
 * NONE and gradients that are wanted later: FORWARD writes the losses and kept (dhidden, dweight
 * and row_grad are not looked at), GRADIENTS with the same other arguments reads kept (and
 * destroys it) and writes the gradients without forming the logits again. */
enum theseus_vocab_phase { THESEUS_VOCAB_ALL = 0, THESEUS_VOCAB_FORWARD = 1, THESEUS_VOCAB_GRADIENTS = 2 };
/* most that is kept: a call with more in its row pieces (V 16-bit values a token) keeps nothing and forms its
 * logits twice.  A bound on memory held from the forward to the backward, which costs a fourth product
 * beyond it: 65536 words, width 5120, both gradients, 1984 tokens (kept) 1607 ns a token, 2112 (not kept) 2256,
 * 4096 2027; reduced losses of as many 1606, 1718, 1559 */
#define THESEUS_VOCAB_MAX_KEPT (256ll << 20)

/* c_i of the gradients is row_grad_i row_weight_i, over the sum of the weights for MEAN.  A
 * token whose row_weight_i is 0 or whose label is ignored adds nothing, whatever its row_grad_i, nor to the
 * gradients one whose c_i is 0 (its hidden state has to be finite all the same where dweight is asked for:
 * 0 times it is added).
 * Target entries with q = 0 (a teacher's -inf) are not looked at; one with q != 0 whose index is
 * outside the vocabulary makes the token's loss NaN (and adds nothing to the gradients but p). */
size_t theseus_vocab_loss_workspace_size(const theseus_vocab_loss_args* args);
size_t theseus_vocab_loss_kept_size(const theseus_vocab_loss_args* args); /* 0: nothing can be kept */
int theseus_vocab_loss(const theseus_vocab_loss_args* args, void* workspace, size_t workspace_bytes,
                       hipStream_t stream);

/* x and y *= *factor for nx and ny bfloat16 values (a NULL of 0 values is left out), nothing moved
 * where the factor (device memory) is 1. */
int theseus_vocab_scale(void* x, long long nx, void* y, long long ny, const float* factor, hipStream_t stream);

/* logits [M][V] bfloat16 or float32, row_stride elements from row to row, M >= 0, V in
 * 1 .. 2^30, k in 1 .. min(V, THESEUS_VOCAB_MAX_TOP).  values [M][k] in the logits' type and
 * indices [M][k], largest first, equal values by the lowest index, NaN above every number;
 * lse [M] = log sum exp(logits / temperature), may be NULL.  Rows are read in whole granules of 16 aligned
 * bytes: up to 15 bytes on either side of the first and last row are read too (never across such a
 * boundary, so never beyond a page) and not looked at. */
size_t theseus_vocab_top_workspace_size(long long rows, long long vocab, int k, int dtype);
int theseus_vocab_top(long long rows, long long vocab, int k, int dtype, float temperature, const void* logits,
                      long long row_stride, void* values, int64_t* indices, float* lse, void* workspace,
                      size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* THESEUS_VOCAB_H */

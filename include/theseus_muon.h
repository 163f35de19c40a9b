/*
 * theseus_muon.h -- C ABI of the orthogonalised updates in libtheseus_wkv7.so (gfx950).
 *
 * A matrix X [m][n] is brought near the orthogonal factor of its polar decomposition by an odd
 * polynomial of its singular values, in products alone (Newton-Schulz), with p = min(m, n):
 *
 *   X_0 = X / max(|X|_F, eps)
 *   A = X_i X_i^T  (m > n: X_i^T X_i),  B = b A + c A^2,  X_{i+1} = a X_i + B X_i  (m > n: X_i B)
 *
 *   theseus_orthogonalize   X_steps of a list of matrices, in bfloat16
 *   theseus_muon_step       the optimizer that steps along it: with g = grad factor,
 *                             momentum = mu momentum + (1 - mu) g
 *                             u = mu momentum + (1 - mu) g  (without nesterov: momentum)
 *                             param = param keep - step X_steps(u)
 *
 * All pointers are device memory on the current device; the lists and ns are read during the call only (host
 * memory).  Nothing is allocated or synchronised, so the calls may be captured into a graph.  Results
 * are deterministic: the same list gives the same bits (in another list a matrix' sums may be cut otherwise).  The
 * products take float16 operands (scaled into its range) and add in float32; X itself is held in two float16 halves, 22
 * bits, the last step's operand in one.  Coefficients that keep the singular values of X_0 .. X_{steps-1} below 3 and
 * |a + b s^2 + c s^4| below 32 for them cannot overflow; others may, and give values that are not finite.
 * Status codes are those of theseus_wkv7.h.
 */
#ifndef THESEUS_MUON_H
#define THESEUS_MUON_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* hipStream_t;

enum theseus_muon_dtype { THESEUS_MUON_BF16 = 0, THESEUS_MUON_FP32 = 1 };

typedef struct theseus_newton_schulz {
    int steps;      /* 1 .. 100                */
    float a, b, c;  /* finite                  */
    float eps;      /* >= 0, less than 1e-30 as 1e-30 */
} theseus_newton_schulz;

typedef struct theseus_orthogonalize_matrix {
    const void* x;          /* [rows][cols], row_stride elements from row to row               */
    void* out;              /* bfloat16 [rows][cols], contiguous                               */
    long long row_stride;   /* cols .. 2^21 (of one row: not used)                             */
    int rows, cols;         /* 0 .. 2^17 (0: skipped)                                          */
    int dtype;              /* theseus_muon_dtype of x                                         */
} theseus_orthogonalize_matrix;

typedef struct theseus_muon_matrix {
    float* param;           /* [rows][cols], contiguous as all of the three; updated in place  */
    const float* grad;      /* read only                                                       */
    float* momentum;        /* updated in place                                                */
    int rows, cols;         /* 0 .. 2^17 (0: skipped)                                          */
    float keep;             /* 1 - lr weight_decay                                             */
    float step;             /* lr, times what the shape asks for                               */
} theseus_muon_matrix;

size_t theseus_orthogonalize_workspace_size(const theseus_orthogonalize_matrix* matrices, int count);
int theseus_orthogonalize(const theseus_orthogonalize_matrix* matrices, int count, const theseus_newton_schulz* ns,
                          void* workspace, size_t workspace_bytes, hipStream_t stream);

/* factor = grad_scale min(1, max_norm / (norm + 1e-6)) with the L2 norm of grad_scale grad over all matrices,
 * formed in device memory ahead of the step; max_norm < 0 or NaN: grad_scale alone, no norm.  result: 3
 * floats of device memory as theseus_adamw_step writes them, norm, factor and 1 where the norm is
 * not finite (without a norm NaN, grad_scale and 0 if there is anything to step; may then be NULL).  With
 * skip_nonfinite a norm that is not finite leaves every param and momentum unchanged. */
size_t theseus_muon_workspace_size(const theseus_muon_matrix* matrices, int count);
int theseus_muon_step(const theseus_muon_matrix* matrices, int count, const theseus_newton_schulz* ns, double momentum,
                      int nesterov, float grad_scale, float max_norm, int skip_nonfinite, float* result, void* workspace,
                      size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* THESEUS_MUON_H */

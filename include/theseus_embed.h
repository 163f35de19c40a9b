/*
 * theseus_embed.h -- C ABI of the token embedding in libtheseus_wkv7.so (gfx950): M rows of
 * a table [V][D] by index, times a factor, and the table's gradient.
 *
 *   theseus_embed_lookup   out_i = scale weight_{ids_i}
 *   theseus_embed_grad     dweight_v = scale sum_{i: ids_i = v} grad_i
 *
 * Pointers are device memory on the current device, tables and rows bfloat16 or float32 (any mix),
 * aligned to their elements.  Products and sums are float32, rounded once to the result's type.
 * The sums run in the tokens' order, in parts whose bounds follow from M, D and the indices alone:
 * results are deterministic.  Nothing is allocated or synchronised, so the calls may be captured
 * into a graph.  Status codes are those of theseus_wkv7.h: sizes out of range
 * THESEUS_WKV7_ERR_SHAPE, an unknown type _ERR_DTYPE.
 */
#ifndef THESEUS_EMBED_H
#define THESEUS_EMBED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* hipStream_t;

enum theseus_embed_dtype { THESEUS_EMBED_BF16 = 0, THESEUS_EMBED_FP32 = 1 };

/* ids [M], M in 0 .. 2^30; weight [V][D], weight_stride >= D elements from row to row, V in
 * 1 .. 2^22, D in 1 .. 2^17; out [M][D].  An index outside 0 .. V-1 makes its row NaN. */
int theseus_embed_lookup(long long rows, long long vocab, int width, int weight_dtype, int out_dtype,
                         const int64_t* ids, const void* weight, long long weight_stride, float scale,
                         void* out, hipStream_t stream);

/* grad [M][D], grad_stride elements from row to row (0: one row for all tokens, else >= D); dweight [V][D] is written whole,
 * rows that no token asks for as 0.  Tokens whose index is `skip` (-1: none) or outside 0 .. V-1
 * add nothing, and their rows of grad are not looked at. */
size_t theseus_embed_grad_workspace_size(long long rows, long long vocab, int width);
int theseus_embed_grad(long long rows, long long vocab, int width, int grad_dtype, int weight_dtype,
                       const int64_t* ids, long long skip, const void* grad, long long grad_stride, float scale,
                       void* dweight, void* workspace, size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* THESEUS_EMBED_H */

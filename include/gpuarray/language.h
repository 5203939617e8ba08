/* Operators of language models: rows of an embedding table, log probabilities
 * of tokens, the gradients of both, and the global norm of many arrays with
 * clipping by it.
 *
 * The reference has none of these.  They stand beside what it does have:
 * GpuArray_take1 gathers rows (src/gpuarray/array.h:348-366),
 * GpuArray_maxandargmax reduces rows of logits (:607-644), and a norm and its
 * clipping are a reduction and an elementwise expression over every array.
 *
 * Common rules
 *   types    values are GA_FLOAT, GA_HALF or GA_BFLOAT16 (norms also
 *            GA_DOUBLE); ids are any integer type of up to 64 bits.  Sums,
 *            softmax statistics and norms are held in 32 bits or more and a
 *            result is rounded once, to nearest even.
 *   layout   rows (the last axis) have unit stride; any other stride is
 *            taken as it is, negative and zero ones too (results must not
 *            overlap themselves, and the memory from a result's first element
 *            to its last holds no other argument).  Rows need not be aligned to more than
 *            their element.
 *   ids      a negative id counts from the end of the vocabulary, as in
 *            GpuArray_take1, except the id `ignore`, which stands for no
 *            token (GA_NO_IGNORE: no id does).  An unsigned one of 2^63 or
 *            more is out of range.  An id out of range never
 *            reads or writes memory: it sets the context's error word, which
 *            `check_error` reads back (blocking), resets and reports as
 *            GA_VALUE_ERROR "Index out of bounds", and which otherwise stays
 *            set for the next checked call.
 *   errors   GA_INVALID_ERROR (shapes, layouts, contexts), GA_VALUE_ERROR (values,
 *            results that overlap an operand or themselves), GA_UNALIGNED_ERROR,
 *            GA_UNSUPPORTED_ERROR (types), GA_XLARGE_ERROR; nothing has been
 *            launched then.
 *   order    results are the same bits on every call with the same arguments.
 *   graphs   a call on a stream that records a graph launches kernels only,
 *            once an earlier call of the same types and sizes has built the kernels
 *            and grown the context's scratch; otherwise it is refused with
 *            GA_UNSUPPORTED_ERROR, and so is a call with `check_error`, which
 *            would wait.  Partial results lie in that scratch, so
 *            graphs recorded from a context are replayed on its stream, one
 *            after the other (as for GpuReduction_call).
 */
#ifndef GPUARRAY_LANGUAGE_H
#define GPUARRAY_LANGUAGE_H

#include <gpuarray/array.h>
#include <gpuarray/buffer.h>

#ifdef __cplusplus
extern "C" {
#endif

/* No id stands for "no token". */
#define GA_NO_IGNORE ((ssize_t)((size_t)1 << (8 * sizeof(ssize_t) - 1)))

/* out[i, :] = scale * table[ids[i], :]
 *   out (n, d), table (v, d), ids (n); out and table may differ in type.
 * A row whose id is `ignore` is zeros; a row whose id is out of range is left
 * as it was. */
GPUARRAY_PUBLIC int GpuArray_embedding(GpuArray *out, const GpuArray *table,
                                       const GpuArray *ids, double scale,
                                       ssize_t ignore, int check_error);

/* Gradient of GpuArray_embedding with respect to the table:
 *   grad[r, :] = scale * sum of dout[i, :] over the i with ids[i] == r
 * with rows of no token zero, or, with `accumulate`, added to what grad holds
 * (rows of no token are not touched then).
 *   grad (v, d), dout (n, d), ids (n); grad and dout may differ in type.
 * The sum of a row runs over its tokens in a fixed order, in 32 bits, and is
 * rounded once.  Ids that are `ignore` or out of range contribute nothing. */
GPUARRAY_PUBLIC int GpuArray_embedding_grad(GpuArray *grad,
                                            const GpuArray *dout,
                                            const GpuArray *ids, double scale,
                                            ssize_t ignore, int accumulate,
                                            int check_error);

/* Largest number of alternatives of GpuArray_token_logprobs. */
#define GA_TOKEN_LOGPROBS_MAX_TOP 64

/* Log probabilities under p(j) = exp(scale * x[j]) / sum_k exp(scale * x[k])
 * for each row x of logits (t, v); scale > 0 is an inverse temperature, in 32
 * bits and with scale * log2(e) in 32 bits too (up to 2.3e38).
 *   logp      (t)     log p of ids[i]; 0 where ids[i] is `ignore`, NaN where
 *                     it is out of range
 *   entropy   (t)     -sum p log p
 *   stats     (t, 2)  largest logit m, and log sum_k exp(scale * (x[k] - m)):
 *                     what GpuArray_token_logprobs_grad needs of a row
 *   top_logp  (t, k)  the k largest log probabilities in descending order and
 *   top_ids   (t, k)  their ids (GA_INT or GA_LONG); of equal logits the lower
 *                     id comes first; k <= GA_TOKEN_LOGPROBS_MAX_TOP, k <= v
 * Every result is GA_FLOAT (but top_ids) and may be NULL; logp and ids go
 * together, top_logp and top_ids too.
 *   Logits of -inf have probability 0.  In a row with nothing but -inf every log probability and
 * the second statistic are -inf, the entropy is 0 and the alternatives are
 * ids 0 to k - 1.  In a row with a NaN or a +inf every value is NaN (the first
 * statistic is the largest number, or NaN if a NaN is a signaling one) and the
 * alternatives are ids 0 to k - 1. */
GPUARRAY_PUBLIC int GpuArray_token_logprobs(GpuArray *logp, GpuArray *entropy,
                                            GpuArray *stats,
                                            GpuArray *top_logp,
                                            GpuArray *top_ids,
                                            const GpuArray *logits,
                                            const GpuArray *ids, double scale,
                                            ssize_t ignore, int check_error);

/* Gradient of sum_i dlogp[i] * logp[i] + dentropy[i] * entropy[i] with respect
 * to the logits:
 *   dlogits[i, j] = scale * (dlogp[i] * ([j == ids[i]] - p(j))
 *                            - dentropy[i] * p(j) * (log p(j) + entropy[i]))
 *   stats and entropy are what GpuArray_token_logprobs left for these logits
 *   and this scale; ids and dlogp go together, entropy and dentropy too, and
 *   either pair may be NULL.  An id that is `ignore` or out of range has no
 *   part through dlogp.  A row with nothing but -inf has gradient 0.
 * dlogits has the shape and type of logits and may be the same array (the
 * gradient then replaces the logits); any other overlap is refused. */
GPUARRAY_PUBLIC int GpuArray_token_logprobs_grad(
    GpuArray *dlogits, const GpuArray *logits, const GpuArray *ids,
    const GpuArray *stats, const GpuArray *dlogp, const GpuArray *entropy,
    const GpuArray *dentropy, double scale, ssize_t ignore, int check_error);

/* norm = sqrt(sum of the squares of all elements of the n arrays), summed in
 * 64 bits, also of doubles whose squares are in none.  norm is 0-d (or has one element), GA_FLOAT or GA_DOUBLE.  The
 * arrays are contiguous, in either order, of any shapes and of mixed types;
 * one that is listed twice counts twice. */
GPUARRAY_PUBLIC int GpuArray_global_norm(GpuArray *norm, const GpuArray **as,
                                         size_t n);

/* rs[i] = as[i] * (max_norm / norm) if the global norm of the as is finite and
 * above max_norm, else rs[i] = as[i], without waiting for the norm on the
 * host.  rs[i] may be as[i] itself (rs == NULL: all of them are) or an array
 * of its shape, type and strides; no other overlap, between any two, is allowed.
 * The factor is rounded to 32 bits (64 for GA_DOUBLE), the product once; where the
 * factor is too small to be a normal number of that type, as[i] is divided by norm first, in 64 bits.
 * norm receives the norm before clipping, and may be NULL. */
GPUARRAY_PUBLIC int GpuArray_clip_global_norm(GpuArray **rs,
                                              const GpuArray **as, size_t n,
                                              double max_norm, GpuArray *norm);

/* The same for a list that is clipped again and again, of any length: an
 * operator that holds the arrays' buffers (retained until it is freed) and a
 * table of them in device memory.  The arrays count as they are when it is
 * made; rs == NULL: for norms alone; rs may be `as`, or name `as` elements, to clip in place.
 * Making one copies the table to the device, and is refused while the stream
 * records a graph; calls may be recorded, and replayed until it is freed. */
typedef struct _GpuGlobalNorm GpuGlobalNorm;
GPUARRAY_PUBLIC int GpuGlobalNorm_new(GpuGlobalNorm **g, gpucontext *ctx,
                                      const GpuArray **as, GpuArray **rs,
                                      size_t n);
GPUARRAY_PUBLIC void GpuGlobalNorm_free(GpuGlobalNorm *g);
/* GpuArray_global_norm and GpuArray_clip_global_norm on its arrays. */
GPUARRAY_PUBLIC int GpuGlobalNorm_norm(const GpuGlobalNorm *g, GpuArray *norm);
GPUARRAY_PUBLIC int GpuGlobalNorm_clip(const GpuGlobalNorm *g, double max_norm,
                                       GpuArray *norm);

#ifdef __cplusplus
}
#endif
#endif

/* Key/value cache held in 8 bits, and attention over it.
 *
 * A cache holds the keys and values of `batch` sequences and `kv_heads` heads
 * of one attention layer, up to `capacity` tokens each, in device memory of
 * its own. Tokens come in blocks of TENSOR_KV_CACHE_BLOCK. A full block's keys
 * (and likewise its values) of one head are held as int8 codes with one f32
 * scale: with a the largest |x| of the block, x being the appended elements
 * rounded to f16,
 *     scale = a / 127,   code = 127 x / a rounded to nearest, ties to even,
 * and stand for the f32 product code * scale. The tokens of the last, partial
 * block are held in f16 until the block is full, so what a cache holds does not
 * depend on how its tokens were split over calls.
 *
 * A token whose key or value holds, in some head, an element that is no
 * finite f16 (NaN, infinite, or an f32 of 65520 and more) is marked in that
 * head: its score is NaN for every query row that sees it, and it reads back
 * as NaN. It has no effect on rows that do not see it nor on its block's
 * scales.
 *
 * No counterpart in the reference (its caches are f16/f32 tensors of the model
 * harnesses). Conventions are those of tensor_ops_ext.h, with these of the
 * cache:
 *   - tensor operands are device tensors; calls enqueue on the SDK stream and
 *     return;
 *   - lengths are kept on the host too, so every check is made before any work
 *     is queued, and a call that is refused leaves the cache as it was. Should
 *     the runtime fail to launch a kernel, the sequences of the launches before
 *     it (256 in each) are done and the others as they were, and the lengths
 *     say which; of an eviction the target is as it was, of a
 *     reorder the cache;
 *   - `counts`, where a call takes it, is a host array of `batch` numbers: of
 *     sequence b only the first counts[b] tokens (or query rows) are there and
 *     the rest of its rows is padding, neither read nor written. NULL: all are
 *     there;
 *   - append, truncate, evict and copy change lengths and are refused while the
 *     SDK stream records a graph. Attention, read and reorder may be recorded: a
 *     replay works on what the cache then holds;
 *   - calls from several host threads are safe; a cache is freed, and replayed
 *     graphs that use it are destroyed, when no call uses it.
 */
#ifndef TENSOR_KV_CACHE_H
#define TENSOR_KV_CACHE_H

#include "tensor_buffer.h"

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TENSOR_KV_CACHE_BLOCK 64

typedef struct TensorKvCache TensorKvCache;

/* An empty cache. head_dim (of keys) and value_dim: 1 to 256, any number;
   capacity up to 2^27, batch up to 65535, kv_heads up to 4096, and batch *
   kv_heads * capacity (in whole blocks) up to 2^31. */
int tensor_kv_cache_create(size_t batch, size_t kv_heads, size_t capacity,
                           size_t head_dim, size_t value_dim,
                           TensorKvCache **result, char *error,
                           size_t error_capacity);
/* Waits for queued work, then frees. NULL is ignored. */
void tensor_kv_cache_free(TensorKvCache *cache);
/* Tokens of a sequence (0 for NULL or a sequence past the batch). */
size_t tensor_kv_cache_length(const TensorKvCache *cache, size_t sequence);
size_t tensor_kv_cache_capacity(const TensorKvCache *cache);
/* Device bytes the cache takes. */
size_t tensor_kv_cache_byte_length(const TensorKvCache *cache);

/* Appends n tokens to every sequence (counts[b] <= n to sequence b): key
   [batch, kv_heads, n, head_dim], value [batch, kv_heads, n, value_dim]. */
int tensor_kv_cache_append_f32(TensorKvCache *cache, const TensorBuffer *key,
                               const TensorBuffer *value,
                               const uint32_t *counts, char *error,
                               size_t error_capacity);
int tensor_kv_cache_append_f16(TensorKvCache *cache, const TensorBuffer *key,
                               const TensorBuffer *value,
                               const uint32_t *counts, char *error,
                               size_t error_capacity);

/* Cuts sequence b to its first lengths[b] tokens (host array, none above the
   present length; NULL empties every sequence). Where a full block is cut, the
   tokens that stay of it go on in f16 as the values they stood for. */
int tensor_kv_cache_truncate(TensorKvCache *cache, const uint32_t *lengths,
                             char *error, size_t error_capacity);

/* The values the cache holds: key [batch, kv_heads, rows, head_dim] and value
   [batch, kv_heads, rows, value_dim] with rows at least the longest length;
   rows from a sequence's length on are left as they were. Either output may be
   NULL. */
int tensor_kv_cache_read_f32(const TensorKvCache *cache, TensorBuffer *key,
                             TensorBuffer *value, char *error,
                             size_t error_capacity);
int tensor_kv_cache_read_f16(const TensorKvCache *cache, TensorBuffer *key,
                             TensorBuffer *value, char *error,
                             size_t error_capacity);

/* Attention over the cache: query [batch, query_heads, n, head_dim], output
   [batch, query_heads, n, value_dim], query head h reads kv head
   h / (query_heads / kv_heads). With causal != 0 the rows are the last tokens
   of their sequence: row i of counts[b] (of n) sees the first
   length - counts[b] + i + 1 tokens, none where that is not positive. With
   causal == 0 every row sees every token (cross attention). The row rules are
   tensor_sdpa_device's: a row that sees nothing, or whose largest score is not
   finite, is zeros; one with a NaN score beside finite ones is NaN. f32 sums
   throughout; with f16 tensors the softmax weights are rounded to f16 in the
   product with the values.
   weights, F32 [batch, kv_heads, tokens] with tokens at least the longest
   length, or NULL: weights[b, h, t] += the softmax weight that token t got,
   summed over the rows and query heads of kv head h (rows whose output is not
   finite, and padded ones, add nothing). They go by scores rounded to f32,
   each weight off by 2^-24 of its score; f32 outputs go by what that rounding
   takes off as well. */
int tensor_kv_cache_attention_f32(const TensorKvCache *cache,
                                  const TensorBuffer *query,
                                  const uint32_t *counts, float scale,
                                  int causal, TensorBuffer *weights,
                                  TensorBuffer *output, char *error,
                                  size_t error_capacity);
int tensor_kv_cache_attention_f16(const TensorKvCache *cache,
                                  const TensorBuffer *query,
                                  const uint32_t *counts, float scale,
                                  int causal, TensorBuffer *weights,
                                  TensorBuffer *output, char *error,
                                  size_t error_capacity);

/* Moves into `target` (another cache of the same batch, heads and dims,
   capacity at least `keep`; what it held is dropped) the tokens that each kv
   head keeps of `cache`, in their order: of a sequence of at most `keep`
   tokens all, else exactly `keep`, namely the first `first` and the last
   `recent` tokens and of the others those of largest weights[b, h, t] (F32
   [batch, kv_heads, tokens], tokens at least the longest length; the earlier
   of two equal ones; NaN counts as lowest). weights NULL: of the others the
   latest, a sliding window behind `first`. first + recent <= keep. Full blocks
   are held anew from the values that the kept tokens stood for.
   kept, U32 [batch, kv_heads, slots] or NULL: the index in `cache` of each
   kept token; target_weights, F32 of the same shape or NULL (needs weights):
   its weight; slots at least keep or the longest length, whichever is less.
   Entries past a head's kept tokens are left as they were. */
int tensor_kv_cache_evict(const TensorKvCache *cache,
                          const TensorBuffer *weights, size_t first,
                          size_t recent, size_t keep, TensorKvCache *target,
                          TensorBuffer *target_weights, TensorBuffer *kept,
                          char *error, size_t error_capacity);

/* ---- several continuations of one prompt ---------------------------------- */

/* An entry of `source` that leaves its sequence of the target as it is. */
#define TENSOR_KV_CACHE_KEEP UINT32_MAX

/* Sequence b of `target` becomes a copy, as it is held, of sequence source[b] of
   `cache` (a host array of the target's batch; an entry may be repeated):
   a prompt into its beams or a free slot, a batch closed up. The target has the
   cache's heads and dims, room for what it gets, and any batch and capacity. It
   may be the cache itself, where no sequence that is copied is replaced. Changes
   lengths: not recorded into a graph. */
int tensor_kv_cache_copy(const TensorKvCache *cache, const uint32_t *source,
                         TensorKvCache *target, char *error,
                         size_t error_capacity);

/* Beams follow their choice (tensor_beam_select, tensor_ops_ext.h), in place: with
   parents U32 [groups, beams], groups * beams the cache's batch, sequence
   g * beams + i becomes what sequence g * beams + parents[g, i] was. 1 to 64
   beams. The parents are on the device: the call does not wait for them, and an
   index not below `beams` leaves its sequence as it is. The sequences of a group
   are of one length, at each replay of a recorded call too. */
int tensor_kv_cache_reorder(TensorKvCache *cache, const TensorBuffer *parents,
                            char *error, size_t error_capacity);

/* tensor_kv_cache_attention of sequences whose tokens follow a prefix that
   several of them share: the first members[0] sequences of `cache` continue
   sequence 0 of `prefix`, the next members[1] sequence 1, and so on (host
   array of the prefix's batch, zeros allowed, in all the cache's batch; NULL:
   equal groups). Each query row sees every token of its prefix and, of its
   sequence's own tokens in `cache`, those that tensor_kv_cache_attention lets it
   see; one softmax goes over both. A prefix's tokens are read once for all of its
   sequences, or once for many. The caches have the same heads and dims. Query
   rows of all sequences and heads together: at most 2^26. */
int tensor_kv_cache_attention_shared_f32(const TensorKvCache *prefix,
                                         const TensorKvCache *cache,
                                         const TensorBuffer *query,
                                         const uint32_t *members,
                                         const uint32_t *counts, float scale,
                                         int causal, TensorBuffer *output,
                                         char *error, size_t error_capacity);
int tensor_kv_cache_attention_shared_f16(const TensorKvCache *prefix,
                                         const TensorKvCache *cache,
                                         const TensorBuffer *query,
                                         const uint32_t *members,
                                         const uint32_t *counts, float scale,
                                         int causal, TensorBuffer *output,
                                         char *error, size_t error_capacity);

#ifdef __cplusplus
}
#endif

#endif

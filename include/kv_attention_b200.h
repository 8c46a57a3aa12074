/* C ABI of the batched KV-cache decode attention (libmoe_b200.so, sm_100a).
 *
 * Replaces, for many sequences at once, the attention arithmetic of
 * MultiHeadAttention::forward_cached (reference attention.rs:344-398): rotate the new queries and keys
 * (rope.rs:170-225, rotate-half pairing of channel j with j + head_dim / 2), append the new keys and
 * values to each sequence's cache (KvCache::append, attention.rs:65-78: post-RoPE rows of
 * kv_heads * head_dim values), then for every new row softmax(q . K^T / sqrt(head_dim)) V over the
 * positions it may see (head_scores, attention.rs:1100-1130; accumulate_head_output, :1133-1160; query
 * head h reads key/value head h / (num_heads / kv_heads)).  The projections around it (query, key,
 * value, output Linear layers) stay with the caller, as they do for the MoE layer.
 *
 * The reference decodes one sequence per call; here `sequences` caches advance together, each with its
 * own length.  All pointers are device pointers unless said otherwise.  Status codes are the moe_status
 * values of moe_b200.h.  Calls on one cache are ordered by the caller (one stream, or events between streams): they share its lengths and
 * its workspace; two captured graphs of one cache may be replayed one after the other, not at once.
 *
 * A cache of MOE_PRECISION_Q4 holds 4 bits a channel.  For every position, kv head and run of 32 channels of its key (after the rotation)
 * and of its value:
 *     step = bf16((high - low) / 15),  base = bf16(low),  code = clamp(round((x - base) / step), 0, 15)   (0 where step is 0)
 *     what the cache stands for = code * step + base
 * in f32 arithmetic, rounding to even, rotation included (two products and their sum, not contracted; the angles are computed in 64 bits).
 * A step's own new positions are read back from the cache like all others.  If a position's key or value of a kv head holds a NaN, an
 * infinity or a number above 2^40 in magnitude, its key and value stand for NaN: what attends to it is NaN, what does not is untouched.
 * A query with an infinity, a NaN or a number above 2^116 (after the rotation) may give NaN, in its own row and head.
 * What the attention rounds on the way: the rotated query to f16 under a power of two of its own (2^-11 of a channel at most), what the cache
 * stands for of a value to bf16 (2^-8 of it), a weight to two bf16 numbers (2^-16), the result to bf16.  Keys are not rounded; scores, the softmax's
 * maximum and sum and the sums of products are f32.  Against 64 bits that is 2.0e-3 to 2.4e-3 of the result, of which its own rounding is 1.7e-3.
 * kv_attention_forward_cached, kv_cache_append, kv_cache_rollback and kv_cache_newest allocate nothing on such a cache, so every step can be
 * captured, and q is left alone; kv_cache_read may grow a buffer, and it waits for the stream.  At most 2^30 positions.
 */
#ifndef KV_ATTENTION_B200_H
#define KV_ATTENTION_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct kv_cache kv_cache_t;

typedef struct {
  int32_t sequences;    /* caches that advance together */
  int32_t num_heads;    /* query heads */
  int32_t kv_heads;     /* key/value heads; num_heads is a multiple (attention.rs:178) */
  int32_t head_dim;     /* 8, 16, 32, 64, 128 or 256 */
  int32_t capacity;     /* positions per sequence (KvCache::with_capacity, attention.rs:39-48) */
  int32_t max_seq_len;  /* length of the RoPE tables (rope.rs:71-97); capacity <= max_seq_len */
  float rope_base;      /* 10000.0 in the reference's configs */
  int32_t rope;         /* 0: no rotation (rope_enabled == false) */
  int32_t precision;    /* MOE_PRECISION_F32 (0) or MOE_PRECISION_BF16 (1): type of q, k, v, out and of the cache;
                           MOE_PRECISION_Q4 (3): bf16 q, k, v and out, the cache in 4 bits (head_dim 32, 64, 128 or 256) */
  int32_t device;
} kv_cache_config_t;

/* KvCache::with_capacity for `sequences` sequences.  InvalidConfig for the shapes the reference refuses
 * (attention.rs:173-186, rope.rs:72-76) and for head_dim values the kernels do not cover. */
int32_t kv_cache_create(const kv_cache_config_t* config, kv_cache_t** out);
void kv_cache_destroy(kv_cache_t* cache);
const char* kv_cache_last_error(const kv_cache_t* cache);

/* KvCache::clear (attention.rs:58-62) for every sequence, or for one when sequence >= 0. */
int32_t kv_cache_clear(kv_cache_t* cache, int32_t sequence, void* stream);

/* KvCache::len of every sequence into host memory (read from the device; synchronises the stream).
 * The capacity checks of the calls below use a host copy of the lengths that every call keeps up to
 * date; a step replayed from a captured CUDA graph advances the device lengths only, and this call
 * brings the host copy back in line.  A replayed step that no longer fits is caught on the device: for a
 * sequence whose cache cannot take the step's rows the kernels store nothing, leave its length alone, write
 * zeros as its merged heads and mark it; the other sequences of the call proceed.  This call reports such a
 * mark as MOE_INVALID_INPUT ("SequenceTooLong", attention.rs:364-371) once and clears it; kv_cache_clear /
 * kv_cache_truncate of the sequence clear it too. */
int32_t kv_cache_lengths(kv_cache_t* cache, int32_t* lengths_host, void* stream);

/* forward_cached without the projections, for sequences first_sequence .. first_sequence + n_sequences - 1
 * (all of them for a decode step, one of them for the prefill of a new request).
 * q [n_sequences * rows_per_sequence, num_heads * head_dim], k and v [same rows, kv_heads * head_dim],
 * rows of one sequence adjacent (row = j * rows_per_sequence + i for the j-th sequence of the range);
 * row i of a sequence sits at position len + i and sees positions 0 ..= len + i.  q, k and v are the
 * projections BEFORE rotation (`project`, attention.rs:920-944, rotates queries and keys; here the call
 * does).  q starts on a 16-byte boundary (InvalidInput where a kernel would load across one; a 4-bit cache takes any).
 * q is scratch: one kernel path rotates it in place, the other rotates in registers and leaves it
 * alone, so its contents after the call are unspecified; k and v are read only.
 * merged [rows, num_heads * head_dim] is the input of the output projection; it may be q itself and overlaps nothing else.
 * SequenceTooLong -> MOE_INVALID_INPUT when a cache would pass its capacity (rope.rs:194-200); nothing
 * is appended in that case. */
int32_t kv_attention_forward_cached(kv_cache_t* cache, int32_t first_sequence, int32_t n_sequences, void* q,
                                    const void* k, const void* v, int32_t rows_per_sequence, void* merged,
                                    void* stream);

/* Drops the newest positions of a sequence (all sequences when sequence < 0) so that `length` remain;
 * a length above the current one is InvalidInput.  Used to replay a decode step at a fixed history. */
int32_t kv_cache_truncate(kv_cache_t* cache, int32_t sequence, int32_t length, void* stream);

/* KvCache::append (attention.rs:65-78) without a query: rotates and stores rows new keys and values for each sequence of the range, layout
 * as above, and moves the lengths on.  Fills a cache whose attention output is not wanted (a prompt's prefix, a cache handed over). */
int32_t kv_cache_append(kv_cache_t* cache, int32_t first_sequence, int32_t n_sequences, const void* k, const void* v,
                        int32_t rows_per_sequence, void* stream);

/* Takes back the newest rows of each sequence of the range (draft tokens that were not accepted).  Unlike kv_cache_truncate it counts from
 * each sequence's own length, on the device, so that a captured step can contain it.  The rows of steps that were skipped for want of room
 * since the last step that was taken are the newest ones: they count first, and taking them back changes nothing else, until kv_cache_lengths
 * has reported the mark; from then on the host knows that they are not there.  More rows than a sequence holds are InvalidInput. */
int32_t kv_cache_rollback(kv_cache_t* cache, int32_t first_sequence, int32_t n_sequences, int32_t rows_per_sequence, void* stream);

/* The newest rows of each sequence of the range as the cache holds them, into device memory: f32
 * [n_sequences * rows_per_sequence, kv_heads * head_dim] each. */
int32_t kv_cache_newest(kv_cache_t* cache, int32_t first_sequence, int32_t n_sequences, int32_t rows_per_sequence, float* keys,
                        float* values, void* stream);

/* Read-only views for tests and for handing a cache back: keys / values of one sequence,
 * [len, kv_heads * head_dim] as f32, into host memory. */
int32_t kv_cache_read(kv_cache_t* cache, int32_t sequence, float* keys_host, float* values_host, void* stream);

#ifdef __cplusplus
}
#endif
#endif

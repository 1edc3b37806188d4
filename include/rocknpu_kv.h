/*
 * rocknpu_kv.h — the 8-bit key/value cache and the attention that reads it, on
 * device buffers: what runs between a layer's q/k/v projections and its output
 * projection.
 *
 * No counterpart in the reference's accelerated path: its ggml plugin leaves
 * attention to the host (crates/rocknpu-llm/src/lib.rs:202 is its plain f32
 * form).
 *
 * Every pointer inside the structures is a DEVICE pointer, the structures
 * themselves are host memory read during the call; `stream` is a hipStream_t.
 * Calls validate what the host can see, enqueue and return without
 * synchronising or allocating. Status codes are those of rocknpu.h (0 ok, -1
 * invalid argument, -3 launch failure). What only the device can see (lengths,
 * page numbers) is checked by the kernels: nothing outside the buffers is read
 * or written whatever it holds. A block whose page number is outside
 * [0, n_pages) or whose place is outside the table is skipped by append and reads
 * as zeros. In attention, a page number outside [0, n_pages) or a scale that is
 * negative or not finite gives NaN in the rows that see the block, and in no other.
 * Any other scale counts as it is, zero too.
 *
 * The cache. A page holds one block of 32 tokens of one kv head: 32 * head_dim
 * int8 codes of keys, then as many of values, and in `scales` one f32 for its
 * keys and one for its values; a value is code * scale. head_dim is 64, 128,
 * 192 or 256. Within a page:
 *   keys    [head_dim / 64][token 0..31][64 dims]
 *   values  [head_dim / 32][dim bits 3-0][token bits 3-2][dim bit 4][token bit 4][token bits 1-0]
 * so that a wave's lanes load 16 bytes each, in one run, in the order in which
 * the matrix instructions take them.
 *
 * table[b][h][i] is the page of the i-th block that sequence b and kv head h
 * hold, in order of position, starts[b][h][i] the position of that block's
 * first token (a multiple of 32). Entries past the blocks in use name the pages
 * that the sequence's next blocks take. dropped[b] counts the blocks that a
 * sequence has lost to eviction, the same for all its heads: with t tokens seen
 * so far it holds ceil(t / 32) - dropped[b] blocks, and its newest block is the
 * last. weights[b][h][i] accumulates the attention weight that block i got.
 *
 * A step adds rows cu[b] .. cu[b + 1] - 1 of its tensors to sequence b, which
 * had past[b] tokens before it; row cu[b] + i is the token at position
 * past[b] + i. All layers of a model share past, cu and dropped.
 */
#ifndef ROCKNPU_KV_H
#define ROCKNPU_KV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ROCKNPU_KV_F32 0
#define ROCKNPU_KV_F16 1
#define ROCKNPU_KV_BF16 2

typedef struct rocknpu_kv_cache {
    uint8_t * pages;         /* [n_pages][64 * head_dim], 16-byte aligned */
    float * scales;          /* [n_pages][2]: keys, values; 8-byte aligned */
    const int32_t * table;   /* [batch][kv_heads][max_blocks] */
    int32_t * starts;        /* [batch][kv_heads][max_blocks] */
    const int32_t * dropped; /* [batch] */
    float * weights;         /* [batch][kv_heads][max_blocks], or NULL */
    int64_t n_pages;
    int32_t batch;           /* at most 4095 */
    int32_t kv_heads;        /* at most 65535 */
    int32_t head_dim;
    int32_t max_blocks;      /* at most 2^26 - 1 */
} rocknpu_kv_cache;

/* Quantises a step's key and value rows (type ROCKNPU_KV_*, [rows][kv_heads]
 * [head_dim], strides in elements, the last dimension contiguous) into their
 * blocks. max_new bounds the rows of any one sequence (above `rows` it is
 * `rows`). A block's scale is the largest of amax / 127 over the new values, the
 * scale it had if it held tokens before, and 2^-100; codes are rint(x * (1 / scale)), codes that the block held
 * before become rint(code * (old scale / scale)) when the scale grows. A new
 * value that is not finite, or an old scale that is negative or not finite, makes
 * the block's scale NaN and its codes zero, and NaN it stays until the block is
 * started anew. The first token of a block sets
 * its entry of `starts` and clears its entry of `weights` (if not NULL). Past
 * tokens must not share a partly filled block with another sequence. */
int rocknpu_hip_kv_append(const rocknpu_kv_cache * cache, uint32_t type, const void * k, int64_t k_row,
                          int64_t k_head, const void * v, int64_t v_row, int64_t v_head, size_t rows,
                          const int32_t * past, const int32_t * cu, size_t max_new, void * stream);

/* The values that the cache stands for: keys and values at positions first[b] ..
 * first[b] + count - 1 of every sequence into k and v, each contiguous
 * [batch][count][kv_heads][head_dim] of `type` (16-byte aligned); zeros for
 * positions at or past tokens[b] and for evicted blocks. */
int rocknpu_hip_kv_read(const rocknpu_kv_cache * cache, const int32_t * first, const int32_t * tokens, size_t count,
                        uint32_t type, void * k, void * v, void * stream);

typedef struct rocknpu_kv_attention_args {
    const void * q;          /* [rows][heads][head_dim] of `type`, strides in elements, last dimension contiguous */
    void * out;              /* the same shape and type, strides its own, without overlap */
    const int32_t * past;    /* [batch] */
    const int32_t * cu;      /* [batch + 1] */
    const int32_t * prefix;  /* [batch], or NULL */
    const float * slopes;    /* [heads], or NULL */
    float * weights_out;     /* [batch][kv_heads][max_blocks], or NULL; may be cache->weights itself */
    int64_t q_row, q_head, out_row, out_head;
    int64_t rows;
    int64_t max_new;         /* bounds the rows of any one sequence; above `rows` it is `rows` */
    int64_t max_tokens;      /* what past + rows are expected to reach: sizes the work split, not the result; 0: unknown */
    uint32_t type;
    int32_t heads;           /* a multiple of kv_heads; head h reads kv head h / (heads / kv_heads) */
    int32_t causal;
    int32_t window;          /* 0: none */
    float scale;
    float softcap;           /* 0: none */
} rocknpu_kv_attention_args;

/* Attention of a step's query rows over the cache (the step's keys and values
 * appended before). For the row at position p and a held key at position s:
 * x = scale * q.k; with softcap, x = softcap * tanh(x / softcap); with slopes,
 * x += slopes[head] * (s - p). The row sees s if s <= p (causal) and s > p -
 * window (window), or if s < prefix[b]; without causal it sees all keys (window
 * and prefix must then be absent). out = sum(exp(x) v) / sum(exp(x)) over what it
 * sees, and 0 where it sees nothing. Scores, the running maximum and sum and the
 * products' sums are f32. The codes enter the matrix instructions exactly, q as
 * f16 for f16 and bf16 calls and as a pair of f16 (to a unit of f32's last place,
 * or 2^-38 of the row's largest) for f32 calls (each row scaled by a power of two
 * first), the weights rounded to 17 bits for f16 and bf16 calls and 24 for f32
 * calls, over f32's range.
 * With weights_out, also weights_out = cache->weights + the weight that each
 * block got from all rows and the kv head's heads (entries past the blocks in
 * use are copied); at most 256 rows times heads per kv head.
 * The workspace (rocknpu_hip_kv_attention_workspace bytes, 256-byte aligned,
 * any contents) is free again when the call's kernels are done. What a call
 * computes may be summed in another order at another max_tokens or on another
 * number of compute units; the same call gives the same bits. */
int rocknpu_hip_kv_attention(const rocknpu_kv_cache * cache, const rocknpu_kv_attention_args * args, void * workspace,
                             size_t workspace_bytes, void * stream);

/* Bytes of workspace for such a call on a GPU of `cus` compute units (cus <= 0:
 * the current device's); 0 for none. Host code only. */
int rocknpu_hip_kv_attention_workspace(const rocknpu_kv_cache * cache, const rocknpu_kv_attention_args * args, int cus,
                                       size_t * bytes);

/* How such a call is shared out over workgroups where the rows of sequence b may
 * see blocks[b] blocks (0: it has no rows): parts[b] of them take sequence b, each
 * a part of its blocks, per kv head and tile of rows. All parts together are at
 * most `slots`, what the launch holds. blocks and parts are HOST arrays of batch
 * entries; host code only, `cus` as above. */
int rocknpu_hip_kv_attention_parts(const rocknpu_kv_cache * cache, const rocknpu_kv_attention_args * args, int cus,
                                   const int32_t * blocks, int32_t * parts, int64_t * slots);

typedef struct rocknpu_kv_evict_args {
    const int32_t * table;   /* [batch][kv_heads][max_blocks], as in the cache */
    const int32_t * starts;
    const float * weights;
    const int32_t * tokens;  /* [batch]: tokens seen so far */
    const int32_t * dropped; /* [batch] */
    int32_t * table_out;     /* the outputs' shapes are the inputs'; each may be its input, or overlap nothing */
    int32_t * starts_out;
    float * weights_out;
    int32_t * dropped_out;   /* [batch]; not `dropped` itself, which every head's workgroup reads */
    int32_t batch;
    int32_t kv_heads;
    int32_t max_blocks;      /* at most 16384 */
    int32_t budget;          /* blocks a sequence may hold */
    int32_t sinks;           /* its first blocks, always kept */
    int32_t recent;          /* its last blocks, always kept, at least 1; sinks + recent <= budget */
} rocknpu_kv_evict_args;

/* Where a sequence holds n > budget blocks, each head keeps its first `sinks`,
 * its last `recent` and, of the others, the budget - sinks - recent of greatest
 * weight (equal weights: the lowest place; NaN ranks lowest). Its entries of
 * table, starts and weights become the kept ones in order, then the evicted ones
 * in order (their pages are the next to be reused: pages that another sequence
 * shares have to be replaced there before the next append), then the rest as they
 * were; dropped_out = dropped + n - budget. Other sequences are copied. */
int rocknpu_hip_kv_evict(const rocknpu_kv_evict_args * args, void * stream);

#ifdef __cplusplus
}
#endif

#endif

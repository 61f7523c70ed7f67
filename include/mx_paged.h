/*
 * mx_paged.h — C ABI of the paged key/value cache: keys and values of many sequences in fixed-size pages of one pool,
 * lengths and page tables in device memory, so that a step captured in a HIP graph replays while its sequences grow.
 * Three calls serve a decoder's layer: mx_paged_store writes a step's new keys and values, mx_paged_decode attends a few
 * new rows of each sequence, mx_paged_prefill attends packed prompts. Each has a form for pages in 8 bits, and the decode one for
 * sequences that share their first keys.
 *
 * The reference has no paged cache: it keeps one contiguous cache per sequence (metal_llama_decoder.mm:664), which
 * mx_attn.h serves. The arithmetic is that of rope_store (src/backend/metal/llama_kernels.h:520-545) and of the attention
 * kernels (llama_kernels.h:552-769, 856-929).
 *
 * The cache. Key `pos` of sequence b lies in page table[b * table_stride + pos / page_size], at row pos % page_size; element d
 * of kv head g of that row is at page * page_stride + row * kv_stride + g * head_stride + d of the pool, for the keys and the
 * values alike. Any order of heads and rows within a page is a choice of the two strides. Sequences may share pages. Rows
 * that hold no key (behind a sequence's end, or in pages of no sequence) are never used, whatever they hold.
 *
 * Arithmetic of the attention calls. Scores, running maxima and sums, accumulators and joins are f32. The probabilities are
 * rounded to the pages' type for their product with the values, as the matrix cores take both operands in one type: half a step
 * of that type on each key's weight, with row_dtype MX_ATTN_F32 too, whose rows are only stored wider. The output is rounded once.
 * A probability that rounds to 0 (in f16 below 2^-25 of the largest) makes NaN of an infinite value at its key. Prompts, and the
 * prefixes of mx_paged_decode_shared, take scores below 2^27 in magnitude: from about 2^30 on (f16; 2^31 in bf16) a row is NaN. The
 * decodes, and a sequence's own keys, take what f32 holds.
 *
 * Device metadata cannot be checked by the host, and no entry of it makes a call read or write outside the pool:
 *   - kv_len outside [0, max_pages * page_size] makes that sequence's outputs NaN, a page outside [0, n_pages) the rows that
 *     attend it (and rows of that sequence that are computed with them); mx_paged_store leaves out the keys and values of a row
 *     that such a page or length would take;
 *   - query rows that see no key (kv_len 0, or rows of a causal call at positions below 0) give zeros and an lse of -inf;
 *   - cu_q entries are clamped to [0, n_rows] and have to ascend; what ranges that run backwards or overlap compute is undefined.
 *
 * Pages in 8 bits. The calls named _e4m3 keep each row of a kv head as head_dim codes of the 8-bit float e4m3 (no infinities,
 * largest 448) and one scale byte e, and the row stands for code x 2^(e - 127): half the memory of 16-bit pages and half the
 * bytes of a decode, at half a step of 2^-4 on each element. The scale is a power of two: quantising and expanding round once and
 * not twice, and a row's values do not depend on how a quotient is rounded. desc->dtype is then the type of the query rows, to which
 * codes are expanded for the matrix cores: exact in bf16, and in f16 as a cache of f16 values would hold them (products past 65504
 * are infinite, below 2^-14 they lose digits). A NaN code, or scale byte 255, stands for NaN.
 *
 * Errors, streams and threading as mx_attn.h (the same codes and mx_attn_last_error()).
 */
#ifndef MX_PAGED_H
#define MX_PAGED_H

#include "mx_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MX_PAGED_MAX_AXES 4

typedef struct mx_paged_desc {
    int32_t n_head;       /* query heads */
    int32_t n_head_kv;    /* key/value heads; n_head % n_head_kv == 0 */
    int32_t head_dim;     /* 64, 128 or 256 */
    int32_t dtype;        /* MX_ATTN_F16 or MX_ATTN_BF16: of the pages and of the query rows */
    int32_t row_dtype;    /* mx_paged_store: of the q|k|v rows (any of the three types); attention: of the output rows, dtype or
                             MX_ATTN_F32 */
    int32_t n_seq;        /* sequences, 0 .. 65535 (0: nothing to do) */
    int32_t n_rows;       /* rows of q (or q|k|v) and of the output; without cu_q every sequence has n_rows / n_seq of them */
    int32_t causal;       /* attention: 1: row t of a sequence's n rows sees keys 0 .. kv_len - n + t; 0: all kv_len keys */
    int32_t page_size;    /* keys per page: a power of two, 16 .. 65536 */
    int32_t n_pages;      /* pages in the pool */
    int32_t max_pages;    /* entries per sequence of the page table */
    int32_t max_q;        /* mx_paged_prefill: the most rows of a sequence, 0: unknown. A hint for the plan, as is ... */
    int32_t max_kv_len;   /* ... the most keys of a sequence, 0: unknown (max_pages * page_size) */
    int32_t reserved;     /* must be 0 */
    int64_t page_stride;  /* elements between pages, rows of a page and heads of a row: multiples of 8 (any with one page or head) */
    int64_t kv_stride;
    int64_t head_stride;
    int64_t table_stride; /* entries between sequences of the page table (>= max_pages) */
    int64_t row_stride;   /* elements between rows of q (>= n_head * head_dim) or q|k|v (>= (n_head + 2 n_head_kv) head_dim) */
    int64_t out_stride;   /* elements between output rows (>= n_head * head_dim); for mx_paged_store those of q_out */
    float scale;          /* attention: score scale, finite; 0 is valid (uniform attention) */
} mx_paged_desc;

/*
 * The scales of pages in 8 bits: that of row `row` of page `page`, kv head g is the byte at page * page_stride + g * head_stride +
 * row (rows of a page lie in a row) of k for the keys, v for the values. The pools' strides in mx_paged_desc count codes, and
 * are multiples of 16 there.
 */
typedef struct mx_paged_scales {
    uint8_t * k;          /* device, 16-byte aligned; written by mx_paged_store_e4m3 */
    uint8_t * v;
    int64_t page_stride;  /* bytes between pages and heads: multiples of 16 (any with one page or head) */
    int64_t head_stride;
    int32_t reserved;     /* must be 0 */
} mx_paged_scales;

/*
 * Rotary embedding. The head_dim / 2 pairs of a head are dealt to 1 .. 4 position axes in order, axis_pairs[a] pairs to axis a,
 * and pair i turns by positions[axis of i] * f(i). One axis is the ordinary embedding; several place image patches or video
 * frames (time, height, width).
 */
typedef struct mx_paged_rope {
    int32_t mode;         /* as mx_attn_rope: 0 adjacent pairs (2i, 2i + 1); 1 split halves (i, i + head_dim / 2); 2 none */
    int32_t n_axes;       /* 1 .. MX_PAGED_MAX_AXES */
    int32_t axis_pairs[MX_PAGED_MAX_AXES]; /* pairs per axis, each >= 1, together head_dim / 2 */
    int32_t axis_restart; /* 0: f(i) = base^(-2i / head_dim), one ladder over the head; 1: f(i) = base^(-j / axis_pairs[a]) for
                             the j-th pair of axis a, a ladder for each axis */
    int32_t reserved;     /* must be 0 */
    double base;          /* >= 1; 64 bits, as are the angles: at far positions 32 lose them */
} mx_paged_rope;

/*
 * The append of a step's new tokens: row r of the q|k|v rows (n_head query heads, n_head_kv key heads, n_head_kv value heads,
 * unrotated) is token t of the n new tokens of its sequence, at cache position kv_len - n + t. Its rotated query goes to
 * q_out, its rotated key and its value into the sequence's page, each rounded once to dtype. Replaces rope_store for a paged
 * cache.
 *
 *   qkv        device, [n_rows][row_stride] of row_dtype
 *   positions  device int32, [n_axes][n_rows]: the rotary positions; NULL (one axis only): the cache positions
 *   k, v       device, the pools, written
 *   table      device int32, [n_seq][table_stride]
 *   kv_len     device int32, [n_seq]: keys of each sequence INCLUDING the new ones
 *   cu_q       device int32, [n_seq + 1]: rows cu_q[b] .. cu_q[b + 1] - 1 are sequence b's, rows from cu_q[n_seq] on are left as
 *              they were; NULL: n_rows / n_seq rows each
 *   q_out      device, [n_rows][out_stride] of dtype, or NULL: queries are not wanted
 *
 * Two rows must not be given the same cache position of the same page. q_out must not overlap qkv.
 */
MX_ATTN_API int32_t mx_paged_store(const mx_paged_desc * desc, const mx_paged_rope * rope, const void * qkv,
                                   const int32_t * positions, void * k, void * v, const int32_t * table,
                                   const int32_t * kv_len, const int32_t * cu_q, void * q_out, mx_attn_stream stream);

/*
 * mx_paged_store into pages in 8 bits. Keys are rotated in 64 bits. The scale of a row is 2^e with e the least (from -127 on) for which
 * its largest finite magnitude is at most 448 x 2^e; each element is divided by it, which is exact, and rounded to nearest even. A
 * row of zeros has scale byte 0. An infinity or NaN becomes a NaN code, and leaves the scale to the others. The queries are rounded
 * to desc->dtype.
 */
MX_ATTN_API int32_t mx_paged_store_e4m3(const mx_paged_desc * desc, const mx_paged_rope * rope, const mx_paged_scales * scales,
                                        const void * qkv, const int32_t * positions, void * k, void * v, const int32_t * table,
                                        const int32_t * kv_len, const int32_t * cu_q, void * q_out, mx_attn_stream stream);

/*
 * Attention of n_rows / n_seq new rows of each sequence (one: a decode step; a few: drafted tokens) over its pages. The work is
 * cut over the sequences' lengths on the device, read by each call (and each replay of a captured one).
 *
 *   q          device, [n_rows][row_stride] of dtype, rotated; rows of sequence b start at b * n_rows / n_seq
 *   k, v       device, the pools
 *   out        device, [n_rows][out_stride] of row_dtype; must not overlap q
 *   lse        device f32, [n_rows][n_head], natural-log log-sum-exp of the scaled scores, or NULL
 *   workspace  device, 256-byte aligned, at least mx_paged_decode_workspace_bytes(desc) bytes, zeroed once by
 *              mx_attn_decode_workspace_init; every call leaves its counters at zero, and one workspace may serve this call,
 *              mx_paged_prefill and the calls of mx_attn.h that keep such counters (mx_attn_decode, _decode_f32, _decode_rope,
 *              _prefill_ws and _prefill_rope_ws), but not mx_self_attention or mx_linear, which write their rows where the
 *              counters lie. Calls that share it (captured ones too) must be ordered. NULL is allowed when the size needed
 *              is 0.
 */
MX_ATTN_API int32_t mx_paged_decode(const mx_paged_desc * desc, const void * q, const void * k, const void * v,
                                    const int32_t * table, const int32_t * kv_len, void * out, float * lse, void * workspace,
                                    size_t ws_bytes, mx_attn_stream stream);

/* mx_paged_decode over pages in 8 bits, with the same workspace. */
MX_ATTN_API int32_t mx_paged_decode_e4m3(const mx_paged_desc * desc, const mx_paged_scales * scales, const void * q, const void * k,
                                         const void * v, const int32_t * table, const int32_t * kv_len, void * out, float * lse,
                                         void * workspace, size_t ws_bytes, mx_attn_stream stream);

/* Workspace bytes mx_paged_decode needs for desc (the strides and pools do not matter). 0 and the last error set for an
 * invalid descriptor. */
MX_ATTN_API size_t mx_paged_decode_workspace_bytes(const mx_paged_desc * desc);

/*
 * Sequences whose first keys are the same: a batch of answers to one prompt, of users behind one system prompt, of questions about one
 * document. The sequences come in n_groups groups, one behind the other, each with a prefix that its sequences share; sequences
 * that no group has share nothing.
 */
typedef struct mx_paged_prefix {
    int32_t n_groups;           /* 0 .. 65535 (0: nothing is shared); groups may be empty */
    int32_t reserved;           /* must be 0 */
    const int32_t * cu_seq;     /* device, [n_groups + 1]: sequences cu_seq[g] .. cu_seq[g + 1] - 1 are group g's; ascending */
    const int32_t * prefix_len; /* device, [n_groups]: the keys that the sequences of a group have in common, from key 0 on; any
                                   number of them, whole pages or not */
} mx_paged_prefix;

/*
 * mx_paged_decode of sequences that share prefixes: the results of mx_paged_decode within its rounding, while each shared key is read
 * once for all rows of its group instead of once a sequence. Two launches: one for the partials of the prefixes, of all query rows of a
 * group on the matrix cores together, and of each sequence's own keys; one that joins them.
 *
 * The keys of a prefix are found through the page table of its group's first sequence, also where that one has 0 keys; the other sequences' entries for whole
 * pages of it are not read, and rows of it in a page that holds keys of a sequence's own (where the prefix ends within a page) are
 * never used. kv_len counts the prefix's keys too. Every row has to see the whole prefix, also where a sequence is alone in its group: one
 * with fewer keys than the prefix (causal: than the prefix and all but one of its new rows), but not 0, or with a prefix_len outside
 * [0, max_pages * page_size], gets NaN; one of 0 keys gets zeros, and takes nothing from its group; one that ends with its prefix has no
 * keys of its own. cu_seq entries are clamped to [0, n_seq]; what ranges that run backwards or overlap compute is undefined, within the
 * buffers.
 *
 *   scales      of pages in 8 bits, or NULL: pages of dtype
 *   workspace   as mx_paged_decode's, at least mx_paged_decode_shared_workspace_bytes(desc, n_groups) bytes, never NULL where there
 *               is work to do. Nothing is kept in it between calls.
 *
 * desc->max_kv_len counts the keys of a sequence behind its prefix here (0: unknown); a sequence of no group has no prefix, and all its
 * keys count. n_rows * n_head at most 2^26. Every workgroup reads all groups: up to a hundred cost little, thousands milliseconds.
 */
MX_ATTN_API int32_t mx_paged_decode_shared(const mx_paged_desc * desc, const mx_paged_scales * scales, const mx_paged_prefix * prefix,
                                           const void * q, const void * k, const void * v, const int32_t * table,
                                           const int32_t * kv_len, void * out, float * lse, void * workspace, size_t ws_bytes,
                                           mx_attn_stream stream);

/* Workspace bytes mx_paged_decode_shared needs for desc and so many groups, or fewer; 0 and the last error set for an invalid
 * descriptor. */
MX_ATTN_API size_t mx_paged_decode_shared_workspace_bytes(const mx_paged_desc * desc, int32_t n_groups);

/*
 * Attention of packed prompts: rows cu_q[b] .. cu_q[b + 1] - 1 are the last rows of sequence b, whose pages hold its keys
 * already (mx_paged_store), those of an earlier chunk or a shared prefix among them. Rows from cu_q[n_seq] on are left as
 * they were. Arguments as mx_paged_decode. With a workspace (mx_paged_prefill_workspace_bytes(desc) bytes, the rules of
 * mx_paged_decode's) the work is cut into equal ranges over the chip, which split a tile of rows between workgroups; NULL: no
 * tile is split.
 */
MX_ATTN_API int32_t mx_paged_prefill(const mx_paged_desc * desc, const void * q, const void * k, const void * v,
                                     const int32_t * table, const int32_t * kv_len, const int32_t * cu_q, void * out, float * lse,
                                     void * workspace, size_t ws_bytes, mx_attn_stream stream);

/* mx_paged_prefill over pages in 8 bits, with the same workspace. */
MX_ATTN_API int32_t mx_paged_prefill_e4m3(const mx_paged_desc * desc, const mx_paged_scales * scales, const void * q, const void * k,
                                          const void * v, const int32_t * table, const int32_t * kv_len, const int32_t * cu_q,
                                          void * out, float * lse, void * workspace, size_t ws_bytes, mx_attn_stream stream);

/* Workspace bytes mx_paged_prefill needs for desc; 0 and the last error set for an invalid descriptor. */
MX_ATTN_API size_t mx_paged_prefill_workspace_bytes(const mx_paged_desc * desc);

#ifdef __cplusplus
}
#endif

#endif /* MX_PAGED_H */

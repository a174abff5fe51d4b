/* qwen3/cache_args.h - the arguments of the kernels of a cache that may be kept in 8 bits and of steps with drafted tokens (kernels.h).
   They are many, and are handed over as a structure in host memory, which the call reads before it returns: a host program fills one once and
   changes what changes.  All pointers are device pointers; `stream` is a cudaStream_t.
   Pages: keys and values [pages, kv heads, 64, d], of the compute type (k_scales, v_scales null) or as e4m3 codes with a scale of a power of two
   a row, [pages, kv heads, 64] bytes (exponent + 127). */
#pragma once

#include <stdint.h>

/* q3_cache_append_*: per-head norm (weights may be null) and rotation (tables may be null) of new rows of q and k, and the write of k and v */
typedef struct q3_cache_append_args {
    const void *qkv;                                  /* [tokens, row]: nq query heads, nkv keys, nkv values, of d each */
    void *q_out, *k_pages, *v_pages, *k_scales, *v_scales;
    const void *q_norm, *k_norm, *cos_tab, *sin_tab;  /* float32 [d]; [positions, rotary_dim / 2] */
    const void *token_seq, *token_pos, *token_place;  /* int32 [tokens]: sequence, position of the rotation, place in the sequence's cache */
    const void *page_table;                           /* int32 [sequences, pages_per_seq] */
    void *stream;
    int64_t n_pages, n_tokens, row;
    double eps;
    int pages_per_seq, nq, nkv, d, rotary_dim, norm_once;   /* norm_once: one rounding, at the end */
} q3_cache_append_args;

/* q3_cache_read_*: pages of codes as pages of values, page j of sequence s to number s * out_pages + j, as far as it holds some of the first
   seq_end[s] rows; rows behind them in a page become zeros */
typedef struct q3_cache_read_args {
    const void *k_pages, *v_pages, *k_scales, *v_scales, *page_table, *seq_end;
    void *k_out, *v_out, *stream;
    int64_t n_pages;
    int pages_per_seq, n_seqs, out_pages, nkv, d, reserved;
} q3_cache_read_args;

/* q3_cache_keep: in each of n_areas areas [pages, kv heads, 64, row_bytes] (scales: a byte a row, or null) row seq_pos0 + path[i] moves to
   seq_pos0 + i; a sequence's path ascends, -1 ends it */
typedef struct q3_cache_keep_args {
    void *store, *scales;
    const void *page_table, *seq_pos0, *path;
    void *stream;
    int64_t n_areas, n_pages;
    int nkv, row_bytes, pages_per_seq, path_len, n_seqs, reserved;
} q3_cache_keep_args;

/* q3_attention_tree_*: the new tokens of every sequence over the cache's pages, which hold their keys and values too, from place seq_pos0 on.  A
   token sees the seq_pos0 earlier rows and, of the new ones, number n where bit n % 64 of tree[token][n / 64] is set (tree null: those up to
   itself); one that sees nothing gets zeros */
typedef struct q3_attention_tree_args {
    const void *q, *k_pages, *v_pages, *k_scales, *v_scales;
    void *out, *parts, *counters;                     /* parts: see q3_attention_tree_*_parts; counters: int32, zero when made and left zero */
    const void *seq_start, *seq_pos0, *page_table, *tree;
    void *status, *stream;
    int64_t n_pages, n_tokens;
    double scale;
    int pages_per_seq, n_seqs, max_new, nq, nkv, d, words, reserved;   /* max_new: the most tokens that a sequence brings; words: of a mask */
} q3_attention_tree_args;

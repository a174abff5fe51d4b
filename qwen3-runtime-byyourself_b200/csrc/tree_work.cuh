// How the attention of a step over the paged cache is shared out over the blocks of a launch, and which of a sequence's new keys a token sees.
//
// The work is a list of items - (sequence, kv head, tile of new tokens) - of as many pages as the sequence has.  The pages of all
// items in a row are cut into ranges of equal length, one a block, wherever they fall: contexts of unequal length take as long as equal ones of
// the same total, and a block has at most a part of an item, some whole ones, and another part.  Parts of an item are added up
// in their order by the block that comes last.  Which part of an item is whose, and so the order of a row's sums, hangs on the lengths of
// all sequences of the step and on nothing else.
#pragma once

#include "common.cuh"

struct TreeStep {
    const int *seq_start, *seq_pos0, *page_table;
    const unsigned long long* tree;                // [tokens, words], null: a token sees the new ones up to itself
    int words, pages_per_seq, n_seqs, nq, nkv;
    int64_t n_pages;
    int max_new;                                   // no sequence brings more tokens (those that one brings beyond are left out)
};

// A range of pages [begin, end) of one item.
struct TreePart {
    int seq, head, tile;                           // head: the kv head
    int begin, end, pages;                         // pages of the item in all
    int64_t item_begin;                            // the item's first page in the list of all
    int item;                                      // its number among the items
};

// `per_tile` new tokens make a tile; `least`: a block is not given fewer pages.
struct TreeShare {
    int64_t from, to, quota;                       // this block's range, and a block's length
};

__device__ __forceinline__ int tree_new(const TreeStep& a, int seq) { return min(a.seq_start[seq + 1] - a.seq_start[seq], a.max_new); }
__device__ __forceinline__ int tree_pages(const TreeStep& a, int seq) {
    const int n_new = tree_new(a, seq);
    return n_new <= 0 ? 0 : min((a.seq_pos0[seq] + n_new + Q3_PAGE_TOKENS - 1) / Q3_PAGE_TOKENS, a.pages_per_seq);
}
__device__ __forceinline__ int tree_tiles(const TreeStep& a, int seq, int per_tile) { return (max(tree_new(a, seq), 0) + per_tile - 1) / per_tile; }

// Called by one whole warp.
__device__ __forceinline__ TreeShare tree_share(const TreeStep& a, int per_tile, int least) {
    const int lane = threadIdx.x & 31;
    long long total = 0;
    for (int s = lane; s < a.n_seqs; s += 32) total += (long long)tree_pages(a, s) * tree_tiles(a, s, per_tile) * a.nkv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    TreeShare t;
    const long long even = (total + gridDim.x - 1) / (long long)gridDim.x;
    t.quota = even > least ? even : least;
    const long long from = (long long)blockIdx.x * t.quota;
    t.from = from < total ? from : total;
    t.to = t.from + t.quota < total ? t.from + t.quota : total;
    return t;
}

// The sequence in whose items page `at` of the list lies, with the list's and the items' count before it.  Called by one whole warp.
__device__ __forceinline__ void tree_find(const TreeStep& a, int per_tile, int64_t at, int& seq, int64_t& before, int& items_before) {
    const int lane = threadIdx.x & 31;
    long long run = 0;
    int items = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        const int n = s < a.n_seqs ? tree_tiles(a, s, per_tile) * a.nkv : 0;
        const long long pages = s < a.n_seqs ? (long long)tree_pages(a, s) * n : 0;
        long long sum = pages;
        int count = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, sum, o);
            const int c = __shfl_up_sync(0xffffffffu, count, o);
            if (lane >= o) { sum += v; count += c; }
        }
        const unsigned hit = __ballot_sync(0xffffffffu, run + sum > at);
        if (hit != 0) {
            const int first = __ffs(hit) - 1;
            seq = s0 + first;
            before = run + __shfl_sync(0xffffffffu, sum - pages, first);
            items_before = items + __shfl_sync(0xffffffffu, count - n, first);
            return;
        }
        run += __shfl_sync(0xffffffffu, sum, 31);
        items += __shfl_sync(0xffffffffu, count, 31);
    }
    seq = a.n_seqs;
    before = run;
    items_before = items;
}

// The part at page `at` of the list, given the sequence that holds it; moves on to the next sequence where it has to.
__device__ __forceinline__ TreePart tree_part(const TreeStep& a, int per_tile, int64_t at, int64_t to, int& seq, int64_t& before, int& items_before) {
    TreePart p;
    while (true) {
        const int pages = tree_pages(a, seq), tiles = tree_tiles(a, seq, per_tile), n = tiles * a.nkv;
        const int64_t in = at - before;
        if (in < (int64_t)pages * n) {
            const int i = (int)(in / pages);
            p.seq = seq;
            p.head = i / tiles;
            p.tile = i - p.head * tiles;
            p.pages = pages;
            p.begin = (int)(in - (int64_t)i * pages);
            p.item_begin = before + (int64_t)i * pages;
            p.end = to - p.item_begin < pages ? (int)(to - p.item_begin) : pages;
            p.item = items_before + i;
            return p;
        }
        before += (int64_t)pages * n;
        items_before += n;
        ++seq;
    }
}

// Bit i: the token sees key `key0 + i` of its sequence (i < 64), `own` being its number among the sequence's n_new new tokens.
__device__ __forceinline__ unsigned long long tree_seen(const unsigned long long* mask, int words, int pos0, int n_new, int own, int key0) {
    const int n0 = key0 - pos0;                    // the number of the new token at bit 0
    if (n0 <= -64) return ~0ull;
    unsigned long long m;
    int upto = n_new - n0;                         // bits from here on are keys behind the end
    if (mask == nullptr) {
        m = ~0ull;
        upto = min(upto, own + 1 - n0);
    } else if (n0 < 0) {
        m = mask[0] << -n0;
    } else {
        const int w = n0 >> 6, sh = n0 & 63;
        m = w < words ? mask[w] >> sh : 0ull;
        if (sh != 0 && w + 1 < words) m |= mask[w + 1] << (64 - sh);
    }
    if (upto <= 0) m = 0ull;
    else if (upto < 64) m &= (1ull << upto) - 1ull;
    if (n0 < 0) m |= (1ull << -n0) - 1ull;         // earlier tokens
    return m;
}

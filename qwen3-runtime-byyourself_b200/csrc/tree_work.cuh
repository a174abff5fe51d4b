// How the attention of a step over the paged cache is shared out over the blocks of a launch, and which of a sequence's new keys a token sees.
//
// The work is a list of items - (sequence, kv head, tile of rows; a row is a new token and a query head of the kv head's group) - of as
// many stretches of UNIT keys as the sequence has.  The stretches of all items in a row are cut into ranges of equal length, one a
// block, wherever they fall: contexts of unequal length take as long as equal ones of the same total, and a block has at most a part of an item, some whole
// ones, and another part.  Which part of an item is whose, and so the order of a row's sums, hangs on the lengths of all sequences of the step and on
// nothing else.
#pragma once

#include "common.cuh"

struct TreeStep {
    const int *seq_start, *seq_pos0, *page_table;
    const unsigned long long* tree;                // [tokens, words], null: a token sees the new ones up to itself
    int words, pages_per_seq, n_seqs, nq, nkv;
    int64_t n_pages;
    int max_new;                                   // no sequence brings more tokens (those that one brings beyond are left out)
};

// A range of stretches [begin, end) of one item.
struct TreePart {
    int seq, head, tile;                           // head: the kv head
    int begin, end, units;                         // units: the item's in all
    int64_t item_begin;                            // the item's first stretch in the list of all
    int item;                                      // its number among the items
};

// A block's range of the list, and the length of a range.
struct TreeShare {
    int64_t from, to, quota;
};

// Where a walk through the list is: a sequence, and the stretches and items before it.
struct TreePlace {
    int64_t before;
    int items_before, seq;
};

// UNIT: keys of a stretch; ROWS: rows of a tile.
template <int UNIT, int ROWS> struct TreeWork {
    static __device__ __forceinline__ int n_new(const TreeStep& a, int seq) { return min(a.seq_start[seq + 1] - a.seq_start[seq], a.max_new); }
    static __device__ __forceinline__ int units(const TreeStep& a, int seq) {
        const int n = n_new(a, seq);
        return n <= 0 ? 0 : (min(a.seq_pos0[seq] + n, a.pages_per_seq * Q3_PAGE_TOKENS) + UNIT - 1) / UNIT;
    }
    static __host__ __device__ __forceinline__ int tiles_of(int n_new, int group) { return n_new <= 0 ? 0 : (int)(((int64_t)n_new * group + ROWS - 1) / ROWS); }
    static __device__ __forceinline__ int tiles(const TreeStep& a, int seq) { return tiles_of(n_new(a, seq), a.nq / a.nkv); }

    // The range of block `block` of `blocks`, of at least `least` stretches.  Called by one whole warp.
    static __device__ __forceinline__ TreeShare share(const TreeStep& a, int least, int block, int blocks) {
        const int lane = threadIdx.x & 31;
        long long total = 0;
        for (int s = lane; s < a.n_seqs; s += 32) total += (long long)units(a, s) * tiles(a, s) * a.nkv;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const long long even = (total + blocks - 1) / (long long)blocks;
        TreeShare t;
        t.quota = even > least ? even : least;
        const long long from = (long long)block * t.quota;
        t.from = from < total ? from : total;
        t.to = t.from + t.quota < total ? t.from + t.quota : total;
        return t;
    }

    // The sequence in whose items stretch `at` lies.  Called by one whole warp.
    static __device__ __forceinline__ TreePlace find(const TreeStep& a, int64_t at) {
        const int lane = threadIdx.x & 31;
        long long run = 0;
        int items = 0;
        TreePlace p;
        for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
            const int s = s0 + lane;
            const int n = s < a.n_seqs ? tiles(a, s) * a.nkv : 0;
            const long long mine = s < a.n_seqs ? (long long)units(a, s) * n : 0;
            long long sum = mine;
            int count = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, sum, o);
                const int c = __shfl_up_sync(0xffffffffu, count, o);
                if (lane >= o) {
                    sum += v;
                    count += c;
                }
            }
            const unsigned hit = __ballot_sync(0xffffffffu, run + sum > at);
            if (hit != 0) {
                const int first = __ffs(hit) - 1;
                p.seq = s0 + first;
                p.before = run + __shfl_sync(0xffffffffu, sum - mine, first);
                p.items_before = items + __shfl_sync(0xffffffffu, count - n, first);
                return p;
            }
            run += __shfl_sync(0xffffffffu, sum, 31);
            items += __shfl_sync(0xffffffffu, count, 31);
        }
        p.seq = a.n_seqs;
        p.before = run;
        p.items_before = items;
        return p;
    }

    // The part of the range up to `to` that begins at stretch `at`, which lies in the list behind `place`; that moves on where it has to.
    static __device__ __forceinline__ TreePart part(const TreeStep& a, int64_t at, int64_t to, TreePlace& place) {
        TreePart p;
        while (true) {
            const int each = units(a, place.seq), per_head = tiles(a, place.seq), n = per_head * a.nkv;
            const int64_t in = at - place.before;
            if (in < (int64_t)each * n) {
                const int i = (int)(in / each);
                p.seq = place.seq;
                p.head = i / per_head;
                p.tile = i - p.head * per_head;
                p.units = each;
                p.begin = (int)(in - (int64_t)i * each);
                p.item_begin = place.before + (int64_t)i * each;
                p.end = to - p.item_begin < each ? (int)(to - p.item_begin) : each;
                p.item = place.items_before + i;
                return p;
            }
            place.before += (int64_t)each * n;
            place.items_before += n;
            ++place.seq;
        }
    }
};

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

// How the attention of a step over the paged cache is shared out over the blocks of a launch, and which of a sequence's new keys a token sees.
//
// The work is a list of items - (sequence, kv head, tile of rows; a row is a new token and a query head of the kv head's group) - of as
// many stretches of UNIT keys as the sequence has.  It is shared out in one of two ways, whatever the sequences' lengths:
//   pieces  every item is cut into equal pieces of at most `quota` stretches, and a block takes one piece.  `quota` is the best of four numbers between
//           the even share and one at which the pieces are certainly no more than the blocks, or that is longer by what a second part would cost a block;
//   ranges  the stretches of all items in a row are cut into ranges of equal length, one a block, wherever they fall: a block has at most a
//           part of an item, some whole ones and another part.  Taken where there are no such pieces.  In the row every item is longer by some stretches
//           before its first one, for the time that beginning and ending it takes: a block with five short items is not the last.
// Parts of an item are added up in their order.  Which part is whose, and so the order of a row's sums, hangs on the lengths of all sequences of the step
// and on nothing else.
#pragma once

#include "../include/qwen3/cache_args.h"
#include "common.cuh"

struct TreeStep {
    const int *seq_start, *seq_pos0, *page_table;
    const unsigned long long* tree;                // [tokens, words], null: a token sees the new ones up to itself
    int words, pages_per_seq, n_seqs, nq, nkv;
    int64_t n_pages;
    int max_new;                                   // no sequence brings more tokens (those that one brings beyond are left out)
};
static inline TreeStep tree_step(const q3_attention_tree_args& a) {
    return {(const int*)a.seq_start, (const int*)a.seq_pos0, (const int*)a.page_table, (const unsigned long long*)a.tree, a.words, a.pages_per_seq, a.n_seqs, a.nq,
            a.nkv, a.n_pages, a.max_new};
}
// What is wrong with the arguments of a tensor-core form (0: nothing).
static inline int tree_refused(const q3_attention_tree_args& a, int d) {
    if (a.nq <= 0 || a.nkv <= 0 || a.nq % a.nkv != 0 || a.d != d || a.n_pages <= 0 || a.pages_per_seq <= 0 ||
        (a.tree != nullptr && (a.words <= 0 || (int64_t)a.words * 64 < a.max_new)))
        return Q3_ERR_BAD_SIZE;
    for (const void* p : {a.q, a.k_pages, a.v_pages, a.k_scales, a.v_scales, (const void*)a.out, (const void*)a.parts})
        if (!aligned16(p)) return Q3_ERR_MISALIGNED;
    return 0;
}

// A range of stretches [begin, end) of one item.
struct TreePart {
    int seq, head, tile;                           // head: the kv head
    int begin, end, item;                          // item: its number among the items
    int parts, slot, slot0, first_block;           // of the item: how many; this one's place in the scratch, the first one's, and the first one's block
    int list_end;                                  // where the block's share goes on
    int t0, n_new, pos0;                           // of the sequence: its first token and how many of the step's, its earlier keys

    // The place of the item's part i in the scratch (a block has two: of the part that it begins with, and of the one that it ends with).
    __device__ __forceinline__ int slot_of(int i) const { return i == 0 ? slot0 : 2 * (first_block + i); }
};

// What of a sequence counts in the list: its items, in the order of their heads and tiles, of so many stretches each.  With LIGHT a stretch of a tile of at most
// half the rows (the last one of a head) costs half of another's: lengths are then counted in halves, those of light items rounded up to whole ones.
struct TreeItems {
    int units, tiles;                              // stretches of an item; twice the tiles of a head, and 1 if the last one is light
};

// What a block has: in the way of ranges stretches [from, to) of the list (none: from >= to), else one piece.
struct TreeShare {
    int from, to, quota;                           // quota: a range's length, or (`pieces`) the most stretches of a piece
    int pieces, pad;                               // 1: pieces; what an item is longer by, counted as lengths are (pieces: 0)
    int seq, before, items_before;                 // where `from` (a piece: the block's number) lies: its sequence, the stretches (pieces) and items before it
    TreeItems items;                               // the sequence's
};

// UNIT: keys of a stretch; ROWS: rows of a tile.
template <int UNIT, int ROWS, bool LIGHT> struct TreeWork {
    static constexpr int COUNT = LIGHT ? 2 : 1;    // of a stretch
    static __device__ __forceinline__ int n_new(const TreeStep& a, int seq) { return max(0, min(a.seq_start[seq + 1] - a.seq_start[seq], a.max_new)); }
    static __host__ __device__ __forceinline__ int tiles_of(int n_new, int group) { return (int)(((int64_t)n_new * group + ROWS - 1) / ROWS); }
    static __device__ __forceinline__ TreeItems items_of(const TreeStep& a, int seq) {
        const int n = n_new(a, seq), group = a.nq / a.nkv;
        const int units = n == 0 ? 0 : (min(a.seq_pos0[seq] + n, a.pages_per_seq * Q3_PAGE_TOKENS) + UNIT - 1) / UNIT, tiles = units > 0 ? tiles_of(n, group) : 0;
        return {units, 2 * tiles + (LIGHT && tiles > 0 && n * group - (tiles - 1) * ROWS <= ROWS / 2 ? 1 : 0)};
    }
    // Tiles of a head, whether the last one is light (0 or 1), the lengths of the others and of a light one.
    static __device__ __forceinline__ int per_head(const TreeItems& i) { return i.tiles >> 1; }
    static __device__ __forceinline__ int light(const TreeItems& i) { return i.tiles & 1; }
    static __device__ __forceinline__ int full(const TreeItems& i) { return i.units * COUNT; }
    static __device__ __forceinline__ int lighter(const TreeItems& i) { return (i.units + 1) & ~1; }
    static __device__ __forceinline__ int cut(int length, int quota) { return (int)((unsigned)(length + quota - 1) / (unsigned)quota); }
    // A head's length, or its pieces of up to `quota`.
    static __device__ __forceinline__ int of_head(const TreeItems& i, int pad) {
        return (per_head(i) - light(i)) * full(i) + light(i) * lighter(i) + per_head(i) * pad;
    }
    static __device__ __forceinline__ int pieces_of_head(const TreeItems& i, int quota) {
        return i.units == 0 ? 0 : (per_head(i) - light(i)) * cut(full(i), quota) + (light(i) ? cut(lighter(i), quota) : 0);
    }

    // The most items and counted stretches that a step can have (the latter have to stay below 2^30).
    static __host__ int64_t most_items(const TreeStep& a) { return (int64_t)a.n_seqs * a.nkv * tiles_of(a.max_new, a.nq / a.nkv); }
    static __host__ int64_t most_units(const TreeStep& a, int spare) {
        return COUNT * most_items(a) * (((int64_t)a.pages_per_seq * Q3_PAGE_TOKENS + UNIT - 1) / UNIT + spare);
    }

    // What block `block` of `blocks` has.  Called by one whole warp; `least`: a block is not given fewer stretches (unless an item has no more), nor so few
    // that adding up an item's parts would take longer than it saves: for an item of u stretches in pieces of q, where a part is added up in `join` times the
    // time of a stretch, q + join u / q is least at q = sqrt(join u); `whole`: where no item has more stretches, none is cut;
    // `spare`: so many stretches take about as long as beginning and ending a part: a piece may be longer than the even share by them, rather than that
    // blocks have several parts, and items count as longer by them.
    static __device__ TreeShare share(const TreeStep& a, int least, int whole, float join, int spare, int block, int blocks) {
        const int lane = threadIdx.x & 31;
        // of up to 64 sequences everything is read once
        const bool few = a.n_seqs <= 64;
        const TreeItems none = {0, 0}, mine = few && lane < a.n_seqs ? items_of(a, lane) : none, mine2 = few && lane + 32 < a.n_seqs ? items_of(a, lane + 32) : none;
        auto each = [&](auto f) {                                        // sum over the sequences, for a head
            int sum = 0;
            if (few) sum = f(mine) + f(mine2);
            else
                for (int s = lane; s < a.n_seqs; s += 32) sum += f(items_of(a, s));
            return __reduce_add_sync(0xffffffffu, sum) * a.nkv;
        };
        int longest = max(mine.units, mine2.units);
        if (!few)
            for (int s = lane; s < a.n_seqs; s += 32) longest = max(longest, items_of(a, s).units);
        longest = __reduce_max_sync(0xffffffffu, longest);
        least = max(least, longest <= whole ? longest : __float2int_rn(sqrtf(join * (float)longest)));
        TreeShare t;
        const int items = each([](const TreeItems& i) { return per_head(i); });
        int total = each([](const TreeItems& i) { return of_head(i, 0); });
        auto even_of = [&] { return (max(least * COUNT, (int)(((unsigned)total + blocks - 1) / (unsigned)blocks)) + COUNT - 1) & ~(COUNT - 1); };
        const int even = even_of();
        t.pieces = 0;
        if (items < blocks) {
            // with pieces of `safe` there are at most items + total / safe of them
            const int safe = max(even, (total + blocks - items - 1) / (blocks - items)), cap = even + spare * COUNT;
            // four numbers at once, eight lanes each
            const int quota = even + (min(safe, cap) - even) * (lane >> 3) / 3;
            int sum = 0;
            for (int s0 = 0; s0 < a.n_seqs; s0 += 8) {
                const int s = s0 + (lane & 7);
                TreeItems i = none;
                if (few) i = {__shfl_sync(0xffffffffu, s0 < 32 ? mine.units : mine2.units, s & 31), __shfl_sync(0xffffffffu, s0 < 32 ? mine.tiles : mine2.tiles, s & 31)};
                else if (s < a.n_seqs) i = items_of(a, s);
                sum += pieces_of_head(i, quota);
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const unsigned fits = __ballot_sync(0xffffffffu, sum * a.nkv <= blocks);
            if (fits != 0) {
                t.pieces = 1;
                t.quota = __shfl_sync(0xffffffffu, quota, __ffs(fits) - 1);
            }
        }
        t.pad = t.pieces ? 0 : spare * COUNT;
        if (!t.pieces) {
            total += items * t.pad;
            t.quota = even_of();
        }
        // where the block's range or piece begins
        const int at = t.pieces ? block : (int)min((int64_t)total, (int64_t)block * t.quota);
        t.from = at;
        t.to = t.pieces ? at + 1 : (int)min((int64_t)total, (int64_t)at + t.quota);
        int run = 0, passed = 0;
        for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
            const int s = s0 + lane;
            const TreeItems here = few ? (s0 == 0 ? mine : mine2) : s < a.n_seqs ? items_of(a, s) : none;
            const int own = a.nkv * (t.pieces ? pieces_of_head(here, t.quota) : of_head(here, t.pad)), count = a.nkv * per_head(here);
            int sum = own, counts = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o), c = __shfl_up_sync(0xffffffffu, counts, o);
                if (lane >= o) {
                    sum += v;
                    counts += c;
                }
            }
            const unsigned hit = __ballot_sync(0xffffffffu, run + sum > at);
            if (hit != 0) {
                const int first = __ffs(hit) - 1;
                t.seq = s0 + first;
                t.before = run + __shfl_sync(0xffffffffu, sum - own, first);
                t.items_before = passed + __shfl_sync(0xffffffffu, counts - count, first);
                t.items = {__shfl_sync(0xffffffffu, here.units, first), __shfl_sync(0xffffffffu, here.tiles, first)};
                return t;
            }
            run += __shfl_sync(0xffffffffu, sum, 31);
            passed += __shfl_sync(0xffffffffu, counts, 31);
        }
        t.from = t.to = 0;                                               // nothing for this block
        t.seq = t.before = t.items_before = 0;
        t.items = none;
        return t;
    }

    // The part at `at` (t.from, then what `next` says) of a block's share; `t` is moved on to the sequence that holds it.  The last part of a range may be
    // empty (begin == end): the range ends before the item's first stretch.
    static __device__ __forceinline__ TreePart part(const TreeStep& a, TreeShare& t, int at, int block) {
        TreePart p;
        while (true) {
            const TreeItems& i = t.items;
            const int head = t.pieces ? pieces_of_head(i, t.quota) : of_head(i, t.pad), in = at - t.before;
            if (in < head * a.nkv) {
                p.seq = t.seq;
                p.t0 = a.seq_start[t.seq];
                p.n_new = n_new(a, t.seq);
                p.pos0 = a.seq_pos0[t.seq];
                p.head = (int)((unsigned)in / (unsigned)head);
                const int in_head = in - p.head * head, a_full = t.pieces ? cut(full(i), t.quota) : full(i) + t.pad;     // numbers that a tile that is not light has
                p.tile = min((int)((unsigned)in_head / (unsigned)a_full), per_head(i) - 1);
                const int off = in_head - p.tile * a_full, light_tile = light(i) && p.tile == per_head(i) - 1 ? 1 : 0;
                const int length = (light_tile ? lighter(i) : full(i)) + t.pad, count = light_tile ? 1 : COUNT;
                p.item = t.items_before + p.head * per_head(i) + p.tile;
                if (t.pieces) {
                    p.parts = cut(length, t.quota);
                    p.begin = (int)((unsigned)(off * i.units) / (unsigned)p.parts);
                    p.end = (int)((unsigned)((off + 1) * i.units) / (unsigned)p.parts);
                    p.first_block = block - off;
                    p.slot0 = 2 * p.first_block;
                    p.slot = 2 * block;
                    p.list_end = at + 1;
                } else {
                    const int item_begin = at - off, to = min(length, t.to - item_begin);
                    p.begin = max(0, off - t.pad) / count;               // (whole: ranges, items and their pads begin with whole stretches)
                    p.end = min(i.units, max(0, to - t.pad) / count);
                    p.first_block = (int)((unsigned)(item_begin + t.pad) / (unsigned)t.quota);
                    p.parts = (int)((unsigned)(item_begin + length - 1) / (unsigned)t.quota) - p.first_block + 1;
                    p.slot0 = 2 * p.first_block + (p.first_block * t.quota >= item_begin ? 0 : 1);
                    p.slot = 2 * block + (at == t.from ? 0 : 1);
                    p.list_end = item_begin + to;
                }
                return p;
            }
            t.before += head * a.nkv;
            t.items_before += per_head(i) * a.nkv;
            t.items = items_of(a, ++t.seq);
        }
    }
    static __device__ __forceinline__ int next(const TreePart& p) { return p.list_end; }
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

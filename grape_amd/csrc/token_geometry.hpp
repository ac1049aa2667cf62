// Which elements of a paged cache a call of the new tokens' kernels touches, and which calls are refused: the expressions that
// the kernels and their entry points use, free of HIP so that a host build can walk over them.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include <algorithm>
#include "../../include/grape_hip.h"

#ifndef GRAPE_HD
#ifdef __HIPCC__
#define GRAPE_HD __host__ __device__ __forceinline__
#else
#define GRAPE_HD inline
#endif
#endif

namespace grape {
namespace token {

// The positions lo <= t < hi that a sequence attends to.  False (and none) where its numbers do not fit the call.
GRAPE_HD bool live_span(int32_t len, int32_t first, uint32_t max_len, uint32_t table_stride, uint32_t page_size, uint32_t& lo, uint32_t& hi) {
    const bool ok = len >= 0 && first >= 0 && (uint32_t)len <= max_len && (uint64_t)len <= (uint64_t)table_stride * page_size;
    lo = ok ? (uint32_t)first : 0;
    hi = ok ? (uint32_t)len : 0;
    if (lo > hi) lo = hi;
    return ok;
}

// Offset of the first head of a page's token, or -1 where the page is outside the cache.
GRAPE_HD int64_t token_offset(const grape_wit_cache& c, int32_t page, uint32_t in_page) {
    if (page < 0 || (uint32_t)page >= c.pages) return -1;
    return page * c.page_stride + (int64_t)in_page * c.token_stride;
}

// Whether a token with this slot and position is written at all (0), is padding (1) or is out of range (2).
GRAPE_HD int append_kind(const grape_wit_cache& c, int64_t slot, int32_t position, uint32_t rot, uint32_t table_rows) {
    if (slot < 0) return 1;
    return slot < (int64_t)c.pages * c.page_size && (rot == 0 || (position >= 0 && (uint32_t)position < table_rows)) ? 0 : 2;
}

// Whether different slots, or heads of one, can share elements of the cache: axes in the order of their strides, each of which
// has to step over all that the ones before it reach.
inline bool cache_overlaps(const grape_wit_cache& c) {
    uint64_t n[3] = {c.pages, c.page_size, c.heads}, st[3] = {(uint64_t)c.page_stride, (uint64_t)c.token_stride, (uint64_t)c.head_stride};
    bool done[3] = {n[0] == 1, n[1] == 1, n[2] == 1};
    unsigned __int128 extent = c.dim;
    for (int step = 0; step < 3; step++) {
        int at = -1;
        for (int i = 0; i < 3; i++)
            if (!done[i] && (at < 0 || st[i] < st[at])) at = i;
        if (at < 0) break;
        if (st[at] < extent) return true;
        extent += (unsigned __int128)(n[at] - 1) * st[at];
        done[at] = true;
    }
    return false;
}

#define GRAPE_REFUSE(cond, msg) \
    if (cond) return msg

inline const char* refuse_cache(const grape_wit_cache* c) {
    GRAPE_REFUSE(!c, "cache is null");
    GRAPE_REFUSE(!c->d_k || !c->d_v, "the cache's keys or values are null");
    GRAPE_REFUSE(!c->pages || !c->page_size || !c->heads || !c->dim, "empty cache");
    GRAPE_REFUSE((uint64_t)c->pages * c->page_size >= (uint64_t)1 << 31, "the cache has 2^31 slots or more");
    GRAPE_REFUSE(c->heads > 65535 || c->dim > 8192, "at most 65535 heads of 8192 elements");
    const int64_t most = (int64_t)1 << 40;
    GRAPE_REFUSE(c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0, "negative stride");
    GRAPE_REFUSE(c->page_stride >= most || c->token_stride >= most || c->head_stride >= most, "stride of 2^40 or more");
    return nullptr;
}

// Units of work of one head and of one token of the append (see wit_append_kernel), pairs of `vec` elements each.
GRAPE_HD uint32_t append_head_units(uint32_t dim, uint32_t rot, uint32_t vec) { return rot / (2 * vec) + (dim - rot + 2 * vec - 1) / (2 * vec); }

inline const char* refuse_append(const grape_wit_rope_append_args* a, const grape_wit_cache* c) {
    GRAPE_REFUSE(!a, "args is null");
    if (const char* m = refuse_cache(c)) return m;
    GRAPE_REFUSE(a->scale < 1 || a->scale > (int64_t)1 << 31, "scale must be in 1..2^31 (the remainder is stored as int32)");
    GRAPE_REFUSE(a->rot % 2 || a->rot > c->dim, "rot must be even and at most dim");
    GRAPE_REFUSE(a->heads > 65535, "at most 65535 heads");
    GRAPE_REFUSE(cache_overlaps(*c), "different slots of the cache share elements");
    GRAPE_REFUSE(a->q_stride < 0 || a->k_stride < 0 || a->v_stride < 0, "negative stride");
    if (a->tokens == 0) return nullptr;
    GRAPE_REFUSE(a->tokens > (uint32_t)1 << 24, "at most 2^24 tokens");          // each workgroup looks through the later ones' slots
    GRAPE_REFUSE(!a->d_k || !a->d_v || !a->d_slots, "d_k, d_v or d_slots is null");
    GRAPE_REFUSE(a->heads && (!a->d_q || !a->d_q_out), "d_q or d_q_out is null");
    GRAPE_REFUSE(a->rot && (!a->d_positions || !a->d_cos || !a->d_sin || !a->table_rows), "the positions or their tables are missing");
    const uint64_t units = (uint64_t)(a->heads + 2 * c->heads) * append_head_units(c->dim, a->rot, 1);
    GRAPE_REFUSE(units >= (uint64_t)1 << 31 || a->tokens * (unsigned __int128)units >= (uint64_t)1 << 38, "tensor too large");
    return nullptr;
}

// How an attention call is cut up.  A workgroup of the scores and of the values takes `rows` query heads of one cache head and a
// chunk of the positions, one of the exponentials a query head and a chunk; with few sequences the chunks are short enough to
// fill the chip (about 8 workgroups a CU), with many they are long.
struct AttentionPlan {
    uint32_t dim64;                    // blocks of 64 elements of a head
    uint32_t rows, tiles;              // query heads of a workgroup, workgroups of a cache head
    bool score_apart;
    uint32_t score_chunk, score_chunks;
    uint32_t exp_chunk, exp_chunks;
    uint32_t blocks, groups;           // blocks of 32 elements of a values workgroup, workgroups of a head's elements
    uint32_t value_chunk, value_chunks;
    bool counted;                      // the scores' and the values' workgroups find their chunk by counting (see find_chunk)
    bool whole;                        // one launch, a workgroup for all positions
    size_t whole_lds;
    uint32_t row_held;                 // entries of a row of scores or exponentials in the workspace
    size_t at_scores, at_exp, at_max, at_sum, at_part, bytes;      // offsets in the workspace
};
constexpr uint32_t kTokenLds = 60 * 1024;      // of a workgroup; of one that takes all positions:
constexpr size_t kWholeLds = 72 * 1024;
constexpr uint32_t kWorkgroups = 4096;
constexpr uint32_t kWholeMost = 256;          // positions of the one launch
constexpr uint32_t kCountedMost = 256;        // sequences whose chunks are counted

inline uint32_t ceil_div(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }

// max_len: how many positions a row attends to at most; `rows`: how many rows there are where it is more than one of each sequence
inline bool attention_plan(uint32_t seqs, uint32_t heads, uint32_t cache_heads, uint32_t dim, uint32_t max_len, AttentionPlan& p, uint32_t rows = 0) {
    if (!seqs || !heads || !cache_heads || !dim || heads > 65535 || seqs > 65535 || heads % cache_heads || dim > 8192 || max_len >= (uint32_t)1 << 31) return false;
    const uint64_t rows_all = (uint64_t)seqs * heads;
    if ((unsigned __int128)rows_all * max_len >= (uint64_t)1 << 38) return false;
    const uint32_t each = heads / cache_heads;
    p.dim64 = ceil_div(dim, 64);
    p.rows = (kTokenLds - 4096) / (5 * 64 * p.dim64);      // five planes of the queries' digits
    p.rows = p.rows < 16 ? p.rows : 16;
    p.rows = p.rows < each ? p.rows : each;
    p.tiles = ceil_div(each, p.rows);
    auto chunk = [&](uint64_t beside, uint32_t step, uint32_t most, uint32_t workgroups) {
        const uint64_t want = beside >= workgroups ? 1 : workgroups / beside;
        uint64_t c = (max_len + want - 1) / want;
        c = (c + step - 1) / step * step;
        c = c < step ? step : c;
        return (uint32_t)(c < most ? c : most);
    };
    const uint64_t beside = (uint64_t)seqs * cache_heads * p.tiles;
    // a score waits in LDS, 8 bytes, beside the positions' offsets and the queries' digits
    const uint32_t left = kTokenLds - 5 * 64 * p.dim64 * p.rows;
    uint32_t score_most = left / (8 * p.rows + 8) / 64 * 64;
    if (score_most > 4096 / p.rows) score_most = 4096 / p.rows / 64 * 64;
    if (score_most < 64) return false;
    // with heads of 512 elements and more the waves share the elements of 16 positions instead of the positions: one sequence
    // of 500 with a head of 4096 is 32 workgroups then and not 8
    p.score_apart = p.dim64 >= 8;
    p.score_chunk = chunk(beside, p.score_apart ? 16 : 64, score_most, kWorkgroups);
    p.score_chunks = ceil_div(max_len, p.score_chunk);
    p.exp_chunk = chunk(rows_all, 1024, (uint32_t)1 << 20, kWorkgroups / 2);
    p.exp_chunks = ceil_div(max_len, p.exp_chunk);
    // four waves share a workgroup's elements, 32 each; those that find none left take every second or fourth step instead
    const uint32_t dim32 = ceil_div(dim, 32);
    p.blocks = dim32 > 2 ? 4 : dim32;
    uint32_t most = kTokenLds / (4 * p.rows + 8) / 64 * 64;
    if (most > 1024) most = 1024;
    if (max_len <= most && (max_len <= 512 || beside >= 256)) {
        // one chunk, so that nothing is left to join; fewer elements a workgroup until the chip is full (300 positions of 8 heads of
        // 128: 19.9 us a call and not 21.3, 64 sequences of up to 1000 90 and not 102; but one of 1000 26 and not 22)
        while (p.blocks > 1 && beside * ceil_div(dim32, p.blocks) < kWorkgroups / 4) p.blocks /= 2;
        p.groups = ceil_div(dim32, p.blocks);
        p.value_chunk = max_len <= 64 ? 64 : ceil_div(max_len, 64) * 64;
    } else {
        p.groups = ceil_div(dim32, p.blocks);
        // no longer than 256 while that leaves few parts to join, as many of max_len's positions may be none, and with several
        // sequences, whose lengths differ (64 of up to 2048, 8 heads of 128: 147 us a call and not 152; 8 of up to 20000 with a
        // window of 1024 39 and not 59); but one of 131072 281 us and not 292 without
        if (p.groups == 1 && (seqs >= 8 || beside * ceil_div(max_len, 256) <= kWorkgroups / 2) && most > 256) most = 256;
        p.value_chunk = chunk(beside * p.groups, p.blocks == 1 ? 128 : 64, most, kWorkgroups / 4);
    }
    p.value_chunks = ceil_div(max_len, p.value_chunk);
    // a launch's first axis, in threads
    if ((uint64_t)cache_heads * p.tiles * std::max<uint64_t>(p.score_chunks, (uint64_t)p.value_chunks * p.groups) >= (uint64_t)1 << 23) return false;
    // lengths that differ (see find_chunk for both sides); more sequences would make each workgroup's count long
    p.counted = seqs >= 8 && seqs <= kCountedMost &&
                (uint64_t)seqs * cache_heads * p.tiles * std::max<uint64_t>(p.score_chunks, (uint64_t)p.value_chunks * p.groups) < (uint64_t)1 << 23;
    // offsets, 64-bit sums of the scores and then of the output, scores, and the queries' digits or the probabilities' ones
    const size_t one = (size_t)5 * 64 * p.dim64 * p.rows, two = (size_t)4 * kWholeMost * p.rows;
    p.whole_lds = 8 * kWholeMost + (size_t)8 * p.rows * (dim > kWholeMost ? dim : kWholeMost) + (size_t)4 * kWholeMost * p.rows + (one > two ? one : two);
    p.whole = p.whole_lds <= kWholeLds && max_len <= kWholeMost && dim <= 256;
    const uint64_t rows_held = (uint64_t)std::max(seqs, rows) * heads;
    if ((unsigned __int128)rows_held * max_len >= (uint64_t)1 << 38) return false;
    p.row_held = max_len;
    const size_t row = (size_t)rows_held * max_len * 4;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    p.at_scores = 0;
    p.at_exp = up(row);
    p.at_max = p.at_exp + up(row);
    p.at_sum = p.at_max + up((size_t)rows_held * p.score_chunks * 4);
    p.at_part = p.at_sum + up((size_t)rows_held * p.exp_chunks * 8);
    p.bytes = p.whole ? 0 : p.at_part + (p.value_chunks > 1 ? (size_t)rows_held * p.value_chunks * dim * 8 : 0);
    return true;
}

// Bytes of workspace, 0 where a call of these sizes is refused.
inline size_t attention_workspace(uint32_t seqs, uint32_t heads, uint32_t cache_heads, uint32_t dim, uint32_t max_len) {
    AttentionPlan p;
    return attention_plan(seqs, heads, cache_heads, dim, max_len, p) ? p.bytes : 0;
}

// n / d for n below 2^31
struct FastDiv {
    uint32_t d, mul, shift;
    GRAPE_HD uint32_t operator()(uint32_t n) const {
        return d == 1 ? n : (uint32_t)(((uint64_t)n * mul) >> 32) >> shift;
    }
};
inline FastDiv fast_div(uint32_t d) {
    // the smallest l with 2^l >= d; mul = floor(2^(31 + l) / d) + 1 is off by at most d / 2^(31 + l) <= 2^-31 a unit of n
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) l++;
    return FastDiv{d, d == 1 ? 0 : (uint32_t)((((uint64_t)1 << (31 + l)) / d) + 1), l - 1};
}

inline const char* refuse_attention(const grape_wit_attention_args* a, const grape_wit_cache* c) {
    GRAPE_REFUSE(!a, "args is null");
    if (const char* m = refuse_cache(c)) return m;
    const int64_t most = (int64_t)1 << 31;
    GRAPE_REFUSE(a->qk_scale < 1 || a->qk_scale > most || a->out_scale < 1 || a->out_scale > most || a->prob_scale < 1 || a->prob_scale > most / 2,
                 "scales must be in 1..2^31, prob_scale in 1..2^30");
    GRAPE_REFUSE(a->bit_shift < 1 || a->bit_shift > 30 || a->index_bits < 1 || a->index_bits > 30, "bit_shift and index_bits must be in 1..30");
    GRAPE_REFUSE(a->heads < 1 || a->heads > 65535 || a->heads % c->heads, "heads must be a multiple of the cache's heads");
    GRAPE_REFUSE(a->q_stride < 0, "negative stride");
    if (a->seqs == 0) return nullptr;
    GRAPE_REFUSE(a->seqs > 65535, "at most 65535 sequences");
    GRAPE_REFUSE(a->max_len >= (uint32_t)1 << 31, "max_len must be below 2^31");
    GRAPE_REFUSE(!a->d_q || !a->d_lens || !a->d_exp_table || !a->d_out, "d_q, d_lens, d_exp_table or d_out is null");
    GRAPE_REFUSE(a->max_len && !a->d_block_table, "d_block_table is null");
    AttentionPlan plan;
    GRAPE_REFUSE(!attention_plan(a->seqs, a->heads, c->heads, c->dim, a->max_len, plan), "tensor too large");
    const size_t need = plan.bytes;
    GRAPE_REFUSE(a->workspace_bytes < need || (need && !a->d_workspace), "the workspace is too small");
    GRAPE_REFUSE((uintptr_t)a->d_workspace & 15, "the workspace must be 16-byte aligned");
    return nullptr;
}

// Products with 4-bit weights.  One token is taken apart by the workgroups that multiply it, and so are up to four while that is
// little work for them (two tokens through 4096 x 4096, groups of 128: 8.0 to 8.5 us a call and not 10.0, four 9.5 and not 10.4); more by
// a launch of its own, into the workspace, in tiles of four, eight or sixteen (four tokens through 16384 x 8192, groups of 128: 24 us
// and not 44, with zero points 30 and not 47).  One word a block of 2048 inputs of a token says whether one of them is above the digits;
// any such word of a tile's tokens sends all of the tile's sums through their rows again.
constexpr uint32_t kQ4Inputs = (uint32_t)1 << 24;          // a thread looks through a row's for those above the digits
inline bool q4_few(uint32_t tokens, uint32_t outputs, uint32_t inputs) {
    const uint64_t tiles = ceil_div(outputs, 16) < 256 ? 256 : ceil_div(outputs, 16);
    return tokens == 1 || (tokens <= 4 && tiles * tokens * ceil_div(inputs, 128) <= 40000);
}
struct Q4Plan {
    uint32_t tile_tokens, token_tiles;
    uint32_t makers;                   // workgroups of one token that make digits
    size_t at_over, bytes;
};
inline Q4Plan q4_plan(uint32_t tokens, uint32_t inputs) {
    Q4Plan p;
    const uint32_t units = ceil_div(inputs, 128);
    p.tile_tokens = tokens <= 4 ? 4 : tokens <= 8 ? 8 : 16;
    p.token_tiles = ceil_div(tokens, p.tile_tokens);
    p.makers = ceil_div(units * 16, 256);
    p.at_over = (size_t)p.token_tiles * units * 32 * 4 * p.tile_tokens * 4;
    p.bytes = p.at_over + (size_t)4 * tokens * p.makers;
    return p;
}
inline size_t q4_workspace(uint32_t tokens, uint32_t outputs, uint32_t inputs, uint32_t group) {
    if (!tokens || !outputs || !inputs || !group || group % 32 || tokens > 65535 || inputs > kQ4Inputs || q4_few(tokens, outputs, inputs)) return 0;
    return q4_plan(tokens, inputs).bytes;
}

inline const char* refuse_q4(const void* d_q, const void* d_x, int64_t x_stride, const void* d_w, int64_t w_stride, const void* d_scales,
                             uint32_t tokens, uint32_t outputs, uint32_t inputs, uint32_t group, int64_t scale, const void* d_workspace, size_t workspace_bytes) {
    GRAPE_REFUSE(scale < 1 || scale > (int64_t)1 << 31, "scale must be in 1..2^31 (the remainder is stored as int32)");
    GRAPE_REFUSE(inputs < 1 || group < 1, "empty inner dimension or group");
    GRAPE_REFUSE(inputs > kQ4Inputs || group > (uint32_t)1 << 30, "at most 2^24 inputs");
    GRAPE_REFUSE(x_stride < 0 || w_stride < 0, "negative stride");
    if (!tokens || !outputs) return nullptr;
    GRAPE_REFUSE(!d_q || !d_x || !d_w || !d_scales, "d_q, d_x, d_w or d_scales is null");
    GRAPE_REFUSE(tokens > 65535, "at most 65535 tokens");
    GRAPE_REFUSE(outputs > (uint32_t)1 << 24, "at most 2^24 outputs");
    const size_t need = q4_workspace(tokens, outputs, inputs, group);
    GRAPE_REFUSE(workspace_bytes < need || (need && !d_workspace), "the workspace is too small");
    GRAPE_REFUSE(need && ((uintptr_t)d_workspace & 15), "the workspace must be 16-byte aligned");
    return nullptr;
}
#undef GRAPE_REFUSE

}  // namespace token
}  // namespace grape

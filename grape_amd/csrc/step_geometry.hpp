// What the calls around a step of new tokens - its pages and slots, the choice of the next tokens - take and refuse, and where
// their entries stand: the expressions that the kernels and their entry points use, free of HIP so that a host build can walk over them.
#pragma once
#include "token_geometry.hpp"

namespace grape {
namespace step {

#define GRAPE_REFUSE(cond, msg) \
    if (cond) return msg

// ---- pages and slots
constexpr uint32_t kPageSeqs = 4096;          // whose prefix sums a workgroup holds in LDS

GRAPE_HD uint32_t pages_of(uint32_t tokens, const token::FastDiv& by_page) { return tokens ? by_page(tokens - 1) + 1 : 0; }

// Pages that no token from `pos` on sees through a window: those before page number out_of_sight(pos), but for the sinks' own.
GRAPE_HD uint32_t out_of_sight(uint32_t pos, uint32_t window, const token::FastDiv& by_page) {
    return window && pos + 1 > window ? by_page(pos + 1 - window) : 0;
}

// One sequence's part of a step: lengths before and after, pages held before and taken by it, pages given back (`first_back` from
// page number `back_from`, and the first `kept_back` pages too, which is a request that is over).
struct Sequence {
    uint32_t len, tokens, held, taken;
    uint32_t kept_back, back_from, back;
    bool ended, ok;
    // what it asks for; false where its numbers do not fit
    GRAPE_HD bool ask(int32_t len_, int32_t new_, uint64_t most, const token::FastDiv& by_page) {
        ended = new_ == -1;
        tokens = new_ > 0 ? (uint32_t)new_ : 0;
        ok = len_ >= 0 && new_ >= -1 && (uint64_t)(uint32_t)len_ + tokens <= most;
        len = len_ >= 0 ? (uint32_t)len_ : 0;
        if (!ok) {
            ended = false;
            tokens = 0;
        }
        held = ok ? pages_of(len, by_page) : 0;
        taken = ok ? pages_of(len + tokens, by_page) - held : 0;
        return ok;
    }
    GRAPE_HD void refuse() { tokens = taken = 0; }
    GRAPE_HD void give_back(uint32_t window, uint32_t sink_pages, const token::FastDiv& by_page) {
        kept_back = back_from = back = 0;
        if (!ok) return;
        const uint32_t from = out_of_sight(len, window, by_page), lo = from > sink_pages ? from : sink_pages;
        const uint32_t to = ended ? held : out_of_sight(len + tokens, window, by_page);
        back_from = lo;
        if (ended) kept_back = sink_pages < held ? sink_pages : held;
        back = kept_back + (to > lo ? to - lo : 0);
    }
    // the number of page j of those given back
    GRAPE_HD uint32_t back_page(uint32_t j) const { return j < kept_back ? j : back_from + (j - kept_back); }
};

inline bool ranges_meet(const void* a, size_t n, const void* b, size_t m) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && n && m && x < y + m && y < x + n;
}

inline const char* refuse_pages(const grape_wit_page_step_args* a) {
    GRAPE_REFUSE(!a, "args is null");
    GRAPE_REFUSE(a->seqs > kPageSeqs, "at most 4096 sequences");
    GRAPE_REFUSE(!a->page_size, "empty pages");
    GRAPE_REFUSE((uint64_t)a->page_size * a->table_stride >= (uint64_t)1 << 31, "a sequence's pages hold 2^31 tokens or more");
    GRAPE_REFUSE((uint64_t)a->seqs * a->table_stride >= (uint64_t)1 << 31, "the block table has 2^31 entries or more");
    GRAPE_REFUSE(a->rows >= (uint32_t)1 << 31 || a->ring >= (uint32_t)1 << 31, "2^31 rows or entries of the ring or more");
    GRAPE_REFUSE(a->window >= (uint32_t)1 << 31 || a->sinks >= (uint32_t)1 << 31, "window and sinks must be below 2^31");
    GRAPE_REFUSE(!a->window && a->sinks, "sinks need a window");
    GRAPE_REFUSE(!a->d_span || !a->d_span_out || !a->d_starts, "d_span, d_span_out or d_starts is null");
    GRAPE_REFUSE(a->seqs && (!a->d_lens || !a->d_new || !a->d_lens_out), "d_lens, d_new or d_lens_out is null");
    GRAPE_REFUSE(a->seqs && a->table_stride && !a->d_block_table, "d_block_table is null");
    GRAPE_REFUSE(a->ring && !a->d_free, "d_free is null");
    GRAPE_REFUSE(a->rows && (!a->d_positions || !a->d_slots), "d_positions or d_slots is null");
    // every workgroup reads the inputs, whatever the others have written by then
    const void* in[] = {a->d_lens, a->d_new, a->d_span};
    const size_t in_bytes[] = {(size_t)4 * a->seqs, (size_t)4 * a->seqs, 8};
    const void* out[] = {a->d_starts, a->d_positions, a->d_slots, a->d_lens_out, a->d_span_out, a->d_block_table, a->d_free};
    const size_t out_bytes[] = {(size_t)4 * a->seqs + 4, (size_t)4 * a->rows, (size_t)8 * a->rows, (size_t)4 * a->seqs, 8, (size_t)4 * a->seqs * a->table_stride, (size_t)4 * a->ring};
    for (int i = 0; i < 3; i++)
        for (int o = 0; o < 7; o++) GRAPE_REFUSE(ranges_meet(in[i], in_bytes[i], out[o], out_bytes[o]), "an output overlaps an input");
    for (int i = 0; i < 7; i++)
        for (int o = i + 1; o < 7; o++) GRAPE_REFUSE(ranges_meet(out[i], out_bytes[i], out[o], out_bytes[o]), "two outputs overlap");
    return nullptr;
}

// ---- the next token
// A workgroup takes a chunk of a row's vocabulary, and counts the row's history for it: 8192 tokens, or half and a quarter where that leaves CUs
// idle (one row of 32000: 5.5 us, by 8192 8.7; 64 rows 12.0 by 4096, 13.7 by 2048, 14.5 by 8192; 256 rows of 131072: 67, by 2048 110).
struct NextPlan {
    uint32_t chunk, chunks;
    size_t bytes;
};
constexpr uint32_t kNextLeast = 2048, kNextMost = 8192;

inline NextPlan next_plan(uint32_t seqs, uint32_t vocab) {
    NextPlan p;
    p.chunk = kNextMost;
    while (p.chunk > kNextLeast && (uint64_t)seqs * token::ceil_div(vocab, p.chunk) < 400) p.chunk /= 2;
    p.chunks = token::ceil_div(vocab, p.chunk);
    p.bytes = (size_t)8 * seqs * p.chunks;
    return p;
}
inline size_t next_workspace(uint32_t seqs, uint32_t vocab) {
    if (!seqs || !vocab || seqs > 65535 || vocab > (uint32_t)1 << 24) return 0;
    return next_plan(seqs, vocab).bytes;
}

inline const char* refuse_next(const grape_wit_next_token_args* a) {
    GRAPE_REFUSE(!a, "args is null");
    GRAPE_REFUSE(a->seqs > 65535, "at most 65535 sequences");
    GRAPE_REFUSE(a->vocab < 1 || a->vocab > (uint32_t)1 << 24, "the vocabulary must have 1 to 2^24 tokens");
    GRAPE_REFUSE(a->scale < 1 || a->scale > (int64_t)1 << 31, "scale must be in 1..2^31 (the remainder is stored as int32)");
    GRAPE_REFUSE(a->history > (uint32_t)1 << 24, "at most 2^24 tokens of history");          // each of up to 2048 workgroups of a row reads it all
    const int64_t most = (int64_t)1 << 40;
    GRAPE_REFUSE(a->logits_stride < 0 || a->history_stride < 0 || a->bias_stride < 0 || a->mask_stride < 0, "negative stride");
    GRAPE_REFUSE(a->logits_stride >= most || a->history_stride >= most || a->bias_stride >= most || a->mask_stride >= most, "stride of 2^40 or more");
    if (!a->seqs) return nullptr;
    GRAPE_REFUSE(!a->d_logits || !a->d_token, "d_logits or d_token is null");
    GRAPE_REFUSE(a->history && (!a->d_history || !a->d_history_lens), "d_history or d_history_lens is null");
    const size_t need = next_workspace(a->seqs, a->vocab);
    GRAPE_REFUSE(a->workspace_bytes < need || !a->d_workspace, "the workspace is too small");
    GRAPE_REFUSE((uintptr_t)a->d_workspace & 15, "the workspace must be 16-byte aligned");
    const size_t all = (size_t)4 * a->seqs * a->vocab, one = (size_t)4 * a->seqs;
    const void* out[] = {a->d_out, a->d_rem, a->d_count, a->d_gap, a->d_token, a->d_max, a->d_workspace};
    const size_t out_bytes[] = {all, all, all, all, one, one, need};
    for (int i = 0; i < 7; i++)
        for (int o = i + 1; o < 7; o++) GRAPE_REFUSE(ranges_meet(out[i], out_bytes[i], out[o], out_bytes[o]), "two outputs overlap");
    const void* in[] = {a->d_logits, a->d_bias};
    const int64_t stride[] = {a->logits_stride, a->bias_stride};
    for (int i = 0; i < 2; i++)
        for (int o = 0; o < 7; o++)
            GRAPE_REFUSE(ranges_meet(in[i], 4 * ((size_t)(a->seqs - 1) * stride[i] + a->vocab), out[o], out_bytes[o]) &&
                             !(i == 0 && o == 0 && in[i] == out[o] && (a->seqs == 1 || stride[i] == (int64_t)a->vocab)), "an output overlaps an input");
    // what the first launch reads beside them must not be what it writes (all but d_token and d_max); entries of the history behind its lengths are not used,
    // so it is not looked at here
    const size_t words = ((size_t)a->seqs - 1) * (size_t)a->mask_stride + (a->vocab + 31) / 32;
    const void* beside[] = {a->d_history_lens, a->d_repetition, a->d_presence, a->d_frequency, a->d_mask};
    const size_t beside_bytes[] = {a->history ? one : 0, one, one, one, 4 * words};
    for (int i = 0; i < 5; i++)
        for (int o = 0; o < 7; o++) GRAPE_REFUSE(o != 4 && o != 5 && ranges_meet(beside[i], beside_bytes[i], out[o], out_bytes[o]), "an output overlaps an input");
    return nullptr;
}

// ---- attention of several tokens a sequence
// A workgroup takes kRows rows of one cache head - the query heads of a token that read it side by side, token after token - and
// positions in tiles of kCols.  Sequence b's tiles of rows are numbered from starts[b] * each / kRows + b on, which leaves none to two
// sequences whatever the lengths are: no workgroup has to know more than its own sequence.
constexpr uint32_t kRows = 32, kCols = 64;

struct WindowPlan {
    uint32_t each, dim64;
    uint32_t tiles;                            // of rows of one cache head, at most
    uint32_t cols;                             // tiles of positions that a tile of rows sees, at most
    uint32_t score_cols, score_chunks;         // of a workgroup of the scores, and workgroups along the positions
    uint32_t exp_cols, exp_chunks;
    uint32_t value_cols, value_chunks, groups;          // and workgroups along a head's elements
    bool packed;                               // operands are made beforehand, see wit_window_pack_kernel:
    uint32_t steps, all_cols, splits;          // steps of 64 elements of theirs, tiles of positions that a sequence's rows see, workgroups of a tile's elements
    size_t at_keys, at_values, at_queries, at_over, at_query_over;
    size_t at_scores, at_exp, at_max, at_sum, at_factors, at_part, bytes;
};
constexpr size_t kFactorBytes = 2 * 1024 * 8 + 64 * 4;
constexpr uint32_t kValueDims = 128;
constexpr uint32_t kValueMost = 511;          // tiles of positions: four products of digits each, 4 * 2^14 * 64 * 511, fit 32 bits
constexpr uint32_t kPackTiles = 8, kPackSteps = 4;          // tiles of rows that operands made beforehand serve at least; steps of a workgroup
constexpr uint64_t kPackProducts = (uint64_t)1 << 30;
constexpr size_t kKeyStepBytes = 3 * kCols * 64, kQueryStepBytes = 3 * kRows * 64, kValueStepBytes = 3 * kCols * 64;
constexpr uint32_t kJoinRows = 4;              // of a workgroup that joins the values' chunks
constexpr uint32_t kOffsetTiles = 16;          // tiles of positions whose offsets a values workgroup holds

inline bool window_plan(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t cache_heads, uint32_t dim, uint32_t max_new, uint32_t max_len, uint32_t window, uint32_t sinks,
                        WindowPlan& p) {
    if (!rows || !seqs || !heads || !cache_heads || !dim || !max_new || !max_len || heads > 65535 || seqs > 65535 || heads % cache_heads || dim > 8192) return false;
    if (max_len >= (uint32_t)1 << 31 || max_new > max_len || window >= (uint32_t)1 << 31 || sinks >= (uint32_t)1 << 31 || rows > (uint32_t)1 << 24) return false;
    p.each = heads / cache_heads;
    p.dim64 = token::ceil_div(dim, 64);
    const uint64_t rows_all = (uint64_t)rows * heads, tiles = (uint64_t)rows * p.each / kRows + seqs;
    if ((unsigned __int128)rows_all * max_len >= (uint64_t)1 << 38) return false;
    uint64_t cols = token::ceil_div(max_len, kCols);
    if (window) cols = std::min<uint64_t>(cols, ((uint64_t)window + kRows + kCols - 1) / kCols + 1 + ((uint64_t)sinks + kCols - 1) / kCols);
    p.tiles = (uint32_t)tiles;
    p.cols = (uint32_t)cols;
    // a launch's first axis in workgroups, the others' limits
    if (tiles * cache_heads >= (uint64_t)1 << 22) return false;
    // tiles of rows that are surely there, and as many workgroups as fill the chip
    const uint64_t beside = std::max<uint64_t>((uint64_t)rows * p.each / kRows, std::min(seqs, rows)) * cache_heads;
    auto chunk = [&](uint64_t workgroups, uint64_t most) {
        const uint64_t want = beside >= workgroups ? 1 : workgroups / beside;
        return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, (cols + want - 1) / want));
    };
    p.score_cols = chunk(p.dim64 > 8 ? 4096 : 768, 32);
    p.score_chunks = token::ceil_div(p.cols, p.score_cols);
    // four tiles or more, which a wave reads at once (4 sequences of 4000: 20 us, and 25 and 40 by two and one), but where that leaves CUs idle (3 of 500: 19 and 11 by one)
    p.exp_cols = std::max(std::min(4u, chunk(256, 16)), chunk(2048, 16));
    p.exp_chunks = token::ceil_div(p.cols, p.exp_cols);
    p.groups = token::ceil_div(dim, kValueDims);
    const uint64_t want = beside * p.groups >= 512 ? 1 : 512 / (beside * p.groups);
    p.value_cols = (uint32_t)std::min<uint64_t>((cols + want - 1) / want, kValueMost);
    p.value_chunks = token::ceil_div(p.cols, p.value_cols);
    if (p.score_chunks > 65535 || p.exp_chunks > 65535 || (uint64_t)p.value_chunks * p.groups > 65535) return false;
    // workgroups without rows or positions, of many sequences that might be long, take their time too; the join's are many where few rows of long
    // heads stand beside many sequences without any
    const uint64_t joins = p.value_chunks > 1 ? (uint64_t)p.dim64 * (kRows / kJoinRows) : 0;
    const uint64_t most = std::max(std::max<uint64_t>(std::max(p.score_chunks, p.exp_chunks), (uint64_t)p.value_chunks * p.groups), joins);
    if (tiles * cache_heads * most >= (uint64_t)1 << 27) return false;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    // Operands are made beforehand where each key and value then serves eight tiles of rows or more (24 sequences of 2000 positions, 32 heads of 128
    // over 8: 32 new tokens 674 us from the cache and 706 so, 12 of 64 tokens 671 and 627), in calls of 2^30 products or more (one such sequence:
    // 64 tokens of 1000 64 and 68 us, 128 of 2000 135 and 127, 512 of 4000 698 and 556), and where they take no more than a few GiB.
    p.steps = p.dim64 == 1 ? 1 : (p.dim64 + 1) / 2 * 2;
    uint64_t all = token::ceil_div(max_len, kCols);
    if (window) all = std::min<uint64_t>(all, ((uint64_t)window + max_new + kCols - 1) / kCols + 1 + ((uint64_t)sinks + kCols - 1) / kCols);
    p.all_cols = (uint32_t)all;
    p.splits = token::ceil_div(p.dim64, kPackSteps);
    const uint64_t cache_tiles = (uint64_t)seqs * p.all_cols * cache_heads;
    const unsigned __int128 key_bytes = (unsigned __int128)cache_tiles * p.steps * kKeyStepBytes, value_bytes = (unsigned __int128)cache_tiles * p.dim64 * kValueStepBytes;
    const uint64_t query_bytes = tiles * cache_heads * p.steps * kQueryStepBytes;
    p.packed = (uint64_t)rows * p.each >= (uint64_t)kPackTiles * kRows * seqs && (unsigned __int128)rows_all * p.cols * kCols * dim >= kPackProducts && key_bytes + value_bytes + query_bytes <= (uint64_t)4 << 30 &&
               (cache_tiles + tiles * cache_heads) * p.splits < (uint64_t)1 << 22;
    const size_t row = (size_t)rows_all * p.cols * kCols * 4;
    p.at_scores = 0;
    p.at_exp = up(row);
    p.at_max = p.at_exp + up(row);
    p.at_sum = p.at_max + up((size_t)rows_all * p.score_chunks * 4);
    p.at_factors = p.at_sum + up((size_t)rows_all * 8);
    p.at_part = p.at_factors + up(kFactorBytes);
    p.at_keys = p.at_part + up(p.value_chunks > 1 ? (size_t)rows_all * p.value_chunks * dim * 8 : 0);
    p.at_values = p.at_keys + (p.packed ? up((size_t)key_bytes) : 0);
    p.at_queries = p.at_values + (p.packed ? up((size_t)value_bytes) : 0);
    p.at_over = p.at_queries + (p.packed ? up((size_t)query_bytes) : 0);
    p.at_query_over = p.at_over + (p.packed ? up((size_t)cache_tiles * p.splits * 4) : 0);
    p.bytes = p.at_query_over + (p.packed ? up((size_t)tiles * cache_heads * p.splits * 4) : 0);
    return true;
}
// Single tokens go the way of attention_plan, with at most this many positions each.
GRAPE_HD uint32_t seen_most(uint32_t max_len, uint32_t window, uint32_t sinks) {
    return window && (uint64_t)window + sinks < max_len ? window + sinks : max_len;
}
inline bool single_plan(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t cache_heads, uint32_t dim, uint32_t max_len, uint32_t window, uint32_t sinks, token::AttentionPlan& p) {
    return rows && max_len && token::attention_plan(seqs, heads, cache_heads, dim, seen_most(max_len, window, sinks), p, rows);
}
inline size_t window_workspace(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t cache_heads, uint32_t dim, uint32_t max_new, uint32_t max_len, uint32_t window, uint32_t sinks) {
    if (max_new == 1) {
        token::AttentionPlan one;
        return single_plan(rows, seqs, heads, cache_heads, dim, max_len, window, sinks, one) ? one.bytes : 0;
    }
    WindowPlan p;
    return window_plan(rows, seqs, heads, cache_heads, dim, max_new, max_len, window, sinks, p) ? p.bytes : 0;
}

// What a sequence brings to a call: its first row, its new tokens, the first one's position.  False (and no tokens) where its
// numbers do not fit the call.
GRAPE_HD bool new_tokens(int32_t s, int32_t e, int32_t len, uint32_t rows, uint32_t max_new, uint32_t max_len, uint64_t most, uint32_t& n, uint32_t& pos) {
    const bool ok = s >= 0 && e >= s && (uint32_t)e <= rows && (uint32_t)(e - s) <= max_new && len >= e - s && (uint32_t)len <= max_len && (uint64_t)(uint32_t)len <= most;
    n = ok ? (uint32_t)(e - s) : 0;
    pos = ok ? (uint32_t)len - n : 0;
    return ok;
}

// The sequence that tile of rows `ti` belongs to; any other where it belongs to none.  One search, ballot(f) asking 64 sequences at a time
// what f says of lane 0 .. 63, for the last one whose tiles start at ti or before.  An entry that is no row of the call starts no tiles, so that the
// others, which ascend, are searched as if it was not there; but where it was asked for its part of the sequences the search ends at one before it, whose
// rows then have no end (not has_rows), and all are gone through.
GRAPE_HD bool is_row(int32_t s, uint32_t rows) { return (uint32_t)s <= rows; }          // rows <= 2^24: no negative one is
GRAPE_HD bool has_rows(int32_t s, int32_t e, uint32_t rows) { return is_row(s, rows) && is_row(e, rows) && s <= e; }
GRAPE_HD uint64_t first_tile(int32_t s, uint32_t b, uint32_t each) { return (uint64_t)(uint32_t)s * each / kRows + b; }
GRAPE_HD uint32_t last_lane(unsigned long long lanes) { return 63u - (uint32_t)__builtin_clzll(lanes); }
template <class Ballot>
GRAPE_HD uint32_t search_tile(const int32_t* starts, uint32_t seqs, uint32_t rows, uint32_t each, uint32_t ti, Ballot ballot) {
    uint32_t lo = 0, left = seqs;
    while (left > 1) {
        const uint32_t step = (left + 63) / 64;
        const unsigned long long before = ballot([&](uint32_t lane) {
            const uint32_t at = lane * step < left ? lo + lane * step : lo + left - 1;
            const int32_t s = starts[at];
            return lane * step < left && is_row(s, rows) && first_tile(s, at, each) <= ti;
        });
        const uint32_t last = before ? last_lane(before) : 0;
        lo += last * step;
        left = left - last * step < step ? left - last * step : step;
    }
    return lo;
}
template <class Ballot>
GRAPE_HD uint32_t scan_for_tile(const int32_t* starts, uint32_t seqs, uint32_t rows, uint32_t each, uint32_t ti, Ballot ballot) {
    for (uint32_t base = 0; base < seqs; base += 64) {
        const unsigned long long here = ballot([&](uint32_t lane) {
            const uint32_t b = base + lane;
            if (b >= seqs) return false;
            const int32_t s = starts[b], e = starts[b + 1];
            return has_rows(s, e, rows) && first_tile(s, b, each) <= ti && (ti - first_tile(s, b, each)) * kRows < (uint64_t)(uint32_t)(e - s) * each;
        });
        if (here) return base + last_lane(here);
    }
    return 0;
}

// The positions that a tile of rows with the tokens at pos0 .. pos1 sees, in tiles: `sink_tiles` from 0 on, then those from tile
// `from` on, `tiles` in all.
struct Seen {
    uint32_t lo, hi, sinks;                    // lo <= t < hi, or t < sinks
    uint32_t sink_tiles, from, tiles;
    GRAPE_HD Seen(uint32_t pos0, uint32_t pos1, uint32_t window, uint32_t sinks_) {
        hi = pos1 + 1;
        lo = window && pos0 + 1 > window ? pos0 + 1 - window : 0;
        sinks = sinks_ < lo ? sinks_ : lo;
        from = lo / kCols;
        sink_tiles = (sinks + kCols - 1) / kCols;
        if (sink_tiles > from) sink_tiles = from;
        tiles = sink_tiles + (hi + kCols - 1) / kCols - from;
    }
    GRAPE_HD uint32_t tile(uint32_t v) const { return v < sink_tiles ? v : v - sink_tiles + from; }
    // and back: the number of a tile that is one of these
    GRAPE_HD uint32_t number(uint32_t tile) const { return tile < sink_tiles ? tile : tile - from + sink_tiles; }
    GRAPE_HD bool any(uint32_t t) const { return t < hi && (t >= lo || t < sinks); }
    // the tiles from <= v < to of v0 .. v0 + n, counted from v0, whose positions all rows see (tokens pos0 .. pos1); sinks' tiles are not counted
    GRAPE_HD void full(uint32_t pos0, uint32_t pos1, uint32_t window, uint32_t v0, uint32_t n, uint32_t& first, uint32_t& last) const {
        const uint32_t lowest = window && pos1 + 1 > window ? (pos1 - window) / kCols + 1 : 0, end = (pos0 + 1) / kCols;
        const uint32_t a = sink_tiles + (lowest > from ? lowest - from : 0), b = end > from ? sink_tiles + end - from : 0;
        first = a > v0 ? (a - v0 < n ? a - v0 : n) : 0;
        last = b > v0 ? (b - v0 < n ? b - v0 : n) : 0;
        if (last < first) last = first;
    }
};
// whether the token at `pos` sees position t
GRAPE_HD bool sees(uint32_t pos, uint32_t t, uint32_t window, uint32_t sinks) { return t <= pos && (!window || t + window > pos || t < sinks); }

inline const char* refuse_window(const grape_wit_window_attention_args* a, const grape_wit_cache* c) {
    GRAPE_REFUSE(!a, "args is null");
    if (const char* m = token::refuse_cache(c)) return m;
    const int64_t most = (int64_t)1 << 31;
    GRAPE_REFUSE(a->qk_scale < 1 || a->qk_scale > most || a->out_scale < 1 || a->out_scale > most || a->prob_scale < 1 || a->prob_scale > most / 2,
                 "scales must be in 1..2^31, prob_scale in 1..2^30");
    GRAPE_REFUSE(a->bit_shift < 1 || a->bit_shift > 30 || a->index_bits < 1 || a->index_bits > 30, "bit_shift and index_bits must be in 1..30");
    GRAPE_REFUSE(a->heads < 1 || a->heads > 65535 || a->heads % c->heads, "heads must be a multiple of the cache's heads");
    GRAPE_REFUSE(a->q_stride < 0, "negative stride");
    GRAPE_REFUSE(a->window >= (uint32_t)1 << 31 || a->sinks >= (uint32_t)1 << 31, "window and sinks must be below 2^31");
    GRAPE_REFUSE(!a->window && a->sinks, "sinks need a window");
    GRAPE_REFUSE(a->max_new > a->max_len, "max_new must be at most max_len");
    if (!a->seqs || !a->rows || !a->max_new) return nullptr;
    GRAPE_REFUSE(a->seqs > 65535, "at most 65535 sequences");
    GRAPE_REFUSE(!a->d_q || !a->d_starts || !a->d_lens || !a->d_exp_table || !a->d_out || !a->d_block_table, "d_q, d_starts, d_lens, d_exp_table, d_block_table or d_out is null");
    GRAPE_REFUSE(a->rows > (uint32_t)1 << 24, "at most 2^24 rows");
    WindowPlan p;
    token::AttentionPlan one;
    GRAPE_REFUSE(a->max_new == 1 ? !single_plan(a->rows, a->seqs, a->heads, c->heads, c->dim, a->max_len, a->window, a->sinks, one)
                                 : !window_plan(a->rows, a->seqs, a->heads, c->heads, c->dim, a->max_new, a->max_len, a->window, a->sinks, p), "tensor too large");
    const size_t need = a->max_new == 1 ? one.bytes : p.bytes;
    GRAPE_REFUSE(a->workspace_bytes < need || (need && !a->d_workspace), "the workspace is too small");
    GRAPE_REFUSE((uintptr_t)a->d_workspace & 15, "the workspace must be 16-byte aligned");
    return nullptr;
}
#undef GRAPE_REFUSE

}  // namespace step
}  // namespace grape

// Host build of grape_amd/csrc/step_geometry.hpp: which calls are refused, what the plans of a step's calls cover, where tokens, tiles
// and pages stand, and the argument structs as the Python helpers pack them.
#include <cstring>
#include "../../grape_amd/csrc/step_geometry.hpp"
using namespace grape;

extern "C" {
const char* refuse_pages(const grape_wit_page_step_args* a) { return step::refuse_pages(a); }
const char* refuse_window(const grape_wit_window_attention_args* a, const grape_wit_cache* c) { return step::refuse_window(a, c); }
const char* refuse_next(const grape_wit_next_token_args* a) { return step::refuse_next(a); }
size_t struct_bytes(int which) {
    return which == 0 ? sizeof(grape_wit_page_step_args) : which == 1 ? sizeof(grape_wit_window_attention_args) : sizeof(grape_wit_next_token_args);
}
size_t window_workspace(uint32_t rows, uint32_t seqs, uint32_t h, uint32_t hk, uint32_t d, uint32_t most, uint32_t n, uint32_t w, uint32_t s) {
    return step::window_workspace(rows, seqs, h, hk, d, most, n, w, s);
}
size_t next_workspace(uint32_t n, uint32_t v) { return step::next_workspace(n, v); }
void next_of(uint32_t n, uint32_t v, uint32_t* o) {
    const step::NextPlan p = step::next_plan(n, v);
    o[0] = p.chunk;
    o[1] = p.chunks;
}
// a sequence's part of a step: whether its numbers fit, tokens, pages held, taken and given back, and the numbers of the latter
int sequence(int32_t len, int32_t n, uint64_t most, uint32_t page, uint32_t window, uint32_t sinks, uint32_t* o, uint32_t room) {
    const token::FastDiv by = token::fast_div(page);
    step::Sequence s;
    const bool ok = s.ask(len, n, most, by);
    s.give_back(window, window ? step::pages_of(sinks, by) : 0, by);
    o[0] = s.tokens;
    o[1] = s.held;
    o[2] = s.taken;
    o[3] = s.back;
    for (uint32_t j = 0; j < s.back && j < room; j++) o[4 + j] = s.back_page(j);
    return ok;
}
int new_tokens(int32_t s, int32_t e, int32_t len, uint32_t rows, uint32_t max_new, uint32_t max_len, uint64_t most, uint32_t* o) {
    return step::new_tokens(s, e, len, rows, max_new, max_len, most, o[0], o[1]);
}
// the sequence that every tile of rows is given to
void tile_owners(const int32_t* starts, uint32_t seqs, uint32_t rows, uint32_t each, uint32_t tiles, uint32_t* o) {
    auto ballot = [](auto f) {
        unsigned long long lanes = 0;
        for (uint32_t lane = 0; lane < 64; lane++) lanes |= (unsigned long long)(f(lane) ? 1 : 0) << lane;
        return lanes;
    };
    for (uint32_t t = 0; t < tiles; t++) {
        o[t] = step::search_tile(starts, seqs, rows, each, t, ballot);
        if (!step::has_rows(starts[o[t]], starts[o[t] + 1], rows)) o[t] = step::scan_for_tile(starts, seqs, rows, each, t, ballot);
    }
}
int sees(uint32_t pos, uint32_t t, uint32_t window, uint32_t sinks) { return step::sees(pos, t, window, sinks); }
// the tiles of positions that tokens pos0 .. pos1 see, and for n of them from v0 on those that all see
uint32_t seen_tiles(uint32_t pos0, uint32_t pos1, uint32_t window, uint32_t sinks, uint32_t v0, uint32_t n, uint32_t* tiles, uint32_t* numbers, uint32_t* full) {
    const step::Seen s(pos0, pos1, window, sinks);
    for (uint32_t v = 0; v < s.tiles; v++) {
        tiles[v] = s.tile(v);
        numbers[v] = s.number(s.tile(v));
    }
    s.full(pos0, pos1, window, v0, n, full[0], full[1]);
    return s.tiles;
}
int any(uint32_t pos0, uint32_t pos1, uint32_t window, uint32_t sinks, uint32_t t) { return step::Seen(pos0, pos1, window, sinks).any(t); }
int window_of(uint32_t rows, uint32_t seqs, uint32_t h, uint32_t hk, uint32_t d, uint32_t most, uint32_t n, uint32_t w, uint32_t s, uint64_t* o) {
    step::WindowPlan p;
    if (!step::window_plan(rows, seqs, h, hk, d, most, n, w, s, p)) return 0;
    const uint64_t v[] = {p.each, p.dim64, p.tiles, p.cols, p.score_cols, p.score_chunks, p.exp_cols, p.exp_chunks, p.value_cols, p.value_chunks, p.groups, p.packed, p.steps,
                          p.all_cols, p.splits, p.at_scores, p.at_exp, p.at_max, p.at_sum, p.at_factors, p.at_part, p.at_keys, p.at_values, p.at_queries, p.at_over,
                          p.at_query_over, p.bytes};
    std::memcpy(o, v, sizeof v);
    return 1;
}
// every field of the structs, in the order in which the helpers pack them
void pages_fields(const grape_wit_page_step_args* a, int64_t* o) {
    const int64_t v[] = {(int64_t)a->d_lens, (int64_t)a->d_new, (int64_t)a->d_span, (int64_t)a->d_block_table, (int64_t)a->d_free, (int64_t)a->d_starts, (int64_t)a->d_positions,
                         (int64_t)a->d_slots, (int64_t)a->d_lens_out, (int64_t)a->d_span_out, a->seqs, a->table_stride, a->ring, a->rows, a->page_size, a->window, a->sinks, a->reserved};
    std::memcpy(o, v, sizeof v);
}
void window_fields(const grape_wit_window_attention_args* a, int64_t* o) {
    const int64_t v[] = {(int64_t)a->d_q, a->q_stride, (int64_t)a->d_block_table, (int64_t)a->d_starts, (int64_t)a->d_lens, (int64_t)a->d_exp_table, (int64_t)a->d_scores,
                         (int64_t)a->d_scores_rem, (int64_t)a->d_shifted, (int64_t)a->d_exp, (int64_t)a->d_prob, (int64_t)a->d_query, (int64_t)a->d_max, (int64_t)a->d_sum,
                         (int64_t)a->d_out, (int64_t)a->d_out_rem, (int64_t)a->d_workspace, (int64_t)a->workspace_bytes, a->qk_scale, a->prob_scale, a->out_scale, a->rows,
                         a->seqs, a->heads, a->max_new, a->max_len, a->table_stride, a->window, a->sinks, a->bit_shift, a->index_bits};
    std::memcpy(o, v, sizeof v);
}
void next_fields(const grape_wit_next_token_args* a, int64_t* o) {
    const int64_t v[] = {(int64_t)a->d_logits, (int64_t)a->d_history, (int64_t)a->d_history_lens, (int64_t)a->d_repetition, (int64_t)a->d_presence, (int64_t)a->d_frequency,
                         (int64_t)a->d_bias, (int64_t)a->d_mask, (int64_t)a->d_out, (int64_t)a->d_rem, (int64_t)a->d_count, (int64_t)a->d_gap, (int64_t)a->d_token, (int64_t)a->d_max,
                         (int64_t)a->d_workspace, (int64_t)a->workspace_bytes, a->logits_stride, a->history_stride, a->bias_stride, a->mask_stride, a->scale, a->seqs, a->vocab,
                         a->history, a->reserved};
    std::memcpy(o, v, sizeof v);
}
}

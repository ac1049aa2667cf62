// Host build of grape_amd/csrc/token_geometry.hpp: which calls are refused, which positions a sequence attends to, where a
// page's tokens stand, and the argument structs as the Python helpers pack them.
#include <cstring>
#include "../../grape_amd/csrc/token_geometry.hpp"
using namespace grape;

extern "C" {
const char* refuse_append(const grape_wit_rope_append_args* a, const grape_wit_cache* c) { return token::refuse_append(a, c); }
const char* refuse_attention(const grape_wit_attention_args* a, const grape_wit_cache* c) { return token::refuse_attention(a, c); }
const char* refuse_q4(const void* q, const void* x, int64_t xs, const void* w, int64_t ws, const void* sc, uint32_t n, uint32_t m, uint32_t k, uint32_t g, int64_t s,
                      const void* sp, size_t sb) {
    return token::refuse_q4(q, x, xs, w, ws, sc, n, m, k, g, s, sp, sb);
}
size_t struct_bytes(int which) { return which == 0 ? sizeof(grape_wit_cache) : which == 1 ? sizeof(grape_wit_rope_append_args) : sizeof(grape_wit_attention_args); }
int overlaps(const grape_wit_cache* c) { return token::cache_overlaps(*c); }
int span(int32_t len, int32_t first, uint32_t max_len, uint32_t stride, uint32_t page, uint32_t* out) {
    return token::live_span(len, first, max_len, stride, page, out[0], out[1]);
}
int64_t offset_of(const grape_wit_cache* c, int32_t page, uint32_t in_page) { return token::token_offset(*c, page, in_page); }
int kind(const grape_wit_cache* c, int64_t slot, int32_t pos, uint32_t rot, uint32_t rows) { return token::append_kind(*c, slot, pos, rot, rows); }
size_t q4_workspace(uint32_t n, uint32_t m, uint32_t k, uint32_t g) { return token::q4_workspace(n, m, k, g); }
size_t workspace(uint32_t s, uint32_t h, uint32_t hk, uint32_t d, uint32_t n) { return token::attention_workspace(s, h, hk, d, n); }
uint32_t divided(uint32_t n, uint32_t d) { return token::fast_div(d)(n); }
// the parts of a plan that bound what the kernels touch
int plan_of(uint32_t s, uint32_t h, uint32_t hk, uint32_t d, uint32_t n, uint64_t* o) {
    token::AttentionPlan p;
    if (!token::attention_plan(s, h, hk, d, n, p)) return 0;
    const uint64_t v[] = {p.dim64, p.rows, p.tiles, p.score_chunk, p.score_chunks, p.exp_chunk, p.exp_chunks, p.blocks, p.groups, p.value_chunk, p.value_chunks,
                          p.at_scores, p.at_exp, p.at_max, p.at_sum, p.at_part, p.bytes, p.whole, p.whole_lds};
    std::memcpy(o, v, sizeof v);
    return 1;
}
int counted(uint32_t s, uint32_t h, uint32_t hk, uint32_t d, uint32_t n) {
    token::AttentionPlan p;
    return token::attention_plan(s, h, hk, d, n, p) ? p.counted : -1;
}
// every field of the structs, in the order in which the helpers pack them
void append_fields(const grape_wit_rope_append_args* a, int64_t* o) {
    const int64_t v[] = {(int64_t)a->d_q, (int64_t)a->d_k, (int64_t)a->d_v, a->q_stride, a->k_stride, a->v_stride, (int64_t)a->d_positions, (int64_t)a->d_slots,
                         (int64_t)a->d_cos, (int64_t)a->d_sin, (int64_t)a->d_q_out, (int64_t)a->d_q_rem, (int64_t)a->d_k_rem, a->tokens, a->heads, a->rot,
                         a->table_rows, a->scale, a->interleaved, a->reserved};
    std::memcpy(o, v, sizeof v);
}
void attention_fields(const grape_wit_attention_args* a, int64_t* o) {
    const int64_t v[] = {(int64_t)a->d_q, a->q_stride, (int64_t)a->d_block_table, (int64_t)a->d_lens, (int64_t)a->d_first, (int64_t)a->d_exp_table, (int64_t)a->d_scores,
                         (int64_t)a->d_scores_rem, (int64_t)a->d_shifted, (int64_t)a->d_exp, (int64_t)a->d_prob, (int64_t)a->d_query, (int64_t)a->d_max, (int64_t)a->d_sum,
                         (int64_t)a->d_out, (int64_t)a->d_out_rem, (int64_t)a->d_workspace, (int64_t)a->workspace_bytes, a->qk_scale, a->prob_scale, a->out_scale, a->seqs,
                         a->heads, a->max_len, a->table_stride, a->bit_shift, a->index_bits};
    std::memcpy(o, v, sizeof v);
}
void cache_fields(const grape_wit_cache* c, int64_t* o) {
    const int64_t v[] = {(int64_t)c->d_k, (int64_t)c->d_v, c->pages, c->page_size, c->heads, c->dim, c->page_stride, c->token_stride, c->head_stride};
    std::memcpy(o, v, sizeof v);
}
}

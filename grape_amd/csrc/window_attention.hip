// Attention of several new tokens a sequence over a paged cache - in their order, or behind a sliding window and a few first tokens -
// with the tensors that a proof of it looks up.
#include <algorithm>
#include <type_traits>
#include "token_device.hpp"
#include "step_geometry.hpp"
#include "token_attention.hpp"

namespace grape {

// ------------------------------------------------------------------------------------------------
// Scores, softmax through the table, products with the values, for tiles of 32 rows: the query heads that read one cache head, token
// after token, so that a key or a value that is read serves 32 rows.  The softmax is the table's, rounded: the row's maximum is
// needed before the first exponential and the sum of all before the first probability, hence a launch for each of the three, and
// a fourth that joins the values' partial sums where the positions are cut up.  Rows of 32 are two operands of a product for each key
// that is loaded; 16 would read keys and values twice as often, 64 leave no registers for the five sums of the planes' products.
//
// 2048 new tokens, 32 heads of 128 over 8, with a proof (1.68 GB written, 0.54 GB of it read again): 47 us operands, 158 scores, 209
// exponentials, 246 values, each of the last three near what it writes and reads at 3.4 to 3.9 TB/s.  One head of 4096: 63 + 113-117 + 18 + 139-144 us; its products alone
// would take 103 at the 2.5 POP/s that the kernel of a large int8 product reaches.  5 drafted tokens of 8 sequences of up to 3000: 35 + 15 + 39 + 5 us, chains of
// dependent loads in short workgroups; a fourth wave of registers (128 of them) or other chunks are no faster.
//
// Both products run on the int8 matrix cores, exactly.  An element of magnitude below 2^23 is three balanced digits of base 256, the bytes
// of x + 0x808080 with their top bits turned over, nine products of planes for a pair of operands and six where the probabilities
// are small; pairs with the same sum of exponents share an accumulator (3 * 2^14 * 8192 elements stay below 2^31).  Where a larger
// element turns up, positions are taken again with x - c, c = 128 (1 + 2^8 + 2^16), whose four digits are the bytes of x with the
// three lower top bits turned over: sum q k = sum (q-c)(k-c) + c (sum (q-c) + sum (k-c)) + c^2 dim.  For a large key these are the sixteen
// positions that its wave takes of each tile of the chunk; with operands made beforehand, or for a large query, all of the chunk; for a large value the
// workgroup's whole chunk.  That is meant to be right, not fast: its operands come element by element with nothing under way.  The 2048 tokens
// above take 655 us without a large element, 2139 with one key, 2454 with one key in a hundred, 769 with one value and 804 with one in a hundred; one head of
// 4096 311, 745, 1664, 440 and 503; five drafted tokens 76, 107, 178, 88 and 93 (each time with the same inputs again and again).
// ------------------------------------------------------------------------------------------------
using step::kCols;
using step::kRows;
constexpr uint32_t kNoElement = 0x00808080;          // whose four digits are all zero
constexpr uint32_t kThreeDigits = 0x00808080;        // added to an element, leaves 24 bits of it where three digits hold it
typedef int v4u_t __attribute__((ext_vector_type(4), aligned(4)));

// rows of a tensor of the proof, or of the workspace, which holds the tiles that are seen side by side
struct Rows {
    int32_t* base;
    size_t stride;
    bool dense;
    __device__ __forceinline__ int32_t* at(size_t row, uint32_t t, uint32_t v) const { return base + row * stride + (dense ? t : v * kCols + t % kCols); }
};

struct WindowArgs {
    grape_wit_window_attention_args a;
    grape_wit_cache c;
    step::WindowPlan plan;
    token::FastDiv page, by_each;
    Scaler qk, out;
    Rows scores, exps;
    int32_t* chunk_max;          // [rows][heads][score chunks]
    unsigned long long* sums;    // [rows][heads]
    int64_t* part;               // [rows][heads][value chunks][dim]
    uint32_t* status;
    bool q_vec, k_vec;           // rows of the queries and of the keys that can be read by four elements
    double limit;                // of a score's product that is rescaled in double precision
    uint32_t along;              // workgroups of a launch's first axis
    double* factors;             // of the exponential table, see make_factors; null where it is read
    uint32_t* differs;
    // operands made beforehand (see wit_window_pack_kernel), and whether an element did not fit
    uint8_t *keys, *values, *queries;
    uint32_t *over, *query_over;
    __device__ __forceinline__ size_t tile_of(uint32_t b, uint32_t kv, uint32_t number) const { return ((size_t)b * c.heads + kv) * plan.all_cols + number; }
};

// the three planes of four elements; `over` gathers bits above the 24
__device__ __forceinline__ void three_planes(v4i_t x, uint32_t out[3], uint32_t& over) {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = (uint32_t)x[j] + kThreeDigits;
    over |= (u[0] | u[1]) | (u[2] | u[3]);
    const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(u[1], u[0], 0x07030602u), d = __builtin_amdgcn_perm(u[3], u[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ kByteTops;
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u) ^ kByteTops;
    out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u) ^ kByteTops;
}
constexpr uint32_t kOver = 0xff000000;

// the four planes of x - kCacheOffset
__device__ __forceinline__ void four_planes(v4i_t x, uint32_t out[4]) {
    transpose4((uint32_t)x[0], (uint32_t)x[1], (uint32_t)x[2], (uint32_t)x[3], out);
#pragma unroll
    for (int k = 0; k < 3; k++) out[k] ^= kByteTops;
}

// A workgroup's rows: rows `at` .. + R of the cache head kv of sequence b, whose n new tokens start at row `first` and position
// `pos`.  Row r is query head r % each of token r / each.  Where there are fewer than kRows, the last one stands in for those that are
// missing: what is written for it is written several times, and the same.
struct RowTile {
    uint32_t b, kv, first, n, pos, at, R, first_pos, last_pos;
    uint32_t lane, wave, col, kg;
    __device__ __forceinline__ bool find(const WindowArgs& p, uint32_t index) {
        lane = threadIdx.x & 63u;
        wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        col = lane & 15u;
        kg = lane >> 4;
        // the heads of one tile are neighbours, so that each die's L2 gets the keys of its own heads where there are eight; long rows first
        kv = index % p.c.heads;
        const uint32_t ti = p.plan.tiles - 1 - index / p.c.heads;
        auto ballot = [&](auto f) { return __ballot(f(lane)); };
        b = step::search_tile(p.a.d_starts, p.a.seqs, p.a.rows, p.plan.each, ti, ballot);
        int32_t s = p.a.d_starts[b], e = p.a.d_starts[b + 1], len = p.a.d_lens[b];
        if (!step::has_rows(s, e, p.a.rows)) {
            b = step::scan_for_tile(p.a.d_starts, p.a.seqs, p.a.rows, p.plan.each, ti, ballot);
            s = p.a.d_starts[b];
            e = p.a.d_starts[b + 1];
            len = p.a.d_lens[b];
        }
        if (!step::new_tokens(s, e, len, p.a.rows, p.a.max_new, p.a.max_len, (uint64_t)p.a.table_stride * p.c.page_size, n, pos)) return false;
        first = (uint32_t)s;
        const uint64_t base = step::first_tile(s, b, p.plan.each);
        if (ti < base) return false;
        const uint64_t local = (uint64_t)(ti - base) * kRows, all = (uint64_t)n * p.plan.each;
        if (local >= all) return false;
        at = (uint32_t)local;
        R = (uint32_t)min((uint64_t)kRows, all - local);
        first_pos = pos_of(p, 0);
        last_pos = pos_of(p, R - 1);
        return true;
    }
    __device__ __forceinline__ uint32_t token(const WindowArgs& p, uint32_t r) const { return p.by_each(at + r); }
    __device__ __forceinline__ uint32_t pos_of(const WindowArgs& p, uint32_t r) const { return pos + token(p, r); }
    __device__ __forceinline__ size_t row(const WindowArgs& p, uint32_t r) const {
        const uint32_t j = token(p, r);
        return (size_t)(first + j) * p.a.heads + kv * p.plan.each + (at + r - j * p.plan.each);
    }
    // what all of the sequence's rows see, by which the operands made beforehand are numbered
    __device__ __forceinline__ step::Seen all_seen(const WindowArgs& p) const { return step::Seen(pos, pos + n - 1, p.a.window, p.a.sinks); }
    __device__ __forceinline__ step::Seen seen(const WindowArgs& p) const { return step::Seen(first_pos, last_pos, p.a.window, p.a.sinks); }
    // the tiles first <= v < last of v0 .. v0 + n whose positions all rows see
    __device__ __forceinline__ void full(const WindowArgs& p, const step::Seen& seen, uint32_t v0, uint32_t n, uint32_t& first, uint32_t& last) const {
        seen.full(first_pos, last_pos, p.a.window, v0, n, first, last);
    }
};

// Offset of position t's token; of the last one that is seen where no row sees t, so that nothing is read but what is there.  -1 where the
// page is outside the cache.
__device__ __forceinline__ int64_t offset_of(const WindowArgs& p, uint32_t b, const step::Seen& seen, uint32_t t) {
    if (!seen.any(t)) t = seen.hi - 1;
    const uint32_t pg = p.page(t);
    return token::token_offset(p.c, p.a.d_block_table[(size_t)b * p.a.table_stride + pg], t - pg * p.c.page_size);
}

// The queries' digits of a block of 512 elements in LDS, [step of 64][plane][lane group][row], 16 bytes each.
constexpr uint32_t kBlockSteps = 8, kHalfQuads = kBlockSteps / 2 * step::kQueryStepBytes / 16 / 256;
__device__ __forceinline__ const int32_t* query_of(const WindowArgs& p, const RowTile& w, uint32_t r) {
    const uint32_t tok = w.token(p, r);
    return p.a.d_q + (int64_t)(w.first + tok) * p.a.q_stride + (size_t)(w.kv * p.plan.each + (w.at + r - tok * p.plan.each)) * p.c.dim;
}
// four elements of a row, `pad` where there is none
__device__ __forceinline__ v4i_t elements(const int32_t* x, uint32_t e, uint32_t dim, bool vec, int32_t pad) {
    v4i_t y = {pad, pad, pad, pad};
    if (vec) {
        if (e < dim) y = *reinterpret_cast<const v4i_t*>(x + e);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
            if (e + j < dim) y[j] = x[e + j];
    }
    return y;
}
__device__ __forceinline__ void stage_queries(const WindowArgs& p, const RowTile& w, uint32_t block, uint32_t* digits, uint32_t& over) {
    const uint32_t steps = min(p.plan.dim64 - kBlockSteps * block, kBlockSteps), e0 = 64 * kBlockSteps * block;
    for (uint32_t i = threadIdx.x; i < kRows * steps * 16; i += blockDim.x) {
        const uint32_t r = i / (steps * 16), quad = i - r * (steps * 16), s = quad >> 4, c = (quad >> 2) & 3u, g = quad & 3u;
        const v4i_t x = elements(query_of(p, w, min(r, w.R - 1)), e0 + 4 * quad, p.c.dim, p.q_vec, 0);
        uint32_t pl[3];
        three_planes(x, pl, over);
        uint32_t* o = digits + (((s * 3 * 4 + g) * kRows + r) << 2) + c;
#pragma unroll
        for (uint32_t k = 0; k < 3; k++) o[k * 16 * kRows] = pl[k];
    }
}

__device__ __forceinline__ uint32_t seen_of_four(const WindowArgs& p, uint32_t pos, uint32_t t) {
    uint32_t there = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) there |= step::sees(pos, t + i, p.a.window, p.a.sinks) ? 1u << i : 0u;
    return there;
}
// Four elements of a tensor of the proof that no later launch of the call reads, which then does not push out of the caches what the next one does.
__device__ __forceinline__ void store_last(int32_t* to, v4u_t x) { __builtin_nontemporal_store(x, reinterpret_cast<v4u_t*>(to)); }
__device__ __forceinline__ void store_four(int32_t* to, v4u_t x, uint32_t there) {
    if (there == 15u) {
        *reinterpret_cast<v4u_t*>(to) = x;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
            if ((there >> i) & 1u) to[i] = x[i];
    }
}

// The scores of a wave's positions with operands of any size, both from memory: sixteen rows at a time, four planes each.
__device__ __forceinline__ void wide_scores(const WindowArgs& p, const RowTile& w, const step::Seen& seen, uint32_t v0, uint32_t tiles, int32_t mx[2], uint32_t& bad) {
    const int32_t* keys = p.c.d_k + (int64_t)w.kv * p.c.head_stride;
    const uint32_t dim = p.c.dim;
#pragma unroll 1
    for (uint32_t tile = 0; tile < tiles; tile++) {
        const uint32_t in_tile = 16 * w.wave + 4 * w.kg, v = v0 + tile, t0 = seen.tile(v) * kCols + in_tile;
        const int64_t k_off = offset_of(p, w.b, seen, seen.tile(v) * kCols + 16 * w.wave + w.col);
        const int32_t* k_row = keys + max(k_off, (int64_t)0);
#pragma unroll 1
        for (uint32_t rb = 0; 16 * rb < w.R; rb++) {
            const uint32_t r = min(16 * rb + w.col, w.R - 1);
            const int32_t* q_row = query_of(p, w, r);
            v4i_t acc[7];
            int32_t k_dot[4] = {0, 0, 0, 0}, q_dot[4] = {0, 0, 0, 0};          // sums of the planes of this lane's parts
#pragma unroll
            for (int g = 0; g < 7; g++) acc[g] = v4i_t{0, 0, 0, 0};
#pragma unroll 1
            for (uint32_t s = 0; s < p.plan.dim64; s++) {
                v4i_t kb[4], qb[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint32_t e = 64 * s + 16 * c + 4 * w.kg;
                    uint32_t pl[4];
                    four_planes(elements(k_row, e, dim, false, (int32_t)kNoElement), pl);
#pragma unroll
                    for (int k = 0; k < 4; k++) kb[k][c] = (int)pl[k];
                    four_planes(elements(q_row, e, dim, false, (int32_t)kNoElement), pl);
#pragma unroll
                    for (int k = 0; k < 4; k++) qb[k][c] = (int)pl[k];
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        k_dot[k] = __builtin_amdgcn_sdot4(kb[k][c], 0x01010101, k_dot[k], false);
                        q_dot[k] = __builtin_amdgcn_sdot4(qb[k][c], 0x01010101, q_dot[k], false);
                    }
#pragma unroll
                    for (int a = 0; a < 4; a++) acc[a + k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kb[k], qb[a], acc[a + k], 0, 0, 0);
                }
            }
            int64_t k_sum = 0, q_sum = 0;
#pragma unroll
            for (int k = 3; k >= 0; k--) {
                k_sum = k_sum * 256 + k_dot[k];
                q_sum = q_sum * 256 + q_dot[k];
            }
#pragma unroll
            for (int d = 16; d <= 32; d <<= 1) {
                k_sum += __shfl_xor(k_sum, d, 64);
                q_sum += __shfl_xor(q_sum, d, 64);
            }
            const uint32_t there = 16 * rb + w.col < w.R ? seen_of_four(p, w.pos_of(p, r), t0) : 0;
            v4u_t q, rem;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const int64_t k_of = __shfl(k_sum, (int)(4 * w.kg + i), 64);
                uint64_t y = 0;
#pragma unroll
                for (int g = 6; g >= 0; g--) y = (y << 8) + (uint64_t)(int64_t)acc[g][i];
                y += (uint64_t)kCacheOffset * (uint64_t)(k_of + q_sum + kCacheOffset * dim);
                uint32_t wide = 0;
                int32_t qi, ri;
                p.qk.apply(__shfl(k_off < 0 ? 1 : 0, (int)(4 * w.kg + i), 64) ? 0 : (int64_t)y, qi, ri, wide);          // a page outside: zero
                q[i] = qi;
                rem[i] = ri;
                if ((there >> i) & 1u) {
                    bad |= wide;
                    if (rb == 0) mx[0] = max(mx[0], qi);
                    else mx[1] = max(mx[1], qi);
                }
            }
            const size_t row = w.row(p, r);
            store_four(p.scores.at(row, t0, v), q, there);
            if (p.a.d_scores_rem) store_four(p.a.d_scores_rem + row * p.a.max_len + t0, rem, there);
        }
    }
}

// A table of exponentials need not be looked into where it is one: entry 2^bit_shift - 1 - d is then round(S exp(-d / S)) with S the
// entry of d = 0.  Written as d = 1024 a + b that is the product of two factors of a thousand each, 16 KB in all, which LDS holds.  These
// workgroups make the factors and compare every entry that a score can meet; where one differs, the entries are read.  That pays from the smallest
// calls on, since it runs beside another launch: 2 new tokens behind 64 positions 24 us either way, 64 behind 1000 (32 heads) 67 us, and 75 read.
constexpr uint32_t kFactors = 1024, kTableGroups = 64;
__device__ __forceinline__ void make_factors(const WindowArgs& p, uint32_t group, double* factors, uint32_t& differs) {
    const uint32_t last = ((uint32_t)1 << p.a.bit_shift) - 1;
    const int32_t top = p.a.d_exp_table[last];
    const double scale = (double)max(top, 1);
    if (threadIdx.x == 0) differs = top < 1;
    for (uint32_t i = threadIdx.x; i < kFactors; i += kBlock) {
        factors[i] = scale * exp(-(double)(i * kFactors) / scale);
        factors[kFactors + i] = exp(-(double)i / scale);
    }
    __syncthreads();
    const uint32_t each = last / kTableGroups + 1, from = group * each, to = min(from + each, last + 1);
    bool other = false;
#pragma unroll 8
    for (uint32_t d = from + threadIdx.x; d < to; d += kBlock) other |= p.a.d_exp_table[last - d] != (int32_t)__builtin_rint(factors[d / kFactors] * factors[kFactors + d % kFactors]);
    if (other) differs = 1;
    __syncthreads();
    if (threadIdx.x == 0) p.differs[group] = differs;
    if (group == 0)
        for (uint32_t i = threadIdx.x; i < 2 * kFactors; i += kBlock) p.factors[i] = factors[i];
}

// Loads of the next positions are issued before this one's stores, so that waiting for them does not wait for the stores; the compiler can
// count on that where every way to the wait has the same number of stores behind the loads.  Tiles that all rows see in full therefore have a
// loop of their own, nothing is under way when it begins, and the other tiles wait for everything in the end.
__device__ __forceinline__ void wait_for_memory() { __builtin_amdgcn_s_waitcnt(0x0f70); }          // vmcnt 0

// The operands of a call with many rows, made once: turning an element into digits costs as much as its products with 32 rows.  Keys of a
// tile of 64 positions: [step][plane][16 positions][lane group][position], queries of a tile of rows: [step][plane][lane group][row], values of a
// tile of 64 positions: [16 elements][plane][lane group][element] - 16 bytes each, what a lane of a product takes.  Positions that nobody sees and
// pages outside the cache are zero.  A workgroup takes 256 elements.  2048 tokens, 40 + 8 heads of 128: 46 us for 64 MB, bound by the chain of
// starts, lengths, pages and elements in one round of workgroups (queries alone 24); with it scores go from 239 to 158 us, values from 319 to 248.
__global__ void __launch_bounds__(256) wit_window_pack_kernel(WindowArgs p) {
    __shared__ double factors[2 * kFactors];
    __shared__ int64_t off[kCols];
    __shared__ uint32_t word[2];
    uint32_t index = blockIdx.x, bad = 0;
    if (p.factors) {
        if (index < kTableGroups) return make_factors(p, index, factors, word[0]);
        index -= kTableGroups;
    }
    if (threadIdx.x < 2) word[threadIdx.x] = 0;
    const uint32_t dim = p.c.dim;
    uint32_t over = 0;
    const uint32_t split = index % p.plan.splits, s0 = split * step::kPackSteps;
    index /= p.plan.splits;
    if (index < p.along) {
        RowTile w;
        if (!w.find(p, index)) return;
        __syncthreads();
        const uint32_t g = threadIdx.x & 3u, r = (threadIdx.x >> 2) % kRows;          // two steps at a time
        const int32_t* q = query_of(p, w, min(r, w.R - 1));
        uint8_t* to = p.queries + (size_t)index * p.plan.steps * step::kQueryStepBytes + (g * kRows + r) * 16;
        for (uint32_t s = s0 + threadIdx.x / (4 * kRows); s < min(s0 + step::kPackSteps, p.plan.steps); s += 2) {
            uint32_t pl[4][3];
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) three_planes(elements(q, 64 * s + 16 * c + 4 * g, dim, p.q_vec, 0), pl[c], over);
#pragma unroll
            for (uint32_t k = 0; k < 3; k++)
                *reinterpret_cast<v4i_t*>(to + (s * 3 + k) * 64 * kRows) = v4i_t{(int)pl[0][k], (int)pl[1][k], (int)pl[2][k], (int)pl[3][k]};
        }
        if (over & kOver) word[0] = 1;
        __syncthreads();
        if (threadIdx.x == 0) p.query_over[(size_t)index * p.plan.splits + split] = word[0];
        return;
    }
    index -= p.along;
    const uint32_t kv = index % p.c.heads, rest = index / p.c.heads, number = rest % p.plan.all_cols, b = rest / p.plan.all_cols;
    uint32_t n, pos;
    if (!step::new_tokens(p.a.d_starts[b], p.a.d_starts[b + 1], p.a.d_lens[b], p.a.rows, p.a.max_new, p.a.max_len, (uint64_t)p.a.table_stride * p.c.page_size, n, pos) || n == 0) return;
    const step::Seen seen(pos, pos + n - 1, p.a.window, p.a.sinks);
    if (number >= seen.tiles) return;
    const uint32_t k0 = seen.tile(number) * kCols;
    if (threadIdx.x < kCols) {
        const uint32_t t = k0 + threadIdx.x;
        const int64_t o = seen.any(t) ? offset_of(p, b, seen, t) : -2;
        if (o == -1) bad |= (uint32_t)kWitIndex;
        off[threadIdx.x] = o;
    }
    __syncthreads();
    const size_t at = p.tile_of(b, kv, number);
    {
        const uint32_t key = threadIdx.x >> 2, g = threadIdx.x & 3u;
        const int64_t o = off[key];
        const int32_t* k = p.c.d_k + (int64_t)kv * p.c.head_stride + max(o, (int64_t)0);
        uint8_t* to = p.keys + at * p.plan.steps * step::kKeyStepBytes + (((key >> 4) * 4 + g) * 16 + (key & 15u)) * 16;
        for (uint32_t s = s0; s < min(s0 + step::kPackSteps, p.plan.steps); s++) {
            uint32_t pl[4][3];
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) {
                v4i_t x = {0, 0, 0, 0};
                if (o >= 0) x = elements(k, 64 * s + 16 * c + 4 * g, dim, p.k_vec, 0);
                three_planes(x, pl[c], over);
            }
#pragma unroll
            for (uint32_t j = 0; j < 3; j++)
                *reinterpret_cast<v4i_t*>(to + (size_t)(s * 3 + j) * kCols * 64) = v4i_t{(int)pl[0][j], (int)pl[1][j], (int)pl[2][j], (int)pl[3][j]};
        }
        if (over & kOver) word[0] = 1;
    }
    over = 0;
    {
        const uint32_t g = threadIdx.x >> 6;
        const int32_t* values = p.c.d_v + (int64_t)kv * p.c.head_stride;
        uint8_t* to = p.values + at * p.plan.dim64 * step::kValueStepBytes;
        for (uint32_t s = s0; s < min(s0 + step::kPackSteps, p.plan.dim64); s++) {
            const uint32_t e = 64 * s + (threadIdx.x & 63u);
            int32_t x[16];
#pragma unroll
            for (uint32_t j = 0; j < 16; j++) {
                const int64_t o = off[16 * g + j];
                x[j] = o >= 0 && e < dim ? values[o + e] : 0;
            }
            uint32_t pl[4][3];
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) three_planes(v4i_t{x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]}, pl[c], over);
#pragma unroll
            for (uint32_t k = 0; k < 3; k++)
                *reinterpret_cast<v4i_t*>(to + ((size_t)((e >> 4) * 3 + k) * 64 + g * 16 + (e & 15u)) * 16) = v4i_t{(int)pl[0][k], (int)pl[1][k], (int)pl[2][k], (int)pl[3][k]};
        }
        if (over & kOver) word[1] = 1;
    }
    __syncthreads();
    if (threadIdx.x == 0) p.over[at * p.plan.splits + split] = word[0] | word[1] << 1;
    if (bad) atomicOr(p.status, bad);
}

// Scores of 32 rows with a chunk of the positions.  A wave takes 16 positions of each tile of 64 and all rows.  Its keys come as operands
// (PACKED), or from the cache into the operand (lane l the elements 64 s + 16 c + 4 (l / 16) .. + 4 of position l % 16); the queries' digits from LDS.
// Five accumulators become a sum in double precision, exact below 2^53, and below 2^50 the quotient of (y + s/2 + 1/2) / s needs no
// second look: it is no nearer than 1 / (2 s) to a whole number, and the product with 1 / s off by at most 2^-52 of itself.
// Bound by vector instructions and stores together where a proof is made (the 2048 tokens above: 158 us, 3.7 TB/s); heads of 4096 reach 1.4 POP/s of
// the 2.5 that a large int8 product does, by 1.05e7 requests of L2, up to 1.3 GB (113 us; 130 when a block of queries was loaded between two barriers and not beside the products).
template <bool PACKED, bool VEC, bool REM>
__global__ void __launch_bounds__(256, 2) wit_window_scores_kernel(WindowArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ int32_t top[4][kRows];
    __shared__ uint32_t q_over;
    uint32_t bad = 0;
    if (!PACKED && blockIdx.x >= p.along) {
        if (blockIdx.y == 0) make_factors(p, blockIdx.x - p.along, reinterpret_cast<double*>(lds), q_over);
        return;
    }
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        uint32_t n, pos;
        for (uint32_t b = threadIdx.x; b < p.a.seqs; b += 256)
            if (!step::new_tokens(p.a.d_starts[b], p.a.d_starts[b + 1], p.a.d_lens[b], p.a.rows, p.a.max_new, p.a.max_len, (uint64_t)p.a.table_stride * p.c.page_size, n, pos))
                atomicOr(p.status, (uint32_t)kWitIndex);
    }
    RowTile w;
    if (!w.find(p, blockIdx.x)) return;
    const step::Seen seen = w.seen(p);
    const step::Seen made = w.all_seen(p);
    const uint32_t v0 = blockIdx.y * p.plan.score_cols;
    if (v0 >= seen.tiles) return;
    const uint32_t tiles = min(p.plan.score_cols, seen.tiles - v0), steps = PACKED ? p.plan.steps : p.plan.dim64, dim = p.c.dim, blocks = (steps + kBlockSteps - 1) / kBlockSteps;
    int64_t* off = reinterpret_cast<int64_t*>(lds + (size_t)min(steps, kBlockSteps) * 3 * 4 * kRows * 4);
    if (threadIdx.x == 0) q_over = 0;
    bool outside = false;
    if constexpr (PACKED) {
        __syncthreads();
        bool over = false;
        for (uint32_t i = threadIdx.x; i < tiles * p.plan.splits; i += 256) over |= p.over[p.tile_of(w.b, w.kv, made.number(seen.tile(v0 + i / p.plan.splits))) * p.plan.splits + i % p.plan.splits] & 1u;
        for (uint32_t i = threadIdx.x; i < p.plan.splits; i += 256) over |= p.query_over[(size_t)blockIdx.x * p.plan.splits + i] != 0;
        if (over) q_over = 1;
    } else {
        for (uint32_t i = threadIdx.x; i < tiles * kCols; i += 256) {
            const int64_t o = offset_of(p, w.b, seen, seen.tile(v0 + i / kCols) * kCols + i % kCols);
            outside |= o < 0;
            off[i] = max(o, (int64_t)0);
        }
        if (outside) bad |= (uint32_t)kWitIndex;
    }
    if (blockIdx.y == 0 && threadIdx.x < w.R) p.sums[w.row(p, threadIdx.x)] = 0;
    uint32_t over = 0;
    auto stage = [&](uint32_t block) {
        if constexpr (PACKED) {
            const uint32_t n = steps * (uint32_t)(step::kQueryStepBytes / 16);
            const v4i_t* from = reinterpret_cast<const v4i_t*>(p.queries + (size_t)blockIdx.x * steps * step::kQueryStepBytes);
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < n; i += 256) reinterpret_cast<v4i_t*>(lds)[i] = from[i];
        } else {
            stage_queries(p, w, block, lds, over);
        }
    };
    __syncthreads();
    if (blocks == 1) {
        stage(0);
        __syncthreads();
    }
    const v4i_t* q_digits = reinterpret_cast<const v4i_t*>(lds) + w.kg * kRows + w.col;
    // PACKED, of more steps than LDS holds: half of what it holds at a time, in turn; the next half is under way while one is used
    v4i_t under_way[kHalfQuads];
    uint32_t turn = 0;
    auto request_half = [&](uint32_t s) {
        const uint32_t n = min(steps - s, kBlockSteps / 2) * (uint32_t)(step::kQueryStepBytes / 16);
        const v4i_t* from = reinterpret_cast<const v4i_t*>(p.queries + ((size_t)blockIdx.x * steps + s) * step::kQueryStepBytes);
#pragma unroll
        for (uint32_t i = 0; i < kHalfQuads; i++) under_way[i] = from[min(threadIdx.x + 256 * i, n - 1)];
    };
    auto store_half = [&](uint32_t half) {
        v4i_t* to = reinterpret_cast<v4i_t*>(lds) + half * kHalfQuads * 256;
#pragma unroll
        for (uint32_t i = 0; i < kHalfQuads; i++) to[threadIdx.x + 256 * i] = under_way[i];
    };
    if (PACKED && blocks > 1) {
        request_half(0);
        store_half(0);
        __syncthreads();
    }
    // PACKED: operands of two steps, each next pair requested as the one before it has been used
    v4i_t x[4], keys[2][3];
    auto request = [&](int half, uint32_t tile, uint32_t s) {
        const uint8_t* from = p.keys + (p.tile_of(w.b, w.kv, made.number(seen.tile(v0 + tile))) * steps + s) * step::kKeyStepBytes + (w.wave * 64 + w.lane) * 16;
#pragma unroll
        for (int k = 0; k < 3; k++) keys[half][k] = *reinterpret_cast<const v4i_t*>(from + k * kCols * 64);
    };
    const int32_t* cache_keys = p.c.d_k + (int64_t)w.kv * p.c.head_stride;
    auto fetch = [&](uint32_t tile, uint32_t s) {
        const int32_t* k = cache_keys + off[tile * kCols + 16 * w.wave + w.col];
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) x[c] = elements(k, 64 * s + 16 * c + 4 * w.kg, dim, VEC, 0);
    };
    if constexpr (PACKED) {
        request(0, 0, 0);
        if (steps > 1) request(1, 0, 1);
    } else {
        fetch(0, 0);
    }
    int32_t mx[2] = {INT32_MIN, INT32_MIN};
    uint32_t pos[2];
    size_t row[2];
#pragma unroll
    for (uint32_t rb = 0; rb < 2; rb++) {
        const uint32_t r = min(16 * rb + w.col, w.R - 1);
        pos[rb] = w.pos_of(p, r);
        row[rb] = w.row(p, r);
    }
    const double scale = (double)p.qk.s, inv = p.qk.inv, half = (double)(p.qk.s >> 1) + 0.5, limit = p.limit;
    bool large = false;
    uint32_t k_over = 0;
    auto body = [&](uint32_t tile, auto all_see) {
        constexpr bool FULL = decltype(all_see)::value;
        v4i_t acc[2][5];
#pragma unroll
        for (int rb = 0; rb < 2; rb++)
#pragma unroll
            for (int g = 0; g < 5; g++) acc[rb][g] = v4i_t{0, 0, 0, 0};
        auto multiply = [&](const v4i_t (&kb)[3], uint32_t step) {
            v4i_t f[3][2];
#pragma unroll
            for (int a = 0; a < 3; a++)
#pragma unroll
                for (int rb = 0; rb < 2; rb++) f[a][rb] = q_digits[(step * 12 + a * 4) * kRows + 16 * rb];
#pragma unroll
            for (int a = 0; a < 3; a++)
#pragma unroll
                for (int k = 0; k < 3; k++)
#pragma unroll
                    for (int rb = 0; rb < 2; rb++) acc[rb][a + k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kb[k], f[a][rb], acc[rb][a + k], 0, 0, 0);
        };
        const uint32_t next_tile = min(tile + 1, tiles - 1);
        auto next_block = [&](uint32_t s) {
            if (blocks > 1 && s % kBlockSteps == 0) {
                __syncthreads();
                stage(s / kBlockSteps);
                __syncthreads();
            }
        };
        if constexpr (PACKED) {
            if (steps == 1) {
                multiply(keys[0], 0);
                request(0, next_tile, 0);
            } else {
                const bool halves = blocks > 1;
#pragma unroll 1
                for (uint32_t s = 0; s < steps; s += 2) {
                    const bool more = s + 2 < steps;
                    const uint32_t in_half = s % (kBlockSteps / 2), at = halves ? turn * (kBlockSteps / 2) + in_half : s;
                    if (halves && in_half == 0) request_half(s + kBlockSteps / 2 < steps ? s + kBlockSteps / 2 : 0);
                    multiply(keys[0], at);
                    request(0, more ? tile : next_tile, more ? s + 2 : 0);
                    multiply(keys[1], at + 1);
                    request(1, more ? tile : next_tile, more ? s + 3 : 1);
                    if (halves && (!more || in_half + 2 == kBlockSteps / 2)) {
                        turn ^= 1;
                        store_half(turn);
                        __syncthreads();
                    }
                }
            }
        } else {
#pragma unroll 1
            for (uint32_t s = 0; s < steps; s++) {
                next_block(s);
                v4i_t kb[3];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t pl[3];
                    three_planes(x[c], pl, k_over);
#pragma unroll
                    for (int k = 0; k < 3; k++) kb[k][c] = (int)pl[k];
                }
                fetch(s + 1 < steps ? tile : next_tile, s + 1 < steps ? s + 1 : 0);
                multiply(kb, s % kBlockSteps);
            }
        }
        // register i of lane l: position 4 (l / 16) + i of the wave's 16, row l % 16 of a block
        const uint32_t in_tile = 16 * w.wave + 4 * w.kg, v = v0 + tile, t0 = seen.tile(v) * kCols + in_tile;
#pragma unroll
        for (uint32_t rb = 0; rb < 2; rb++) {
            __builtin_amdgcn_sched_barrier(0);
            const uint32_t there = FULL ? 15u : seen_of_four(p, pos[rb], t0);
            v4u_t q, rem;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                double y;
                if (steps < 4) {          // two of the sums fit 32 bits: 2 * 2^14 * 192 * 2^8 + 2^14 * 192
                    const int32_t low = (acc[rb][1][i] << 8) + acc[rb][0][i], high = (acc[rb][4][i] << 8) + acc[rb][3][i];
                    y = __builtin_fma((double)high, 0x1p24, __builtin_fma((double)acc[rb][2][i], 0x1p16, (double)low));
                } else {
                    y = (double)acc[rb][4][i];
#pragma unroll
                    for (int g = 3; g >= 0; g--) y = __builtin_fma(y, 256.0, (double)acc[rb][g][i]);
                }
                const double t = y + half, quotient = __builtin_floor(t * inv);
                const bool here = (there >> i) & 1u;
                large |= here && __builtin_fabs(t) >= limit;
                q[i] = (int32_t)quotient;
                if constexpr (REM) rem[i] = (int32_t)__builtin_fma(-quotient, scale, y);
                mx[rb] = max(mx[rb], here ? q[i] : INT32_MIN);
            }
            int32_t* to = p.scores.at(row[rb], t0, v);
            if constexpr (FULL) *reinterpret_cast<v4u_t*>(to) = q;
            else store_four(to, q, there);
            if constexpr (REM) {
                int32_t* to_rem = p.a.d_scores_rem + row[rb] * p.a.max_len + t0;
                if constexpr (FULL) store_last(to_rem, rem);
                else store_four(to_rem, rem, there);
            }
        }
        if constexpr (!FULL) wait_for_memory();
    };
    uint32_t full0, full1, tile = 0;
    w.full(p, seen, v0, tiles, full0, full1);
#pragma unroll 1
    for (; tile < full0; tile++) body(tile, std::false_type{});
    wait_for_memory();
#pragma unroll 1
    for (; tile < full1; tile++) body(tile, std::true_type{});
#pragma unroll 1
    for (; tile < tiles; tile++) body(tile, std::false_type{});
    if (__any((over & kOver) != 0 || outside) && w.lane == 0) q_over = 1;          // what all threads made for all waves
    large |= (k_over & kOver) != 0;
    __syncthreads();
    if (q_over || __any(large)) {
        mx[0] = mx[1] = INT32_MIN;
        wide_scores(p, w, seen, v0, tiles, mx, bad);
    }
#pragma unroll
    for (int rb = 0; rb < 2; rb++) {
        mx[rb] = max(mx[rb], __shfl_xor(mx[rb], 16, 64));
        mx[rb] = max(mx[rb], __shfl_xor(mx[rb], 32, 64));
        if (w.kg == 0) top[w.wave][16 * rb + w.col] = mx[rb];
    }
    __syncthreads();
    if (threadIdx.x < w.R) {
        int32_t m = top[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < 4; i++) m = max(m, top[i][threadIdx.x]);
        p.chunk_max[w.row(p, threadIdx.x) * p.plan.score_chunks + blockIdx.y] = m;
    }
    if (bad) atomicOr(p.status, bad);
}

// Exponentials of 32 rows and a chunk of the positions, and the rows' sums, to which the chunks add.  A wave takes 256 positions of a row
// at a time, two of them under way.  The table's entries are 4 MB, of which a wave asks for 64 lines at a time: reading them is bound by L2
// (606 us for the 2048 tokens above, the factors' products 208: 0.8 GB at 3.9 TB/s).
template <bool FACTORS, bool SHIFTED>
__global__ void __launch_bounds__(256) wit_window_exp_kernel(WindowArgs p) {
    __shared__ int32_t top[kRows];
    __shared__ unsigned long long sums[kRows];
    __shared__ double factors[FACTORS ? 2 * kFactors : 1];
    RowTile w;
    if (!w.find(p, blockIdx.x)) return;
    const step::Seen seen = w.seen(p);
    const uint32_t v0 = blockIdx.y * p.plan.exp_cols;
    if (v0 >= seen.tiles) return;
    const uint32_t tiles = min(p.plan.exp_cols, seen.tiles - v0), parts = (seen.tiles - 1) / p.plan.score_cols + 1;
    if (threadIdx.x < kRows) {
        top[threadIdx.x] = INT32_MIN;
        sums[threadIdx.x] = 0;
    }
    bool computed = false;
    if constexpr (FACTORS) {
        computed = !__any(p.differs[w.lane] != 0);
        if (computed)
            for (uint32_t i = threadIdx.x; i < 2 * kFactors; i += 256) factors[i] = p.factors[i];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < parts * kRows; i += 256) {
        const uint32_t r = i % kRows;
        if (r < w.R) atomicMax(&top[r], p.chunk_max[w.row(p, r) * p.plan.score_chunks + i / kRows]);
    }
    __syncthreads();
    if (blockIdx.y == 0 && p.a.d_max && threadIdx.x < w.R) p.a.d_max[w.row(p, threadIdx.x)] = top[threadIdx.x];
    uint32_t bad = 0;
    const uint32_t last = ((uint32_t)1 << p.a.bit_shift) - 1, mine = w.wave < w.R ? (w.R - 1 - w.wave) / 4 + 1 : 0;          // rows of the wave
    uint32_t full0, full1;
    w.full(p, seen, v0, tiles, full0, full1);
    if (!computed) full1 = full0;
    auto entry = [&](uint32_t d) { return (int32_t)__builtin_rint(factors[d / kFactors] * factors[kFactors + d % kFactors]); };
    const uint32_t groups = (full1 - full0 + 3) / 4, items = mine * groups;
    if (items) {
        // item i: four tiles, group i % groups, of the wave's row i / groups; two items at a time, each in registers of its own.  Lanes behind
        // the last tile take it again, and leave it out of the sum.
        struct Item {
            uint32_t r, g, t, v;
            size_t row;
        };
        uint32_t k = 0, g = 0;
        auto next_item = [&]() {
            Item a;
            a.r = w.wave + 4 * k;
            a.g = g;
            a.row = w.row(p, a.r);
            a.v = v0 + min(full0 + 4 * g + w.lane / 16, full1 - 1);
            a.t = seen.tile(a.v) * kCols + 4 * w.lane % kCols;
            if (++g == groups) {
                g = 0;
                if (k + 1 < mine) k++;
            }
            return a;
        };
        auto load = [&](const Item& a) { return *reinterpret_cast<const v4u_t*>(p.scores.at(a.row, a.t, a.v)); };
        unsigned long long sum = 0;
        auto work = [&](const Item& a, const v4u_t& x) {
            const int32_t mx = top[a.r];
            v4u_t e, shifted;
            unsigned long long four = 0;
            uint32_t most = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint32_t below = (uint32_t)mx - (uint32_t)x[j];
                most = max(most, below);
                shifted[j] = (int32_t)(0 - below);
                e[j] = entry(min(below, last));          // entry 0 stands in for those before it
                four += (uint32_t)e[j];
            }
            if (most > last) bad |= (uint32_t)kWitIndex;
            if constexpr (SHIFTED) store_last(p.exps.at(a.row, a.t, a.v), e);          // 240 -> 221 us; not so a workspace's, which stays in the caches (47, values 57 -> 53)
            else *reinterpret_cast<v4u_t*>(p.exps.at(a.row, a.t, a.v)) = e;
            if constexpr (SHIFTED) store_last(p.a.d_shifted + a.row * p.a.max_len + a.t, shifted);
            sum += full0 + 4 * a.g + w.lane / 16 < full1 ? four : 0;
            if (a.g + 1 == groups) {
#pragma unroll
                for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
                if (w.lane == 0) sums[a.r] = sum;
                sum = 0;
            }
        };
        Item a = next_item();
        v4u_t x = load(a);
        uint32_t it = 0;
        wait_for_memory();
#pragma unroll 1
        for (; it + 2 <= items; it += 2) {
            const Item b = next_item();
            const v4u_t y = load(b);
            __builtin_amdgcn_sched_barrier(0);
            work(a, x);
            a = next_item();
            x = load(a);
            __builtin_amdgcn_sched_barrier(0);
            work(b, y);
        }
        if (it < items) work(a, x);
    }
    __syncthreads();
    // the other tiles, four rows of one at a time
    const uint32_t others = tiles - (full1 - full0), quads = (w.R + 3) / 4;
    for (uint32_t i = w.wave; i < others * quads; i += 4) {
        const uint32_t j = i / quads, r = 4 * (i - j * quads) + w.lane / 16, v = v0 + (j < full0 ? j : j - full0 + full1), t = seen.tile(v) * kCols + 4 * w.col;
        const uint32_t rr = min(r, w.R - 1), there = r < w.R ? seen_of_four(p, w.pos_of(p, rr), t) : 0;
        const size_t row = w.row(p, rr);
        const int32_t mx = top[rr];
        const int32_t* from = p.scores.at(row, t, v);
        v4u_t x = {mx, mx, mx, mx}, e, shifted;
        if (there == 15u) {
            x = *reinterpret_cast<const v4u_t*>(from);
        } else {
#pragma unroll
            for (uint32_t m = 0; m < 3; m++)
                if ((there >> m) & 1u) x[m] = from[m];
            if (there >> 3) x[3] = from[3];
        }
        unsigned long long sum = 0;
#pragma unroll
        for (uint32_t m = 0; m < 4; m++) {
            const uint32_t below = (uint32_t)mx - (uint32_t)x[m];
            const int64_t idx = (int64_t)last - below;
            const bool ok = idx >= 0 && idx < ((int64_t)1 << p.a.index_bits);
            e[m] = computed ? entry(min(below, last)) : p.a.d_exp_table[ok ? idx : 0];
            shifted[m] = (int32_t)(0 - below);
            if ((there >> m) & 1u) {
                if (!ok) bad |= (uint32_t)kWitIndex;
                if (e[m] < 0) bad |= (uint32_t)kWitSum;
                sum += (unsigned long long)max(e[m], 0);
            }
        }
        store_four(p.exps.at(row, t, v), e, there);
        if constexpr (SHIFTED) store_four(p.a.d_shifted + row * p.a.max_len + t, shifted, there);
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
        if (w.col == 0 && r < w.R) atomicAdd(&sums[r], sum);
    }
    __syncthreads();
    if (threadIdx.x < w.R) atomicAdd(&p.sums[w.row(p, threadIdx.x)], sums[threadIdx.x]);
    if (bad) atomicOr(p.status, bad);
}

// Probabilities of 32 rows and their products with 128 elements of the values, over a chunk of the positions.  Eight threads a row make
// the digits of 64 positions in LDS; a wave takes 32 elements and all rows, and turns its values into operands in registers.  A
// probability is floor((e P + floor(S/2)) / S) from one product in double precision, as the scores' quotients are, where S is below 2^28 and P
// at most 2^22; the remainder of the division gives the lookup's query.  Four waves of 32 elements leave 256 registers each, of which the sums
// take 80 to 112 and spill a few.  Heads of more than 128 elements are divided among workgroups that make the probabilities again (one head of
// 4096: 140 us, 0.74 POP/s of six products of planes, 1.4e7 requests of L2).
constexpr uint32_t kValueThreads = 256;
constexpr uint64_t kPlainSum = (uint64_t)1 << 28;
enum Written { kNone, kBoth, kSome };          // of the probabilities and queries
typedef int v2u_t __attribute__((ext_vector_type(2), aligned(4)));

template <int PP>
struct ValueLds {
    uint32_t digits[2][PP * 4 * kRows * 4];
    int64_t off[2][step::kOffsetTiles * kCols];
    unsigned long long p_sum[kRows];
    uint32_t third[2], wide, outside;          // the last tile with digits in the third plane (and 1), of even and odd ones; whether a page is outside the cache
    uint32_t large;                            // whether a row's sum is kPlainSum or more
};

template <int PP, bool WIDE, Written W, bool PACKED>
__device__ __forceinline__ bool window_values(const WindowArgs& p, const RowTile& w, const step::Seen& seen, ValueLds<PP>& lds, uint32_t group, uint32_t chunk, uint32_t& bad) {
    constexpr int VP = WIDE ? 4 : 3, G = PP + VP - 1;
    constexpr uint32_t K = step::kOffsetTiles;
    const step::Seen made = w.all_seen(p);
    const uint32_t v0 = chunk * p.plan.value_cols, tiles = min(p.plan.value_cols, seen.tiles - v0), dim = p.c.dim;
    // of the probabilities: this thread's row and its eight positions of a tile
    const uint32_t r = threadIdx.x >> 3, part = threadIdx.x & 7u, rr = min(r, w.R - 1), pos = w.pos_of(p, rr);
    const size_t row = w.row(p, rr);
    unsigned long long sum = p.sums[row], all = 0;
    if (sum == 0) {
        bad |= (uint32_t)kWitSum;
        sum = 1;
    }
    if (!WIDE && r < w.R && group == 0 && chunk == 0 && part == 0 && p.a.d_sum) store_sum(&p.a.d_sum[row], sum, bad);
    const double inv = 1.0 / (double)sum, scale = (double)p.a.prob_scale, half = (double)(sum >> 1) + 0.5, whole_sum = (double)sum, odd = (double)(sum & 1) - 1.0;
    // Both choose between loops that meet at barriers, so they are the workgroup's: read behind a barrier that follows what is written to them, and
    // written again behind another one.
    bool plain = false, outside = false;
    // of the values: elements e0 + 2 col, + 1; lanes behind the last element take it again
    const uint32_t e0 = group * step::kValueDims + 32 * w.wave, el = e0 + 2 * w.col;
    const bool pairs = dim % 2 == 0;
    const int32_t* values = p.c.d_v + (int64_t)w.kv * p.c.head_stride;
    const int32_t *value0 = values + (pairs ? min(el, dim - 2) : min(el, dim - 1)), *value1 = values + min(el + 1, dim - 1);
    auto make_offsets = [&](uint32_t tile) {
        const uint32_t n = min(K, tiles - tile) * kCols;
        for (uint32_t i = threadIdx.x; i < n; i += kValueThreads) {
            const int64_t o = offset_of(p, w.b, seen, seen.tile(v0 + tile + i / kCols) * kCols + i % kCols);
            lds.off[(tile / K) & 1][i] = max(o, (int64_t)0);
            if (o < 0) lds.outside = 1;
        }
    };
    auto offsets = [&](uint32_t tile) { return lds.off[(tile / K) & 1] + (tile % K) * kCols; };
    v2u_t x[16];
    v4u_t e[2];
    v4i_t vb[2][VP];          // the tile's operands, of the elements 2 col, + 1 or (PACKED) col, 16 + col
    auto request = [&](uint32_t tile) {
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {
            const uint32_t block = min(e0 / 16 + j, 4 * p.plan.dim64 - 1);
            const uint8_t* from = p.values + p.tile_of(w.b, w.kv, made.number(seen.tile(v0 + tile))) * p.plan.dim64 * step::kValueStepBytes + (size_t)block * 3 * 1024 + w.lane * 16;
#pragma unroll
            for (int k = 0; k < 3; k++) vb[j][k] = *reinterpret_cast<const v4i_t*>(from + k * 1024);
        }
    };
    auto fetch_values = [&](uint32_t tile) {
        const int64_t* o = offsets(tile) + 16 * w.kg;
        if (pairs) {
#pragma unroll
            for (uint32_t j = 0; j < 16; j++) x[j] = *reinterpret_cast<const v2u_t*>(value0 + o[j]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 16; j++) x[j] = v2u_t{value0[o[j]], value1[o[j]]};
        }
    };
    auto fetch_exps = [&](uint32_t tile, auto all_see) {
        const uint32_t t = seen.tile(v0 + tile) * kCols + 8 * part;
        const int32_t* from = p.exps.at(row, t, v0 + tile);
        if constexpr (decltype(all_see)::value) {
            e[0] = *reinterpret_cast<const v4u_t*>(from);
            e[1] = *reinterpret_cast<const v4u_t*>(from + 4);
        } else {
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
                const uint32_t there = seen_of_four(p, pos, t + 4 * h);
                if (there == 15u) {
                    e[h] = *reinterpret_cast<const v4u_t*>(from + 4 * h);
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) e[h][j] = (there >> j) & 1u ? from[4 * h + j] : 0;
                }
            }
        }
    };
    v4i_t acc[2][2][G];          // [element of a pair][block of rows][exponent]
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int rb = 0; rb < 2; rb++)
#pragma unroll
            for (int g = 0; g < G; g++) acc[j][rb][g] = v4i_t{0, 0, 0, 0};
    uint32_t over = 0;
    // a tile and, if it is not the last one, the loads of the next; FULL: all rows see this tile's positions and the next one's
    auto body = [&](uint32_t tile, auto all_see) {
        constexpr bool FULL = decltype(all_see)::value;
        // operands and probabilities first, then the next tile's loads, then this one's stores
        if constexpr (!PACKED) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const v4i_t y = {x[4 * c][j], x[4 * c + 1][j], x[4 * c + 2][j], x[4 * c + 3][j]};
                    uint32_t v[4];
                    if constexpr (WIDE) four_planes(y, v);
                    else three_planes(y, v, over);
#pragma unroll
                    for (int k = 0; k < VP; k++) vb[j][k][c] = (int)v[k];
                }
        }
        const uint32_t t = seen.tile(v0 + tile) * kCols + 8 * part, there = FULL ? 255u : seen_of_four(p, pos, t) | seen_of_four(p, pos, t + 4) << 4;
        v4u_t pr[2], query[2];
        if (FULL || plain) {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const double num = __builtin_fma((double)max(e[j / 4][j % 4], 0), scale, half), q = __builtin_floor(num * inv);
                pr[j / 4][j % 4] = (int32_t)q;
                if constexpr (W != kNone) query[j / 4][j % 4] = (int32_t)__builtin_fma(2.0, __builtin_fma(-q, whole_sum, num), odd);
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const uint32_t ej = (uint32_t)max(e[j / 4][j % 4], 0), pj = probability(ej, (uint64_t)p.a.prob_scale, sum, inv);
                pr[j / 4][j % 4] = (int32_t)pj;
                if constexpr (W != kNone) {
                    uint32_t wide = 0;
                    int32_t qj;
                    store_sum(&qj, lookup_query(ej, p.a.prob_scale, sum, pj), wide);
                    query[j / 4][j % 4] = qj;
                    if (((there >> j) & 1u) && p.a.d_query) bad |= wide;
                }
            }
        }
        if (FULL || tile + 1 < tiles) {
            if constexpr (!PACKED) {
                if ((tile + 1) % K == 0) {
                    make_offsets(tile + 1);
                    __syncthreads();
                    outside = __builtin_amdgcn_readfirstlane((int)lds.outside) != 0;
                }
                fetch_values(tile + 1);
            }
            fetch_exps(tile + 1, all_see);
        }
        if constexpr (W != kNone) {
            const size_t o = row * p.a.max_len + t;
            if constexpr (W == kBoth && FULL) {
#pragma unroll
                for (uint32_t h = 0; h < 2; h++) {
                    *reinterpret_cast<v4u_t*>(p.a.d_prob + o + 4 * h) = pr[h];
                    *reinterpret_cast<v4u_t*>(p.a.d_query + o + 4 * h) = query[h];
                }
            } else {
#pragma unroll
                for (uint32_t h = 0; h < 2; h++) {
                    if (W == kBoth || p.a.d_prob) store_four(p.a.d_prob + o + 4 * h, pr[h], (there >> (4 * h)) & 15u);
                    if (W == kBoth || p.a.d_query) store_four(p.a.d_query + o + 4 * h, query[h], (there >> (4 * h)) & 15u);
                }
                wait_for_memory();
            }
        }
        uint32_t pl[2][4];
#pragma unroll
        for (uint32_t h = 0; h < 2; h++) {
            v4i_t d;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                d[j] = (there >> (4 * h + j)) & 1u ? pr[h][j] : 0;
                if (!PACKED && !FULL && outside && offset_of(p, w.b, seen, t + 4 * h + j) < 0) d[j] = 0;          // a page outside: no value
                if constexpr (WIDE) all += (uint32_t)d[j];
            }
            if constexpr (PP == 3) {
                uint32_t none = 0;
                three_planes(d, pl[h], none);
            } else {
                transpose4(digits_of(d[0]), digits_of(d[1]), digits_of(d[2]), digits_of(d[3]), pl[h]);
            }
        }
        if (PP == 3 && __any((pl[0][2] | pl[1][2]) != 0) && w.lane == 0) lds.third[tile & 1] = tile + 1;
        uint64_t* to = reinterpret_cast<uint64_t*>(lds.digits[tile & 1]) + ((part >> 1) * kRows + r) * 2 + (part & 1u);
#pragma unroll
        for (int k = 0; k < PP; k++) to[k * 8 * kRows] = ((uint64_t)pl[1][k] << 32) | pl[0][k];
        __syncthreads();
        const v4i_t* pa = reinterpret_cast<const v4i_t*>(lds.digits[tile & 1]) + w.kg * kRows + w.col;
        auto multiply = [&](auto a) {
            constexpr int A = decltype(a)::value;
            v4i_t f[2];
#pragma unroll
            for (uint32_t rb = 0; rb < 2; rb++) f[rb] = pa[A * 4 * kRows + 16 * rb];
#pragma unroll
            for (int k = 0; k < VP; k++)
#pragma unroll
                for (uint32_t rb = 0; rb < 2; rb++)
#pragma unroll
                    for (int j = 0; j < 2; j++) acc[j][rb][A + k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vb[j][k], f[rb], acc[j][rb][A + k], 0, 0, 0);
        };
        multiply(std::integral_constant<int, 0>{});
        multiply(std::integral_constant<int, 1>{});
        if (PP > 3 || lds.third[tile & 1] == tile + 1) multiply(std::integral_constant<int, 2>{});
        if constexpr (PP > 3) multiply(std::integral_constant<int, 3>{});
        if constexpr (PACKED) request(FULL ? tile + 1 : min(tile + 1, tiles - 1));
    };
    if constexpr (PACKED) request(0);
    __syncthreads();
    if (threadIdx.x < 2) lds.third[threadIdx.x] = 0;
    if (threadIdx.x == 0) lds.outside = 0;
    if (sum >= kPlainSum) lds.large = 1;
    __syncthreads();
    plain = PP == 3 && __builtin_amdgcn_readfirstlane((int)lds.large) == 0;
    if constexpr (PACKED) {
        for (uint32_t i = threadIdx.x; i < tiles * p.plan.splits; i += kValueThreads)
            if (p.over[p.tile_of(w.b, w.kv, made.number(seen.tile(v0 + i / p.plan.splits))) * p.plan.splits + i % p.plan.splits] & 2u) over = kOver;
    } else {
        make_offsets(0);
        __syncthreads();
        outside = __builtin_amdgcn_readfirstlane((int)lds.outside) != 0;
        fetch_values(0);
    }
    fetch_exps(0, std::false_type{});
    wait_for_memory();
    uint32_t full0, full1, tile = 0;
    w.full(p, seen, v0, tiles, full0, full1);
#pragma unroll 1
    for (; tile < full0; tile++) body(tile, std::false_type{});
    wait_for_memory();
#pragma unroll 1
    for (; plain && tile + 1 < full1 && !outside; tile++) body(tile, std::true_type{});
#pragma unroll 1
    for (; tile < tiles; tile++) body(tile, std::false_type{});
    if constexpr (WIDE) {
#pragma unroll
        for (int k = 4; k >= 1; k >>= 1) all += __shfl_xor(all, k, 64);
        if (part == 0) lds.p_sum[r] = all;
    } else {
        if (__any((over & kOver) != 0) && w.lane == 0) lds.wide = 1;
    }
    __syncthreads();
    if (!WIDE && lds.wide) return true;
    const bool whole = seen.tiles <= p.plan.value_cols;          // all positions of the rows are this workgroup's
#pragma unroll
    for (uint32_t rb = 0; rb < 2; rb++) {
        const uint32_t q_row = 16 * rb + w.col;
        if (q_row >= w.R) continue;
        const size_t at = w.row(p, q_row);
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t j = PACKED ? i / 4 : i % 2, m = PACKED ? i % 4 : i / 2, e1 = PACKED ? e0 + 16 * j + 4 * w.kg + m : e0 + 8 * w.kg + i;
            if (e1 >= dim) break;
            uint64_t y = WIDE ? (uint64_t)kCacheOffset * lds.p_sum[q_row] : 0, z = 0;
#pragma unroll
            for (int g = G - 1; g >= 0; g--) z = (z << 8) + (uint64_t)(int64_t)acc[j][rb][g][m];
            y += z;
            if (whole) {
                int32_t q, rem;
                p.out.apply((int64_t)y, q, rem, bad);
                p.a.d_out[at * dim + e1] = q;
                if (p.a.d_out_rem) p.a.d_out_rem[at * dim + e1] = rem;
            } else {
                p.part[(at * p.plan.value_chunks + chunk) * dim + e1] = (int64_t)y;
            }
        }
    }
    return false;
}

template <int PP, Written W, bool GROUPS, bool PACKED>          // what the first group of elements writes; whether there are others
__global__ void __launch_bounds__(kValueThreads, 2) wit_window_values_kernel(WindowArgs p) {
    __shared__ __attribute__((aligned(16))) ValueLds<PP> lds;
    RowTile w;
    if (!w.find(p, blockIdx.x)) return;
    const step::Seen seen = w.seen(p);
    const uint32_t group = GROUPS ? blockIdx.y % p.plan.groups : 0, chunk = GROUPS ? blockIdx.y / p.plan.groups : blockIdx.y;
    if (chunk * p.plan.value_cols >= seen.tiles) return;
    uint32_t bad = 0;
    if (threadIdx.x == 0) lds.wide = lds.large = 0;          // behind window_values' first barrier the others write them
    bool wide;
    if (W != kNone && GROUPS && group) wide = window_values<PP, false, kNone, PACKED>(p, w, seen, lds, group, chunk, bad);
    else wide = window_values<PP, false, W, PACKED>(p, w, seen, lds, group, chunk, bad);
    if (wide) window_values<PP, true, kNone, false>(p, w, seen, lds, group, chunk, bad);
    if (bad) atomicOr(p.status, bad);
}

// The chunks' partial sums of 64 elements of a row, a wave each.
__global__ void __launch_bounds__(64 * step::kJoinRows) wit_window_join_kernel(WindowArgs p) {
    RowTile w;
    if (!w.find(p, blockIdx.x)) return;
    const step::Seen seen = w.seen(p);
    const uint32_t r = blockIdx.z * step::kJoinRows + w.wave, e = blockIdx.y * 64 + w.lane, dim = p.c.dim;
    if (seen.tiles <= p.plan.value_cols || r >= w.R || e >= dim) return;
    const uint32_t parts = (seen.tiles - 1) / p.plan.value_cols + 1;
    uint32_t bad = 0;
    const size_t row = w.row(p, r);
    int64_t y = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < parts; i++) y += p.part[(row * p.plan.value_chunks + i) * dim + e];
    int32_t q, rem;
    p.out.apply(y, q, rem, bad);
    p.a.d_out[row * dim + e] = q;
    if (p.a.d_out_rem) p.a.d_out_rem[row * dim + e] = rem;
    if (bad) atomicOr(p.status, bad);
}

}  // namespace grape

using namespace grape;

extern "C" {

size_t grape_wit_window_attention_workspace(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t cache_heads, uint32_t dim, uint32_t max_new, uint32_t max_len, uint32_t window, uint32_t sinks) {
    return step::window_workspace(rows, seqs, heads, cache_heads, dim, max_new, max_len, window, sinks);
}

int grape_wit_window_attention(const grape_wit_window_attention_args* args, const grape_wit_cache* cache, grape_stream_t st) {
    GRAPE_REQUIRE(initialised(), "grape_init has not been called");
    GRAPE_REFUSED_IF(step::refuse_window(args, cache));
    if (!args->seqs || !args->rows || !args->max_new) return GRAPE_OK;
    if (args->max_new == 1) return attend_single(*args, *cache, st);          // heads by sixteen and not rows by 32, one launch for few positions (24 sequences behind a window of 1024: 79 us, and 84 here)
    WindowArgs p;
    p.a = *args;
    p.c = *cache;
    const grape_wit_window_attention_args& a = p.a;
    step::window_plan(a.rows, a.seqs, a.heads, p.c.heads, p.c.dim, a.max_new, a.max_len, a.window, a.sinks, p.plan);
    const step::WindowPlan& pl = p.plan;
    uint8_t* ws = (uint8_t*)a.d_workspace;
    const size_t cols = (size_t)pl.cols * kCols;
    p.scores = a.d_scores ? Rows{a.d_scores, a.max_len, true} : Rows{(int32_t*)(ws + pl.at_scores), cols, false};
    p.exps = a.d_exp ? Rows{a.d_exp, a.max_len, true} : Rows{(int32_t*)(ws + pl.at_exp), cols, false};
    p.chunk_max = (int32_t*)(ws + pl.at_max);
    p.sums = (unsigned long long*)(ws + pl.at_sum);
    p.part = (int64_t*)(ws + pl.at_part);
    p.keys = ws + pl.at_keys;
    p.values = ws + pl.at_values;
    p.queries = ws + pl.at_queries;
    p.over = (uint32_t*)(ws + pl.at_over);
    p.query_over = (uint32_t*)(ws + pl.at_query_over);
    p.page = token::fast_div(p.c.page_size);
    p.by_each = token::fast_div(pl.each);
    p.qk = scaler(a.qk_scale);
    p.out = scaler(a.out_scale);
    p.limit = std::min(0x1p50, 2147483647.0 * (double)a.qk_scale);
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status);
    if (rc) return rc;
    auto aligned = [&](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    p.k_vec = p.c.dim % 4 == 0 && ((p.c.page_stride | p.c.token_stride | p.c.head_stride) & 3) == 0 && aligned(p.c.d_k);
    p.q_vec = p.c.dim % 4 == 0 && a.q_stride % 4 == 0 && aligned(a.d_q);
    p.along = pl.tiles * p.c.heads;
    p.factors = nullptr;
    if (a.bit_shift <= 20 && a.index_bits >= a.bit_shift) {
        p.factors = (double*)(ws + pl.at_factors);
        p.differs = (uint32_t*)(p.factors + 2 * kFactors);
    }
    const size_t score_lds = std::max<size_t>((size_t)std::min(pl.packed ? pl.steps : pl.dim64, kBlockSteps) * 12 * kRows * 16 + (pl.packed ? 0 : (size_t)pl.score_cols * kCols * 8), p.factors ? 2 * kFactors * sizeof(double) : 0);
    const dim3 scores(p.along + (p.factors && !pl.packed ? kTableGroups : 0), pl.score_chunks), exps(p.along, pl.exp_chunks), values(p.along, pl.value_chunks * pl.groups);
    using std::integral_constant;
    auto scores_of = [&](auto packed, auto by_four) {
        constexpr bool P = decltype(packed)::value, V = decltype(by_four)::value;
        if (a.d_scores_rem) wit_window_scores_kernel<P, V, true><<<scores, 256, score_lds, s>>>(p);
        else wit_window_scores_kernel<P, V, false><<<scores, 256, score_lds, s>>>(p);
    };
    if (pl.packed) {
        wit_window_pack_kernel<<<(p.factors ? kTableGroups : 0) + (p.along + a.seqs * pl.all_cols * p.c.heads) * pl.splits, 256, 0, s>>>(p);
        GRAPE_LAUNCH_CHECK();
        scores_of(std::true_type{}, std::true_type{});
    } else if (p.k_vec) {
        scores_of(std::false_type{}, std::true_type{});
    } else {
        scores_of(std::false_type{}, std::false_type{});
    }
    GRAPE_LAUNCH_CHECK();
    if (p.factors && a.d_shifted) wit_window_exp_kernel<true, true><<<exps, 256, 0, s>>>(p);
    else if (p.factors) wit_window_exp_kernel<true, false><<<exps, 256, 0, s>>>(p);
    else if (a.d_shifted) wit_window_exp_kernel<false, true><<<exps, 256, 0, s>>>(p);
    else wit_window_exp_kernel<false, false><<<exps, 256, 0, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    auto values_of = [&](auto planes, auto written) {
        constexpr int PP = decltype(planes)::value;
        constexpr Written W = decltype(written)::value;
        if (pl.packed && pl.groups > 1) wit_window_values_kernel<PP, W, true, true><<<values, kValueThreads, 0, s>>>(p);
        else if (pl.packed) wit_window_values_kernel<PP, W, false, true><<<values, kValueThreads, 0, s>>>(p);
        else if (pl.groups > 1) wit_window_values_kernel<PP, W, true, false><<<values, kValueThreads, 0, s>>>(p);
        else wit_window_values_kernel<PP, W, false, false><<<values, kValueThreads, 0, s>>>(p);
    };
    auto values_by = [&](auto planes) {
        if (a.d_prob && a.d_query) values_of(planes, integral_constant<Written, kBoth>{});
        else if (a.d_prob || a.d_query) values_of(planes, integral_constant<Written, kSome>{});
        else values_of(planes, integral_constant<Written, kNone>{});
    };
    if (a.prob_scale <= ((int64_t)1 << 22)) values_by(integral_constant<int, 3>{});
    else values_by(integral_constant<int, 4>{});
    GRAPE_LAUNCH_CHECK();
    if (pl.value_chunks > 1) {
        wit_window_join_kernel<<<dim3(p.along, pl.dim64, kRows / step::kJoinRows), 64 * step::kJoinRows, 0, s>>>(p);
        GRAPE_LAUNCH_CHECK();
    }
    return GRAPE_OK;
}

}  // extern "C"

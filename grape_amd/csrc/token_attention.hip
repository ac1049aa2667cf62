// Attention of one new token a sequence over a paged cache of keys and values, with the tensors that a proof of it looks up.
#include <algorithm>
#include "token_device.hpp"

namespace grape {

// ------------------------------------------------------------------------------------------------
// Attention of one token a sequence: scores, softmax through the table, products with the values.
//
// The softmax is the table's, rounded, so a running maximum cannot be corrected later by a factor: the maximum of the whole row
// is needed before the first exponential and the sum of all before the first probability.  Hence three launches, each over
// chunks of the positions, and a fourth that joins the values' partial sums.  Keys and values are read once; what goes between
// the launches is 4 bytes a head and position.
//
// Both products run on the matrix cores: a cache element x is taken as x - c, c = 128 (1 + 2^8 + 2^16), whose balanced digits
// are the bytes of x with three top bits turned over, and c times the sum of the other operand is added in the end.  The pairs
// of planes with the same sum of exponents share an accumulator: 4 * 2^14 * 8192 elements (1024 positions) stay below 2^31.
// ------------------------------------------------------------------------------------------------
constexpr int64_t kCacheOffset = 0x808080;
constexpr uint32_t kByteTops = 0x80808080;          // of a plane's four bytes

struct AttendArgs {
    grape_wit_attention_args a;
    grape_wit_cache c;
    token::AttentionPlan plan;
    token::FastDiv page;
    Scaler qk, out;
    int32_t* chunk_max;          // [seqs][heads][score chunks]
    unsigned long long* sums;    // [seqs][heads][exp chunks]
    int64_t* part;               // [seqs][heads][value chunks][dim]
    uint32_t* status;
};

__device__ __forceinline__ bool span_of(const AttendArgs& p, uint32_t b, uint32_t& lo, uint32_t& hi) {
    return token::live_span(p.a.d_lens[b], p.a.d_first ? p.a.d_first[b] : 0, p.a.max_len, p.a.table_stride, p.c.page_size, lo, hi);
}

// The sequence, the chunk of `size` positions and the positions that are number `index` when the sequences' chunks are counted, one
// at least of each; false where there are fewer.  Where lengths differ, many of max_len's chunks are of no sequence: counted, their
// workgroups come last, when all others are under way (64 sequences of up to 2048, 8 heads of 128: 147 us a call and not 156, 24 with
// a window of 256 of up to 5000 29 and not 39).  It costs each workgroup a wait for the lengths (64 sequences of 1024 each: 153 and
// not 149), so that few sequences keep the plain order.  All lanes of a wave together.
__device__ __forceinline__ bool find_chunk(const AttendArgs& p, uint32_t index, uint32_t size, uint32_t& b, uint32_t& chunk, uint32_t& lo, uint32_t& hi, bool& fits) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t before = 0;
    for (uint32_t base = 0; base < p.a.seqs; base += 64) {
        uint32_t l = 0, h = 0, n = 0;
        bool ok = true;
        if (base + lane < p.a.seqs) {
            ok = span_of(p, base + lane, l, h);
            n = l < h ? (h - l - 1) / size + 1 : 1;
        }
        uint32_t sum = n;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint32_t y = __shfl_up(sum, d, 64);
            if (lane >= d) sum += y;
        }
        const unsigned long long past = __ballot(before + sum > index);
        if (past) {
            const int at = __ffsll(past) - 1;
            b = base + (uint32_t)at;
            chunk = index - before - (uint32_t)__builtin_amdgcn_readlane((int)(sum - n), at);
            lo = (uint32_t)__builtin_amdgcn_readlane((int)l, at);
            hi = (uint32_t)__builtin_amdgcn_readlane((int)h, at);
            fits = __builtin_amdgcn_readlane((int)ok, at) != 0;
            return true;
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    }
    return false;
}

// The offsets of a chunk's positions t0 .. t0 + n, made by all threads of a workgroup.  The first page of each thread is
// requested before the sequence's length is known where it does not depend on it, so that the two loads are under way together.
struct Offsets {
    int32_t page = -1;
    uint32_t t = 0;
    bool early = false;
    __device__ __forceinline__ int32_t load(const AttendArgs& p, uint32_t b, uint32_t pos) const {
        return p.a.d_block_table[(size_t)b * p.a.table_stride + p.page(pos)];
    }
    __device__ __forceinline__ void request(const AttendArgs& p, uint32_t b, uint64_t start, uint32_t most) {
        early = p.a.d_first == nullptr;
        t = (uint32_t)start + threadIdx.x;
        if (early && threadIdx.x < most && start + threadIdx.x < p.a.max_len && p.page(t) < p.a.table_stride) page = load(p, b, t);
    }
    __device__ __forceinline__ bool store(const AttendArgs& p, uint32_t b, uint32_t t0, uint32_t n, uint32_t filled, int64_t* off) const {
        bool outside = false;
        for (uint32_t i = threadIdx.x; i < filled; i += blockDim.x) {
            int64_t o = -1;
            if (i < n) {
                const int32_t pg = early && i == threadIdx.x ? page : load(p, b, t0 + i);
                o = token::token_offset(p.c, pg, t0 + i - p.page(t0 + i) * p.c.page_size);
                outside |= o < 0;
            }
            off[i] = o;
        }
        return outside;
    }
};

// four elements from x; those from `n` on are whatever comes first
template <bool VEC>
__device__ __forceinline__ v4i_t load4(const int32_t* x, uint32_t at, uint32_t n) {
    if constexpr (VEC) {
        return *reinterpret_cast<const v4i_t*>(x + (at < n ? at : 0));          // n is a multiple of 4
    } else {
        v4i_t v;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) v[j] = x[at + j < n ? at + j : 0];
        return v;
    }
}

typedef int v2i_t __attribute__((ext_vector_type(2)));
template <bool VEC>
__device__ __forceinline__ v2i_t load2(const int32_t* x, uint32_t at, uint32_t n) {
    if constexpr (VEC) {
        return *reinterpret_cast<const v2i_t*>(x + (at < n ? at : 0));
    } else {
        v2i_t v;
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) v[j] = x[at + j < n ? at + j : 0];
        return v;
    }
}

// The query heads of a workgroup: R heads from h0 of sequence b, which read the cache's head kv.
struct Tile {
    uint32_t b, kv, h0, R;
    size_t row0;                 // of the rows [seqs][heads]
    uint32_t lane, wave, col, kg;
    __device__ __forceinline__ Tile(const AttendArgs& p, uint32_t b_, uint32_t head_tile) : b(b_) {
        const uint32_t each = p.a.heads / p.c.heads;
        kv = head_tile / p.plan.tiles;
        const uint32_t tile = head_tile - kv * p.plan.tiles;
        h0 = kv * each + tile * p.plan.rows;
        R = min(p.plan.rows, each - tile * p.plan.rows);
        row0 = (size_t)b * p.a.heads + h0;
        lane = threadIdx.x & 63u;
        wave = threadIdx.x >> 6;
        col = lane & 15u;
        kg = lane >> 4;
    }
    // Row m of a product is query head 4 (m % 4) + m / 4: register i of lane l then holds head 4 i + l / 16 at column l % 16, and
    // four heads need one register of every lane.  Rows past the last head repeat it; nothing of them is kept.
    __device__ __forceinline__ uint32_t row() const {
        const uint32_t head = 4 * (col & 3u) + (col >> 2);
        return head < R ? head : R - 1;
    }
};

// The queries' digits in LDS, [step of 64][plane 0..4][lane group][row], 16 bytes each, with plane 4 what a top digit of 128
// carries; and the queries' sums.  q4: this thread's first four elements, requested by first().
struct Queries {
    int32_t q4[4];
    __device__ __forceinline__ void load(const AttendArgs& p, const Tile& w, uint32_t i) {
        const uint32_t steps = p.plan.dim64, r = i / (steps * 16), quad = i - r * (steps * 16);
        const int32_t* q = p.a.d_q + w.b * p.a.q_stride + (size_t)(w.h0 + r) * p.c.dim;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) q4[j] = 4 * quad + j < p.c.dim ? q[4 * quad + j] : 0;
    }
    __device__ __forceinline__ void first(const AttendArgs& p, const Tile& w) {
        if (threadIdx.x < w.R * p.plan.dim64 * 16) load(p, w, threadIdx.x);
    }
    __device__ __forceinline__ void store(const AttendArgs& p, const Tile& w, uint32_t* digits, unsigned long long* q_sum, uint32_t* over_any) {
        const uint32_t steps = p.plan.dim64;
        for (uint32_t i = threadIdx.x; i < w.R * steps * 16; i += blockDim.x) {
            const uint32_t r = i / (steps * 16), quad = i - r * (steps * 16), s = quad >> 4, c = (quad >> 2) & 3u, g = quad & 3u;
            if (i != threadIdx.x) load(p, w, i);
            uint32_t d[4], pl[4], carry = 0;
            long long sum = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                d[j] = digits_of(q4[j]);
                sum += q4[j];
                carry |= q4[j] > kDigitTop ? 1u << (8 * j) : 0u;
            }
            transpose4(d[0], d[1], d[2], d[3], pl);
            uint32_t* o = digits + (((s * 5 * 4 + g) * w.R + r) << 2) + c;
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) o[k * 16 * w.R] = pl[k];
            o[4 * 16 * w.R] = carry;
            if (carry) *over_any = 1;
            // sixteen neighbouring lanes are of one row
#pragma unroll
            for (int k = 8; k >= 1; k >>= 1) sum += __shfl_xor(sum, k, 64);
            if ((i & 15u) == 0) atomicAdd(&q_sum[r], (unsigned long long)sum);
        }
    }
};

// Products of the queries with n keys (less their offset): sink(row, position, whether there is one, 64-bit sum), called by all
// lanes of a wave together, 16 neighbouring ones for one row.  A wave takes 16
// positions: lane l reads those elements 64 s + 16 c + 4 (l / 16) .. + 4 of position l % 16 that make up its operand of step s
// (any order of a step's elements will do, as long as the queries' digits have the same), whole lines among the lanes.
template <bool VEC, uint32_t WAVES, class F>
__device__ __forceinline__ void score_products(const AttendArgs& p, const Tile& w, uint32_t n, const int64_t* off, const uint32_t* digits, bool over, bool apart, F sink) {
    const uint32_t steps = p.plan.dim64, R = w.R, row = w.row(), dim = p.c.dim;
    const int32_t* keys = p.c.d_k + (int64_t)w.kv * p.c.head_stride;
    // the waves take different positions, or (apart) different steps of the same ones
    for (uint32_t at = apart ? 0 : 16 * w.wave; at < n; at += apart ? 16 : 16 * WAVES) {
        const int32_t* k = keys + max(off[min(at + w.col, n - 1)], (int64_t)0);
        v4i_t acc[8];
#pragma unroll
        for (int g = 0; g < 8; g++) acc[g] = v4i_t{0, 0, 0, 0};
        // two steps at a time: their keys are requested together, and other waves multiply meanwhile
        for (uint32_t s = apart ? 2 * w.wave : 0; s < steps; s += apart ? 2 * WAVES : 2) {
            v4i_t x[8];
#pragma unroll
            for (uint32_t c = 0; c < 8; c++) {
                if (64 * s + 16 * c < dim) x[c] = load4<VEC>(k, 64 * s + 16 * c + 4 * w.kg, dim);
                else x[c] = v4i_t{0, 0, 0, 0};
            }
#pragma unroll
            for (uint32_t u = 0; u < 2; u++) {
                if (s + u >= steps) break;
                v4i_t kb[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const v4i_t y = x[4 * u + c];
                    uint32_t pl[4];
                    transpose4((uint32_t)y[0], (uint32_t)y[1], (uint32_t)y[2], (uint32_t)y[3], pl);
#pragma unroll
                    for (int k2 = 0; k2 < 4; k2++) kb[k2][c] = (int)(k2 < 3 ? pl[k2] ^ kByteTops : pl[k2]);
                }
                const v4i_t* qa = reinterpret_cast<const v4i_t*>(digits) + ((s + u) * 5 * 4 + w.kg) * R + row;
#pragma unroll
                for (int a = 0; a < 4; a++) {
                    const v4i_t f = qa[a * 4 * R];
#pragma unroll
                    for (int k2 = 0; k2 < 4; k2++) acc[a + k2] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, kb[k2], acc[a + k2], 0, 0, 0);
                }
                if (over) {
                    const v4i_t f = qa[4 * 4 * R];
#pragma unroll
                    for (int k2 = 0; k2 < 4; k2++) acc[4 + k2] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, kb[k2], acc[4 + k2], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            if (4 * i >= R) break;
            const uint32_t r = 4 * i + w.kg;
            uint64_t y = 0;
#pragma unroll
            for (int g = 7; g >= 0; g--) y = (y << 8) + (uint64_t)(int64_t)acc[g][i];
            sink(r, at + w.col, r < R && at + w.col < n, y);
        }
    }
}

// Such sums, [row][stride] in LDS, rescaled and written; the largest score of each row goes to largest(r, max).
template <class F>
__device__ __forceinline__ void score_rows(const AttendArgs& p, const Tile& w, uint32_t t0, uint32_t n, const int64_t* off, const uint64_t* sums, uint32_t stride,
                                           const unsigned long long* q_sum, uint32_t& bad, F largest) {
    for (uint32_t r = w.wave; r < w.R; r += 4) {
        const size_t o = (w.row0 + r) * p.a.max_len + t0;
        const uint64_t more = (uint64_t)kCacheOffset * q_sum[r];
        int32_t mx = INT32_MIN;
        for (uint32_t i = w.lane; i < n; i += 64) {
            const int64_t y = off[i] < 0 ? 0 : (int64_t)(sums[r * stride + i] + more);          // a page outside: zero
            int32_t q, rem;
            p.qk.apply(y, q, rem, bad);
            p.a.d_scores[o + i] = q;
            if (p.a.d_scores_rem) p.a.d_scores_rem[o + i] = rem;
            mx = max(mx, q);
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) mx = max(mx, __shfl_xor(mx, d, 64));
        if (w.lane == 0) largest(r, mx);
    }
}

// Exponentials of the scores t0 + i of row `row`, i = from, from + step, ... below n, and their sum.  Bound by the gathers'
// latency: eight are under way a thread.
constexpr uint32_t kExpAhead = 8;
__device__ __forceinline__ unsigned long long exponentials(const AttendArgs& p, size_t row, uint32_t t0, uint32_t from, uint32_t step, uint32_t n, int32_t mx, uint32_t& bad) {
    const size_t o = row * p.a.max_len + t0;
    unsigned long long sum = 0;
    for (uint32_t t = from; t < n; t += step * kExpAhead) {
        int32_t x[kExpAhead], e[kExpAhead];
#pragma unroll
        for (uint32_t j = 0; j < kExpAhead; j++) x[j] = t + j * step < n ? p.a.d_scores[o + t + j * step] : mx;
#pragma unroll
        for (uint32_t j = 0; j < kExpAhead; j++) {
            const int64_t idx = (int64_t)x[j] - mx + (((int64_t)1 << p.a.bit_shift) - 1);
            const bool ok = idx >= 0 && idx < ((int64_t)1 << p.a.index_bits);
            e[j] = p.a.d_exp_table[ok ? idx : 0];
            if (!ok && t + j * step < n) bad |= (uint32_t)kWitIndex;
        }
#pragma unroll
        for (uint32_t j = 0; j < kExpAhead; j++) {
            const uint32_t i = t + j * step;
            if (i >= n) break;
            if (e[j] < 0) bad |= (uint32_t)kWitSum;
            p.a.d_exp[o + i] = e[j];
            if (p.a.d_shifted) p.a.d_shifted[o + i] = (int32_t)((int64_t)x[j] - mx);
            sum += (unsigned long long)(e[j] < 0 ? 0 : e[j]);
        }
    }
    return sum;
}

// floor((e * scale + sum / 2) / sum) for e <= sum: the quotient is at most `scale`, so one product in double precision is off by one at most
__device__ __forceinline__ uint32_t probability(uint32_t e, uint64_t scale, uint64_t sum, double inv) {
    const uint64_t num = e * scale + (sum >> 1);
    uint64_t q = (uint64_t)((double)num * inv);
    const int64_t rest = (int64_t)(num - q * sum);
    if (rest < 0) q--;
    else if (rest >= (int64_t)sum) q++;
    return (uint32_t)q;
}

// 2 * scale * e - sum * (2 * prob - 1), within 0 .. 2 sum: less than 2^63
__device__ __forceinline__ uint64_t lookup_query(uint32_t e, int64_t scale, uint64_t sum, uint32_t prob) {
    return (uint64_t)e * 2 * (uint64_t)scale - sum * (2 * (uint64_t)prob - 1);
}

// Where a tensor of the proof holds a sum or a query, its low 32 bits; the bit says that they are not all of it.
__device__ __forceinline__ void store_sum(int32_t* to, uint64_t x, uint32_t& bad) {
    bad |= x > (uint64_t)INT32_MAX ? (uint32_t)kWitSumWide : 0u;
    *to = (int32_t)x;
}

// The threads of a workgroup that share a query head: as many as there are for each, a power of two, in lanes side by side.
struct RowThreads {
    uint32_t each, r, from, lanes;
    bool mine, leads;            // of a row that there is; the first of its lanes in a wave
    __device__ __forceinline__ RowThreads(uint32_t threads, uint32_t R) {
        each = threads;
        while (each * R > threads) each >>= 1;
        r = threadIdx.x / each;
        from = threadIdx.x - r * each;
        lanes = min(each, 64u);
        mine = r < R;
        leads = threadIdx.x % lanes == 0;
    }
    template <class T, class F>
    __device__ __forceinline__ T all(T v, F f) const {
        for (uint32_t k = lanes / 2; k >= 1; k >>= 1) v = f(v, __shfl_xor(v, k, 64));
        return v;
    }
};

// Probabilities of this thread's positions of its row, from load(position), its exponential; written if `write`, and their digits
// in LDS: [step of 32][plane][lane group][row], operands of 8 positions each, zero up to a whole number of 32 positions and for
// pages outside the cache.  Returns the sum of the probabilities that the values are multiplied with.
template <int PP, uint32_t AHEAD, class F>          // planes of the probabilities, positions under way a thread
__device__ __forceinline__ unsigned long long probabilities(const AttendArgs& p, const Tile& w, const RowThreads& row, uint32_t t0, uint32_t n, const int64_t* off,
                                                            unsigned long long sum, bool write, uint32_t* digits, uint32_t& bad, F load) {
    const size_t o = (w.row0 + row.r) * p.a.max_len + t0;
    const double inv = 1.0 / (double)sum;
    const uint32_t filled = (n + 31) / 32 * 32;
    unsigned long long all = 0;
#pragma unroll 1
    for (uint32_t first = row.from; first < filled; first += AHEAD * row.each) {
        uint32_t e[AHEAD];
#pragma unroll
        for (uint32_t a = 0; a < AHEAD; a++) e[a] = first + a * row.each < n ? load(first + a * row.each) : 0;
#pragma unroll
        for (uint32_t a = 0; a < AHEAD; a++) {
            const uint32_t i = first + a * row.each;
            if (i >= filled) break;
            uint32_t pr = 0;
            if (i < n) {
                pr = probability(e[a], (uint64_t)p.a.prob_scale, sum, inv);
                if (write) {
                    if (p.a.d_prob) p.a.d_prob[o + i] = (int32_t)pr;
                    if (p.a.d_query) store_sum(&p.a.d_query[o + i], lookup_query(e[a], p.a.prob_scale, sum, pr), bad);
                }
                if (off[i] < 0) pr = 0;
            }
            all += pr;
            const uint32_t d = digits_of((int32_t)pr);
            uint8_t* out = reinterpret_cast<uint8_t*>(digits) + ((((i >> 5) * PP * 4 + ((i >> 3) & 3u)) * w.R + row.r) << 3) + (i & 7u);
#pragma unroll
            for (int k = 0; k < PP; k++) out[k * 32 * w.R] = (uint8_t)(d >> (8 * k));
        }
    }
    return row.all(all, [](unsigned long long x, unsigned long long y) { return x + y; });
}

// Products of the probabilities with 32 elements (from e) of n values.  A wave takes 32 positions a step: lane l reads the
// elements 2 (l % 16), + 1 of the positions 8 (l / 16) .. + 8, a line among 16 lanes, and turns four positions' words into the
// planes of four positions, in registers.  Every next step is on its way while this one multiplies.
template <bool VEC, int PP>
struct ValueProducts {
    static constexpr int G = PP + 3;
    v2i_t next[8];
    v4i_t acc[2][G];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int g = 0; g < G; g++) acc[j][g] = v4i_t{0, 0, 0, 0};
    }
    __device__ __forceinline__ void fetch(const AttendArgs& p, const Tile& w, const int64_t* off, uint32_t e, uint32_t s) {
        const int32_t* v = p.c.d_v + (int64_t)w.kv * p.c.head_stride;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const int64_t at = off[s * 32 + w.kg * 8 + i];
            next[i] = load2<VEC>(v + (at < 0 ? 0 : at), e + 2 * w.col, p.c.dim);
        }
    }
    // steps s, s + apart, ... below `halves`; the first has been fetched
    __device__ __forceinline__ void run(const AttendArgs& p, const Tile& w, const int64_t* off, const uint32_t* digits, uint32_t e, uint32_t s, uint32_t apart, uint32_t halves) {
        const uint32_t row = w.row();
        for (; s < halves; s += apart) {
            v2i_t x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = next[i];
            if (s + apart < halves) fetch(p, w, off, e, s + apart);
            long pa[PP];
#pragma unroll
            for (int k = 0; k < PP; k++) pa[k] = reinterpret_cast<const long*>(digits)[((s * PP + k) * 4 + w.kg) * w.R + row];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                uint32_t p0[4], p1[4];
                transpose4((uint32_t)x[0][j], (uint32_t)x[1][j], (uint32_t)x[2][j], (uint32_t)x[3][j], p0);
                transpose4((uint32_t)x[4][j], (uint32_t)x[5][j], (uint32_t)x[6][j], (uint32_t)x[7][j], p1);
#pragma unroll
                for (int k2 = 0; k2 < 3; k2++) p0[k2] ^= kByteTops, p1[k2] ^= kByteTops;
#pragma unroll
                for (int k2 = 0; k2 < 4; k2++) {
                    const long vb = (long)(((uint64_t)p1[k2] << 32) | p0[k2]);
#pragma unroll
                    for (int k = 0; k < PP; k++) acc[j][k + k2] = __builtin_amdgcn_mfma_i32_16x16x32_i8(pa[k], vb, acc[j][k + k2], 0, 0, 0);
                }
            }
        }
    }
    // added to 64-bit sums [row][width] in LDS, this wave's 32 elements from `at`, as far as they are within the width
    __device__ __forceinline__ void add(const Tile& w, unsigned long long* total, uint32_t width, uint32_t at) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t r = 4 * i + w.kg, el = at + 2 * w.col + j;
                if (4 * i < w.R && r < w.R && el < width) {
                    uint64_t y = 0;
#pragma unroll
                    for (int g = G - 1; g >= 0; g--) y = (y << 8) + (uint64_t)(int64_t)acc[j][g][i];
                    atomicAdd(&total[r * width + el], (unsigned long long)y);
                }
            }
    }
};

__device__ __forceinline__ void write_out(const AttendArgs& p, size_t row, uint32_t e, int64_t y, uint32_t& bad) {
    int32_t q, rem;
    p.out.apply(y, q, rem, bad);
    p.a.d_out[row * p.c.dim + e] = q;
    if (p.a.d_out_rem) p.a.d_out_rem[row * p.c.dim + e] = rem;
}

// Rows with nothing to attend to: elements e0 .. e0 + width of the output, and the maximum and sum if `rows`.
__device__ __forceinline__ void write_empty(const AttendArgs& p, const Tile& w, uint32_t e0, uint32_t width, bool rows) {
    for (uint32_t i = threadIdx.x; i < w.R * width; i += blockDim.x) {
        const uint32_t r = i / width, e = e0 + i - r * width;
        if (e >= p.c.dim) continue;
        p.a.d_out[(w.row0 + r) * p.c.dim + e] = 0;
        if (p.a.d_out_rem) p.a.d_out_rem[(w.row0 + r) * p.c.dim + e] = 0;
    }
    if (rows && threadIdx.x < w.R) {
        if (p.a.d_max) p.a.d_max[w.row0 + threadIdx.x] = 0;
        if (p.a.d_sum) p.a.d_sum[w.row0 + threadIdx.x] = 0;
    }
}

// ---- the launches over chunks
// Scores of `rows` query heads with a chunk of the keys.  Bound by reading the keys: 131072 positions of 8 heads of 128 for 32 query
// heads, 570 MB with what is written, 121 us, 4.7 TB/s, as a copy.
template <bool VEC>
__global__ void __launch_bounds__(256, 4) wit_attend_scores_kernel(AttendArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ unsigned long long q_sum[16];
    __shared__ uint32_t over_any;
    const uint32_t per_chunk = p.c.heads * p.plan.tiles, index = blockIdx.x / per_chunk, within = blockIdx.x - index * per_chunk;
    uint32_t b = blockIdx.y, chunk = index, lo, hi, bad = 0;
    bool fits;
    if (p.plan.counted && !find_chunk(p, index, p.plan.score_chunk, b, chunk, lo, hi, fits)) return;
    const Tile w(p, b, within);
    // what does not depend on the sequence's length is requested beside it
    Queries queries;
    queries.first(p, w);
    Offsets offsets;
    offsets.request(p, w.b, (uint64_t)chunk * p.plan.score_chunk, p.plan.score_chunk);
    if (!p.plan.counted) fits = span_of(p, w.b, lo, hi);
    if (!fits && chunk == 0 && within == 0 && threadIdx.x == 0) atomicOr(p.status, (uint32_t)kWitIndex);
    const uint64_t start = (uint64_t)lo + (uint64_t)chunk * p.plan.score_chunk;
    if (start >= hi) return;
    const uint32_t t0 = (uint32_t)start, n = min(hi - t0, p.plan.score_chunk);
    if (threadIdx.x < 16) q_sum[threadIdx.x] = 0;
    if (threadIdx.x == 0) over_any = 0;
    // behind the digits: the positions' offsets and the scores' 64-bit sums, so that nothing but the keys is read or written on
    // the way (waiting for any other load or store would wait for all keys requested before it)
    int64_t* off = reinterpret_cast<int64_t*>(lds + (size_t)5 * 16 * p.plan.dim64 * p.plan.rows);
    uint64_t* sums = reinterpret_cast<uint64_t*>(off + p.plan.score_chunk);
    if (offsets.store(p, w.b, t0, n, n, off)) bad |= (uint32_t)kWitIndex;
    const bool apart = p.plan.score_apart;
    if (apart)
        for (uint32_t i = threadIdx.x; i < w.R * p.plan.score_chunk; i += 256) sums[i] = 0;
    __syncthreads();
    queries.store(p, w, lds, q_sum, &over_any);
    __syncthreads();
    score_products<VEC, 4>(p, w, n, off, lds, over_any != 0, apart, [&](uint32_t r, uint32_t i, bool there, uint64_t y) {
        if (!there) return;
        uint64_t* sum = &sums[r * p.plan.score_chunk + i];
        if (apart) atomicAdd(reinterpret_cast<unsigned long long*>(sum), (unsigned long long)y);
        else *sum = y;
    });
    __syncthreads();
    score_rows(p, w, t0, n, off, sums, p.plan.score_chunk, q_sum, bad,
               [&](uint32_t r, int32_t mx) { p.chunk_max[(w.row0 + r) * p.plan.score_chunks + chunk] = mx; });
    if (bad) atomicOr(p.status, bad);
}

template <class T, class F>
__device__ __forceinline__ T block_all(T v, F f) {
    __shared__ T sh[kBlock / 64];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < kBlock / 64; w++) v = f(v, sh[w]);
    __syncthreads();
    return v;
}

// Exponentials of a chunk of one row, and their sum.  Bound by the gathers: 32 rows of 131072, 31 us, 135 a nanosecond from a table
// of 4 MB that the L2 of each die shares with the scores.
__global__ void __launch_bounds__(kBlock) wit_attend_exp_kernel(AttendArgs p) {
    const uint32_t b = blockIdx.z;
    const size_t row = (size_t)b * p.a.heads + blockIdx.y;
    uint32_t lo, hi, bad = 0;
    span_of(p, b, lo, hi);
    const uint64_t start = (uint64_t)lo + (uint64_t)blockIdx.x * p.plan.exp_chunk;
    if (start >= hi) return;
    const uint32_t t0 = (uint32_t)start, n = min(hi - t0, p.plan.exp_chunk), parts = (hi - lo - 1) / p.plan.score_chunk + 1;
    int32_t mx = INT32_MIN;
    for (uint32_t i = threadIdx.x; i < parts; i += kBlock) mx = max(mx, p.chunk_max[row * p.plan.score_chunks + i]);
    mx = block_all(mx, [](int32_t x, int32_t y) { return max(x, y); });
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.a.d_max) p.a.d_max[row] = mx;
    unsigned long long sum = exponentials(p, row, t0, threadIdx.x, kBlock, n, mx, bad);
    sum = block_all(sum, [](unsigned long long x, unsigned long long y) { return x + y; });
    if (threadIdx.x == 0) p.sums[row * p.plan.exp_chunks + blockIdx.x] = sum;
    if (bad) atomicOr(p.status, bad);
}

// Probabilities of a chunk of the positions for `rows` query heads, and their products with 32 * blocks elements of the values.
// The waves take different blocks of 32 elements, or every second or fourth step.  Bound by reading the values: the
// 131072 positions' 587 MB with probabilities and queries in 128 us, 4.6 TB/s.
constexpr uint32_t kProbAhead = 4;
template <bool VEC, int PP>
__global__ void __launch_bounds__(256, 4) wit_attend_values_kernel(AttendArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ unsigned long long e_sum[16], p_sum[16];
    const uint32_t per_chunk = p.c.heads * p.plan.tiles * p.plan.groups, index = blockIdx.x / per_chunk, within = blockIdx.x - index * per_chunk;
    const uint32_t group = within % p.plan.groups;
    uint32_t b = blockIdx.y, chunk = index, lo, hi, bad = 0;
    bool fits;
    if (p.plan.counted && !find_chunk(p, index, p.plan.value_chunk, b, chunk, lo, hi, fits)) return;
    const Tile w(p, b, within / p.plan.groups);
    Offsets offsets;
    offsets.request(p, w.b, (uint64_t)chunk * p.plan.value_chunk, p.plan.value_chunk);
    if (!p.plan.counted) span_of(p, w.b, lo, hi);
    const uint64_t start = (uint64_t)lo + (uint64_t)chunk * p.plan.value_chunk;
    const bool direct = hi - lo <= p.plan.value_chunk;          // the whole row is this workgroup's
    const uint32_t e0 = group * p.plan.blocks * 32, width = p.plan.blocks * 32, dim = p.c.dim;
    if (start >= hi) {
        if (lo == hi && chunk == 0) write_empty(p, w, e0, width, group == 0);
        return;
    }
    const uint32_t t0 = (uint32_t)start, n = min(hi - t0, p.plan.value_chunk);
    int64_t* off = reinterpret_cast<int64_t*>(lds + (size_t)p.plan.value_chunk * w.R * PP / 4);        // behind the digits
    if (threadIdx.x < 16) e_sum[threadIdx.x] = p_sum[threadIdx.x] = 0;
    offsets.store(p, w.b, t0, n, (n + 63) / 64 * 64, off);
    __syncthreads();
    const uint32_t block = w.wave % p.plan.blocks, apart = 4 / p.plan.blocks, e = e0 + 32 * block, halves = e < dim ? (n + 31) / 32 : 0, s = w.wave / p.plan.blocks;
    ValueProducts<VEC, PP> products;
    if (s < halves) products.fetch(p, w, off, e, s);            // under way while the probabilities are computed
    const uint32_t parts = (hi - lo - 1) / p.plan.exp_chunk + 1;
    const RowThreads row(256, w.R);
    const size_t at = w.row0 + min(row.r, w.R - 1);
    if (row.mine) {
        unsigned long long sum = 0;
        for (uint32_t i = row.from; i < parts; i += row.each) sum += p.sums[at * p.plan.exp_chunks + i];
        sum = row.all(sum, [](unsigned long long x, unsigned long long y) { return x + y; });
        if (row.leads) atomicAdd(&e_sum[row.r], sum);
    }
    __syncthreads();
    if (row.mine) {
        unsigned long long sum = e_sum[row.r];
        if (sum == 0) {
            bad |= (uint32_t)kWitSum;
            sum = 1;
        }
        if (chunk == 0 && group == 0 && row.from == 0 && p.a.d_sum) store_sum(&p.a.d_sum[at], sum, bad);
        const int32_t* exps = p.a.d_exp + at * p.a.max_len + t0;
        const unsigned long long mine = probabilities<PP, kProbAhead>(p, w, row, t0, n, off, sum, group == 0, lds, bad, [&](uint32_t i) { return (uint32_t)max(exps[i], 0); });
        if (row.leads) atomicAdd(&p_sum[row.r], mine);
    }
    __syncthreads();
    products.clear();
    products.run(p, w, off, lds, e, s, apart, halves);
    __syncthreads();
    unsigned long long* total = reinterpret_cast<unsigned long long*>(lds);          // [rows][32 * blocks]
    for (uint32_t i = threadIdx.x; i < w.R * width; i += 256) total[i] = (unsigned long long)kCacheOffset * p_sum[i / width];
    __syncthreads();
    products.add(w, total, width, 32 * block);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < w.R * width; i += 256) {
        const uint32_t r = i / width, el = e0 + i - r * width;
        if (el >= dim) continue;
        if (direct) write_out(p, w.row0 + r, el, (int64_t)total[i], bad);
        else p.part[((w.row0 + r) * p.plan.value_chunks + chunk) * dim + el] = (int64_t)total[i];
    }
    if (bad) atomicOr(p.status, bad);
}

// The chunks' partial sums of 64 elements of one row.  A wave for each four chunks, at most sixteen: with few of them the rows are
// many, and more waves would only stand in line (64 sequences of 32 heads of 128 and 8 chunks: 5.2 us, with sixteen waves 11.2).
constexpr uint32_t kJoinThreads = 1024;
__global__ void __launch_bounds__(kJoinThreads) wit_attend_join_kernel(AttendArgs p) {
    __shared__ int64_t sh[kJoinThreads];
    const uint32_t h = blockIdx.y, b = blockIdx.z, e = blockIdx.x * 64 + (threadIdx.x & 63u), dim = p.c.dim;
    const size_t row = (size_t)b * p.a.heads + h;
    uint32_t lo, hi, bad = 0;
    span_of(p, b, lo, hi);
    if (hi - lo <= p.plan.value_chunk) return;
    const uint32_t parts = (hi - lo - 1) / p.plan.value_chunk + 1;
    const uint32_t waves = blockDim.x >> 6;
    int64_t y = 0;
    if (e < dim) {
#pragma unroll 8
        for (uint32_t i = threadIdx.x >> 6; i < parts; i += waves) y += p.part[(row * p.plan.value_chunks + i) * dim + e];
    }
    sh[threadIdx.x] = y;
    __syncthreads();
    if (threadIdx.x < 64 && e < dim) {
        for (uint32_t i = 1; i < waves; i++) y += sh[threadIdx.x + 64 * i];
        write_out(p, row, e, y, bad);
    }
    if (bad) atomicOr(p.status, bad);
}

// ---- the same in one launch, a workgroup for all positions of its query heads (at most kWholeMost): what goes from step to step
// stays on chip.  A few positions leave nothing but latencies - of loads that depend on each other, and of instructions that run
// once - so eight waves share the positions, and the softmax takes one position a thread in short loops.  37 positions of 32 heads of 128:
// 10.2 us.
constexpr uint32_t kWholeWaves = 8, kWholeThreads = 64 * kWholeWaves;
template <bool VEC, int PP>
__global__ void __launch_bounds__(kWholeThreads, 4) wit_attend_whole_kernel(AttendArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ unsigned long long q_sum[16], e_sum[16], p_sum[16];
    __shared__ int32_t row_max[16];
    __shared__ uint32_t over_any;
    constexpr uint32_t C = token::kWholeMost;
    const Tile w(p, blockIdx.y, blockIdx.x);
    const uint32_t dim = p.c.dim;
    uint32_t lo, hi, bad = 0;
    Queries queries;
    queries.first(p, w);
    Offsets offsets;
    offsets.request(p, w.b, 0, C);
    const bool fits = span_of(p, w.b, lo, hi);
    if (!fits && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(p.status, (uint32_t)kWitIndex);
    if (lo == hi) {
        write_empty(p, w, 0, dim, true);
        return;
    }
    const uint32_t n = hi - lo;
    int64_t* off = reinterpret_cast<int64_t*>(lds);                                        // [C]
    unsigned long long* total = reinterpret_cast<unsigned long long*>(off + C);            // the scores' sums [rows][C], then the output's [rows][dim]
    uint32_t* scores = reinterpret_cast<uint32_t*>(total + (size_t)w.R * max(dim, C));      // [rows][C], then the exponentials
    uint32_t* digits = scores + w.R * C;                                                    // of the queries, then of the probabilities
    if (threadIdx.x < 16) {
        q_sum[threadIdx.x] = e_sum[threadIdx.x] = p_sum[threadIdx.x] = 0;
        row_max[threadIdx.x] = INT32_MIN;
    }
    if (threadIdx.x == 0) over_any = 0;
    __syncthreads();
    const uint32_t filled = (n + 31) / 32 * 32;
    if (offsets.store(p, w.b, lo, n, filled, off)) bad |= (uint32_t)kWitIndex;
    queries.store(p, w, digits, q_sum, &over_any);
    __syncthreads();
    score_products<VEC, kWholeWaves>(p, w, n, off, digits, over_any != 0, false, [&](uint32_t r, uint32_t i, bool there, uint64_t y) {
        if (there) total[r * C + i] = y;
    });
    // the values' first step is under way during the softmax
    const uint32_t dim32 = (dim + 31) / 32, blocks = dim32 > 4 ? 8 : dim32 > 2 ? 4 : dim32, apart = kWholeWaves / blocks, block = w.wave % blocks, s = w.wave / blocks, halves = (n + 31) / 32;
    ValueProducts<VEC, PP> products;
    if (32 * block < dim && s < halves) products.fetch(p, w, off, 32 * block, s);
    __syncthreads();
    const RowThreads row(kWholeThreads, w.R);
    const uint32_t r = row.r, from = row.from, each = row.each;
    const bool mine = row.mine, leads = row.leads;
    const size_t o = (w.row0 + min(r, w.R - 1)) * p.a.max_len + lo;
    if (mine) {
        const uint64_t more = (uint64_t)kCacheOffset * q_sum[r];
        int32_t mx = INT32_MIN;
#pragma unroll 1
        for (uint32_t i = from; i < n; i += each) {
            int32_t q, rem;
            p.qk.apply(off[i] < 0 ? 0 : (int64_t)(total[r * C + i] + more), q, rem, bad);          // a page outside the cache: zero
            if (p.a.d_scores) p.a.d_scores[o + i] = q;
            if (p.a.d_scores_rem) p.a.d_scores_rem[o + i] = rem;
            scores[r * C + i] = (uint32_t)q;
            mx = max(mx, q);
        }
        mx = row.all(mx, [](int32_t x, int32_t y) { return max(x, y); });
        if (leads) atomicMax(&row_max[r], mx);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < w.R * dim; i += kWholeThreads) total[i] = 0;
    if (mine) {
        const int32_t mx = row_max[r];
        unsigned long long sum = 0;
#pragma unroll 1
        for (uint32_t first = from; first < n; first += 4 * each) {          // four gathers under way a thread
            int32_t x[4], e[4];
#pragma unroll
            for (uint32_t a = 0; a < 4; a++) {
                const uint32_t i = first + a * each;
                x[a] = i < n ? (int32_t)scores[r * C + i] : mx;          // its own positions only: the others' become exponentials meanwhile
                const int64_t idx = (int64_t)x[a] - mx + (((int64_t)1 << p.a.bit_shift) - 1);
                const bool ok = idx >= 0 && idx < ((int64_t)1 << p.a.index_bits);
                if (!ok && i < n) bad |= (uint32_t)kWitIndex;
                e[a] = p.a.d_exp_table[ok ? idx : 0];
            }
#pragma unroll
            for (uint32_t a = 0; a < 4; a++) {
                const uint32_t i = first + a * each;
                if (i >= n) break;
                if (p.a.d_shifted) p.a.d_shifted[o + i] = (int32_t)((int64_t)x[a] - mx);
                if (p.a.d_exp) p.a.d_exp[o + i] = e[a];
                if (e[a] < 0) bad |= (uint32_t)kWitSum;
                e[a] = max(e[a], 0);
                scores[r * C + i] = (uint32_t)e[a];
                sum += (uint32_t)e[a];
            }
        }
        sum = row.all(sum, [](unsigned long long x, unsigned long long y) { return x + y; });
        if (leads) atomicAdd(&e_sum[r], sum);
    }
    __syncthreads();
    if (mine) {
        unsigned long long sum = e_sum[r];
        if (sum == 0) {
            bad |= (uint32_t)kWitSum;
            sum = 1;
        }
        if (from == 0) {
            if (p.a.d_max) p.a.d_max[w.row0 + r] = row_max[r];
            if (p.a.d_sum) store_sum(&p.a.d_sum[w.row0 + r], sum, bad);
        }
        const unsigned long long all = probabilities<PP, 1>(p, w, row, lo, n, off, sum, true, digits, bad, [&](uint32_t i) { return scores[r * C + i]; });
        if (leads) atomicAdd(&p_sum[r], all);
    }
    __syncthreads();
    for (uint32_t el = 32 * block; el < dim && s < halves; el += 32 * blocks) {
        if (el != 32 * block) products.fetch(p, w, off, el, s);
        products.clear();
        products.run(p, w, off, digits, el, s, apart, halves);
        products.add(w, total, dim, el);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < w.R * dim; i += kWholeThreads) {
        const uint32_t row = i / dim;
        write_out(p, w.row0 + row, i - row * dim, (int64_t)(total[i] + (unsigned long long)kCacheOffset * p_sum[row]), bad);
    }
    if (bad) atomicOr(p.status, bad);
}

}  // namespace grape

using namespace grape;

extern "C" {

size_t grape_wit_paged_attention_workspace(uint32_t seqs, uint32_t heads, uint32_t cache_heads, uint32_t dim, uint32_t max_len) {
    return token::attention_workspace(seqs, heads, cache_heads, dim, max_len);
}

int grape_wit_paged_attention(const grape_wit_attention_args* args, const grape_wit_cache* cache, grape_stream_t st) {
    GRAPE_REQUIRE(initialised(), "grape_init has not been called");
    GRAPE_REFUSED_IF(token::refuse_attention(args, cache));
    if (args->seqs == 0) return GRAPE_OK;
    AttendArgs p;
    p.a = *args;
    p.c = *cache;
    grape_wit_attention_args& a = p.a;
    token::attention_plan(a.seqs, a.heads, p.c.heads, p.c.dim, a.max_len, p.plan);
    const token::AttentionPlan& pl = p.plan;
    uint8_t* ws = (uint8_t*)a.d_workspace;
    if (!pl.whole && !a.d_scores) a.d_scores = (int32_t*)(ws + pl.at_scores);
    if (!pl.whole && !a.d_exp) a.d_exp = (int32_t*)(ws + pl.at_exp);
    p.chunk_max = (int32_t*)(ws + pl.at_max);
    p.sums = (unsigned long long*)(ws + pl.at_sum);
    p.part = (int64_t*)(ws + pl.at_part);
    p.page = token::fast_div(p.c.page_size);
    p.qk = scaler(a.qk_scale);
    p.out = scaler(a.out_scale);
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status);
    if (rc) return rc;
    auto aligned = [&](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    const bool vec = p.c.dim % 4 == 0 && ((p.c.page_stride | p.c.token_stride | p.c.head_stride) & 3) == 0 && aligned(p.c.d_k) && aligned(p.c.d_v);
    const int planes = a.prob_scale <= ((int64_t)1 << 22) ? 3 : 4;
    if (pl.whole) {
        const dim3 grid(p.c.heads * pl.tiles, a.seqs);
        if (vec && planes == 3) wit_attend_whole_kernel<true, 3><<<grid, kWholeThreads, pl.whole_lds, s>>>(p);
        else if (vec) wit_attend_whole_kernel<true, 4><<<grid, kWholeThreads, pl.whole_lds, s>>>(p);
        else if (planes == 3) wit_attend_whole_kernel<false, 3><<<grid, kWholeThreads, pl.whole_lds, s>>>(p);
        else wit_attend_whole_kernel<false, 4><<<grid, kWholeThreads, pl.whole_lds, s>>>(p);
        GRAPE_LAUNCH_CHECK();
        return GRAPE_OK;
    }
    const size_t score_lds = (size_t)pl.dim64 * 5 * 64 * pl.rows + (size_t)pl.score_chunk * 8 * (pl.rows + 1);
    const size_t value_lds = std::max<size_t>((size_t)pl.value_chunk * (pl.rows * planes + 8), (size_t)pl.rows * pl.blocks * 32 * 8);
    // the heads of one chunk are neighbours: they read the same tokens' lines of memory at the same time
    const uint32_t head_tiles = p.c.heads * pl.tiles;
    const uint32_t along = pl.counted ? a.seqs : 1, across = pl.counted ? 1 : a.seqs;
    const dim3 score_grid(std::max(1u, pl.score_chunks) * head_tiles * along, across), value_grid(std::max(1u, pl.value_chunks) * head_tiles * pl.groups * along, across);
    if (vec) wit_attend_scores_kernel<true><<<score_grid, 256, score_lds, s>>>(p);
    else wit_attend_scores_kernel<false><<<score_grid, 256, score_lds, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    if (a.max_len) {
        wit_attend_exp_kernel<<<dim3(pl.exp_chunks, a.heads, a.seqs), kBlock, 0, s>>>(p);
        GRAPE_LAUNCH_CHECK();
    }
    if (vec && planes == 3) wit_attend_values_kernel<true, 3><<<value_grid, 256, value_lds, s>>>(p);
    else if (vec) wit_attend_values_kernel<true, 4><<<value_grid, 256, value_lds, s>>>(p);
    else if (planes == 3) wit_attend_values_kernel<false, 3><<<value_grid, 256, value_lds, s>>>(p);
    else wit_attend_values_kernel<false, 4><<<value_grid, 256, value_lds, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    if (pl.value_chunks > 1) {
        const uint32_t waves = std::min(kJoinThreads / 64, (pl.value_chunks + 3) / 4);
        wit_attend_join_kernel<<<dim3(pl.dim64, a.heads, a.seqs), 64 * waves, 0, s>>>(p);
        GRAPE_LAUNCH_CHECK();
    }
    return GRAPE_OK;
}

}  // extern "C"

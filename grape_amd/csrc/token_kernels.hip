// The witness of new tokens: rotation and append to a paged cache, attention of one token a sequence over that cache, and
// products with 4-bit weights.  The arithmetic is that of witness_kernels.hip: exact 64-bit products, rescaled.
#include <algorithm>
#include "common.hpp"
#include "token_geometry.hpp"
#include "witness_device.hpp"

namespace grape {

typedef int v4i_t __attribute__((ext_vector_type(4)));

// rescale64 for a scale that is the same for a whole launch: where it is no power of two the quotient comes from a product in
// double precision.  That is off by at most 2^-52 of itself, 2^11 for the largest dividend, so a second one of what is left
// over is off by one at most.
struct Scaler {
    int64_t s;
    double inv;
    int sh;
    __device__ __forceinline__ void apply(int64_t y, int32_t& q, int32_t& r, uint32_t& bad) const {
        const int64_t t = y + (s >> 1);
        int64_t qq;
        if (sh >= 0) {
            qq = t >> sh;
        } else {
            qq = (int64_t)floor((double)t * inv);
            int64_t rest = t - qq * s;
            if (rest < 0 || rest >= s) {
                qq += (int64_t)floor((double)rest * inv);
                rest = t - qq * s;
                if (rest < 0) qq--;
                else if (rest >= s) qq++;
            }
        }
        bad |= (qq != (int64_t)(int32_t)qq) ? (uint32_t)kWitQuotient : 0u;
        q = (int32_t)qq;
        r = (int32_t)(y - qq * s);
    }
};
static Scaler scaler(int64_t s) { return Scaler{s, 1.0 / (double)s, log2_exact(s)}; }

// x = sum_p d_p 256^p with d_p in -128..127 for p < 3: the bytes of the word.  The top digit is 128 above kDigitTop and does
// not fit its byte there.
constexpr int32_t kDigitTop = 0x7f7f7f7f;
__device__ __forceinline__ uint32_t digits_of(int32_t x) { return ((uint32_t)x + 0x00808080u) ^ 0x00808080u; }

// out[p] = byte p of w0, w1, w2, w3
__device__ __forceinline__ void transpose4(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t out[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w1, w0, 0x05010400u), b = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(w1, w0, 0x07030602u), d = __builtin_amdgcn_perm(w3, w2, 0x07030602u);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// ------------------------------------------------------------------------------------------------
// Rotation and append.  A unit is one pair of a rotated head or two elements that only move; a token's units are those of its
// query heads, its key heads and its value heads.
// ------------------------------------------------------------------------------------------------
struct AppendArgs {
    grape_wit_rope_append_args a;
    grape_wit_cache c;
    uint32_t units, head_units;   // of a token, of a head
    uint64_t total;
    int shift;
    uint32_t* status;
};

__global__ void __launch_bounds__(kBlock) wit_append_kernel(AppendArgs p) {
    const uint64_t i = (uint64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= p.total) return;
    const grape_wit_rope_append_args& a = p.a;
    const grape_wit_cache& c = p.c;
    const uint32_t t = (uint32_t)(i / p.units), u = (uint32_t)(i - (uint64_t)t * p.units);
    const uint32_t hh = u / p.head_units, j = u - hh * p.head_units;
    auto kind = [&](uint32_t tok) { return token::append_kind(c, a.d_slots[tok], a.rot ? a.d_positions[tok] : 0, a.rot, a.table_rows); };
    const int64_t slot = a.d_slots[t];
    const int k = kind(t);
    if (k == 2 && u == 0) atomicOr(p.status, (uint32_t)kWitIndex);
    if (k) return;
    const bool is_q = hh < a.heads, is_k = !is_q && hh < a.heads + c.heads;
    const uint32_t h = is_q ? hh : is_k ? hh - a.heads : hh - a.heads - c.heads;
    const int32_t* x = is_q ? a.d_q + t * a.q_stride : is_k ? a.d_k + t * a.k_stride : a.d_v + t * a.v_stride;
    x += (size_t)h * c.dim;
    int32_t *q, *r = nullptr;
    if (is_q) {
        const size_t o = ((size_t)t * a.heads + h) * c.dim;
        q = a.d_q_out + o;
        if (a.d_q_rem) r = a.d_q_rem + o;
    } else {
        const int64_t pg = slot / c.page_size;
        q = (is_k ? c.d_k : c.d_v) + token::token_offset(c, (int32_t)pg, (uint32_t)(slot - pg * c.page_size)) + h * c.head_stride;
        if (is_k && a.d_k_rem) r = a.d_k_rem + ((size_t)t * c.heads + h) * c.dim;
        for (uint32_t o = t + 1; o < a.tokens; o++)
            if (a.d_slots[o] == slot && kind(o) == 0) {
                q = nullptr;
                break;
            }
    }
    uint32_t bad = 0;
    if ((is_q || is_k) && 2 * j < a.rot) {
        const uint32_t half = a.rot / 2, e0 = a.interleaved ? 2 * j : j, e1 = a.interleaved ? 2 * j + 1 : j + half;
        const size_t row = (size_t)a.d_positions[t] * half + j;
        const int64_t x0 = x[e0], x1 = x[e1], cs = a.d_cos[row], sn = a.d_sin[row];
        int32_t q0, r0, q1, r1;
        rescale64(x0 * cs - x1 * sn, a.scale, p.shift, q0, r0, bad);
        rescale64(x0 * sn + x1 * cs, a.scale, p.shift, q1, r1, bad);
        if (q) q[e0] = q0, q[e1] = q1;
        if (r) r[e0] = r0, r[e1] = r1;
    } else {
        for (uint32_t e = 2 * j; e < std::min(2 * j + 2, c.dim); e++) {
            if (q) q[e] = x[e];
            if (r) r[e] = 0;
        }
    }
    if (bad) atomicOr(p.status, bad);
}

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
constexpr uint32_t kByteTops = 0x00808080;

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

// The offsets of a chunk's positions t0 .. t0 + n, made by all 256 threads of a workgroup.  The first page of each thread is
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
        for (uint32_t i = threadIdx.x; i < filled; i += 256) {
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

// Scores of `rows` query heads with a chunk of the keys.  A wave takes 16 positions: lane l reads those elements 64 s + 16 c +
// 4 (l / 16) .. + 4 of position l % 16 that make up its operand of step s (any order of a step's elements will do, as long as
// the queries' digits in LDS have the same), whole lines among the lanes.  Bound by reading the keys.
template <bool VEC>
__global__ void __launch_bounds__(256, 4) wit_attend_scores_kernel(AttendArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ unsigned long long q_sum[16];
    __shared__ uint32_t over_any;
    const uint32_t per_chunk = p.c.heads * p.plan.tiles, chunk = blockIdx.x / per_chunk, head_tile = blockIdx.x - chunk * per_chunk;
    const uint32_t b = blockIdx.y, kv = head_tile / p.plan.tiles, tile = head_tile - kv * p.plan.tiles;
    const uint32_t each = p.a.heads / p.c.heads, h0 = kv * each + tile * p.plan.rows, R = min(p.plan.rows, each - tile * p.plan.rows);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, col = lane & 15u, kg = lane >> 4, dim = p.c.dim, steps = p.plan.dim64;
    uint32_t lo, hi, bad = 0;
    // what does not depend on the sequence's length is requested beside it
    const uint32_t items = R * steps * 16;
    auto query = [&](uint32_t i, int32_t v[4]) {
        const uint32_t r = i / (steps * 16), quad = i - r * (steps * 16);
        const int32_t* q = p.a.d_q + b * p.a.q_stride + (size_t)(h0 + r) * dim;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) v[j] = 4 * quad + j < dim ? q[4 * quad + j] : 0;
    };
    int32_t q4[4] = {0, 0, 0, 0};
    if (threadIdx.x < items) query(threadIdx.x, q4);
    Offsets offsets;
    offsets.request(p, b, (uint64_t)chunk * p.plan.score_chunk, p.plan.score_chunk);
    const bool fits = span_of(p, b, lo, hi);
    if (!fits && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(p.status, (uint32_t)kWitIndex);
    const uint64_t start = (uint64_t)lo + (uint64_t)chunk * p.plan.score_chunk;
    if (start >= hi) return;
    const uint32_t t0 = (uint32_t)start, n = min(hi - t0, p.plan.score_chunk);
    if (threadIdx.x < 16) q_sum[threadIdx.x] = 0;
    if (threadIdx.x == 0) over_any = 0;
    // behind the digits: the positions' offsets and the scores' 64-bit sums, so that nothing but the keys is read or written on
    // the way (waiting for any other load or store would wait for all keys requested before it)
    int64_t* off = reinterpret_cast<int64_t*>(lds + (size_t)5 * 16 * steps * p.plan.rows);
    uint64_t* sums = reinterpret_cast<uint64_t*>(off + p.plan.score_chunk);            // [row][position]
    if (offsets.store(p, b, t0, n, n, off)) bad |= (uint32_t)kWitIndex;
    __syncthreads();
    // the queries' digits: [step][plane 0..4][lane group][row], 16 bytes each; plane 4 holds what a top digit of 128 carries
    for (uint32_t i = threadIdx.x; i < items; i += 256) {
        const uint32_t r = i / (steps * 16), quad = i - r * (steps * 16), s = quad >> 4, c = (quad >> 2) & 3u, g = quad & 3u;
        if (i != threadIdx.x) query(i, q4);
        uint32_t w[4], pl[4], carry = 0;
        long long sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            w[j] = digits_of(q4[j]);
            sum += q4[j];
            carry |= q4[j] > kDigitTop ? 1u << (8 * j) : 0u;
        }
        transpose4(w[0], w[1], w[2], w[3], pl);
        uint32_t* o = lds + (((s * 5 * 4 + g) * R + r) << 2) + c;
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) o[k * 16 * R] = pl[k];
        o[4 * 16 * R] = carry;
        if (carry) over_any = 1;
        // sixteen neighbouring lanes are of one row
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
        if ((i & 15u) == 0) atomicAdd(&q_sum[r], (unsigned long long)sum);
    }
    __syncthreads();
    const bool over = over_any != 0;
    // row m of the product is query head 4 (m % 4) + m / 4: register i of lane l then holds head 4 i + l / 16 at position l % 16,
    // and four heads need one register of every lane
    const uint32_t head = 4 * (col & 3u) + (col >> 2), row = head < R ? head : R - 1;
    const int32_t* keys = p.c.d_k + (int64_t)kv * p.c.head_stride;
    for (uint32_t at = 16 * wave; at < n; at += 64) {
        const int32_t* k = keys + max(off[min(at + col, n - 1)], (int64_t)0);
        v4i_t acc[8];
#pragma unroll
        for (int g = 0; g < 8; g++) acc[g] = v4i_t{0, 0, 0, 0};
        // two steps at a time: their keys are requested together, and other waves multiply meanwhile
        for (uint32_t s = 0; s < steps; s += 2) {
            v4i_t x[8];
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) x[c] = load4<VEC>(k, 64 * s + 16 * c + 4 * kg, dim);
            if (s + 1 < steps) {
#pragma unroll
                for (uint32_t c = 4; c < 8; c++) x[c] = load4<VEC>(k, 64 * s + 16 * c + 4 * kg, dim);
            }
#pragma unroll
            for (uint32_t u = 0; u < 2; u++) {
                if (s + u >= steps) break;
                v4i_t kb[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const v4i_t w = x[4 * u + c];
                    uint32_t pl[4];
                    transpose4((uint32_t)w[0] ^ kByteTops, (uint32_t)w[1] ^ kByteTops, (uint32_t)w[2] ^ kByteTops, (uint32_t)w[3] ^ kByteTops, pl);
#pragma unroll
                    for (int k2 = 0; k2 < 4; k2++) kb[k2][c] = (int)pl[k2];
                }
                const v4i_t* qa = reinterpret_cast<const v4i_t*>(lds) + ((s + u) * 5 * 4 + kg) * R + row;
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
        if (at + col < n) {
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t r = 4 * i + kg;
                if (4 * i < R && r < R) {
                    uint64_t y = 0;
#pragma unroll
                    for (int g = 7; g >= 0; g--) y = (y << 8) + (uint64_t)(int64_t)acc[g][i];
                    sums[r * p.plan.score_chunk + at + col] = y;
                }
            }
        }
    }
    __syncthreads();
    for (uint32_t r = wave; r < R; r += 4) {
        const size_t row = (size_t)b * p.a.heads + h0 + r, o = row * p.a.max_len + t0;
        const uint64_t more = (uint64_t)kCacheOffset * q_sum[r];
        int32_t mx = INT32_MIN;
        for (uint32_t i = lane; i < n; i += 64) {
            const int64_t y = off[i] < 0 ? 0 : (int64_t)(sums[r * p.plan.score_chunk + i] + more);          // a page outside: zero
            int32_t q, rem;
            p.qk.apply(y, q, rem, bad);
            p.a.d_scores[o + i] = q;
            if (p.a.d_scores_rem) p.a.d_scores_rem[o + i] = rem;
            mx = max(mx, q);
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) mx = max(mx, __shfl_xor(mx, d, 64));
        if (lane == 0) p.chunk_max[row * p.plan.score_chunks + chunk] = mx;
    }
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

// Exponentials of a chunk of one row, and their sum.  Bound by the gathers' latency: eight are under way a thread.
constexpr uint32_t kExpAhead = 8;
__global__ void __launch_bounds__(kBlock) wit_attend_exp_kernel(AttendArgs p) {
    const uint32_t h = blockIdx.y, b = blockIdx.z;
    const size_t row = (size_t)b * p.a.heads + h, o = row * p.a.max_len;
    uint32_t lo, hi, bad = 0;
    span_of(p, b, lo, hi);
    const uint64_t start = (uint64_t)lo + (uint64_t)blockIdx.x * p.plan.exp_chunk;
    if (start >= hi) return;
    const uint32_t t0 = (uint32_t)start, t1 = min(hi, t0 + p.plan.exp_chunk), parts = (hi - lo - 1) / p.plan.score_chunk + 1;
    int32_t mx = INT32_MIN;
    for (uint32_t i = threadIdx.x; i < parts; i += kBlock) mx = max(mx, p.chunk_max[row * p.plan.score_chunks + i]);
    mx = block_all(mx, [](int32_t x, int32_t y) { return max(x, y); });
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.a.d_max) p.a.d_max[row] = mx;
    unsigned long long sum = 0;
    for (uint32_t t = t0 + threadIdx.x; t < t1; t += kBlock * kExpAhead) {
        int32_t x[kExpAhead], e[kExpAhead];
#pragma unroll
        for (uint32_t j = 0; j < kExpAhead; j++) x[j] = t + j * kBlock < t1 ? p.a.d_scores[o + t + j * kBlock] : mx;
#pragma unroll
        for (uint32_t j = 0; j < kExpAhead; j++) {
            const int64_t idx = (int64_t)x[j] - mx + (((int64_t)1 << p.a.bit_shift) - 1);
            const bool ok = idx >= 0 && idx < ((int64_t)1 << p.a.index_bits);
            e[j] = p.a.d_exp_table[ok ? idx : 0];
            if (!ok && t + j * kBlock < t1) bad |= (uint32_t)kWitIndex;
        }
#pragma unroll
        for (uint32_t j = 0; j < kExpAhead; j++) {
            const uint32_t i = t + j * kBlock;
            if (i >= t1) break;
            if (e[j] < 0) bad |= (uint32_t)kWitSum;
            p.a.d_exp[o + i] = e[j];
            if (p.a.d_shifted) p.a.d_shifted[o + i] = (int32_t)((int64_t)x[j] - mx);
            sum += (unsigned long long)(e[j] < 0 ? 0 : e[j]);
        }
    }
    sum = block_all(sum, [](unsigned long long x, unsigned long long y) { return x + y; });
    if (threadIdx.x == 0) p.sums[row * p.plan.exp_chunks + blockIdx.x] = sum;
    if (bad) atomicOr(p.status, bad);
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

// Probabilities of a chunk of the positions for `rows` query heads, and their products with 32 * blocks elements of the values.
// A wave reads a line among 16 lanes and turns four positions' words into the planes of four positions, in registers.
// The waves of a workgroup take different blocks of 64 elements, or every second or fourth step.  Bound by reading the values.
constexpr uint32_t kProbAhead = 2;   // four positions each under way a lane
template <bool VEC, int PP>          // PP: planes of the probabilities
__global__ void __launch_bounds__(256, 4) wit_attend_values_kernel(AttendArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ unsigned long long p_sum[16];
    const uint32_t per_chunk = p.c.heads * p.plan.tiles * p.plan.groups, chunk = blockIdx.x / per_chunk, within = blockIdx.x - chunk * per_chunk;
    const uint32_t b = blockIdx.y, head_tile = within / p.plan.groups, group = within - head_tile * p.plan.groups;
    const uint32_t kv = head_tile / p.plan.tiles, tile = head_tile - kv * p.plan.tiles;
    const uint32_t each = p.a.heads / p.c.heads, h0 = kv * each + tile * p.plan.rows, R = min(p.plan.rows, each - tile * p.plan.rows);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, col = lane & 15u, kg = lane >> 4, dim = p.c.dim;
    uint32_t lo, hi, bad = 0;
    Offsets offsets;
    offsets.request(p, b, (uint64_t)chunk * p.plan.value_chunk, p.plan.value_chunk);
    span_of(p, b, lo, hi);
    const uint64_t start = (uint64_t)lo + (uint64_t)chunk * p.plan.value_chunk;
    const bool direct = hi - lo <= p.plan.value_chunk;          // the whole row is this workgroup's
    const uint32_t e0 = group * p.plan.blocks * 32, width = p.plan.blocks * 32;
    const size_t row0 = (size_t)b * p.a.heads + h0;
    if (start >= hi) {
        if (lo == hi && chunk == 0) {                      // nothing to attend to
            for (uint32_t i = threadIdx.x; i < R * width; i += 256) {
                const uint32_t r = i / width, e = e0 + i - r * width;
                if (e >= dim) continue;
                p.a.d_out[(row0 + r) * dim + e] = 0;
                if (p.a.d_out_rem) p.a.d_out_rem[(row0 + r) * dim + e] = 0;
            }
            if (group == 0 && threadIdx.x < R) {
                if (p.a.d_max) p.a.d_max[row0 + threadIdx.x] = 0;
                if (p.a.d_sum) p.a.d_sum[row0 + threadIdx.x] = 0;
            }
        }
        return;
    }
    const uint32_t t0 = (uint32_t)start, n = min(hi - t0, p.plan.value_chunk), steps = (n + 63) / 64;
    // [step of 32][plane][lane group][row] operands of 8 positions each, and the positions' offsets
    int64_t* off = reinterpret_cast<int64_t*>(lds + (size_t)p.plan.value_chunk * R * PP / 4);
    if (threadIdx.x < 16) p_sum[threadIdx.x] = 0;
    offsets.store(p, b, t0, n, steps * 64, off);
    __syncthreads();
    // A wave takes 32 positions x 32 elements a step: lane l reads the elements 2 (l % 16), + 1 of the positions 8 (l / 16) ..
    // + 8.  Its first step is on its way while the probabilities are computed, and each next one while this one multiplies.
    const uint32_t block = wave % p.plan.blocks, apart = 4 / p.plan.blocks, e = e0 + 32 * block, halves = e < dim ? (n + 31) / 32 : 0;
    const int32_t* v = p.c.d_v + (int64_t)kv * p.c.head_stride;
    auto fetch = [&](v2i_t x[8], uint32_t s) {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const int64_t at = off[s * 32 + kg * 8 + i];
            x[i] = load2<VEC>(v + (at < 0 ? 0 : at), e + 2 * col, dim);
        }
    };
    v2i_t next[8];
    uint32_t s = wave / p.plan.blocks;
    if (s < halves) fetch(next, s);
    const uint32_t quads = steps * 16, parts = (hi - lo - 1) / p.plan.exp_chunk + 1;
    for (uint32_t r = wave; r < R; r += 4) {
        const size_t row = row0 + r;
        unsigned long long sum = 0;
        for (uint32_t i = lane; i < parts; i += 64) sum += p.sums[row * p.plan.exp_chunks + i];
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (sum == 0) {
            bad |= (uint32_t)kWitSum;
            sum = 1;
        }
        if (chunk == 0 && group == 0 && lane == 0 && p.a.d_sum) p.a.d_sum[row] = (int32_t)sum;
        const double inv = 1.0 / (double)sum;
        unsigned long long mine = 0;
        for (uint32_t first = lane; first < quads; first += 64 * kProbAhead) {
            int32_t ex[kProbAhead][4];
#pragma unroll
            for (uint32_t a = 0; a < kProbAhead; a++)
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t i = 4 * (first + 64 * a) + j;
                    ex[a][j] = i < n ? p.a.d_exp[row * p.a.max_len + t0 + i] : 0;
                }
#pragma unroll
            for (uint32_t a = 0; a < kProbAhead; a++) {
                const uint32_t quad = first + 64 * a;
                if (quad >= quads) break;
                uint32_t w[4], pl[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t i = 4 * quad + j;
                    uint32_t pr = 0;
                    if (i < n) {
                        const size_t o = row * p.a.max_len + t0 + i;
                        const uint32_t ev = ex[a][j] < 0 ? 0 : (uint32_t)ex[a][j];
                        pr = probability(ev, (uint64_t)p.a.prob_scale, sum, inv);
                        if (group == 0) {
                            if (p.a.d_prob) p.a.d_prob[o] = (int32_t)pr;
                            if (p.a.d_query) p.a.d_query[o] = (int32_t)((uint64_t)ev * 2 * (uint64_t)p.a.prob_scale - sum * (2 * (uint64_t)pr - 1));
                        }
                        if (off[i] < 0) pr = 0;                     // a page outside the cache
                    }
                    mine += pr;
                    w[j] = digits_of((int32_t)pr);
                }
                transpose4(w[0], w[1], w[2], w[3], pl);
                uint32_t* o = lds + ((((quad >> 3) * PP * 4 + ((quad >> 1) & 3u)) * R + r) << 1) + (quad & 1u);
#pragma unroll
                for (int k = 0; k < PP; k++) o[k * 8 * R] = pl[k];
            }
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) mine += __shfl_xor(mine, o, 64);
        if (lane == 0) p_sum[r] = mine;
    }
    __syncthreads();
    constexpr int G = PP + 3;
    v4i_t acc[2][G];
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int g = 0; g < G; g++) acc[j][g] = v4i_t{0, 0, 0, 0};
    // row m of the product is query head 4 (m % 4) + m / 4, as in the scores
    const uint32_t head = 4 * (col & 3u) + (col >> 2), row = head < R ? head : R - 1;
    for (; s < halves; s += apart) {
        v2i_t x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = next[i];
        if (s + apart < halves) fetch(next, s + apart);
        long pa[PP];
#pragma unroll
        for (int k = 0; k < PP; k++) pa[k] = reinterpret_cast<const long*>(lds)[((s * PP + k) * 4 + kg) * R + row];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            uint32_t p0[4], p1[4];
            transpose4((uint32_t)x[0][j] ^ kByteTops, (uint32_t)x[1][j] ^ kByteTops, (uint32_t)x[2][j] ^ kByteTops, (uint32_t)x[3][j] ^ kByteTops, p0);
            transpose4((uint32_t)x[4][j] ^ kByteTops, (uint32_t)x[5][j] ^ kByteTops, (uint32_t)x[6][j] ^ kByteTops, (uint32_t)x[7][j] ^ kByteTops, p1);
#pragma unroll
            for (int k2 = 0; k2 < 4; k2++) {
                const long vb = (long)(((uint64_t)p1[k2] << 32) | p0[k2]);
#pragma unroll
                for (int k = 0; k < PP; k++) acc[j][k + k2] = __builtin_amdgcn_mfma_i32_16x16x32_i8(pa[k], vb, acc[j][k + k2], 0, 0, 0);
            }
        }
    }
    __syncthreads();
    unsigned long long* total = reinterpret_cast<unsigned long long*>(lds);          // [rows][32 * blocks]
    for (uint32_t i = threadIdx.x; i < R * width; i += 256) total[i] = (unsigned long long)kCacheOffset * p_sum[i / width];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t r = 4 * i + kg;
            if (4 * i < R && r < R) {
                uint64_t y = 0;
#pragma unroll
                for (int g = G - 1; g >= 0; g--) y = (y << 8) + (uint64_t)(int64_t)acc[j][g][i];
                atomicAdd(&total[r * width + 32 * block + 2 * col + j], (unsigned long long)y);
            }
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < R * width; i += 256) {
        const uint32_t r = i / width, el = e0 + i - r * width;
        if (el >= dim) continue;
        if (direct) {
            int32_t q, rem;
            p.out.apply((int64_t)total[i], q, rem, bad);
            p.a.d_out[(row0 + r) * dim + el] = q;
            if (p.a.d_out_rem) p.a.d_out_rem[(row0 + r) * dim + el] = rem;
        } else {
            p.part[((row0 + r) * p.plan.value_chunks + chunk) * dim + el] = (int64_t)total[i];
        }
    }
    if (bad) atomicOr(p.status, bad);
}

// The chunks' partial sums of 64 elements of one row, sixteen threads an element.
constexpr uint32_t kJoinThreads = 1024;
__global__ void __launch_bounds__(kJoinThreads) wit_attend_join_kernel(AttendArgs p) {
    __shared__ int64_t sh[kJoinThreads];
    const uint32_t h = blockIdx.y, b = blockIdx.z, e = blockIdx.x * 64 + (threadIdx.x & 63u), dim = p.c.dim;
    const size_t row = (size_t)b * p.a.heads + h;
    uint32_t lo, hi, bad = 0;
    span_of(p, b, lo, hi);
    if (hi - lo <= p.plan.value_chunk) return;
    const uint32_t parts = (hi - lo - 1) / p.plan.value_chunk + 1;
    int64_t y = 0;
    if (e < dim) {
#pragma unroll 8
        for (uint32_t i = threadIdx.x >> 6; i < parts; i += kJoinThreads / 64) y += p.part[(row * p.plan.value_chunks + i) * dim + e];
    }
    sh[threadIdx.x] = y;
    __syncthreads();
    if (threadIdx.x < 64 && e < dim) {
#pragma unroll
        for (uint32_t i = 1; i < kJoinThreads / 64; i++) y += sh[threadIdx.x + 64 * i];
        int32_t q, r;
        p.out.apply(y, q, r, bad);
        p.a.d_out[row * dim + e] = q;
        if (p.a.d_out_rem) p.a.d_out_rem[row * dim + e] = r;
    }
    if (bad) atomicOr(p.status, bad);
}

// ------------------------------------------------------------------------------------------------
// Products with 4-bit weights.
// ------------------------------------------------------------------------------------------------
struct Q4Args {
    int32_t *q, *r;
    const int32_t* x;
    int64_t x_stride;
    const uint8_t* w;
    int64_t w_stride;
    const int32_t* scales;
    const uint8_t* zeros;
    uint32_t tokens, outputs, inputs, group, groups;
    Scaler scale;
    uint32_t* status;
};

// Any group: a wave a row and up to four tokens, its lanes over the row's bytes.
__global__ void __launch_bounds__(kBlock) wit_q4_any_kernel(Q4Args p) {
    const uint32_t m = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6), n0 = blockIdx.y * 4, lane = threadIdx.x & 63u;
    if (m >= p.outputs) return;
    const uint8_t* w = p.w + m * p.w_stride;
    int64_t y[4] = {0, 0, 0, 0};
    for (uint32_t i = lane; 2 * i < p.inputs; i += 64) {
        const uint32_t byte = w[i];
#pragma unroll
        for (uint32_t half = 0; half < 2; half++) {
            const uint32_t k = 2 * i + half;
            if (k >= p.inputs) break;
            const size_t at = (size_t)m * p.groups + k / p.group;
            const int64_t v = (int64_t)p.scales[at] * ((int32_t)((byte >> (4 * half)) & 15u) - (p.zeros ? (int32_t)p.zeros[at] : 8));
#pragma unroll
            for (uint32_t n = 0; n < 4; n++)
                if (n0 + n < p.tokens) y[n] += (int64_t)((uint64_t)v * (uint64_t)(int64_t)p.x[(n0 + n) * p.x_stride + k]);
        }
    }
    uint32_t bad = 0;
#pragma unroll
    for (uint32_t n = 0; n < 4; n++) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) y[n] += __shfl_xor((long long)y[n], off, 64);
        if (lane == 0 && n0 + n < p.tokens) {
            int32_t q, r;
            p.scale.apply(y[n], q, r, bad);
            const size_t o = (size_t)(n0 + n) * p.outputs + m;
            p.q[o] = q;
            if (p.r) p.r[o] = r;
        }
    }
    if (bad) atomicOr(p.status, bad);
}

// Groups of whole 32s, on the matrix cores.  The input x = sum_p d_p 256^p (balanced digits, four planes) gives four columns a
// token, a tile of 16 columns holds four tokens, and a weight byte is one nibble of the packed byte moved to the upper half
// with its top bit turned over: 16 (w - 8) as a signed byte.  A lane's 16 packed bytes are then 32 of the row's weights, the
// even ones and the odd ones an operand each, with the digits laid out in the same order.  After each step (GS inputs, which
// lie in one group) the 32-bit sums are scaled and added to 64-bit ones: 128 * 128 * 128 * 16 stays far below 2^31.  Zero
// points other than 8 add (8 - z) * sum of digits, which one more product, with ones, gives in the same registers.
// A workgroup takes 16 rows and its eight waves take the row's steps of 128 inputs in turn, so that 4096 rows fill the chip
// and a wave's share is in flight at once; the digits, scales and zero points are staged in LDS meanwhile.
constexpr int kQ4Waves = 8, kQ4Ahead = 4;
constexpr uint32_t kQ4Lds = 60 * 1024;       // of digits, scales and zero points; a longer input goes through in pieces

template <int GS>
__device__ __forceinline__ v4i_t q4_load(const uint8_t* row, uint32_t bytes, uint32_t unit, uint32_t kg) {
    constexpr int CB = GS / 8;               // bytes of a lane's share of GS inputs
    union { v4i_t v; uint8_t b[16]; uint32_t u[4]; uint2 d[2]; } o;
    const uint32_t base = unit * 64;
    if (base + 64 <= bytes) {
#pragma unroll
        for (int c = 0; c < 16 / CB; c++) {
            const uint8_t* s = row + base + c * (GS / 2) + kg * CB;
            if constexpr (CB == 16) __builtin_memcpy(&o.v, s, 16);
            else if constexpr (CB == 8) __builtin_memcpy(&o.d[c], s, 8);
            else __builtin_memcpy(&o.u[c], s, 4);
        }
    } else {
#pragma unroll
        for (int c = 0; c < 16 / CB; c++)
#pragma unroll
            for (int i = 0; i < CB; i++) {
                const uint32_t at = base + c * (GS / 2) + kg * CB + i;
                o.b[c * CB + i] = at < bytes ? row[at] : 0x88;
            }
    }
    return o.v;
}

// Eight inputs' digits, x[0..7] from an even place: the even ones' bytes of plane p in lo[p], the odd ones' in hi[p].
__device__ __forceinline__ bool q4_digits(const int32_t* x, uint32_t lo[4], uint32_t hi[4]) {
    uint32_t d[8];
    bool over = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        d[i] = digits_of(x[i]);
        over |= x[i] > kDigitTop;
    }
    transpose4(d[0], d[2], d[4], d[6], lo);
    transpose4(d[1], d[3], d[5], d[7], hi);
    return over;
}

// Where the word of plane p of token n (of `nt`) and the inputs 8 e .. 8 e + 7 stands, among the operands of the product: units
// of 128 inputs, 2 operands of 16 bytes a lane group (GS = 128, 64) or 4 of 8 (GS = 32).  `odd`: the odd inputs' word.
template <int GS>
__device__ __forceinline__ uint32_t q4_word(uint32_t e, uint32_t n, uint32_t p, uint32_t nt, uint32_t odd) {
    const uint32_t unit = e >> 4, in = e & 15u, cols = 4 * nt;
    if constexpr (GS == 128) {               // lane group in / 4; operand = parity; word in % 4
        return ((((unit * 2 + odd) * 4 + (in >> 2)) * cols + 4 * n + p) << 2) + (in & 3u);
    } else if constexpr (GS == 64) {         // operand in / 8; lane group (in % 8) / 2; words: two even, two odd
        return ((((unit * 2 + (in >> 3)) * 4 + ((in >> 1) & 3u)) * cols + 4 * n + p) << 2) + 2 * odd + (in & 1u);
    } else {                                 // operand in / 4; lane group in % 4; words: even, odd
        return ((((unit * 4 + (in >> 2)) * 4 + (in & 3u)) * cols + 4 * n + p) << 1) + odd;
    }
}

template <int GS, bool ZEROS, int NT>        // NT: tiles of four tokens
__global__ void __launch_bounds__(64 * kQ4Waves) wit_q4_kernel(Q4Args p, uint32_t piece) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ uint32_t over_any;
    constexpr int OPS = GS == 32 ? 4 : 2, STEPS = 128 / GS;      // operands and scalings of a unit
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, col = lane & 15u, kg = lane >> 4;
    const uint32_t m0 = blockIdx.x * 16, n0 = blockIdx.y * 4 * NT, nt = min(4u * NT, p.tokens - n0), cols = 4 * nt;
    const uint32_t row = min(m0 + col, p.outputs - 1), bytes = (p.inputs + 1) / 2, units = (p.inputs + 127) / 128;
    const uint8_t* w = p.w + row * p.w_stride;
    // columns past the tokens read the first ones' digits again; nothing of them is kept
    uint32_t at_col[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) at_col[j] = 16 * j + col < cols ? 16 * j + col : 0;
    int64_t y[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) y[j][i] = 0;
    uint32_t* sc = lds;                                          // [groups of the piece][20]: 16 rows' scales, 4 words of zero points
    const uint32_t piece_groups = (min(piece, units) * 128 - 1) / p.group + 2;
    uint32_t* xd = lds + ((piece_groups * 20 + 3) & ~3u);
    if (threadIdx.x == 0) over_any = 0;
    for (uint32_t u0 = 0; u0 < units; u0 += piece) {
        const uint32_t u1 = min(units, u0 + piece);
        v4i_t a[kQ4Ahead];
#pragma unroll
        for (int s = 0; s < kQ4Ahead; s++)
            if (u0 + wave + s * kQ4Waves < u1) a[s] = q4_load<GS>(w, bytes, u0 + wave + s * kQ4Waves, kg);
        __syncthreads();
        // digits of the piece
        const uint32_t eighths = (u1 - u0) * 16;
        for (uint32_t i = threadIdx.x; i < eighths * nt; i += 64 * kQ4Waves) {
            const uint32_t n = i / eighths, e = i - n * eighths, k = 8 * (u0 * 16 + e);
            const int32_t* x = p.x + (n0 + n) * p.x_stride + k;
            int32_t v[8];
            if (k + 8 <= p.inputs) __builtin_memcpy(v, x, 32);
            else
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = k + j < p.inputs ? x[j] : 0;
            uint32_t lo[4], hi[4];
            if (q4_digits(v, lo, hi)) over_any = 1;
#pragma unroll
            for (int pl = 0; pl < 4; pl++) {
                xd[q4_word<GS>(e, n, pl, nt, 0)] = lo[pl];
                xd[q4_word<GS>(e, n, pl, nt, 1)] = hi[pl];
            }
        }
        const uint32_t g0 = u0 * 128 / p.group, gn = (min(u1 * 128, p.inputs) - 1) / p.group - g0 + 1;
        for (uint32_t i = threadIdx.x; i < gn * 16; i += 64 * kQ4Waves) {
            const uint32_t r = i / gn, g = i - r * gn;
            const size_t at = (size_t)min(m0 + r, p.outputs - 1) * p.groups + g0 + g;
            sc[g * 20 + r] = (uint32_t)p.scales[at];
            if (ZEROS) reinterpret_cast<uint8_t*>(sc + g * 20 + 16)[r] = p.zeros[at];
        }
        __syncthreads();
        for (uint32_t u = u0 + wave; u < u1; u += kQ4Waves * kQ4Ahead) {
#pragma unroll
            for (int s = 0; s < kQ4Ahead; s++) {
                const uint32_t unit = u + s * kQ4Waves;
                if (unit < u1) {
                    const v4i_t wv = a[s];
                    if (unit + kQ4Ahead * kQ4Waves < u1) a[s] = q4_load<GS>(w, bytes, unit + kQ4Ahead * kQ4Waves, kg);
                    v4i_t even, odd;
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const uint32_t x = (uint32_t)wv[c] ^ 0x88888888u;
                        even[c] = (int)((x << 4) & 0xf0f0f0f0u);
                        odd[c] = (int)(x & 0xf0f0f0f0u);
                    }
#pragma unroll
                    for (int st = 0; st < STEPS; st++) {
                        const uint32_t g = (unit * 128 + st * GS) / p.group - g0;
                        if (unit * 128 + st * GS >= p.inputs) break;
                        const v4i_t scale = *reinterpret_cast<const v4i_t*>(sc + g * 20 + 4 * kg);
                        const uint32_t zero = ZEROS ? sc[g * 20 + 16 + kg] : 0;
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            v4i_t acc = {0, 0, 0, 0}, ones = {0, 0, 0, 0};
                            if constexpr (GS == 32) {
                                const uint32_t o = (((unit - u0) * OPS + st) * 4 + kg) * cols + at_col[j];
                                const long b = *reinterpret_cast<const long*>(xd + (o << 1));
                                union { uint32_t u[2]; long l; } f = {{(uint32_t)even[st], (uint32_t)odd[st]}};
                                acc = __builtin_amdgcn_mfma_i32_16x16x32_i8(f.l, b, acc, 0, 0, 0);
                                if (ZEROS) ones = __builtin_amdgcn_mfma_i32_16x16x32_i8(0x0101010101010101L, b, ones, 0, 0, 0);
                            } else {
#pragma unroll
                                for (int op = 0; op < OPS / STEPS; op++) {
                                    const uint32_t o = (((unit - u0) * OPS + st + op) * 4 + kg) * cols + at_col[j];
                                    const v4i_t b = *reinterpret_cast<const v4i_t*>(xd + (o << 2));
                                    v4i_t f;
                                    if constexpr (GS == 128) f = op ? odd : even;
                                    else f = v4i_t{even[2 * st], even[2 * st + 1], odd[2 * st], odd[2 * st + 1]};
                                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, b, acc, 0, 0, 0);
                                    if (ZEROS) {
                                        const v4i_t o1 = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
                                        ones = __builtin_amdgcn_mfma_i32_16x16x64_i8(o1, b, ones, 0, 0, 0);
                                    }
                                }
                            }
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                int32_t v = acc[i] >> 4;
                                if (ZEROS) v += (8 - (int32_t)((zero >> (8 * i)) & 255u)) * ones[i];
                                y[j][i] += (int64_t)v * scale[i];
                            }
                        }
                    }
                }
            }
        }
    }
    // planes of a token stand in four neighbouring columns; then the waves' sums
    __syncthreads();
    int64_t* sum = reinterpret_cast<int64_t*>(lds);              // [wave][16 rows][4 NT tokens]
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            int64_t v = (int64_t)((uint64_t)y[j][i] << (8 * (col & 3u)));
            v += __shfl_xor((long long)v, 1, 64);
            v += __shfl_xor((long long)v, 2, 64);
            if ((col & 3u) == 0) sum[(wave * 16 + 4 * kg + i) * 4 * NT + 4 * j + (col >> 2)] = v;
        }
    __syncthreads();
    uint32_t bad = 0;
    for (uint32_t i = threadIdx.x; i < 16 * 4 * NT; i += 64 * kQ4Waves) {
        const uint32_t r = i & 15u, n = i >> 4, m = m0 + r;
        if (n >= nt || m >= p.outputs) continue;
        int64_t v = 0;
#pragma unroll
        for (int wv = 0; wv < kQ4Waves; wv++) v += sum[(wv * 16 + r) * 4 * NT + n];
        if (over_any) {
            // inputs above kDigitTop: their top digit is 128, which the byte held as -128; 2^32 of each is missing
            const int32_t* x = p.x + (n0 + n) * p.x_stride;
            const uint8_t* wr = p.w + m * p.w_stride;
            uint64_t more = 0;
            for (uint32_t k = 0; k < p.inputs; k++)
                if (x[k] > kDigitTop) {
                    const size_t at = (size_t)m * p.groups + k / p.group;
                    more += (uint64_t)((int64_t)p.scales[at] * ((int32_t)((wr[k >> 1] >> (4 * (k & 1u))) & 15u) - (p.zeros ? (int32_t)p.zeros[at] : 8)));
                }
            v += (int64_t)(more << 32);
        }
        int32_t q, rr;
        p.scale.apply(v, q, rr, bad);
        const size_t o = (size_t)(n0 + n) * p.outputs + m;
        p.q[o] = q;
        if (p.r) p.r[o] = rr;
    }
    if (bad) atomicOr(p.status, bad);
}

template <int GS, bool ZEROS>
static void q4_launch(const Q4Args& p, hipStream_t s) {
    const uint32_t nt = std::min(p.tokens, 4u), units = (p.inputs + 127) / 128;
    const uint32_t piece = std::min(units, kQ4Lds / (512 * nt + 80 * std::max(1u, 128 / p.group)));
    const uint32_t piece_groups = (uint32_t)(((uint64_t)piece * 128 - 1) / p.group) + 2;
    const size_t bytes = std::max<size_t>(((piece_groups * 20 + 3) & ~3u) * 4 + (size_t)piece * 512 * nt, kQ4Waves * 16 * 4 * 8);
    wit_q4_kernel<GS, ZEROS, 1><<<dim3((p.outputs + 15) / 16, (p.tokens + 3) / 4), 64 * kQ4Waves, bytes, s>>>(p, piece);
}

}  // namespace grape

using namespace grape;

#define GRAPE_REFUSED_IF(expr)           \
    if (const char* why = (expr)) {      \
        set_error("%s: %s", __func__, why); \
        return GRAPE_EINVAL;             \
    }

extern "C" {

int grape_wit_rope_append(const grape_wit_rope_append_args* args, const grape_wit_cache* cache, grape_stream_t st) {
    GRAPE_REQUIRE(initialised(), "grape_init has not been called");
    GRAPE_REFUSED_IF(token::refuse_append(args, cache));
    if (args->tokens == 0) return GRAPE_OK;
    AppendArgs p;
    p.a = *args;
    p.c = *cache;
    const grape_wit_rope_append_args& a = p.a;
    p.head_units = token::append_head_units(p.c.dim, a.rot, 1);
    p.units = (a.heads + 2 * p.c.heads) * p.head_units;
    p.total = (uint64_t)a.tokens * p.units;
    p.shift = log2_exact(a.scale);
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status, s);
    if (rc) return rc;
    wit_append_kernel<<<blocks_for(p.total), kBlock, 0, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    return GRAPE_OK;
}

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
    if (!a.d_scores) a.d_scores = (int32_t*)(ws + pl.at_scores);
    if (!a.d_exp) a.d_exp = (int32_t*)(ws + pl.at_exp);
    p.chunk_max = (int32_t*)(ws + pl.at_max);
    p.sums = (unsigned long long*)(ws + pl.at_sum);
    p.part = (int64_t*)(ws + pl.at_part);
    p.page = token::fast_div(p.c.page_size);
    p.qk = scaler(a.qk_scale);
    p.out = scaler(a.out_scale);
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status, s);
    if (rc) return rc;
    auto aligned = [&](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    const bool vec = p.c.dim % 4 == 0 && ((p.c.page_stride | p.c.token_stride | p.c.head_stride) & 3) == 0 && aligned(p.c.d_k) && aligned(p.c.d_v);
    const int planes = a.prob_scale <= ((int64_t)1 << 22) ? 3 : 4;
    const size_t score_lds = (size_t)pl.dim64 * 5 * 64 * pl.rows + (size_t)pl.score_chunk * 8 * (pl.rows + 1);
    const size_t value_lds = std::max<size_t>((size_t)pl.value_chunk * (pl.rows * planes + 8), (size_t)pl.rows * pl.blocks * 32 * 8);
    // the heads of one chunk are neighbours: they read the same tokens' lines of memory at the same time
    const uint32_t head_tiles = p.c.heads * pl.tiles;
    const dim3 score_grid(std::max(1u, pl.score_chunks) * head_tiles, a.seqs), value_grid(std::max(1u, pl.value_chunks) * head_tiles * pl.groups, a.seqs);
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
        wit_attend_join_kernel<<<dim3(pl.dim64, a.heads, a.seqs), kJoinThreads, 0, s>>>(p);
        GRAPE_LAUNCH_CHECK();
    }
    return GRAPE_OK;
}

int grape_wit_matvec_q4(int32_t* d_q, int32_t* d_r, const int32_t* d_x, int64_t x_stride, const uint8_t* d_w, int64_t w_stride,
                        const int32_t* d_scales, const uint8_t* d_zeros, uint32_t tokens, uint32_t outputs, uint32_t inputs,
                        uint32_t group, int64_t scale, grape_stream_t st) {
    GRAPE_REQUIRE(initialised(), "grape_init has not been called");
    GRAPE_REFUSED_IF(token::refuse_q4(d_q, d_x, x_stride, d_w, w_stride, d_scales, tokens, outputs, inputs, group, scale));
    if (tokens == 0 || outputs == 0) return GRAPE_OK;
    Q4Args p;
    p.q = d_q; p.r = d_r; p.x = d_x; p.x_stride = x_stride; p.w = d_w; p.w_stride = w_stride; p.scales = d_scales; p.zeros = d_zeros;
    p.tokens = tokens; p.outputs = outputs; p.inputs = inputs; p.group = group;
    p.groups = (inputs - 1) / group + 1;
    p.scale = scaler(scale);
    hipStream_t s = as_stream(st);
    int rc = wit_status_word(&p.status, s);
    if (rc) return rc;
    if (group % 32) wit_q4_any_kernel<<<dim3((outputs + 3) / 4, (tokens + 3) / 4), kBlock, 0, s>>>(p);
    else if (group % 64) d_zeros ? q4_launch<32, true>(p, s) : q4_launch<32, false>(p, s);
    else if (group % 128) d_zeros ? q4_launch<64, true>(p, s) : q4_launch<64, false>(p, s);
    else d_zeros ? q4_launch<128, true>(p, s) : q4_launch<128, false>(p, s);
    GRAPE_LAUNCH_CHECK();
    return GRAPE_OK;
}

}  // extern "C"

// The step around new tokens: their pages, positions and slots from the requests' lengths, and the choice of the next token.
#include <algorithm>
#include "token_device.hpp"
#include "step_geometry.hpp"

namespace grape {

// ------------------------------------------------------------------------------------------------
// Pages and slots.  One launch: every workgroup makes the prefix sums of all sequences' tokens, pages and pages given back for
// itself, in LDS, and then takes its share of the rows, the new pages and the ones given back, each of which finds its sequence by
// halving.  Nothing that a workgroup reads is written by another one: the lengths and the ring's span go to places of their own,
// entries of the table are read below the pages held and written above, and the ring is written behind its last entry alone.
// Bound by latency: 7.5 us for one more token of 64 sequences, 10 for a few prompts among running answers, 12.6 for 1023 sequences behind a window: two
// rounds of loads with the scans between them.
// ------------------------------------------------------------------------------------------------
struct PageArgs {
    grape_wit_page_step_args a;
    token::FastDiv by_page;
    uint32_t sink_pages;
    uint32_t* status;
};
struct Two {
    uint64_t a, b;
};
// The sums of v over the threads before this one, and of all of them.
template <uint32_t THREADS>
__device__ __forceinline__ Two before_me(Two v, Two& all, Two* waves) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    Two sum = v;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t x = __shfl_up(sum.a, d, 64), y = __shfl_up(sum.b, d, 64);
        if (lane >= d) sum.a += x, sum.b += y;
    }
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    Two base{sum.a - v.a, sum.b - v.b};
    all = Two{0, 0};
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 64; w++) {
        if (w < wave) base.a += waves[w].a, base.b += waves[w].b;
        all.a += waves[w].a;
        all.b += waves[w].b;
    }
    return base;
}

// The number of the n ascending sums that are at most `x`: the sequence that x belongs to.
__device__ __forceinline__ uint32_t find_sequence(const uint32_t* sums, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (sums[mid] <= x) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) wit_page_step_kernel(PageArgs p) {
    extern __shared__ uint32_t lds[];
    __shared__ Two waves[2][THREADS / 64];
    __shared__ uint32_t top[2];
    const grape_wit_page_step_args& a = p.a;
    uint32_t *to_token = lds, *to_page = lds + a.seqs, *to_back = lds + 2 * a.seqs;          // sums up to and with each sequence
    int32_t *lens = reinterpret_cast<int32_t*>(lds + 3 * a.seqs), *news = lens + a.seqs;
    const uint64_t most = (uint64_t)a.page_size * a.table_stride;
    uint32_t bad = 0;
    for (uint32_t b = threadIdx.x; b < a.seqs; b += THREADS) {
        lens[b] = a.d_lens[b];
        news[b] = a.d_new[b];
    }
    const uint32_t head_in = (uint32_t)a.d_span[0], count_in = (uint32_t)a.d_span[1];
    const bool ring_ok = count_in <= a.ring && (head_in < a.ring || (head_in == 0 && a.ring == 0));
    const uint32_t head = ring_ok ? head_in : 0, count = ring_ok ? count_in : 0, room = ring_ok ? a.ring - count : 0;
    if (!ring_ok) bad |= (uint32_t)kWitIndex;
    if (threadIdx.x < 2) top[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t each = (a.seqs + THREADS - 1) / THREADS, b0 = min(threadIdx.x * each, a.seqs), b1 = min(b0 + each, a.seqs);
    step::Sequence s;
    auto ask = [&](uint32_t b) { return s.ask(lens[b], news[b], most, p.by_page); };
    Two wanted{0, 0}, all, back{0, 0}, all_back;          // tokens and pages; pages given back
    for (uint32_t b = b0; b < b1; b++) {
        if (!ask(b)) bad |= (uint32_t)kWitIndex;
        wanted.a += s.tokens;
        wanted.b += s.taken;
    }
    wanted = before_me<THREADS>(wanted, all, waves[0]);
    // sequences are served in their order until the rows or the free pages run out; from there on none is
    uint32_t served_tokens = 0, served_pages = 0;
    for (uint32_t b = b0; b < b1; b++) {
        ask(b);
        wanted.a += s.tokens;
        wanted.b += s.taken;
        const bool served = wanted.a <= a.rows && wanted.b <= count;
        if (served) served_tokens = (uint32_t)wanted.a, served_pages = (uint32_t)wanted.b;
        else s.refuse();
        s.give_back(a.window, p.sink_pages, p.by_page);
        back.a += s.back;
        to_token[b] = served ? (uint32_t)wanted.a : UINT32_MAX;
        to_page[b] = (uint32_t)wanted.b;
        to_back[b] = s.back;
    }
    // the largest sums that were served
    if (served_tokens) atomicMax(&top[0], served_tokens);
    if (served_pages) atomicMax(&top[1], served_pages);
    back = before_me<THREADS>(back, all_back, waves[1]);
    const uint32_t rows = top[0], taken = top[1], kept = (uint32_t)min(all_back.a, (uint64_t)room);
    const bool mine = blockIdx.x == 0;          // of what is written once
    for (uint32_t b = b0; b < b1; b++) {
        const bool served = to_token[b] != UINT32_MAX;
        if (!served) {
            to_token[b] = rows;
            to_page[b] = taken;
        }
        back.a += to_back[b];
        to_back[b] = (uint32_t)back.a;
        if (mine) {
            const bool ok = ask(b);
            a.d_starts[b + 1] = (int32_t)to_token[b];
            a.d_lens_out[b] = !ok ? lens[b] : s.ended ? 0 : (int32_t)(s.len + (served ? s.tokens : 0));
        }
    }
    if (mine && threadIdx.x == 0) {
        a.d_starts[0] = 0;
        const uint32_t at = head + taken;
        a.d_span_out[0] = (int32_t)(ring_ok ? (at >= a.ring && a.ring ? at - a.ring : at) : head_in);
        a.d_span_out[1] = (int32_t)(ring_ok ? count - taken + kept : count_in);
        if (all.a > a.rows || all.b > count || all_back.a > kept) bad |= (uint32_t)kWitPages;
    }
    __syncthreads();
    auto ring_at = [&](uint32_t k) {
        const uint32_t at = head + k;
        return at >= a.ring ? at - a.ring : at;
    };
    // page number i of sequence b, which held `held` and whose first new one is number `first` of those taken
    auto page_at = [&](uint32_t b, uint32_t i, uint32_t held, uint32_t first) {
        return i < held ? a.d_block_table[(size_t)b * a.table_stride + i] : a.d_free[ring_at(first + i - held)];
    };
    // rows, new pages and pages given back, each from a wave of its own on, so that none waits for the loads of another kind
    auto up = [](uint64_t x) { return (x + 63) / 64 * 64; };
    const uint64_t page0 = up(a.rows), back0 = page0 + up(taken), end = back0 + kept;
    for (uint64_t at = (uint64_t)blockIdx.x * THREADS + threadIdx.x; at < end; at += (uint64_t)gridDim.x * THREADS) {
        if (at < page0) {
            const uint32_t r = (uint32_t)at;
            if (r >= a.rows) continue;
            int32_t pos = 0;
            int64_t slot = -1;
            if (r < rows) {
                const uint32_t b = find_sequence(to_token, a.seqs, r), had = (uint32_t)lens[b], t = had + (r - (b ? to_token[b - 1] : 0)), i = p.by_page(t);
                const int32_t page = page_at(b, i, step::pages_of(had, p.by_page), b ? to_page[b - 1] : 0);
                pos = (int32_t)t;
                if (page >= 0) slot = (int64_t)page * a.page_size + (t - i * a.page_size);
                else bad |= (uint32_t)kWitIndex;
            }
            a.d_positions[r] = pos;
            a.d_slots[r] = slot;
        } else if (at < back0) {
            const uint32_t k = (uint32_t)(at - page0);
            if (k >= taken) continue;
            const uint32_t b = find_sequence(to_page, a.seqs, k);
            a.d_block_table[(size_t)b * a.table_stride + step::pages_of((uint32_t)lens[b], p.by_page) + (k - (b ? to_page[b - 1] : 0))] = a.d_free[ring_at(k)];
        } else {
            const uint32_t k = (uint32_t)(at - back0), b = find_sequence(to_back, a.seqs, k);
            ask(b);
            if (b ? to_token[b] == to_token[b - 1] : to_token[b] == 0) s.refuse();
            s.give_back(a.window, p.sink_pages, p.by_page);
            const int32_t page = page_at(b, s.back_page(k - (b ? to_back[b - 1] : 0)), s.held, b ? to_page[b - 1] : 0);
            if (page < 0) bad |= (uint32_t)kWitIndex;
            a.d_free[ring_at(count + k)] = page;
        }
    }
    if (bad) atomicOr(p.status, bad);
}

// ------------------------------------------------------------------------------------------------
// The next token.  A workgroup counts a row's history for its chunk of the vocabulary in LDS, applies what the counts, biases and
// mask ask for and keeps its largest logit; a second launch joins the chunks and writes how far each logit is below the row's largest.
// Bound by memory: 4 bytes read a logit, up to 16 written, and 4 read again for the distances.  256 rows of 131072: 67 + 5 us, 2 TB/s, held up by
// the vector instructions of the counting and the adjusting (half of the time); one row of 32000: 5.5 + 3 us, two chains of loads.  Lists of the tokens
// that occur, so that only these are divided, were slower than dividing where a count is not zero.
// ------------------------------------------------------------------------------------------------
constexpr int32_t kLowest = INT32_MIN;          // of a token that must not be chosen
struct NextArgs {
    grape_wit_next_token_args a;
    step::NextPlan plan;
    Scaler scale;
    unsigned long long* part;          // [seqs][chunks]: the larger the logit, then the smaller the token, the larger the number
    uint32_t* status;
};

__device__ __forceinline__ unsigned long long rank_of(int32_t z, uint32_t token) {
    return ((unsigned long long)((uint32_t)z ^ 0x80000000u) << 32) | (uint32_t)~token;
}
__device__ __forceinline__ int32_t value_of(unsigned long long rank) { return (int32_t)((uint32_t)(rank >> 32) ^ 0x80000000u); }

constexpr uint32_t kNextThreads = 512, kNextAhead = 4;          // of a workgroup; tokens of the history asked for at once by a thread
__device__ __forceinline__ unsigned long long block_largest(unsigned long long v) {
    __shared__ unsigned long long sh[kNextThreads / 64];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = max(v, __shfl_xor(v, off, 64));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (uint32_t w = 1; w < kNextThreads / 64; w++) v = max(v, sh[w]);
    return v;
}

// four entries of a row, wherever it starts; those from n on are 0 and left as they were
typedef int v4u_t __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ v4i_t row4(const int32_t* x, uint32_t at, uint32_t n) {
    if (at + 4 <= n) return *reinterpret_cast<const v4u_t*>(x + at);
    v4i_t v = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t j = 0; j < 3; j++)
        if (at + j < n) v[j] = x[at + j];
    return v;
}
__device__ __forceinline__ void put4(int32_t* x, uint32_t at, uint32_t n, v4i_t v) {
    if (at + 4 <= n) {
        *reinterpret_cast<v4u_t*>(x + at) = v;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 3; j++)
            if (at + j < n) x[at + j] = v[j];
    }
}

// One way of the repetition's division, x * mul / by: in double precision where every product stays below 2^50 (see Penalty).
struct Division {
    double mul, by, inv, half;
    Division() = default;
    __device__ __forceinline__ Division(int64_t mul_, int64_t by_) : mul((double)mul_), by((double)by_), inv(1.0 / (double)by_), half((double)(by_ >> 1) + 0.5) {}
};

// What a token that occurs in the history loses.  With `scale` and the repetition's factor up to 2^18 a product of int32 stays below 2^50, and
// the quotient of (y + by/2 + 1/2) / by is no nearer than 1 / (2 by) to a whole number while its product with 1 / by is off by at most 2^-52 of
// itself: one product gives it.  Sums that leave 2^53 are no longer exact, and far outside int32.
struct Penalty {
    Division up, down;                         // of logits above zero, and of the others
    Scaler wide_up, wide_down;
    int64_t scale, repetition, whole_presence, whole_frequency;
    double presence, frequency;
    bool divides, plain;
    __device__ __forceinline__ void apply(int32_t x, uint32_t count, double& y, int32_t& rem) const {
        y = (double)x;
        rem = 0;
        if (divides) {
            if (plain) {
                const double t = __builtin_fma(y, x > 0 ? up.mul : down.mul, x > 0 ? up.half : down.half), q = __builtin_floor(t * (x > 0 ? up.inv : down.inv));
                rem = (int32_t)(__builtin_fma(-q, x > 0 ? up.by : down.by, t) - (x > 0 ? up.half : down.half));
                y = q;
            } else {
                const int64_t product = (int64_t)x * (x > 0 ? scale : repetition), by = x > 0 ? repetition : scale;
                int32_t q;
                uint32_t beyond = 0;          // a quotient beyond int32 is still one of 64 bits
                if (x > 0) wide_up.apply(product, q, rem, beyond);
                else wide_down.apply(product, q, rem, beyond);
                // up to 2^62, which a penalty of up to 2^55 may bring back to where every bit counts
                y = (double)((beyond ? (product - rem) / by : (int64_t)q) - (whole_frequency * (int64_t)count + whole_presence));
                return;
            }
        }
        y -= __builtin_fma(frequency, (double)count, presence);
    }
};

__global__ void __launch_bounds__(kNextThreads, 6) wit_next_adjust_kernel(NextArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t counts[];
    const grape_wit_next_token_args& a = p.a;
    const uint32_t b = blockIdx.y, v0 = blockIdx.x * p.plan.chunk, n = min(a.vocab - v0, p.plan.chunk);
    const int32_t *logits = a.d_logits + b * a.logits_stride + v0, *bias = a.d_bias ? a.d_bias + b * a.bias_stride + v0 : nullptr;
    const uint32_t* mask = a.d_mask ? reinterpret_cast<const uint32_t*>(a.d_mask) + b * a.mask_stride + v0 / 32 : nullptr;
    uint32_t bad = 0;
    // a thread's logits are all under way while the history is counted
    constexpr uint32_t kFours = step::kNextMost / (4 * kNextThreads);
    v4i_t x[kFours];
#pragma unroll
    for (uint32_t k = 0; k < kFours; k++) {
        const uint32_t i = 4 * (threadIdx.x + k * kNextThreads);
        x[k] = i < n ? row4(logits, i, n) : v4i_t{0, 0, 0, 0};
    }
    int32_t len = a.history ? a.d_history_lens[b] : 0;
    const int32_t* history = a.history ? a.d_history + b * a.history_stride : nullptr;
    int32_t seen[kNextAhead];
    auto fetch = [&](uint32_t from) {
#pragma unroll
        for (uint32_t k = 0; k < kNextAhead; k++) {
            const uint32_t at = from + threadIdx.x + k * kNextThreads;
            seen[k] = at < a.history ? history[at] : -1;
        }
    };
    fetch(0);
    for (uint32_t k = threadIdx.x; k < p.plan.chunk / 4; k += kNextThreads) reinterpret_cast<v4i_t*>(counts)[k] = v4i_t{0, 0, 0, 0};
    if (len < 0 || (uint32_t)len > a.history) {
        bad |= (uint32_t)kWitIndex;
        len = len < 0 ? 0 : (int32_t)a.history;
    }
    Penalty penalty;
    penalty.scale = a.scale;
    penalty.repetition = a.d_repetition ? a.d_repetition[b] : a.scale;
    if (penalty.repetition < 1) bad |= (uint32_t)kWitIndex;
    penalty.divides = a.d_repetition && penalty.repetition >= 1;
    penalty.plain = a.scale <= (1 << 18) && penalty.repetition <= (1 << 18);
    if (penalty.divides) {
        penalty.up = Division(a.scale, penalty.repetition);
        penalty.down = Division(penalty.repetition, a.scale);
        penalty.wide_up = Scaler{penalty.repetition, penalty.up.inv, -1};
        penalty.wide_down = p.scale;
    }
    penalty.whole_presence = a.d_presence ? a.d_presence[b] : 0;
    penalty.whole_frequency = a.d_frequency ? a.d_frequency[b] : 0;
    penalty.presence = (double)penalty.whole_presence;
    penalty.frequency = (double)penalty.whole_frequency;
    __syncthreads();
    for (uint32_t from = 0; from < (uint32_t)len; from += kNextAhead * kNextThreads) {
        if (from) fetch(from);
#pragma unroll
        for (uint32_t k = 0; k < kNextAhead; k++) {
            const int32_t t = seen[k];
            if (from + threadIdx.x + k * kNextThreads >= (uint32_t)len) break;
            if (t >= (int32_t)a.vocab) bad |= (uint32_t)kWitIndex;
            const uint32_t at = (uint32_t)t - v0;
            if (t >= 0 && at < n) atomicAdd(&counts[at], 1u);
        }
    }
    const size_t o = (size_t)b * a.vocab + v0;
    __syncthreads();
    int32_t best = kLowest;
    uint32_t best_at = 0;
#pragma unroll
    for (uint32_t k = 0; k < kFours; k++) {
        const uint32_t i = 4 * (threadIdx.x + k * kNextThreads);
        if (i >= n) break;
        const v4i_t more = bias ? row4(bias, i, n) : v4i_t{0, 0, 0, 0};
        const uint32_t allowed = mask ? mask[i / 32] >> (i & 31u) : ~0u;
        const v4i_t c = *reinterpret_cast<const v4i_t*>(counts + i);
        v4i_t z, rem = {0, 0, 0, 0};
        // a sum at either end of int32 may have left it, or stand where excluded tokens do
        uint32_t edge = ~0u;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const bool chosen = ((allowed >> j) & 1u) && min(x[k][j], more[j]) != kLowest;
            const int32_t sum = __builtin_elementwise_add_sat((int)x[k][j], (int)more[j]);
            edge = min(edge, ((uint32_t)sum ^ 0x80000000u) + 1u);
            z[j] = chosen ? sum : kLowest;
        }
        if ((c[0] | c[1] | c[2] | c[3]) || edge < 2) {
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                if (!(c[j] || edge < 2) || !((allowed >> j) & 1u) || min(x[k][j], more[j]) == kLowest || i + j >= n) continue;
                double y = (double)x[k][j];
                int32_t r = 0;
                if (c[j]) penalty.apply(x[k][j], (uint32_t)c[j], y, r);
                rem[j] = r;
                y += (double)more[j];
                const bool beyond = y <= (double)kLowest || y > (double)INT32_MAX;
                if (beyond) bad |= (uint32_t)kWitQuotient;
                z[j] = beyond ? (y < 0.0 ? kLowest + 1 : INT32_MAX) : (int32_t)y;
            }
        }
        if (i + 4 > n) {
#pragma unroll
            for (uint32_t j = 1; j < 4; j++) z[j] = i + j < n ? z[j] : kLowest;
        }
        const int32_t most = max(max(z[0], z[1]), max(z[2], z[3]));
        if (most > best) {
            best = most;
            best_at = v0 + i + (z[0] == most ? 0 : z[1] == most ? 1 : z[2] == most ? 2 : 3);
        }
        if (a.d_out) put4(a.d_out + o, i, n, z);
        if (a.d_rem) put4(a.d_rem + o, i, n, rem);
        if (a.d_count) put4(a.d_count + o, i, n, c);
        if (a.d_gap) put4(a.d_gap + o, i, n, z);          // the second launch takes it from the largest
    }
    const unsigned long long largest = block_largest(rank_of(best, best_at));
    if (threadIdx.x == 0) p.part[(size_t)b * p.plan.chunks + blockIdx.x] = largest;
    if (bad) atomicOr(p.status, bad);
}

__global__ void __launch_bounds__(kNextThreads) wit_next_choose_kernel(NextArgs p) {
    const grape_wit_next_token_args& a = p.a;
    const uint32_t b = blockIdx.y;
    unsigned long long best = 0;
    for (uint32_t i = threadIdx.x; i < p.plan.chunks; i += kNextThreads) best = max(best, p.part[(size_t)b * p.plan.chunks + i]);
    best = block_largest(best);
    const int32_t top = value_of(best);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.d_token[b] = top == kLowest ? -1 : (int32_t)~(uint32_t)best;
        if (a.d_max) a.d_max[b] = top;
    }
    if (!a.d_gap) return;
    const uint32_t v0 = blockIdx.x * p.plan.chunk, n = min(a.vocab - v0, p.plan.chunk);
    int32_t* gap = a.d_gap + (size_t)b * a.vocab + v0;
    uint32_t bad = 0;
    for (uint32_t i = 4 * threadIdx.x; i < n; i += 4 * kNextThreads) {
        v4i_t z = row4(gap, i, n);
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t below = z[j] == kLowest ? 0u : (uint32_t)top - (uint32_t)z[j];
            if (below > (uint32_t)INT32_MAX && i + j < n) bad |= (uint32_t)kWitSumWide;
            z[j] = (int32_t)below;
        }
        put4(gap, i, n, z);
    }
    if (bad) atomicOr(p.status, bad);
}

}  // namespace grape

using namespace grape;

extern "C" {

int grape_wit_page_step(const grape_wit_page_step_args* args, grape_stream_t st) {
    GRAPE_REQUIRE(initialised(), "grape_init has not been called");
    GRAPE_REFUSED_IF(step::refuse_pages(args));
    PageArgs p;
    p.a = *args;
    p.by_page = token::fast_div(p.a.page_size);
    p.sink_pages = p.a.window ? (uint32_t)(((uint64_t)p.a.sinks + p.a.page_size - 1) / p.a.page_size) : 0;
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status);
    if (rc) return rc;
    // every workgroup makes the sums, of up to four sequences a thread; waves fewer meet sooner (64 sequences 7.5 us, and 8.8 by 1024 threads, 600 10.4 and 11.3,
    // 1023 12.5 and 14.4, but 2048 16.4 and 15.3, 4096 25 and 17)
    const uint32_t threads = p.a.seqs <= 1024 ? 256 : 1024, workgroups = std::min(256u, token::ceil_div(p.a.rows, threads) + token::ceil_div(p.a.seqs, 128));
    const size_t lds = (size_t)20 * p.a.seqs;
    if (threads == 256) wit_page_step_kernel<256><<<std::max(1u, workgroups), 256, lds, s>>>(p);
    else wit_page_step_kernel<1024><<<std::max(1u, workgroups), 1024, lds, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    return GRAPE_OK;
}

size_t grape_wit_next_token_workspace(uint32_t seqs, uint32_t vocab) { return step::next_workspace(seqs, vocab); }

int grape_wit_next_token(const grape_wit_next_token_args* args, grape_stream_t st) {
    GRAPE_REQUIRE(initialised(), "grape_init has not been called");
    GRAPE_REFUSED_IF(step::refuse_next(args));
    if (args->seqs == 0) return GRAPE_OK;
    NextArgs p;
    p.a = *args;
    const grape_wit_next_token_args& a = p.a;
    p.plan = step::next_plan(a.seqs, a.vocab);
    p.scale = scaler(a.scale);
    p.part = (unsigned long long*)a.d_workspace;
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status);
    if (rc) return rc;
    const dim3 grid(p.plan.chunks, a.seqs);
    const size_t lds = (size_t)4 * p.plan.chunk;
    wit_next_adjust_kernel<<<grid, kNextThreads, lds, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    const dim3 join(a.d_gap ? p.plan.chunks : 1, a.seqs);
    wit_next_choose_kernel<<<join, kNextThreads, 0, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    return GRAPE_OK;
}

}  // extern "C"

// The witness of new tokens: rotation and append to a paged cache, and products with 4-bit weights (their attention is in
// token_attention.hip).  The arithmetic is that of witness_kernels.hip: exact 64-bit products, rescaled.
#include <algorithm>
#include <type_traits>
#include "token_device.hpp"

namespace grape {

// ------------------------------------------------------------------------------------------------
// Rotation and append.  A unit is W pairs of a rotated head or 2 W elements that only move; a token's units are those of its
// query heads, its key heads and its value heads.  W = 4: a unit is two 16-byte loads and two to four 16-byte stores.  Bound by
// memory (2048 tokens of one head of 4096 elements, 302 MB: 79 us, 3.8 TB/s; units of 16 bytes took 94); with few tokens by two
// loads that depend on each other, the position and its row of the tables (one token: 3.4 us).
//
// Of several tokens with one slot the last one has to stay, whatever the order in which they are written: a workgroup looks for
// its tokens' slots among those of the later tokens first.  It reads 8 bytes a later token for that, beside some hundred units of
// 32 bytes and more each; with many tokens it asks a table of one bit a hash value before it compares.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kAppendTokens = 1024;     // tokens of a workgroup at most
constexpr uint32_t kAppendFilter = 8;        // tokens from which the table of bits is used
struct AppendArgs {
    grape_wit_rope_append_args a;
    grape_wit_cache c;
    uint32_t units, head_units, per;         // of a token, of a head, of a workgroup
    uint64_t total;
    token::FastDiv by_units, by_head, by_page;
    Scaler scale;
    uint32_t* status;
};

template <int W>
struct Elements {
    int32_t v[W];
    __device__ __forceinline__ void load(const int32_t* x) {
        if constexpr (W == 4) *reinterpret_cast<v4i_t*>(v) = *reinterpret_cast<const v4i_t*>(x);
        else v[0] = *x;
    }
    __device__ __forceinline__ void store(int32_t* x) const {
        if constexpr (W == 4) *reinterpret_cast<v4i_t*>(x) = *reinterpret_cast<const v4i_t*>(v);
        else *x = v[0];
    }
};

template <int W>
__global__ void __launch_bounds__(kBlock) wit_append_kernel(AppendArgs p) {
    __shared__ uint32_t shadowed[kAppendTokens / 32], bits[2048];
    const grape_wit_rope_append_args& a = p.a;
    const grape_wit_cache& c = p.c;
    const uint64_t u0 = (uint64_t)blockIdx.x * p.per;
    const uint32_t t0 = (uint32_t)(u0 / p.units), skip = (uint32_t)(u0 - (uint64_t)t0 * p.units), n = (uint32_t)min((uint64_t)p.per, p.total - u0);
    const uint32_t tokens = (skip + n - 1) / p.units + 1;          // of this workgroup
    auto kind = [&](int64_t slot, uint32_t tok) { return token::append_kind(c, slot, a.rot ? a.d_positions[tok] : 0, a.rot, a.table_rows); };
    if (t0 + 1 < a.tokens) {
        const bool filter = tokens > kAppendFilter;
        for (uint32_t i = threadIdx.x; i < (tokens + 31) / 32; i += kBlock) shadowed[i] = 0;
        auto hash = [](int64_t slot) { return ((uint32_t)slot * 2654435761u) >> 16; };
        if (filter) {
            for (uint32_t i = threadIdx.x; i < 2048; i += kBlock) bits[i] = 0;
            __syncthreads();
            for (uint32_t j = threadIdx.x; j < tokens; j += kBlock) {
                const uint32_t h = hash(a.d_slots[t0 + j]);
                atomicOr(&bits[h >> 5], 1u << (h & 31u));
            }
        }
        __syncthreads();
        for (uint32_t o = t0 + 1 + threadIdx.x; o < a.tokens; o += kBlock) {
            const int64_t slot = a.d_slots[o];
            if (slot < 0) continue;
            if (filter) {
                const uint32_t h = hash(slot);
                if (!((bits[h >> 5] >> (h & 31u)) & 1u)) continue;
            }
            for (uint32_t j = 0; j < tokens && t0 + j < o; j++)
                if (a.d_slots[t0 + j] == slot && kind(slot, o) == 0) atomicOr(&shadowed[j >> 5], 1u << (j & 31u));
        }
        __syncthreads();
    }
    const uint32_t half = a.rot / 2, rotated = a.rot / (2 * W);
    uint32_t bad = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kBlock) {
        const uint32_t j = p.by_units(skip + i), t = t0 + j, u = skip + i - j * p.units, hh = p.by_head(u), m = u - hh * p.head_units;
        const bool is_q = hh < a.heads, is_k = !is_q && hh < a.heads + c.heads, turns = (is_q || is_k) && m < rotated;
        const uint32_t h = is_q ? hh : is_k ? hh - a.heads : hh - a.heads - c.heads;
        const int32_t* x = (is_q ? a.d_q + t * a.q_stride : is_k ? a.d_k + t * a.k_stride : a.d_v + t * a.v_stride) + (size_t)h * c.dim;
        // the unit's two parts: side by side, or half a rotation apart; the second may lie past the head's end
        const bool halves = turns && !a.interleaved;
        const uint32_t e0 = (halves ? W : 2 * W) * m, e1 = halves ? e0 + half : e0 + W;
        const bool second = e1 < c.dim;
        Elements<W> x0, x1;
        x0.load(x + e0);
        if (second) x1.load(x + e1);
        const int64_t slot = a.d_slots[t];
        if (slot < 0) continue;
        const int k = kind(slot, t);
        if (k) {
            if (u == 0) bad |= (uint32_t)kWitIndex;
            continue;
        }
        int32_t *q = nullptr, *r = nullptr;
        if (is_q) {
            const size_t o = ((size_t)t * a.heads + h) * c.dim;
            q = a.d_q_out + o;
            if (a.d_q_rem) r = a.d_q_rem + o;
        } else {
            if (t0 + 1 >= a.tokens || !((shadowed[j >> 5] >> (j & 31u)) & 1u)) {
                const uint32_t pg = p.by_page((uint32_t)slot);
                q = (is_k ? c.d_k : c.d_v) + token::token_offset(c, (int32_t)pg, (uint32_t)slot - pg * c.page_size) + h * c.head_stride;
            }
            if (is_k && a.d_k_rem) r = a.d_k_rem + ((size_t)t * c.heads + h) * c.dim;
        }
        Elements<W> r0, r1;
#pragma unroll
        for (int w = 0; w < W; w++) r0.v[w] = r1.v[w] = 0;
        if (turns) {
            const size_t row = (size_t)a.d_positions[t] * half + W * m;
            Elements<W> cs, sn;
            cs.load(a.d_cos + row);
            sn.load(a.d_sin + row);
            Elements<W> q0, q1;
            auto turn = [&](int32_t y0, int32_t y1, int w, int32_t& o0, int32_t& s0, int32_t& o1, int32_t& s1) {
                p.scale.apply((int64_t)y0 * cs.v[w] - (int64_t)y1 * sn.v[w], o0, s0, bad);
                p.scale.apply((int64_t)y0 * sn.v[w] + (int64_t)y1 * cs.v[w], o1, s1, bad);
            };
            if (a.interleaved) {
                // elements in the order of memory: pair w is elements 2 w and 2 w + 1 of the 2 W
                auto at = [&](Elements<W>& y0, Elements<W>& y1, int e) -> int32_t& { return e < W ? y0.v[e] : y1.v[e - W]; };
#pragma unroll
                for (int w = 0; w < W; w++) turn(at(x0, x1, 2 * w), at(x0, x1, 2 * w + 1), w, at(q0, q1, 2 * w), at(r0, r1, 2 * w), at(q0, q1, 2 * w + 1), at(r0, r1, 2 * w + 1));
            } else {
#pragma unroll
                for (int w = 0; w < W; w++) turn(x0.v[w], x1.v[w], w, q0.v[w], r0.v[w], q1.v[w], r1.v[w]);
            }
            x0 = q0;
            x1 = q1;
        }
        if (q) {
            x0.store(q + e0);
            if (second) x1.store(q + e1);
        }
        if (r) {
            r0.store(r + e0);
            if (second) r1.store(r + e1);
        }
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
    token::FastDiv by_group;
    Scaler scale;
    uint32_t* status;
    uint32_t *digits, *over;     // of the inputs, where a launch of its own makes them
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
            const size_t at = (size_t)m * p.groups + p.by_group(k);
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

// Groups of whole 32s, on the matrix cores.  The input x = sum_p d_p 256^p (balanced digits, four planes) gives a token four rows of
// the first operand, and a weight byte of the second is one nibble of the packed byte moved to the upper half with its top bit
// turned over: 16 (w - 8) as a signed byte.  A lane's 16 packed bytes are 32 of the row's weights, the even ones and the odd ones an
// operand each, with the digits laid out in the same order.  Lane l then holds the four planes of token l / 16 for weight row
// l % 16, the row whose bytes it has read: one scale a lane.  After each step (GS inputs, which lie in one group) two planes at a
// time are put together in 32 bits (128 * 128 * 8 * 257 and the zero points' part stay below 2^31), scaled and added in 64 bits.
// Zero points other than 8 add (8 - z) * sum of digits; one more product, with ones, gives those sums in the same registers.
// The waves of a workgroup take consecutive shares of a tile of 16 rows' inputs, so that 4096 rows fill the chip; what a wave needs
// next is requested some units of 128 inputs ahead.
constexpr int kQ4Waves = 8, kQ4Threads = 64 * kQ4Waves;
// waves of a workgroup for up to four tokens at most: four scales a lane need the registers of twice as many
constexpr uint32_t q4_most_waves(int gs) { return gs == 32 ? 8 : 16; }

// N bytes of a weight row of `bytes`, from `at`.  Where they pass the row's end, the row's last N are read and shifted instead (a
// loop over bytes takes a load's latency for each: one token through 16384 x 1000 9.9 us a call and not 7.2, 4096 x 2033 9.4 and
// not 7.2); what stands behind the end then meets digits of zero, whatever it is.
template <int N>
__device__ __forceinline__ void q4_bytes(const uint8_t* s, uint32_t at, uint32_t bytes, uint32_t* out) {
    if (bytes >= N) {
        const uint32_t from = min(at, bytes - N), past = at - from;
        uint64_t v[2] = {0, 0};
        __builtin_memcpy(v, s + from, N);
        if (past) {
            if (past & 8u) v[0] = v[1];
            const uint32_t bits = 8 * (past & 7u);
            v[0] >>= bits;
            if (bits) v[0] |= v[1] << (64 - bits);
            v[1] >>= bits;
        }
        __builtin_memcpy(out, v, N);
    } else {
#pragma unroll
        for (int j = 0; j < N / 4; j++) {
            out[j] = 0;
#pragma unroll 1
            for (uint32_t b = 0; b < 4; b++) out[j] |= (at + 4 * j + b < bytes ? (uint32_t)s[at + 4 * j + b] : 0u) << (8 * b);
        }
    }
}

// Four units of 128 inputs of 16 weight rows.  A wave reads 256 bytes in a row among 16 neighbouring lanes, then turns them over
// through 4 KB of LDS of its own into the operands, where 16 neighbouring lanes hold 16 rows: read as operands in the first place,
// every lane's 16 bytes would be a line of memory of their own, and so would the scales (22.5 MB of weights with scales and zero
// points for each 64 took 17.7 us that way).  Scales and zero points are read by lane 4 r + s for row r and unit s.
template <int GS>
struct Q4Quad {
    static constexpr int STEPS = 128 / GS;          // scalings of a unit
    v4i_t w[4];
    int32_t scale[STEPS];
    uint32_t zeros;                                 // a byte a step
    __device__ __forceinline__ void load(const Q4Args& p, uint32_t m0, uint32_t unit, uint32_t lane) {
        const uint32_t bytes = (p.inputs + 1) / 2, at = unit * 64 + 16 * (lane & 15u);
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint8_t* s = p.w + min(m0 + 4 * i + (lane >> 4), p.outputs - 1) * p.w_stride;
            q4_bytes<16>(s, at, bytes, reinterpret_cast<uint32_t*>(&w[i]));
        }
        const uint32_t row = min(m0 + (lane >> 2), p.outputs - 1), u = unit + (lane & 3u);
        const size_t first = (size_t)row * p.groups;
        zeros = 0;
        if (p.group == GS && (u + 1) * STEPS <= p.groups) {          // neighbours
            __builtin_memcpy(scale, p.scales + first + u * STEPS, 4 * STEPS);
            if (p.zeros) __builtin_memcpy(&zeros, p.zeros + first + u * STEPS, STEPS);
            return;
        }
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            const uint32_t g = min(p.by_group(min(u * 128 + st * GS, p.inputs - 1)), p.groups - 1);
            scale[st] = p.scales[first + g];
            if (p.zeros) zeros |= (uint32_t)p.zeros[first + g] << (8 * st);
        }
    }
    // 16 bytes: chunk c of row r stands at 16 r + (c ^ r), so that the sixteen rows' equal chunks spread over the banks
    __device__ __forceinline__ void store(uint8_t* lds, uint32_t lane) const {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t r = 4 * i + (lane >> 4), c = lane & 15u;
            *reinterpret_cast<v4i_t*>(lds + 16 * (16 * r + (c ^ r))) = w[i];
        }
    }
};

// A lane's 16 bytes of unit s of its row, and its scales: GS / 2 bytes of a step lie among the four lane groups.
template <int GS>
struct Q4Unit {
    static constexpr int STEPS = 128 / GS, CB = GS / 8;
    v4i_t w;
    int32_t scale[STEPS], zero[STEPS];
    // straight from memory, every lane for itself
    __device__ __forceinline__ void load(const Q4Args& p, uint32_t row, uint32_t unit, uint32_t kg) {
        const uint8_t* s = p.w + row * p.w_stride;
        const uint32_t bytes = (p.inputs + 1) / 2, base = unit * 64;
        union { v4i_t v; uint32_t u[4]; } o;
        if (CB < 16 && base + 64 <= bytes) {          // several shifts less
#pragma unroll
            for (int c = 0; c < 16 / CB; c++) __builtin_memcpy(o.u + c * CB / 4, s + base + c * (GS / 2) + kg * CB, CB);
        } else {
#pragma unroll
            for (int c = 0; c < 16 / CB; c++) q4_bytes<CB>(s, base + c * (GS / 2) + kg * CB, bytes, o.u + c * CB / 4);
        }
        w = o.v;
        const size_t first = (size_t)row * p.groups;
        if (p.group == GS && (unit + 1) * STEPS <= p.groups) {          // neighbours
            __builtin_memcpy(scale, p.scales + first + unit * STEPS, 4 * STEPS);
            uint8_t z[STEPS];
            if (p.zeros) __builtin_memcpy(z, p.zeros + first + unit * STEPS, STEPS);
#pragma unroll
            for (int st = 0; st < STEPS; st++) zero[st] = p.zeros ? z[st] : 8;
            return;
        }
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            const uint32_t g = min(p.by_group(unit * 128 + st * GS), p.groups - 1);
            scale[st] = p.scales[first + g];
            zero[st] = p.zeros ? (int32_t)p.zeros[first + g] : 8;
        }
    }
    // from four units that have been turned over
    __device__ __forceinline__ void take(const Q4Quad<GS>& q, const uint8_t* lds, uint32_t s, uint32_t lane, bool zeros) {
        const uint32_t r = lane & 15u, kg = lane >> 4;
        union { v4i_t v; uint32_t u[4]; uint2 d[2]; } o;
#pragma unroll
        for (uint32_t c = 0; c < 16 / CB; c++) {
            const uint32_t at = 64 * s + c * (GS / 2) + kg * CB, chunk = at >> 4;
            const uint8_t* from = lds + 16 * (16 * r + (chunk ^ r)) + (at & 15u);
            if constexpr (CB == 16) o.v = *reinterpret_cast<const v4i_t*>(from);
            else if constexpr (CB == 8) o.d[c] = *reinterpret_cast<const uint2*>(from);
            else o.u[c] = *reinterpret_cast<const uint32_t*>(from);
        }
        w = o.v;
        const uint32_t z = zeros ? (uint32_t)__shfl((int)q.zeros, 4 * r + s, 64) : 0u;
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            scale[st] = __shfl(q.scale[st], 4 * r + s, 64);
            zero[st] = (int32_t)((z >> (8 * st)) & 255u);
        }
    }
};

// what one lane of a wave wrote to LDS is there for the others
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Where the word of plane pl of token n (of `cols` / 4) and the inputs 8 e .. 8 e + 7 stands, in words, among the first operands:
// [unit][operand][lane group][column] of 16 bytes (GS = 32: of 8, four operands a unit instead of two).  `odd`: the odd inputs' word.
template <int GS>
__device__ __forceinline__ size_t q4_word(uint32_t e, uint32_t n, uint32_t pl, uint32_t cols, uint32_t odd) {
    const uint32_t in = e & 15u, col = 4 * n + pl;
    const size_t unit = e >> 4;
    if constexpr (GS == 128) return ((((unit * 2 + odd) * 4 + (in >> 2)) * cols + col) << 2) + (in & 3u);
    else if constexpr (GS == 64) return ((((unit * 2 + (in >> 3)) * 4 + ((in >> 1) & 3u)) * cols + col) << 2) + 2 * odd + (in & 1u);
    else return ((((unit * 4 + (in >> 2)) * 4 + (in & 3u)) * cols + col) << 1) + odd;
}

// Digits of eight inputs of token n, from 8 e; true where one has a top digit of 128, which its byte holds as -128.
template <int GS>
__device__ __forceinline__ bool q4_digits(const Q4Args& p, uint32_t n, uint32_t e, uint32_t* out, uint32_t e_out, uint32_t n_out, uint32_t cols) {
    const uint32_t k = 8 * e;
    const int32_t* x = p.x + n * p.x_stride + k;
    int32_t v[8];
    if (k + 8 <= p.inputs) __builtin_memcpy(v, x, 32);
    else
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = k + j < p.inputs ? x[j] : 0;
    uint32_t d[8], lo[4], hi[4];
    bool over = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        d[i] = digits_of(v[i]);
        over |= v[i] > kDigitTop;
    }
    transpose4(d[0], d[2], d[4], d[6], lo);
    transpose4(d[1], d[3], d[5], d[7], hi);
#pragma unroll
    for (int pl = 0; pl < 4; pl++) {
        out[q4_word<GS>(e_out, n_out, pl, cols, 0)] = lo[pl];
        out[q4_word<GS>(e_out, n_out, pl, cols, 1)] = hi[pl];
    }
    return over;
}

// One unit of 128 inputs: the sums of planes 0, 1 and of planes 2, 3 of NT tiles of four tokens.  operand(op, j): the digits.
template <int GS, int NT, class F>
__device__ __forceinline__ void q4_unit(const Q4Unit<GS>& x, bool zeros, int64_t (*y)[2], F operand) {
    v4i_t even, odd;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t w = (uint32_t)x.w[c] ^ 0x88888888u;
        even[c] = (int)((w << 4) & 0xf0f0f0f0u);
        odd[c] = (int)(w & 0xf0f0f0f0u);
    }
    const v4i_t none = {0, 0, 0, 0}, one = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
#pragma unroll
    for (int st = 0; st < 128 / GS; st++) {
        // all tiles' products before the first one's sums are looked at
        v4i_t acc[NT], ones[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) acc[j] = ones[j] = none;
        if constexpr (GS == 32) {
            const long w = (long)(((uint64_t)(uint32_t)odd[st] << 32) | (uint32_t)even[st]);
            long d[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) d[j] = operand(st, j);
#pragma unroll
            for (int j = 0; j < NT; j++) acc[j] = __builtin_amdgcn_mfma_i32_16x16x32_i8(d[j], w, acc[j], 0, 0, 0);
            if (zeros) {
#pragma unroll
                for (int j = 0; j < NT; j++) ones[j] = __builtin_amdgcn_mfma_i32_16x16x32_i8(d[j], 0x0101010101010101L, ones[j], 0, 0, 0);
            }
        } else {
            v4i_t d[GS / 64][NT];
#pragma unroll
            for (int op = 0; op < GS / 64; op++)
#pragma unroll
                for (int j = 0; j < NT; j++) d[op][j] = operand(st + op, j);
#pragma unroll
            for (int op = 0; op < GS / 64; op++) {
                v4i_t w;
                if constexpr (GS == 128) w = op ? odd : even;
                else w = v4i_t{even[2 * st], even[2 * st + 1], odd[2 * st], odd[2 * st + 1]};
#pragma unroll
                for (int j = 0; j < NT; j++) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(d[op][j], w, acc[j], 0, 0, 0);
            }
            if (zeros) {
#pragma unroll
                for (int op = 0; op < GS / 64; op++)
#pragma unroll
                    for (int j = 0; j < NT; j++) ones[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(d[op][j], one, ones[j], 0, 0, 0);
            }
        }
        const int32_t up = 8 - x.zero[st];
#pragma unroll
        for (int j = 0; j < NT; j++) {
            int32_t s[4];
#pragma unroll
            for (int i = 0; i < 4; i++) s[i] = (acc[j][i] >> 4) + (zeros ? __mul24(up, ones[j][i]) : 0);
            y[j][0] += (int64_t)(s[0] + 256 * s[1]) * x.scale[st];
            y[j][1] += (int64_t)(s[2] + 256 * s[3]) * x.scale[st];
        }
    }
}

// What inputs above kDigitTop of token n are short of in row m: 2^32 of each.
__device__ __forceinline__ uint64_t q4_over(const Q4Args& p, uint32_t n, uint32_t m) {
    const int32_t* x = p.x + n * p.x_stride;
    const uint8_t* w = p.w + m * p.w_stride;
    uint64_t more = 0;
    for (uint32_t k = 0; k < p.inputs; k++)
        if (x[k] > kDigitTop) {
            const size_t at = (size_t)m * p.groups + p.by_group(k);
            more += (uint64_t)((int64_t)p.scales[at] * ((int32_t)((w[k >> 1] >> (4 * (k & 1u))) & 15u) - (p.zeros ? (int32_t)p.zeros[at] : 8)));
        }
    return more << 32;
}

__device__ __forceinline__ void q4_out(const Q4Args& p, uint32_t n, uint32_t m, int64_t y, uint32_t& bad) {
    int32_t q, r;
    p.scale.apply(y, q, r, bad);
    const size_t o = (size_t)n * p.outputs + m;
    p.q[o] = q;
    if (p.r) p.r[o] = r;
}

// Up to four tokens: a workgroup makes their digits itself, in LDS (a longer input goes through in pieces), while its first weights
// are under way.  One token through 4096 x 4096, groups of 128: 5.7 us, as long as a launch and a chain of loads take; 11008 x 4096,
// groups of 64 with zero points, 26 MB: 12.1 us, 2.1 TB/s.  Not the memory bounds that (all 688 workgroups are resident, 11 MB requested at
// the start) but the chain in each: inputs, digits, weights turned over, a second quad, the join; and the digits are made 688 times
// and LDS waits 7.5e5 cycles for its banks in 2.1e5 instructions.  blockDim: as many waves as share a tile's inputs, 4 KB of LDS each
// behind the digits.
template <int GS>
__global__ void __launch_bounds__(64 * q4_most_waves(GS), GS == 32 ? 2 : 4) wit_q4_few_kernel(Q4Args p, uint32_t piece) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ uint32_t over_any;
    constexpr int OPS = GS == 32 ? 4 : 2;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, col = lane & 15u, kg = lane >> 4;
    const uint32_t nt = p.tokens, cols = 4 * nt, units = (p.inputs + 127) / 128, m0 = blockIdx.x * 16;
    const uint32_t at_col = col < cols ? col : 0;          // rows past the tokens' planes: nothing of them is kept
    uint8_t* turned = reinterpret_cast<uint8_t*>(lds + (size_t)piece * 128 * nt) + 4096 * wave;
    if (threadIdx.x == 0) over_any = 0;
    int64_t y[1][2] = {{0, 0}};
    for (uint32_t u0 = 0; u0 < units; u0 += piece) {
        // shares of whole fours
        const uint32_t un = min(units - u0, piece), share = ((un + waves - 1) / waves + 3) / 4 * 4;
        const uint32_t first = min(wave * share, un), last = min(first + share, un);          // of this wave, in the piece
        Q4Quad<GS> next;
        if (first < last) next.load(p, m0, u0 + first, lane);
        __syncthreads();                                    // the digits of the piece before are not needed any more
        for (uint32_t i = threadIdx.x; i < un * 16 * nt; i += blockDim.x) {
            const uint32_t n = i / (un * 16), e = i - n * (un * 16);
            if (q4_digits<GS>(p, n, u0 * 16 + e, lds, e, n, cols)) over_any = 1;
        }
        __syncthreads();
#pragma unroll 1
        for (uint32_t u = first; u < last; u += 4) {
            const Q4Quad<GS> quad = next;
            if (u + 4 < last) next.load(p, m0, u0 + u + 4, lane);
            wave_sync();
            quad.store(turned, lane);
            wave_sync();
#pragma unroll 1
            for (uint32_t s = 0; s < 4 && u + s < last; s++) {
                Q4Unit<GS> x;
                x.take(quad, turned, s, lane, p.zeros != nullptr);
                q4_unit<GS, 1>(x, p.zeros != nullptr, y, [&](int op, int) {
                    const uint32_t o = (((u + s) * OPS + op) * 4 + kg) * cols + at_col;
                    if constexpr (GS == 32) return reinterpret_cast<const long*>(lds)[o];
                    else return reinterpret_cast<const v4i_t*>(lds)[o];
                });
            }
        }
    }
    __syncthreads();
    int64_t* sum = reinterpret_cast<int64_t*>(lds);          // [wave][lane]
    sum[threadIdx.x] = y[0][0] + (int64_t)((uint64_t)y[0][1] << 16);
    __syncthreads();
    if (wave == 0 && kg < nt && m0 + col < p.outputs) {
        int64_t v = 0;
        for (uint32_t k = 0; k < waves; k++) v += sum[64 * k + lane];
        if (over_any) v += (int64_t)q4_over(p, kg, m0 + col);
        uint32_t bad = 0;
        q4_out(p, kg, m0 + col, v, bad);
        if (bad) atomicOr(p.status, bad);
    }
}

// More tokens: their digits are made once, by a launch of its own, and read from L2 as operands, 4 NT tokens at a time for RT tiles
// of 16 rows.  For 16 tokens through 4096 x 11008 (14.3 us, of which reading the weights would take 5) those are 180 MB, 12 TB/s: what a
// chain reaches that requests a unit's digits when it multiplies them, with eight waves a CU; the rate of L2 itself was not measured.
// 64 tokens 39 us a call, 256 142: weights and digits are read again for each sixteen.  Digits in LDS for 128 rows at a time ask for 22 MB instead, but leave a workgroup a CU of which each waits for
// its next weights, and sums to be joined: 14.8 and 3.9 us.
template <int GS>
__global__ void __launch_bounds__(kBlock) wit_q4_digits_kernel(Q4Args p, uint32_t tile_tokens) {
    __shared__ uint32_t over;
    const uint32_t units = (p.inputs + 127) / 128, n = blockIdx.y, e = blockIdx.x * kBlock + threadIdx.x, tile = n / tile_tokens, cols = 4 * tile_tokens;
    if (threadIdx.x == 0) over = 0;
    __syncthreads();
    uint32_t* out = p.digits + (size_t)tile * units * 32 * cols;          // 128 inputs of a column are 32 words
    if (e < units * 16 && q4_digits<GS>(p, n, e, out, e, n - tile * tile_tokens, cols)) over = 1;
    __syncthreads();
    if (threadIdx.x == 0) p.over[(size_t)n * gridDim.x + blockIdx.x] = over;
}

// Whether the weights go through LDS: with scales for each 64 or 32 the lanes of a row load short pieces, and many.  Four tokens
// through 16384 x 8192, with zero points: 39 us and not 55 with groups of 32, 33 and not 39 with groups of 64.  With sixteen the registers
// are not enough for it (96 us and not 90).
constexpr bool q4_turns(int gs, int nt) { return gs < 128 && nt < 4; }
template <int GS, int NT, int RT>
__global__ void __launch_bounds__(kQ4Threads, 2) wit_q4_many_kernel(Q4Args p, uint32_t makers) {
    constexpr int kQ4ManyAhead = 2, OPS = GS == 32 ? 4 : 2;
    constexpr uint32_t COLS = 16 * NT;
    // the weights to be turned over, 4 KB a wave and tile, and in the end the waves' sums
    constexpr bool kTurns = q4_turns(GS, NT);
    constexpr size_t kTurned = kTurns ? kQ4Waves * RT * 4096 : 0, kSums = sizeof(int64_t) * kQ4Waves * RT * NT * 64;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kTurned > kSums ? kTurned : kSums];
    __shared__ uint32_t over_any;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, col = lane & 15u, kg = lane >> 4;
    const uint32_t units = (p.inputs + 127) / 128, m0 = blockIdx.x * 16 * RT, n0 = blockIdx.y * 4 * NT;
    const uint32_t* digits = p.digits + (size_t)blockIdx.y * units * 32 * COLS;
    if (threadIdx.x == 0) over_any = 0;
    int64_t y[RT][NT][2];
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < NT; j++) y[t][j][0] = y[t][j][1] = 0;
    // shares of whole fours where the weights go through LDS, unless that leaves most waves without one
    const uint32_t even = (units + kQ4Waves - 1) / kQ4Waves, share = kTurns && even > 2 ? (even + 3) / 4 * 4 : even;
    const uint32_t first = min(wave * share, units), last = min(first + share, units);
    typedef typename std::conditional<GS == 32, long, v4i_t>::type operand_t;
    if constexpr (kTurns) {
        uint8_t* turned = lds + wave * RT * 4096;
        Q4Quad<GS> next[RT];
#pragma unroll
        for (int t = 0; t < RT; t++)
            if (first < last) next[t].load(p, m0 + 16 * t, first, lane);
        operand_t d[OPS][NT];                                    // the next unit's digits
        auto fetch = [&](uint32_t u) {
#pragma unroll
            for (int op = 0; op < OPS; op++)
#pragma unroll
                for (int j = 0; j < NT; j++) d[op][j] = reinterpret_cast<const operand_t*>(digits)[(((size_t)u * OPS + op) * 4 + kg) * COLS + 16 * j + col];
        };
        if (first < last) fetch(first);
#pragma unroll 1
        for (uint32_t u = first; u < last; u += 4) {
            Q4Quad<GS> quad[RT];
            wave_sync();
#pragma unroll
            for (int t = 0; t < RT; t++) {
                quad[t] = next[t];
                quad[t].store(turned + 4096 * t, lane);
                if (u + 4 < last) next[t].load(p, m0 + 16 * t, u + 4, lane);
            }
            wave_sync();
#pragma unroll 1
            for (uint32_t s = 0; s < 4 && u + s < last; s++) {
                operand_t now[OPS][NT];
#pragma unroll
                for (int op = 0; op < OPS; op++)
#pragma unroll
                    for (int j = 0; j < NT; j++) now[op][j] = d[op][j];
                if (u + s + 1 < last) fetch(u + s + 1);
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    Q4Unit<GS> x;
                    x.take(quad[t], turned + 4096 * t, s, lane, p.zeros != nullptr);
                    q4_unit<GS, NT>(x, p.zeros != nullptr, y[t], [&](int op, int j) { return now[op][j]; });
                }
            }
        }
    } else {
        Q4Unit<GS> next[kQ4ManyAhead][RT];
#pragma unroll
        for (int s = 0; s < kQ4ManyAhead; s++)
#pragma unroll
            for (int t = 0; t < RT; t++)
                if (first + s < last) next[s][t].load(p, min(m0 + 16 * t + col, p.outputs - 1), first + s, kg);
#pragma unroll 1
        for (uint32_t u = first; u < last; u++) {
            operand_t d[OPS][NT];
#pragma unroll
            for (int op = 0; op < OPS; op++)
#pragma unroll
                for (int j = 0; j < NT; j++) d[op][j] = reinterpret_cast<const operand_t*>(digits)[(((size_t)u * OPS + op) * 4 + kg) * COLS + 16 * j + col];
            Q4Unit<GS> x[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                x[t] = next[0][t];
#pragma unroll
                for (int s = 0; s + 1 < kQ4ManyAhead; s++) next[s][t] = next[s + 1][t];
                if (u + kQ4ManyAhead < last) next[kQ4ManyAhead - 1][t].load(p, min(m0 + 16 * t + col, p.outputs - 1), u + kQ4ManyAhead, kg);
            }
#pragma unroll
            for (int t = 0; t < RT; t++) q4_unit<GS, NT>(x[t], p.zeros != nullptr, y[t], [&](int op, int j) { return d[op][j]; });
        }
    }
    __syncthreads();
    int64_t(*sum)[RT * NT * 64] = reinterpret_cast<int64_t(*)[RT * NT * 64]>(lds);
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < NT; j++) sum[wave][(t * NT + j) * 64 + lane] = y[t][j][0] + (int64_t)((uint64_t)y[t][j][1] << 16);
    __syncthreads();
    const uint32_t over_words = min(4u * NT, p.tokens - n0) * makers;
    for (uint32_t i = threadIdx.x; i < over_words; i += kQ4Threads)
        if (p.over[(size_t)n0 * makers + i]) over_any = 1;
    __syncthreads();
    uint32_t bad = 0;
    for (uint32_t i = threadIdx.x; i < RT * NT * 64; i += kQ4Threads) {
        const uint32_t m = m0 + 16 * (i / (64 * NT)) + (i & 15u), n = n0 + 4 * (i / 64 % NT) + ((i >> 4) & 3u);
        if (m >= p.outputs || n >= p.tokens) continue;
        int64_t v = 0;
#pragma unroll
        for (int k = 0; k < kQ4Waves; k++) v += sum[k][i];
        if (over_any) v += (int64_t)q4_over(p, n, m);
        q4_out(p, n, m, v, bad);
    }
    if (bad) atomicOr(p.status, bad);
}

template <int GS>
static int q4_launch(const Q4Args& p, hipStream_t s) {
    const uint32_t units = (p.inputs + 127) / 128, tiles = (p.outputs + 15) / 16;
    if (token::q4_few(p.tokens, p.outputs, p.inputs)) {
        // a wave for each four units of 128 inputs, and no more than sixteen a CU where that leaves four
        uint32_t waves = std::min((units + 3) / 4, std::min(q4_most_waves(GS), std::max(4u, 16u * kNumCU / tiles)));
        const uint32_t share = ((units + waves - 1) / waves + 3) / 4 * 4;
        waves = (units + share - 1) / share;
        const uint32_t piece = std::min(units, token::kTokenLds / (512 * p.tokens) / 4 * 4);
        wit_q4_few_kernel<GS><<<tiles, 64 * waves, (size_t)piece * 512 * p.tokens + 4096 * waves, s>>>(p, piece);
        GRAPE_LAUNCH_CHECK();
        return GRAPE_OK;
    }
    const token::Q4Plan plan = token::q4_plan(p.tokens, p.inputs);
    wit_q4_digits_kernel<GS><<<dim3(plan.makers, p.tokens), kBlock, 0, s>>>(p, plan.tile_tokens);
    GRAPE_LAUNCH_CHECK();
    // two tiles of rows share the digits where that still leaves a workgroup for each CU (and the registers are enough)
    constexpr int kMost = GS == 32 ? 0 : GS == 64 ? 4 : 1;          // from which NT on
    const uint32_t nt = plan.tile_tokens / 4;
    const bool two = kMost && nt >= kMost && (uint64_t)(tiles + 1) / 2 * plan.token_tiles >= (uint64_t)kNumCU;
    const dim3 grid(two ? (tiles + 1) / 2 : tiles, plan.token_tiles);
    if constexpr (GS == 128) {
        if (two && nt == 1) wit_q4_many_kernel<GS, 1, 2><<<grid, kQ4Threads, 0, s>>>(p, plan.makers);
        else if (two && nt == 2) wit_q4_many_kernel<GS, 2, 2><<<grid, kQ4Threads, 0, s>>>(p, plan.makers);
    }
    if constexpr (GS >= 64) {
        if (two && nt == 4) wit_q4_many_kernel<GS, 4, 2><<<grid, kQ4Threads, 0, s>>>(p, plan.makers);
    }
    if (!two && nt == 1) wit_q4_many_kernel<GS, 1, 1><<<grid, kQ4Threads, 0, s>>>(p, plan.makers);
    else if (!two && nt == 2) wit_q4_many_kernel<GS, 2, 1><<<grid, kQ4Threads, 0, s>>>(p, plan.makers);
    else if (!two) wit_q4_many_kernel<GS, 4, 1><<<grid, kQ4Threads, 0, s>>>(p, plan.makers);
    GRAPE_LAUNCH_CHECK();
    return GRAPE_OK;
}

}  // namespace grape

using namespace grape;

extern "C" {

int grape_wit_rope_append(const grape_wit_rope_append_args* args, const grape_wit_cache* cache, grape_stream_t st) {
    GRAPE_REQUIRE(initialised(), "grape_init has not been called");
    GRAPE_REFUSED_IF(token::refuse_append(args, cache));
    if (args->tokens == 0) return GRAPE_OK;
    AppendArgs p;
    p.a = *args;
    p.c = *cache;
    const grape_wit_rope_append_args& a = p.a;
    auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    const bool vec = p.c.dim % 4 == 0 && a.rot % 8 == 0 && ((a.q_stride | a.k_stride | a.v_stride | p.c.page_stride | p.c.token_stride | p.c.head_stride) & 3) == 0 &&
                     aligned(a.d_q) && aligned(a.d_k) && aligned(a.d_v) && aligned(a.d_cos) && aligned(a.d_sin) && aligned(a.d_q_out) && aligned(a.d_q_rem) &&
                     aligned(a.d_k_rem) && aligned(p.c.d_k) && aligned(p.c.d_v);
    p.head_units = token::append_head_units(p.c.dim, a.rot, vec ? 4 : 1);
    p.units = (a.heads + 2 * p.c.heads) * p.head_units;
    p.total = (uint64_t)a.tokens * p.units;
    // one unit a thread as long as that fills the chip, then longer shares (2048 tokens of a head of 4096: 80 us; in twice as many 83)
    uint64_t per = std::max<uint64_t>(kBlock, (p.total + 2047) / 2048);
    per = std::min<uint64_t>((per + kBlock - 1) / kBlock * kBlock, (uint64_t)(kAppendTokens - 2) * p.units);
    p.per = (uint32_t)per;
    p.by_units = token::fast_div(p.units);
    p.by_head = token::fast_div(p.head_units);
    p.by_page = token::fast_div(p.c.page_size);
    p.scale = scaler(a.scale);
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status);
    if (rc) return rc;
    const unsigned grid = (unsigned)((p.total + per - 1) / per);
    if (vec) wit_append_kernel<4><<<grid, kBlock, 0, s>>>(p);
    else wit_append_kernel<1><<<grid, kBlock, 0, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    return GRAPE_OK;
}

size_t grape_wit_matvec_q4_workspace(uint32_t tokens, uint32_t outputs, uint32_t inputs, uint32_t group) {
    return token::q4_workspace(tokens, outputs, inputs, group);
}

int grape_wit_matvec_q4(int32_t* d_q, int32_t* d_r, const int32_t* d_x, int64_t x_stride, const uint8_t* d_w, int64_t w_stride,
                        const int32_t* d_scales, const uint8_t* d_zeros, uint32_t tokens, uint32_t outputs, uint32_t inputs,
                        uint32_t group, int64_t scale, void* d_workspace, size_t workspace_bytes, grape_stream_t st) {
    GRAPE_REQUIRE(initialised(), "grape_init has not been called");
    GRAPE_REFUSED_IF(token::refuse_q4(d_q, d_x, x_stride, d_w, w_stride, d_scales, tokens, outputs, inputs, group, scale, d_workspace, workspace_bytes));
    if (tokens == 0 || outputs == 0) return GRAPE_OK;
    Q4Args p;
    p.q = d_q; p.r = d_r; p.x = d_x; p.x_stride = x_stride; p.w = d_w; p.w_stride = w_stride; p.scales = d_scales; p.zeros = d_zeros;
    p.tokens = tokens; p.outputs = outputs; p.inputs = inputs; p.group = group;
    p.groups = (inputs - 1) / group + 1;
    p.by_group = token::fast_div(group);
    p.scale = scaler(scale);
    p.digits = (uint32_t*)d_workspace;
    p.over = (uint32_t*)((uint8_t*)d_workspace + token::q4_plan(tokens, inputs).at_over);
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status);
    if (rc) return rc;
    if (group % 32) {
        wit_q4_any_kernel<<<dim3((outputs + 3) / 4, (tokens + 3) / 4), kBlock, 0, s>>>(p);
        GRAPE_LAUNCH_CHECK();
        return GRAPE_OK;
    }
    return group % 64 ? q4_launch<32>(p, s) : group % 128 ? q4_launch<64>(p, s) : q4_launch<128>(p, s);
}

}  // extern "C"

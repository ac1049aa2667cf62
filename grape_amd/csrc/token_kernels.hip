// The witness of new tokens: rotation and append to a paged cache, and products with 4-bit weights (their attention is in
// token_attention.hip).  The arithmetic is that of witness_kernels.hip: exact 64-bit products, rescaled.
#include <algorithm>
#include "token_device.hpp"

namespace grape {

// ------------------------------------------------------------------------------------------------
// Rotation and append.  A unit is W pairs of a rotated head or 2 W elements that only move; a token's units are those of its
// query heads, its key heads and its value heads.  W = 4: a unit is two 16-byte loads and two to four 16-byte stores.  Bound by
// memory; with few tokens by two loads that depend on each other, the position and its row of the tables.
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
    const int rc = wit_status_word(&p.status, s);
    if (rc) return rc;
    const unsigned grid = (unsigned)((p.total + per - 1) / per);
    if (vec) wit_append_kernel<4><<<grid, kBlock, 0, s>>>(p);
    else wit_append_kernel<1><<<grid, kBlock, 0, s>>>(p);
    GRAPE_LAUNCH_CHECK();
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

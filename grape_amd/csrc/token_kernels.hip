// The witness of new tokens: rotation and append to a paged cache, attention of one token a sequence over that cache, and
// products with 4-bit weights.  The arithmetic is that of witness_kernels.hip: exact 64-bit products, rescaled.
#include <algorithm>
#include "common.hpp"
#include "token_geometry.hpp"
#include "witness_device.hpp"

namespace grape {

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
// ------------------------------------------------------------------------------------------------
struct AttendArgs {
    grape_wit_attention_args a;
    grape_wit_cache c;
    int qk_shift, out_shift;
    uint32_t* status;
};

__device__ __forceinline__ bool span_of(const AttendArgs& p, uint32_t b, uint32_t& lo, uint32_t& hi) {
    return token::live_span(p.a.d_lens[b], p.a.d_first ? p.a.d_first[b] : 0, p.a.max_len, p.a.table_stride, p.c.page_size, lo, hi);
}

__device__ __forceinline__ int64_t token_at(const AttendArgs& p, uint32_t b, uint32_t t) {
    const uint32_t pg = t / p.c.page_size;
    return token::token_offset(p.c, p.a.d_block_table[(size_t)b * p.a.table_stride + pg], t - pg * p.c.page_size);
}

__global__ void __launch_bounds__(kBlock) wit_attend_scores_kernel(AttendArgs p) {
    const uint32_t t = blockIdx.x * kBlock + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
    uint32_t lo, hi, bad = 0;
    if (!span_of(p, b, lo, hi)) bad = kWitIndex;
    if (t >= lo && t < hi) {
        const int64_t at = token_at(p, b, t);
        int64_t s = 0;
        if (at < 0) bad |= (uint32_t)kWitIndex;
        else {
            const int32_t* k = p.c.d_k + at + (int64_t)(h / (p.a.heads / p.c.heads)) * p.c.head_stride;
            const int32_t* q = p.a.d_q + b * p.a.q_stride + (size_t)h * p.c.dim;
            for (uint32_t d = 0; d < p.c.dim; d++) s += (int64_t)q[d] * k[d];
        }
        const size_t o = ((size_t)b * p.a.heads + h) * p.a.max_len + t;
        int32_t q, r;
        rescale64(s, p.a.qk_scale, p.qk_shift, q, r, bad);
        p.a.d_scores[o] = q;
        if (p.a.d_scores_rem) p.a.d_scores_rem[o] = r;
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

__global__ void __launch_bounds__(kBlock) wit_attend_softmax_kernel(AttendArgs p) {
    const uint32_t h = blockIdx.x, b = blockIdx.y;
    const size_t row = (size_t)b * p.a.heads + h, o = row * p.a.max_len;
    uint32_t lo, hi, bad = 0;
    span_of(p, b, lo, hi);
    int32_t mx = INT32_MIN;
    for (uint32_t t = lo + threadIdx.x; t < hi; t += kBlock) mx = max(mx, p.a.d_scores[o + t]);
    mx = block_all(mx, [](int32_t x, int32_t y) { return max(x, y); });
    unsigned long long sum = 0;
    for (uint32_t t = lo + threadIdx.x; t < hi; t += kBlock) {
        const int64_t d = (int64_t)p.a.d_scores[o + t] - mx, idx = d + (((int64_t)1 << p.a.bit_shift) - 1);
        const bool ok = idx >= 0 && idx < ((int64_t)1 << p.a.index_bits);
        const int32_t e = p.a.d_exp_table[ok ? idx : 0];
        if (!ok) bad |= (uint32_t)kWitIndex;
        if (e < 0) bad |= (uint32_t)kWitSum;
        p.a.d_exp[o + t] = e;
        if (p.a.d_shifted) p.a.d_shifted[o + t] = (int32_t)d;
        sum += (unsigned long long)(e < 0 ? 0 : e);
    }
    sum = block_all(sum, [](unsigned long long x, unsigned long long y) { return x + y; });
    if (lo < hi && sum == 0) bad |= (uint32_t)kWitSum;
    if (threadIdx.x == 0) {
        if (p.a.d_max) p.a.d_max[row] = lo < hi ? mx : 0;
        if (p.a.d_sum) p.a.d_sum[row] = lo < hi && sum == 0 ? 1 : (int32_t)sum;
    }
    if (sum == 0) sum = 1;
    for (uint32_t t = lo + threadIdx.x; t < hi; t += kBlock) {
        const int32_t e = p.a.d_exp[o + t];
        const unsigned long long ev = e < 0 ? 0 : e, pr = (ev * p.a.prob_scale + (sum >> 1)) / sum;
        p.a.d_prob[o + t] = (int32_t)pr;
        if (p.a.d_query) p.a.d_query[o + t] = (int32_t)(ev * 2 * p.a.prob_scale - sum * (2 * pr - 1));
    }
    if (bad) atomicOr(p.status, bad);
}

__global__ void __launch_bounds__(kBlock) wit_attend_values_kernel(AttendArgs p) {
    const uint32_t d = blockIdx.x * kBlock + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
    if (d >= p.c.dim) return;
    const size_t row = (size_t)b * p.a.heads + h;
    uint32_t lo, hi, bad = 0;
    span_of(p, b, lo, hi);
    int64_t y = 0;
    for (uint32_t t = lo; t < hi; t++) {
        const int64_t at = token_at(p, b, t);
        if (at >= 0) y += (int64_t)p.a.d_prob[row * p.a.max_len + t] * p.c.d_v[at + (int64_t)(h / (p.a.heads / p.c.heads)) * p.c.head_stride + d];
    }
    int32_t q, r;
    rescale64(y, p.a.out_scale, p.out_shift, q, r, bad);
    p.a.d_out[row * p.c.dim + d] = q;
    if (p.a.d_out_rem) p.a.d_out_rem[row * p.c.dim + d] = r;
    if (bad) atomicOr(p.status, bad);
}

// ------------------------------------------------------------------------------------------------
// Products with 4-bit weights, one thread an output.
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
    int64_t scale;
    int shift;
    uint32_t* status;
};

__global__ void __launch_bounds__(kBlock) wit_q4_kernel(Q4Args p) {
    const uint64_t i = (uint64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= (uint64_t)p.tokens * p.outputs) return;
    const uint32_t n = (uint32_t)(i / p.outputs), m = (uint32_t)(i - (uint64_t)n * p.outputs);
    const int32_t* x = p.x + n * p.x_stride;
    const uint8_t* w = p.w + m * p.w_stride;
    int64_t y = 0;
    for (uint32_t g = 0; g < p.groups; g++) {
        const size_t at = (size_t)m * p.groups + g;
        const int32_t zero = p.zeros ? p.zeros[at] : 8;
        int64_t part = 0;
        for (uint64_t k = (uint64_t)g * p.group; k < std::min<uint64_t>((uint64_t)(g + 1) * p.group, p.inputs); k++)
            part += (int64_t)x[k] * (int32_t)(((w[k >> 1] >> (4 * (k & 1))) & 15) - zero);
        y += part * p.scales[at];
    }
    uint32_t bad = 0;
    int32_t q, r;
    rescale64(y, p.scale, p.shift, q, r, bad);
    p.q[i] = q;
    if (p.r) p.r[i] = r;
    if (bad) atomicOr(p.status, bad);
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
    const size_t row = (size_t)a.seqs * a.heads * a.max_len;
    int32_t* ws = (int32_t*)a.d_workspace;
    if (!a.d_scores) a.d_scores = ws;
    if (!a.d_exp) a.d_exp = ws + row;
    if (!a.d_prob) a.d_prob = ws + 2 * row;
    p.qk_shift = log2_exact(a.qk_scale);
    p.out_shift = log2_exact(a.out_scale);
    hipStream_t s = as_stream(st);
    const int rc = wit_status_word(&p.status, s);
    if (rc) return rc;
    wit_attend_scores_kernel<<<dim3(std::max(1u, blocks_for(a.max_len)), a.heads, a.seqs), kBlock, 0, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    wit_attend_softmax_kernel<<<dim3(a.heads, a.seqs), kBlock, 0, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    wit_attend_values_kernel<<<dim3(blocks_for(p.c.dim), a.heads, a.seqs), kBlock, 0, s>>>(p);
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
    p.scale = scale; p.shift = log2_exact(scale);
    hipStream_t s = as_stream(st);
    int rc = wit_status_word(&p.status, s);
    if (rc) return rc;
    wit_q4_kernel<<<blocks_for((size_t)tokens * outputs), kBlock, 0, s>>>(p);
    GRAPE_LAUNCH_CHECK();
    return GRAPE_OK;
}

}  // extern "C"

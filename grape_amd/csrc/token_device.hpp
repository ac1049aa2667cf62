// What the new tokens' kernels share: the rescaling of a whole launch, and integers as planes of signed bytes for the matrix cores.
#pragma once
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
        const int64_t t = (int64_t)((uint64_t)y + (uint64_t)(s >> 1));
        int64_t qq;
        if (sh >= 0) {
            qq = t >> sh;
        } else {
            auto left = [&]() { return (int64_t)((uint64_t)t - (uint64_t)qq * (uint64_t)s); };
            qq = (int64_t)floor((double)t * inv);
            int64_t rest = left();
            if (rest < 0 || rest >= s) {
                qq += (int64_t)floor((double)rest * inv);
                rest = left();
                if (rest < 0) qq--;
                else if (rest >= s) qq++;
            }
        }
        bad |= (qq != (int64_t)(int32_t)qq) ? (uint32_t)kWitQuotient : 0u;
        q = (int32_t)qq;
        r = (int32_t)((uint64_t)y - (uint64_t)qq * (uint64_t)s);
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

}  // namespace grape

#define GRAPE_REFUSED_IF(expr)              \
    if (const char* why = (expr)) {         \
        set_error("%s: %s", __func__, why); \
        return GRAPE_EINVAL;                \
    }

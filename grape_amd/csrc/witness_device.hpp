// What the witness kernels share: the rescaling rule, the bits of the sticky status word and the word itself.
#pragma once
#include "common.hpp"

namespace grape {

enum WitFlag : uint32_t { kWitQuotient = 1, kWitIndex = 2, kWitSum = 4, kWitSquares = 8, kWitSumWide = 16 };

// floor((y + s/2) / s) and the centred remainder; s > 0, sh = log2(s) or -1 when s is no power of 2
__device__ __forceinline__ void rescale64(int64_t y, int64_t s, int sh, int32_t& q, int32_t& r, uint32_t& bad) {
    const int64_t t = y + (s >> 1);
    int64_t qq;
    if (sh >= 0) {
        qq = t >> sh;                         // arithmetic shift floors
    } else {
        qq = t / s;
        if ((t % s != 0) && (t < 0)) qq -= 1;  // C division truncates; floor wanted
    }
    bad |= (qq != (int64_t)(int32_t)qq) ? (uint32_t)kWitQuotient : 0u;
    q = (int32_t)qq;
    r = (int32_t)(y - qq * s);
}

// log2(s), or -1 where s is no power of 2
static inline int log2_exact(int64_t s) {
    if (s <= 0 || (s & (s - 1)) != 0) return -1;
    int sh = 0;
    while ((((int64_t)1) << sh) != s) sh++;
    return sh;
}

// the current device's status word
int wit_status_word(uint32_t** out);

}  // namespace grape

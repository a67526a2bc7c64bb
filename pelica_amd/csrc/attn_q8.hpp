// 8-bit cache values as f16.
#pragma once
#include "attn_common.hpp"

namespace pelica {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));

// The integers n of a word's bytes times a scale, in f16: a byte n + 128 behind
// 0x64 is the f16 number 1024 + 128 + n, exact, as is n after the subtraction;
// the product is rounded once.  7 instructions for 4 values.
__device__ __forceinline__ half4 q8_word(uint32_t w, half2 s) {
    w ^= 0x80808080u;
    const half2 lo = __builtin_bit_cast(half2, __builtin_amdgcn_perm(w, 0x64646464u, 0x00050004u));
    const half2 hi = __builtin_bit_cast(half2, __builtin_amdgcn_perm(w, 0x64646464u, 0x00070006u));
    const half2 off = {(_Float16)1152, (_Float16)1152};
    const half2 a = (lo - off) * s, b = (hi - off) * s;
    return half4{a[0], a[1], b[0], b[1]};
}
__device__ __forceinline__ half2 q8_scale(uint16_t s) {
    const _Float16 x = __builtin_bit_cast(_Float16, s);
    return half2{x, x};
}
__device__ __forceinline__ half8 q8_values(u32x2 w, uint16_t s) {
    const half2 x = q8_scale(s);
    return cat8(q8_word(w[0], x), q8_word(w[1], x));
}

}  // namespace pelica

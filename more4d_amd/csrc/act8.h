// The 8-bit form of a block of 32 channels (act8.hip: format and reasons), shared by the kernels that write or read it.
#pragma once
#include "common.h"

namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4q __attribute__((ext_vector_type(4)));

M4D_DEV float step_of(unsigned b) { return __builtin_bit_cast(float, b << 23); }      // 2^(b - 127); 255 -> +inf (times code 0: NaN)

// stored exponent byte of a block from the bits of its largest magnitude (as integers NaN > inf > every finite value):
// max = 1.f * 2^E gives e = E - 6, one more if 1.f > 127 / 64 (mantissa above 0x7e0000), within [-126, 121]; 255 = not finite
M4D_DEV unsigned block_exp(unsigned top) {
    const unsigned b = (top >> 23) + ((top & 0x7fffffu) > 0x7e0000u ? 1u : 0u);
    return top >= 0x7f800000u ? 255u : min(b > 7u ? b - 6u : 1u, 248u);
}
M4D_DEV float block_inv(unsigned b) { return __builtin_bit_cast(float, (254u - b) << 23); }      // 2^-e of a finite block: a normal number

// four values -> four codes in a dword.  x * 2^-e is exact, so adding 1.5 * 2^23 in the same fma rounds it to an integer, half to even, and
// leaves the code as the low byte.  cap: the block's exponent was capped at 121, values up to 128 steps saturate.
M4D_DEV unsigned encode4(float a, float b, float c, float d, float inv, bool cap) {
    const float magic = 12582912.f;
    float f[4] = {fmaf(a, inv, magic), fmaf(b, inv, magic), fmaf(c, inv, magic), fmaf(d, inv, magic)};
    if (cap) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = fminf(fmaxf(f[e], magic - 127.f), magic + 127.f);
    }
    const unsigned u0 = __builtin_bit_cast(unsigned, f[0]), u1 = __builtin_bit_cast(unsigned, f[1]);
    const unsigned u2 = __builtin_bit_cast(unsigned, f[2]), u3 = __builtin_bit_cast(unsigned, f[3]);
    const unsigned lo = __builtin_amdgcn_perm(u1, u0, 0x0c0c0400u), hi = __builtin_amdgcn_perm(u3, u2, 0x04000c0cu);      // bytes 0 of u0, u1 | u2, u3
    return lo | hi;
}

M4D_DEV float decode1(unsigned c, int e, float step) { return (float)((int)(c << (24 - 8 * e)) >> 24) * step; }
M4D_DEV void decode8(const u32x2& c, float step, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = decode1(c[e >> 2], e & 3, step);
}

}  // namespace

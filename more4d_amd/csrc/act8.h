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

// a lane's value and its neighbours' (lane ^ 1, lane ^ 2) within groups of four, largest
M4D_DEV unsigned max_xor1(unsigned v) { return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true)); }
M4D_DEV unsigned max_xor2(unsigned v) { return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true)); }

// bits of the largest magnitude of the values in n dwords (bf16: two in a dword, compared as 16-bit integers)
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <typename T, int N> M4D_DEV unsigned top_bits(const unsigned (&w)[N]) {
    if constexpr (sizeof(T) == 2) {
        u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
        for (int i = 1; i < N; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
        return (unsigned)max(m[0], m[1]) << 16;
    } else {
        unsigned m = w[0] & 0x7fffffffu;
#pragma unroll
        for (int i = 1; i < N; ++i) m = max(m, w[i] & 0x7fffffffu);
        return m;
    }
}
template <typename T, int N> M4D_DEV float value_of(const unsigned (&w)[N], int e) {
    return __builtin_bit_cast(float, sizeof(T) == 2 ? (e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16) : w[e]);
}
// values 4 q .. 4 q + 3 -> codes; b: the block's exponent byte (255: zeros)
template <typename T, int N> M4D_DEV unsigned encode_of(const unsigned (&w)[N], int q, unsigned b, float inv, bool cap) {
    const unsigned c = encode4(value_of<T>(w, 4 * q), value_of<T>(w, 4 * q + 1), value_of<T>(w, 4 * q + 2), value_of<T>(w, 4 * q + 3), inv, cap);
    return b == 255u ? 0u : c;
}

M4D_DEV float decode1(unsigned c, int e, float step) { return (float)((int)(c << (24 - 8 * e)) >> 24) * step; }
M4D_DEV void decode8(const u32x2& c, float step, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = decode1(c[e >> 2], e & 3, step);
}

}  // namespace

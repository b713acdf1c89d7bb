// Activations kept in 8 bits for the backward pass (m4d_act_quant8, m4d_act_dequant8, m4d_act_dequant8_t, m4d_act_bwd8).
//
// A row is cut into blocks of 32 consecutive channels.  A block stores ONE byte b = e + 127 and 32 codes round_half_even(x / 2^e), where
// e >= -126 is the smallest integer with max|x| <= 127 * 2^e; it stands for code * 2^e.  The step is a power of two, so both the division
// and the value read back are exact in float32 (and in bf16: a code has 7 bits), whoever computes them, and the 1-byte step lets the block be
// short: at 32 channels the rounding error of normal data (step / sqrt(12), step between 1 and 2 times max / 127) is the one that an exact
// float32 step reaches at 128 channels.  e is capped at 121 so that every code stands for a finite number (codes then saturate at 127);
// a block holding an infinity or NaN stores b = 255 and zero codes, which reads back as 0 * inf = NaN: a step that overflowed must not pass
// through the checkpoint as ordinary numbers.
//
// All four kernels are one pass over the data and bound by HBM; a "unit" is 8 channels of a row (16 bytes of bf16, 8 bytes of codes), four
// units are a block.  Rows of codes are padded to whole blocks, so the code side is always aligned; the other side takes 16-byte accesses
// where its rows are 16-byte aligned and element accesses otherwise.  21840 x 13824 bf16 (a copy of 2 GiB runs at 4.9 TB/s): act_quant8 183 us = 5.0
// TB/s, act_bwd8 302 us = 5.0, act_dequant8_t with GELU 245 us = 3.7 (its activation's instructions); 21840 x 5120 float32: act_quant8 112 us, act_dequant8 138.
#include "act8.h"
#include "more4d_hip.h"

namespace {

struct Act8Args {
    const void* in;       // quant: x;  bwd: dy
    void* out;            // dequant / bwd / transposed output
    int8_t* codes; uint8_t* exps;
    int64_t ld_in, ld_out, rows;
    int C, nb;            // channels, blocks per row (codes row stride = 32 * nb)
    int64_t rows_pad;     // transposed output: columns written (rows .. rows_pad are zero)
    int vec;              // 1: the T side has 16-byte aligned rows
};

// walks the units (row, j) of a [rows, nu] grid with a stride of gridDim.x * blockDim.x units: one division per thread, not per unit
struct UnitWalk {
    int64_t row; int j;
    int64_t q; int r, nu;
    M4D_DEV UnitWalk(int nu_) : nu(nu_) {
        const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, stride = (int64_t)gridDim.x * blockDim.x;
        row = first / nu; j = (int)(first - row * nu);
        q = stride / nu; r = (int)(stride - q * nu);
    }
    M4D_DEV void next() {
        row += q; j += r;
        if (j >= nu) { j -= nu; ++row; }
    }
};

template <typename T>
M4D_DEV void load_unit(const T* src, int n, bool vec, float (&v)[8]) {      // n <= 8 valid channels, the others read as 0
    if (vec && n == 8) {
        const f32x4 a = load4(src), b = load4(src + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? (float)src[e] : 0.f;
    }
}
template <>
M4D_DEV void load_unit<bf16_t>(const bf16_t* src, int n, bool vec, float (&v)[8]) {
    if (vec && n == 8) {
        const bf16x8 a = *reinterpret_cast<const bf16x8*>(src);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? (float)src[e] : 0.f;
    }
}
template <typename T>
M4D_DEV void store_unit(T* dst, int n, bool vec, const float (&v)[8]) {
    if (vec && n == 8) {
        if constexpr (sizeof(T) == 2) {
            bf16x8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (bf16_t)v[e];
            *reinterpret_cast<bf16x8*>(dst) = o;
        } else {
            store4((float*)dst, f32x4{v[0], v[1], v[2], v[3]});
            store4((float*)dst + 4, f32x4{v[4], v[5], v[6], v[7]});
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) dst[e] = (T)v[e];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void act_quant8_kernel(Act8Args p) {
    const int nu = p.nb * 4;
    for (UnitWalk w(nu); w.row < p.rows; w.next()) {
        const int c0 = w.j * 8, n = min(8, p.C - c0);
        constexpr int ND = 2 * sizeof(T);             // dwords of a unit
        unsigned v[ND];
        const T* src = (const T*)p.in + w.row * p.ld_in + c0;
        if (p.vec && n == 8) {
#pragma unroll
            for (int i = 0; i < ND / 4; ++i) {
                const u32x4q d = reinterpret_cast<const u32x4q*>(src)[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i * 4 + e] = d[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                if constexpr (sizeof(T) == 2) {
                    bf16x2 b = {(bf16_t)0.f, (bf16_t)0.f};
                    if (2 * i < n) b[0] = src[2 * i];
                    if (2 * i + 1 < n) b[1] = src[2 * i + 1];
                    v[i] = __builtin_bit_cast(unsigned, b);
                } else v[i] = i < n ? __builtin_bit_cast(unsigned, src[i]) : 0u;
            }
        }
        const unsigned b = block_exp(max_xor2(max_xor1(top_bits<T>(v))));      // the block's four units are four neighbouring lanes
        const float inv = block_inv(min(b, 248u));
        const u32x2 c = {encode_of<T>(v, 0, b, inv, b == 248u), encode_of<T>(v, 1, b, inv, b == 248u)};
        *reinterpret_cast<u32x2*>(p.codes + (w.row * p.nb) * 32 + c0) = c;
        if ((w.j & 3) == 0) p.exps[w.row * p.nb + (w.j >> 2)] = (uint8_t)b;
    }
}

// gelu_tanh as x s(2u) with 2u log2 e = x (c0 + c1 x^2) in one multiply-add: the transposed reader evaluates it at the rate of HBM, and common.h's
// form, which rounds like the forward's, has three instructions more.  (x^2 may overflow: the exponential is then 0 or inf, the result x or -0.)
M4D_DEV float gelu_f(float x) {
    const float c0 = -2.3022081981f, c1 = -0.1029432396f;      // -2 log2(e) sqrt(2 / pi), times 0.044715
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * fmaf(c1, x * x, c0)));
}
template <int ACT> M4D_DEV float act_f(float x) {
    return ACT == 1 ? silu_f(x) : ACT == 2 ? gelu_f(x) : ACT == 3 ? gelu_erf_f(x) : x;
}

// act'(x).  Beyond |x| = 128 the three derivatives are 0 or 1 in float32, and clamping there keeps the polynomials finite; x * 0 brings
// back the NaN that the clamp would lose.
template <int ACT> M4D_DEV float dact_f(float x0) {
    const float x = fminf(fmaxf(x0, -128.f), 128.f);
    float d;
    if constexpr (ACT == 2) {      // gelu_tanh = x s(2u), s the logistic function, u = k0 (x + k1 x^3):  s + x s (1 - s) 2 u'
        const float k0 = 0.7978845608028654f, k1 = 0.044715f, x2 = x * x;
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(k0 * x * (1.0f + k1 * x2) * -2.8853900817779268f));
        d = s + x * s * (1.0f - s) * (2.0f * k0) * (1.0f + 3.0f * k1 * x2);
    } else if constexpr (ACT == 1) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-x));
        d = s * (1.0f + x * (1.0f - s));
    } else {
        d = 0.5f * (1.0f + erff(x * 0.7071067811865476f)) + x * __expf(-0.5f * x * x) * 0.3989422804014327f;
    }
    return fmaf(x0, 0.f, d);
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_dequant8_kernel(Act8Args p) {
    const int nu = (p.C + 7) >> 3;
    for (UnitWalk w(nu); w.row < p.rows; w.next()) {
        const int c0 = w.j * 8, n = min(8, p.C - c0);
        const u32x2 c = *reinterpret_cast<const u32x2*>(p.codes + (w.row * p.nb) * 32 + c0);
        float v[8];
        decode8(c, step_of(p.exps[w.row * p.nb + (w.j >> 2)]), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = act_f<ACT>(v[e]);
        store_unit<T>((T*)p.out + w.row * p.ld_out + c0, n, p.vec, v);
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_bwd8_kernel(Act8Args p) {
    const int nu = (p.C + 7) >> 3;
    for (UnitWalk w(nu); w.row < p.rows; w.next()) {
        const int c0 = w.j * 8, n = min(8, p.C - c0);
        const u32x2 c = *reinterpret_cast<const u32x2*>(p.codes + (w.row * p.nb) * 32 + c0);
        float d[8], v[8];
        load_unit<T>((const T*)p.in + w.row * p.ld_in + c0, n, p.vec, d);
        decode8(c, step_of(p.exps[w.row * p.nb + (w.j >> 2)]), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = d[e] * dact_f<ACT>(v[e]);
        store_unit<T>((T*)p.out + w.row * p.ld_out + c0, n, p.vec, v);
    }
}

// out[c, r] = act(value[r, c]), columns rows .. rows_pad zero: the weight gradient's operand (the token axis becomes the K of the GEMM).
// Tile: 128 channels x 64 dwords of rows (bf16: two rows in a dword, fp32: one), in LDS as [channel][dword] with the 16-byte chunks of a
// channel XORed by channel / 8: the 16 x 4 (unit, dword) pairs that a wave writes per channel land in 64 different banks, and a lane reads its
// 8 (4) rows of a channel as one 16-byte chunk.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_dequant8_t_kernel(Act8Args p) {
    constexpr int RPD = 4 / sizeof(T);          // rows per dword
    constexpr int TR = 64 * RPD;                // rows of a tile
    __shared__ __attribute__((aligned(16))) unsigned tile[128 * 64];
    const int t = threadIdx.x;
    const int64_t r0 = (int64_t)blockIdx.x * TR;
    const int c0 = blockIdx.y * 128;
    const int cg = t & 15;                      // unit (8 channels) of the tile
    const int col = c0 + cg * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = i * 16 + (t >> 4);        // dword of the tile's rows
        float v[RPD][8];
#pragma unroll
        for (int h = 0; h < RPD; ++h) {
            const int64_t r = r0 + d * RPD + h;
            if (r < p.rows && col < p.C) {
                const u32x2 c = *reinterpret_cast<const u32x2*>(p.codes + (r * p.nb) * 32 + col);
                decode8(c, step_of(p.exps[r * p.nb + (col >> 5)]), v[h]);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[h][e] = act_f<ACT>(v[h][e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[h][e] = 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            unsigned w;
            if constexpr (RPD == 2) {
                bf16x2 b;
                b[0] = (bf16_t)v[0][e]; b[1] = (bf16_t)v[RPD - 1][e];
                w = __builtin_bit_cast(unsigned, b);
            } else w = __builtin_bit_cast(unsigned, v[0][e]);
            tile[(cg * 8 + e) * 64 + (((d >> 2) ^ cg) << 2) + (d & 3)] = w;
        }
    }
    __syncthreads();
    const int ch = t & 15;                      // chunk: rows ch * 4 * RPD ..
    const int64_t r = r0 + ch * 4 * RPD;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int cl = i * 16 + (t >> 4);
        if (c0 + cl >= p.C || r >= p.rows_pad) continue;
        const uint4 w = *reinterpret_cast<const uint4*>(&tile[cl * 64 + ((ch ^ (cl >> 3)) << 2)]);
        *reinterpret_cast<uint4*>((T*)p.out + (int64_t)(c0 + cl) * p.ld_out + r) = w;      // (rows_pad and ld_out: whole chunks)
    }
}

unsigned grid_of(int64_t units) {
    const int64_t n = (units + 255) / 256;
    return (unsigned)(n < 256 * 32 ? n : 256 * 32);
}

}  // namespace

// the activation as a template parameter: a runtime switch per element was a fifth of the transposed reader's time
#define ACT8_ONE(KERNEL, ACT)                                                                                           \
    do {                                                                                                                \
        if (dt == M4D_BF16) hipLaunchKernelGGL((KERNEL<bf16_t, ACT>), grid, block, 0, (hipStream_t)stream, p);           \
        else hipLaunchKernelGGL((KERNEL<float, ACT>), grid, block, 0, (hipStream_t)stream, p);                          \
    } while (0)
#define ACT8_BY_ACT(KERNEL)                                                                                             \
    do {                                                                                                                \
        if (act == 1) ACT8_ONE(KERNEL, 1);                                                                              \
        else if (act == 2) ACT8_ONE(KERNEL, 2);                                                                         \
        else ACT8_ONE(KERNEL, 3);                                                                                       \
    } while (0)
#define DT_OK(dt) ((dt) == M4D_BF16 || (dt) == M4D_F32)
#define ACT8_COMMON(name)                                                                                              \
    M4D_CHECK_ARG(DT_OK(dt), name ": bad dtype %d", (int)dt);                                                           \
    M4D_CHECK_ARG(codes && exps && rows > 0 && C > 0, name ": null pointer or empty (rows=%lld C=%d)", (long long)rows, C); \
    M4D_CHECK_ARG(C <= (1 << 24) && rows < (1ll << 38), name ": too large");                                            \
    M4D_CHECK_ARG(((uintptr_t)codes % 16) == 0, name ": codes must be 16-byte aligned");                                \
    const int nb = (C + 31) / 32, es = dt == M4D_BF16 ? 2 : 4;                                                          \
    (void)es

extern "C" int m4d_act_quant8(m4d_dtype dt, const void* x, int64_t ldx, int8_t* codes, uint8_t* exps, int64_t rows, int C,
                              m4d_stream stream) {
    ACT8_COMMON("act_quant8");
    M4D_CHECK_ARG(x && (rows == 1 || ldx >= C), "act_quant8: null input or row stride %lld below C=%d", (long long)ldx, C);
    Act8Args p{};
    p.in = x; p.ld_in = ldx; p.codes = codes; p.exps = exps; p.rows = rows; p.C = C; p.nb = nb;
    p.vec = ((uintptr_t)x % 16) == 0 && (ldx * es) % 16 == 0;
    dim3 grid(grid_of(rows * nb * 4)), block(256);
    if (dt == M4D_BF16) hipLaunchKernelGGL(act_quant8_kernel<bf16_t>, grid, block, 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(act_quant8_kernel<float>, grid, block, 0, (hipStream_t)stream, p);
    M4D_CHECK_LAUNCH("act_quant8");
    return 0;
}

extern "C" int m4d_act_dequant8(m4d_dtype dt, const int8_t* codes, const uint8_t* exps, void* out, int64_t ldo, int64_t rows, int C, int act,
                                m4d_stream stream) {
    ACT8_COMMON("act_dequant8");
    M4D_CHECK_ARG(act >= 0 && act <= 3, "act_dequant8: bad activation %d", act);
    M4D_CHECK_ARG(out && (rows == 1 || ldo >= C), "act_dequant8: null output or row stride %lld below C=%d", (long long)ldo, C);
    Act8Args p{};
    p.out = out; p.ld_out = ldo; p.codes = (int8_t*)codes; p.exps = (uint8_t*)exps; p.rows = rows; p.C = C; p.nb = nb;
    p.vec = ((uintptr_t)out % 16) == 0 && (ldo * es) % 16 == 0;
    dim3 grid(grid_of(rows * ((C + 7) / 8))), block(256);
    if (act == 0) ACT8_ONE(act_dequant8_kernel, 0);
    else ACT8_BY_ACT(act_dequant8_kernel);
    M4D_CHECK_LAUNCH("act_dequant8");
    return 0;
}

extern "C" int m4d_act_dequant8_t(m4d_dtype dt, const int8_t* codes, const uint8_t* exps, void* out, int64_t ldo, int64_t rows, int64_t rows_pad,
                                  int C, int act, m4d_stream stream) {
    ACT8_COMMON("act_dequant8_t");
    M4D_CHECK_ARG(act >= 0 && act <= 3, "act_dequant8_t: bad activation %d", act);
    M4D_CHECK_ARG(out && rows_pad >= rows && ldo >= rows_pad, "act_dequant8_t: null output, rows_pad < rows or row stride below rows_pad");
    M4D_CHECK_ARG(((uintptr_t)out % 16) == 0 && (rows_pad * es) % 16 == 0 && (ldo * es) % 16 == 0,
                  "act_dequant8_t: output rows and rows_pad must be multiples of 16 bytes");
    const int tr = dt == M4D_BF16 ? 128 : 64;
    const int64_t gx = (rows_pad + tr - 1) / tr;
    const int gy = (C + 127) / 128;
    M4D_CHECK_ARG(gx < (1ll << 31) && gy <= 65535, "act_dequant8_t: too large");
    Act8Args p{};
    p.out = out; p.ld_out = ldo; p.codes = (int8_t*)codes; p.exps = (uint8_t*)exps; p.rows = rows; p.C = C; p.nb = nb;
    p.rows_pad = rows_pad;
    dim3 grid((unsigned)gx, (unsigned)gy), block(256);
    if (act == 0) ACT8_ONE(act_dequant8_t_kernel, 0);
    else ACT8_BY_ACT(act_dequant8_t_kernel);
    M4D_CHECK_LAUNCH("act_dequant8_t");
    return 0;
}

extern "C" int m4d_act_bwd8(m4d_dtype dt, const void* dy, int64_t ldy, const int8_t* codes, const uint8_t* exps, void* out, int64_t ldo, int64_t rows,
                            int C, int act, m4d_stream stream) {
    ACT8_COMMON("act_bwd8");
    M4D_CHECK_ARG(act >= 1 && act <= 3, "act_bwd8: bad activation %d", act);
    M4D_CHECK_ARG(dy && out && (rows == 1 || (ldy >= C && ldo >= C)), "act_bwd8: null pointer or row stride below C=%d", C);
    Act8Args p{};
    p.in = dy; p.ld_in = ldy; p.out = out; p.ld_out = ldo; p.codes = (int8_t*)codes; p.exps = (uint8_t*)exps;
    p.rows = rows; p.C = C; p.nb = nb;
    p.vec = ((uintptr_t)dy % 16) == 0 && ((uintptr_t)out % 16) == 0 && (ldy * es) % 16 == 0 && (ldo * es) % 16 == 0;
    dim3 grid(grid_of(rows * ((C + 7) / 8))), block(256);
    ACT8_BY_ACT(act_bwd8_kernel);
    M4D_CHECK_LAUNCH("act_bwd8");
    return 0;
}

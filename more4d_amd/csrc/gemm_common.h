// Shared pieces of the GEMM kernels (gemm.hip, gemm_packed.hip): argument block, LDS swizzle, XCD-aware tile order,
// fused epilogue.  See gemm.hip for the design notes.
#pragma once
#include <type_traits>

#include "common.h"
#include "more4d_hip.h"

#define GLOBAL_AS __attribute__((address_space(1)))
#define LDS_AS __attribute__((address_space(3)))

namespace {

struct GemmArgs {
    const void* A; const void* W; const void* bias; void* out;
    const float* gate;
    int64_t lda, ldw, ldc, M, N, K, gate_stride, rows_per_sample;
    int epilogue, bias_on_m;
    int tiles_m, tiles_n;
    int64_t a_bs1, a_bs2, w_bs1, w_bs2;   // batched launches (gridDim.y = nb1 * nb2): element offsets of batch (i1, i2); out += batch * M * ldc
    int nb1;                               // 0 = not batched
    // stacked taps (m4d_gemm_bt_taps, the conv weight gradient on the wide kernel): the M rows are tap_rows-row groups t = dt * tap_kh + dh
    // of the SAME tap_rows rows of A, read tap_s1 * dt + tap_s2 * dh elements further along K (0 = off)
    int tap_rows, tap_kh;
    int64_t tap_s1, tap_s2;
    // split-K tail (m4d_gemm_bt_ws): the launch over the full tile rounds uses `remap_n` (< tiles_m*tiles_n) logical tiles; the tail
    // launch has ksplit > 0: block b computes K-slice b % ksplit of logical tile tile_base + b / ksplit into its float32 slab of `ws`
    int remap_n, tile_base, ksplit;
    int tile_off;   // chunked launches (M4D_GEMM_CHUNK): this launch covers logical tiles [tile_off, tile_off + remap_n)
    float* ws;
    int abl;   // timing ablations (tools only; results wrong when != 0): 1 no DMA, 2 frags once, 4 no barriers, 8 no MFMA
    unsigned* sync;   // persistent wide kernel: 8 arrival counters (one per XCD, 128 bytes apart, zeroed before the launch) or nullptr
};

// Shared projection with low-rank adapters (adapters.hip): behind the K loop a tile adds, for every adapter that one of its rows names,
// the product of that adapter's rows of u (= s x A^T, other rows read as zero) with its B.
struct GemmAdArgs : GemmArgs {
    const void* u;              // T [M, u_stride(R)] (u_hi)
    const void* up;             // T [G, N, R]
    const int* row_adapter;     // [M], -1 = none
    const int* tile_off;        // [tiles_m + 1] into tile_list
    const int* tile_list;       // adapters of the rows of each tile, each once
    const int* tile_one;        // [tiles_m] the adapter that ALL rows of the tile name, or -1 (wide kernel only)
    int R;                      // multiple of 16
};

// A row of u holds float32 ranks in one piece, bf16 as hi + lo of 16 bits (split2) in blocks of 32 ranks, the last may have 16: [hi | lo] of each.  One
// rounding to bf16 here would put an error of up to 2^-8 of the adapter's part on an output that is itself rounded once; 32 ranks of both parts
// are one 64-element K-tile of the 256 x 256 kernel.
template <typename T> struct Parts { static constexpr int N = sizeof(T) == 2 ? 2 : 1; };
template <typename T> M4D_DEV int u_stride(int R) { return R * Parts<T>::N; }
template <typename T> M4D_DEV int u_hi(int r) { return Parts<T>::N == 2 ? 2 * (r & ~31) + (r & 31) : r; }      // lo: min(32, R - (r & ~31)) further

constexpr int ROWB = 128;  // bytes of K per LDS row

M4D_DEV int lds_off(int row, int chunk) { return row * ROWB + ((chunk ^ ((row >> 1) & 7)) << 4); }

// XCD-aware, banded tile order -> (tm, tn)
M4D_DEV void tile_coords(const GemmArgs& p, int& tm, int& tn, int bid) {
    if (p.ksplit > 0) bid = p.tile_base + bid / p.ksplit;      // tail launch: logical tile id, no XCD remap
    else {
        const int nwg = p.remap_n > 0 ? p.remap_n : p.tiles_m * p.tiles_n;
        const int q = nwg >> 3, r = nwg & 7, xcd = bid & 7, idx = bid >> 3;
        bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx + p.tile_off;
    }
    constexpr int GM = 8;
    const int band = bid / (GM * p.tiles_n);
    const int band_rows = min(GM, p.tiles_m - band * GM);
    const int in_band = bid - band * GM * p.tiles_n;
    tm = band * GM + in_band % band_rows;
    tn = in_band / band_rows;
    if (M4D_ABL(p) & 16) { tm = 0; tn = 0; }          // ablation: every workgroup reads the same panels (all L2 hits)
    if (M4D_ABL(p) & 32) { tm = blockIdx.x % p.tiles_m; tn = blockIdx.x / p.tiles_m; }   // ablation: naive order
}
M4D_DEV void tile_coords(const GemmArgs& p, int& tm, int& tn) { tile_coords(p, tm, tn, (int)blockIdx.x); }

// Epilogue for one 32(n) x 32(m) accumulator tile: this lane holds column m, rows nb0 + 8*rq + 4*hi + [0,4).
// bf16 outputs are widened to 16-byte stores: a v_permlane32_swap per dword exchanges the 4-column groups of the two
// half-waves so lanes 0-31 own columns 16j..16j+7 and lanes 32-63 columns 16j+8..16j+15 of their row (cdna guide T21:
// the store tail is issue-bound, half the instructions = half the tail).
template <typename T>
M4D_DEV void epilogue_tile(const GemmArgs& p, const f32x16& acc, int64_t m, int64_t nb0, int hi, float bias_m,
                           const float* grow, int64_t n_lo = 0) {   // columns below n_lo belong to the neighbouring tile
    const T* bias = (const T*)p.bias;
    f32x4 v[4];
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
        const int64_t nb = nb0 + rq * 8 + hi * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[rq][e] = acc[rq * 4 + e];
        if (bias) {
            if (p.bias_on_m) { v[rq] += bias_m; }
            else if (nb < p.N) { v[rq] += load4(bias + nb); }
        }
        switch (p.epilogue) {
            case M4D_EPI_GELU_TANH:
#pragma unroll
                for (int e = 0; e < 4; ++e) v[rq][e] = gelu_tanh_f(v[rq][e]);
                break;
            case M4D_EPI_GELU_ERF:
#pragma unroll
                for (int e = 0; e < 4; ++e) v[rq][e] = gelu_erf_f(v[rq][e]);
                break;
            case M4D_EPI_SILU:
#pragma unroll
                for (int e = 0; e < 4; ++e) v[rq][e] = silu_f(v[rq][e]);
                break;
            default: break;
        }
    }
    if (p.epilogue == M4D_EPI_RESID_GATE) {
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
            const int64_t nb = nb0 + rq * 8 + hi * 4;
            if (nb >= p.N || nb < n_lo) continue;
            float* r = (float*)p.out + m * p.ldc + nb;
            f32x4 x = load4(r);
            f32x4 g = {1.f, 1.f, 1.f, 1.f};
            if (grow) g = load4(grow + nb);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += round_through<T>(v[rq][e]) * g[e];
            store4(r, x);
        }
    } else if (p.epilogue == M4D_EPI_STORE_F32) {
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
            const int64_t nb = nb0 + rq * 8 + hi * 4;
            if (nb >= p.N) continue;
            if (!p.nb1) {      // (batched split-K partial sums keep their float32 accumulators)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[rq][e] = round_through<T>(v[rq][e]);
            }
            store4((float*)p.out + m * p.ldc + nb, v[rq]);
        }
    } else {
        if constexpr (sizeof(T) == 2) {
            if ((p.N & 7) == 0 && (p.ldc & 7) == 0) {     // both half-waves of a row take the same branch: N % 8 == 0
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    union { bf16x4 h; unsigned u[2]; } a, b;
#pragma unroll
                    for (int e = 0; e < 4; ++e) { a.h[e] = (bf16_t)v[2 * j][e]; b.h[e] = (bf16_t)v[2 * j + 1][e]; }
                    const auto r0 = __builtin_amdgcn_permlane32_swap(a.u[0], b.u[0], false, false);
                    const auto r1 = __builtin_amdgcn_permlane32_swap(a.u[1], b.u[1], false, false);
                    const int64_t nb = nb0 + j * 16 + hi * 8;
                    if (nb < p.N)
                        *reinterpret_cast<uint4*>((T*)p.out + m * p.ldc + nb) = make_uint4(r0[0], r1[0], r0[1], r1[1]);
                }
                return;
            }
        }
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
            const int64_t nb = nb0 + rq * 8 + hi * 4;
            if (nb >= p.N) continue;
            store4((T*)p.out + m * p.ldc + nb, v[rq]);
        }
    }
}

// The adapters' part of a wave's NI x MI accumulator blocks (32 x 32 each; rows m_base + 32 mi + lane, columns n_base + 32 ni + lane of W):
// acc += up_g[n, :] . u[m, :] over the rank, for every step-th adapter of the tile from `first` on.  The operands come straight from L2 in the
// MFMA layout (16 bytes per lane and 16 ranks; a block's 32 rows of R ranks are contiguous memory): through LDS they would need two more
// barriers.  All loads of 64 ranks (32 with 256 accumulators) are issued before their first product, so a tile pays one L2
// latency for them and adapter, not four (two).
// Rows of u that name another adapter (or none: their u was never written) are replaced by zero before the product, not multiplied by zero; and
// where a wave's rows do not all name the adapter, an infinity or NaN in its B must not meet those zeros, nor be left out where a row's own u is
// zero or infinite.  float32 then forms the products apart and adds them in the adapter's rows only; bf16 adds what is not finite by add_bad (a VALU
// instruction on its accumulators takes them out of the AGPRs: 200 spilled registers in the 256 x 256 kernel).
// AdTile: what the extension has to know about its tile, loaded in front of the K loop (behind it these would be three dependent trips to L2).
// order (or nullptr): the row behind each row of the tiles.
template <int MI> struct AdTile { int i0, i1, g0; int ra[MI], row[MI]; };
template <int MI>
M4D_DEV AdTile<MI> adapters_tile(const GemmAdArgs& p, int tile, int64_t m_base, int lane, int first = 0, const int* order = nullptr) {
    AdTile<MI> a;
    a.i0 = __builtin_amdgcn_readfirstlane(p.tile_off[tile]) + first;
    a.i1 = __builtin_amdgcn_readfirstlane(p.tile_off[tile + 1]);
    a.g0 = a.i0 < a.i1 ? __builtin_amdgcn_readfirstlane(p.tile_list[a.i0]) : 0;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const int64_t m = m_base + mi * 32 + (lane & 31);
        a.row[mi] = m >= p.M ? 0 : order ? order[m] : (int)m;
        a.ra[mi] = m < p.M ? p.row_adapter[a.row[mi]] : -1;
    }
    return a;
}
// bits of a fragment's largest magnitude as a float32 (integers order like magnitudes, NaN on top)
M4D_DEV unsigned frag_top(const bf16x8& f) {
    typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const u16x8 v = __builtin_bit_cast(u16x8, f) & (unsigned short)0x7fff;
    const u16x2 a = __builtin_elementwise_max(u16x2{v[0], v[1]}, u16x2{v[2], v[3]}), b = __builtin_elementwise_max(u16x2{v[4], v[5]}, u16x2{v[6], v[7]});
    const u16x2 m = __builtin_elementwise_max(a, b);
    return (unsigned)max(m[0], m[1]) << 16;
}
M4D_DEV unsigned frag_top(const f32x8& f) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __builtin_bit_cast(unsigned, f[e]) & 0x7fffffffu);
    return m;
}
// bf16, 16 ranks of a block: what an infinity or NaN in B adds to the columns of acc that are its adapter's, as products of +-3.3e38 with +-3.3e38
// (they overflow to the infinity that is wanted; zeros everywhere else), those of one sign together.  u: the part that has its sign.
//   b = +-inf, u not 0: sign(b) sign(u) inf;   b = +-inf, u = 0, or b = NaN: inf, then -inf;   (u = NaN: the product itself)
template <int MI>
M4D_DEV void add_bad(const bf16x8& b, const bf16x8 (&u)[MI], const bool (&own)[MI], f32x16 (&acc)[MI]) {
    const bf16_t big = (bf16_t)3.3e38f, none = (bf16_t)0.f;
    auto pick = [&](const bf16x8& f, bf16_t v, auto which) {
        bf16x8 r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = which((float)f[e]) ? v : none;
        return r;
    };
    const float inf = __builtin_inff();
    const bf16x8 bp = pick(b, big, [&](float v) { return v == inf; }), bm = pick(b, -big, [&](float v) { return v == -inf; });
    const bf16x8 bi = pick(b, big, [&](float v) { return fabsf(v) == inf; }), bn = pick(b, big, [&](float v) { return v != v; });
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const bool o = own[mi];
        const bf16x8 up = pick(u[mi], big, [&](float v) { return o && v > 0.f; }), um = pick(u[mi], -big, [&](float v) { return o && v < 0.f; });
        mma32(bp, up, acc[mi]);
        mma32(bm, um, acc[mi]);
        mma32(bp, um, acc[mi]);
        mma32(bm, up, acc[mi]);
#pragma unroll
        for (int sign = 0; sign < 2; ++sign) {
            mma32(bi, pick(u[mi], sign ? -big : big, [&](float v) { return o && v == 0.f; }), acc[mi]);
            mma32(bn, pick(u[mi], sign ? -big : big, [&](float) { return o; }), acc[mi]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}
// B's fragment for the product itself: 1 with its sign in the place of an infinity (an infinite u is to meet no zero there), 1 of a NaN
M4D_DEV bf16x8 without_bad(const bf16x8& b) {
    bf16x8 r = b;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = (float)b[e];
        if (!(fabsf(v) < __builtin_inff())) r[e] = (bf16_t)(v < 0.f ? -1.f : 1.f);
    }
    return r;
}
template <typename T, int NI, int MI>
M4D_DEV void adapters_extend(const GemmAdArgs& p, f32x16 (&acc)[NI][MI], const AdTile<MI>& a, int64_t n_base, int lane, int step = 1,
                             int k0 = 0) {      // k0: ranks in front of it are already in
    typedef typename Frag8<T>::type frag_t;
    constexpr int U = sizeof(T) != 2 ? 1 : NI * MI < 16 ? 4 : 2;      // 16-rank steps in flight, as registers allow (float32 is MFMA-bound)
    const int li = lane & 31, hi = lane >> 5;
    if (a.i0 >= a.i1 || k0 >= p.R) return;
    const T* pu[MI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) pu[mi] = (const T*)p.u + (int64_t)a.row[mi] * u_stride<T>(p.R) + hi * 8;
    int64_t nr[NI];                                   // (columns beyond N are computed from row N - 1 and not stored)
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) nr[ni] = min(n_base + ni * 32 + li, p.N - 1) * p.R + hi * 8;
    for (int i = a.i0; i < a.i1; i += step) {
        const int g = i == a.i0 ? a.g0 : __builtin_amdgcn_readfirstlane(p.tile_list[i]);
        bool mine = false, all = true;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) { mine |= a.ra[mi] == g; all &= a.ra[mi] == g; }
        if (!__any(mine)) continue;                   // none of this wave's rows
        const bool mixed = !__all(all);
        const T* b = (const T*)p.up + (int64_t)g * p.N * p.R;
        // C steps of 16 ranks: all loads (without predicates: rows of other adapters are replaced after the load), then the products.  u's parts as they
        // lie in a block of 32 ranks, in the order in which the 256 x 256 kernel's K loop takes them: a row that two of its tiles write (the last one
        // is shifted inwards) has to get the same bits from both.
        auto chunk = [&](auto C_T, int k) {
            constexpr int C = decltype(C_T)::value, NP = Parts<T>::N, W = C == 1 ? 16 : 32;      // (bf16: C = 1 is the last block of 16)
            frag_t fu[C][NP][MI], fb[C][NI];
            auto load_u = [&](int s, int q, int mi) { return *reinterpret_cast<const frag_t*>(pu[mi] + (NP == 2 ? 2 * k + (s >> 1) * 64 + (s & 1) * 16 + q * W : k + s * 16)); };
            auto load_b = [&](int s, int ni) { return *reinterpret_cast<const frag_t*>(b + nr[ni] + k + s * 16); };
#pragma unroll
            for (int s = 0; s < C; ++s) {
#pragma unroll
                for (int q = 0; q < NP; ++q)
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi) fu[s][q][mi] = load_u(s, q, mi);
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) fb[s][ni] = load_b(s, ni);
            }
            if (mixed) {
                unsigned top = 0;
#pragma unroll
                for (int s = 0; s < C; ++s) {
#pragma unroll
                    for (int q = 0; q < NP; ++q)
#pragma unroll
                        for (int mi = 0; mi < MI; ++mi)
                            if (a.ra[mi] != g) fu[s][q][mi] = frag_t{};
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) top = max(top, frag_top(fb[s][ni]));
                }
                if (__any(top >= 0x7f800000u)) {
                    if constexpr (sizeof(T) == 2) {
                        bool own[MI];
#pragma unroll
                        for (int mi = 0; mi < MI; ++mi) own[mi] = a.ra[mi] == g;
#pragma unroll 1
                        for (int s = 0; s < C; ++s) {      // (rolled up and from memory again: it must not add to the registers of the rest)
                            frag_t us[MI];
#pragma unroll
                            for (int mi = 0; mi < MI; ++mi) us[mi] = load_u(s, 0, mi);
#pragma unroll
                            for (int ni = 0; ni < NI; ++ni) add_bad<MI>(load_b(s, ni), us, own, acc[ni]);
                        }
#pragma unroll
                        for (int s = 0; s < C; ++s) {
#pragma unroll
                            for (int q = 0; q < NP; ++q)
#pragma unroll
                                for (int mi = 0; mi < MI; ++mi) fu[s][q][mi] = own[mi] ? load_u(s, q, mi) : frag_t{};
#pragma unroll
                            for (int ni = 0; ni < NI; ++ni) fb[s][ni] = without_bad(load_b(s, ni));
                        }
                    } else {
#pragma unroll
                        for (int ni = 0; ni < NI; ++ni) {
#pragma unroll
                            for (int mi = 0; mi < MI; ++mi) {
                                f32x16 sum;
#pragma unroll
                                for (int q = 0; q < 16; ++q) sum[q] = 0.f;
                                mma32(fb[0][ni], fu[0][0][mi], sum);
#pragma unroll
                                for (int q = 0; q < 16; ++q) acc[ni][mi][q] += a.ra[mi] == g ? sum[q] : 0.f;
                                __builtin_amdgcn_sched_barrier(0);
                            }
                            fb[0][ni] = frag_t{};
                        }
#pragma unroll
                        for (int mi = 0; mi < MI; ++mi) fu[0][0][mi] = frag_t{};
                    }
                }
            }
#pragma unroll
            for (int s2 = 0; s2 < C; s2 += 2)
#pragma unroll
                for (int q = 0; q < NP; ++q)
#pragma unroll
                    for (int s = s2; s < s2 + 2 && s < C; ++s)
#pragma unroll
                        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
                            for (int mi = 0; mi < MI; ++mi) mma32(fb[s][ni], fu[s][q][mi], acc[ni][mi]);
        };
        int k = k0;
        for (; k + 16 * U <= p.R; k += 16 * U) chunk(std::integral_constant<int, U>{}, k);
        if constexpr (U == 4)
            if (k + 32 <= p.R) { chunk(std::integral_constant<int, 2>{}, k); k += 32; }
        if constexpr (U > 1)
            if (k < p.R) chunk(std::integral_constant<int, 1>{}, k);
    }
}

// wave-uniform 64-bit value forced into SGPRs (keeps the DMA in its  vgpr_offset + sgpr_base  addressing form)
M4D_DEV const char* uniform_ptr(const char* q) {
    const unsigned long long v = (unsigned long long)q;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
    return (const char*)(((unsigned long long)hi << 32) | lo);
}

// Epilogue of one 64(m) x 64(n) half of a wave's sub-tile THROUGH LDS.  The accumulator layout gives every lane its own
// output ROW (lane = m), so direct stores touch 64 different rows per instruction (16-byte pieces of 64 cache lines:
// measured 1.4 TB/s, 16 % of a K = 5120 GEMM).  Here the half-tile is written to a wave-private LDS region with bias /
// activation / gate applied, then read back row-wise so that 8 (bf16) or 16 (fp32) consecutive lanes cover one
// contiguous 128 / 256-byte row segment of the output.  16-byte chunks are XOR-swizzled by the row index.
template <typename T>
M4D_DEV void epilogue_half_lds(const GemmArgs& p, char* wl, const f32x16& a00, const f32x16& a01, const f32x16& a10,
                               const f32x16& a11, int64_t m_base, int64_t n_base, int64_t m_lo, int64_t n_lo, int lane) {
    // a[ni][mi2]: a00 = (ni 0, mi2 0), a01 = (ni 0, mi2 1), a10 = (ni 1, mi2 0), a11 = (ni 1, mi2 1)
    const int li = lane & 31, hi = lane >> 5;
    const T* bias = (const T*)p.bias;
    const bool f32out = p.epilogue == M4D_EPI_RESID_GATE || p.epilogue == M4D_EPI_STORE_F32;
#pragma unroll
    for (int mi2 = 0; mi2 < 2; ++mi2) {
        const int r = mi2 * 32 + li;
        const int64_t m = m_base + r;
        const float bm = (bias && p.bias_on_m) ? (float)bias[m] : 0.f;
        const float* grow = (p.epilogue == M4D_EPI_RESID_GATE && p.gate) ? p.gate + (m / p.rows_per_sample) * p.gate_stride : nullptr;
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
            const f32x16& acc = ni == 0 ? (mi2 == 0 ? a00 : a01) : (mi2 == 0 ? a10 : a11);
#pragma unroll
            for (int rq = 0; rq < 4; ++rq) {
                const int nl = ni * 32 + rq * 8 + hi * 4;
                const int64_t nb = n_base + nl;
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[rq * 4 + e];
                if (bias) { if (p.bias_on_m) v += bm; else v += load4(bias + nb); }
                if (p.epilogue == M4D_EPI_GELU_TANH) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = gelu_tanh_f(v[e]);
                } else if (p.epilogue == M4D_EPI_GELU_ERF) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = gelu_erf_f(v[e]);
                } else if (p.epilogue == M4D_EPI_SILU) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = silu_f(v[e]);
                }
                if (f32out) {
                    if (!p.nb1) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = round_through<T>(v[e]);
                    }
                    if (grow) v = v * load4(grow + nb);
                    const int ch = nl >> 2;                                   // 16 chunks of 4 floats per 256-byte row
                    *reinterpret_cast<f32x4*>(wl + r * 256 + ((ch ^ (r & 15)) << 4)) = v;
                } else {
                    const int ch = nl >> 3;                                   // 8 chunks of 8 bf16 per 128-byte row
                    store4(reinterpret_cast<T*>(wl + r * 128 + ((ch ^ (r & 7)) << 4) + (nl & 4) * 2), v);
                }
            }
        }
    }
    // wave-private region: program order + the compiler's lgkmcnt wait order the reads after the writes
    if (f32out) {
        const int ch = lane & 15;
        const int64_t nb = n_base + ch * 4;
#pragma unroll
        for (int it = 0; it < 16; ++it) {
            const int r = it * 4 + (lane >> 4);
            const int64_t m = m_base + r;
            f32x4 v = *reinterpret_cast<const f32x4*>(wl + r * 256 + ((ch ^ (r & 15)) << 4));
            if (m < m_lo || nb < n_lo) continue;
            float* dst = (float*)p.out + m * p.ldc + nb;
            if (p.epilogue == M4D_EPI_RESID_GATE) v += load4(dst);
            store4(dst, v);
        }
    } else {
        const int ch = lane & 7;
        const int64_t nb = n_base + ch * 8;
#pragma unroll
        for (int it = 0; it < 8; ++it) {
            const int r = it * 8 + (lane >> 3);
            const int64_t m = m_base + r;
            const uint4 v = *reinterpret_cast<const uint4*>(wl + r * 128 + ((ch ^ (r & 7)) << 4));
            if (m < m_lo || nb + 8 <= n_lo) continue;      // a chunk straddling n_lo rewrites identical values (benign)
            *reinterpret_cast<uint4*>((T*)p.out + m * p.ldc + nb) = v;
        }
    }
}

}  // namespace

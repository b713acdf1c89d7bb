// adapter_gemm_kernel: the shared projection with its adapters for the sizes between one row and the 256 x 256 tiles of gemm_wide.h, bf16 and
// float32.  out[m, n] = x W^T (+ bias) + u_g up_g^T for a BM x BN tile, BM = 32 MI WM, BN = 32 NI WN, WM x WN waves (four; bf16 from 64 x 128
// up: eight).
//
// What bounds these sizes is latency: a tile's K loop is serial, and with one or two waves per SIMD little else hides a trip to memory.  So the K tiles
// (128 bytes of a row) run through a ring of NST LDS stages filled by direct-to-LDS loads, NST - 1 tiles in flight; the fragments of the next
// 16 channels are read while the MFMAs of these run, across the one barrier of a tile too; and the requests for the tile NST ahead are issued
// one by one behind MFMAs.  (Reading a tile's fragments behind its barrier, all requests in front of it: 1.6 times the time at 512 x 5120 x
// 4096.)  Where the tiles do not fill the chip, K is cut into S slices (gridDim.y) whose float32 partial tiles a second kernel joins in slice
// order.  Counted (profiles/adapters_counters.log): 986 x 5120 x 4096 bf16, 55 us: the MFMAs are busy for 51 % of the CUs' busy time, 46 bytes/ns
// from L2 to each of 216 CUs, no LDS bank conflicts; 322 x 1536 x 4096 float32, 54 us: 73 %, of which a sixth is rows that pad 322 to 384, at 1.9 GHz.
// LDS image and swizzle are those of gemm.hip; rows beyond M and N are staged from the last row and not stored, 16-byte chunks beyond K are
// staged from a page of zeros.
#pragma once
#include "gemm_common.h"

namespace {

struct AdGemmArgs : GemmAdArgs {
    int S;             // K slices; > 1: float32 partial sums to ws [S, M, N]
    const int* order;  // [M] the row of x, u and out behind each row of the tiles, or nullptr: the same
};

__device__ __attribute__((aligned(16))) const unsigned zero_page[4] = {0u, 0u, 0u, 0u};

template <typename T, int MI, int NI, int WM, int WN>
struct AdGemmShape {
    static constexpr int BM = 32 * MI * WM, BN = 32 * NI * WN;
    static constexpr int STAGE = (BM + BN) * ROWB;
    static constexpr int NST = STAGE * 4 <= 131072 ? 4 : 3;
    static constexpr int THREADS = 64 * WM * WN;
    static constexpr int LDS = NST * STAGE;
};

template <typename T, int MI, int NI, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void adapter_gemm_kernel(AdGemmArgs p) {
    typedef AdGemmShape<T, MI, NI, WM, WN> Sh;
    typedef typename Frag8<T>::type frag_t;
    extern __shared__ __attribute__((aligned(16))) char ad_smem[];
    constexpr int ES = sizeof(T), KT = ROWB / ES, KSTEPS = KT / 16, NST = Sh::NST, BM = Sh::BM, BN = Sh::BN;
    constexpr int NW = WM * WN, NU = (BM + BN) / (8 * NW);      // staging instructions per wave and K tile (8 rows x 128 bytes each)
    static_assert((BM + BN) % (8 * NW) == 0, "whole requests");
    int tm, tn;
    tile_coords(p, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int li = lane & 31, hi = lane >> 5, wm = wave / WN, wn = wave % WN;
    const unsigned lds_base = (unsigned)(uintptr_t)(LDS_AS char*)ad_smem;

    const int nk = (int)((p.K + KT - 1) / KT), per = (nk + p.S - 1) / p.S;
    const int kt0 = (int)blockIdx.y * per, kt1 = min(nk, kt0 + per);
    const int tail = (int)(p.K * ES - (int64_t)(nk - 1) * ROWB);      // bytes of the last K tile

    // unit j = wave + NW i: rows 8 j + (lane >> 3) of the stage (x rows, then W rows), physical chunk lane & 7
    const char* src[NU];
    int lc16[NU];
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const int j = wave + NW * i, r = j * 8 + (lane >> 3);
        const bool isx = j * 8 < BM;
        const int rr = isx ? r : r - BM;
        int64_t row = isx ? min(m0 + rr, p.M - 1) : min(n0 + rr, p.N - 1);
        if (isx && p.order) row = p.order[row];
        lc16[i] = (((lane & 7) ^ ((rr >> 1) & 7)) << 4);
        src[i] = (isx ? (const char*)p.A + row * p.lda * ES : (const char*)p.W + row * p.ldw * ES) + lc16[i];
    }
    // request i of K tile kt into its stage; chunks beyond the end of K come from the page of zeros
    auto request = [&](int kt, unsigned dst, int i) {
        const char* s = src[i] + (int64_t)kt * ROWB;
        if (kt == nk - 1 && lc16[i] >= tail) s = (const char*)zero_page;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(dst + i * (NW * 1024)), "v"(s) : "memory", "m0");
    };
    auto stage_of = [&](int kt) { return (unsigned)((kt - kt0) % NST) * Sh::STAGE; };
    auto dst_of = [&](int kt) { return __builtin_amdgcn_readfirstlane(lds_base + stage_of(kt) + wave * 1024); };
    // all but the youngest n tiles' requests (n <= 3) have landed, of this wave; then of all, and nobody reads an older stage any more
    auto arrive = [&](int n) {
        if (n >= 3) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"(3 * NU) : "memory");
        else if (n == 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"(2 * NU) : "memory");
        else if (n == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"(NU) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    f32x16 acc[NI][MI];
#pragma unroll
    for (int a = 0; a < NI; ++a)
#pragma unroll
        for (int b = 0; b < MI; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
    frag_t fa[2][MI], fw[2][NI];
    auto read = [&](unsigned stage, int kk, frag_t (&a)[MI], frag_t (&w)[NI]) {
        const char* sA = ad_smem + stage;
        const char* sW = sA + BM * ROWB;
        const int c0 = (kk * 16 + hi * 8) * ES / 16;
        auto rd = [&](const char* s, int row) {
            if constexpr (ES == 2) return *reinterpret_cast<const frag_t*>(s + lds_off(row, c0));
            else {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(s + lds_off(row, c0)), h4 = *reinterpret_cast<const f32x4*>(s + lds_off(row, c0 + 1));
                return (frag_t)__builtin_shufflevector(lo, h4, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        };
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = rd(sA, (wm * MI + i) * 32 + li);
#pragma unroll
        for (int i = 0; i < NI; ++i) w[i] = rd(sW, (wn * NI + i) * 32 + li);
    };
    // K tile kt, its first fragments in set 0.  MORE: requests tile kt - 1 + NST into the stage of tile kt - 1 (request i in phase i * KSTEPS / NU);
    // NEXT: at the end tile kt + 1 has landed and its first fragments are in set 0.  NQ = requests issued before the last phase.
    constexpr int NQ = (NU * (KSTEPS - 1) + KSTEPS - 1) / KSTEPS;
    auto tile = [&](int kt, auto MORE_T, auto NEXT_T, int younger) {
        constexpr bool MORE = decltype(MORE_T)::value, NEXT = decltype(NEXT_T)::value;
        const unsigned cur = stage_of(kt), nxt = stage_of(kt + 1);
        unsigned dst = 0;
        if constexpr (MORE) dst = dst_of(kt - 1);
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
            constexpr int LASTK = KSTEPS - 1;
            const int c = kk & 1;
            if (kk < LASTK) read(cur, kk + 1, fa[c ^ 1], fw[c ^ 1]);
            __builtin_amdgcn_sched_barrier(0);
            int q = (NU * kk + KSTEPS - 1) / KSTEPS;                 // the phase's first request (all constants after unrolling)
            const int q1 = (NU * (kk + 1) + KSTEPS - 1) / KSTEPS;
#pragma unroll
            for (int m = 0; m < MI * NI; ++m) {
                mma32(fw[c][m / MI], fa[c][m % MI], acc[m / MI][m % MI]);
                __builtin_amdgcn_sched_barrier(0);
                if (m == 0 && kk == LASTK && NEXT) {
                    if constexpr (MORE) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"((NST - 3) * NU + NQ) : "memory");
                    else arrive(younger);
                    read(nxt, 0, fa[c ^ 1], fw[c ^ 1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (MORE) {
                    if (q < q1) request(kt - 1 + NST, dst, q++);
                    if (m == MI * NI - 1)
                        while (q < q1) request(kt - 1 + NST, dst, q++);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };
    const AdTile<MI> ad_tile = adapters_tile<MI>(p, tm, m0 + wm * MI * 32, lane, (int)blockIdx.y, p.order);      // (a slice takes every S-th adapter)
    const int n_tiles = kt1 - kt0;
    if (n_tiles > 0) {
#pragma unroll
        for (int s = 0; s < NST; ++s)
            if (s < n_tiles) {
                const unsigned dst = dst_of(kt0 + s);
#pragma unroll
                for (int i = 0; i < NU; ++i) request(kt0 + s, dst, i);
            }
        arrive(min(NST, n_tiles) - 1);
        read(stage_of(kt0), 0, fa[0], fw[0]);
        int kt = kt0;
        if (n_tiles > 1) {
            tile(kt, std::false_type{}, std::true_type{}, min(NST, n_tiles) - 2);
            ++kt;
        }
        for (; kt - 1 + NST < kt1; ++kt) tile(kt, std::true_type{}, std::true_type{}, 0);
        for (; kt < kt1 - 1; ++kt) tile(kt, std::false_type{}, std::true_type{}, kt1 - 2 - kt);
        tile(kt, std::false_type{}, std::false_type{}, 0);
    }
    adapters_extend<T, NI, MI>(p, acc, ad_tile, n0 + wn * NI * 32, lane, p.S);

    // out of the accumulator layout (lane = row) through LDS: 4 consecutive columns per lane, whole rows per group of lanes
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    constexpr int EN = NI % 2 ? 1 : NI;                      // column blocks of 32 in one trip (three: one after the other)
    constexpr int NCH = EN * 8;                              // 16-byte chunks of a row of them
    char* wl = ad_smem + wave * 32 * NCH * 16;
    static_assert(NW * 32 * NCH * 16 <= Sh::LDS, "the epilogue's block fits");
    const T* bias = (const T*)p.bias;
    const int ch = lane % NCH;
    float* part = p.S > 1 ? p.ws + (int64_t)blockIdx.y * p.M * p.N : nullptr;
#pragma unroll
    for (int nb = 0; nb < NI; nb += EN) {
        const int64_t n = n0 + (wn * NI + nb) * 32 + ch * 4;
        f32x4 bv = {0.f, 0.f, 0.f, 0.f};
        if (p.S == 1 && bias && n < p.N) bv = load4(bias + n);
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
            for (int ni = 0; ni < EN; ++ni)
#pragma unroll
                for (int rq = 0; rq < 4; ++rq) {
                    const int c = ni * 8 + rq * 2 + hi;
                    const f32x16& a = acc[nb + ni][mi];
                    const f32x4 v = {a[rq * 4], a[rq * 4 + 1], a[rq * 4 + 2], a[rq * 4 + 3]};
                    *reinterpret_cast<f32x4*>(wl + li * NCH * 16 + ((c ^ (li & (NCH - 1))) << 4)) = v;
                }
            // (wave-private region: program order and the compiler's lgkmcnt waits order the reads behind the writes)
#pragma unroll
            for (int it = 0; it < NCH / 2; ++it) {
                const int r = it * (64 / NCH) + lane / NCH;
                const f32x4 v = *reinterpret_cast<const f32x4*>(wl + r * NCH * 16 + ((ch ^ (r & (NCH - 1))) << 4));
                const int64_t m = m0 + (wm * MI + mi) * 32 + r;
                if (m < p.M && n < p.N) {
                    if (part) store4(part + m * p.N + n, v);
                    else store4((T*)p.out + (p.order ? p.order[m] : m) * p.ldc + n, v + bv);
                }
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void adapter_gemm_join_kernel(AdGemmArgs p) {
    const int64_t n4 = p.N / 4, total = p.M * n4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / n4, n = (i - m * n4) * 4;
        f32x4 v = load4(p.ws + m * p.N + n);
        for (int s = 1; s < p.S; ++s) v += load4(p.ws + ((int64_t)s * p.M + m) * p.N + n);
        if (p.bias) v += load4((const T*)p.bias + n);
        store4((T*)p.out + (p.order ? p.order[m] : m) * p.ldc + n, v);
    }
}

// D += A(16 x 32) * B(32 x 16): lane = (i = l & 15, q = l >> 4) holds the 8 consecutive k at 8 q of row i; D: column l & 15, rows 4 q + [0, 4)
M4D_DEV void mma16(const bf16x8& a, const bf16x8& b, f32x4& c) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
M4D_DEV void mma16(const f32x8& a, const f32x8& b, f32x4& c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
}

// 8 consecutive elements of a row at k, those at or beyond K as zero (rows are whole 16-byte chunks)
template <typename T> M4D_DEV typename Frag8<T>::type load_k8(const T* row, int k, int K);
template <> M4D_DEV bf16x8 load_k8<bf16_t>(const bf16_t* row, int k, int K) {
    bf16x8 v = {};
    if (k < K) v = *reinterpret_cast<const bf16x8*>(row + k);
    return v;
}
template <> M4D_DEV f32x8 load_k8<float>(const float* row, int k, int K) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    if (k < K) a = load4(row + k);
    if (k + 4 < K) b = load4(row + k + 4);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Up to 16 rows (single tokens, modulation vectors): one pass over W, which is all the traffic there is.  A workgroup owns 16 rows of W, its
// eight waves take 256 bytes of them each in turn straight into registers (every byte is used once: LDS would only add a trip); the adapters
// of the batch are dealt to the waves like further K steps, and the waves' sums meet in LDS in wave order.  2 rows, 1536 -> 9216: 8.5 us (the 28 MB of
// W at 3.3 TB/s: most of it is the ramp).
constexpr int SKINNY_WAVES = 8;
template <typename T>
__global__ __launch_bounds__(64 * SKINNY_WAVES) void adapter_gemv_kernel(AdGemmArgs p) {
    typedef typename Frag8<T>::type frag_t;
    __shared__ f32x4 red[SKINNY_WAVES][64];
    constexpr int U = 4, KS = 32 * U;               // K elements of a wave's step
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, i16 = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const T* w = (const T*)p.W + min(n0 + i16, p.N - 1) * p.ldw + q * 8;
    const int row = min(i16, (int)p.M - 1);         // (lanes beyond the last row compute copies of it and store nothing)
    const T* x = (const T*)p.A + row * p.lda + q * 8;
    const int K = (int)p.K;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    int k0 = wave * KS;
    for (; k0 + KS <= K; k0 += SKINNY_WAVES * KS) {
        frag_t fw[U], fx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) fw[u] = *reinterpret_cast<const frag_t*>(w + k0 + u * 32);
#pragma unroll
        for (int u = 0; u < U; ++u) fx[u] = *reinterpret_cast<const frag_t*>(x + k0 + u * 32);
#pragma unroll
        for (int u = 0; u < U; ++u) mma16(fw[u], fx[u], acc);
    }
    for (int u = 0; u < U && k0 + u * 32 < K; ++u) {      // the last, partial step of one wave
        const int k = k0 + u * 32;
        mma16(load_k8<T>(w, k, K - q * 8), load_k8<T>(x, k, K - q * 8), acc);
    }
    const int ra = p.row_adapter[row];
    for (int i = p.tile_off[0] + wave; i < p.tile_off[1]; i += SKINNY_WAVES) {      // (at most 16 rows: one tile)
        const int g = p.tile_list[i];
        const T* b = (const T*)p.up + ((int64_t)g * p.N + min(n0 + i16, p.N - 1)) * p.R;
        const T* u = (const T*)p.u + (int64_t)row * u_stride<T>(p.R);
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < p.R; k += 32) {
            const int w = min(32, p.R - k), ks = min(q * 8, w - 8);
            const frag_t zero = {};
            frag_t fb = *reinterpret_cast<const frag_t*>(b + k + ks);
            if (q * 8 >= w) fb = zero;
#pragma unroll
            for (int h = 0; h < Parts<T>::N; ++h) {
                const frag_t fu = *reinterpret_cast<const frag_t*>(u + u_hi<T>(k) + h * w + ks);
                mma16(fb, q * 8 >= w ? zero : fu, sum);
            }
        }
        if (ra == g) acc += sum;                    // (see adapters_extend: rows of other adapters see nothing of this one)
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
        const int64_t n = n0 + q * 4;
        if (i16 < p.M && n < p.N) {
            f32x4 v = red[0][lane];
#pragma unroll
            for (int k = 1; k < SKINNY_WAVES; ++k) v += red[k][lane];
            if (p.bias) v += load4((const T*)p.bias + n);
            store4((T*)p.out + (int64_t)i16 * p.ldc + n, v);
        }
    }
}

}  // namespace

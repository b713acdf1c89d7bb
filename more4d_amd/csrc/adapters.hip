// Low-rank adapters of many requests beside a shared projection (m4d_adapter_down, m4d_linear_adapters, m4d_adapter_grad).
//
//   y = x W^T + bias + s_g (x A_g^T) B_g^T          g = the adapter that the row names (none: the shared projection alone)
//
// forward:   u = s_g x A_g^T  (m4d_adapter_down), then ONE GEMM over K with u B_g^T added behind its K loop (m4d_linear_adapters): a separate
//            pass over y would read and write it once more and round it twice;
// backward:  v = s_g dy B_g is the same down projection (with B^T for A), dx = dy W + v A_g the same GEMM (with W^T, A^T), and
//            dA_g = sum_rows v^T x, dB_g = sum_rows dy^T u are m4d_adapter_grad: products that contract over the rows.
//
// Rows are worked on in SLOTS: the plan lists the rows adapter by adapter, each adapter's list padded (slot_row = -1) to whole PIECES of 64
// slots, so a workgroup never sees two adapters whatever the order of the requests, and one-row requests of one adapter share a piece.
// u is written twice: by rows, the GEMM's operand (gemm_common.h: u_hi), and as the operand of the row contraction in the order in which its MFMA
// lanes read it, [slot / 16][rank / 32][part][lane][8] with lane = rank % 32 + 32 * (slot % 16 / 8) (read row by row, 16 bytes of 32 ranks each,
// these loads cost the address unit as much as x's); pad slots and ranks hold zero.
// Rounding: u (or v) is nowhere rounded to bf16 once, which would put an error of the size of the result's own rounding on it (gradients: 0.0024 of
// their size instead of 0.0017; y and dx more with every rank, 0.0019 at 128): it is kept as a sum of two parts, u = hi + lo to 16 bits, at
// twice the products, which are not what bounds the row contraction and 32 more of K = 1536 .. 5120 per 32 ranks in the GEMM.
//
// The operand of a down projection is laid out once (m4d_adapter_pack) in the order in which the MFMA lanes read it: chunks of 64 channels, 32
// ranks, and within them lane (rank l & 31, channels 32 (l >> 5) + [0, 32) as four 8-element fragments).  With that order of the channels a
// lane holds a whole 32-channel block of its row, so the same pass that multiplies x by A can write x's 8-bit form (act8.h): a training
// step that keeps its inputs in 8 bits reads them once.
#include "act8.h"
#include "adapters_gemm.h"

extern "C" __attribute__((visibility("hidden"))) int m4d_launch_gemm_wide_adapters(const void* args, unsigned nwg, hipStream_t st);

namespace {

constexpr int PIECE = 64;

// ---------------------------------------------------------------- layout of a bank
struct PackArgs {
    const void *a, *b;          // [G, rank, K], [G, N, rank]
    void *a_down, *b_up, *b_down, *a_up;
    int G, rank, K, N, R;
};
M4D_DEV int64_t down_elems(int G, int R, int K) { return (int64_t)G * ((K + 63) / 64) * ((R + 31) / 32) * 2048; }

// one element of the down layout of an operand [rank, K] of adapter g: index -> (rank, channel)
template <typename T>
M4D_DEV void pack_down(const PackArgs& p, void* out, int K, bool from_b, int64_t i) {
    const int e = (int)(i & 7), lane = (int)(i >> 3) & 63, kk = (int)(i >> 9) & 3, rts = (p.R + 31) / 32, nc = (K + 63) / 64;
    int64_t j = i >> 11;
    const int rt = (int)(j % rts);
    j /= rts;
    const int c = (int)(j % nc);
    const int64_t g = j / nc;
    const int r = rt * 32 + (lane & 31), k = c * 64 + (lane >> 5) * 32 + kk * 8 + e;
    T v = (T)0.f;
    if (r < p.rank && k < K) v = from_b ? ((const T*)p.b)[(g * K + k) * p.rank + r] : ((const T*)p.a)[(g * p.rank + r) * K + k];
    ((T*)out)[i] = v;
}
// one element of the up layout [rows, R] (rows = N from b, K from a)
template <typename T>
M4D_DEV void pack_up(const PackArgs& p, void* out, int rows, bool from_a, int64_t i) {
    const int r = (int)(i % p.R);
    const int64_t j = i / p.R, n = j % rows, g = j / rows;
    T v = (T)0.f;
    if (r < p.rank) v = from_a ? ((const T*)p.a)[(g * p.rank + r) * rows + n] : ((const T*)p.b)[(g * rows + n) * p.rank + r];
    ((T*)out)[i] = v;
}
template <typename T>
__global__ __launch_bounds__(256) void adapter_pack_kernel(PackArgs p) {
    const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, st = (int64_t)gridDim.x * 256;
    if (blockIdx.y == 0 && p.a_down) for (int64_t i = i0; i < down_elems(p.G, p.R, p.K); i += st) pack_down<T>(p, p.a_down, p.K, false, i);
    if (blockIdx.y == 1 && p.b_up) for (int64_t i = i0; i < (int64_t)p.G * p.N * p.R; i += st) pack_up<T>(p, p.b_up, p.N, false, i);
    if (blockIdx.y == 2 && p.b_down) for (int64_t i = i0; i < down_elems(p.G, p.R, p.N); i += st) pack_down<T>(p, p.b_down, p.N, true, i);
    if (blockIdx.y == 3 && p.a_up) for (int64_t i = i0; i < (int64_t)p.G * p.K * p.R; i += st) pack_up<T>(p, p.a_up, p.K, true, i);
}

// ---------------------------------------------------------------- down projection
struct DownArgs {
    const void* x; const void* a; const float* scale;
    void* u; void* ut;
    int8_t* codes; uint8_t* exps;
    const int *slot_row, *piece_adapter;
    int64_t ldx;
    int K, R, n_pieces;
    int KS;                // K slices (gridDim.y); > 1: unscaled float32 sums to part [KS, n_pieces, R rounded up to 32, 64]
    float* part;
    int split;             // u as the projection's operand (gemm_common.h: u_hi); 0: [rows, R], rounded once
};

// bf16, the projection's operand: v = hi + lo to 16 bits, hi being v cut off towards zero (its predecessor where v is a bf16 number itself), so that
// both parts have v's sign: hi * b + lo * b is then what v * b is for an infinite b or v too (parts of v rounded to nearest give inf - inf or 0 * inf).
M4D_DEV void split2(float v, bf16_t& hi, bf16_t& lo) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    if (!isfinite(v)) { hi = lo = (bf16_t)v; return; }
    const float h = __builtin_bit_cast(float, (u & 0x7fffffffu) != 0u && (u & 0xffffu) == 0u ? u - 0x10000u : u & 0xffff0000u);
    hi = (bf16_t)h; lo = (bf16_t)(v - h);
}
M4D_DEV void split2(float v, float& hi, float&) { hi = v; }

// four ranks (r .. r + 3, r a multiple of 4) of a row of u
template <typename T>
M4D_DEV void store_u(T* row, int r, int R, const f32x4& v) {
    T hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split2(v[e], hi[e], lo[e]);
    T* d = row + u_hi<T>(r);
    store4(d, f32x4{(float)hi[0], (float)hi[1], (float)hi[2], (float)hi[3]});
    if constexpr (Parts<T>::N == 2) store4(d + min(32, R - (r & ~31)), f32x4{(float)lo[0], (float)lo[1], (float)lo[2], (float)lo[3]});
}

// four ranks (r .. r + 3) of one slot to u and / or ut, scaled
template <typename T>
M4D_DEV void down_store(const DownArgs& p, int64_t piece, int g, int slot, int row, int r, f32x4 v) {
    const float sc = p.scale[g];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = row >= 0 ? v[e] * sc : 0.f;
    if (p.u && row >= 0 && r < p.R) {
        if (p.split) store_u((T*)p.u + (int64_t)row * u_stride<T>(p.R), r, p.R, v);
        else store4((T*)p.u + (int64_t)row * p.R + r, v);
    }
    if (p.ut) {
        const int64_t s = piece * PIECE + slot;
        T* d = (T*)p.ut + (((s >> 4) * ((p.R + 31) >> 5) + (r >> 5)) * (64 * Parts<T>::N) + (r & 31) + ((slot >> 3) & 1) * 32) * 8 + (slot & 7);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T hi = (T)v[e];
            d[e * 8] = hi;
            if constexpr (Parts<T>::N == 2) d[512 + e * 8] = (T)(isfinite((float)hi) ? v[e] - (float)hi : 0.f);      // (inf - inf would be NaN)
        }
    }
}

// u of one piece: 64 slots x RT * 32 ranks, a chunk of 64 channels at a time.  Bound by reading x once; the operand comes from L2, as many bytes
// again at 64 ranks.  Rows and operand go to LDS by direct loads, whole 128-byte lines of a row per request (straight into registers, a lane of
// the MFMA layout wants 16 bytes of a row of its own, and the address unit then handles 64 lines per request: 85 us for 21840 x 5120 at rank
// 64, against 46 us of HBM time), NST - 1 chunks in flight, one barrier per chunk, two workgroups per CU.
// Wave (s, h): slots 32 s + [0, 32) and rank tiles h, h + 2, ...; with one rank tile h takes every other 16 channels instead.  QUANT: four
// more waves write the codes, 16 of the piece's rows each, two lanes per block of 32 channels, out of the same LDS.  (The waves that request
// chunks cannot also store: loads and stores share one counter, only loads return in order, so a wait that must not pass too early has to
// wait for the stores as well, and little stays in flight: 128 us instead of 75 + 40 at 21840 x 5120.)
// DEEP: fewer workgroups than CUs, each with the LDS of a whole CU: up to twelve chunks in flight, because alone a workgroup waits for memory (0.5
// us a chunk with four stages).  21840 x 5120, rank 64: 60 - 68 us (3.7 TB/s of x), with codes 96 - 107 (floors 46 and 69), and 7 - 13 more for the join.
template <typename T, int RT, bool DEEP> struct DownShape {
    static constexpr int XB = 64 * 64 * sizeof(T), AB = RT * 64 * 32 * sizeof(T), STAGE = XB + AB;
    static constexpr int NST = DEEP ? (STAGE * 12 <= 144 * 1024 ? 12 : 144 * 1024 / STAGE) : STAGE * 4 <= 80 * 1024 ? 4 : STAGE * 3 <= 80 * 1024 ? 3 : 2;
    static constexpr int LDS = NST * STAGE;
};
// s_waitcnt vmcnt(N * NU) lgkmcnt(0); s_barrier  with N = min(n, MAX)
template <int MAX, int NU>
M4D_DEV void wait_younger(int n) {
    if constexpr (MAX > 0) {
        if (n < MAX) { wait_younger<MAX - 1, NU>(n); return; }
    }
    static_assert(MAX * NU < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"(MAX * NU) : "memory");
}
template <typename T, int RT, bool QUANT, bool DEEP>
__global__ __launch_bounds__(QUANT ? 512 : 256, 2) void adapter_down_kernel(DownArgs p) {
    typedef DownShape<T, RT, DEEP> Sh;
    typedef typename Frag8<T>::type frag_t;
    extern __shared__ __attribute__((aligned(16))) char ad_smem[];
    constexpr int ES = sizeof(T), NST = Sh::NST, RB = 64 * ES, CPR = RB / 16, RPU = 1024 / RB;      // bytes, 16-byte chunks of a row; rows of a request
    constexpr int NX = 64 / RPU / 4, NA = Sh::AB / 4096, NU = NX + NA;                               // requests of a wave and chunk
    constexpr int NT = RT == 1 ? 1 : RT / 2;
    const int t = threadIdx.x, lane = t & 63, li = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6), s = wave & 1, h = wave >> 1;
    // more than RT * 32 ranks: ny workgroups read the same rows; numbered so that they run next to each other on one XCD and share them in its L2
    const int rts = (p.R + 31) / 32, ny = (rts + RT - 1) / RT, b8 = blockIdx.x >> 3;
    const int piece = (b8 / ny) * 8 + (blockIdx.x & 7), rt0 = (b8 % ny) * RT;
    if (piece >= p.n_pieces) return;
    const int g = __builtin_amdgcn_readfirstlane(p.piece_adapter[piece]);
    const int* sr = p.slot_row + (int64_t)piece * PIECE;
    const int nc = (p.K + 63) >> 6, nb = (p.K + 31) >> 5, per = (nc + p.KS - 1) / p.KS, c0 = (int)blockIdx.y * per, c1 = min(nc, c0 + per);
    const int tail = (p.K - (nc - 1) * 64) * ES;         // bytes of the last chunk of a row
    const unsigned lds_base = (unsigned)(uintptr_t)(LDS_AS char*)ad_smem;
    auto swz = [](int r) { return ES == 2 ? (r >> 1) & 7 : r & 15; };      // 16-byte chunk c of row r sits at chunk c ^ swz(r)
    if constexpr (QUANT) {
        if (wave >= 4) {
            if (rt0 == 0) {
                // this lane's row, and where its codes and exponents go
                const int qr = (wave - 4) * 16 + (lane >> 2), qrow = sr[qr];
                int8_t* qc = p.codes + (int64_t)max(qrow, 0) * nb * 32 + (lane & 3) * 16;
                uint8_t* qe = p.exps + (int64_t)max(qrow, 0) * nb;
                unsigned even = 0;                           // the exponents of the even chunk before an odd one
                for (int c = c0; c < c1; ++c) {
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // the barrier of chunk c
                    const char* st = ad_smem + ((c - c0) % NST) * Sh::STAGE;
                    unsigned v[4 * ES];                               // 16 channels, half a block
#pragma unroll
                    for (int k = 0; k < ES; ++k) {
                        const u32x4q d = *reinterpret_cast<const u32x4q*>(st + qr * RB + ((((lane & 3) * ES + k) ^ swz(qr)) << 4));
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[k * 4 + e] = d[e];
                    }
                    const unsigned b = block_exp(max_xor1(top_bits<T>(v)));
                    const float inv = block_inv(min(b, 248u));
                    u32x4q q4;
#pragma unroll
                    for (int k = 0; k < 4; ++k) q4[k] = encode_of<T>(v, k, b, inv, b == 248u);
                    const int blk = c * 2 + ((lane >> 1) & 1);
                    if (qrow >= 0 && blk < nb) *reinterpret_cast<u32x4q*>(qc + (int64_t)c * 64) = q4;
                    // exponents: the row's two bytes meet in its first lane, and where rows of bytes are 4-byte aligned two chunks' go out as one dword
                    // (bytes one at a time are 32 cache lines a store)
                    const unsigned both = b | ((unsigned)__builtin_amdgcn_mov_dpp((int)b, 0x4E, 0xF, 0xF, true) << 8);
                    if ((lane & 3) == 0 && qrow >= 0) {
                        if (nb & 3) {
                            qe[c * 2] = (uint8_t)both;
                            if (c * 2 + 1 < nb) qe[c * 2 + 1] = (uint8_t)(both >> 8);
                        } else if (c & 1) {
                            if (c == c0) *reinterpret_cast<uint16_t*>(qe + c * 2) = (uint16_t)both;
                            else *reinterpret_cast<unsigned*>(qe + c * 2 - 2) = (both << 16) | even;
                        } else if (c == c1 - 1) *reinterpret_cast<uint16_t*>(qe + c * 2) = (uint16_t)both;
                    }
                    even = both;
                }
            } else {
                for (int c = c0; c < c1; ++c) asm volatile("s_barrier" ::: "memory");
            }
            if constexpr (RT == 1) {                         // (the barriers of the join below)
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __syncthreads();
            }
            return;
        }
    }
    const char* sx[NX];
    int cb[NX];
#pragma unroll
    for (int i = 0; i < NX; ++i) {
        const int r = (wave + 4 * i) * RPU + lane / CPR, rw = sr[r];
        cb[i] = ((lane % CPR) ^ swz(r)) * 16;
        sx[i] = (const char*)p.x + (int64_t)(rw >= 0 ? rw : sr[0]) * p.ldx * ES + cb[i];      // (pad slots compute copies of the first row)
    }
    const char* sa[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        const int o = (wave + 4 * i) * 1024, rt = o / (2048 * ES), in = o % (2048 * ES);
        sa[i] = (const char*)p.a + (((int64_t)g * nc * rts + min(rt0 + rt, rts - 1)) * 2048) * ES + in + lane * 16;
    }
    auto request = [&](int c) {
        const unsigned dst = __builtin_amdgcn_readfirstlane(lds_base + (unsigned)((c - c0) % NST) * Sh::STAGE + wave * 1024);
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const char* q = sx[i] + (int64_t)c * RB;
            if (c == nc - 1 && cb[i] >= tail) q = (const char*)zero_page;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(dst + i * 4096), "v"(q) : "memory", "m0");
        }
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const char* q = sa[i] + (int64_t)c * rts * 2048 * ES;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(dst + Sh::XB + i * 4096), "v"(q) : "memory", "m0");
        }
    };
    f32x16 acc[NT];
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[k][q] = 0.f;
    const int row = sr[s * 32 + li];
#pragma unroll
    for (int i = 0; i < NST - 1; ++i)
        if (c0 + i < c1) request(c0 + i);
    for (int c = c0; c < c1; ++c) {
        // chunk c has landed when at most the younger chunks' requests are pending (only loads are counted: a store in flight makes the wait
        // stricter); behind the barrier everybody's has, and nobody reads chunk c - 1 any more, whose stage the next request overwrites
        wait_younger<NST - 2, NU>(c1 - 1 - c);
        if (c + NST - 1 < c1) request(c + NST - 1);
        const char* st = ad_smem + ((c - c0) % NST) * Sh::STAGE;
        auto frag = [&](const char* q, int o0, int o1) {
            if constexpr (ES == 2) return *reinterpret_cast<const frag_t*>(q + o0);
            else return (frag_t)__builtin_shufflevector(*reinterpret_cast<const f32x4*>(q + o0), *reinterpret_cast<const f32x4*>(q + o1), 0, 1, 2, 3, 4, 5, 6, 7);
        };
        frag_t x[4];
        const int r = s * 32 + li;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const int ch = (hi * 32 + kk * 8) * ES / 16;
            x[kk] = frag(st + r * RB, (ch ^ swz(r)) << 4, ((ch + 1) ^ swz(r)) << 4);
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            if (RT == 1 && (kk & 1) != h) continue;          // (wave-uniform)
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                const char* q = st + Sh::XB + (((RT == 1 ? 0 : h + 2 * k) * 4 + kk) * 64 + lane) * 8 * ES;
                mma32(frag(q, 0, 16), x[kk], acc[k]);
            }
        }
    }
    if constexpr (RT == 1) {                                 // join the two halves of the channels
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        float* red = reinterpret_cast<float*>(ad_smem) + s * 1024 + lane;
        if (h == 1) {
#pragma unroll
            for (int q = 0; q < 16; ++q) red[q * 64] = acc[0][q];
        }
        __syncthreads();
        if (h == 1) return;
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[0][q] += red[q * 64];
    }
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const int rt = rt0 + (RT == 1 ? 0 : h + 2 * k), r = rt * 32 + q4 * 8 + hi * 4, slot = s * 32 + li;
            if (rt >= rts) continue;
            const f32x4 v = {acc[k][q4 * 4], acc[k][q4 * 4 + 1], acc[k][q4 * 4 + 2], acc[k][q4 * 4 + 3]};
            if (p.part) {
                float* d = p.part + (((int64_t)blockIdx.y * p.n_pieces + piece) * rts * 32 + r) * PIECE + slot;
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e * PIECE] = v[e];
            } else down_store<T>(p, piece, g, slot, row, r, v);
        }
}

// The same for at most 16 rows (single tokens): a workgroup takes 16 ranks of one adapter, its eight waves the chunks of K in turn, straight from
// memory into the 16 x 16 x 32 MFMA; all rows are multiplied by every adapter and only its own are kept.  One launch instead of slices and
// their join (12 us): K = 5120, rank 32, six adapters 9 us; K = 1536, rank 16, two adapters 4.
template <typename T>
__global__ __launch_bounds__(64 * SKINNY_WAVES) void adapter_down16_kernel(DownArgs p, const int* row_adapter, const int* adapters, int rows) {
    typedef typename Frag8<T>::type frag_t;
    __shared__ f32x4 red[SKINNY_WAVES][64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, i16 = lane & 15, q = lane >> 4;
    const int g = adapters[blockIdx.x], r0 = blockIdx.y * 16, nc = (p.K + 63) >> 6, rts = (p.R + 31) >> 5;
    const int row = min(i16, rows - 1);
    // of a chunk's packed operand (channel 32 hi + 8 kk + e at [rt][kk][rank + 32 hi][e]) quarter q of the wave takes hi = q & 1, kk = 2 j + (q >> 1)
    const T* a = (const T*)p.a + ((int64_t)g * nc * rts + (r0 >> 5)) * 2048 + (q >> 1) * 512 + ((r0 & 16) + i16 + 32 * (q & 1)) * 8;
    const T* x = (const T*)p.x + (int64_t)row * p.ldx + (q & 1) * 32 + (q >> 1) * 8;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    int c = wave;
    constexpr int U = 4;
    for (; c + (U - 1) * SKINNY_WAVES < nc - 1; c += U * SKINNY_WAVES) {      // whole chunks: all loads first
        frag_t fa[U][2], fx[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                fa[u][j] = *reinterpret_cast<const frag_t*>(a + (int64_t)(c + u * SKINNY_WAVES) * rts * 2048 + j * 1024);
                fx[u][j] = *reinterpret_cast<const frag_t*>(x + (c + u * SKINNY_WAVES) * 64 + j * 16);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) mma16(fa[u][j], fx[u][j], acc);
    }
    for (; c < nc; c += SKINNY_WAVES)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            mma16(*reinterpret_cast<const frag_t*>(a + (int64_t)c * rts * 2048 + j * 1024), load_k8<T>(x, c * 64 + j * 16, p.K - (q & 1) * 32 - (q >> 1) * 8), acc);
    red[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && i16 < rows && row_adapter[i16] == g) {
        f32x4 v = red[0][lane];
#pragma unroll
        for (int k = 1; k < SKINNY_WAVES; ++k) v += red[k][lane];
        const f32x4 w = v * p.scale[g];
        if (p.split) store_u((T*)p.u + (int64_t)i16 * u_stride<T>(p.R), r0 + q * 4, p.R, w);
        else store4((T*)p.u + (int64_t)i16 * p.R + r0 + q * 4, w);
    }
}

// the K slices' sums of four ranks of one slot, in slice order
template <typename T>
__global__ __launch_bounds__(256) void adapter_down_join_kernel(DownArgs p) {
    const int t = threadIdx.x, slot = t & 63, r = (blockIdx.y * 4 + (t >> 6)) * 4;
    const int64_t piece = blockIdx.x;
    const int64_t R32 = (p.R + 31) / 32 * 32;
    if (r >= R32) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < p.KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += p.part[((k * p.n_pieces + piece) * R32 + r + e) * PIECE + slot];
    down_store<T>(p, piece, p.piece_adapter[piece], slot, p.slot_row[piece * PIECE + slot], r, v);
}

// ---------------------------------------------------------------- contraction over the rows
struct GradArgs {
    const void* vt;                 // T, packed: [slot / 16][rank / 32][parts][64][8]
    const void* x;                  // T [rows, C] (row stride ldx), or
    const int8_t* codes; const uint8_t* exps;      // its 8-bit form (act8.hip)
    float* ws;                      // [n_chunks, R, C]
    void* out;                      // T [G, rank, C], or [G, C, rank]
    const int *slot_row, *chunks, *chunk_off;
    int64_t ldx;
    int C, R, rank, n_adapters, transposed;
};

// four consecutive columns of a row as T
template <typename T> struct Quad;
template <> struct Quad<bf16_t> { typedef bf16x4 type; };
template <> struct Quad<float> { typedef f32x4 type; };

// ws[chunk][r][c] = sum over the chunk's slots of vt[r][slot] * x[row of slot][c].  A workgroup owns 128 columns of one chunk, its four waves take
// 16 slots each in turn.  The contraction runs over ROWS, so the MFMA wants 8 rows of one column per lane: a lane loads 4 consecutive columns
// of 8 rows and regroups them in registers into 4 fragments, fragment f = column 4 * lane + f, so that no LDS transpose is needed and a lane
// ends with 4 consecutive columns of the result.  The chunk's row numbers sit in LDS, and PF steps of rows are in flight while one is used.
// Bound by reading x once: 21840 x 5120, rank 64: 61 - 66 us from bf16 (floor 46), 54 - 60 from codes (its conversions; floor 24); the sums
// of its chunks are joined in 7 us.
constexpr int CHUNK_PIECES = 64;       // most pieces in a chunk (the row numbers in LDS)
template <typename T, bool CODES, int RT>
__global__ __launch_bounds__(256, 2) void adapter_grad_kernel(GradArgs p) {
    typedef typename Frag8<T>::type frag_t;
    typedef typename Quad<T>::type quad_t;
    constexpr int PF = 2, NP = Parts<T>::N;
    constexpr int RED = RT * 4 * 16 * 64 * 4;
    __shared__ __attribute__((aligned(16))) char smem[RED > CHUNK_PIECES * PIECE * 4 ? RED : CHUNK_PIECES * PIECE * 4];
    int* rows = reinterpret_cast<int*>(smem);
    float* red = reinterpret_cast<float*>(smem);
    const int t = threadIdx.x, lane = t & 63, li = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int c = blockIdx.x * 128 + li * 4, r0 = blockIdx.z * (RT * 32);
    const int* ch = p.chunks + 3 * blockIdx.y;
    const int s0 = ch[0] * PIECE, n = ch[1] * PIECE - s0;
    for (int i = t; i < n; i += 256) rows[i] = p.slot_row[s0 + i];
    const bool cin = c < p.C;
    const int cc = cin ? c : 0;                     // (columns beyond C are computed from the first ones and not stored)
    const int nb = (p.C + 31) >> 5, rts = (p.R + 31) >> 5;
    const T* pv[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) pv[rt] = (const T*)p.vt + ((int64_t)(s0 >> 4) * rts + min((int)blockIdx.z * RT + rt, rts - 1)) * (512 * NP) + lane * 8;
    f32x16 acc[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[rt][f][q] = 0.f;
    __syncthreads();
    struct Step {
        frag_t v[RT][NP];
        quad_t x[8];
        int code[8];
        unsigned char ex[8];
    };
    // (pad slots, -1, read the chunk's first row: what they read is replaced by zero in use() — their v is zero, but zero times an infinity is not)
    const int row0 = rows[0];
    auto load = [&](int s, Step& b) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int q = 0; q < NP; ++q) b.v[rt][q] = *reinterpret_cast<const frag_t*>(pv[rt] + (int64_t)(s >> 4) * rts * (512 * NP) + q * 512);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = rows[s + hi * 8 + j];
            const int64_t row = r >= 0 ? r : row0;
            if constexpr (CODES) {
                b.code[j] = *reinterpret_cast<const int*>(p.codes + row * nb * 32 + cc);
                b.ex[j] = p.exps[row * nb + (cc >> 5)];
            } else b.x[j] = *reinterpret_cast<const quad_t*>((const T*)p.x + row * p.ldx + cc);
        }
    };
    auto use = [&](int s, Step& b) {
        if (s + PIECE >= n && rows[s + 15] < 0) {   // (uniform: only an adapter's last piece has pad slots)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (rows[s + hi * 8 + j] < 0) {
                    if constexpr (CODES) { b.code[j] = 0; b.ex[j] = 1; }
                    else b.x[j] = quad_t{};
                }
        }
        if constexpr (CODES) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) b.x[j][e] = (T)decode1((unsigned)b.code[j], e, step_of(b.ex[j]));      // exact in T
        }
        // two parts of v have signs of their own: an infinity of x meets the first one only (inf - inf would be NaN where v inf is an infinity)
        bool bad = false;
        if constexpr (NP == 2 && !CODES) {
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const u32x2 w = __builtin_bit_cast(u32x2, b.x[j]);
                const unsigned d[2] = {w[0], w[1]};
                top = max(top, top_bits<T>(d));
            }
            bad = __any(top >= 0x7f800000u);
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            frag_t fx;
#pragma unroll
            for (int j = 0; j < 8; ++j) fx[j] = b.x[j][f];
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                if (q == 1 && bad)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!isfinite((float)fx[j])) fx[j] = (T)0.f;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) mma32(b.v[rt][q], fx, acc[rt][f]);
            }
        }
    };
    // (n is whole pieces: every wave has n / 64 steps.  Requests beyond the end repeat the last step's rows: a branch around them would make the
    // compiler wait for everything in flight at its join)
    const int ns = n >> 6, last = (ns - 1) * 64 + wave * 16;
    Step b[PF];
#pragma unroll
    for (int i = 0; i < PF; ++i) load(min(wave * 16 + 64 * i, last), b[i]);
    int k = 0;
    for (; k + PF <= ns; k += PF) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int s = wave * 16 + 64 * (k + i);
            use(s, b[i]);
            load(min(s + 64 * PF, last), b[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < PF - 1; ++i)
        if (k + i < ns) use(wave * 16 + 64 * (k + i), b[i]);
    for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (wave == w) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    f32x4* d = reinterpret_cast<f32x4*>(red) + (rt * 16 + q) * 64 + lane;
                    const f32x4 v = {acc[rt][0][q], acc[rt][1][q], acc[rt][2][q], acc[rt][3][q]};
                    *d = w == 0 ? v : *d + v;
                }
        }
    }
    __syncthreads();
    if (!cin) return;
    float* out = p.ws + (int64_t)blockIdx.y * p.R * p.C + c;
#pragma unroll
    for (int i = 0; i < RT * 4; ++i) {
        const int k = i * 4 + wave, rt = k >> 4, q = k & 15;
        const int r = r0 + rt * 32 + (q & 3) + 8 * (q >> 2) + 4 * hi;
        if (r < p.R) store4(out + (int64_t)r * p.C, reinterpret_cast<const f32x4*>(red)[k * 64 + lane]);
    }
}

// out[g] = sum of the partial products of g's chunks, in chunk order (no atomics: the same bits every time); 16 ranks x 16 columns a workgroup,
// one output a thread: at one adapter of rank 16 and 1536 channels that is still 96 workgroups
template <typename T>
__global__ __launch_bounds__(256) void adapter_grad_join_kernel(GradArgs p) {
    const int t = threadIdx.x, g = blockIdx.z;
    // partial sums are read along the columns; a transposed output is written along the ranks
    const int cl = t & 15, rl = t >> 4;
    const int c = blockIdx.x * 16 + cl, r = blockIdx.y * 16 + rl;
    const int i0 = g < p.n_adapters ? p.chunk_off[g] : 0, i1 = g < p.n_adapters ? p.chunk_off[g + 1] : 0;
    float v = 0.f;
    if (c < p.C) {
        const float* w = p.ws + (int64_t)r * p.C + c;
        const int64_t st = (int64_t)p.R * p.C;
        int i = i0;
        for (; i + 8 <= i1; i += 8) {
            float b[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) b[k] = w[(i + k) * st];
#pragma unroll
            for (int k = 0; k < 8; ++k) v += b[k];
        }
        for (; i < i1; ++i) v += w[i * st];
    }
    if (!p.transposed) {
        if (c < p.C && r < p.rank) ((T*)p.out)[((int64_t)g * p.rank + r) * p.C + c] = (T)v;
        return;
    }
    __shared__ float tile[16][17];
    tile[cl][rl] = v;
    __syncthreads();
    const int c2 = blockIdx.x * 16 + rl, r2 = blockIdx.y * 16 + cl;
    if (c2 < p.C && r2 < p.rank) ((T*)p.out)[((int64_t)g * p.C + c2) * p.rank + r2] = (T)tile[rl][cl];
}

bool dt_ok(int dt) { return dt == M4D_BF16 || dt == M4D_F32; }

int cus() {
    static std::atomic<int> n[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) { (void)hipGetLastError(); return 256; }
    if (dev < 0 || dev >= 64) return 256;
    int v = n[dev].load(std::memory_order_relaxed);
    if (v == 0) {
        if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) { (void)hipGetLastError(); v = 256; }
        n[dev].store(v, std::memory_order_relaxed);
    }
    return v;
}

enum { GEMV16 = 0, TILE_64x64, TILE_64x128, TILE_128x128, TILE_256x128, WIDE_256x256, TILE_128x192 };
struct Choice { int kind, S; int64_t head; };      // head rows on the 256 x 256 kernel, the others on `kind` in S slices of K

double wide_round_us(int64_t K, double wide_ad) { return (double)(K / 64) * 1.03 + 10.0 + wide_ad; }
// Which kernel, and into how many slices of K: the least estimated time.  A CU runs its workgroups in rounds; a round costs a fixed part (filling
// the ring, epilogue) and c per 128-byte K tile.  c is what the tile stages from L2 at the 55 - 64 bytes/ns that a CU's K loop gets (fp32: the
// MFMA rate), so larger tiles are cheaper per product and smaller ones waste less of a round; slices pay for writing and joining float32 partial
// tiles.  Measured c (us, bf16 / fp32): 64 x 64 0.30 / 0.70 alone on a CU and 0.42 / 1.25 as one of two, 64 x 128 0.36 / 1.16, 128 x 128
// 0.55 / 2.1, 128 x 192 0.66 / -, 256 x 128 0.78 / 4.0, 256 x 256 (gemm_wide.h) 1.03.  These are of runs too short for the board's power limit: many
// rounds take longer than they say, whichever the tile (256 x 256, 21840 x 5120 x 5120: 650 us by them, 870 - 990 measured), and there the 256 x 256 tiles
// are ahead by a quarter.  Against every kind and number of slices (profiles/adapters_gemm_sweep.log): within 8 % of the best at 33 bf16 and 5 % at 11 float32
// shapes, e.g. 64 x 5120 x 4096 64 x 64 in 3 slices, 986 x 5120 x 4096 128 x 192 whole (63 us; 256 x 128 74).
Choice choose_whole(bool bf16, int64_t M, int64_t N, int64_t K, bool wide_ok, double wide_ad, int ncu, double& t_best) {
    t_best = 1e30;
#ifdef M4D_ABLATIONS
    { const char* v = getenv("M4D_ADAPTER_GEMM"); if (v) { const int c = atoi(v); if (c / 100 != WIDE_256x256 || wide_ok) return Choice{c / 100, c % 100 ? c % 100 : 1, 0}; } }
#endif
    const double es = bf16 ? 2 : 4, wbytes = (double)N * K * es;
    const int64_t nk = (int64_t)((K * es + ROWB - 1) / ROWB);
    Choice best{TILE_64x64, 1, 0};
    auto offer = [&](double t, int kind, int S) { if (t < t_best) { t_best = t; best = Choice{kind, S, 0}; } };
    if (M <= 16) offer(4.0 + wbytes * (1.0 + M / 24.0) / 6.0e6, GEMV16, 1);
    if (wide_ok) {
        const int64_t tiles = ((M + 255) / 256) * ((N + 255) / 256);
        offer((double)((tiles + ncu - 1) / ncu) * wide_round_us(K, wide_ad), WIDE_256x256, 1);
    }
    static const struct { int kind, bm, bn, occ; double c[2][2], fix; } cfg[5] = {
        {TILE_64x64, 64, 64, 2, {{0.30, 0.42}, {0.70, 1.25}}, 4.0}, {TILE_64x128, 64, 128, 1, {{0.36, 0.36}, {1.16, 1.16}}, 4.0},
        {TILE_128x128, 128, 128, 1, {{0.55, 0.55}, {2.1, 2.1}}, 5.0}, {TILE_256x128, 256, 128, 1, {{0.78, 0.78}, {4.0, 4.0}}, 7.0},
        {TILE_128x192, 128, 192, 1, {{0.66, 0.66}, {1e6, 1e6}}, 6.0}};      // (bf16 only)
    for (const auto& f : cfg) {
        const int64_t tiles = ((M + f.bm - 1) / f.bm) * ((N + f.bn - 1) / f.bn);
        for (int S = 1; S <= 16; ++S) {
            const int64_t per = (nk + S - 1) / S;
            if (S > 1 && (per < 4 || (nk + per - 1) / per != S || tiles * S > 4 * ncu || (double)S * M * N > 6.4e7)) continue;      // (at most 256 MB of slices)
            const int64_t blocks = tiles * S, rounds = (blocks + (int64_t)ncu * f.occ - 1) / ((int64_t)ncu * f.occ);
            const int shared = blocks > ncu && f.occ > 1;
            double t = rounds * (per * f.c[bf16 ? 0 : 1][shared] + f.fix);
            const double floor = wbytes / 6.0e6;
            if (t < floor) t = floor;
            if (S > 1) t += 4.5 + (double)M * N * (8.0 * S + es) / 7.0e6;
            offer(t, f.kind, S);
        }
    }
    return best;
}
// The 256 x 256 kernel's last round may leave most CUs idle (11776 x 1536 x 8960: 276 tiles on 256 CUs).  Whole rounds of it for the rows in
// front and the remaining rows on whatever is fastest for them, 8 us for one more launch: 11776 x 1536 x 8960 392 us -> 338, 21840 x 1536 x 1536
// 130 -> 112, 3584 x 5120 x 5120 217 -> 184; 4400 x 4100 x 1024 70 -> 72, and nothing (under 2 % by the estimate) at many rounds.
Choice choose(bool bf16, int64_t M, int64_t N, int64_t K, bool wide_ok, bool split_ok, double wide_ad, int ncu) {
    double t;
    Choice best = choose_whole(bf16, M, N, K, wide_ok, wide_ad, ncu, t);
    const int64_t tn = (N + 255) / 256, rounds = ((M + 255) / 256) * tn / ncu, head = rounds * ncu / tn * 256;
    if (wide_ok && split_ok && head > 0 && head < M) {
        double t2;
        Choice rest = choose_whole(bf16, M - head, N, K, false, wide_ad, ncu, t2);
        if (rounds * wide_round_us(K, wide_ad) + t2 + 8.0 < 0.98 * t) { best = rest; best.head = head; }
    }
    return best;
}

}  // namespace

#define PLAN_OK(name)                                                                                                          \
    M4D_CHECK_ARG(dt_ok(dt), name ": bad dtype %d", (int)dt);                                                                   \
    M4D_CHECK_ARG(plan && plan->rows > 0 && plan->rows < (1ll << 31) && plan->n_pieces >= 0 && plan->n_pieces < (1 << 25), name ": bad plan"); \
    M4D_CHECK_ARG(R > 0 && R % 16 == 0 && R <= 512, name ": padded rank R=%d must be a multiple of 16, at most 512", R);          \
    const int es = dt == M4D_BF16 ? 2 : 4

extern "C" int64_t m4d_adapter_down_elems(int G, int R, int64_t K) { return (int64_t)G * ((K + 63) / 64) * ((R + 31) / 32) * 2048; }

extern "C" int m4d_adapter_pack(m4d_dtype dt, const void* a, const void* b, int G, int rank, int64_t K, int64_t N, int R, void* a_down, void* b_up,
                                void* b_down, void* a_up, m4d_stream stream) {
    M4D_CHECK_ARG(dt_ok(dt), "adapter_pack: bad dtype %d", (int)dt);
    M4D_CHECK_ARG(a && b && G > 0 && rank > 0 && R >= rank && R % 16 == 0 && R <= 512 && K > 0 && N > 0 && K < (1 << 30) && N < (1 << 30),
                  "adapter_pack: bad adapters (G=%d rank=%d R=%d K=%lld N=%lld)", G, rank, R, (long long)K, (long long)N);
    M4D_CHECK_ARG(((uintptr_t)a_down % 16) == 0 && ((uintptr_t)b_up % 16) == 0 && ((uintptr_t)b_down % 16) == 0 && ((uintptr_t)a_up % 16) == 0,
                  "adapter_pack: pointers must be 16-byte aligned");
    PackArgs p{a, b, a_down, b_up, b_down, a_up, G, rank, (int)K, (int)N, R};
    const int64_t most = (int64_t)G * (R + 31) * ((K > N ? K : N) + 63);
    const int64_t nblk = (most + 1023) / 1024;
    dim3 grid((unsigned)(nblk < 1024 ? nblk : 1024), b_down || a_up ? 4 : 2);
    if (dt == M4D_BF16) hipLaunchKernelGGL(adapter_pack_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(adapter_pack_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, p);
    M4D_CHECK_LAUNCH("adapter_pack");
    return 0;
}

template <typename T, int RT, bool QUANT, bool DEEP>
static int launch_down_q(const DownArgs& p, hipStream_t st) {
    constexpr int LDS = DownShape<T, RT, DEEP>::LDS;
    static PerDeviceOnce configured;
    if (configured.pending()) {
        if (hipFuncSetAttribute((const void*)adapter_down_kernel<T, RT, QUANT, DEEP>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) {
            (void)hipGetLastError();
            m4d_set_error("adapter_down: cannot enable %d bytes of LDS", LDS);
            return -3;
        }
        configured.mark();
    }
    const int ny = ((p.R + 31) / 32 + RT - 1) / RT;
    hipLaunchKernelGGL((adapter_down_kernel<T, RT, QUANT, DEEP>), dim3((unsigned)((p.n_pieces + 7) / 8 * 8 * ny), (unsigned)p.KS), dim3(QUANT ? 512 : 256), LDS, st, p);
    M4D_CHECK_LAUNCH("adapter_down");
    if (p.part) {
        hipLaunchKernelGGL(adapter_down_join_kernel<T>, dim3((unsigned)p.n_pieces, (unsigned)((p.R + 31) / 32 * 2)), dim3(256), 0, st, p);
        M4D_CHECK_LAUNCH("adapter_down(join)");
    }
    return 0;
}
template <typename T, int RT>
static int launch_down(const DownArgs& p, hipStream_t st) {
    const int64_t blocks = (int64_t)p.n_pieces * p.KS * (((p.R + 31) / 32 + RT - 1) / RT);
    if (blocks <= cus()) return p.codes ? launch_down_q<T, RT, true, true>(p, st) : launch_down_q<T, RT, false, true>(p, st);
    return p.codes ? launch_down_q<T, RT, true, false>(p, st) : launch_down_q<T, RT, false, false>(p, st);
}

// K slices of a down projection: the least estimated time.  A piece's K loop is serial, 0.5 us a chunk of 64 channels, and a CU works through the
// pieces it is dealt; slices shorten the loop where pieces are few (16 pieces, K = 4096: whole 32 us, in eight slices and joined 10) and even out
// the CUs' shares where they are not much more than CUs (341 on 256); writing and joining the float32 sums costs 4 us and their bytes.
static int down_slices(int n_pieces, int64_t K, int R) {
    const int nc = (int)((K + 63) / 64), ncu = cus();
#ifdef M4D_ABLATIONS
    { const char* v = getenv("M4D_ADAPTER_KS"); if (v && atoi(v) > 0) { const int per = (nc + atoi(v) - 1) / atoi(v); return (nc + per - 1) / per; } }
#endif
    int best = 1;
    double t_best = 1e30;
    for (int ks = 1; ks <= 16 && (ks == 1 || nc / ks >= 8); ++ks) {
        const int per = (nc + ks - 1) / ks;
        if ((nc + per - 1) / per != ks) continue;                  // (no empty slices)
        const double rounds = (double)(((int64_t)n_pieces * ks + ncu - 1) / ncu);
        double t = rounds * (per * 0.47 + 2.0);
        if (ks > 1) t += 4.0 + (double)ks * n_pieces * ((R + 31) / 32) * 32 * PIECE * 8 / 4.5e6;
        if (t < t_best) { t_best = t; best = ks; }
    }
    return best;
}
// at most 16 rows, and only u wanted (serving single tokens): adapter_down16_kernel
static bool down_few(const m4d_adapter_plan* plan, const void* ut, const void* codes) { return plan->rows <= 16 && !ut && !codes; }

extern "C" int64_t m4d_adapter_down_workspace(const m4d_adapter_plan* plan, int64_t K, int R, int slots) {
    if (!plan || K <= 0 || R <= 0 || (plan->rows <= 16 && !slots)) return 0;
    const int ks = down_slices(plan->n_pieces, K, R);
    return ks > 1 ? (int64_t)ks * plan->n_pieces * ((R + 31) / 32 * 32) * PIECE : 0;
}

static int down(m4d_dtype dt, const void* x, int64_t ldx, const void* a_down, const float* scale, const m4d_adapter_plan* plan, void* u, int split,
                void* ut, int8_t* codes, uint8_t* exps, int64_t K, int R, float* ws, int64_t ws_floats, m4d_stream stream) {
    PLAN_OK("adapter_down");
    M4D_CHECK_ARG(x && a_down && scale && (u || ut) && (codes == nullptr) == (exps == nullptr), "adapter_down: null pointer");
    M4D_CHECK_ARG(K > 0 && K < (1 << 30) && (K * es) % 16 == 0 && (ldx * es) % 16 == 0 && (plan->rows == 1 || ldx >= K),
                  "adapter_down: rows of K=%lld elements (row stride %lld) must be multiples of 16 bytes", (long long)K, (long long)ldx);
    M4D_CHECK_ARG(((uintptr_t)x % 16) == 0 && ((uintptr_t)a_down % 16) == 0 && ((uintptr_t)u % 16) == 0 && ((uintptr_t)ut % 16) == 0 &&
                  ((uintptr_t)codes % 16) == 0 && ((uintptr_t)exps % 4) == 0 && ((uintptr_t)ws % 16) == 0, "adapter_down: pointers must be 16-byte aligned");
    if (plan->n_pieces == 0) return 0;
    M4D_CHECK_ARG(plan->slot_row && plan->piece_adapter, "adapter_down: bad plan");
    const int ks = down_slices(plan->n_pieces, K, R);
    if (down_few(plan, ut, codes)) {
        M4D_CHECK_ARG(plan->row_adapter && plan->tiles[0] && plan->n_listed > 0 && plan->n_listed <= 16, "adapter_down: bad plan");
        DownArgs p{x, a_down, scale, u, nullptr, nullptr, nullptr, nullptr, nullptr, ldx, (int)K, R, plan->n_pieces, 1, nullptr, split};
        dim3 grid((unsigned)plan->n_listed, (unsigned)(R / 16)), block(64 * SKINNY_WAVES);
        if (dt == M4D_BF16) hipLaunchKernelGGL(adapter_down16_kernel<bf16_t>, grid, block, 0, (hipStream_t)stream, p, plan->row_adapter, plan->tiles[0], (int)plan->rows);
        else hipLaunchKernelGGL(adapter_down16_kernel<float>, grid, block, 0, (hipStream_t)stream, p, plan->row_adapter, plan->tiles[0], (int)plan->rows);
        M4D_CHECK_LAUNCH("adapter_down");
        return 0;
    }
    const int64_t need = m4d_adapter_down_workspace(plan, K, R, 1);
    M4D_CHECK_ARG(need == 0 || (ws && ws_floats >= need), "adapter_down: workspace of %lld floats needed", (long long)need);
    DownArgs p{x, a_down, scale, u, ut, codes, exps, plan->slot_row, plan->piece_adapter, ldx, (int)K, R,
               plan->n_pieces, ks, ks > 1 ? ws : nullptr, split};
    hipStream_t st = (hipStream_t)stream;
    if (dt == M4D_BF16) return R <= 32 ? launch_down<bf16_t, 1>(p, st) : R <= 64 ? launch_down<bf16_t, 2>(p, st) : launch_down<bf16_t, 4>(p, st);
    return R <= 32 ? launch_down<float, 1>(p, st) : launch_down<float, 2>(p, st);
}
extern "C" int m4d_adapter_down(m4d_dtype dt, const void* x, int64_t ldx, const void* a_down, const float* scale, const m4d_adapter_plan* plan,
                                void* u, void* ut, int8_t* codes, uint8_t* exps, int64_t K, int R, float* ws, int64_t ws_floats, m4d_stream stream) {
    return down(dt, x, ldx, a_down, scale, plan, u, 0, ut, codes, exps, K, R, ws, ws_floats, stream);
}

template <typename T, int MI, int NI, int WM, int WN>
static int launch_gemm(AdGemmArgs& p, hipStream_t st) {
    typedef AdGemmShape<T, MI, NI, WM, WN> Sh;
    static PerDeviceOnce configured;
    if (configured.pending()) {
        if (hipFuncSetAttribute((const void*)adapter_gemm_kernel<T, MI, NI, WM, WN>, hipFuncAttributeMaxDynamicSharedMemorySize, Sh::LDS) != hipSuccess) {
            (void)hipGetLastError();
            m4d_set_error("linear_adapters: cannot enable %d bytes of LDS", Sh::LDS);
            return -3;
        }
        configured.mark();
    }
    const int64_t tm = (p.M + Sh::BM - 1) / Sh::BM, tn = (p.N + Sh::BN - 1) / Sh::BN;
    M4D_CHECK_ARG(tm * tn < (1ll << 31), "linear_adapters: too many tiles");
    p.tiles_m = (int)tm; p.tiles_n = (int)tn;
    hipLaunchKernelGGL((adapter_gemm_kernel<T, MI, NI, WM, WN>), dim3((unsigned)(tm * tn), (unsigned)p.S), dim3(Sh::THREADS), Sh::LDS, st, p);
    M4D_CHECK_LAUNCH("linear_adapters");
    if (p.S > 1) {
        const int64_t nblk = (p.M * (p.N / 4) + 255) / 256;
        hipLaunchKernelGGL(adapter_gemm_join_kernel<T>, dim3((unsigned)(nblk < 4096 ? nblk : 4096)), dim3(256), 0, st, p);
        M4D_CHECK_LAUNCH("linear_adapters(join)");
    }
    return 0;
}

static bool wide_shape(m4d_dtype dt, int64_t M, int64_t N, int64_t K) { return dt == M4D_BF16 && K % 64 == 0 && M >= 512 && N >= 512; }
// what the adapters of a 256 x 256 tile add to its time, us (its direct loads take 32 consecutive rows each: it does not see row_order).  Measured
// per adapter: rank 16 0.7, rank 32 1.5, rank 64 3.0, rank 128 5.5.  The other tiles take interleaved rows in order and have one or two adapters each.
static double wide_adapters_us(const m4d_adapter_plan* plan, int R) { return plan->row_order ? 0.045 * R * plan->n_wide / (double)((plan->rows + 255) / 256) : 0.0; }

static int u_parts(m4d_dtype dt) { return dt == M4D_BF16 ? Parts<bf16_t>::N : Parts<float>::N; }
// the down projection's slices and the GEMM's run one after the other: one workspace, the larger of the two
extern "C" int64_t m4d_linear_adapters_workspace(m4d_dtype dt, const m4d_adapter_plan* plan, int64_t N, int64_t K, int R, int slots) {
    if (!plan || plan->rows <= 0 || N <= 0 || K <= 0) return 0;
    const int64_t M = plan->rows;
    int64_t most = m4d_adapter_down_workspace(plan, K, R, slots);      // (whether the wide kernel can run depends on the output's alignment too: room for either choice)
    for (int w = 0; w < 2; ++w) {
        const Choice c = choose(dt == M4D_BF16, M, N, K, w && wide_shape(dt, M, N, K), !plan->row_order, wide_adapters_us(plan, R), cus());
        if (c.S > 1 && c.S * (M - c.head) * N > most) most = c.S * (M - c.head) * N;
    }
    return most;
}

extern "C" int m4d_linear_adapters(m4d_dtype dt, const void* x, int64_t ldx, const void* W, int64_t ldw, const void* bias, const void* a_down,
                                   const float* scale, const void* b_up, const m4d_adapter_plan* plan, void* u, void* ut, int8_t* codes,
                                   uint8_t* exps, void* out, int64_t ldo, int64_t N, int64_t K, int R, float* ws, int64_t ws_floats, m4d_stream stream) {
    PLAN_OK("linear_adapters");
    const int64_t M = plan->rows;
    M4D_CHECK_ARG(x && W && out && a_down && u && b_up, "linear_adapters: null pointer");
    M4D_CHECK_ARG(N > 0 && K > 0 && K < (1 << 30) && N < (1ll << 31) && (K * es) % 16 == 0, "linear_adapters: K*sizeof(T) must be a multiple of 16 (K=%lld)", (long long)K);
    M4D_CHECK_ARG(N % 4 == 0 && ldo % 4 == 0 && (M == 1 || ldo >= N), "linear_adapters: N and the output's row stride must be multiples of 4 (N=%lld ldo=%lld)",
                  (long long)N, (long long)ldo);
    M4D_CHECK_ARG((ldx * es) % 16 == 0 && (ldw * es) % 16 == 0 && (M == 1 || ldx >= K) && ldw >= K, "linear_adapters: rows must be 16-byte aligned");
    M4D_CHECK_ARG(((uintptr_t)x % 16) == 0 && ((uintptr_t)W % 16) == 0 && ((uintptr_t)out % 16) == 0 && ((uintptr_t)u % 16) == 0 && ((uintptr_t)b_up % 16) == 0,
                  "linear_adapters: pointers must be 16-byte aligned");
    M4D_CHECK_ARG(((uintptr_t)bias % (4 * es)) == 0, "linear_adapters: bias must be aligned to four elements");
    M4D_CHECK_ARG(plan->row_adapter && plan->tiles_off[0] && plan->tiles_off[1] && plan->tiles_off[2] && plan->tiles[0] && plan->tiles[1] && plan->tiles[2] && plan->tile_one,
                  "linear_adapters: bad plan");
    const bool bf16 = dt == M4D_BF16;
    // (the wide kernel's lanes hold the offsets of 32 rows in 32 bits)
    const bool wide_ok = wide_shape(dt, M, N, K) && ldo % 8 == 0 && ((uintptr_t)out % 32) == 0 && ldx <= (1 << 25) && ldw <= (1 << 25);
    const Choice c = choose(bf16, M, N, K, wide_ok, !plan->row_order, wide_adapters_us(plan, R), cus());
    M4D_CHECK_ARG(c.S == 1 || (ws && ws_floats >= c.S * (M - c.head) * N && ((uintptr_t)ws % 16) == 0), "linear_adapters: workspace of %lld floats needed",
                  (long long)(c.S * (M - c.head) * N));
    const int rc = down(dt, x, ldx, a_down, scale, plan, u, 1, ut, codes, exps, K, R, ws, ws_floats, stream);
    if (rc != 0) return rc;
    AdGemmArgs p{};
    p.A = x; p.W = W; p.bias = bias; p.out = out; p.lda = ldx; p.ldw = ldw; p.ldc = ldo; p.M = M; p.N = N; p.K = K;
    p.rows_per_sample = M; p.epilogue = M4D_EPI_STORE;
    p.u = u; p.up = b_up; p.row_adapter = plan->row_adapter; p.order = plan->row_order; p.R = R; p.S = c.S; p.ws = ws;
    hipStream_t st = (hipStream_t)stream;
    const int64_t rows_wide = c.kind == WIDE_256x256 ? M : c.head;
    if (rows_wide > 0) {
        p.M = rows_wide;
        p.tile_off = plan->tiles_off[3]; p.tile_list = plan->tiles[3]; p.tile_one = plan->tile_one;
        p.tiles_m = (int)((rows_wide + 255) / 256); p.tiles_n = (int)((N + 255) / 256);
        M4D_CHECK_ARG((int64_t)p.tiles_m * p.tiles_n < (1ll << 31), "linear_adapters: too many tiles");
        m4d_count_launch(M4D_KC_GEMM_WIDE);
        if (m4d_launch_gemm_wide_adapters(static_cast<const GemmAdArgs*>(&p), (unsigned)(p.tiles_m * p.tiles_n), st) != 0) {
            (void)hipGetLastError();
            m4d_set_error("linear_adapters: cannot enable 128 KiB LDS");
            return -3;
        }
        M4D_CHECK_LAUNCH("linear_adapters");
        if (rows_wide == M) return 0;
        // the rows behind it (whole tiles of 256 in front, so every tile table goes on at its own row)
        p.A = (const char*)x + rows_wide * ldx * es; p.u = (const char*)u + rows_wide * R * u_parts(dt) * es; p.out = (char*)out + rows_wide * ldo * es;
        p.row_adapter = plan->row_adapter + rows_wide; p.M = p.rows_per_sample = M - rows_wide;
    }
    const int tl = c.kind == GEMV16 || c.kind == TILE_64x64 || c.kind == TILE_64x128 ? 0 : c.kind == TILE_128x128 || c.kind == TILE_128x192 ? 1 : 2;      // tile heights 64, 128, 256
    p.tile_off = plan->tiles_off[tl] + (rows_wide >> (6 + tl)); p.tile_list = plan->tiles[tl];
    m4d_count_launch(M4D_KC_GEMM_GENERIC);
    switch (c.kind) {
        case GEMV16: {
            M4D_CHECK_ARG(p.M <= 16, "linear_adapters: too many rows");
            dim3 grid((unsigned)((N + 15) / 16)), block(64 * SKINNY_WAVES);
            if (bf16) hipLaunchKernelGGL(adapter_gemv_kernel<bf16_t>, grid, block, 0, st, p);
            else hipLaunchKernelGGL(adapter_gemv_kernel<float>, grid, block, 0, st, p);
            M4D_CHECK_LAUNCH("linear_adapters");
            return 0;
        }
        case TILE_64x64: return bf16 ? launch_gemm<bf16_t, 1, 1, 2, 2>(p, st) : launch_gemm<float, 1, 1, 2, 2>(p, st);
        case TILE_64x128: return bf16 ? launch_gemm<bf16_t, 1, 1, 2, 4>(p, st) : launch_gemm<float, 1, 2, 2, 2>(p, st);
        case TILE_128x128: return bf16 ? launch_gemm<bf16_t, 1, 2, 4, 2>(p, st) : launch_gemm<float, 2, 2, 2, 2>(p, st);
        case TILE_128x192: return launch_gemm<bf16_t, 1, 3, 4, 2>(p, st);
        default: return bf16 ? launch_gemm<bf16_t, 2, 2, 4, 2>(p, st) : launch_gemm<float, 4, 2, 2, 2>(p, st);
    }
}

// the coarsest chunks that still give three workgroups for two CUs (two fit on one; coarser: fewer partial sums to write and join)
static int chunk_level(const m4d_adapter_plan* plan, int64_t C, int R) {
    const int64_t blocks = ((C + 127) / 128) * (R <= 64 ? 1 : (R + 63) / 64);
    for (int l = 0; l < 3; ++l)
        if (2 * blocks * plan->n_chunks[l] >= 3 * cus()) return l;
    return 3;
}

extern "C" int64_t m4d_adapter_grad_workspace(const m4d_adapter_plan* plan, int64_t C, int R) {
    return plan && C > 0 && R > 0 ? (int64_t)plan->n_chunks[chunk_level(plan, C, R)] * R * C : 0;
}

extern "C" int m4d_adapter_grad(m4d_dtype dt, const void* vt, const void* x, int64_t ldx, const int8_t* codes, const uint8_t* exps,
                                const m4d_adapter_plan* plan, float* ws, int64_t ws_floats, void* out, int transposed, int G, int rank, int64_t C,
                                int R, m4d_stream stream) {
    PLAN_OK("adapter_grad");
    M4D_CHECK_ARG(out && G > 0 && G <= 65535 && rank > 0 && rank <= R, "adapter_grad: bad adapters (G=%d rank=%d R=%d)", G, rank, R);
    M4D_CHECK_ARG(C > 0 && C < (1 << 30) && C % 4 == 0, "adapter_grad: C=%lld must be a multiple of 4", (long long)C);
    const int lv = chunk_level(plan, C, R), nch = plan->n_chunks[lv];
    M4D_CHECK_ARG(plan->n_adapters <= G && nch <= 65535, "adapter_grad: the plan names adapter %d of %d, in %d chunks", plan->n_adapters - 1, G, nch);
    hipStream_t st = (hipStream_t)stream;
    GradArgs p{vt, x, codes, exps, ws, out, plan->slot_row, plan->chunks[lv], plan->chunk_off[lv], ldx,
               (int)C, R, rank, plan->n_adapters, transposed};
    if (nch > 0) {
        M4D_CHECK_ARG(vt && ws && ws_floats >= (int64_t)nch * R * C, "adapter_grad: workspace of %lld floats needed", (long long)nch * R * C);
        M4D_CHECK_ARG((x != nullptr) != (codes != nullptr) && (codes == nullptr) == (exps == nullptr), "adapter_grad: either x or its codes");
        M4D_CHECK_ARG(!x || (ldx * es) % 16 == 0, "adapter_grad: rows must be 16-byte aligned");
        M4D_CHECK_ARG(((uintptr_t)vt % 16) == 0 && ((uintptr_t)x % 16) == 0 && ((uintptr_t)codes % 16) == 0 && ((uintptr_t)ws % 16) == 0,
                      "adapter_grad: pointers must be 16-byte aligned");
        M4D_CHECK_ARG(plan->slot_row && p.chunks && p.chunk_off, "adapter_grad: bad plan");
        const int rt = R <= 32 ? 1 : 2;
        dim3 grid((unsigned)((C + 127) / 128), (unsigned)nch, (unsigned)((R + rt * 32 - 1) / (rt * 32)));
#define GRAD(T, CD)                                                                                         \
    do {                                                                                                    \
        if (rt == 1) hipLaunchKernelGGL((adapter_grad_kernel<T, CD, 1>), grid, dim3(256), 0, st, p);         \
        else hipLaunchKernelGGL((adapter_grad_kernel<T, CD, 2>), grid, dim3(256), 0, st, p);                 \
    } while (0)
        if (dt == M4D_BF16) { if (codes) GRAD(bf16_t, true); else GRAD(bf16_t, false); }
        else { if (codes) GRAD(float, true); else GRAD(float, false); }
#undef GRAD
        M4D_CHECK_LAUNCH("adapter_grad");
    }
    dim3 jg((unsigned)((C + 15) / 16), (unsigned)((rank + 15) / 16), (unsigned)G);
    if (dt == M4D_BF16) hipLaunchKernelGGL(adapter_grad_join_kernel<bf16_t>, jg, dim3(256), 0, st, p);
    else hipLaunchKernelGGL(adapter_grad_join_kernel<float>, jg, dim3(256), 0, st, p);
    M4D_CHECK_LAUNCH("adapter_grad(join)");
    return 0;
}

// The whole backward of a frozen projection with adapters in one call: W^T, v = s dy B (with its slots), dx = dy W + v A, dA, dB.  Workspace: W^T, v,
// its slots, then the largest of what the passes need, which run one after the other.
namespace {
struct BwdSpace { int64_t wt, v, vt, rest, total; };
int64_t up64(int64_t n) { return (n + 63) / 64 * 64; }
BwdSpace bwd_space(m4d_dtype dt, const m4d_adapter_plan* plan, int64_t N, int64_t K, int R, bool dx, bool da, bool db) {
    const int64_t per = dt == M4D_BF16 ? 2 : 1;                  // elements of T in a float
    BwdSpace b{};
    int64_t at = 0;
    b.wt = at; if (dx) at += up64((K * N + per - 1) / per);
    b.v = at; if (dx) at += up64((plan->rows * R * u_parts(dt) + per - 1) / per);
    b.vt = at; if (da) at += up64((int64_t)plan->n_pieces * 4 * ((R + 31) / 32) * 512 * u_parts(dt) / per);
    b.rest = at;
    int64_t most = 0;
    auto take = [&](int64_t n) { if (n > most) most = n; };
    if (dx) take(m4d_linear_adapters_workspace(dt, plan, K, N, R, da));
    else if (da) take(m4d_adapter_down_workspace(plan, N, R, 1));
    if (da) take(m4d_adapter_grad_workspace(plan, K, R));
    if (db) take(m4d_adapter_grad_workspace(plan, N, R));
    b.total = at + most;
    return b;
}
}  // namespace

extern "C" int64_t m4d_linear_adapters_bwd_workspace(m4d_dtype dt, const m4d_adapter_plan* plan, int64_t N, int64_t K, int R, int need_dx, int need_da,
                                                     int need_db) {
    if (!plan || plan->rows <= 0 || N <= 0 || K <= 0 || R <= 0) return 0;
    return bwd_space(dt, plan, N, K, R, need_dx, need_da, need_db).total;
}

extern "C" int m4d_linear_adapters_bwd(m4d_dtype dt, const void* dy, int64_t ldy, const void* W, int64_t ldw, const void* b_down, const float* scale,
                                       const void* a_up, const m4d_adapter_plan* plan, const void* x, int64_t ldx, const int8_t* codes,
                                       const uint8_t* exps, const void* ut, void* dx, void* da, void* db, int G, int rank, int64_t N, int64_t K, int R,
                                       float* ws, int64_t ws_floats, m4d_stream stream) {
    PLAN_OK("linear_adapters_bwd");
    M4D_CHECK_ARG(dx || da || db, "linear_adapters_bwd: nothing to compute");
    M4D_CHECK_ARG((N * es) % 16 == 0, "linear_adapters_bwd: rows of dy (N=%lld) must be whole 16-byte chunks", (long long)N);
    const BwdSpace s = bwd_space(dt, plan, N, K, R, dx, da, db);
    M4D_CHECK_ARG(s.total == 0 || (ws && ws_floats >= s.total && ((uintptr_t)ws % 16) == 0), "linear_adapters_bwd: workspace of %lld floats needed", (long long)s.total);
    float* rest = ws + s.rest;
    const int64_t nrest = s.total - s.rest;
    int rc = 0;
    void* vt = da ? (void*)(ws + s.vt) : nullptr;
    if (dx) {
        rc = m4d_transpose(dt, W, ldw, ws + s.wt, N, N, K, stream);
        if (rc == 0) {
            if (plan->n_pieces == 0) rc = m4d_gemm_bt(dt, dy, ldy, ws + s.wt, N, nullptr, 0, dx, K, plan->rows, K, N, M4D_EPI_STORE, nullptr, 0, 0, stream);
            else rc = m4d_linear_adapters(dt, dy, ldy, ws + s.wt, N, nullptr, b_down, scale, a_up, plan, ws + s.v, vt, nullptr, nullptr, dx, K, K, N, R, rest, nrest, stream);
        }
    } else if (da) rc = m4d_adapter_down(dt, dy, ldy, b_down, scale, plan, nullptr, vt, nullptr, nullptr, N, R, rest, nrest, stream);
    if (rc == 0 && da) rc = m4d_adapter_grad(dt, vt, x, ldx, codes, exps, plan, rest, nrest, da, 0, G, rank, K, R, stream);
    if (rc == 0 && db) rc = m4d_adapter_grad(dt, ut, dy, ldy, nullptr, nullptr, plan, rest, nrest, db, 1, G, rank, N, R, stream);
    return rc;
}

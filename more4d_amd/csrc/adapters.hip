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
// u is written twice: [row][R], the GEMM's operand, and [R][slot], the operand of the row contraction (its 8 consecutive slots of one
// rank are one 16-byte load in the MFMA layout; pad slots hold zero).  u and v are rounded to T like every other operand of an MFMA here: the
// error this puts on an output is the one its own final rounding has, or less.
#include "gemm_common.h"

extern "C" __attribute__((visibility("hidden"))) void m4d_launch_gemm_generic_adapters(const void* args, int bf16, unsigned nwg, hipStream_t st);
extern "C" __attribute__((visibility("hidden"))) int m4d_launch_gemm_wide_adapters(const void* args, unsigned nwg, hipStream_t st);

namespace {

constexpr int PIECE = 64;

struct DownArgs {
    const void* x; const void* a; const float* scale;
    void* u; void* ut;
    const int *slot_row, *piece_adapter;
    int64_t ldx, n_slots;
    int K, R;
};

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

// u of one piece: 64 slots x RT * 32 ranks, K split over the workgroup's four waves (64 elements each in turn), joined in LDS in wave order
template <typename T, int RT>
__global__ __launch_bounds__(256) void adapter_down_kernel(DownArgs p) {
    typedef typename Frag8<T>::type frag_t;
    __shared__ float red[RT * 2 * 16 * 64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 31, hi = lane >> 5;
    const int piece = blockIdx.x, r0 = blockIdx.y * (RT * 32);
    const int g = p.piece_adapter[piece];
    int row[2];
    const T* px[2];
    const T* pa[RT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        row[s] = p.slot_row[(int64_t)piece * PIECE + s * 32 + li];
        px[s] = (const T*)p.x + (int64_t)max(row[s], 0) * p.ldx;
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) pa[rt] = (const T*)p.a + ((int64_t)g * p.R + min(r0 + rt * 32 + li, p.R - 1)) * p.K;
    f32x16 acc[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[rt][s][q] = 0.f;
    for (int kc = wave * 64; kc < p.K; kc += 256) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const int k = kc + kk * 16 + hi * 8;
            frag_t fx[2], fa[RT];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                fx[s] = frag_t{};
                if (row[s] >= 0) fx[s] = load_k8<T>(px[s], k, p.K);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) fa[rt] = load_k8<T>(pa[rt], k, p.K);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int s = 0; s < 2; ++s) mma32(fa[rt], fx[s], acc[rt][s]);
        }
    }
    for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        float* d = red + ((rt * 2 + s) * 16 + q) * 64 + lane;
                        *d = w == 0 ? acc[rt][s][q] : *d + acc[rt][s][q];
                    }
        }
        __syncthreads();
    }
    const float sc = p.scale[g];
    // wave -> (rank quad q4 = wave) of every (rt, s): ranks rt*32 + q4*8 + hi*4 + [0, 4) of slot s*32 + li
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int r = r0 + rt * 32 + wave * 8 + hi * 4;
            if (r >= p.R) continue;
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = sc * red[((rt * 2 + s) * 16 + wave * 4 + e) * 64 + lane];
            const int64_t slot = (int64_t)piece * PIECE + s * 32 + li;
            if (p.u && row[s] >= 0) store4((T*)p.u + (int64_t)row[s] * p.R + r, v);
            if (p.ut) {
#pragma unroll
                for (int e = 0; e < 4; ++e) ((T*)p.ut)[(r + e) * p.n_slots + slot] = (T)(row[s] >= 0 ? v[e] : 0.f);
            }
        }
}

struct GradArgs {
    const void* vt;                 // T [R, n_slots]
    const void* x;                  // T [rows, C] (row stride ldx), or
    const int8_t* codes; const uint8_t* exps;      // its 8-bit form (csrc/act8.hip)
    float* ws;                      // [n_chunks, R, C]
    void* out;                      // T [G, rank, C], or [G, C, rank]
    const int *slot_row, *chunks, *chunk_off;
    int64_t ldx, n_slots;
    int C, R, rank, n_adapters, transposed;
};

// four consecutive columns of a row as T
template <typename T> struct Quad;
template <> struct Quad<bf16_t> { typedef bf16x4 type; };
template <> struct Quad<float> { typedef f32x4 type; };

// ws[chunk][r][c] = sum over the chunk's slots of vt[r][slot] * x[row of slot][c].  A workgroup owns 128 columns of one chunk, its four waves take
// 16 slots each in turn.  The contraction runs over ROWS, so the MFMA wants 8 rows of one column per lane: a lane loads 4 consecutive columns
// of 8 rows and regroups them in registers into 4 fragments, fragment f = column 4 * lane + f, so that no LDS transpose is needed and a lane
// ends with 4 consecutive columns of the result.
template <typename T, bool CODES, int RT>
__global__ __launch_bounds__(256) void adapter_grad_kernel(GradArgs p) {
    typedef typename Frag8<T>::type frag_t;
    typedef typename Quad<T>::type quad_t;
    __shared__ float red[RT * 4 * 16 * 64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 31, hi = lane >> 5;
    const int c = blockIdx.x * 128 + li * 4, r0 = blockIdx.z * (RT * 32);
    const int* ch = p.chunks + 3 * blockIdx.y;
    const int s0 = ch[0] * PIECE, s1 = ch[1] * PIECE;
    const bool cin = c < p.C;
    const int nb = (p.C + 31) >> 5;
    const T* pv[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) pv[rt] = (const T*)p.vt + (int64_t)min(r0 + rt * 32 + li, p.R - 1) * p.n_slots + hi * 8;
    f32x16 acc[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[rt][f][q] = 0.f;
    for (int s = s0 + wave * 16; s < s1; s += 64) {
        quad_t xr[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = p.slot_row[s + hi * 8 + j];
            xr[j] = quad_t{};
            if (row >= 0 && cin) {
                if constexpr (CODES) {
                    const int cd = *reinterpret_cast<const int*>(p.codes + ((int64_t)row * nb) * 32 + c);
                    const float step = __builtin_bit_cast(float, (unsigned)p.exps[(int64_t)row * nb + (c >> 5)] << 23);
#pragma unroll
                    for (int e = 0; e < 4; ++e) xr[j][e] = (T)((float)((cd << (24 - 8 * e)) >> 24) * step);
                } else {
                    xr[j] = *reinterpret_cast<const quad_t*>((const T*)p.x + (int64_t)row * p.ldx + c);
                }
            }
        }
        frag_t fv[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) fv[rt] = *reinterpret_cast<const frag_t*>(pv[rt] + s);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            frag_t fx;
#pragma unroll
            for (int j = 0; j < 8; ++j) fx[j] = xr[j][f];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) mma32(fv[rt], fx, acc[rt][f]);
        }
    }
    for (int w = 0; w < 4; ++w) {
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
        __syncthreads();
    }
    if (!cin) return;
    float* out = p.ws + (int64_t)blockIdx.y * p.R * p.C + c;
#pragma unroll
    for (int i = 0; i < RT * 4; ++i) {
        const int k = i * 4 + wave, rt = k >> 4, q = k & 15;
        const int r = r0 + rt * 32 + (q & 3) + 8 * (q >> 2) + 4 * hi;
        if (r < p.R) store4(out + (int64_t)r * p.C, reinterpret_cast<const f32x4*>(red)[k * 64 + lane]);
    }
}

// out[g] = sum of the partial products of g's chunks, in chunk order (no atomics: the same bits every time); 16 ranks x 64 columns a workgroup
template <typename T>
__global__ __launch_bounds__(256) void adapter_grad_join_kernel(GradArgs p) {
    __shared__ float tile[64][17];
    const int t = threadIdx.x, cl = t & 63, c = blockIdx.x * 64 + cl, r0 = blockIdx.y * 16, g = blockIdx.z;
    const int i0 = g < p.n_adapters ? p.chunk_off[g] : 0, i1 = g < p.n_adapters ? p.chunk_off[g + 1] : 0;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < p.C)
        for (int i = i0; i < i1; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += p.ws[((int64_t)i * p.R + r0 + j * 4 + (t >> 6)) * p.C + c];
    if (!p.transposed) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + j * 4 + (t >> 6);
            if (c < p.C && r < p.rank) ((T*)p.out)[((int64_t)g * p.rank + r) * p.C + c] = (T)v[j];
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[cl][j * 4 + (t >> 6)] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = j * 256 + t, cc = k >> 4, r = k & 15;
        if (blockIdx.x * 64 + cc < (unsigned)p.C && r0 + r < p.rank)
            ((T*)p.out)[((int64_t)g * p.C + blockIdx.x * 64 + cc) * p.rank + r0 + r] = (T)tile[cc][r];
    }
}

bool dt_ok(int dt) { return dt == M4D_BF16 || dt == M4D_F32; }

}  // namespace

#define PLAN_OK(name)                                                                                                          \
    M4D_CHECK_ARG(dt_ok(dt), name ": bad dtype %d", (int)dt);                                                                   \
    M4D_CHECK_ARG(plan && plan->rows > 0 && plan->rows < (1ll << 31) && plan->n_pieces >= 0 && plan->n_pieces < (1 << 25), name ": bad plan"); \
    M4D_CHECK_ARG(R > 0 && R % 16 == 0 && R <= 512, name ": padded rank R=%d must be a multiple of 16, at most 512", R);          \
    const int es = dt == M4D_BF16 ? 2 : 4

extern "C" int m4d_adapter_down(m4d_dtype dt, const void* x, int64_t ldx, const void* a, const float* scale, const m4d_adapter_plan* plan,
                                void* u, void* ut, int64_t K, int R, m4d_stream stream) {
    PLAN_OK("adapter_down");
    M4D_CHECK_ARG(x && a && scale && (u || ut), "adapter_down: null pointer");
    M4D_CHECK_ARG(K > 0 && K < (1 << 30) && (K * es) % 16 == 0 && (ldx * es) % 16 == 0 && (plan->rows == 1 || ldx >= K),
                  "adapter_down: rows of K=%lld elements (row stride %lld) must be multiples of 16 bytes", (long long)K, (long long)ldx);
    M4D_CHECK_ARG(((uintptr_t)x % 16) == 0 && ((uintptr_t)a % 16) == 0 && ((uintptr_t)u % 16) == 0 && ((uintptr_t)ut % 16) == 0,
                  "adapter_down: pointers must be 16-byte aligned");
    if (plan->n_pieces == 0) return 0;
    M4D_CHECK_ARG(plan->slot_row && plan->piece_adapter, "adapter_down: bad plan");
    DownArgs p{x, a, scale, u, ut, plan->slot_row, plan->piece_adapter, ldx, (int64_t)plan->n_pieces * PIECE, (int)K, R};
    hipStream_t st = (hipStream_t)stream;
#define DOWN(T, RT) hipLaunchKernelGGL((adapter_down_kernel<T, RT>), dim3((unsigned)plan->n_pieces, (unsigned)((R + RT * 32 - 1) / (RT * 32))), dim3(256), 0, st, p)
    if (dt == M4D_BF16) { if (R <= 32) DOWN(bf16_t, 1); else DOWN(bf16_t, 2); }
    else { if (R <= 32) DOWN(float, 1); else DOWN(float, 2); }
#undef DOWN
    M4D_CHECK_LAUNCH("adapter_down");
    return 0;
}

extern "C" int m4d_linear_adapters(m4d_dtype dt, const void* x, int64_t ldx, const void* W, int64_t ldw, const void* bias, const void* u,
                                   const void* b, const m4d_adapter_plan* plan, void* out, int64_t ldo, int64_t N, int64_t K, int R,
                                   m4d_stream stream) {
    PLAN_OK("linear_adapters");
    const int64_t M = plan->rows;
    M4D_CHECK_ARG(x && W && out && u && b, "linear_adapters: null pointer");
    M4D_CHECK_ARG(N > 0 && K > 0 && K < (1 << 30) && (K * es) % 16 == 0, "linear_adapters: K*sizeof(T) must be a multiple of 16 (K=%lld)", (long long)K);
    M4D_CHECK_ARG(N % 4 == 0 && ldo % 4 == 0 && (M == 1 || ldo >= N), "linear_adapters: N and the output's row stride must be multiples of 4 (N=%lld ldo=%lld)",
                  (long long)N, (long long)ldo);
    M4D_CHECK_ARG((ldx * es) % 16 == 0 && (ldw * es) % 16 == 0 && (M == 1 || ldx >= K) && ldw >= K, "linear_adapters: rows must be 16-byte aligned");
    M4D_CHECK_ARG(((uintptr_t)x % 16) == 0 && ((uintptr_t)W % 16) == 0 && ((uintptr_t)out % 16) == 0 && ((uintptr_t)u % 16) == 0 && ((uintptr_t)b % 16) == 0,
                  "linear_adapters: pointers must be 16-byte aligned");
    M4D_CHECK_ARG(plan->row_adapter && plan->tiles256_off && plan->tiles256 && plan->tiles128_off && plan->tiles128, "linear_adapters: bad plan");
    GemmAdArgs p{};
    p.A = x; p.W = W; p.bias = bias; p.out = out; p.lda = ldx; p.ldw = ldw; p.ldc = ldo; p.M = M; p.N = N; p.K = K;
    p.rows_per_sample = M; p.epilogue = M4D_EPI_STORE;
    p.u = u; p.up = b; p.row_adapter = plan->row_adapter; p.R = R;
    hipStream_t st = (hipStream_t)stream;
    // the rule of m4d_gemm_bt: 256 x 256 tiles for big bf16 problems with whole 64-element K tiles and 16-byte output rows
    const bool wide = dt == M4D_BF16 && K % 64 == 0 && M >= 512 && N >= 512 && ldo % 8 == 0 && ((uintptr_t)out % 32) == 0;
    const int bt = wide ? 256 : 128;
    const int64_t tm = (M + bt - 1) / bt, tn = (N + bt - 1) / bt;
    M4D_CHECK_ARG(tm * tn < (1ll << 31), "linear_adapters: too many tiles");
    p.tiles_m = (int)tm; p.tiles_n = (int)tn;
    p.tile_off = wide ? plan->tiles256_off : plan->tiles128_off;
    p.tile_list = wide ? plan->tiles256 : plan->tiles128;
    if (wide) {
        if (m4d_launch_gemm_wide_adapters(&p, (unsigned)(tm * tn), st) != 0) { m4d_set_error("linear_adapters: cannot enable 128 KiB LDS"); return -3; }
    } else m4d_launch_gemm_generic_adapters(&p, dt == M4D_BF16, (unsigned)(tm * tn), st);
    M4D_CHECK_LAUNCH("linear_adapters");
    m4d_count_launch(wide ? M4D_KC_GEMM_WIDE : M4D_KC_GEMM_GENERIC);
    return 0;
}

extern "C" int64_t m4d_adapter_grad_workspace(const m4d_adapter_plan* plan, int64_t C, int R) {
    return plan ? (int64_t)plan->n_chunks * R * C : 0;
}

extern "C" int m4d_adapter_grad(m4d_dtype dt, const void* vt, const void* x, int64_t ldx, const int8_t* codes, const uint8_t* exps,
                                const m4d_adapter_plan* plan, float* ws, int64_t ws_floats, void* out, int transposed, int G, int rank, int64_t C,
                                int R, m4d_stream stream) {
    PLAN_OK("adapter_grad");
    M4D_CHECK_ARG(out && G > 0 && G <= 65535 && rank > 0 && rank <= R, "adapter_grad: bad adapters (G=%d rank=%d R=%d)", G, rank, R);
    M4D_CHECK_ARG(C > 0 && C < (1 << 30) && C % 4 == 0, "adapter_grad: C=%lld must be a multiple of 4", (long long)C);
    M4D_CHECK_ARG(plan->n_adapters <= G && plan->n_chunks <= 65535, "adapter_grad: the plan names adapter %d of %d", plan->n_adapters - 1, G);
    hipStream_t st = (hipStream_t)stream;
    GradArgs p{vt, x, codes, exps, ws, out, plan->slot_row, plan->chunks, plan->chunk_off, ldx, (int64_t)plan->n_pieces * PIECE,
               (int)C, R, rank, plan->n_adapters, transposed};
    if (plan->n_chunks > 0) {
        M4D_CHECK_ARG(vt && ws && ws_floats >= (int64_t)plan->n_chunks * R * C, "adapter_grad: workspace of %lld floats needed",
                      (long long)plan->n_chunks * R * C);
        M4D_CHECK_ARG((x != nullptr) != (codes != nullptr) && (codes == nullptr) == (exps == nullptr), "adapter_grad: either x or its codes");
        M4D_CHECK_ARG(!x || (ldx * es) % 16 == 0, "adapter_grad: rows must be 16-byte aligned");
        M4D_CHECK_ARG(((uintptr_t)vt % 16) == 0 && ((uintptr_t)x % 16) == 0 && ((uintptr_t)codes % 16) == 0 && ((uintptr_t)ws % 16) == 0,
                      "adapter_grad: pointers must be 16-byte aligned");
        M4D_CHECK_ARG(plan->slot_row && plan->chunks && plan->chunk_off, "adapter_grad: bad plan");
        const int rt = R <= 32 ? 1 : 2;
        dim3 grid((unsigned)((C + 127) / 128), (unsigned)plan->n_chunks, (unsigned)((R + rt * 32 - 1) / (rt * 32)));
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
    dim3 jg((unsigned)((C + 63) / 64), (unsigned)((rank + 15) / 16), (unsigned)G);
    if (dt == M4D_BF16) hipLaunchKernelGGL(adapter_grad_join_kernel<bf16_t>, jg, dim3(256), 0, st, p);
    else hipLaunchKernelGGL(adapter_grad_join_kernel<float>, jg, dim3(256), 0, st, p);
    M4D_CHECK_LAUNCH("adapter_grad(join)");
    return 0;
}

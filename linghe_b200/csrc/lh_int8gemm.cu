// Matrix product in 8-bit integers with one scale per token and one per output channel, and the
// token-wise quantiser in front of it:
//
//   c[m,n] = (sum_k a[m,k] * b[n,k]) * a_s[m] * b_s[n]        a [M,K], b [N,K] int8, sums in 32-bit integers
//   a_s[m] = max(amax_k |x[m,k] / smooth[k]| / 127, 1e-30);   a = nearest(x / smooth / a_s)
//
// The integer sums are exact for K <= 131071 (2^31 / 128^2), so the result does not depend on how k is split:
// the kernels below split it freely and agree bit for bit.
#include "lh_eight.cuh"
#include "lh_umma.cuh"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace lh {

namespace {

constexpr int64_t kInt8MaxK = 131071 / 16 * 16;

// ---- token-wise quantiser ---------------------------------------------------------------------
// A team of warps takes a row, a lane 32 bytes of it.  Rows that 16 warps hold that way (HOLD: 8192 elements of a 16-bit
// type, 4096 of float32) stay in registers between the maximum and the codes, longer ones are walked twice, the second
// time through L2.  Small registers, so that six rows of 4096 are in flight on an SM: that is what it waits for.
constexpr int kTokWarps = 16;

struct TokenParams {
    const uint8_t* x;
    const float* smooth;
    int64_t M;
    int K, wide;
    uint8_t* q;
    float* s;
};

// the elements at column c over max(smooth, 1e-30)
template <typename T>
__device__ __forceinline__ void smoothed(const Lane<T>& x, const float* smooth, int c, float2 (&e)[Lane<T>::V][4]) {
#pragma unroll
    for (int v = 0; v < Lane<T>::V; ++v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[v][i] = x.v[v].get(i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float4 m = *reinterpret_cast<const float4*>(smooth + c + 8 * v + 4 * h);
            float2 &lo = e[v][2 * h], &hi = e[v][2 * h + 1];
            lo = make_float2(__fdiv_rn(lo.x, max_nan(m.x, kScaleFloor)), __fdiv_rn(lo.y, max_nan(m.y, kScaleFloor)));
            hi = make_float2(__fdiv_rn(hi.x, max_nan(m.z, kScaleFloor)), __fdiv_rn(hi.y, max_nan(m.w, kScaleFloor)));
        }
    }
}

template <typename T, bool HOLD, bool SMOOTH>
__global__ void __launch_bounds__(32 * kTokWarps, SMOOTH ? 2 : 3) token_quant_kernel(const TokenParams p, int team) {
    constexpr int ES = sizeof(T), SPAN = kSpan<T>, V = Lane<T>::V;
    __shared__ float part[kTokWarps];
    grid_go();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, teams = (blockDim.x >> 5) / team;
    const int64_t row = int64_t(blockIdx.x) * teams + warp / team;
    const bool any = row < p.M, wide = p.wide != 0;
    const uint8_t* x = p.x + (any ? row : 0) * p.K * ES;
    const int first = (warp % team * 32 + lane) * SPAN, stride = team * 32 * SPAN;
    float amax = 0.f;
    Lane<T> w;
    float2 e[SMOOTH ? V : 1][4];      // the quotients by the smoothing factors are kept, values are unpacked again
    for (int c = first; any && c < p.K; c += stride) {          // HOLD: once at most
        w.load(x + int64_t(c) * ES, wide);
        if constexpr (SMOOTH) smoothed(w, p.smooth, c, e);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (!SMOOTH)
#pragma unroll
                for (int i = 0; i < 4; ++i) e[0][i] = w.v[v].get(i);
            amax = max_nan(amax, amax_pairs(e[SMOOTH ? v : 0]));
        }
        if (HOLD) break;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    if (team > 1) {
        if (lane == 0) part[warp] = amax;
        __syncthreads();
        amax = part[warp / team * team + min(lane & 15, team - 1)];
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    }
    if (!any) return;
    const Divisor d(code_scale<CODES_INT8>(amax));
    if (lane == 0 && warp % team == 0) p.s[row] = d.s;
    for (int c = first; c < p.K; c += stride) {
        if constexpr (!HOLD) {
            w.load(x + int64_t(c) * ES, wide);
            if constexpr (SMOOTH) smoothed(w, p.smooth, c, e);
        }
        Codes<V> q;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (!SMOOTH)
#pragma unroll
                for (int i = 0; i < 4; ++i) e[0][i] = w.v[v].get(i);
            q.w[v] = encode8<CODES_INT8>(e[SMOOTH ? v : 0], d);
        }
        q.store(p.q + row * p.K + c);
        if (HOLD) break;
    }
}

// ---- the product ------------------------------------------------------------------------------
struct Int8Params {
    const uint8_t *a, *b;
    const float *a_s, *b_s;
    uint8_t* c;
    int64_t M;
    int N, K;
    int out_dtype;
    int wide;            // a row of c starts on a 32-byte boundary
};

__device__ __forceinline__ void store_one(const Int8Params& p, int64_t at, float v) {
    if (p.out_dtype == LH_F32) reinterpret_cast<float*>(p.c)[at] = v;
    else if (p.out_dtype == LH_BF16) reinterpret_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(p.c)[at] = __float2half_rn(v);
}

// NC (a multiple of 16) sums of one row from column col on, scaled, rounded and stored
template <int NC>
__device__ __forceinline__ void store_row(const Int8Params& p, int64_t row, int col, const uint32_t* v, float sa) {
    if (row >= p.M || col >= p.N) return;
    const int64_t at = row * p.N + col;
    if (p.wide && col + NC <= p.N) {
#pragma unroll
        for (int h = 0; h < NC; h += 16) {
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 sb = *reinterpret_cast<const float4*>(p.b_s + col + h + i);
                f[i] = __int2float_rn(int(v[h + i])) * sa * sb.x;
                f[i + 1] = __int2float_rn(int(v[h + i + 1])) * sa * sb.y;
                f[i + 2] = __int2float_rn(int(v[h + i + 2])) * sa * sb.z;
                f[i + 3] = __int2float_rn(int(v[h + i + 3])) * sa * sb.w;
            }
            if (p.out_dtype == LH_F32) {
                uint8_t* dst = p.c + (at + h) * 4;
#pragma unroll
                for (int j = 0; j < 16; j += 8)
                    st_global_256(dst + 4 * j, make_uint4(__float_as_uint(f[j]), __float_as_uint(f[j + 1]), __float_as_uint(f[j + 2]), __float_as_uint(f[j + 3])),
                                  make_uint4(__float_as_uint(f[j + 4]), __float_as_uint(f[j + 5]), __float_as_uint(f[j + 6]), __float_as_uint(f[j + 7])));
            } else {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = p.out_dtype == LH_BF16 ? pack_bf16x2(f[2 * j], f[2 * j + 1]) : pack_f16x2(f[2 * j], f[2 * j + 1]);
                st_global_256(p.c + (at + h) * 2, make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7]));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (col + i < p.N) store_one(p, at + i, __int2float_rn(int(v[i])) * sa * p.b_s[col + i]);
    }
}

// Few tokens: the weights are read once and there is next to no arithmetic, so what counts is to have all of
// them in flight at once.  A CTA takes 16 channels, its warps share k in steps of 64; a lane loads 16 bytes of two channels
// per step straight into the fragments of mma.m16n8k32 (k may be in any order as long as both operands agree, so
// a lane's 16 consecutive bytes serve as the two 4-byte pieces of two instructions).  Eight tokens fill the n = 8 of
// the instruction; NT such groups.  The weights are asked for before the wait for the kernel that writes the codes.
constexpr int kRowsSteps = 4;      // steps of a warp in flight

__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT>
__global__ void __launch_bounds__(512) int8_rows_kernel(const Int8Params p) {
    extern __shared__ int red[];                     // [warps][NT][16][8]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int g = lane >> 2, tig = lane & 3;
    const int n0 = blockIdx.x * 16;
    const bool r0 = n0 + g < p.N, r1 = n0 + g + 8 < p.N;
    const uint8_t* b0 = p.b + int64_t(n0 + g) * p.K;
    const uint8_t* b1 = b0 + int64_t(8) * p.K;
    const int steps = (p.K + 63) >> 6;
    int acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0;
    bool waited = false;
    for (int s0 = warp; s0 < steps; s0 += warps * kRowsSteps) {
        uint4 w0[kRowsSteps], w1[kRowsSteps];
#pragma unroll
        for (int i = 0; i < kRowsSteps; ++i) {
            const int k = (s0 + i * warps) * 64 + tig * 16;
            w0[i] = w1[i] = make_uint4(0, 0, 0, 0);
            if (k < p.K) {                           // K is a multiple of 16
                if (r0) w0[i] = __ldg(reinterpret_cast<const uint4*>(b0 + k));
                if (r1) w1[i] = __ldg(reinterpret_cast<const uint4*>(b1 + k));
            }
        }
        if (!waited) { grid_wait(); waited = true; }
#pragma unroll
        for (int i = 0; i < kRowsSteps; ++i) {
            const int k = (s0 + i * warps) * 64 + tig * 16;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (k < p.K && j * 8 + g < p.M) x = *reinterpret_cast<const uint4*>(p.a + int64_t(j * 8 + g) * p.K + k);
                mma_s8(acc[j], w0[i].x, w1[i].x, w0[i].y, w1[i].y, x.x, x.y);
                mma_s8(acc[j], w0[i].z, w1[i].z, w0[i].w, w1[i].w, x.z, x.w);
            }
        }
    }
    if (!waited) grid_wait();
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        int* d = red + (warp * NT + j) * 128;
        *reinterpret_cast<int2*>(d + g * 8 + tig * 2) = make_int2(acc[j][0], acc[j][1]);
        *reinterpret_cast<int2*>(d + (g + 8) * 8 + tig * 2) = make_int2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    // thread = (token, channel): 16 consecutive threads write 16 consecutive channels
    for (int i = threadIdx.x; i < NT * 128; i += blockDim.x) {
        const int m = i >> 4, ch = i & 15;
        if (m >= p.M || n0 + ch >= p.N) continue;
        const int* d = red + (m >> 3) * 128 + ch * 8 + (m & 7);
        int v = 0;
        for (int w = 0; w < warps; ++w) v += d[w * NT * 128];
        store_one(p, int64_t(m) * p.N + n0 + ch, __int2float_rn(v) * p.a_s[m] * p.b_s[n0 + ch]);
    }
}

// The tensor-core kernels: 128 x TN tiles of c, k in stages of 128 bytes brought in by TMA, int32 sums in
// tensor memory.
constexpr int IM = 128, IKB = 128;
constexpr int I_ATILE = IM * IKB;

// D s32 (format 2), A and B s8 (format 1), both K-major, M = 128, N = tn
__host__ __device__ constexpr uint32_t i8_idesc(int tm, int tn) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(tn >> 3) << 17) | (uint32_t(tm >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 lanes x 32 columns: register i of a thread holds column i of its lane
__device__ __forceinline__ void tmem_ld_row32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t tmem_alloc(uint32_t* slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    return 0;
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// Large products: one persistent CTA per SM walks tiles (column tile fastest); warp 0 TMA, warp 1 MMA, warps 2-9
// read the sums of the tile before out of the other tensor-memory buffer, scale and store them.
template <int TN>
struct BigTile {
    static constexpr int STAGE = I_ATILE + TN * IKB;
    static constexpr int STAGES = TN == 256 ? 4 : 6;
    static constexpr int BAR_OFF = STAGES * STAGE;
    static constexpr int SMEM = 1024 + BAR_OFF + 256;
    static constexpr int EPI_WARPS = 8;
    static constexpr int THREADS = 32 * (2 + EPI_WARPS);
    static_assert(SMEM <= 232448, "shared memory");
};

template <int TN>
__global__ void __launch_bounds__(BigTile<TN>::THREADS, 1)
int8_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Int8Params p) {
    using C = BigTile<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;       // two buffers of TN tensor-memory columns
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int kblocks = (p.K + IKB - 1) / IKB, tiles_n = (p.N + TN - 1) / TN;
    const int64_t tiles = (p.M + IM - 1) / IM * tiles_n;
    if (t == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], C::EPI_WARPS); }
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b);
    }
    if (warp == 1) tmem_alloc(slot, 2 * TN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(slot);
    grid_wait();

    if (warp == 0) {
        int s = 0;
        uint32_t ph = 0;
        bool first = true, ok = true;
        for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
            const int m0 = int(tile / tiles_n) * IM, n0 = int(tile % tiles_n) * TN;
            for (int kb = 0; kb < kblocks; ++kb) {
                if (!first) {
                    ok = __all_sync(0xffffffffu, mbar_wait_inline(&empty[s], ph ^ 1u, DEVERR_EMPTY_WAIT));
                    if (!ok) break;
                }
                if (elect_one()) {
                    uint8_t* st = smem + size_t(s) * C::STAGE;
                    mbar_expect_tx(&full[s], C::STAGE);
                    tma_load_2d(st, &map_a, kb * IKB, m0, &full[s]);
                    tma_load_2d(st + I_ATILE, &map_b, kb * IKB, n0, &full[s]);
                }
                if (++s == C::STAGES) { s = 0; ph ^= 1u; first = false; }
            }
        }
    } else if (warp == 1) {
        int s = 0;
        uint32_t ph = 0, n = 0;                       // n: tiles so far
        bool ok = true;
        for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++n) {
            const uint32_t buf = n & 1u;
            if (n >= 2) ok = __all_sync(0xffffffffu, mbar_wait_inline(&acc_empty[buf], ((n >> 1) & 1u) ^ 1u, DEVERR_PART_WAIT));
            for (int kb = 0; kb < kblocks && ok; ++kb) {
                ok = __all_sync(0xffffffffu, mbar_wait_inline(&full[s], ph, DEVERR_FULL_WAIT));
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t a = smem_u32(smem + size_t(s) * C::STAGE);
                    const uint64_t da = umma_desc(a), db = umma_desc(a + I_ATILE);
#pragma unroll
                    for (int k4 = 0; k4 < IKB / 32; ++k4)
                        umma_i8(tmem + buf * TN, da + 2 * k4, db + 2 * k4, i8_idesc(IM, TN), (kb | k4) != 0);
                    umma_commit(&empty[s]);
                    if (kb == kblocks - 1) umma_commit(&acc_full[buf]);
                }
                if (++s == C::STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint32_t n = 0;
        bool ok = true;
        for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++n) {
            const int64_t row = tile / tiles_n * IM + quarter * 32 + lane;
            const int n0 = int(tile % tiles_n) * TN + half * (TN / 2);
            const uint32_t buf = n & 1u;
            const float sa = row < p.M ? p.a_s[row] : 0.f;
            ok = __all_sync(0xffffffffu, mbar_wait_inline(&acc_full[buf], (n >> 1) & 1u, DEVERR_PART_WAIT));
            if (!ok) break;
            tc_fence_after();
            const uint32_t base = tmem + (uint32_t(quarter * 32) << 16) + buf * TN + half * (TN / 2);
#pragma unroll
            for (int c = 0; c < TN / 2; c += 32) {
                uint32_t v[32];
                tmem_ld_row32(base + c, v);
                if (c == TN / 2 - 32) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_empty[buf]);
                }
                store_row<32>(p, row, n0 + c, v, sa);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free(tmem, 2 * TN);
}

// Products of few tiles: a cluster of S CTAs shares k of one tile, adds the partial sums through distributed
// shared memory and stores a share of the rows each.  The cluster's rank is the part of k.
template <int TN>
struct SplitTile {
    static constexpr int STAGE = I_ATILE + TN * IKB;
    static constexpr int STAGES = TN == 256 ? 4 : TN == 128 ? 6 : 8;
    static constexpr int BAR_OFF = STAGES * STAGE;
    static constexpr int SMEM = 1024 + BAR_OFF + 256;
    static constexpr int THREADS = 192;
    static_assert(SMEM <= 232448 && IM * TN * 4 <= BAR_OFF, "shared memory");
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint4 ld_cluster(uint32_t addr, uint32_t rank) {
    uint4 v;
    asm volatile(
        "{\n\t.reg .b32 r;\n\t"
        "mapa.shared::cluster.u32 r, %4, %5;\n\t"
        "ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [r];\n\t}"
        : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}

template <int TN>
__global__ void __launch_bounds__(SplitTile<TN>::THREADS)
int8_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Int8Params p, int S) {
    using C = SplitTile<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
    uint64_t* empty = full + C::STAGES;
    uint64_t* done = empty + C::STAGES;
    uint32_t* slot = reinterpret_cast<uint32_t*>(done + 1);
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int rank = S > 1 ? int(cluster_rank()) : 0;
    const int tiles_n = (p.N + TN - 1) / TN, tile = blockIdx.x / S;
    const int m0 = tile / tiles_n * IM, n0 = tile % tiles_n * TN;
    const int kblocks = (p.K + IKB - 1) / IKB;
    const int kb0 = int(int64_t(kblocks) * rank / S), nkb = int(int64_t(kblocks) * (rank + 1) / S) - kb0;
    if (t == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(done, 1);
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b);
    }
    if (warp == 1) tmem_alloc(slot, TN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(slot);
    bool ok = true;
    if (warp == 0) {
        // the weights of the first stages do not depend on the kernel before this one
        const int early = min(nkb, C::STAGES);
        if (elect_one())
            for (int i = 0; i < early; ++i) {
                mbar_expect_tx(&full[i], C::STAGE);
                tma_load_2d(smem + size_t(i) * C::STAGE + I_ATILE, &map_b, (kb0 + i) * IKB, n0, &full[i]);
            }
        grid_wait();
        int s = 0;
        uint32_t ph = 0;
        for (int i = 0; i < nkb; ++i) {
            if (i >= C::STAGES) {
                ok = __all_sync(0xffffffffu, mbar_wait_inline(&empty[s], ph ^ 1u, DEVERR_EMPTY_WAIT));
                if (!ok) break;
            }
            if (elect_one()) {
                uint8_t* st = smem + size_t(s) * C::STAGE;
                if (i >= C::STAGES) {
                    mbar_expect_tx(&full[s], C::STAGE);
                    tma_load_2d(st + I_ATILE, &map_b, (kb0 + i) * IKB, n0, &full[s]);
                }
                tma_load_2d(st, &map_a, (kb0 + i) * IKB, m0, &full[s]);
            }
            if (++s == C::STAGES) { s = 0; ph ^= 1u; }
        }
    } else if (warp == 1) {
        int s = 0;
        uint32_t ph = 0;
        for (int i = 0; i < nkb; ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait_inline(&full[s], ph, DEVERR_FULL_WAIT));
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t a = smem_u32(smem + size_t(s) * C::STAGE);
                const uint64_t da = umma_desc(a), db = umma_desc(a + I_ATILE);
#pragma unroll
                for (int k4 = 0; k4 < IKB / 32; ++k4)
                    umma_i8(tmem, da + 2 * k4, db + 2 * k4, i8_idesc(IM, TN), (i | k4) != 0);
                umma_commit(&empty[s]);
                if (i == nkb - 1) umma_commit(done);
            }
            if (++s == C::STAGES) { s = 0; ph ^= 1u; }
        }
    }
    grid_wait();                                             // the scales of the tokens come from the kernel before, too
    // the sums are complete (S > 1: and the stages free for them)
    __syncwarp();
    const bool have = mbar_wait_inline(done, 0, DEVERR_PART_WAIT);
    tc_fence_after();
    const int quarter = warp & 3;
    if (S == 1) {
        if (warp >= 2 && have) {
            const int64_t row = int64_t(m0) + quarter * 32 + lane;
            const float sa = row < p.M ? p.a_s[row] : 0.f;
#pragma unroll 1
            for (int c = 0; c < TN; c += 32) {
                uint32_t v[32];
                tmem_ld_row32(tmem + (uint32_t(quarter * 32) << 16) + c, v);
                store_row<32>(p, row, n0 + c, v, sa);
            }
        }
    } else {
        const uint32_t part = smem_u32(smem);
        if (warp >= 2 && __all_sync(0xffffffffu, have)) {
            const int r = quarter * 32 + lane;
            if (int64_t(m0) + quarter * 32 < p.M) {          // whole warps without a row of c keep out
#pragma unroll 1
                for (int c = 0; c < TN; c += 32) {
                    uint32_t v[32];
                    tmem_ld_row32(tmem + (uint32_t(quarter * 32) << 16) + c, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {            // 16-byte pieces, xor-ed with the row against bank conflicts
                        const uint32_t at = uint32_t(r * TN * 4) + ((uint32_t(c / 4 + i) ^ uint32_t(r & 7)) << 4);
                        *reinterpret_cast<uint4*>(smem + at) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync();
        // rank r stores rows r, r + S, ...: 16 columns per thread
        constexpr int PER = TN / 16;                         // threads per row
        const int rows = int(min(int64_t(IM), p.M - m0));
        const int mine = (rows - rank + S - 1) / S;
        for (int i = t; i < mine * PER; i += C::THREADS) {
            const int r = (i / PER) * S + rank, c = (i % PER) * 16;
            uint32_t v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0u;
            for (int k = 0; k < S; ++k) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 w = ld_cluster(part + uint32_t(r * TN * 4) + ((uint32_t(c / 4 + j) ^ uint32_t(r & 7)) << 4), uint32_t(k));
                    v[4 * j] += w.x; v[4 * j + 1] += w.y; v[4 * j + 2] += w.z; v[4 * j + 3] += w.w;
                }
            }
            store_row<16>(p, int64_t(m0) + r, n0 + c, v, p.a_s[m0 + r]);
        }
        __syncwarp();
        cluster_sync();                                      // nobody leaves while others read its sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free(tmem, TN);
}

// one launch: `dependent` lets it start while the kernel before it in the stream still runs (the kernels here wait for that
// kernel before they touch what it writes), `cluster` CTAs share distributed shared memory
template <typename T> struct Same { using type = T; };   // keeps an argument out of the deduction
template <typename... Args>
int launch(const char* what, void (*kern)(Args...), unsigned grid, unsigned block, size_t smem, unsigned cluster, bool dependent,
           cudaStream_t stream, typename Same<Args>::type... args) {
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return int(e); }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (dependent) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = unsigned(n);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) { (void)cudaGetLastError(); set_error("%s: %s", what, cudaGetErrorString(e)); return int(e); }
    return LH_OK;
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int int8_check(const char* what, int64_t M, int64_t N, int64_t K, int out_dtype) {
    if (out_dtype != LH_BF16 && out_dtype != LH_F16 && out_dtype != LH_F32) return fail_arg("%s: bad out dtype", what);
    if (M < 0 || N <= 0 || K <= 0 || (K % 16) || K > kInt8MaxK)
        return fail_arg("%s: need N > 0 and K a positive multiple of 16, at most %lld (M=%lld N=%lld K=%lld)", what, (long long)kInt8MaxK,
                        (long long)M, (long long)N, (long long)K);
    if (M > 0x7fffffff - 256 || N > 0x7fffffff - 256) return fail_arg("%s: size out of range", what);
    return LH_OK;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// arguments checked, M > 0
int int8_product(Int8Params p, bool dependent, cudaStream_t stream) {
    const int sms = sm_count();
    const int64_t es = p.out_dtype == LH_F32 ? 4 : 2;
    p.wide = (p.N * es) % 32 == 0 && aligned(p.c, 32) && aligned(p.b_s, 16);
    if (p.M <= 16) {
        const int steps = (p.K + 63) / 64;
        const int warps = std::max(2, std::min(16, (steps + kRowsSteps - 1) / kRowsSteps));
        const unsigned grid = unsigned(ceil_div(p.N, 16));
        if (p.M <= 8) return launch("int8_rows_kernel", int8_rows_kernel<1>, grid, 32u * warps, size_t(warps) * 512, 1, dependent, stream, p);
        return launch("int8_rows_kernel", int8_rows_kernel<2>, grid, 32u * warps, size_t(warps) * 1024, 1, dependent, stream, p);
    }
    CUtensorMap ma, mb;
    auto maps = [&](int tn) -> int {
        if (int rc = make_tensor_map(&ma, p.a, LH_U8, uint64_t(p.M), uint64_t(p.K), uint64_t(p.K), IM, IKB, 1)) return rc;
        return make_tensor_map(&mb, p.b, LH_U8, uint64_t(p.N), uint64_t(p.K), uint64_t(p.K), uint32_t(tn), IKB, 1);
    };
    auto tiles = [&](int tn) { return ceil_div(p.M, IM) * ceil_div(p.N, tn); };
    if (tiles(256) >= sms) {
        using C = BigTile<256>;
        if (int rc = maps(256)) return rc;
        return launch("int8_tile_kernel", int8_tile_kernel<256>, unsigned(std::min<int64_t>(tiles(256), sms)), C::THREADS, C::SMEM, 1, dependent, stream, ma, mb, p);
    }
    if (tiles(128) >= sms) {
        using C = BigTile<128>;
        if (int rc = maps(128)) return rc;
        return launch("int8_tile_kernel", int8_tile_kernel<128>, unsigned(std::min<int64_t>(tiles(128), sms)), C::THREADS, C::SMEM, 1, dependent, stream, ma, mb, p);
    }
    const int kblocks = int(ceil_div(p.K, IKB));
    auto split = [&](int tn) {
        int s = 1;
        while (s < 8 && tiles(tn) * s * 2 <= sms && kblocks / (s * 2) >= 2) s *= 2;
        return s;
    };
    auto go = [&](auto tag) {
        constexpr int TN = decltype(tag)::value;
        using C = SplitTile<TN>;
        if (int rc = maps(TN)) return rc;
        const int s = split(TN);
        return launch("int8_split_kernel", int8_split_kernel<TN>, unsigned(tiles(TN) * s), C::THREADS, C::SMEM, unsigned(s), dependent, stream, ma, mb, p, s);
    };
    if (tiles(64) <= sms / 2) return go(std::integral_constant<int, 64>{});
    return go(std::integral_constant<int, 128>{});
}

int token_launch(TokenParams p, int dtype, cudaStream_t stream) {
    p.wide = (int64_t(p.K) * (dtype == LH_F32 ? 4 : 2)) % 32 == 0 && aligned(p.x, 32);
    const int span = dtype == LH_F32 ? 8 : 16;
    const int64_t warps = ceil_div(p.K, 32 * span);
    const bool hold = warps <= kTokWarps;
    const int team = hold ? int(warps) : kTokWarps, teams = std::max(1, 4 / team);
    const int64_t grid = ceil_div(p.M, teams);
    if (grid > 0x7fffffff) return fail_arg("token_quant_int8: too many rows");
    auto go = [&](auto kern) { return launch("token_quant_kernel", kern, unsigned(grid), 32u * team * teams, 0, 1, false, stream, p, team); };
    auto with = [&](auto type) {
        using T = decltype(type);
        if (p.smooth) return hold ? go(token_quant_kernel<T, true, true>) : go(token_quant_kernel<T, false, true>);
        return hold ? go(token_quant_kernel<T, true, false>) : go(token_quant_kernel<T, false, false>);
    };
    if (dtype == LH_BF16) return with(__nv_bfloat16{});
    if (dtype == LH_F16) return with(__half{});
    return with(float{});
}

int token_check(const char* what, const void* x, const float* smooth, int dtype, int64_t M, int64_t K, const void* q, const float* s) {
    if (dtype != LH_BF16 && dtype != LH_F16 && dtype != LH_F32) return fail_arg("%s: dtype must be bf16, f16 or f32", what);
    if (M < 0 || K <= 0 || (K % 16) || K > 0x3fffffff) return fail_arg("%s: need K a positive multiple of 16 (M=%lld K=%lld)", what, (long long)M, (long long)K);
    if (M == 0) return LH_OK;
    if (!x || !q || !s) return fail_arg("%s: NULL pointer", what);
    if (!aligned(x, 16) || !aligned(q, 16) || !aligned(smooth, 16)) return fail_arg("%s: pointers must be 16-byte aligned", what);
    return LH_OK;
}

}  // namespace

int token_quant_int8(const void* x, const float* smooth, int dtype, int64_t M, int64_t K, void* q, float* s, cudaStream_t stream) {
    if (int rc = token_check("token_quant_int8", x, smooth, dtype, M, K, q, s)) return rc;
    if (M == 0) return LH_OK;
    TokenParams t{};
    t.x = static_cast<const uint8_t*>(x); t.smooth = smooth; t.M = M; t.K = int(K); t.q = static_cast<uint8_t*>(q); t.s = s;
    return token_launch(t, dtype, stream);
}

int int8_gemm(const void* a, const void* b, const float* a_s, const float* b_s, void* c, int64_t M, int64_t N, int64_t K, int out_dtype,
              bool dependent, cudaStream_t stream) {
    if (int rc = int8_check("int8_gemm", M, N, K, out_dtype)) return rc;
    if (M == 0) return LH_OK;
    if (!a || !b || !a_s || !b_s || !c) return fail_arg("int8_gemm: NULL pointer");
    if (!aligned(a, 16) || !aligned(b, 16) || !aligned(c, 16)) return fail_arg("int8_gemm: pointers must be 16-byte aligned");
    Int8Params p{};
    p.a = static_cast<const uint8_t*>(a); p.b = static_cast<const uint8_t*>(b); p.a_s = a_s; p.b_s = b_s; p.c = static_cast<uint8_t*>(c);
    p.M = M; p.N = int(N); p.K = int(K); p.out_dtype = out_dtype;
    return int8_product(p, dependent, stream);
}

int int8_linear(const void* x, const float* smooth, int dtype, const void* b, const float* b_s, void* q, float* s, void* c, int64_t M,
                int64_t N, int64_t K, int out_dtype, cudaStream_t stream) {
    // everything is checked before anything is launched
    if (int rc = int8_check("int8_linear", M, N, K, out_dtype)) return rc;
    if (int rc = token_check("int8_linear", x, smooth, dtype, M, K, q, s)) return rc;
    if (M == 0) return LH_OK;
    if (!b || !b_s || !c) return fail_arg("int8_linear: NULL pointer");
    if (!aligned(b, 16) || !aligned(c, 16)) return fail_arg("int8_linear: pointers must be 16-byte aligned");
    if (int rc = token_quant_int8(x, smooth, dtype, M, K, q, s, stream)) return rc;
    return int8_gemm(q, b, s, b_s, c, M, N, K, out_dtype, true, stream);
}

}  // namespace lh

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
#include <atomic>
#include <initializer_list>
#include <type_traits>

namespace lh {

namespace {

constexpr int64_t kInt8MaxK = 131071 / 16 * 16;

// ---- token-wise quantiser ---------------------------------------------------------------------
// A team of warps takes a row, a lane 32 bytes of it.  Rows that 16 warps hold that way (HOLD: 8192 elements of a 16-bit
// type, 4096 of float32) stay in registers between the maximum and the codes, longer ones are walked twice, the second
// time through L2.  Small registers, so that six rows of 4096 are in flight on an SM: that is what it waits for (8192 x 4096 bf16
// 24.0 us, floor 15.4; smoothed, with a division per element, 42.4; float32 41.6, floor 25.6).
constexpr int kTokWarps = 16;

struct TokenParams {
    const uint8_t* x;
    const float* smooth;
    int64_t M;
    int K, wide;
    uint8_t* q;
    float* s;
};

// eight elements over max(smooth, 1e-30)
__device__ __forceinline__ void smooth8(const float* smooth, float2* e) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float4 m = *reinterpret_cast<const float4*>(smooth + 4 * h);
        float2 &lo = e[2 * h], &hi = e[2 * h + 1];
        lo = make_float2(__fdiv_rn(lo.x, max_nan(m.x, kScaleFloor)), __fdiv_rn(lo.y, max_nan(m.y, kScaleFloor)));
        hi = make_float2(__fdiv_rn(hi.x, max_nan(m.z, kScaleFloor)), __fdiv_rn(hi.y, max_nan(m.w, kScaleFloor)));
    }
}

// the elements at column c over max(smooth, 1e-30)
template <typename T>
__device__ __forceinline__ void smoothed(const Lane<T>& x, const float* smooth, int c, float2 (&e)[Lane<T>::V][4]) {
#pragma unroll
    for (int v = 0; v < Lane<T>::V; ++v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[v][i] = x.v[v].get(i);
        smooth8(smooth + c + 8 * v, e[v]);
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
    int wide;            // N is a multiple of 4 and the scales of b are aligned: four columns at a time
    int mapped;          // c has a tensor map
};

__device__ __forceinline__ void store_one(const Int8Params& p, int64_t at, float v) {
    if (p.out_dtype == LH_F32) reinterpret_cast<float*>(p.c)[at] = v;
    else if (p.out_dtype == LH_BF16) reinterpret_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(p.c)[at] = __float2half_rn(v);
}

// What an epilogue warp keeps in shared memory: the scales of its columns, fetched while the sums are not there yet, and
// 32 rows x 128 bytes in which a piece of the result is turned from one row per lane to whole 128-byte lines.  One row per
// lane straight to global memory is 32 lines per instruction: the store of a 256 x 256 tile took longer than 1024 of k.
struct alignas(1024) EpiWarp {
    static constexpr int COLS = 128, LD = 17;
    uint8_t buf[32 * 128];
    float sb[COLS];
};

// rows of c that no tensor map can describe (not a multiple of 16 bytes long): 32 rows (lane = row) x 16 columns through
// shared memory, then 16 neighbouring lanes per row, element by element
__device__ __forceinline__ void store_ragged(const Int8Params& p, int64_t row0, int col, const uint32_t* v, float sa, EpiWarp& w, const float* sb) {
    const int lane = threadIdx.x & 31;
    if (col >= p.N) return;
    float* turn = reinterpret_cast<float*>(w.buf);
#pragma unroll
    for (int i = 0; i < 16; ++i) turn[lane * EpiWarp::LD + i] = __int2float_rn(int(v[i])) * sa * sb[i];
    __syncwarp();
    const int c = col + (lane & 15);
#pragma unroll 4
    for (int r = 0; r < 32; r += 2) {
        const int64_t row = row0 + r + (lane >> 4);
        if (row < p.M && c < p.N) store_one(p, row * p.N + c, turn[(r + (lane >> 4)) * EpiWarp::LD + (lane & 15)]);
    }
    __syncwarp();
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src_smem, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x),
                 "r"(y), "r"(smem_u32(src_smem))
                 : "memory");
}

// 32 rows (lane = row) x 32 columns, scaled and rounded, into bytes [64 half, 64 half + 64) of the rows of the buffer (16-bit
// types) or all 128 (float32), laid out with the 128-byte swizzle: 16-byte piece i of row r lies at piece i ^ (r & 7)
__device__ __forceinline__ void turn_piece(const Int8Params& p, const uint32_t* v, float sa, EpiWarp& w, const float* sb, int half) {
    const int lane = threadIdx.x & 31;
    uint8_t* row = w.buf + lane * 128;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        const float4 s0 = *reinterpret_cast<const float4*>(sb + i), s1 = *reinterpret_cast<const float4*>(sb + i + 4);
        const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __int2float_rn(int(v[i + j])) * sa * s[j];
        if (p.out_dtype == LH_F32) {
#pragma unroll
            for (int j = 0; j < 8; j += 4)
                *reinterpret_cast<float4*>(row + ((((i + j) >> 2) ^ (lane & 7)) << 4)) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = p.out_dtype == LH_BF16 ? pack_bf16x2(f[2 * j], f[2 * j + 1]) : pack_f16x2(f[2 * j], f[2 * j + 1]);
            *reinterpret_cast<uint4*>(row + (((4 * half + (i >> 3)) ^ (lane & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
}

// scales of COLS columns from n0 on into shared memory, 0 past the last
__device__ __forceinline__ void fetch_scales(const Int8Params& p, int n0, int cols, float* sb) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    for (int i = lane; i < cols; i += 32) sb[i] = n0 + i < p.N ? p.b_s[n0 + i] : 0.f;
    __syncwarp();
}

// Few tokens: the weights are read once and there is next to no arithmetic, so what counts is to have all of
// them in flight at once.  A CTA takes 16 channels, its warps share k in steps of 64; a lane loads 16 bytes of two channels
// per step straight into the fragments of mma.m16n8k32 (k may be in any order as long as both operands agree, so
// a lane's 16 consecutive bytes serve as the two 4-byte pieces of two instructions).  Eight tokens fill the n = 8 of
// the instruction; NT such groups.  The weights are asked for before the wait for the kernel that writes the codes.  64 registers,
// so that two CTAs of 16 warps are on an SM.  bf16 results, weights from HBM (sets of them in turn that exceed L2): 1 x 4096 x 4096
// 5.9 us (floor 2.6), 8 x 4096 x 4096 6.3, 1 x 8192 x 8192 14.4 (floor 10.3), 4 x 4096 x 14336 13.8 (floor 9.0); weights in L2: 1 x
// 4096 x 4096 4.1, 5.5 with one CTA on an SM.  A warp has four steps in flight and asks for the next four when it has used them.
constexpr int kRowsSteps = 4;      // steps of a warp in flight

__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A warp's weights of steps s0, s0 + warps, ...: 16 bytes of two channels per lane and step.
struct RowWeights {
    uint4 w0[kRowsSteps], w1[kRowsSteps];
    __device__ __forceinline__ void load(const Int8Params& p, int n0, int s0, int warps) {
        const int lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
        const bool r0 = n0 + g < p.N, r1 = n0 + g + 8 < p.N;
        const uint8_t* b0 = p.b + int64_t(n0 + g) * p.K;
        const uint8_t* b1 = b0 + int64_t(8) * p.K;
#pragma unroll
        for (int i = 0; i < kRowsSteps; ++i) {
            const int k = (s0 + i * warps) * 64 + tig * 16;
            w0[i] = w1[i] = make_uint4(0, 0, 0, 0);
            if (k < p.K) {                           // K is a multiple of 16
                if (r0) w0[i] = __ldg(reinterpret_cast<const uint4*>(b0 + k));
                if (r1) w1[i] = __ldg(reinterpret_cast<const uint4*>(b1 + k));
            }
        }
    }
    __device__ __forceinline__ void multiply(int* acc, int i, uint4 x) const {
        mma_s8(acc, w0[i].x, w1[i].x, w0[i].y, w1[i].y, x.x, x.y);
        mma_s8(acc, w0[i].z, w1[i].z, w0[i].w, w1[i].w, x.z, x.w);
    }
};

// The warps' sums of 16 channels and NT groups of eight tokens, added and stored: thread = (token, channel), so that 16
// consecutive threads write 16 consecutive channels.  red: [warps][NT][16][8]
template <int NT>
__device__ __forceinline__ void rows_finish(const Int8Params& p, int (&acc)[NT][4], int* red, const float* a_s, int n0) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        int* d = red + (warp * NT + j) * 128;
        *reinterpret_cast<int2*>(d + g * 8 + tig * 2) = make_int2(acc[j][0], acc[j][1]);
        *reinterpret_cast<int2*>(d + (g + 8) * 8 + tig * 2) = make_int2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 128; i += blockDim.x) {
        const int m = i >> 4, ch = i & 15;
        if (m >= p.M || n0 + ch >= p.N) continue;
        const int* d = red + (m >> 3) * 128 + ch * 8 + (m & 7);
        int v = 0;
        for (int w = 0; w < warps; ++w) v += d[w * NT * 128];
        store_one(p, int64_t(m) * p.N + n0 + ch, __int2float_rn(v) * a_s[m] * p.b_s[n0 + ch]);
    }
}

template <int NT>
__global__ void __launch_bounds__(512, NT == 1 ? 2 : 1) int8_rows_kernel(const Int8Params p) {
    extern __shared__ __align__(16) int red[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int g = lane >> 2, tig = lane & 3;
    const int n0 = blockIdx.x * 16;
    const int steps = (p.K + 63) >> 6;
    int acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0;
    bool waited = false;
    for (int s0 = warp; s0 < steps; s0 += warps * kRowsSteps) {
        RowWeights w;
        w.load(p, n0, s0, warps);
        if (!waited) { grid_wait(); waited = true; }
#pragma unroll
        for (int i = 0; i < kRowsSteps; ++i) {
            const int k = (s0 + i * warps) * 64 + tig * 16;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (k < p.K && j * 8 + g < p.M) x = *reinterpret_cast<const uint4*>(p.a + int64_t(j * 8 + g) * p.K + k);
                w.multiply(acc[j], i, x);
            }
        }
    }
    if (!waited) grid_wait();
    rows_finish<NT>(p, acc, red, p.a_s, n0);
}

// One token with the quantiser inside: every CTA makes the token's codes itself (from L2, while its weights are on their way).
// As long as all CTAs run at once that costs about what the kernel in front does, and the second launch is saved: one token
// through 4096 x 4096 (bf16) takes 5.5 us on the GPU either way and 0.5 us less a call with the weights in L2 (7.1 us from HBM),
// through 1024 x 1024 3.8 us.  With more
// tokens or channels the repeated work is longer than the launch (6 x 8192 x 2048: 14 us, 5.5 in two kernels).
// The arithmetic is that of token_quant_kernel; CTA 0 leaves codes and scale in the workspaces.
constexpr int kFusedMaxK = 16384;

template <typename T, bool SMOOTH>
__global__ void __launch_bounds__(512, 2) int8_one_token_kernel(const Int8Params p, const TokenParams tok) {
    extern __shared__ __align__(16) int red[];       // [warps][16][8] sums, then the codes of the token
    __shared__ int amax;
    constexpr int ES = sizeof(T);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
    const int n0 = blockIdx.x * 16, steps = (p.K + 63) >> 6;
    uint8_t* codes = reinterpret_cast<uint8_t*>(red + warps * 128);
    RowWeights w;
    w.load(p, n0, warp, warps);
    if (t == 0) amax = 0;
    __syncthreads();
    auto element8 = [&](int c, float2* e) {
        Vec8<T> v;
        v.load(tok.x + int64_t(c) * ES);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = v.get(i);
        if constexpr (SMOOTH) smooth8(tok.smooth + c, e);
    };
    float a = 0.f;
    for (int c = t * 8; c < p.K; c += blockDim.x * 8) {
        float2 e[4];
        element8(c, e);
        a = max_nan(a, amax_pairs(e));
    }
    // of numbers without a sign the bits are in the order of the values, a NaN's above infinity's
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(a) & 0x7fffffffu);
    if (lane == 0) atomicMax(&amax, int(bits));
    __syncthreads();
    const Divisor d(code_scale<CODES_INT8>(__int_as_float(amax)));
    for (int c = t * 8; c < p.K; c += blockDim.x * 8) {
        float2 e[4];
        element8(c, e);
        const uint2 q = encode8<CODES_INT8>(e, d);
        *reinterpret_cast<uint2*>(codes + c) = q;
        if (blockIdx.x == 0) *reinterpret_cast<uint2*>(tok.q + c) = q;
    }
    if (blockIdx.x == 0 && t == 0) tok.s[0] = d.s;
    __syncthreads();
    int acc[1][4] = {{0, 0, 0, 0}};
    for (int s0 = warp; s0 < steps; s0 += warps * kRowsSteps) {
        if (s0 != warp) w.load(p, n0, s0, warps);
#pragma unroll
        for (int i = 0; i < kRowsSteps; ++i) {
            const int k = (s0 + i * warps) * 64 + (lane & 3) * 16;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (k < p.K && lane < 4) x = *reinterpret_cast<const uint4*>(codes + k);
            w.multiply(acc[0], i, x);
        }
    }
    __shared__ float scale;
    if (t == 0) scale = d.s;
    rows_finish<1>(p, acc, red, &scale, n0);         // its barrier is between
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
}
// NC (a multiple of 64) columns of 32 rows from tensor memory to c; read() is called when all of them are in registers
template <int NC, typename F>
__device__ __forceinline__ void store_sums(const Int8Params& p, const CUtensorMap* map_c, uint32_t taddr, int64_t row0, int n0, float sa, EpiWarp& w, F read) {
    const int lane = threadIdx.x & 31;
    const bool f32 = p.out_dtype == LH_F32;
    uint32_t v[2][32];
    tmem_ld_row32(taddr, v[0]);
#pragma unroll
    for (int c = 0; c < NC; c += 32) {
        const uint32_t* u = v[(c / 32) & 1];
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (c + 32 < NC) tmem_ld_row32(taddr + c + 32, v[(c / 32 + 1) & 1]);      // the next piece on its way while this one is stored
        else read();
        if (!p.mapped) {
            store_ragged(p, row0, n0 + c, u, sa, w, w.sb + c);
            store_ragged(p, row0, n0 + c + 16, u + 16, sa, w, w.sb + c + 16);
            continue;
        }
        const bool first = f32 || (c & 32) == 0;
        if (first) {                              // the copy before has read the buffer
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
        }
        turn_piece(p, u, sa, w, w.sb + c, (c >> 5) & 1);
        if (f32 || (c & 32) != 0) {
            fence_async_smem();
            __syncwarp();
            const int x = n0 + (f32 ? c : c - 32);
            if (lane == 0) {
                if (row0 < p.M && x < p.N) tma_store_2d(map_c, w.buf, x, int(row0));
                bulk_commit();
            }
        }
    }
}
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// A wait that gave up ends the loop of its warp. What the two issuing warps have issued may still be in flight then, to shared
// memory and tensor memory that other CTAs own once this one is gone: both leave their loops only when it is complete, or after
// another time limit. s, ph: the stage a warp would use next and the parity of its pass over the ring; first: its first pass.
template <int STAGES>
__device__ __forceinline__ void drain_copies(uint64_t* full, int s, uint32_t ph, bool first) {
    for (int i = 0; i < STAGES; ++i)
        if (i < s || !first) mbar_wait_inline(&full[i], i < s ? ph : ph ^ 1u, DEVERR_FULL_WAIT);
}
// the commit of the last stage stands for all MMAs before it
template <int STAGES>
__device__ __forceinline__ void drain_mmas(uint64_t* empty, int s, uint32_t ph, bool first) {
    if (s > 0) mbar_wait_inline(&empty[s - 1], ph, DEVERR_EMPTY_WAIT);
    else if (!first) mbar_wait_inline(&empty[STAGES - 1], ph ^ 1u, DEVERR_EMPTY_WAIT);
}

// Products of many tiles and little k: one persistent CTA per SM walks tiles (column tile fastest); warp 0 TMA, warp 1 MMA,
// warps 2-9 read the sums of the tile before out of the other tensor-memory buffer, scale and store them.  A tile has a quarter of the
// sums of one of the kernel for pairs of SMs below: ahead where k is short (4096 x 8192 x 512 bf16 30 us, 34 there), far behind
// where it is long (8192 x 8192 x 4096 266 us, 177 there).
template <int TN>
struct BigTile {
    static constexpr int STAGE = I_ATILE + TN * IKB;
    static constexpr int STAGES = 5;
    static constexpr int EPI_WARPS = 8;
    static constexpr int EPI_OFF = STAGES * STAGE;
    static constexpr int BAR_OFF = EPI_OFF + EPI_WARPS * int(sizeof(EpiWarp));
    static constexpr int SMEM = 1024 + BAR_OFF + 256;
    static constexpr int THREADS = 32 * (2 + EPI_WARPS);
    static_assert(SMEM <= 232448, "shared memory");
};

template <int TN>
__global__ void __launch_bounds__(BigTile<TN>::THREADS, 1)
int8_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_c, const __grid_constant__ Int8Params p) {
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
        drain_copies<C::STAGES>(full, s, ph, first);
    } else if (warp == 1) {
        int s = 0;
        uint32_t ph = 0, n = 0;                       // n: tiles so far
        bool first = true, ok = true;
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
                if (++s == C::STAGES) { s = 0; ph ^= 1u; first = false; }
            }
        }
        drain_mmas<C::STAGES>(empty, s, ph, first);
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        EpiWarp& epi = reinterpret_cast<EpiWarp*>(smem + C::EPI_OFF)[warp - 2];
        uint32_t n = 0;
        bool ok = true;
        for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++n) {
            const int64_t row0 = tile / tiles_n * IM + quarter * 32;
            const int n0 = int(tile % tiles_n) * TN + half * (TN / 2);
            const uint32_t buf = n & 1u;
            const float sa = row0 + lane < p.M ? p.a_s[row0 + lane] : 0.f;
            fetch_scales(p, n0, TN / 2, epi.sb);
            ok = __all_sync(0xffffffffu, mbar_wait_inline(&acc_full[buf], (n >> 1) & 1u, DEVERR_PART_WAIT));
            if (!ok) break;
            tc_fence_after();
            store_sums<TN / 2>(p, &map_c, tmem + (uint32_t(quarter * 32) << 16) + buf * TN + half * (TN / 2), row0, n0, sa, epi, [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[buf]);
            });
        }
        if (lane == 0) bulk_wait_all();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free(tmem, 2 * TN);
}

// The largest products: two CTAs of a cluster (a pair of SMs) share a 256 x 256 tile, tcgen05.mma.cta_group::2.  Each
// brings in its 128 rows of a and its 128 rows of b, half of what the pair multiplies, so an SM takes 32 KB per 128 bytes of k
// for 128 x 256 sums; a CTA alone takes 48, 96 bytes per cycle at the full rate of the tensor cores, more than L2 gives (bf16
// results, 8192 x 8192 x 4096: 201 us against 177, 8192^3: 485 against 364 to 379, by the card).  From about 4096 of k on the power limit bounds it: 0.40 us per 128
// of k where a short run takes 0.26; below 1024 of k the stores do, about 5 us per tile.  The leader (rank 0) issues for both; full[] counts in the leader's shared memory what both
// bring, commits arrive in both CTAs, both read their half of the sums.
struct PairTile {
    static constexpr int TN = 256, TM = 256;
    static constexpr int STAGE = 2 * I_ATILE;         // a: 16 KB, b: 16 KB
    static constexpr int STAGES = 5;
    static constexpr int EPI_WARPS = 8;
    static constexpr int EPI_OFF = STAGES * STAGE;
    static constexpr int BAR_OFF = EPI_OFF + EPI_WARPS * int(sizeof(EpiWarp));
    static constexpr int SMEM = 1024 + BAR_OFF + 256;
    static constexpr int THREADS = 32 * (2 + EPI_WARPS);
    static_assert(SMEM <= 232448, "shared memory");
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void umma2_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrives on the barrier of this offset in both CTAs when the MMAs issued so far are complete
__device__ __forceinline__ void umma2_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"(uint16_t(3))
                 : "memory");
}
// a tile into this CTA's shared memory, its bytes counted on a barrier of the pair
__device__ __forceinline__ void tma2_load_2d(void* dst_smem, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst_smem)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// bounded wait for arrivals from both CTAs
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, int code) {
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 22); ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (done) return true;
    }
    atomicCAS(&g_device_status, 0, code);
    return false;
}

// Tiles in the order of row bands of 8 tiles, down a column of a band before the next column: the tiles in flight then
// share as few rows of a and of b as can be, and both stay in L2 where one of them alone would not.
__device__ __forceinline__ void band_tile(int64_t tile, int tiles_m, int tiles_n, int& tm, int& tn) {
    constexpr int BAND = 8;
    const int64_t per_band = int64_t(BAND) * tiles_n;
    const int band = int(tile / per_band), rest = int(tile - band * per_band);
    const int rows = min(BAND, tiles_m - band * BAND);
    tn = rest / rows;
    tm = band * BAND + (rest - tn * rows);
}

__global__ void __launch_bounds__(PairTile::THREADS, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_c, const __grid_constant__ Int8Params p) {
    using C = PairTile;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);   // used in the leader
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;
    uint64_t* acc_empty = acc_full + 2;                                // used in the leader
    uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const uint32_t rank = cluster_rank();
    const int kblocks = (p.K + IKB - 1) / IKB, tiles_n = (p.N + C::TN - 1) / C::TN, tiles_m = int((p.M + C::TM - 1) / C::TM);
    const int64_t tiles = int64_t(tiles_m) * tiles_n;
    const int64_t first = blockIdx.x >> 1, step = gridDim.x >> 1;
    if (t == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 2 * C::EPI_WARPS); }
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                              // the other CTA's barriers are set up, too
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(slot);
    grid_wait();

    if (warp == 0) {
        int s = 0;
        uint32_t ph = 0;
        bool fresh = true, ok = true;
        for (int64_t tile = first; tile < tiles && ok; tile += step) {
            int tm, tn;
            band_tile(tile, tiles_m, tiles_n, tm, tn);
            const int m0 = tm * C::TM + int(rank) * IM, n0 = tn * C::TN + int(rank) * 128;
            for (int kb = 0; kb < kblocks; ++kb) {
                if (!fresh) {
                    ok = __all_sync(0xffffffffu, mbar_wait_inline(&empty[s], ph ^ 1u, DEVERR_EMPTY_WAIT));
                    if (!ok) break;
                }
                if (elect_one()) {
                    uint8_t* st = smem + size_t(s) * C::STAGE;
                    const uint32_t bar = mapa(smem_u32(&full[s]), 0);
                    if (rank == 0) mbar_expect_tx(&full[s], 2 * C::STAGE);
                    tma2_load_2d(st, &map_a, kb * IKB, m0, bar);
                    tma2_load_2d(st + I_ATILE, &map_b, kb * IKB, n0, bar);
                }
                if (++s == C::STAGES) { s = 0; ph ^= 1u; fresh = false; }
            }
        }
        if (rank == 0) drain_copies<C::STAGES>(full, s, ph, fresh);       // what both have brought in
    } else if (warp == 1) {
        int s = 0;
        uint32_t ph = 0, n = 0;
        bool fresh = true, ok = rank == 0;
        for (int64_t tile = first; tile < tiles && ok; tile += step, ++n) {
            const uint32_t buf = n & 1u;
            if (n >= 2) ok = __all_sync(0xffffffffu, mbar_wait_cluster(&acc_empty[buf], ((n >> 1) & 1u) ^ 1u, DEVERR_PART_WAIT));
            for (int kb = 0; kb < kblocks && ok; ++kb) {
                ok = __all_sync(0xffffffffu, mbar_wait_cluster(&full[s], ph, DEVERR_FULL_WAIT));
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t a = smem_u32(smem + size_t(s) * C::STAGE);
                    const uint64_t da = umma_desc(a), db = umma_desc(a + I_ATILE);
#pragma unroll
                    for (int k4 = 0; k4 < IKB / 32; ++k4)
                        umma2_i8(tmem + buf * C::TN, da + 2 * k4, db + 2 * k4, i8_idesc(C::TM, C::TN), (kb | k4) != 0);
                    umma2_commit(&empty[s]);
                    if (kb == kblocks - 1) umma2_commit(&acc_full[buf]);
                }
                if (++s == C::STAGES) { s = 0; ph ^= 1u; fresh = false; }
            }
        }
        drain_mmas<C::STAGES>(empty, s, ph, fresh);                       // rank 1 has issued none
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        EpiWarp& epi = reinterpret_cast<EpiWarp*>(smem + C::EPI_OFF)[warp - 2];
        uint32_t n = 0;
        bool ok = true;
        for (int64_t tile = first; tile < tiles && ok; tile += step, ++n) {
            int tm, tn;
            band_tile(tile, tiles_m, tiles_n, tm, tn);
            const int64_t row0 = int64_t(tm) * C::TM + rank * IM + quarter * 32;
            const int n0 = tn * C::TN + half * 128;
            const uint32_t buf = n & 1u;
            const float sa = row0 + lane < p.M ? p.a_s[row0 + lane] : 0.f;
            fetch_scales(p, n0, 128, epi.sb);
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(&acc_full[buf], (n >> 1) & 1u, DEVERR_PART_WAIT));
            if (!ok) break;
            tc_fence_after();
            store_sums<128>(p, &map_c, tmem + (uint32_t(quarter * 32) << 16) + buf * C::TN + half * 128, row0, n0, sa, epi, [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(mapa(smem_u32(&acc_empty[buf]), 0)) : "memory");
            });
        }
        if (lane == 0) bulk_wait_all();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();                              // neither leaves while the other's copies, MMAs or arrivals may still reach it
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Products of few tiles: a cluster of S CTAs shares k of one tile; the rank is the part of k.  Rank r owns the rows r, r + S,
// ... of the tile: every CTA writes its sums of them to its own place in the owner's shared memory (stores to the other
// SMs that nobody waits for; reading them from there instead took twice as long), and behind one cluster barrier the
// owner adds them up and stores the result.  What bounds it is the step of the warp that issues the MMAs (wait, four MMAs, commit),
// 0.27 us per 128 bytes of k: a CTA alone on the GPU takes that with 3 to 7 stages and 64 columns (0.29 with 128, and with 2 stages),
// 0.27 still without its loads, 0.22 without its MMAs; with 128 CTAs 0.29 and 0.34.  So k is split as far as there are SMs.
template <int TN>
struct SplitTile {
    static constexpr int STAGE = I_ATILE + TN * IKB;
    static constexpr int STAGES = TN == 128 ? 4 : 6;
    static constexpr int SUM_OFF = STAGES * STAGE;                 // the ranks' sums of the rows of this CTA
    static constexpr int BAR_OFF = SUM_OFF + (IM + 8) * TN * 4;    // S * ceil(IM / S) rows at most
    static constexpr int SMEM = 1024 + BAR_OFF + 256;
    static constexpr int THREADS = 192;
    static_assert(SMEM <= 232448 && 4 * int(sizeof(EpiWarp)) <= SUM_OFF && TN <= EpiWarp::COLS, "shared memory");
};

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t rank, uint4 v) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mapa(addr, rank)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <int TN>
__global__ void __launch_bounds__(SplitTile<TN>::THREADS)
int8_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_c, const __grid_constant__ Int8Params p, int S) {
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
    if (S > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");     // waited for before the first store to another CTA
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
        bool first = true;
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
            if (++s == C::STAGES) { s = 0; ph ^= 1u; first = false; }
        }
        drain_copies<C::STAGES>(full, s, ph, first);
    } else if (warp == 1) {
        int s = 0;
        uint32_t ph = 0;
        bool first = true;
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
            if (++s == C::STAGES) { s = 0; ph ^= 1u; first = false; }
        }
        drain_mmas<C::STAGES>(empty, s, ph, first);
    }
    grid_wait();                                             // the scales of the tokens come from the kernel before, too
    // the sums are complete (S > 1: and the stages free for them)
    __syncwarp();
    const bool have = mbar_wait_inline(done, 0, DEVERR_PART_WAIT);
    tc_fence_after();
    const int quarter = warp & 3;
    if (S == 1) {
        if (warp >= 2 && __all_sync(0xffffffffu, have) && int64_t(m0) + quarter * 32 < p.M) {
            // the stages are free, the scales and the turning room take their place
            EpiWarp& epi = reinterpret_cast<EpiWarp*>(smem)[warp - 2];
            const int64_t row0 = int64_t(m0) + quarter * 32;
            const float sa = row0 + lane < p.M ? p.a_s[row0 + lane] : 0.f;
            fetch_scales(p, n0, TN, epi.sb);
            store_sums<TN>(p, &map_c, tmem + (uint32_t(quarter * 32) << 16), row0, n0, sa, epi, []() {});
            if (lane == 0) bulk_wait_all();
            __syncwarp();
        }
    } else {
        // place of the sums of rank k for the owner's i-th row: ((k * per + i) * TN) floats, its 16-byte pieces xor-ed with the
        // row against bank conflicts
        const int per = (IM + S - 1) / S;
        const uint32_t sums = smem_u32(smem + C::SUM_OFF);
        __syncwarp();
        cluster_wait();                                      // every CTA of the cluster has started: its shared memory is there
        if (warp >= 2 && __all_sync(0xffffffffu, have) && int64_t(m0) + quarter * 32 < p.M) {   // whole warps without a row of c keep out
            const int r = quarter * 32 + lane, owner = r % S, i = r / S;
            const uint32_t at = sums + uint32_t((rank * per + i) * TN * 4);
#pragma unroll 1
            for (int c = 0; c < TN; c += 32) {
                uint32_t v[32];
                tmem_ld_row32(tmem + (uint32_t(quarter * 32) << 16) + c, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    st_cluster(at + ((uint32_t(c / 4 + j) ^ uint32_t(i & 7)) << 4), uint32_t(owner), make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
            }
        }
        __syncwarp();
        cluster_sync();
        const int rows = int(min(int64_t(IM), p.M - m0));
        const int mine = (rows - rank + S - 1) / S;
        constexpr int PER = TN / 4;                          // four columns per thread: a warp stores 128 columns of a row
        for (int q = t; q < mine * PER; q += C::THREADS) {
            const int i = q / PER, c = (q % PER) * 4, col = n0 + c;
            uint4 v = make_uint4(0, 0, 0, 0);
#pragma unroll 4
            for (int k = 0; k < S; ++k) {
                const uint4 w = *reinterpret_cast<const uint4*>(smem + C::SUM_OFF + ((k * per + i) * TN * 4) + ((uint32_t(c / 4) ^ uint32_t(i & 7)) << 4));
                v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
            }
            const int64_t row = int64_t(m0) + i * S + rank;
            const float sa = p.a_s[row];
            if (p.wide && col + 4 <= p.N) {
                const float4 sb = *reinterpret_cast<const float4*>(p.b_s + col);
                const float f[4] = {__int2float_rn(int(v.x)) * sa * sb.x, __int2float_rn(int(v.y)) * sa * sb.y, __int2float_rn(int(v.z)) * sa * sb.z, __int2float_rn(int(v.w)) * sa * sb.w};
                const int64_t to = row * p.N + col;
                if (p.out_dtype == LH_F32) *reinterpret_cast<float4*>(p.c + to * 4) = make_float4(f[0], f[1], f[2], f[3]);
                else if (p.out_dtype == LH_BF16) *reinterpret_cast<uint2*>(p.c + to * 2) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
                else *reinterpret_cast<uint2*>(p.c + to * 2) = make_uint2(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]));
            } else {
                const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < p.N) store_one(p, row * p.N + col + j, __int2float_rn(int(u[j])) * sa * p.b_s[col + j]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_free(tmem, TN);
}

// one launch: `dependent` lets it start while the kernel before it in the stream still runs (the kernels here wait for that
// kernel before they touch what it writes), `cluster` CTAs share distributed shared memory
template <auto KERN, typename... Args>
int launch(const char* what, unsigned grid, unsigned block, size_t smem, unsigned cluster, bool dependent,
           cudaStream_t stream, const Args&... args) {
    if (smem > 48 * 1024)                        // a constant of the kernel
        if (int rc = allow_smem<KERN>(int(smem))) return rc;
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, KERN, args...);
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

// Warps that share k in the kernels for few tokens: as many as have all their weights in flight at once, at most 16; 8 where there
// are more CTAs of 16 channels than two per SM, so that the next ones load while these finish (1 x 8192 x 8192 14.7 us, 16.6
// with 16 warps; 4 x 4096 x 14336 17.1 and 14.5).
int rows_warps(int64_t N, int64_t K) {
    const int64_t most = N > 32 * int64_t(sm_count()) ? 8 : 16;
    return int(std::max<int64_t>(2, std::min<int64_t>(most, ceil_div(ceil_div(K, 64), kRowsSteps))));
}

// How many clusters of s CTAs of the split kernel run at once on the current device (asked once per device, tile and s): where
// there are more of them a second wave doubles the time.
template <int TN>
int query_clusters(int s) {
    using C = SplitTile<TN>;
    if (allow_smem<int8_split_kernel<TN>>(C::SMEM) != LH_OK) return 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(s));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(s);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, int8_split_kernel<TN>, &cfg) != cudaSuccess) { (void)cudaGetLastError(); return 0; }
    return n;
}
int split_clusters(int tn, int s) {
    static std::atomic<int> known[64][2][9];      // clusters + 1, 0 = not asked
    int dev = 0;
    sm_count(&dev);
    std::atomic<int>* at = dev >= 0 && dev < 64 ? &known[dev][tn == 64][s] : nullptr;
    if (at && at->load(std::memory_order_relaxed)) return at->load(std::memory_order_relaxed) - 1;
    const int n = tn == 64 ? query_clusters<64>(s) : query_clusters<128>(s);
    if (at) at->store(n + 1, std::memory_order_relaxed);
    return n;
}

// arguments checked, M > 0
int int8_product(Int8Params p, bool dependent, cudaStream_t stream) {
    const int sms = sm_count();
    const int64_t es = p.out_dtype == LH_F32 ? 4 : 2;
    p.wide = p.N % 4 == 0 && aligned(p.b_s, 16);
    if (p.M <= 16) {
        const int warps = rows_warps(p.N, p.K);
        const unsigned grid = unsigned(ceil_div(p.N, 16));
        if (p.M <= 8) return launch<int8_rows_kernel<1>>("int8_rows_kernel", grid, 32u * warps, size_t(warps) * 512, 1, dependent, stream, p);
        return launch<int8_rows_kernel<2>>("int8_rows_kernel", grid, 32u * warps, size_t(warps) * 1024, 1, dependent, stream, p);
    }
    CUtensorMap ma, mb, mc{};
    p.mapped = (p.N * es) % 16 == 0;
    if (p.mapped)
        if (int rc = make_tensor_map(&mc, p.c, p.out_dtype, uint64_t(p.M), uint64_t(p.N), uint64_t(p.N * es), 32, uint32_t(128 / es), 1)) return rc;
    auto maps = [&](int tn) -> int {
        if (int rc = make_tensor_map(&ma, p.a, LH_U8, uint64_t(p.M), uint64_t(p.K), uint64_t(p.K), IM, IKB, 1)) return rc;
        return make_tensor_map(&mb, p.b, LH_U8, uint64_t(p.N), uint64_t(p.K), uint64_t(p.K), uint32_t(tn), IKB, 1);
    };
    // Which kernel, by an estimate in microseconds: the slowest CTA's MMAs per 128 bytes of k, at least its stores, or what all
    // CTAs bring in through L2 at 9.5 TB/s, and what follows the last MMA: the join of a split k, or stores that nothing hides (longest
    // where rows have to be written element by element).  Plus 4 for the launch it follows the measured times within 3 us in most cases
    // (bf16 results): 32 x 4096 x 4096 8.3 us (128 columns, k in 4; whole 15.1), 300 x 1024 x 8192 13.7 (128 columns, in 4;
    // 64 in 2 15.7; whole 24.6), 4096 x 8192 x 512 30 (tile; pair 34), 8192 x 8192 x 4096 177 (pair; tile 266).  Where it is wrong:
    // 1000 x 1111 x 2064 14.4 (128 columns, in 2; 64 columns, whole, 12.4), 512 x 4096 x 4096 16.4 (pair; 128 columns 17.8; tile,
    // which is not considered for so few tiles, 14.5).
    const int kblocks = int(ceil_div(p.K, IKB));
    enum { SPLIT64, SPLIT128, TILE, PAIR };
    int kind = PAIR, parts = 1;
    double best = 1e30;
    auto consider = [&](int which, int s, int64_t count, int64_t at_once, int nkb, int tm, int tn, double per_block, double stores, double join) {
        const double rows = double(std::min<int64_t>(p.M, tm));
        const double mma = double(ceil_div(count, at_once)) * std::max(nkb * per_block, stores);
        const double l2 = double(count) * s * nkb * IKB * (rows + tn) / 9.5e6;
        const double cost = std::max(mma, l2) + join;
        if (cost < best) { best = cost; kind = which; parts = s; }
    };
    auto tiles = [&](int tm, int tn) { return ceil_div(p.M, tm) * ceil_div(p.N, tn); };
    consider(PAIR, 1, tiles(256, 256), sms / 2, kblocks, 256, 256, 0.38, 5.0, p.mapped ? 0.0 : 9.0);
    if (tiles(IM, 128) > sms) consider(TILE, 1, tiles(IM, 128), sms, kblocks, IM, 128, 0.33, 2.1, p.mapped ? 0.0 : 4.0);
    for (const int tn : {64, 128}) {
        const int64_t n = tiles(IM, tn);
        if (n > sms) continue;
        const double per_block = tn == 64 ? 0.29 : 0.33;
        for (const int s : {1, 2, 3, 4, 6, 8})
            if (s <= kblocks && (s == 1 || n <= split_clusters(tn, s)))
                consider(tn == 64 ? SPLIT64 : SPLIT128, s, n, n, int(ceil_div(kblocks, s)), IM, tn, per_block, 0.0,
                         s > 1 ? (tn == 64 ? 0.7 : 1.0) + 0.008 * double(std::min<int64_t>(p.M, IM)) : p.mapped ? (tn == 64 ? 0.9 : 2.0) : tn == 64 ? 2.5 : 6.5);
    }
    if (kind == PAIR) {
        using C = PairTile;
        if (int rc = maps(128)) return rc;
        return launch<int8_pair_kernel>("int8_pair_kernel", unsigned(2 * std::min<int64_t>(tiles(256, 256), sms / 2)), C::THREADS, C::SMEM, 2, dependent,
                      stream, ma, mb, mc, p);
    }
    if (kind == TILE) {
        using C = BigTile<128>;
        if (int rc = maps(128)) return rc;
        return launch<int8_tile_kernel<128>>("int8_tile_kernel", unsigned(std::min<int64_t>(tiles(IM, 128), sms)), C::THREADS, C::SMEM, 1, dependent, stream,
                      ma, mb, mc, p);
    }
    auto go = [&](auto tag) {
        constexpr int TN = decltype(tag)::value;
        using C = SplitTile<TN>;
        if (int rc = maps(TN)) return rc;
        return launch<int8_split_kernel<TN>>("int8_split_kernel", unsigned(tiles(IM, TN) * parts), C::THREADS, C::SMEM, unsigned(parts), dependent, stream, ma, mb,
                      mc, p, parts);
    };
    return kind == SPLIT64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

int token_launch(TokenParams p, int dtype, cudaStream_t stream) {
    p.wide = (int64_t(p.K) * (dtype == LH_F32 ? 4 : 2)) % 32 == 0 && aligned(p.x, 32);
    const int span = dtype == LH_F32 ? 8 : 16;
    const int64_t warps = ceil_div(p.K, 32 * span);
    const bool hold = warps <= kTokWarps;
    const int team = hold ? int(warps) : kTokWarps, teams = std::max(1, 4 / team);
    const int64_t grid = ceil_div(p.M, teams);
    if (grid > 0x7fffffff) return fail_arg("token_quant_int8: too many rows");
    const unsigned threads = 32u * team * teams;
    const char* what = "token_quant_kernel";
    auto with = [&](auto type) {
        using T = decltype(type);
        if (p.smooth)
            return hold ? launch<token_quant_kernel<T, true, true>>(what, unsigned(grid), threads, 0, 1, false, stream, p, team)
                        : launch<token_quant_kernel<T, false, true>>(what, unsigned(grid), threads, 0, 1, false, stream, p, team);
        return hold ? launch<token_quant_kernel<T, true, false>>(what, unsigned(grid), threads, 0, 1, false, stream, p, team)
                    : launch<token_quant_kernel<T, false, false>>(what, unsigned(grid), threads, 0, 1, false, stream, p, team);
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
    if (M == 1 && K <= kFusedMaxK && N <= 32 * int64_t(sm_count())) {      // two CTAs of 16 channels per SM
        Int8Params p{};
        p.b = static_cast<const uint8_t*>(b); p.b_s = b_s; p.c = static_cast<uint8_t*>(c);
        p.M = M; p.N = int(N); p.K = int(K); p.out_dtype = out_dtype;
        TokenParams t{};
        t.x = static_cast<const uint8_t*>(x); t.smooth = smooth; t.M = M; t.K = int(K); t.q = static_cast<uint8_t*>(q); t.s = s;
        const int warps = rows_warps(N, K);
        const size_t smem = size_t(warps) * 512 + size_t(K);
        const unsigned grid = unsigned(ceil_div(N, 16)), threads = 32u * warps;
        const char* what = "int8_one_token_kernel";
        auto with = [&](auto type) {
            using T = decltype(type);
            return smooth ? launch<int8_one_token_kernel<T, true>>(what, grid, threads, smem, 1, false, stream, p, t)
                          : launch<int8_one_token_kernel<T, false>>(what, grid, threads, smem, 1, false, stream, p, t);
        };
        if (dtype == LH_BF16) return with(__nv_bfloat16{});
        if (dtype == LH_F16) return with(__half{});
        return with(float{});
    }
    if (int rc = token_quant_int8(x, smooth, dtype, M, K, q, s, stream)) return rc;
    return int8_gemm(q, b, s, b_s, c, M, N, K, out_dtype, true, stream);
}

}  // namespace lh

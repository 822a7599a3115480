// SwiGLU that keeps its input as an 8-bit checkpoint, and its gradient from the checkpoint:
//
//   y = silu(x1) * x2 [* w_row],  x = [x1 | x2] [M, 2n];   codes of x in blocks of 1x128, [M, 2n], scales [M, 2n/128]
//   with x1, x2 the values of the codes, s = sigmoid(x1):
//   dw = sum g * x1 * s * x2;   gw = g * w;   dx1 = gw * x2 * s * (1 + x1 * (1 - s));   dx2 = gw * x1 * s
//
// Forward: 4 bytes read and 2 + 2 written per output element of a 16-bit type; backward: 2 + 2 read, 4 written.
// Nothing is read twice, so both are streams: no shared memory but for the row sum of dw.  A team of 1, 2, 4 or 8
// warps takes a row (dw is a sum over it), a lane 8 columns at a time: 16 lanes hold a block, so its maximum is
// four shuffles, and a warp's accesses are 512 (codes: 256) consecutive bytes.
#include "lh_eight.cuh"

#include <algorithm>
#include <initializer_list>

namespace lh {

namespace {

constexpr int kSilu8Threads = 256;

struct Silu8Params {
    const uint8_t *x, *g, *xq;
    const float* xs;
    const void* w;        // float32 or bf16 [M], may be NULL
    int w_bf16;
    int64_t M;
    int n;
    uint8_t *y, *q, *dx;
    float* s;
    void* dw;
};

__device__ __forceinline__ float row_weight(const Silu8Params& p, int64_t row) {
    if (!p.w) return 1.f;
    return p.w_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.w)[row]) : static_cast<const float*>(p.w)[row];
}

// VEC: 8-element vectors of x1 and of x2 that a lane has in flight
template <typename T, int CK, int VEC>
__global__ void __launch_bounds__(kSilu8Threads) silu8_fwd_kernel(const Silu8Params p, int team) {
    constexpr int ES = sizeof(T);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, teams = kSilu8Threads / 32 / team;
    const int64_t row = int64_t(blockIdx.x) * teams + warp / team;
    if (row >= p.M) return;                             // whole warps
    const int nb = p.n >> 7;
    const uint8_t* x1 = p.x + row * 2 * p.n * ES;
    const float wt = row_weight(p, row);
    const int stride = team * 256;
    for (int c0 = (warp % team) * 256; c0 < p.n; c0 += VEC * stride) {     // the same for all lanes of a warp
        Vec8<T> a[VEC], b[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const int c = c0 + k * stride + lane * 8;
            a[k].zero(); b[k].zero();
            if (c < p.n) {
                a[k].load(x1 + int64_t(c) * ES);
                b[k].load(x1 + (int64_t(p.n) + c) * ES);
            }
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            if (c0 + k * stride >= p.n) break;           // the same for all lanes
            const int c = c0 + k * stride + lane * 8;
            const bool live = c < p.n;
            float2 va[4], vb[4];
            Vec8<T> y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                va[i] = a[k].get(i);
                vb[i] = b[k].get(i);
                y.set(i, mul2(mul2(mul2(va[i], sigmoid_fast2(va[i])), vb[i]), splat2(wt)));
            }
            const float sa = code_scale<CK>(block_amax(amax_pairs(va))), sb = code_scale<CK>(block_amax(amax_pairs(vb)));
            if (live) {
                y.store(p.y + (row * p.n + c) * ES);
                uint8_t* q = p.q + row * 2 * p.n + c;
                *reinterpret_cast<uint2*>(q) = encode8<CK>(va, Divisor(sa));
                *reinterpret_cast<uint2*>(q + p.n) = encode8<CK>(vb, Divisor(sb));
                if ((lane & 15) == 0) {
                    float* s = p.s + row * 2 * nb + (c >> 7);
                    s[0] = sa;
                    s[nb] = sb;
                }
            }
        }
    }
}

template <typename T, int CK, int VEC>
__global__ void __launch_bounds__(kSilu8Threads) silu8_bwd_kernel(const Silu8Params p, int team) {
    constexpr int ES = sizeof(T);
    __shared__ float part[kSilu8Threads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, teams = kSilu8Threads / 32 / team;
    const int64_t row = int64_t(blockIdx.x) * teams + warp / team;
    const int nb = p.n >> 7, stride = team * 256;
    float2 acc = make_float2(0.f, 0.f);
    if (row < p.M) {                                     // whole warps
        const uint8_t* xq = p.xq + row * 2 * p.n;
        const uint8_t* g = p.g + row * p.n * ES;
        const float* xs = p.xs + row * 2 * nb;
        uint8_t* dx = p.dx + row * 2 * p.n * ES;
        const float wt = row_weight(p, row);
        for (int c0 = (warp % team) * 256; c0 < p.n; c0 += VEC * stride) {
            Vec8<T> gv[VEC];
            uint2 q1[VEC], q2[VEC];
            float s1[VEC], s2[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const int c = c0 + k * stride + lane * 8;
                if (c < p.n) {
                    gv[k].load(g + int64_t(c) * ES);
                    q1[k] = *reinterpret_cast<const uint2*>(xq + c);
                    q2[k] = *reinterpret_cast<const uint2*>(xq + p.n + c);
                    s1[k] = xs[c >> 7];
                    s2[k] = xs[nb + (c >> 7)];
                }
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const int c = c0 + k * stride + lane * 8;
                if (c >= p.n) break;
                float2 x1[4], x2[4];
                decode8<CK>(q1[k], s1[k], x1);
                decode8<CK>(q2[k], s2[k], x2);
                Vec8<T> d1, d2;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 sg = sigmoid_fast2(x1[i]), gr = gv[k].get(i);
                    const float2 si = mul2(x1[i], sg);                                 // silu(x1)
                    acc = fma2(mul2(gr, si), x2[i], acc);
                    const float2 gw = mul2(gr, splat2(wt));
                    // s * (1 + x1 * (1 - s)) = s + si * (1 - s)
                    const float2 ds = fma2(si, make_float2(1.f - sg.x, 1.f - sg.y), sg);
                    d1.set(i, mul2(mul2(gw, x2[i]), ds));
                    d2.set(i, mul2(gw, si));
                }
                d1.store(dx + int64_t(c) * ES);
                d2.store(dx + (int64_t(p.n) + c) * ES);
            }
        }
    }
    if (!p.w) return;
    float v = acc.x + acc.y;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (team > 1) {
        if (lane == 0) part[warp] = v;
        __syncthreads();
        if (warp % team == 0) {
            v = part[warp];
            for (int i = 1; i < team; ++i) v += part[warp + i];
        }
    }
    if (lane == 0 && warp % team == 0 && row < p.M) {
        if (p.w_bf16) static_cast<__nv_bfloat16*>(p.dw)[row] = __float2bfloat16_rn(v);
        else static_cast<float*>(p.dw)[row] = v;
    }
}

// warps per row: one vector of eight columns per lane where the row is that wide, at most eight warps
int silu8_team(int64_t n, int vec) {
    int team = 1;
    while (team < 8 && team * 256 * vec < n) team *= 2;
    return team;
}

template <typename T, int CK>
int silu8_go(const Silu8Params& p, bool backward, cudaStream_t stream) {
    constexpr int VEC = sizeof(T) == 4 ? 1 : 2;
    const int team = silu8_team(p.n, VEC), teams = kSilu8Threads / 32 / team;
    const int64_t grid = (p.M + teams - 1) / teams;
    if (grid > 0x7fffffff) return fail_arg("silu_checkpoint: too many rows");
    if (backward) silu8_bwd_kernel<T, CK, VEC><<<unsigned(grid), kSilu8Threads, 0, stream>>>(p, team);
    else silu8_fwd_kernel<T, CK, VEC><<<unsigned(grid), kSilu8Threads, 0, stream>>>(p, team);
    return check_launch(backward ? "silu8_bwd_kernel" : "silu8_fwd_kernel");
}

int silu8_dispatch(const Silu8Params& p, int dtype, int codes, bool backward, cudaStream_t stream) {
    if (dtype == LH_BF16) return codes == CODES_INT8 ? silu8_go<__nv_bfloat16, CODES_INT8>(p, backward, stream) : silu8_go<__nv_bfloat16, CODES_E4M3>(p, backward, stream);
    if (dtype == LH_F16) return codes == CODES_INT8 ? silu8_go<__half, CODES_INT8>(p, backward, stream) : silu8_go<__half, CODES_E4M3>(p, backward, stream);
    return codes == CODES_INT8 ? silu8_go<float, CODES_INT8>(p, backward, stream) : silu8_go<float, CODES_E4M3>(p, backward, stream);
}

int silu8_check(const char* what, int dtype, int codes, const void* w, int w_dtype, int64_t M, int64_t n) {
    if (dtype != LH_BF16 && dtype != LH_F16 && dtype != LH_F32) return fail_arg("%s: dtype must be bf16, f16 or f32", what);
    if (codes != CODES_INT8 && codes != CODES_E4M3) return fail_arg("%s: codes must be 1 (int8) or 2 (e4m3)", what);
    if (w && w_dtype != LH_F32 && w_dtype != LH_BF16) return fail_arg("%s: weights must be f32 or bf16", what);
    if (M < 0 || n <= 0 || (n % 128) != 0 || n > 0x3fffffff) return fail_arg("%s: need n %% 128 == 0 (M=%lld n=%lld)", what, (long long)M, (long long)n);
    return LH_OK;
}

bool unaligned16(std::initializer_list<const void*> ps) {
    uintptr_t a = 0;
    for (const void* q : ps) a |= reinterpret_cast<uintptr_t>(q);
    return (a & 15) != 0;
}

}  // namespace

int silu8_fwd(const void* x, const void* w, int dtype, int w_dtype, int codes, int64_t M, int64_t n, void* y, void* q, float* s, cudaStream_t stream) {
    if (int rc = silu8_check("silu_checkpoint_fwd", dtype, codes, w, w_dtype, M, n)) return rc;
    if (M == 0) return LH_OK;
    if (!x || !y || !q || !s) return fail_arg("silu_checkpoint_fwd: NULL pointer");
    if (unaligned16({x, y, q})) return fail_arg("silu_checkpoint_fwd: pointers must be 16-byte aligned");
    Silu8Params p{};
    p.x = static_cast<const uint8_t*>(x); p.w = w; p.w_bf16 = w_dtype == LH_BF16; p.M = M; p.n = int(n);
    p.y = static_cast<uint8_t*>(y); p.q = static_cast<uint8_t*>(q); p.s = s;
    return silu8_dispatch(p, dtype, codes, false, stream);
}

int silu8_bwd(const void* g, const void* q, const float* s, const void* w, int dtype, int w_dtype, int codes, int64_t M, int64_t n,
              void* dx, void* dw, cudaStream_t stream) {
    if (int rc = silu8_check("silu_checkpoint_bwd", dtype, codes, w, w_dtype, M, n)) return rc;
    if (M == 0) return LH_OK;
    if (!g || !q || !s || !dx || (w && !dw)) return fail_arg("silu_checkpoint_bwd: NULL pointer");
    if (unaligned16({g, q, dx})) return fail_arg("silu_checkpoint_bwd: pointers must be 16-byte aligned");
    Silu8Params p{};
    p.g = static_cast<const uint8_t*>(g); p.xq = static_cast<const uint8_t*>(q); p.xs = s; p.w = w; p.w_bf16 = w_dtype == LH_BF16;
    p.M = M; p.n = int(n); p.dx = static_cast<uint8_t*>(dx); p.dw = dw;
    return silu8_dispatch(p, dtype, codes, true, stream);
}

}  // namespace lh

// SwiGLU that keeps its input as an 8-bit checkpoint, and its gradient from the checkpoint:
//
//   y = silu(x1) * x2 [* w_row],  x = [x1 | x2] [M, 2n];   codes of x in blocks of 1x128, [M, 2n], scales [M, 2n/128]
//   with x1, x2 the values of the codes, s = sigmoid(x1):
//   dw = sum g * x1 * s * x2;   gw = g * w;   dx1 = gw * x2 * s * (1 + x1 * (1 - s));   dx2 = gw * x1 * s
//
// Forward: 4 bytes read and 2 + 2 written per output element of a 16-bit type; backward: 2 + 2 read, 4 written.
// Nothing is read twice, so both are streams and HBM bounds them; what has to be kept up is the number of loads in flight.  A lane
// takes 32 bytes of x1 and of x2 (16 elements of a 16-bit type), so a block is eight lanes and its maximum three shuffles.
// Forward: a warp is done after one span, four warps to a CTA, 64 registers (16384 x 8192 bf16: 173 us, 95 % of the measured copy
// bandwidth; warps that walk a row 182 - 190, CTAs of eight warps 180).  Backward: a team of warps takes a row, since dw is a sum
// over it; 48 registers where every lane has one span (162 us, 102 %; 177 with 64 registers and a warp per row).
#include "lh_eight.cuh"

#include <algorithm>
#include <initializer_list>

namespace lh {

namespace {

constexpr int kSilu8FwdThreads = 128;
constexpr int kSilu8Threads = 256;

struct Silu8Params {
    const uint8_t *x, *g, *xq;
    const float* xs;
    const void* w;        // float32 or bf16 [M], may be NULL
    int w_bf16, wide;
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

// writes the codes and the scale of a lane's elements, whose block the lanes of an aligned group of 128 / kSpan share
template <int CK, typename T>
__device__ __forceinline__ void put_codes(const Lane<T>& x, bool live, uint8_t* q, float* scale, bool first) {
    constexpr int V = Lane<T>::V;
    float2 e[V][4];
    float amax = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[v][i] = x.v[v].get(i);
        amax = max_nan(amax, amax_pairs(e[v]));
    }
#pragma unroll
    for (int m = 8 / V; m >= 1; m >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, m));
    if (!live) return;               // not the zeros of a lane past the row: they would take the slow division
    const Divisor d(code_scale<CK>(amax));
    Codes<V> c;
#pragma unroll
    for (int v = 0; v < V; ++v) c.w[v] = encode8<CK>(e[v], d);
    c.store(q);
    if (first) *scale = d.s;
}

// a warp takes one span of 32 * kSpan columns of one row
template <typename T, int CK>
__global__ void __launch_bounds__(kSilu8FwdThreads, 1024 / kSilu8FwdThreads) silu8_fwd_kernel(const Silu8Params p, uint32_t spans) {
    constexpr int ES = sizeof(T), SPAN = kSpan<T>, V = SPAN / 8;
    const int lane = threadIdx.x & 31;
    const uint32_t unit = blockIdx.x * (kSilu8FwdThreads / 32) + (threadIdx.x >> 5);
    const uint32_t row32 = unit / spans;
    const int64_t row = row32;
    if (row >= p.M) return;                             // whole warps
    const int nb = p.n >> 7, c = int(unit - row32 * spans) * 32 * SPAN + lane * SPAN;
    const bool wide = p.wide != 0, live = c < p.n;
    const uint8_t* x1 = p.x + (row * 2 * p.n + c) * ES;
    const float wt = row_weight(p, row);
    Lane<T> a, b, y;
    a.zero();
    b.zero();
    if (live) {
        a.load(x1, wide);
        b.load(x1 + int64_t(p.n) * ES, wide);
    }
    uint8_t* q = p.q + row * 2 * p.n + c;
    float* scale = p.s + row * 2 * nb + (c >> 7);
    const bool first = (c & 127) == 0;
    put_codes<CK>(a, live, q, scale, first);
    put_codes<CK>(b, live, q + p.n, scale + nb, first);
    if (!live) return;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 va = a.v[v].get(i);
            y.v[v].set(i, mul2(mul2(mul2(va, sigmoid_fast2(va)), b.v[v].get(i)), splat2(wt)));
        }
    y.store(p.y + (row * p.n + c) * ES, wide);
}

// AHEAD: a lane has more than one span, the next one's loads are in flight while one is worked on
template <typename T, int CK, bool AHEAD>
__global__ void __launch_bounds__(kSilu8Threads, AHEAD ? 4 : 5) silu8_bwd_kernel(const Silu8Params p, int team) {
    constexpr int ES = sizeof(T), SPAN = kSpan<T>, V = SPAN / 8;
    __shared__ float part[kSilu8Threads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, teams = (blockDim.x >> 5) / team;
    const int64_t row = int64_t(blockIdx.x) * teams + warp / team;
    const int nb = p.n >> 7;
    const bool wide = p.wide != 0;
    float2 acc = make_float2(0.f, 0.f);
    if (row < p.M) {                                     // whole warps
        const uint8_t* xq = p.xq + row * 2 * p.n;
        const uint8_t* g = p.g + row * p.n * ES;
        const float* xs = p.xs + row * 2 * nb;
        uint8_t* dx = p.dx + row * 2 * p.n * ES;
        const float wt = row_weight(p, row);
        const int step = team * 32 * SPAN;
        Lane<T> g_next;
        Codes<V> q1_next, q2_next;
        float s1_next = 0.f, s2_next = 0.f;
        auto fetch = [&](int c) {
            if (c >= p.n) return;
            g_next.load(g + int64_t(c) * ES, wide);
            q1_next.load(xq + c);
            q2_next.load(xq + p.n + c);
            s1_next = xs[c >> 7];
            s2_next = xs[nb + (c >> 7)];
        };
        int c = (warp % team) * 32 * SPAN + lane * SPAN;
        fetch(c);
        for (; c < p.n; c += AHEAD ? step : p.n) {
            Lane<T> d1, d2;
            const Lane<T> gv = g_next;
            const Codes<V> q1 = q1_next, q2 = q2_next;
            const float s1 = s1_next, s2 = s2_next;
            if (AHEAD) fetch(c + step);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float2 x1[4], x2[4];
                decode8<CK>(q1.w[v], s1, x1);
                decode8<CK>(q2.w[v], s2, x2);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 sg = sigmoid_fast2(x1[i]), gr = gv.v[v].get(i);
                    const float2 si = mul2(x1[i], sg);                                 // silu(x1)
                    if (p.w) acc = fma2(mul2(gr, si), x2[i], acc);
                    const float2 gw = mul2(gr, splat2(wt));
                    // s * (1 + x1 * (1 - s)) = s + si * (1 - s)
                    const float2 ds = fma2(si, make_float2(1.f - sg.x, 1.f - sg.y), sg);
                    d1.v[v].set(i, mul2(mul2(gw, x2[i]), ds));
                    d2.v[v].set(i, mul2(gw, si));
                }
            }
            d1.store(dx + int64_t(c) * ES, wide);
            d2.store(dx + (int64_t(p.n) + c) * ES, wide);
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

// Warps per row: one for each span, at most eight; of the numbers that need as many steps the smallest, so that the last
// step is as full as can be.
int silu8_team(int spans) {
    const int steps = (spans + 7) / 8;
    return (spans + steps - 1) / steps;
}

template <typename T, int CK>
int silu8_go(const Silu8Params& p, bool backward, cudaStream_t stream) {
    if (backward) {
        // A warp alone on a row needs no barrier for the row's sum: 71 us against 90 (40001 x 1408, weighted), as long as
        // the rows fill the machine and are short; 8 warps on a row of 8192 take 162 us, one 177.
        const int spans = int((p.n + 32 * kSpan<T> - 1) / (32 * kSpan<T>));
        const int team = spans <= 4 && p.M >= 32 * sm_count() ? 1 : silu8_team(spans), teams = std::max(1, kSilu8Threads / 64 / team);
        const unsigned grid = unsigned((p.M + teams - 1) / teams), threads = 32u * team * teams;
        if (spans > team) silu8_bwd_kernel<T, CK, true><<<grid, threads, 0, stream>>>(p, team);
        else silu8_bwd_kernel<T, CK, false><<<grid, threads, 0, stream>>>(p, team);
        return check_launch("silu8_bwd_kernel");
    }
    const int64_t spans = (p.n + 32 * kSpan<T> - 1) / (32 * kSpan<T>);
    silu8_fwd_kernel<T, CK><<<unsigned((p.M * spans + kSilu8FwdThreads / 32 - 1) / (kSilu8FwdThreads / 32)), kSilu8FwdThreads, 0, stream>>>(p, uint32_t(spans));
    return check_launch("silu8_fwd_kernel");
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
    // the kernels number the warps' shares of the rows (at least 128 columns each) in 32 bits
    if (M > 0x7fffffff || M * (n / 128) > 0x7fffffff) return fail_arg("%s: too many rows (M=%lld n=%lld)", what, (long long)M, (long long)n);
    return LH_OK;
}

bool unaligned(std::initializer_list<const void*> ps, uintptr_t to = 16) {
    uintptr_t a = 0;
    for (const void* q : ps) a |= reinterpret_cast<uintptr_t>(q);
    return (a & (to - 1)) != 0;
}

}  // namespace

int silu8_fwd(const void* x, const void* w, int dtype, int w_dtype, int codes, int64_t M, int64_t n, void* y, void* q, float* s, cudaStream_t stream) {
    if (int rc = silu8_check("silu_checkpoint_fwd", dtype, codes, w, w_dtype, M, n)) return rc;
    if (M == 0) return LH_OK;
    if (!x || !y || !q || !s) return fail_arg("silu_checkpoint_fwd: NULL pointer");
    if (unaligned({x, y, q})) return fail_arg("silu_checkpoint_fwd: pointers must be 16-byte aligned");
    Silu8Params p{};
    p.x = static_cast<const uint8_t*>(x); p.w = w; p.w_bf16 = w_dtype == LH_BF16; p.M = M; p.n = int(n);
    p.wide = !unaligned({x, y}, 32);
    p.y = static_cast<uint8_t*>(y); p.q = static_cast<uint8_t*>(q); p.s = s;
    return silu8_dispatch(p, dtype, codes, false, stream);
}

int silu8_bwd(const void* g, const void* q, const float* s, const void* w, int dtype, int w_dtype, int codes, int64_t M, int64_t n,
              void* dx, void* dw, cudaStream_t stream) {
    if (int rc = silu8_check("silu_checkpoint_bwd", dtype, codes, w, w_dtype, M, n)) return rc;
    if (M == 0) return LH_OK;
    if (!g || !q || !s || !dx || (w && !dw)) return fail_arg("silu_checkpoint_bwd: NULL pointer");
    if (unaligned({g, q, dx})) return fail_arg("silu_checkpoint_bwd: pointers must be 16-byte aligned");
    Silu8Params p{};
    p.g = static_cast<const uint8_t*>(g); p.xq = static_cast<const uint8_t*>(q); p.xs = s; p.w = w; p.w_bf16 = w_dtype == LH_BF16;
    p.wide = !unaligned({g, dx}, 32);
    p.M = M; p.n = int(n); p.dx = static_cast<uint8_t*>(dx); p.dw = dw;
    return silu8_dispatch(p, dtype, codes, true, stream);
}

}  // namespace lh

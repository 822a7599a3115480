// The two norms around a residual sum as one operator, forward and backward:
//
//   p = o * r_post * post,  r_post = rsqrt(mean(o^2) + eps)      o: output of the block, [M, n]
//   h = round(x + alpha * gate * p)                              x: residual stream
//   y = h * r_pre * pre,    r_pre  = rsqrt(mean(h^2) + eps)      input of the next block
//
// and for gradients dy of y and dh_in of h, with hn = h * r_pre, on = o * r_post:
//
//   t  = dy * pre;   dh = dx = dh_in + r_pre * (t - hn * mean(t * hn))
//   dp = alpha * gate * dh;   u = dp * post;   do = r_post * (u - on * mean(u * on))
//   dpre = sum dy * hn;   dpost = sum dp * on;   dgate = sum alpha * dh * on * post
//
// Both are one pass over HBM: 8 bytes per element forward (16-bit types), 12 backward, 10 with o and h
// kept as 8-bit codes.  What has to be waited for is the row: two sums over it, one after the other, so
// a row's tensors are brought to shared memory by bulk copies several rows ahead of the row being
// worked on, and a thread keeps the columns it owns (the 8-element vectors t and t + NT of a row) for the
// whole walk: gamma and the gradient sums of those columns stay in its registers.
#include "lh_eight.cuh"

#include <algorithm>
#include <type_traits>

namespace lh {

namespace {

constexpr int kPairMaxN = 8192;
constexpr int kPairMaxThreads = kPairMaxN / 16;
constexpr int kPairMaxStages = 4;
constexpr int kPairSmem = 227 * 1024;      // shared memory of an SM that CTAs can ask for
constexpr int kPairSlack = 1536;           // per CTA: static shared memory, what the system reserves, rounding

struct PairParams {
    const uint8_t *x, *o, *post, *pre, *gate;   // forward: x, o.  backward: o, h (values or codes)
    const uint8_t *dy, *dh, *hsrc;
    const float *os_in, *hs_in;                 // scales of the codes of o and h, [M, n / 128]
    int64_t M, G;                               // gate: G rows, row i takes gate row i % G
    int n;
    int stages;
    float alpha, eps, inv_n;
    uint8_t *h, *y, *dx, *dout;
    float *r_post, *r_pre;
    uint8_t *oq, *hq;                           // checkpoints of o and h (forward)
    float *os, *hs;
    float* part;                                // backward: the CTAs' sums
    uint8_t* dgate;
};

// Sum over the CTA.  buf has a place for each of 16 warps, those of absent warps zeroed; it is written
// again only behind another barrier of the caller.
__device__ __forceinline__ float cta_sum(float v, float* buf) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    float4 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = reinterpret_cast<const float4*>(buf)[i];
    float r = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) r += (s[i].x + s[i].y) + (s[i].z + s[i].w);
    return r;
}

// the codes of one block of 128 elements (16 lanes, eight elements each) and its scale; every lane of a warp comes here
template <int CK>
__device__ __forceinline__ void put_codes(const float2* e, bool live, uint8_t* q, float* scales, int64_t row, int n, int col) {
    const float scale = code_scale<CK>(block_amax(amax_pairs(e)));
    if (live) {     // blocks do not straddle the end of a row: n is a multiple of 128
        *reinterpret_cast<uint2*>(q + row * n + col) = encode8<CK>(e, Divisor(scale));
        if ((threadIdx.x & 15) == 0) scales[row * (n >> 7) + (col >> 7)] = scale;
    }
}

enum : int { GATE_NONE = 0, GATE_ROW = 1, GATE_ROWS = 2 };

// ---- forward ---------------------------------------------------------------------------------
// A gate of several rows is brought in with the row; where there is one row of it or none, alpha * gate * post is
// one float32 coefficient per column.
template <typename T, int CK, bool ROWS>
__global__ void __launch_bounds__(kPairMaxThreads, sizeof(T) == 2 ? 2 : 1) pair_fwd_kernel(const PairParams p) {
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t full[kPairMaxStages];
    __shared__ __align__(16) float sum_o[16], sum_h[16];
    constexpr int ES = sizeof(T), NTEN = ROWS ? 3 : 2;
    const int t = threadIdx.x, nt = blockDim.x, S = p.stages;
    const uint32_t row_bytes = uint32_t(p.n) * ES, stage_bytes = NTEN * row_bytes;
    const int64_t step = gridDim.x;

    auto fetch = [&](int64_t row, int s) {
        uint8_t* dst = ring + size_t(s) * stage_bytes;
        mbar_expect_tx(&full[s], stage_bytes);
        bulk_g2s(dst, p.o + row * row_bytes, row_bytes, &full[s]);
        bulk_g2s(dst + row_bytes, p.x + row * row_bytes, row_bytes, &full[s]);
        if (ROWS) bulk_g2s(dst + 2 * row_bytes, p.gate + (row % p.G) * row_bytes, row_bytes, &full[s]);
    };
    if (t == 0) {
        for (int s = 0; s < S; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
        for (int s = 0; s < S && blockIdx.x + s * step < p.M; ++s) fetch(blockIdx.x + s * step, s);
    }
    if (t < 16) sum_o[t] = sum_h[t] = 0.f;

    const int col[2] = {t * 8, (t + nt) * 8};
    const bool live[2] = {col[0] < p.n, col[1] < p.n};
    Vec8<T> pre[2];
    float2 coef[8];      // alpha * post [* gate]
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        Vec8<T> w, g;
        w.zero(); g.zero(); pre[v].zero();
        if (live[v]) {
            w.load(p.post + col[v] * ES);
            if (!ROWS && p.gate) g.load(p.gate + col[v] * ES);
            if (ES == 2) pre[v].load(p.pre + col[v] * ES);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            coef[4 * v + i] = mul2(w.get(i), splat2(p.alpha));
            if (!ROWS && p.gate) coef[4 * v + i] = mul2(coef[4 * v + i], g.get(i));
        }
    }
    __syncthreads();

    bool dead = false;
    int s = 0;
    uint32_t phase = 0;
    for (int64_t row = blockIdx.x; row < p.M; row += step) {
        mbar_wait_or_mark<true>(&full[s], phase, DEVERR_FULL_WAIT, dead);
        const uint8_t* so = ring + size_t(s) * stage_bytes;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            Vec8<T> o;
            o.zero();
            if (live[v]) o.load(so + col[v] * ES);
            float2 e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                e[i] = o.get(i);
                acc = fma2(e[i], e[i], acc);
            }
            if constexpr (CK != CODES_NONE) put_codes<CK>(e, live[v], p.oq, p.os, row, p.n, col[v]);
        }
        const float rp = __frsqrt_rn(fmaf(cta_sum(acc.x + acc.y, sum_o), p.inv_n, p.eps));

        Vec8<T> h[2];
        acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            h[v].zero();
            if (live[v]) {
                Vec8<T> x, o, g;
                o.load(so + col[v] * ES);
                x.load(so + row_bytes + col[v] * ES);
                if (ROWS) g.load(so + 2 * row_bytes + col[v] * ES);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 q = mul2(o.get(i), splat2(rp));
                    if (ROWS) q = mul2(q, g.get(i));
                    h[v].set(i, fma2(q, coef[4 * v + i], x.get(i)));
                }
                h[v].store(p.h + row * row_bytes + col[v] * ES);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc = fma2(h[v].get(i), h[v].get(i), acc);
        }
        const float rh = __frsqrt_rn(fmaf(cta_sum(acc.x + acc.y, sum_h), p.inv_n, p.eps));
        // behind that barrier every thread has read the stage
        if (t == 0) {
            if (row + S * step < p.M) fetch(row + S * step, s);
            p.r_post[row] = rp;
            p.r_pre[row] = rh;
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            if (live[v]) {
                Vec8<T> y, w;
                if (ES == 2) w = pre[v]; else w.load(p.pre + col[v] * ES);
#pragma unroll
                for (int i = 0; i < 4; ++i) y.set(i, mul2(mul2(h[v].get(i), splat2(rh)), w.get(i)));
                y.store(p.y + row * row_bytes + col[v] * ES);
            }
            if constexpr (CK != CODES_NONE) {
                float2 e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = h[v].get(i);
                put_codes<CK>(e, live[v], p.hq, p.hs, row, p.n, col[v]);
            }
        }
        if (++s == S) { s = 0; phase ^= 1u; }
    }
}

// ---- backward --------------------------------------------------------------------------------
// Rows in the order of the gate's groups (all rows of gate row 0 first): position j is row
// j / R + (j % R) * G, R = M / G.  CTA b takes the positions [first(b), first(b + 1)), so that every CTA
// has the same share of rows whatever the number of groups, and a group's gradient is the sum of at most one
// sum per CTA.  A group that lies inside one CTA is written by it; one that several share goes through scratch.
//
// B = sum dh * on is the one sum behind two gradients: dgate = alpha * post * B over the gate's group, and
// dpost = alpha * sum over the groups of gate * B.  With one gate row or none the CTAs keep B alone (and the
// sum for dpre), the reduction forms both; with several rows dpost has sums of its own.
__host__ __device__ __forceinline__ int64_t pair_first(int64_t b, int64_t grid, int64_t M) {
    const int64_t q = M / grid, r = M % grid;
    return b * q + (b < r ? b : r);
}

// scratch: [grid][PART_ROWS][n] float32
enum : int { PART_PRE = 0, PART_POST = 1, PART_HEAD = 2, PART_TAIL = 3, PART_ROWS = 4 };   // PART_POST: B itself with one gate row or none

template <typename T, int CK, int GATE>
__global__ void __launch_bounds__(kPairMaxThreads, 1) pair_bwd_kernel(const PairParams p) {
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t full[kPairMaxStages];
    __shared__ __align__(16) float sum_h[16], sum_o[16];
    constexpr bool ROWS = GATE == GATE_ROWS;
    constexpr int ES = sizeof(T), CS = CK == CODES_NONE ? ES : 1;   // bytes of an element of dy / of o and h
    const int t = threadIdx.x, nt = blockDim.x, S = p.stages;
    const uint32_t row_bytes = uint32_t(p.n) * ES, code_bytes = uint32_t(p.n) * CS;
    const bool has_dh = p.dh != nullptr;
    // a stage: dy | o | h | gate row (if the gate has several) | dh (if given)
    const uint32_t off_o = row_bytes, off_h = off_o + code_bytes, off_g = off_h + code_bytes, off_dh = off_g + (ROWS ? row_bytes : 0u),
                   stage_bytes = off_dh + (has_dh ? row_bytes : 0u);
    const int64_t G = ROWS ? p.G : 1, R = p.M / G;
    const int64_t begin = pair_first(blockIdx.x, gridDim.x, p.M), end = pair_first(blockIdx.x + 1, gridDim.x, p.M);

    auto fetch = [&](int64_t j, int s) {
        const int64_t g = ROWS ? j / R : 0, row = ROWS ? g + (j - g * R) * G : j;
        uint8_t* dst = ring + size_t(s) * stage_bytes;
        mbar_expect_tx(&full[s], stage_bytes);
        bulk_g2s(dst, p.dy + row * row_bytes, row_bytes, &full[s]);
        bulk_g2s(dst + off_h, p.hsrc + row * code_bytes, code_bytes, &full[s]);
        bulk_g2s(dst + off_o, p.o + row * code_bytes, code_bytes, &full[s]);
        if (has_dh) bulk_g2s(dst + off_dh, p.dh + row * row_bytes, row_bytes, &full[s]);
        if (ROWS) bulk_g2s(dst + off_g, p.gate + g * row_bytes, row_bytes, &full[s]);
    };
    if (t == 0) {
        for (int s = 0; s < S; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
        for (int s = 0; s < S && begin + s < end; ++s) fetch(begin + s, s);
    }
    if (t < 16) sum_h[t] = sum_o[t] = 0.f;

    const int col[2] = {t * 8, (t + nt) * 8};
    const bool live[2] = {col[0] < p.n, col[1] < p.n};
    Vec8<T> pre[2];
    float2 coef[8];      // alpha * post [* gate]
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        Vec8<T> w, g;
        w.zero(); g.zero(); pre[v].zero();
        if (live[v]) {
            w.load(p.post + col[v] * ES);
            if (GATE == GATE_ROW) g.load(p.gate + col[v] * ES);
            if (ES == 2) pre[v].load(p.pre + col[v] * ES);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            coef[4 * v + i] = mul2(w.get(i), splat2(p.alpha));
            if (GATE == GATE_ROW) coef[4 * v + i] = mul2(coef[4 * v + i], g.get(i));
        }
    }
    float2 a_pre[8], a_b[8], a_post[ROWS ? 8 : 1];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a_pre[i] = a_b[i] = make_float2(0.f, 0.f);
        if (ROWS) a_post[i] = make_float2(0.f, 0.f);
    }
    __syncthreads();

    // scales of the codes and 1/rms of a row, fetched one row ahead
    struct RowScalars { float so[2], sh[2], rp, rh; };
    auto scalars = [&](int64_t j) {
        RowScalars q{};
        if (j < end) {
            const int64_t g = ROWS ? j / R : 0, row = ROWS ? g + (j - g * R) * G : j;
            q.rp = p.r_post[row];
            q.rh = p.r_pre[row];
            if constexpr (CK != CODES_NONE) {
#pragma unroll
                for (int v = 0; v < 2; ++v)
                    if (live[v]) {
                        const int64_t at = row * (p.n >> 7) + (col[v] >> 7);
                        q.so[v] = p.os_in[at];
                        q.sh[v] = p.hs_in[at];
                    }
            }
        }
        return q;
    };
    // this CTA's sum of the gradient of gate row g, whose positions are [g R, (g + 1) R)
    auto flush_gate = [&](int64_t g) {
        const bool whole = g * R >= begin && (g + 1) * R <= end;
        float* slot = p.part + (int64_t(blockIdx.x) * PART_ROWS + (g * R < begin ? PART_HEAD : PART_TAIL)) * p.n;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            float2 d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                d[i] = mul2(a_b[4 * v + i], coef[4 * v + i]);
                a_b[4 * v + i] = make_float2(0.f, 0.f);
            }
            if (live[v]) {
                if (whole) {
                    Vec8<T> w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) w.set(i, d[i]);
                    w.store(p.dgate + g * row_bytes + col[v] * ES);
                } else {
                    float4* dst = reinterpret_cast<float4*>(slot + col[v]);
                    dst[0] = make_float4(d[0].x, d[0].y, d[1].x, d[1].y);
                    dst[1] = make_float4(d[2].x, d[2].y, d[3].x, d[3].y);
                }
            }
        }
    };

    bool dead = false;
    int s = 0;
    uint32_t phase = 0;
    RowScalars next = scalars(begin);
    int64_t g = ROWS ? begin / R : 0, g_end = (g + 1) * R;      // group of the row, position where it ends
    for (int64_t j = begin; j < end; ++j) {
        const RowScalars cur = next;
        next = scalars(j + 1);
        if (ROWS && j == g_end) { flush_gate(g); ++g; g_end += R; }
        const int64_t row = ROWS ? g + (j - g * R) * G : j;
        mbar_wait_or_mark<true>(&full[s], phase, DEVERR_FULL_WAIT, dead);
        const uint8_t* st = ring + size_t(s) * stage_bytes;

        auto values = [&](uint32_t off, int v, float scale, float2* e) {   // o or h
            if constexpr (CK == CODES_NONE) {
                Vec8<T> w;
                w.load(st + off + col[v] * ES);
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = w.get(i);
            } else {
                decode8<CK>(*reinterpret_cast<const uint2*>(st + off + col[v]), scale, e);
            }
        };
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < 2; ++v)
            if (live[v]) {
                Vec8<T> dy, w;
                float2 h[4];
                dy.load(st + col[v] * ES);
                values(off_h, v, cur.sh[v], h);
                if (ES == 2) w = pre[v]; else w.load(p.pre + col[v] * ES);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc = fma2(mul2(dy.get(i), w.get(i)), h[i], acc);
            }
        const float rh = cur.rh, rp = cur.rp;
        const float ch = cta_sum(acc.x + acc.y, sum_h) * p.inv_n * rh * rh;      // mean(t * hn) * r_pre
        acc = make_float2(0.f, 0.f);
        float2 u[8];
#pragma unroll
        for (int v = 0; v < 2; ++v)
            if (live[v]) {
                Vec8<T> dy, din, w, gt, dx;
                float2 h[4], o[4];
                dy.load(st + col[v] * ES);
                values(off_h, v, cur.sh[v], h);
                values(off_o, v, cur.so[v], o);
                if (has_dh) din.load(st + off_dh + col[v] * ES); else din.zero();
                if (ES == 2) w = pre[v]; else w.load(p.pre + col[v] * ES);
                if (ROWS) gt.load(st + off_g + col[v] * ES);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 hn = mul2(h[i], splat2(rh)), gy = dy.get(i), on = mul2(o[i], splat2(rp));
                    float2 d = fma2(hn, splat2(-ch), mul2(mul2(gy, w.get(i)), splat2(rh)));
                    d = add2(d, din.get(i));
                    dx.set(i, d);
                    a_pre[4 * v + i] = fma2(gy, hn, a_pre[4 * v + i]);
                    a_b[4 * v + i] = fma2(d, on, a_b[4 * v + i]);
                    if constexpr (ROWS) {
                        d = mul2(d, gt.get(i));
                        a_post[4 * v + i] = fma2(d, on, a_post[4 * v + i]);
                    }
                    u[4 * v + i] = mul2(d, coef[4 * v + i]);
                    acc = fma2(u[4 * v + i], o[i], acc);
                }
                dx.store(p.dx + row * row_bytes + col[v] * ES);
            }
        const float co = cta_sum(acc.x + acc.y, sum_o) * p.inv_n * rp * rp;      // mean(u * on) * r_post
#pragma unroll
        for (int v = 0; v < 2; ++v)
            if (live[v]) {
                Vec8<T> d;
                float2 o[4];
                values(off_o, v, cur.so[v], o);
#pragma unroll
                for (int i = 0; i < 4; ++i) d.set(i, fma2(mul2(o[i], splat2(rp)), splat2(-co), mul2(u[4 * v + i], splat2(rp))));
                d.store(p.dout + row * row_bytes + col[v] * ES);
            }
        __syncthreads();      // every thread has read the stage
        if (t == 0 && j + S < end) fetch(j + S, s);
        if (++s == S) { s = 0; phase ^= 1u; }
    }
    if (ROWS) flush_gate(g);      // begin < end: the grid has no more CTAs than there are rows
    float* part = p.part + int64_t(blockIdx.x) * PART_ROWS * p.n;
#pragma unroll
    for (int v = 0; v < 2; ++v)
        if (live[v]) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 *a = a_pre + 4 * v + 2 * i, *b = ROWS ? a_post + (ROWS ? 4 * v + 2 * i : 0) : a_b + 4 * v + 2 * i;
                reinterpret_cast<float4*>(part + PART_PRE * p.n + col[v])[i] = make_float4(a[0].x, a[0].y, a[1].x, a[1].y);
                reinterpret_cast<float4*>(part + PART_POST * p.n + col[v])[i] = make_float4(b[0].x, b[0].y, b[1].x, b[1].y);
            }
        }
}

// The CTAs' sums, added in the order of the CTAs: blockIdx.y 0 dpre, 1 dpost (and the gradient of a gate of one row),
// from 2 on the gate's groups that several CTAs share.
template <typename T>
__global__ void __launch_bounds__(1024) pair_reduce_kernel(const float* part, int ctas, int64_t M, int64_t G, int n, float alpha,
                                                           const T* post, const T* gate, float* dpost, float* dpre, T* dgate) {
    __shared__ float red[32][33];
    const int c = threadIdx.x & 31, l = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + c;             // n is a multiple of 128
    const int64_t R = M / G;
    // where there are fewer groups than borders between CTAs every group is looked at, else every border
    const int64_t borders = ctas - 1, looks = G > 1 ? (G <= borders ? G : borders) : 0;
    for (int64_t k = blockIdx.y; k < 2 + looks; k += gridDim.y) {
        int64_t b0 = 0, b1 = ctas, g = 0;            // CTAs [b0, b1), their rows of scratch
        int first = int(k), others = int(k);
        if (k >= 2) {
            g = k - 2;
            if (G > borders) {
                const int64_t at = pair_first(k - 1, ctas, M);        // where CTA k - 1 begins
                g = at / R;
                if (at == g * R || pair_first(k - 2, ctas, M) > g * R) continue;   // between two groups, or not the group's first border
            }
            b0 = g * R * ctas / M;
            while (b0 > 0 && pair_first(b0, ctas, M) > g * R) --b0;
            while (pair_first(b0 + 1, ctas, M) <= g * R) ++b0;
            b1 = b0 + 1;
            while (b1 < ctas && pair_first(b1, ctas, M) < (g + 1) * R) ++b1;
            if (b1 == b0 + 1) continue;              // one CTA has the whole group and has written it
            first = PART_TAIL;
            others = PART_HEAD;
        }
        float a = 0.f;
        for (int64_t b = b0 + l; b < b1; b += 32) a += part[(b * PART_ROWS + (b == b0 ? first : others)) * n + col];
        red[l][c] = a;
        __syncthreads();
        if (l == 0) {
            float v = red[0][c];
#pragma unroll
            for (int i = 1; i < 32; ++i) v += red[i][c];
            if (k == 0) {
                dpre[col] = v;
            } else if (k == 1) {
                if (G > 1) v *= alpha;
                else {
                    v *= alpha;
                    if (gate) {
                        dgate[col] = T(v * float(post[col]));
                        v *= float(gate[col]);
                    }
                }
                dpost[col] = v;
            } else {
                dgate[g * n + col] = T(v);
            }
        }
        __syncthreads();
    }
}

int pair_threads(int64_t n) { return int((n / 16 + 31) / 32 * 32); }

// CTAs per SM and stages for rows of `bytes` per stage: `threads` in all on an SM, at least two stages
void pair_shape(int threads_per_sm, int nt, int64_t bytes, int& per_sm, int& stages) {
    per_sm = std::max(1, std::min(32, threads_per_sm / nt));
    while (true) {
        stages = int(std::min<int64_t>(kPairMaxStages, (kPairSmem / per_sm - kPairSlack) / bytes));
        if (stages >= 2 || per_sm == 1) break;
        per_sm = (per_sm + 1) / 2;
    }
    stages = std::max(stages, 1);
}

constexpr int kPairBwdThreadsPerSm = 512;   // 128 registers a thread

template <typename F>
int pair_launch(F kern, int64_t grid, int nt, int64_t smem, const PairParams& p, const char* what, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return int(e); }
    kern<<<unsigned(grid), nt, size_t(smem), stream>>>(p);
    return check_launch(what);
}

template <typename T>
int pair_fwd_typed(PairParams& p, int ck, cudaStream_t stream) {
    const int nt = pair_threads(p.n);
    const bool gated = p.gate && p.G > 1;
    const int64_t bytes = int64_t(p.n) * sizeof(T) * (gated ? 3 : 2);
    int per_sm;
    pair_shape(1024 / (sizeof(T) == 2 ? 1 : 2), nt, bytes, per_sm, p.stages);
    const int64_t grid = std::min<int64_t>(p.M, int64_t(sm_count()) * per_sm);
    auto go = [&](auto kern) { return pair_launch(kern, grid, nt, bytes * p.stages, p, "pair_fwd_kernel", stream); };
    if (ck == CODES_INT8) return gated ? go(pair_fwd_kernel<T, CODES_INT8, true>) : go(pair_fwd_kernel<T, CODES_INT8, false>);
    if (ck == CODES_E4M3) return gated ? go(pair_fwd_kernel<T, CODES_E4M3, true>) : go(pair_fwd_kernel<T, CODES_E4M3, false>);
    return gated ? go(pair_fwd_kernel<T, CODES_NONE, true>) : go(pair_fwd_kernel<T, CODES_NONE, false>);
}

int64_t pair_bwd_grid(int64_t M, int64_t n) {
    return std::min<int64_t>(M, int64_t(sm_count()) * std::max(1, std::min(32, kPairBwdThreadsPerSm / pair_threads(n))));
}

template <typename T>
int pair_bwd_typed(PairParams& p, int ck, float* dpost, float* dpre, cudaStream_t stream) {
    const int nt = pair_threads(p.n);
    const int64_t code = ck == CODES_NONE ? int64_t(sizeof(T)) : 1;
    const int64_t bytes = p.n * (int64_t(sizeof(T)) * (1 + (p.dh ? 1 : 0) + (p.gate && p.G > 1 ? 1 : 0)) + 2 * code);
    int per_sm;
    pair_shape(kPairBwdThreadsPerSm, nt, bytes, per_sm, p.stages);
    const int64_t grid = std::min(pair_bwd_grid(p.M, p.n), int64_t(sm_count()) * per_sm);
    auto go = [&](auto kern) { return pair_launch(kern, grid, nt, bytes * p.stages, p, "pair_bwd_kernel", stream); };
    int rc;
    auto with = [&](auto codes) {
        constexpr int CK = decltype(codes)::value;
        if (!p.gate) return go(pair_bwd_kernel<T, CK, GATE_NONE>);
        return p.G > 1 ? go(pair_bwd_kernel<T, CK, GATE_ROWS>) : go(pair_bwd_kernel<T, CK, GATE_ROW>);
    };
    if (ck == CODES_INT8) rc = with(std::integral_constant<int, CODES_INT8>{});
    else if (ck == CODES_E4M3) rc = with(std::integral_constant<int, CODES_E4M3>{});
    else rc = with(std::integral_constant<int, CODES_NONE>{});
    if (rc) return rc;
    const int64_t looks = p.gate && p.G > 1 ? std::min<int64_t>(p.G, grid - 1) : 0;
    pair_reduce_kernel<T><<<dim3(unsigned(p.n / 32), unsigned(2 + std::min<int64_t>(looks, 8))), 1024, 0, stream>>>(
        p.part, int(grid), p.M, p.gate ? p.G : 1, p.n, p.alpha, reinterpret_cast<const T*>(p.post), reinterpret_cast<const T*>(p.gate),
        dpost, dpre, reinterpret_cast<T*>(p.dgate));
    return check_launch("pair_reduce_kernel");
}

bool unaligned(std::initializer_list<const void*> ps) {
    uintptr_t a = 0;
    for (const void* q : ps) a |= reinterpret_cast<uintptr_t>(q);
    return (a & 15) != 0;
}

int pair_check(const char* what, int dtype, int64_t M, int64_t n, const void* gate, int64_t G, int codes) {
    if (dtype != LH_BF16 && dtype != LH_F16 && dtype != LH_F32) return fail_arg("%s: dtype must be bf16, f16 or f32", what);
    if (M < 0 || n <= 0 || n > kPairMaxN || (n % 128) != 0)
        return fail_arg("%s: need n %% 128 == 0 and n <= %d (M=%lld n=%lld)", what, kPairMaxN, (long long)M, (long long)n);
    if (codes < CODES_NONE || codes > CODES_E4M3) return fail_arg("%s: codes must be 0 (none), 1 (int8) or 2 (e4m3)", what);
    if (gate && M > 0 && (G <= 0 || M % G != 0)) return fail_arg("%s: the rows must be a multiple of the gate's rows (M=%lld, gate rows %lld)", what, (long long)M, (long long)G);
    return LH_OK;
}

}  // namespace

int64_t pair_bwd_scratch(int64_t M, int64_t n) {
    if (M <= 0 || n <= 0 || n > kPairMaxN) return 0;
    return pair_bwd_grid(M, n) * PART_ROWS * n * 4;
}

int pair_fwd(const void* x, const void* o, const void* post, const void* pre, const void* gate, int dtype, int64_t M, int64_t n,
             int64_t G, float alpha, float eps, int codes, void* h, void* y, float* r_post, float* r_pre, void* oq, float* os,
             void* hq, float* hs, cudaStream_t stream) {
    if (int rc = pair_check("rmsnorm_pair_fwd", dtype, M, n, gate, G, codes)) return rc;
    if (M == 0) return LH_OK;
    if (!x || !o || !post || !pre || !h || !y || !r_post || !r_pre) return fail_arg("rmsnorm_pair_fwd: NULL pointer");
    if (codes && (!oq || !os || !hq || !hs)) return fail_arg("rmsnorm_pair_fwd: NULL checkpoint pointer");
    if (unaligned({x, o, post, pre, gate, h, y}) || (codes && unaligned({oq, hq}))) return fail_arg("rmsnorm_pair_fwd: pointers must be 16-byte aligned");
    PairParams p{};
    auto b = [](const void* q) { return static_cast<const uint8_t*>(q); };
    p.x = b(x); p.o = b(o); p.post = b(post); p.pre = b(pre); p.gate = b(gate);
    p.M = M; p.G = G; p.n = int(n); p.alpha = alpha; p.eps = eps; p.inv_n = 1.0f / float(n);
    p.h = static_cast<uint8_t*>(h); p.y = static_cast<uint8_t*>(y); p.r_post = r_post; p.r_pre = r_pre;
    p.oq = static_cast<uint8_t*>(oq); p.os = os; p.hq = static_cast<uint8_t*>(hq); p.hs = hs;
    if (dtype == LH_BF16) return pair_fwd_typed<__nv_bfloat16>(p, codes, stream);
    if (dtype == LH_F16) return pair_fwd_typed<__half>(p, codes, stream);
    return pair_fwd_typed<float>(p, codes, stream);
}

int pair_bwd(const void* dy, const void* dh, const void* o, const float* os, const void* h, const float* hs, const void* post,
             const void* pre, const void* gate, const float* r_post, const float* r_pre, int dtype, int64_t M, int64_t n, int64_t G,
             float alpha, int codes, void* dx, void* dout, float* dpost, float* dpre, void* dgate, void* scratch,
             int64_t scratch_bytes, cudaStream_t stream) {
    if (int rc = pair_check("rmsnorm_pair_bwd", dtype, M, n, gate, G, codes)) return rc;
    if (!dpost || !dpre || (gate && !dgate)) return fail_arg("rmsnorm_pair_bwd: NULL pointer");
    if (M == 0) {      // sums over no rows
        for (float* d : {dpost, dpre}) {
            const cudaError_t e = cudaMemsetAsync(d, 0, size_t(n) * 4, stream);
            if (e != cudaSuccess) { set_error("cudaMemsetAsync: %s", cudaGetErrorString(e)); return int(e); }
        }
        if (gate && G > 0) {
            const cudaError_t e = cudaMemsetAsync(dgate, 0, size_t(G) * n * (dtype == LH_F32 ? 4 : 2), stream);
            if (e != cudaSuccess) { set_error("cudaMemsetAsync: %s", cudaGetErrorString(e)); return int(e); }
        }
        return LH_OK;
    }
    if (!dy || !o || !h || !post || !pre || !r_post || !r_pre || !dx || !dout || !scratch) return fail_arg("rmsnorm_pair_bwd: NULL pointer");
    if (codes && (!os || !hs)) return fail_arg("rmsnorm_pair_bwd: NULL scales");
    if (unaligned({dy, dh, o, h, post, pre, gate, dx, dout, dgate, scratch})) return fail_arg("rmsnorm_pair_bwd: pointers must be 16-byte aligned");
    if (scratch_bytes < pair_bwd_scratch(M, n)) return fail_arg("rmsnorm_pair_bwd: scratch too small (%lld < %lld bytes)", (long long)scratch_bytes, (long long)pair_bwd_scratch(M, n));
    PairParams p{};
    auto b = [](const void* q) { return static_cast<const uint8_t*>(q); };
    p.dy = b(dy); p.dh = b(dh); p.o = b(o); p.os_in = os; p.hsrc = b(h); p.hs_in = hs; p.post = b(post); p.pre = b(pre); p.gate = b(gate);
    p.r_post = const_cast<float*>(r_post); p.r_pre = const_cast<float*>(r_pre);
    p.M = M; p.G = G; p.n = int(n); p.alpha = alpha; p.inv_n = 1.0f / float(n);
    p.dx = static_cast<uint8_t*>(dx); p.dout = static_cast<uint8_t*>(dout); p.dgate = static_cast<uint8_t*>(gate ? dgate : nullptr);
    p.part = static_cast<float*>(scratch);
    if (dtype == LH_BF16) return pair_bwd_typed<__nv_bfloat16>(p, codes, dpost, dpre, stream);
    if (dtype == LH_F16) return pair_bwd_typed<__half>(p, codes, dpost, dpre, stream);
    return pair_bwd_typed<float>(p, codes, dpost, dpre, stream);
}

}  // namespace lh

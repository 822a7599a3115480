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
// kept as 8-bit codes.  What has to be waited for is the row: two sums over it, one after the other.  The codes save memory between
// the passes and little time: decoding them, some of them twice, costs the gradient 41 instructions per element instead of 35
// (16384 x 4096 bf16 from tensors, int8, e4m3: 142, 131, 127 us; without dh 127, 128, 124, where the bytes would allow 83 from codes).
#include "lh_eight.cuh"

#include <algorithm>
#include <type_traits>

namespace lh {

namespace {

constexpr int kPairMaxN = 8192;
constexpr int kPairMaxThreads = kPairMaxN / 16;
constexpr int kPairOneMaxN = 5120;          // backward, rows of one vector a thread: up to 640 threads, 96 registers each
constexpr int kPairThreadsPerSm = 512;     // backward, 128 registers a thread
constexpr int kPairMaxStages = 4;
constexpr int kPairSmem = 227 * 1024;      // shared memory of an SM that CTAs can ask for
constexpr int kPairSlack = 5120;           // per CTA: static shared memory, what the system reserves, rounding

struct PairParams {
    const uint8_t *x, *o, *post, *pre, *gate;   // forward: x, o.  backward: o, h (values or codes)
    const uint8_t *dy, *dh, *hsrc;
    const float *os_in, *hs_in;                 // scales of the codes of o and h, [M, n / 128]
    int64_t M, G;                               // gate: G rows, row i takes gate row i % G
    int n;
    int stages, wide;
    float alpha, eps, inv_n;
    uint8_t *h, *y, *dx, *dout;
    float *r_post, *r_pre;
    uint8_t *oq, *hq;                           // checkpoints of o and h (forward)
    float *os, *hs;
    float* part;                                // backward: the CTAs' sums
    uint8_t* dgate;
};

// Sum over the CTA.  buf has a place for each of W warps, those of absent warps zeroed; it is written
// again only behind another barrier of the caller.
template <int W = 16>
__device__ __forceinline__ float cta_sum(float v, float* buf) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buf[threadIdx.x & (W - 1)];
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

enum : int { GATE_NONE = 0, GATE_ROW = 1, GATE_GROUPS = 2, GATE_EACH = 3 };   // gate rows: none, one, fewer than rows, as many as rows

// ---- forward ---------------------------------------------------------------------------------
// One CTA per row, a thread 32 consecutive bytes of it in registers, every load of the row asked for at once: with
// 64 registers 1024 threads are resident, so four rows of 4096 are on their way to an SM while others are normalised
// or stored.  Coefficients (the same for every row) come from L1 and L2: with the row where registers allow it (16-bit
// types without checkpoints, 87 us; 88 where they are fetched when wanted), behind the sums elsewhere (with int8
// checkpoints 122 us, 155 - 175 the other way).
// Measured at 16384 x 4096, bf16: 87 us (94 % of the measured copy bandwidth), 92 with a gate.  A persistent walk fed by bulk copies through a
// shared-memory ring took 92 - 102 us whatever its depth, order of rows, rows per step or cache hints, and 4.2 us
// instead of 3.2 for 16 rows.

// the codes of one block of 128 elements (16 / V lanes, 8 V elements each) and its scale; every lane of a warp comes here
template <int CK, typename T>
__device__ __forceinline__ void put_codes(const Lane<T>& d, bool live, uint8_t* q, float* scales, int64_t row, int n, int col) {
    constexpr int V = Lane<T>::V;
    float2 e[V][4];
    float amax = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[v][i] = d.v[v].get(i);
        amax = max_nan(amax, amax_pairs(e[v]));
    }
#pragma unroll
    for (int m = 8 / V; m >= 1; m >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, m));
    if (live) {     // blocks do not straddle the end of a row: n is a multiple of 128
        const Divisor div(code_scale<CK>(amax));
        Codes<V> c;
#pragma unroll
        for (int v = 0; v < V; ++v) c.w[v] = encode8<CK>(e[v], div);
        c.store(q + row * n + col);
        if ((threadIdx.x & (16 / V - 1)) == 0) scales[row * (n >> 7) + (col >> 7)] = div.s;
    }
}

template <typename T, int CK>
__global__ void __launch_bounds__(kPairMaxN * sizeof(T) / 32, sizeof(T) == 2 ? 2 : 1) pair_fwd_kernel(const PairParams p) {
    constexpr int ES = sizeof(T), V = Lane<T>::V, W = 32 / V;
    constexpr bool EARLY = ES == 2 && CK == CODES_NONE;
    __shared__ float sum_o[W], sum_h[W];
    const int t = threadIdx.x, col = t * 8 * V;
    const bool live = col < p.n, wide = p.wide != 0;
    const int64_t row_bytes = int64_t(p.n) * ES, row = blockIdx.x, at = row * row_bytes + col * ES;
    Lane<T> o, x, post, pre, gate;
    o.zero(); x.zero(); post.zero(); pre.zero(); gate.zero();
    if (live) {
        o.load(p.o + at, wide);
        x.load(p.x + at, wide);
        if (p.gate && (EARLY || p.G > 1)) gate.load(p.gate + (uint32_t(row) % uint32_t(p.G)) * row_bytes + col * ES, wide);   // fewer than 2^31 rows
        if (EARLY) {
            post.load(p.post + col * ES, wide);
            pre.load(p.pre + col * ES, wide);
        }
    }
    if (t < W) sum_o[t] = sum_h[t] = 0.f;
    __syncthreads();
    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = fma2(o.v[v].get(i), o.v[v].get(i), acc);
    if constexpr (CK != CODES_NONE) put_codes<CK>(o, live, p.oq, p.os, row, p.n, col);
    const float r_post = rsqrtf(fmaf(cta_sum<W>(acc.x + acc.y, sum_o), p.inv_n, p.eps));
    const float scaled = r_post * p.alpha;
    if (!EARLY && live) {
        post.load(p.post + col * ES, wide);
        if (p.gate && p.G == 1) gate.load(p.gate + col * ES, wide);
    }
    acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 w = post.v[v].get(i);
            if (p.gate) w = mul2(w, gate.v[v].get(i));
            x.v[v].set(i, fma2(mul2(o.v[v].get(i), splat2(scaled)), w, x.v[v].get(i)));      // h, as it is stored
            acc = fma2(x.v[v].get(i), x.v[v].get(i), acc);
        }
    if (!live) acc = make_float2(0.f, 0.f);        // of a row without a finite norm, 0 * r_post is not 0
    if (live) x.store(p.h + at, wide);
    if constexpr (CK != CODES_NONE) put_codes<CK>(x, live, p.hq, p.hs, row, p.n, col);
    const float r_pre = rsqrtf(fmaf(cta_sum<W>(acc.x + acc.y, sum_h), p.inv_n, p.eps));
    if (t == 0) {
        p.r_post[row] = r_post;
        p.r_pre[row] = r_pre;
    }
    if (!EARLY && live) pre.load(p.pre + col * ES, wide);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[v].set(i, mul2(mul2(x.v[v].get(i), splat2(r_pre)), pre.v[v].get(i)));
    if (live) x.store(p.y + at, wide);
}

// ---- backward --------------------------------------------------------------------------------
// Rows in the order of the gate's groups (all rows of gate row 0 first): position j is row
// j / R + (j % R) * G, R = M / G.  CTA b takes the positions [first(b), first(b + 1)), so that every CTA
// has the same share of rows whatever the number of groups, and a group's gradient is the sum of at most one
// sum per CTA.  A group that lies inside one CTA is written by it; one that several share goes through scratch.
//
// B = sum dh * on is the one sum behind two gradients: dgate = alpha * post * B over the gate's group, and
// dpost = alpha * sum over the groups of gate * B.  With one gate row or none the CTAs keep B alone (and the
// sum for dpre), the reduction forms both; with several rows B starts again with every group, and dpost's sums, which
// grow at the end of a group only, stay in shared memory.  Where every row has a gate row of its own that comes in with
// the row, dgate is written row by row and B's place taken by dpost's sum.
__host__ __device__ __forceinline__ int64_t pair_first(int64_t b, int64_t grid, int64_t M) {
    const int64_t q = M / grid, r = M % grid;
    return b * q + (b < r ? b : r);
}

// scratch: [grid][PART_ROWS][n] float32
enum : int { PART_PRE = 0, PART_POST = 1, PART_HEAD = 2, PART_TAIL = 3, PART_ROWS = 4 };   // PART_POST: B itself with one gate row or none

// Eight elements of o or h as they lie in shared memory: values, or codes that a block's scale makes values of.
template <typename T, int CK>
struct Kept {
    uint2 w;
    __device__ __forceinline__ void load(const uint8_t* p, int col) { w = *reinterpret_cast<const uint2*>(p + col); }
    __device__ __forceinline__ void get(float2* e) const {
        decode4<CK>(w.x, e[0], e[1]);
        decode4<CK>(w.y, e[2], e[3]);
    }
};
template <typename T>
struct Kept<T, CODES_NONE> {
    Vec8<T> w;
    __device__ __forceinline__ void load(const uint8_t* p, int col) { w.load(p + col * int(sizeof(T))); }
    __device__ __forceinline__ void get(float2* e) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = w.get(i);
    }
};

__device__ __forceinline__ void copy4_async(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// global -> shared bulk copy of what no other kernel reads soon
__device__ __forceinline__ void bulk_once(void* dst_smem, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
                     smem_u32(dst_smem)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Sums over the CTA of two values.  buf: a place for each of W (16 or 32) warps and value, those of absent warps zeroed.
template <int W>
__device__ __forceinline__ float2 cta_sum2(float a, float b, float* buf) {
    const bool up = (threadIdx.x & 16) != 0;          // the halves of a warp take a value each after the first exchange
    float v = up ? b : a;
    v += __shfl_xor_sync(0xffffffffu, up ? a : b, 16);
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 15) == 0) buf[(threadIdx.x & 16) * (W / 16) + (threadIdx.x >> 5)] = v;
    __syncthreads();
    const float* mine = buf + (threadIdx.x & 16) * (W / 16) + (threadIdx.x & 15);
    v = mine[0];
    if (W == 32) v += mine[16];
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    const float o = __shfl_xor_sync(0xffffffffu, v, 16);
    return up ? make_float2(o, v) : make_float2(v, o);
}

// A row passes three times through the registers: (1) sum t * hn, (2) dx, the sums over rows, u and sum u * on,
// (3) do.  The two sums of a row are joined with its neighbours': between two barriers a CTA does (3) of row i, (2) of
// row i + 1 and (1) of row i + 2, and the barrier exchanges the sums of the latter two.  That is one barrier and one
// reduction's latency per row, with 16 to 20 warps on an SM to hide it for 16-bit rows up to 5120 columns and 8 to 16 elsewhere.  Rows come in by bulk copies,
// their 1/rms and the scales of their codes by 4-byte copies two rows further ahead.
template <typename T, int CK, int GATE, int V>
__global__ void __launch_bounds__(V == 1 ? kPairOneMaxN / 8 : kPairMaxThreads, 1) pair_bwd_kernel(const PairParams p) {
    extern __shared__ __align__(128) uint8_t ring[];
    constexpr int NB = kPairMaxN / 128, SC = 2 * NB + 2;
    constexpr int DEPTH = kPairMaxStages + 3;      // behind the barrier of row i: row i in pass 3 up to row i + S + 2 on its way
    __shared__ uint64_t full[kPairMaxStages];
    constexpr int W = V == 1 ? 32 : 16;       // warps of a CTA, at most
    __shared__ float sums[2][2 * W];
    __shared__ float scal[DEPTH][SC];        // scales of o, of h, 1/rms of o, of h
    constexpr bool GROUPS = GATE == GATE_GROUPS, EACH = GATE == GATE_EACH;
    constexpr int ES = sizeof(T), CS = CK == CODES_NONE ? ES : 1;   // bytes of an element of dy / of o and h
    const int t = threadIdx.x, nt = blockDim.x, S = p.stages, nb = p.n >> 7;
    const uint32_t row_bytes = uint32_t(p.n) * ES, code_bytes = uint32_t(p.n) * CS;
    const bool has_dh = p.dh != nullptr;
    // a stage: dy | o | h | gate row (if every row has one) | dh (if given)
    const uint32_t off_o = row_bytes, off_h = off_o + code_bytes, off_g = off_h + code_bytes, off_dh = off_g + (EACH ? row_bytes : 0u),
                   stage_bytes = off_dh + (has_dh ? row_bytes : 0u);
    const int G = GROUPS ? int(p.G) : 1, R = int(p.M) / G;          // fewer than 2^31 rows
    const int begin = int(pair_first(blockIdx.x, gridDim.x, p.M)), end = int(pair_first(blockIdx.x + 1, gridDim.x, p.M));

    // a position, its gate row and its row; one step on costs no division
    struct At { int j, g, left, row; };
    auto start = [&](int j) {
        At a{j, 0, 0, j};
        if (GROUPS) {
            a.g = j / R;
            const int k = j - a.g * R;
            a.left = R - k;
            a.row = a.g + k * G;
        }
        return a;
    };
    auto advance = [&](At& a) {
        ++a.j;
        if (!GROUPS) ++a.row;
        else if (--a.left == 0) { ++a.g; a.left = R; a.row = a.g; }
        else a.row += G;
    };
    __shared__ At ahead;           // the position to be fetched next; thread 0 alone uses it
    auto fetch = [&](int s) {
        const int64_t row = ahead.row;
        uint64_t policy;             // its lines go first when L2 needs room: 4 % at 16384 x 4096
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        uint8_t* dst = ring + size_t(s) * stage_bytes;
        mbar_expect_tx(&full[s], stage_bytes);
        bulk_once(dst, p.dy + row * row_bytes, row_bytes, &full[s], policy);
        bulk_once(dst + off_h, p.hsrc + row * code_bytes, code_bytes, &full[s], policy);
        bulk_once(dst + off_o, p.o + row * code_bytes, code_bytes, &full[s], policy);
        if (has_dh) bulk_once(dst + off_dh, p.dh + row * row_bytes, row_bytes, &full[s], policy);
        if (EACH) bulk_once(dst + off_g, p.gate + row * row_bytes, row_bytes, &full[s], policy);
        advance(ahead);
    };
    // one group of 4-byte copies per row, an empty one past the last
    const int nsc = CK == CODES_NONE ? 2 : 2 * nb + 2;               // fewer than threads
    At sc_at = start(begin);
    int sc_slot = 0;
    auto fetch_scalars = [&]() {
        if (sc_at.j < end && t < nsc) {
            const int k = CK == CODES_NONE ? t + 2 * nb : t;
            const float* src = k < nb ? p.os_in + int64_t(sc_at.row) * nb + k : k < 2 * nb ? p.hs_in + int64_t(sc_at.row) * nb + (k - nb)
                               : k == 2 * nb ? p.r_post + sc_at.row : p.r_pre + sc_at.row;
            copy4_async(&scal[sc_slot][k], src);
        }
        copies_commit();
        advance(sc_at);
        if (++sc_slot == DEPTH) sc_slot = 0;
    };
    if (t == 0) {
        for (int s = 0; s < S; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
        ahead = start(begin);
        for (int s = 0; s < S && begin + s < end; ++s) fetch(s);
    }
    for (int i = 0; i < S + 2; ++i) fetch_scalars();
    if (t < 2 * W) sums[0][t] = sums[1][t] = 0.f;

    int col[V];
    bool live[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        col[v] = (t + v * nt) * 8;
        live[v] = col[v] < p.n;
    }
    Vec8<T> pre[V];
    float2 coef[4 * V];      // alpha * post [* gate]
    auto coefficients = [&](int g) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            Vec8<T> w, q;
            w.zero(); q.zero();
            if (live[v]) {
                w.load(p.post + col[v] * ES);
                if (GATE == GATE_ROW || GROUPS) q.load(p.gate + int64_t(g) * row_bytes + col[v] * ES);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                coef[4 * v + i] = mul2(w.get(i), splat2(p.alpha));
                if (GATE == GATE_ROW || GROUPS) coef[4 * v + i] = mul2(coef[4 * v + i], q.get(i));
            }
        }
    };
#pragma unroll
    for (int v = 0; v < V; ++v) {
        pre[v].zero();
        if (ES == 2 && live[v]) pre[v].load(p.pre + col[v] * ES);
    }
    At at2 = start(begin);         // row of pass 2
    coefficients(at2.g);
    float2 a_pre[4 * V], a_b[4 * V];
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) a_pre[i] = a_b[i] = make_float2(0.f, 0.f);
    // dpost's sums of GATE_GROUPS, behind the ring, each thread's own
    float4* a_post = reinterpret_cast<float4*>(ring + size_t(S) * stage_bytes) + t;
    if constexpr (GROUPS)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) a_post[i * nt] = make_float4(0.f, 0.f, 0.f, 0.f);

    // What the elements of vector v are multiplied by to be hn (which 1) or on (0): 1/rms, times the scale of the codes' block.
    auto factor = [&](const float* sc, int which, int v) {
        const float r = sc[2 * nb + which];
        return CK == CODES_NONE ? r : r * sc[(which ? nb : 0) + (col[v] >> 7)];
    };
    Kept<T, CK> ok[V];       // o of the row between passes 2 and 3
    auto pass1 = [&](const uint8_t* st, const float* sc) {
        float part = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (live[v]) {
                Vec8<T> dy, w;
                Kept<T, CK> hk;
                float2 h[4], acc = make_float2(0.f, 0.f);
                dy.load(st + col[v] * ES);
                hk.load(st + off_h, col[v]);
                hk.get(h);
                if (ES == 2) w = pre[v]; else w.load(p.pre + col[v] * ES);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc = fma2(mul2(dy.get(i), w.get(i)), h[i], acc);
                part = fmaf(acc.x + acc.y, factor(sc, 1, v), part);
            }
        return part;
    };
    auto pass2 = [&](const uint8_t* st, const float* sc, float ch, float2* u, uint8_t* dx_row) {   // ch: mean(t * hn)
        const float rh = sc[2 * nb + 1];
        float part = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (live[v]) {
                Vec8<T> dy, din, w, gt, dx, dg;
                Kept<T, CK> hk;
                float2 h[4], o[4], acc = make_float2(0.f, 0.f);
                dy.load(st + col[v] * ES);
                hk.load(st + off_h, col[v]);
                hk.get(h);
                ok[v].load(st + off_o, col[v]);
                ok[v].get(o);
                if (has_dh) din.load(st + off_dh + col[v] * ES); else din.zero();
                if (ES == 2) w = pre[v]; else w.load(p.pre + col[v] * ES);
                if (EACH) gt.load(st + off_g + col[v] * ES);
                const float fh = factor(sc, 1, v), fo = factor(sc, 0, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 hn = mul2(h[i], splat2(fh)), on = mul2(o[i], splat2(fo)), gy = dy.get(i);
                    float2 d = fma2(fma2(hn, splat2(-ch), mul2(gy, w.get(i))), splat2(rh), din.get(i));
                    dx.set(i, d);
                    a_pre[4 * v + i] = fma2(gy, hn, a_pre[4 * v + i]);
                    if constexpr (EACH) {
                        dg.set(i, mul2(mul2(d, on), coef[4 * v + i]));
                        d = mul2(d, gt.get(i));
                    }
                    a_b[4 * v + i] = fma2(d, on, a_b[4 * v + i]);
                    u[4 * v + i] = mul2(d, coef[4 * v + i]);
                    acc = fma2(u[4 * v + i], on, acc);
                }
                dx.store(dx_row + col[v] * ES);
                if (EACH) dg.store(p.dgate + (dx_row - p.dx) + col[v] * ES);
                part += acc.x + acc.y;
            }
        if constexpr (GROUPS) {
            // the last row of its group here: the group's gradient, its share of dpost, and B starts again
            if (at2.left == 1 || at2.j + 1 == end) {
                const int g0 = at2.g * R;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (live[v]) {
                        Vec8<T> w, q;
                        w.load(p.post + col[v] * ES);
                        q.load(p.gate + int64_t(at2.g) * row_bytes + col[v] * ES);
                        float2 d[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) d[i] = mul2(mul2(w.get(i), splat2(p.alpha)), a_b[4 * v + i]);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float4& sum = a_post[(2 * v + i) * nt];
                            const float2 lo = mul2(a_b[4 * v + 2 * i], q.get(2 * i)), hi = mul2(a_b[4 * v + 2 * i + 1], q.get(2 * i + 1));
                            sum = make_float4(sum.x + lo.x, sum.y + lo.y, sum.z + hi.x, sum.w + hi.y);
                            a_b[4 * v + 2 * i] = a_b[4 * v + 2 * i + 1] = make_float2(0.f, 0.f);
                        }
                        if (g0 >= begin && g0 + R <= end) {
                            Vec8<T> out;
#pragma unroll
                            for (int i = 0; i < 4; ++i) out.set(i, d[i]);
                            out.store(p.dgate + int64_t(at2.g) * row_bytes + col[v] * ES);
                        } else {
                            float4* dst = reinterpret_cast<float4*>(p.part + (int64_t(blockIdx.x) * PART_ROWS + (g0 < begin ? PART_HEAD : PART_TAIL)) * p.n + col[v]);
                            dst[0] = make_float4(d[0].x, d[0].y, d[1].x, d[1].y);
                            dst[1] = make_float4(d[2].x, d[2].y, d[3].x, d[3].y);
                        }
                    }
                if (at2.j + 1 < end) coefficients(at2.g + 1);
            }
        }
        return part;
    };
    auto pass3 = [&](const float* sc, float co, const float2* u, uint8_t* row) {      // co: mean(u * on)
        const float rp = sc[2 * nb];
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (live[v]) {
                Vec8<T> d;
                float2 o[4];
                ok[v].get(o);
                const float c = -co * rp * factor(sc, 0, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) d.set(i, fma2(o[i], splat2(c), mul2(u[4 * v + i], splat2(rp))));
                d.store(row + col[v] * ES);
            }
    };

    bool dead = false;
    float2 u[4 * V];
    copies_wait<0>();
    __syncthreads();
    mbar_wait_or_mark<true>(&full[0], 0u, DEVERR_FULL_WAIT, dead);
    uint8_t *dx_row = p.dx + int64_t(at2.row) * row_bytes, *do_row = p.dout + int64_t(at2.row) * row_bytes;
    auto next_row = [&]() {
        advance(at2);
        if (GROUPS) {
            dx_row = p.dx + int64_t(at2.row) * row_bytes;
            do_row = p.dout + int64_t(at2.row) * row_bytes;
        } else {
            dx_row += row_bytes;
            do_row += row_bytes;
        }
    };
    if (S >= 2) {
        int sl = 0, sc = 0, par = 0;                 // stage, slot of the scalars of the row of pass 2
        uint32_t ph = 0;
        const uint8_t* st = ring;
        float2 sum = cta_sum2<W>(pass1(st, scal[0]), 0.f, sums[par]);
        par ^= 1;
        float part2 = pass2(st, scal[0], sum.x * p.inv_n, u, dx_row);
        while (true) {
            const bool more = at2.j + 1 < end;
            const int done = sl, sc3 = sc;
            float part1 = 0.f;
            if (more) {
                if (++sl == S) { sl = 0; ph ^= 1u; }
                if (++sc == DEPTH) sc = 0;
                st = ring + size_t(sl) * stage_bytes;
                mbar_wait_or_mark<true>(&full[sl], ph, DEVERR_FULL_WAIT, dead);
                part1 = pass1(st, scal[sc]);
            }
            copies_wait<1>();
            sum = cta_sum2<W>(part1, part2, sums[par]);
            par ^= 1;
            // behind that barrier every thread has read the stage of the row whose pass 2 came before it
            if (t == 0 && !dead && at2.j + S < end) fetch(done);      // a barrier whose copies did not come is not armed again
            fetch_scalars();
            pass3(scal[sc3], sum.y * p.inv_n, u, do_row);
            if (!more) break;
            next_row();
            part2 = pass2(st, scal[sc], sum.x * p.inv_n, u, dx_row);
        }
    } else {
        // one row fills the shared memory (pair_shape): float32 rows with a gradient of h from 7168 columns on, from 6400 with groups of
        // gate rows, from 5760 with a gate per element; without one 8192 with groups, from 7168 with a gate per element; from codes 8192
        // with a gate per element and a gradient of h.  4096 x 8192: 208 us, 1.7 times the floor
        int sc = 0;
        uint32_t ph = 0;
        while (true) {
            float2 sum = cta_sum2<W>(pass1(ring, scal[sc]), 0.f, sums[0]);
            const float part = pass2(ring, scal[sc], sum.x * p.inv_n, u, dx_row);
            fetch_scalars();
            copies_wait<0>();
            sum = cta_sum2<W>(part, 0.f, sums[1]);
            if (t == 0 && !dead && at2.j + 1 < end) fetch(0);
            pass3(scal[sc], sum.x * p.inv_n, u, do_row);
            if (at2.j + 1 == end) break;
            next_row();
            if (++sc == DEPTH) sc = 0;
            ph ^= 1u;
            mbar_wait_or_mark<true>(&full[0], ph, DEVERR_FULL_WAIT, dead);
        }
    }
    if (t == 0 && dead) {    // rows that the wait gave up on may still be on their way to this CTA's shared memory: one more time limit
        const int fetched = ahead.j - begin;
        for (int i = max(0, fetched - S); i < fetched; ++i) mbar_wait_inline(&full[i % S], uint32_t(i / S) & 1u, DEVERR_FULL_WAIT);
    }
    grid_go();
    copies_wait<0>();
    float* out = p.part + int64_t(blockIdx.x) * PART_ROWS * p.n;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (live[v]) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 *a = a_pre + 4 * v + 2 * i, *b = a_b + 4 * v + 2 * i;
                reinterpret_cast<float4*>(out + PART_PRE * p.n + col[v])[i] = make_float4(a[0].x, a[0].y, a[1].x, a[1].y);
                reinterpret_cast<float4*>(out + PART_POST * p.n + col[v])[i] = GROUPS ? a_post[(2 * v + i) * nt] : make_float4(b[0].x, b[0].y, b[1].x, b[1].y);
            }
        }
}

// The CTAs' sums, added in the order of the CTAs: blockIdx.y 0 dpre, 1 dpost (and the gradient of a gate of one row),
// from 2 on the gate's groups that several CTAs share.
template <typename T>
__global__ void __launch_bounds__(256) pair_reduce_kernel(const float* part, int ctas, int M, int G, int n, float alpha, const T* post,
                                                           const T* gate, float* dpost, float* dpre, T* dgate) {
    __shared__ float red[32][33];
    grid_wait();                                     // for the kernel whose sums these are
    const int c = (threadIdx.x & 7) * 4, l = threadIdx.x >> 3;       // four columns, every 32nd CTA's sums
    const int R = M / G, q = M / ctas, rest = M % ctas;
    auto first_of = [&](int b) { return b * q + min(b, rest); };                 // pair_first
    auto owner = [&](int j) { return j < rest * (q + 1) ? j / (q + 1) : rest + (j - rest * (q + 1)) / q; };   // the CTA of a position
    // where there are fewer groups than borders between CTAs every group is looked at, else every border
    const int borders = ctas - 1, looks = G > 1 && G < M ? min(G, borders) : 0;
    for (int k = blockIdx.y; k < 2 + looks; k += gridDim.y) {
        int b0 = 0, b1 = ctas, g = 0;                // CTAs [b0, b1), their rows of scratch
        int first = k, others = k;
        if (k >= 2) {
            g = k - 2;
            if (G > borders) {
                const int at = first_of(k - 1);      // where CTA k - 1 begins
                g = at / R;
                if (at == g * R || first_of(k - 2) > g * R) continue;   // between two groups, or not the group's first border
            }
            b0 = owner(g * R);
            b1 = owner((g + 1) * R - 1) + 1;
            if (b1 == b0 + 1) continue;              // one CTA has the whole group and has written it
            first = PART_TAIL;
            others = PART_HEAD;
        }
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int b = b0 + l; b < b1; b += 8 * 32) {  // eight loads in flight; the order of the sum is that of the CTAs l, l + 32, ...
            float4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = b + 32 * i;
                v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (at < b1) v[i] = *reinterpret_cast<const float4*>(part + (int64_t(at) * PART_ROWS + (at == b0 ? first : others)) * n + blockIdx.x * 32 + c);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) a = make_float4(a.x + v[i].x, a.y + v[i].y, a.z + v[i].z, a.w + v[i].w);
        }
        red[l][c] = a.x; red[l][c + 1] = a.y; red[l][c + 2] = a.z; red[l][c + 3] = a.w;
        __syncthreads();
        if (threadIdx.x < 32) {
            const int col = blockIdx.x * 32 + threadIdx.x;          // n is a multiple of 128
            float v = red[0][threadIdx.x];
#pragma unroll
            for (int i = 1; i < 32; ++i) v += red[i][threadIdx.x];
            if (k == 0) {
                dpre[col] = v;
            } else if (k == 1) {
                v *= alpha;
                if (G == 1 && gate) {
                    dgate[col] = T(v * float(post[col]));
                    v *= float(gate[col]);
                }
                dpost[col] = v;
            } else {
                dgate[int64_t(g) * n + col] = T(v);
            }
        }
        __syncthreads();
    }
}

// With two vectors of eight elements a thread the backward kernel wants 128 registers, so 512 threads fill an SM: CTAs of rows of
// up to 4096 columns share it, wider ones are alone on it and leave up to seven of 16 warps out.  16-bit rows of 4097 to 5120 columns
// therefore take one vector a thread, 17 to 20 warps of 96 registers: fp16 at 5005 x 5120 75 -> 61 us, from int8 73 -> 66, with
// a gate per sample 86 -> 75; 8192 x 4224 109 -> 91.  Up to 6144 columns that is 80 registers, which spill (5005 x 5120 67 and
// 87 us); float32 rows gain nothing from int8 (106 -> 109) and 1 to 7 % without codes; one vector a thread with 64 registers
// and 32 warps is a quarter slower at 4096 columns.
template <typename T>
int pair_vectors(int64_t n) { return sizeof(T) == 2 && n > 4096 && n <= kPairOneMaxN ? 1 : 2; }
int pair_per_sm(int64_t n) { return std::max(1, std::min(32, kPairThreadsPerSm / int((n / 16 + 31) / 32 * 32))); }
// Stages of `bytes` each, with `fixed` bytes beside them; fewer CTAs per SM where there is no room for two stages
void pair_shape(int64_t bytes, int64_t fixed, int& per_sm, int& stages) {
    while (true) {
        stages = int(std::min<int64_t>(kPairMaxStages, (kPairSmem / per_sm - kPairSlack - fixed) / bytes));
        if (stages >= 2 || per_sm == 1) break;
        per_sm = (per_sm + 1) / 2;
    }
    stages = std::max(stages, 1);
}


template <void (*KERN)(PairParams)>
int pair_launch(int64_t grid, int nt, int64_t smem, const PairParams& p, const char* what, cudaStream_t stream) {
    // the same limit for every call: another thread's launch of this kernel with other sizes may come in between
    if (smem > 0)
        if (int rc = allow_smem<KERN>(kPairSmem - kPairSlack)) return rc;
    KERN<<<unsigned(grid), nt, size_t(smem), stream>>>(p);
    return check_launch(what);
}

template <typename T>
int pair_fwd_typed(const PairParams& p, int ck, cudaStream_t stream) {
    const int nt = int((p.n * sizeof(T) / 32 + 31) / 32 * 32);
    const char* what = "pair_fwd_kernel";
    if (ck == CODES_INT8) return pair_launch<pair_fwd_kernel<T, CODES_INT8>>(p.M, nt, 0, p, what, stream);
    if (ck == CODES_E4M3) return pair_launch<pair_fwd_kernel<T, CODES_E4M3>>(p.M, nt, 0, p, what, stream);
    return pair_launch<pair_fwd_kernel<T, CODES_NONE>>(p.M, nt, 0, p, what, stream);
}

int64_t pair_bwd_grid(int64_t M, int64_t n) {
    return std::min<int64_t>(M, int64_t(sm_count()) * pair_per_sm(n));
}

template <typename T>
int pair_bwd_typed(PairParams& p, int ck, float* dpost, float* dpre, cudaStream_t stream) {
    const int vectors = pair_vectors<T>(p.n), nt = int((p.n / (8 * vectors) + 31) / 32 * 32);
    const int64_t code = ck == CODES_NONE ? int64_t(sizeof(T)) : 1;
    const bool each = p.gate && p.G == p.M && p.M > 1, groups = p.gate && p.G > 1 && !each;
    const int64_t bytes = p.n * (int64_t(sizeof(T)) * (1 + (p.dh ? 1 : 0) + (each ? 1 : 0)) + 2 * code);
    int per_sm = pair_per_sm(p.n);
    const int64_t fixed = groups ? int64_t(nt) * 32 * vectors : 0;
    pair_shape(bytes, fixed, per_sm, p.stages);
    const int64_t grid = std::min(pair_bwd_grid(p.M, p.n), int64_t(sm_count()) * per_sm);
    const int64_t smem = bytes * p.stages + fixed;
    const char* what = "pair_bwd_kernel";
    int rc;
    auto with = [&](auto codes, auto width) {
        constexpr int CK = decltype(codes)::value, V = decltype(width)::value;
        if (!p.gate) return pair_launch<pair_bwd_kernel<T, CK, GATE_NONE, V>>(grid, nt, smem, p, what, stream);
        if (p.G == 1) return pair_launch<pair_bwd_kernel<T, CK, GATE_ROW, V>>(grid, nt, smem, p, what, stream);
        return each ? pair_launch<pair_bwd_kernel<T, CK, GATE_EACH, V>>(grid, nt, smem, p, what, stream)
                    : pair_launch<pair_bwd_kernel<T, CK, GATE_GROUPS, V>>(grid, nt, smem, p, what, stream);
    };
    auto of = [&](auto codes) {
        if constexpr (sizeof(T) == 2)
            if (vectors == 1) return with(codes, std::integral_constant<int, 1>{});
        return with(codes, std::integral_constant<int, 2>{});
    };
    if (ck == CODES_INT8) rc = of(std::integral_constant<int, CODES_INT8>{});
    else if (ck == CODES_E4M3) rc = of(std::integral_constant<int, CODES_E4M3>{});
    else rc = of(std::integral_constant<int, CODES_NONE>{});
    if (rc) return rc;
    const int64_t looks = groups ? std::min<int64_t>(p.G, grid - 1) : 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(p.n / 32), unsigned(2 + std::min<int64_t>(looks, 8)));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];      // it may be set up while the last CTAs above still run
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, pair_reduce_kernel<T>, static_cast<const float*>(p.part), int(grid), int(p.M), p.gate ? int(p.G) : 1,
                                             p.n, p.alpha, reinterpret_cast<const T*>(p.post), reinterpret_cast<const T*>(p.gate), dpost, dpre,
                                             reinterpret_cast<T*>(p.dgate));
    if (e != cudaSuccess) { (void)cudaGetLastError(); set_error("pair_reduce_kernel: %s", cudaGetErrorString(e)); return int(e); }
    return LH_OK;
}

bool unaligned(std::initializer_list<const void*> ps, uintptr_t to = 16) {
    uintptr_t a = 0;
    for (const void* q : ps) a |= reinterpret_cast<uintptr_t>(q);
    return (a & (to - 1)) != 0;
}

int pair_check(const char* what, int dtype, int64_t M, int64_t n, const void* gate, int64_t G, int codes) {
    if (dtype != LH_BF16 && dtype != LH_F16 && dtype != LH_F32) return fail_arg("%s: dtype must be bf16, f16 or f32", what);
    if (M > 0x7fffffff) return fail_arg("%s: too many rows", what);
    if (M < 0 || n <= 0 || n > kPairMaxN || (n % 128) != 0)
        return fail_arg("%s: need n %% 128 == 0 and n <= %d (M=%lld n=%lld)", what, kPairMaxN, (long long)M, (long long)n);
    if (codes < CODES_NONE || codes > CODES_E4M3) return fail_arg("%s: codes must be 0 (none), 1 (int8) or 2 (e4m3)", what);
    if (gate && M > 0 && (G <= 0 || M % G != 0)) return fail_arg("%s: the rows must be a multiple of the gate's rows (M=%lld, gate rows %lld)", what, (long long)M, (long long)G);
    return LH_OK;
}

}  // namespace

int64_t pair_bwd_scratch(int64_t M, int64_t n) {
    if (M <= 0 || n <= 0 || n > kPairMaxN || (n % 128) != 0) return 0;     // sizes that the call refuses (or has nothing to do for)
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
    p.wide = !unaligned({x, o, h, y, post, pre, gate}, 32);
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

// Shared device pieces of the operators that keep activations in eight bits: 8-element vectors of
// the three input types, and codes of 1x128 blocks (or of whole rows) in int8 or e4m3.
//
//   scale = max(amax / top, 1e-30), top = 127 (int8) or 448 (e4m3), a correctly rounded float32
//   code  = nearest(x / scale), the quotient a correctly rounded float32 too
// so that codes and scales equal the PyTorch expression bit for bit.  A NaN or an infinity in a block
// gives the block a NaN scale: nothing of it comes back as a finite value.
#pragma once
#include "lh_common.cuh"

#include <type_traits>

namespace lh {

enum : int { CODES_NONE = 0, CODES_INT8 = 1, CODES_E4M3 = 2 };

// ---- eight consecutive elements as float32 ------------------------------------------------
template <typename T>
struct Vec8 {
    static constexpr int WORDS = sizeof(T) == 4 ? 8 : 4;   // 32-bit words
    uint32_t w[WORDS];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0u;
    }
    // p: 16-byte aligned, global or shared
    __device__ __forceinline__ void load(const void* p) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + 4 * i);
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    }
    __device__ __forceinline__ void store(void* p) const {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4)
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p) + 4 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
    // element pair i (0..3)
    __device__ __forceinline__ float2 get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        } else if constexpr (std::is_same<T, __half>::value) {
            return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        } else {
            return bf16x2_to_f2(w[i]);
        }
    }
    __device__ __forceinline__ void set(int i, float2 v) {
        if constexpr (sizeof(T) == 4) {
            w[2 * i] = __float_as_uint(v.x);
            w[2 * i + 1] = __float_as_uint(v.y);
        } else if constexpr (std::is_same<T, __half>::value) {
            w[i] = pack_f16x2(v.x, v.y);
        } else {
            w[i] = pack_bf16x2(v.x, v.y);
        }
    }
};

// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// max(|a|, |b|, |c|), a NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float amax_pairs(const float2* v) {   // four pairs
    const float a = max3_nan(v[0].x, v[0].y, v[1].x), b = max3_nan(v[1].y, v[2].x, v[2].y);
    return max3_nan(max3_nan(a, b, v[3].x), v[3].y, 0.f);
}

// RN(a / 127) by the sequence of div448 (checked against division for every mantissa)
__device__ __forceinline__ float div127(float a) {
    constexpr float c = 1.0f / 127.0f;
    const float q = a * c;
    return fmaf(fmaf(-127.0f, q, a), c, q);
}

// NaN in, or an infinity (whose residual is NaN): a NaN scale
template <int CK>
__device__ __forceinline__ float code_scale(float amax) {
    return max_nan(CK == CODES_INT8 ? div127(amax) : div448(amax), kScaleFloor);
}

// the codes of 8 elements under one scale, in two words
template <int CK>
__device__ __forceinline__ uint2 encode8(const float2* v, const Divisor& d) {
    float2 q[4];
    if (d.tiny) {   // the residual of the fast exact quotient could underflow: rare, the scale of a block of zeros among them
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = make_float2(__fdiv_rn(v[i].x, d.s), __fdiv_rn(v[i].y, d.s));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = quot_exact2(make_float2(-v[i].x, -v[i].y), splat2(d.s), splat2(d.ny));
    }
    if constexpr (CK == CODES_E4M3) {
        return make_uint2(cvt_e4m3x4(q[0].x, q[0].y, q[1].x, q[1].y), cvt_e4m3x4(q[2].x, q[2].y, q[3].x, q[3].y));
    } else {
        // adding 1.5 * 2^23 rounds |q| <= 127 to the nearest integer, ties to even, and leaves it in the low byte
        constexpr float magic = 12582912.0f;
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 m = add2(q[i], splat2(magic));
            b[2 * i] = __float_as_uint(m.x);
            b[2 * i + 1] = __float_as_uint(m.y);
        }
        return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                          __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
    }
}

// four codes of a word as float32, not yet scaled
template <int CK>
__device__ __forceinline__ void decode4(uint32_t w, float2& lo, float2& hi) {
    if constexpr (CK == CODES_E4M3) {
        uint32_t a, b;
        asm("{\n\t.reg .b16 l, h;\n\t"
            "mov.b32 {l, h}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(a), "=r"(b)
            : "r"(w));
        lo = __half22float2(*reinterpret_cast<const __half2*>(&a));
        hi = __half22float2(*reinterpret_cast<const __half2*>(&b));
    } else {
        // biased by 128 a code is a byte, and 2^23 + byte a float32 with that byte at its end
        const uint32_t u = w ^ 0x80808080u;
        constexpr float bias = 8388608.0f + 128.0f;
        lo = add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7650)), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7651))), splat2(-bias));
        hi = add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7652)), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7653))), splat2(-bias));
    }
}
template <int CK>
__device__ __forceinline__ void decode8(uint2 w, float scale, float2* v) {
    decode4<CK>(w.x, v[0], v[1]);
    decode4<CK>(w.y, v[2], v[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], splat2(scale));
}

// ---- a lane's share of a row: 32 bytes of a 16-bit type (16 elements) or of float32 (8) --------
template <typename T> constexpr int kSpan = 32 / int(sizeof(T));

template <typename T>
struct Lane {
    static constexpr int V = kSpan<T> / 8;
    Vec8<T> v[V];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i].zero();
    }
    // wide: p is 32-byte aligned, else 16
    __device__ __forceinline__ void load(const uint8_t* p, bool wide) {
        if (wide) {
            uint4 a, b;
            ld_global_256(p, a, b);
            put(a, b);
        } else {
            put(*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(p + 16));
        }
    }
    __device__ __forceinline__ void put(const uint4& a, const uint4& b) {
        constexpr int H = V - 1, J = 4 * (2 - V);
        v[0].w[0] = a.x; v[0].w[1] = a.y; v[0].w[2] = a.z; v[0].w[3] = a.w;
        v[H].w[J] = b.x; v[H].w[J + 1] = b.y; v[H].w[J + 2] = b.z; v[H].w[J + 3] = b.w;
    }
    __device__ __forceinline__ void store(uint8_t* p, bool wide) const {
        constexpr int H = V - 1, J = 4 * (2 - V);
        const uint4 a = make_uint4(v[0].w[0], v[0].w[1], v[0].w[2], v[0].w[3]), b = make_uint4(v[H].w[J], v[H].w[J + 1], v[H].w[J + 2], v[H].w[J + 3]);
        if (wide) {
            st_global_256(p, a, b);
        } else {
            *reinterpret_cast<uint4*>(p) = a;
            *reinterpret_cast<uint4*>(p + 16) = b;
        }
    }
};
template <int V>
struct Codes {                     // V times eight codes
    uint2 w[V];
    __device__ __forceinline__ void load(const uint8_t* p) {
        if constexpr (V == 2) {
            const uint4 q = *reinterpret_cast<const uint4*>(p);
            w[0] = make_uint2(q.x, q.y);
            w[1] = make_uint2(q.z, q.w);
        } else {
            w[0] = *reinterpret_cast<const uint2*>(p);
        }
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
        if constexpr (V == 2) *reinterpret_cast<uint4*>(p) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
        else *reinterpret_cast<uint2*>(p) = w[0];
    }
};

}  // namespace lh

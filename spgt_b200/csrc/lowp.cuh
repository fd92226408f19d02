// Element types of the training operators (fp32, bf16, fp16), the activations with their derivatives, and the 8-bit checkpoint
// format: 32 consecutive values share a step 2^(E - 127), the smallest of which |value| < 127.5 steps, E >= 1; a code is the value
// in steps, rounded to nearest even.  value / step is exact, so a code does not depend on how it is computed, and code * step has
// seven significant bits: exact in fp32 and in bf16.  A block that holds an infinity or a NaN has E = 255 and restores as NaN.
// (64 steps of the largest block, E = 249, would be an infinity: its codes end at 63.)
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "tc_common.cuh"

namespace spgt {

constexpr int Q8_BLOCK = 32;

template <class T> struct alignas(16) Pack { static constexpr int N = 16 / (int)sizeof(T); T v[N]; };   // 16 bytes of values

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

template <class T, int N> __device__ __forceinline__ void load_pack(const T* p, float (&v)[N]) {
    static_assert(N == Pack<T>::N, "16 bytes");
    const Pack<T> q = *reinterpret_cast<const Pack<T>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(q.v[i]);
}
template <class T, int N> __device__ __forceinline__ void store_pack(T* p, const float (&v)[N]) {
    static_assert(N == Pack<T>::N, "16 bytes");
    Pack<T> q;
#pragma unroll
    for (int i = 0; i < N; ++i) q.v[i] = from_f32<T>(v[i]);
    *reinterpret_cast<Pack<T>*>(p) = q;
}
// ---- activations of the training operators: a NaN stays a NaN, as in the library's --------------------------------------------
// sigmoid from the approximate base-2 exponential and reciprocal.  The exponent z log2(e), rounded, with the rounded constant gives a relative
// error of up to 1.3 |z| 2^-24; the two instructions and the sum add 0.9 x 2^-21: below 2^-19 in all for |z| < 16.  Results under 2^-126
// are zero, and nothing but a NaN gives a NaN.
__device__ __forceinline__ float sigmoid_f(float z) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}
__device__ __forceinline__ float silu_value(float z) { return z * sigmoid_f(z); }
__device__ __forceinline__ float silu_slope(float z) { const float s = sigmoid_f(z); return s * fmaf(z, 1.0f - s, 1.0f); }
template <int N> __device__ __forceinline__ void act_values(int act, float (&z)[N]) {
    if (act == SPGT_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = z[i] < 0.0f ? 0.0f : z[i];
    } else if (act == SPGT_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = silu_value(z[i]);
    } else if (act == SPGT_ACT_SILU2) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = silu_value(silu_value(z[i]));
    }
}
// d *= act'(z)
template <int N> __device__ __forceinline__ void act_slopes(int act, const float (&z)[N], float (&d)[N]) {
    if (act == SPGT_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = z[i] > 0.0f ? d[i] : (z[i] == z[i] ? 0.0f : z[i]);
    } else if (act == SPGT_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] *= silu_slope(z[i]);
    } else if (act == SPGT_ACT_SILU2) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] *= silu_slope(silu_value(z[i])) * silu_slope(z[i]);
    }
}

// The same for pairs of values: two fp32 operations per instruction.
__device__ __forceinline__ float2 pair(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 sigmoid2(float2 z) {
    const float2 y = mul2(z, pair(-1.4426950408889634f));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(y.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(y.y));
    e = add2(e, pair(1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    return r;
}
__device__ __forceinline__ float2 silu2(float2 z) { return mul2(z, sigmoid2(z)); }
__device__ __forceinline__ float2 silu_slope2(float2 z) {
    const float2 s = sigmoid2(z), t = fma2(s, pair(-1.0f), pair(1.0f));      // 1 - s
    return fma2(mul2(z, s), t, s);
}
template <int ACT> __device__ __forceinline__ float2 act_value2(float2 z) {
    if constexpr (ACT == SPGT_ACT_RELU) return make_float2(z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y);
    else if constexpr (ACT == SPGT_ACT_SILU) return silu2(z);
    else if constexpr (ACT == SPGT_ACT_SILU2) return silu2(silu2(z));
    else return z;
}
template <int ACT> __device__ __forceinline__ float2 act_slope2(float2 z, float2 d) {
    if constexpr (ACT == SPGT_ACT_RELU) return make_float2(z.x > 0.0f ? d.x : (z.x == z.x ? 0.0f : z.x), z.y > 0.0f ? d.y : (z.y == z.y ? 0.0f : z.y));
    else if constexpr (ACT == SPGT_ACT_SILU) return mul2(d, silu_slope2(z));
    else if constexpr (ACT == SPGT_ACT_SILU2) return mul2(d, mul2(silu_slope2(silu2(z)), silu_slope2(z)));
    else return d;
}
// 16 bytes of values as pairs
__device__ __forceinline__ void unpack_pairs(const uint4& r, float2 (&v)[2], float) {
    v[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    v[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
}
__device__ __forceinline__ void unpack_pairs(const uint4& r, float2 (&v)[4], __nv_bfloat16) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
}
__device__ __forceinline__ void unpack_pairs(const uint4& r, float2 (&v)[4], __half) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
}
__device__ __forceinline__ uint4 pack_pairs(const float2 (&v)[2], float) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
}
__device__ __forceinline__ uint32_t pack_pair(float2 v, __nv_bfloat16) { const __nv_bfloat162 h = __float22bfloat162_rn(v); return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ uint32_t pack_pair(float2 v, __half) { const __half2 h = __float22half2_rn(v); return *reinterpret_cast<const uint32_t*>(&h); }
template <class T> __device__ __forceinline__ uint4 pack_pairs(const float2 (&v)[4], T t) {
    return make_uint4(pack_pair(v[0], t), pack_pair(v[1], t), pack_pair(v[2], t), pack_pair(v[3], t));
}

// ---- 8-bit checkpoints ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t q8_magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }   // orders NaN > inf > finite
// E of a block from its largest magnitude: 127.5 = 1.1111111b * 2^6, so adding 2^16 carries into the exponent from 127.5 / 64 on
__device__ __forceinline__ uint32_t q8_exponent(uint32_t magnitude) {
    if (magnitude >= 0x7f800000u) return 255u;
    const uint32_t e = (magnitude + 0x10000u) >> 23;
    return (e < 7u ? 7u : e) - 6u;
}
__device__ __forceinline__ float q8_step(uint32_t e) { return __uint_as_float(e << 23); }                 // E = 255: infinity, and 0 * infinity is NaN
__device__ __forceinline__ float q8_inverse(uint32_t e) { return e == 255u ? 0.0f : __uint_as_float((254u - e) << 23); }
// Four codes.  1.5 * 2^23 + x / step has the code, rounded to nearest even, in its low byte.
__device__ __forceinline__ uint32_t q8_encode(float a, float b, float c, float d, float inverse, bool finite) {
    constexpr float magic = 12582912.0f;
    const uint32_t x = __float_as_uint(fmaf(a, inverse, magic)), y = __float_as_uint(fmaf(b, inverse, magic));
    const uint32_t z = __float_as_uint(fmaf(c, inverse, magic)), w = __float_as_uint(fmaf(d, inverse, magic));
    const uint32_t q = __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
    return finite ? q : 0u;
}
template <int N> __device__ __forceinline__ void q8_codes(uint32_t e, const float (&v)[N], uint32_t (&q)[N / 4]) {
    const float inverse = q8_inverse(e), most = 63.0f * __uint_as_float(249u << 23);
    float u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = v[i];
    if (e == 249u) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = fminf(fmaxf(u[i], -most), most);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) q[i] = q8_encode(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3], inverse, e != 255u);
}
__device__ __forceinline__ void q8_decode(uint32_t codes, float step, float (&v)[4]) {
    const uint32_t u = codes ^ 0x80808080u;                                                               // code + 128 in each byte
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + i)) - 8388736.0f) * step;
}
// N consecutive values from an N-aligned offset: they lie in one block
template <int N> __device__ __forceinline__ void q8_load(const int8_t* codes, const uint8_t* steps, int64_t at, float (&v)[N]) {
    static_assert(N == 4 || N == 8, "one or two words");
    const float step = q8_step(__ldg(steps + (at >> 5)));
    if constexpr (N == 4) {
        q8_decode(__ldg(reinterpret_cast<const uint32_t*>(codes + at)), step, v);
    } else {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(codes + at));
        float lo[4], hi[4];
        q8_decode(q.x, step, lo);
        q8_decode(q.y, step, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = lo[i]; v[4 + i] = hi[i]; }
    }
}
// The lanes that share a block (8 with four values each, 4 with eight) write it; all of them call this together.
template <int N> __device__ __forceinline__ void q8_store(int8_t* codes, uint8_t* steps, int64_t at, const float (&v)[N], uint32_t lanes) {
    static_assert(N == 4 || N == 8, "one or two words");
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, q8_magnitude(v[i]));
#pragma unroll
    for (int o = Q8_BLOCK / N / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(lanes, m, o));
    const uint32_t e = q8_exponent(m);
    uint32_t q[N / 4];
    q8_codes(e, v, q);
    if constexpr (N == 4) *reinterpret_cast<uint32_t*>(codes + at) = q[0];
    else *reinterpret_cast<uint2*>(codes + at) = make_uint2(q[0], q[1]);
    if ((at & (Q8_BLOCK - 1)) == 0) steps[at >> 5] = (uint8_t)e;
}

// Calls f with a value of the C type of an element type code (SPGT_F32, SPGT_BF16, SPGT_F16).
template <class F> inline int with_type(int dtype, F&& f) {
    if (dtype == SPGT_F32) return f(float{});
    if (dtype == SPGT_BF16) return f(__nv_bfloat16{});
    if (dtype == SPGT_F16) return f(__half{});
    return SPGT_ERR_SHAPE;
}

}  // namespace spgt

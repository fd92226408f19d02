// Activation checkpoints in 8 bits (format: lowp.cuh).  compress: codes and steps of x, and act(x) in the same pass when wanted;
// restore: the values, or a gradient times act'(values).  A thread takes 16 bytes of values at a time, so neighbouring lanes share a
// block and every access is coalesced.  fp32: two such, loaded together, so that enough is under way (46 M values, compress 46 -> 41 us,
// with an activation 67 -> 63; four 37 and 64, but 75 instead of 64 for its gradient); 16-bit types: one (28 us, two 29).  Bound by HBM:
// an activation and its gradient on 46 M fp32 values take 63 + 63 us, the bytes alone 63 + 63; on bf16 40 + 39, the bytes 35 + 35.
#include "lowp.cuh"

namespace spgt {

constexpr int C8_THREADS = 256;
template <class T> constexpr int c8_each = sizeof(T) == 4 ? 2 : 1;

template <class T, bool ACT> __global__ void __launch_bounds__(C8_THREADS)
compress8_kernel(const T* x, int act, T* y, int8_t* codes, uint8_t* steps, int64_t n) {
    constexpr int N = Pack<T>::N, EACH = c8_each<T>;
    const int64_t first = ((int64_t)blockIdx.x * (EACH * C8_THREADS) + threadIdx.x) * N;
    float v[EACH][N];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
        const int64_t at = first + u * (C8_THREADS * N);
        if (at + N <= n) {
            load_pack(x + at, v[u]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[u][i] = at + i < n ? to_f32(x[at + i]) : 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
        const int64_t at = first + u * (C8_THREADS * N);
        // (whole blocks: lanes past the end take part with zeros and write nothing)
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, q8_magnitude(v[u][i]));
#pragma unroll
        for (int o = Q8_BLOCK / N / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (at < n) {
            const uint32_t e = q8_exponent(m);
            uint32_t q[N / 4];
            q8_codes(e, v[u], q);
            if ((at & (Q8_BLOCK - 1)) == 0) steps[at >> 5] = (uint8_t)e;
            if constexpr (ACT) act_values(act, v[u]);
            if (at + N <= n) {
                if constexpr (N == 4) *reinterpret_cast<uint32_t*>(codes + at) = q[0];
                else *reinterpret_cast<uint2*>(codes + at) = make_uint2(q[0], q[1]);
                if constexpr (ACT) store_pack(y + at, v[u]);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (at + i < n) {
                        codes[at + i] = (int8_t)(q[i / 4] >> (8 * (i % 4)));
                        if constexpr (ACT) y[at + i] = from_f32<T>(v[u][i]);
                    }
            }
        }
    }
}

// fp16: a value that rounds past the largest finite one (a code of 64 steps of 1024) is that one; a NaN is not touched
template <class T> __device__ __forceinline__ float in_range(float v) { return v; }
template <> __device__ __forceinline__ float in_range<__half>(float v) { return fabsf(v) > 65504.0f ? copysignf(65504.0f, v) : v; }

template <class T, bool GRAD> __global__ void __launch_bounds__(C8_THREADS)
restore8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ steps, const T* dy, int act, T* out, int64_t n) {
    constexpr int N = Pack<T>::N, EACH = c8_each<T>;
    const int64_t first = ((int64_t)blockIdx.x * (EACH * C8_THREADS) + threadIdx.x) * N;
    float v[EACH][N], d[EACH][N];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
        const int64_t at = first + u * (C8_THREADS * N);
        if (at + N <= n) {
            q8_load(codes, steps, at, v[u]);
            if constexpr (GRAD) load_pack(dy + at, d[u]);
        } else if (at < n) {
            const float step = q8_step(steps[at >> 5]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[u][i] = at + i < n ? (float)codes[at + i] * step : 0.0f;
                if constexpr (GRAD) d[u][i] = at + i < n ? to_f32(dy[at + i]) : 0.0f;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
        const int64_t at = first + u * (C8_THREADS * N);
        if (at >= n) return;
        if constexpr (GRAD) {
            act_slopes(act, v[u], d[u]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) d[u][i] = in_range<T>(v[u][i]);
        }
        if (at + N <= n) {
            store_pack(out + at, d[u]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < n) out[at + i] = from_f32<T>(d[u][i]);
        }
    }
}

static inline unsigned c8_blocks(int64_t n, int per_thread) { return (unsigned)ceil_div<int64_t>(n, (int64_t)C8_THREADS * per_thread); }
static inline bool c8_size(int64_t n) { return n >= 0 && n <= ((int64_t)1 << 38); }

}  // namespace spgt

using namespace spgt;

extern "C" int spgt_compress8(const void* x, int dtype, int act, void* y, int8_t* codes, uint8_t* steps, int64_t n, spgt_stream_t stream) {
    if (!c8_size(n) || act < SPGT_ACT_NONE || act > SPGT_ACT_SILU2 || dtype < SPGT_F32 || dtype > SPGT_F16) return SPGT_ERR_SHAPE;
    if (n == 0) return SPGT_OK;
    if (!x || !codes || !steps) return SPGT_ERR_NULL;
    if (!aligned16(x) || !aligned16(codes) || (y && !aligned16(y))) return SPGT_ERR_ALIGN;
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        const unsigned blocks = c8_blocks(n, Pack<T>::N * c8_each<T>);
        if (y) compress8_kernel<T, true><<<blocks, C8_THREADS, 0, (cudaStream_t)stream>>>((const T*)x, act, (T*)y, codes, steps, n);
        else compress8_kernel<T, false><<<blocks, C8_THREADS, 0, (cudaStream_t)stream>>>((const T*)x, act, nullptr, codes, steps, n);
        return launch_status();
    });
}

extern "C" int spgt_restore8(const int8_t* codes, const uint8_t* steps, const void* dy, int act, void* out, int dtype, int64_t n,
                             spgt_stream_t stream) {
    if (!c8_size(n) || act < SPGT_ACT_NONE || act > SPGT_ACT_SILU2 || dtype < SPGT_F32 || dtype > SPGT_F16) return SPGT_ERR_SHAPE;
    if (n == 0) return SPGT_OK;
    if (!codes || !steps || !out) return SPGT_ERR_NULL;
    if (!aligned16(codes) || !aligned16(out) || (dy && !aligned16(dy))) return SPGT_ERR_ALIGN;
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        const unsigned blocks = c8_blocks(n, Pack<T>::N * c8_each<T>);
        if (dy) restore8_kernel<T, true><<<blocks, C8_THREADS, 0, (cudaStream_t)stream>>>(codes, steps, (const T*)dy, act, (T*)out, n);
        else restore8_kernel<T, false><<<blocks, C8_THREADS, 0, (cudaStream_t)stream>>>(codes, steps, nullptr, act, (T*)out, n);
        return launch_status();
    });
}

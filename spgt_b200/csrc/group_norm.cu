// Group normalisation with an activation, channels last, forward and backward:
//   m, v: mean and (biased) variance over a sample's P pixels and the cg channels of a group;  xh = (x - m) (v + eps)^-1/2,
//   y = act(xh w + b);   dz = dy act'(xh w + b),  db = sum dz,  dw = sum dz xh,
//   dx = (v + eps)^-1/2 (w dz - mean(w dz) - xh mean(w dz xh)),  means over the group.
// The backward pass reads x, or an 8-bit checkpoint of it (lowp.cuh), and the forward's statistics.
//
// A sample is one contiguous run of P C values.  It is read in 16-byte vectors whatever C is: vector j starts at channel
// (head + j V) mod C, which repeats every K = C / gcd(C, V) vectors, so a thread that steps by multiples of K always holds the same
// channels and keeps their parameters and sums in registers.  Up to V - 1 values before the first 16-byte boundary of a sample
// (head) and after its last (tail) are taken one by one.
// Variances are sums of squared distances from a mean throughout: within a thread's vectors, then merged with
// M2 = M2a + M2b + (ma - mb)^2 na nb / (na + nb), so a mean far from zero costs no digits.  All sums have a fixed order.
#include "lowp.cuh"

namespace spgt {

constexpr int GN_MAX_THREADS = 512, GN_UNROLL = 4;

struct GnShape {
    int64_t L;                  // values of a sample
    int N, C, G, cg;
    int V, K, mult;             // values per vector, vectors per period, periods of channels in one period of vectors
    int R, iters, tiles;        // vector rows a block takes at once, how many times per tile, tiles per sample
    int threads;
};
struct GnParams {
    GnShape s;
    const void *x, *dy;         // x: values, or NULL and the checkpoint
    const int8_t* codes; const uint8_t* steps;
    void* out;                  // y or dx
    int8_t* out_codes; uint8_t* out_steps;
    const float *w, *b;
    float2* stats;              // [N][G] mean, 1 / sqrt(var + eps)
    float4* partial;            // [N][tiles][G] count, mean, M2
    float2 *chan, *sums;        // [N][tiles][C], [N][C]: sum dz, sum dz xh
    float *dw, *db;
    float eps;
    int act;
};

// Where a block's tile lies in its sample.
struct GnTile {
    int n, tile, head, tail, col, row;
    int64_t base, nv, j0, j1;   // offset of the first vector, vectors of the sample, the tile's vectors
    bool active;
    __device__ __forceinline__ GnTile(const GnShape& s, int item) {
        n = item / s.tiles; tile = item - n * s.tiles;
        const int64_t start = n * s.L;
        head = (int)((uint32_t)(-start) & (uint32_t)(s.V - 1));
        if (head > s.L) head = (int)s.L;
        base = start + head;
        nv = (s.L - head) / s.V;
        tail = (int)(s.L - head - nv * s.V);
        const int64_t tv = (int64_t)s.K * s.R * s.iters;
        j0 = tile * tv;
        j1 = j0 + tv < nv ? j0 + tv : nv;
        row = threadIdx.x / s.K; col = threadIdx.x - row * s.K;
        active = row < s.R;
        if (tile != 0) head_here = 0; else head_here = head;
        tail_here = tile == s.tiles - 1 ? tail : 0;
    }
    int head_here, tail_here;   // single values this tile takes
    // offset in the sample of single value e of this tile (e < head_here + tail_here)
    __device__ __forceinline__ int64_t single(int e, const GnShape& s) const { return e < head_here ? e : s.L - tail_here + (e - head_here); }
    // vectors that the thread of (row, col) takes
    __device__ __forceinline__ int count(int r, int c, const GnShape& s) const {
        const int64_t left = j1 - j0 - ((int64_t)r * s.K + c);
        return left <= 0 ? 0 : (int)((left + s.R * s.K - 1) / (s.R * s.K));
    }
};
// first channel of a thread's vectors; channel i is (first + i) mod C
__device__ __forceinline__ int gn_channel(const GnTile& t, const GnShape& s) { return (int)((t.head + (int64_t)t.col * s.V) % s.C); }
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ---- forward statistics -----------------------------------------------------------------------------------------------------------
// JOINT: a vector lies in one group (cg a multiple of V, no head), so its V values are one set; else a set per channel.
template <class T, bool JOINT> __global__ void __launch_bounds__(GN_MAX_THREADS)
gn_stats_kernel(const GnParams p) {
    constexpr int V = Pack<T>::N, S = JOINT ? 1 : V;
    extern __shared__ float2 s_set[];                       // [R K S] mean, M2
    const GnShape& s = p.s;
    const GnTile t(s, blockIdx.x);
    const T* x = (const T*)p.x + t.base;
    if (t.active) {
        float mean[S], m2[S], n = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) mean[i] = m2[i] = 0.0f;
        // U vectors: their mean, the squared distances from it, then the merge
        auto take = [&](auto count, int64_t j) {
            constexpr int U = decltype(count)::value;
            float v[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) load_pack(x + (j + (int64_t)u * s.R * s.K) * V, v[u]);
            constexpr float per = JOINT ? (float)(U * V) : (float)U;
            const float total = n + per, fb = per / total, fm = n * fb;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                float m = 0.0f, q = 0.0f;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if constexpr (JOINT) {
#pragma unroll
                        for (int k = 0; k < V; ++k) m += v[u][k];
                    } else m += v[u][i];
                }
                m *= 1.0f / per;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if constexpr (JOINT) {
#pragma unroll
                        for (int k = 0; k < V; ++k) { const float d = v[u][k] - m; q = fmaf(d, d, q); }
                    } else { const float d = v[u][i] - m; q = fmaf(d, d, q); }
                }
                const float d = m - mean[i];
                mean[i] = fmaf(d, fb, mean[i]);
                m2[i] += fmaf(d * fm, d, q);
            }
            n = total;
        };
        int64_t j = t.j0 + (int64_t)t.row * s.K + t.col;
        const int64_t step = (int64_t)s.R * s.K;
        for (; j + (GN_UNROLL - 1) * step < t.j1; j += GN_UNROLL * step) take(std::integral_constant<int, GN_UNROLL>{}, j);
        for (; j < t.j1; j += step) take(std::integral_constant<int, 1>{}, j);
#pragma unroll
        for (int i = 0; i < S; ++i) s_set[((int64_t)t.row * s.K + t.col) * S + i] = make_float2(mean[i], m2[i]);
    }
    __syncthreads();
    // groups: a warp each.  Single values are sets of one, held by lane.
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    float one = 0.0f;
    int one_group = -1;
    if (lane < t.head_here + t.tail_here) {
        const int64_t at = t.single(lane, s);
        one = to_f32(((const T*)p.x)[t.n * s.L + at]);
        one_group = (int)(at % s.C) / s.cg;
    }
    for (int g = threadIdx.x >> 5; g < s.G; g += warps) {
        const int per_row = JOINT ? s.cg / V : s.mult * s.cg, sets = s.R * per_row;
        auto at = [&](int i, float& cnt) {
            const int r = i / per_row, k = i - r * per_row;
            if constexpr (JOINT) {
                const int col = g * per_row + k;
                cnt = (float)(V * t.count(r, col, s));
                return s_set[r * s.K + col];
            } else {
                const int c = g * s.cg + k % s.cg, first = t.head % s.C;
                const int pos = (c >= first ? c - first : c - first + s.C) + k / s.cg * s.C;
                cnt = (float)t.count(r, pos / V, s);
                return s_set[r * s.K * V + pos];
            }
        };
        float cnt = one_group == g ? 1.0f : 0.0f, sum = one_group == g ? one : 0.0f;
        for (int i = lane; i < sets; i += 32) {
            float c;
            const float2 e = at(i, c);
            cnt += c; sum = fmaf(c, e.x, sum);
        }
        cnt = warp_sum(cnt); sum = warp_sum(sum);
        const float mean = cnt > 0.0f ? sum / cnt : 0.0f;
        float m2 = one_group == g ? (one - mean) * (one - mean) : 0.0f;
        for (int i = lane; i < sets; i += 32) {
            float c;
            const float2 e = at(i, c);
            const float d = e.x - mean;
            m2 += fmaf(c * d, d, e.y);
        }
        m2 = warp_sum(m2);
        if (lane == 0) p.partial[((int64_t)t.n * s.tiles + t.tile) * s.G + g] = make_float4(cnt, mean, m2, 0.0f);
    }
}

// a warp per (sample, group)
__global__ void __launch_bounds__(256) gn_merge_kernel(const GnParams p) {
    const GnShape& s = p.s;
    const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= (int64_t)s.N * s.G) return;
    const int n = (int)(i / s.G), g = (int)(i - (int64_t)n * s.G);
    const float4* e = p.partial + (int64_t)n * s.tiles * s.G + g;
    float sum = 0.0f;
    const float total = (float)(s.L / s.C) * (float)s.cg;
    for (int k = lane; k < s.tiles; k += 32) { const float4 v = e[(int64_t)k * s.G]; sum = fmaf(v.x, v.y, sum); }
    const float mean = warp_sum(sum) / total;
    float m2 = 0.0f;
    for (int k = lane; k < s.tiles; k += 32) { const float4 v = e[(int64_t)k * s.G]; const float d = v.y - mean; m2 += fmaf(v.x * d, d, v.z); }
    m2 = warp_sum(m2);
    if (lane == 0) p.stats[i] = make_float2(mean, rsqrtf(m2 / total + p.eps));
}

// ---- forward: y --------------------------------------------------------------------------------------------------------------------
template <class T, bool KEEP> __global__ void __launch_bounds__(GN_MAX_THREADS)
gn_apply_kernel(const GnParams p) {
    constexpr int V = Pack<T>::N;
    const GnShape& s = p.s;
    const GnTile t(s, blockIdx.x);
    const float2* stats = p.stats + (int64_t)t.n * s.G;
    if (threadIdx.x < t.head_here + t.tail_here) {
        const int64_t at = t.single(threadIdx.x, s);
        const int c = (int)(at % s.C);
        const float2 st = stats[c / s.cg];
        float z[1] = {fmaf(to_f32(((const T*)p.x)[t.n * s.L + at]) - st.x, st.y * (p.w ? p.w[c] : 1.0f), p.b ? p.b[c] : 0.0f)};
        act_values(p.act, z);
        ((T*)p.out)[t.n * s.L + at] = from_f32<T>(z[0]);
    }
    if (!t.active) return;
    float mean[V], a[V], b[V];
    const int first = gn_channel(t, s);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = (first + i) % s.C;
        const float2 st = stats[c / s.cg];
        mean[i] = st.x; a[i] = st.y * (p.w ? p.w[c] : 1.0f); b[i] = p.b ? p.b[c] : 0.0f;
    }
    const T* x = (const T*)p.x + t.base;
    T* y = (T*)p.out + t.base;
    const int64_t step = (int64_t)s.R * s.K;
#pragma unroll 4
    for (int64_t j = t.j0 + (int64_t)t.row * s.K + t.col; j < t.j1; j += step) {
        float v[V];
        load_pack(x + j * V, v);
        // (C a multiple of 32: the lanes that share a block of the checkpoint take part together)
        if constexpr (KEEP) q8_store(p.out_codes, p.out_steps, t.base + j * V, v, (Q8_BLOCK / V == 8 ? 0xffu : 0xfu) << (threadIdx.x & 31 & ~(Q8_BLOCK / V - 1)));
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = fmaf(v[i] - mean[i], a[i], b[i]);
        act_values(p.act, v);
        store_pack(y + j * V, v);
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------
template <class T, bool CODES, int V> __device__ __forceinline__ void gn_load_x(const GnParams& p, int64_t at, float (&v)[V]) {
    if constexpr (CODES) q8_load(p.codes, p.steps, at, v);
    else load_pack((const T*)p.x + at, v);
}
template <class T, bool CODES> __device__ __forceinline__ float gn_load_single(const GnParams& p, int64_t at) {
    if constexpr (CODES) return (float)p.codes[at] * q8_step(p.steps[at >> 5]);
    else return to_f32(((const T*)p.x)[at]);
}

// sums of dz and dz xh of each channel over a tile's pixels
template <class T, bool CODES> __global__ void __launch_bounds__(GN_MAX_THREADS)
gn_bwd_sums_kernel(const GnParams p) {
    constexpr int V = Pack<T>::N;
    extern __shared__ float2 s_sum[];                       // [R][K V]
    __shared__ float2 s_one[2 * V];
    __shared__ int s_one_channel[2 * V];
    const GnShape& s = p.s;
    const GnTile t(s, blockIdx.x);
    const float2* stats = p.stats + (int64_t)t.n * s.G;
    const int singles = t.head_here + t.tail_here;
    if (threadIdx.x < singles) {
        const int64_t at = t.single(threadIdx.x, s);
        const int c = (int)(at % s.C);
        const float2 st = stats[c / s.cg];
        const float xm = gn_load_single<T, CODES>(p, t.n * s.L + at) - st.x;
        const float z[1] = {fmaf(xm, st.y * (p.w ? p.w[c] : 1.0f), p.b ? p.b[c] : 0.0f)};
        float d[1] = {to_f32(((const T*)p.dy)[t.n * s.L + at])};
        act_slopes(p.act, z, d);
        s_one[threadIdx.x] = make_float2(d[0], d[0] * xm);
        s_one_channel[threadIdx.x] = c;
    }
    if (t.active) {
        float mean[V], a[V], b[V], A[V], B[V];
        const int first = gn_channel(t, s);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (first + i) % s.C;
            const float2 st = stats[c / s.cg];
            mean[i] = st.x; a[i] = st.y * (p.w ? p.w[c] : 1.0f); b[i] = p.b ? p.b[c] : 0.0f;
            A[i] = B[i] = 0.0f;
        }
        const T* dy = (const T*)p.dy + t.base;
        const int64_t step = (int64_t)s.R * s.K;
#pragma unroll 2
        for (int64_t j = t.j0 + (int64_t)t.row * s.K + t.col; j < t.j1; j += step) {
            float v[V], d[V], z[V];
            gn_load_x<T, CODES>(p, t.base + j * V, v);
            load_pack(dy + j * V, d);
#pragma unroll
            for (int i = 0; i < V; ++i) { v[i] -= mean[i]; z[i] = fmaf(v[i], a[i], b[i]); }
            act_slopes(p.act, z, d);
#pragma unroll
            for (int i = 0; i < V; ++i) { A[i] += d[i]; B[i] = fmaf(d[i], v[i], B[i]); }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) s_sum[((int64_t)t.row * s.K + t.col) * V + i] = make_float2(A[i], B[i]);
    }
    __syncthreads();
    const int phase = t.head % s.C;
    for (int c = threadIdx.x; c < s.C; c += blockDim.x) {
        float A = 0.0f, B = 0.0f;
        const int pos = c >= phase ? c - phase : c - phase + s.C;
        for (int r = 0; r < s.R; ++r)
            for (int m = 0; m < s.mult; ++m) { const float2 v = s_sum[r * s.K * V + pos + m * s.C]; A += v.x; B += v.y; }
        for (int e = 0; e < singles; ++e)
            if (s_one_channel[e] == c) { A += s_one[e].x; B += s_one[e].y; }
        p.chan[((int64_t)t.n * s.tiles + t.tile) * s.C + c] = make_float2(A, B * stats[c / s.cg].y);
    }
}

// over the tiles: a warp per (sample, channel)
__global__ void __launch_bounds__(256) gn_bwd_merge_kernel(const GnParams p) {
    const GnShape& s = p.s;
    const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= (int64_t)s.N * s.C) return;
    const int64_t n = i / s.C, c = i - n * s.C;
    float A = 0.0f, B = 0.0f;
    for (int k = lane; k < s.tiles; k += 32) { const float2 v = p.chan[(n * s.tiles + k) * s.C + c]; A += v.x; B += v.y; }
    A = warp_sum(A); B = warp_sum(B);
    if (lane == 0) p.sums[i] = make_float2(A, B);
}
// over the samples
__global__ void __launch_bounds__(256) gn_bwd_params_kernel(const GnParams p) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.s.C) return;
    float A = 0.0f, B = 0.0f;
    for (int n = 0; n < p.s.N; ++n) { const float2 v = p.sums[(int64_t)n * p.s.C + c]; A += v.x; B += v.y; }
    if (p.db) p.db[c] = A;
    if (p.dw) p.dw[c] = B;
}

template <class T, bool CODES> __global__ void __launch_bounds__(GN_MAX_THREADS)
gn_bwd_apply_kernel(const GnParams p) {
    constexpr int V = Pack<T>::N;
    extern __shared__ float2 s_group[];                     // [G] means of w dz and w dz xh
    const GnShape& s = p.s;
    const GnTile t(s, blockIdx.x);
    const float2* stats = p.stats + (int64_t)t.n * s.G;
    const int lane = threadIdx.x & 31;
    const float total = (float)(s.L / s.C) * (float)s.cg;
    for (int g = threadIdx.x >> 5; g < s.G; g += blockDim.x >> 5) {
        float c1 = 0.0f, c2 = 0.0f;
        for (int k = lane; k < s.cg; k += 32) {
            const int c = g * s.cg + k;
            const float2 v = p.sums[(int64_t)t.n * s.C + c];
            const float w = p.w ? p.w[c] : 1.0f;
            c1 = fmaf(w, v.x, c1); c2 = fmaf(w, v.y, c2);
        }
        c1 = warp_sum(c1); c2 = warp_sum(c2);
        if (lane == 0) s_group[g] = make_float2(c1 / total, c2 / total);
    }
    __syncthreads();
    if (threadIdx.x < t.head_here + t.tail_here) {
        const int64_t at = t.single(threadIdx.x, s);
        const int c = (int)(at % s.C);
        const float2 st = stats[c / s.cg], k = s_group[c / s.cg];
        const float xm = gn_load_single<T, CODES>(p, t.n * s.L + at) - st.x, a = st.y * (p.w ? p.w[c] : 1.0f);
        const float z[1] = {fmaf(xm, a, p.b ? p.b[c] : 0.0f)};
        float d[1] = {to_f32(((const T*)p.dy)[t.n * s.L + at])};
        act_slopes(p.act, z, d);
        ((T*)p.out)[t.n * s.L + at] = from_f32<T>(fmaf(a, d[0], -st.y * k.x) - xm * (st.y * st.y * k.y));
    }
    if (!t.active) return;
    float mean[V], a[V], b[V], k1[V], k2[V];
    const int first = gn_channel(t, s);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = (first + i) % s.C;
        const float2 st = stats[c / s.cg], k = s_group[c / s.cg];
        mean[i] = st.x; a[i] = st.y * (p.w ? p.w[c] : 1.0f); b[i] = p.b ? p.b[c] : 0.0f;
        k1[i] = -st.y * k.x; k2[i] = -st.y * st.y * k.y;
    }
    const T* dy = (const T*)p.dy + t.base;
    T* dx = (T*)p.out + t.base;
    const int64_t step = (int64_t)s.R * s.K;
#pragma unroll 2
    for (int64_t j = t.j0 + (int64_t)t.row * s.K + t.col; j < t.j1; j += step) {
        float v[V], d[V], z[V];
        gn_load_x<T, CODES>(p, t.base + j * V, v);
        load_pack(dy + j * V, d);
#pragma unroll
        for (int i = 0; i < V; ++i) { v[i] -= mean[i]; z[i] = fmaf(v[i], a[i], b[i]); }
        act_slopes(p.act, z, d);
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = fmaf(v[i], k2[i], fmaf(a[i], d[i], k1[i]));
        store_pack(dx + j * V, d);
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------
static int gn_shape(int N, int64_t P, int C, int G, int dtype, GnShape& s) {
    if (N < 0 || P < 0 || C <= 0 || G <= 0 || C % G || dtype < SPGT_F32 || dtype > SPGT_F16) return SPGT_ERR_SHAPE;
    s = GnShape{};
    s.V = dtype == SPGT_F32 ? 4 : 8;
    int d = s.V;
    while (C % d) d >>= 1;                                  // gcd(C, V): V is a power of two
    s.K = C / d; s.mult = s.V / d;
    if (s.K > GN_MAX_THREADS || P > ((int64_t)1 << 40) / C) return SPGT_ERR_SHAPE;
    s.N = N; s.L = P * C; s.C = C; s.G = G; s.cg = C / G;
    s.R = (s.K > 64 ? GN_MAX_THREADS : 256) / s.K;
    s.threads = ceil_div(s.R * s.K, 32) * 32;
    // tiles of up to 16 rows of vectors per thread, fewer where that leaves SMs without a tile
    const int64_t rows = ceil_div<int64_t>(s.L / s.V, (int64_t)s.R * s.K);
    int64_t iters = N > 0 ? rows * N / (4 * num_sms()) : 1;
    iters = iters < 1 ? 1 : iters > 16 ? 16 : iters;
    s.iters = (int)iters;
    const int64_t tiles = ceil_div<int64_t>(rows, iters) < 1 ? 1 : ceil_div<int64_t>(rows, iters);
    if (tiles * (N > 0 ? N : 1) > 0x7fffffff) return SPGT_ERR_SHAPE;
    s.tiles = (int)tiles;
    return SPGT_OK;
}

}  // namespace spgt

using namespace spgt;

extern "C" size_t spgt_group_norm_workspace_bytes(int N, int64_t P, int C, int G, int dtype) {
    GnShape s;
    if (gn_shape(N, P, C, G, dtype, s)) return 0;
    return (size_t)s.N * s.tiles * s.G * sizeof(float4) + 16;
}
extern "C" size_t spgt_group_norm_bwd_workspace_bytes(int N, int64_t P, int C, int G, int dtype) {
    GnShape s;
    if (gn_shape(N, P, C, G, dtype, s)) return 0;
    return ((size_t)s.N * s.tiles + s.N) * s.C * sizeof(float2) + 16;
}

extern "C" int spgt_group_norm_fwd(const void* x, const float* w, const float* b, void* y, float* stats, int8_t* codes, uint8_t* steps,
                                   int N, int64_t P, int C, int G, float eps, int act, int dtype, void* workspace, size_t workspace_bytes,
                                   spgt_stream_t stream) {
    GnParams p{};
    if (int e = gn_shape(N, P, C, G, dtype, p.s)) return e;
    if (act < SPGT_ACT_NONE || act > SPGT_ACT_SILU2) return SPGT_ERR_SHAPE;
    if (N == 0 || P == 0) return SPGT_OK;
    if (!x || !y || !stats || !workspace || !codes != !steps) return SPGT_ERR_NULL;
    if (workspace_bytes < spgt_group_norm_workspace_bytes(N, P, C, G, dtype)) return SPGT_ERR_WORKSPACE;
    if (!aligned16(x) || !aligned16(y) || !aligned16(stats) || !aligned16(workspace) || (codes && !aligned16(codes))) return SPGT_ERR_ALIGN;
    p.x = x; p.out = y; p.w = w; p.b = b; p.stats = (float2*)stats; p.partial = (float4*)workspace; p.eps = eps; p.act = act;
    p.out_codes = codes; p.out_steps = steps;
    const GnShape& s = p.s;
    const cudaStream_t st = (cudaStream_t)stream;
    const bool joint = s.cg % s.V == 0, keep = codes && C % Q8_BLOCK == 0;
    const size_t smem = (size_t)s.R * s.K * (joint ? 1 : s.V) * sizeof(float2);
    const unsigned items = (unsigned)((int64_t)N * s.tiles);
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        if (joint) gn_stats_kernel<T, true><<<items, s.threads, smem, st>>>(p);
        else gn_stats_kernel<T, false><<<items, s.threads, smem, st>>>(p);
        if (int e = launch_status()) return e;
        gn_merge_kernel<<<(unsigned)ceil_div<int64_t>((int64_t)N * G, 8), 256, 0, st>>>(p);
        if (int e = launch_status()) return e;
        if (keep) gn_apply_kernel<T, true><<<items, s.threads, 0, st>>>(p);
        else gn_apply_kernel<T, false><<<items, s.threads, 0, st>>>(p);
        if (int e = launch_status()) return e;
        return codes && !keep ? spgt_compress8(x, dtype, SPGT_ACT_NONE, nullptr, codes, steps, N * s.L, stream) : (int)SPGT_OK;
    });
}

extern "C" int spgt_group_norm_bwd(const void* dy, const void* x, const int8_t* codes, const uint8_t* steps, const float* w, const float* b,
                                   const float* stats, void* dx, float* dw, float* db, int N, int64_t P, int C, int G, int act, int dtype,
                                   void* workspace, size_t workspace_bytes, spgt_stream_t stream) {
    GnParams p{};
    if (int e = gn_shape(N, P, C, G, dtype, p.s)) return e;
    if (act < SPGT_ACT_NONE || act > SPGT_ACT_SILU2) return SPGT_ERR_SHAPE;
    const cudaStream_t st = (cudaStream_t)stream;
    if (N == 0 || P == 0) {                                 // no pixels: the parameters' gradients are zero
        if (dw && cudaMemsetAsync(dw, 0, (size_t)C * sizeof(float), st) != cudaSuccess) return launch_status();
        if (db && cudaMemsetAsync(db, 0, (size_t)C * sizeof(float), st) != cudaSuccess) return launch_status();
        return SPGT_OK;
    }
    if (!dy || !dx || !stats || !workspace || (!x && !codes) || (codes && !steps)) return SPGT_ERR_NULL;
    if (workspace_bytes < spgt_group_norm_bwd_workspace_bytes(N, P, C, G, dtype)) return SPGT_ERR_WORKSPACE;
    if (!aligned16(dy) || !aligned16(dx) || !aligned16(stats) || !aligned16(workspace) || (codes ? !aligned16(codes) : !aligned16(x))) return SPGT_ERR_ALIGN;
    p.dy = dy; p.x = x; p.codes = codes; p.steps = steps; p.w = w; p.b = b; p.stats = (float2*)stats; p.out = dx; p.dw = dw; p.db = db; p.act = act;
    const GnShape& s = p.s;
    p.sums = (float2*)workspace;
    p.chan = p.sums + (int64_t)N * C;
    const unsigned items = (unsigned)((int64_t)N * s.tiles);
    const size_t smem = (size_t)s.R * s.K * s.V * sizeof(float2);
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        if (codes) gn_bwd_sums_kernel<T, true><<<items, s.threads, smem, st>>>(p);
        else gn_bwd_sums_kernel<T, false><<<items, s.threads, smem, st>>>(p);
        if (int e = launch_status()) return e;
        gn_bwd_merge_kernel<<<(unsigned)ceil_div<int64_t>((int64_t)N * C, 8), 256, 0, st>>>(p);
        if (int e = launch_status()) return e;
        if (dw || db) gn_bwd_params_kernel<<<(unsigned)ceil_div(C, 256), 256, 0, st>>>(p);
        if (int e = launch_status()) return e;
        if (codes) gn_bwd_apply_kernel<T, true><<<items, s.threads, (size_t)G * sizeof(float2), st>>>(p);
        else gn_bwd_apply_kernel<T, false><<<items, s.threads, (size_t)G * sizeof(float2), st>>>(p);
        return launch_status();
    });
}

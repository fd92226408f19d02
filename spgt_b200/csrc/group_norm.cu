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
//
// Each way is a pass for the sums, which leaves a word per group and tile, and a pass for the results, whose blocks merge their
// sample's words themselves.  Both read x, so they take turns over units of samples that L2 could hold: the first pass asks it to keep what
// it reads, the second to let go of what it reads and writes.  Launches are chained (common.cuh), which hides their gaps.
// Measured, in a graph, with what reading x (and dy) and writing the result once takes at the measured copy rate: 64 x 106 x 106 x 128
// fp32 172 us (112; reading x twice from memory would take 168, so what L2 keeps is lost again in the eight passes' starts and ends), the
// same in bf16 109 (56), 8 x 211 x 211 x 42 bf16 23.5 (9.1; two waves' latencies), 43 x 43 x 128 fp32 7.1 (0.3; two launches), 16 x 106 x 106
// x 128 fp32 with a checkpoint 52 (32), 8 x 211 x 211 x 44 bf16 with one, for which x is read a third time, 34 (12); backward of 4 x 71 x 71
// x 128 fp32 15.5 (4.7), of 64 x 106 x 106 x 128 bf16 182 (84), of 16 x 106 x 106 x 128 fp32 from a checkpoint 63 (32), of 8 x 211 x 211 x 44
// bf16 from one 35.3 (12).
// One launch in which a cluster of 8 or 16 blocks shares a sample and meets in the middle is no faster: 178 to 191 us, 37 and 9.5 for
// the first three.
#include "lowp.cuh"
#include <type_traits>

namespace spgt {

constexpr int GN_MAX_WORK = 512;        // threads of a block, most, and vectors that they take at once: their sets, 8 bytes a value, fit 48 KB
static_assert(GN_MAX_WORK * 8 * sizeof(float2) <= 48 * 1024, "no opt-in to more shared memory");

struct GnShape {
    int64_t L;                  // values of a sample
    int N, C, G, cg;
    int V, K, mult;             // values per vector, vectors per period, periods of channels in one period of vectors
    int R, iters, tiles;        // vector rows a block takes at once, how many times per tile, tiles per sample
    int work;                   // threads
    int lanes;                  // threads that work on a group together
    int unit;                   // samples per unit
};
struct GnParams {
    GnShape s;
    const void *x, *dy;         // x: values, or NULL and the checkpoint
    const int8_t* codes; const uint8_t* steps;
    void* out;                  // y or dx
    int8_t* out_codes; uint8_t* out_steps;
    const float *w, *b;
    float2* stats;              // [N][G] mean, 1 / sqrt(var + eps)
    float2* words;              // [N][tiles][G] a tile's mean and M2, or its sums of w dz and w dz xh
    float2* chan;               // [N][tiles][C]: sum dz, sum dz xh
    float *dw, *db;
    float eps;
    int act, first;             // first: sample of the unit
    bool last;                  // the launch that adds up dw and db
};

// Where a block's tile lies.
struct GnTask {
    int64_t base, first;        // offsets of the tile's first vector and of its sample
    int n, tile, left;          // left: vectors of the tile
    int head, head_here, tail_here;      // single values before the sample's first vector; those this tile takes, before and after
};
template <int V> __device__ __forceinline__ GnTask gn_task(const GnShape& s, int n, int tile) {
    GnTask t;
    t.n = n; t.tile = tile;
    t.first = n * s.L;
    t.head = (int)((uint32_t)(-t.first) & (uint32_t)(V - 1));
    if (t.head > s.L) t.head = (int)s.L;
    const int64_t nv = (s.L - t.head) / V, tv = (int64_t)s.K * s.R * s.iters, j0 = tile * tv;
    t.base = t.first + t.head + j0 * V;
    t.left = (int)(nv - j0 < tv ? (nv > j0 ? nv - j0 : 0) : tv);
    t.head_here = tile == 0 ? t.head : 0;
    t.tail_here = tile == s.tiles - 1 ? (int)(s.L - t.head - nv * V) : 0;
    return t;
}
// A thread's place in the rows of vectors.
struct GnThread {
    int row, col, mine, period;
    bool active;
    __device__ __forceinline__ GnThread(const GnShape& s) {
        row = threadIdx.x / s.K; col = threadIdx.x - row * s.K;
        active = row < s.R; mine = threadIdx.x; period = s.R * s.K;
    }
};
// vectors that the thread of (row, col) takes of a tile
__device__ __forceinline__ int gn_count(const GnTask& t, const GnShape& s, int row, int col) {
    const int period = s.R * s.K, left = t.left - (row * s.K + col);
    return left <= 0 ? 0 : (left + period - 1) / period;
}
// offset in the sample of single value e of a tile
__device__ __forceinline__ int64_t gn_single(const GnTask& t, const GnShape& s, int e) { return e < t.head_here ? e : s.L - t.tail_here + (e - t.head_here); }
// f(i, channel, group) for the values i of a thread's vectors: (head + col V + i) mod C
template <int V, class F> __device__ __forceinline__ void gn_channels(const GnTask& t, const GnThread& me, const GnShape& s, F&& f) {
    int c = me.col * V + t.head;
    if (c >= s.C) c %= s.C;
    int g = c / s.cg, r = c - g * s.cg;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        f(i, c, g);
        ++c; ++r;
        if (r == s.cg) { r = 0; ++g; }
        if (c == s.C) { c = 0; g = 0; }
    }
}
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// L2 policies: kept for the next pass, or let go.
__device__ __forceinline__ uint64_t gn_keep() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint64_t gn_drop() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
template <class T> __device__ __forceinline__ uint4 gn_raw(const T* p, uint64_t policy) {
    uint4 v;
    asm volatile("ld.global.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p), "l"(policy));
    return v;
}
// f(j, loaded) for batches of U of the thread's vectors of a tile, which are j, j + period, ... in vectors from the tile's first; those past
// its end are for f to leave out.  load() runs B batches ahead, and loads the thread's last vector in the place of those, so that
// no branch keeps the loads apart.
template <int U, int B, class L, class F> __device__ __forceinline__ void gn_vectors(const GnTask& t, const GnThread& me, L&& load, F&& f) {
    if (!me.active || me.mine >= t.left) return;
    const int period = me.period, last = t.left - 1 - (t.left - 1 - me.mine) % period;
    decltype(load(0)) r[B][U];
    auto fetch = [&](decltype(load(0)) (&to)[U], int j) {
#pragma unroll
        for (int u = 0; u < U; ++u) to[u] = load(min(j + u * period, last));
    };
#pragma unroll
    for (int b = 0; b < B; ++b)
        if (me.mine + b * U * period < t.left) fetch(r[b], me.mine + b * U * period);
    for (int j = me.mine; j < t.left; j += B * U * period) {
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int jb = j + b * U * period;
            if (jb < t.left) {
                f(jb, r[b]);
                if (jb + B * U * period < t.left) fetch(r[b], jb + B * U * period);
            }
        }
    }
}
// The same in two parts, so that the first batches can be under way before what f needs.
template <int U, int B, class L> struct GnStream {
    using Loaded = std::invoke_result_t<L, int>;
    const L load;
    const int mine, period, left, last;
    Loaded r[B][U];
    __device__ __forceinline__ GnStream(const GnTask& t, const GnThread& me, L l)
        : load(l), mine(me.mine), period(me.period), left(me.active ? t.left : 0), last(t.left - 1 - (t.left - 1 - me.mine) % me.period) {}
    __device__ __forceinline__ void fetch(Loaded (&to)[U], int j) {
        if (j >= left) return;
#pragma unroll
        for (int u = 0; u < U; ++u) to[u] = load(min(j + u * period, last));
    }
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int b = 0; b < B; ++b) fetch(r[b], mine + b * U * period);
    }
    template <class F> __device__ __forceinline__ void run(F&& f) {
        for (int j = mine; j < left; j += B * U * period) {
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int jb = j + b * U * period;
                if (jb < left) {
                    f(jb, r[b]);
                    fetch(r[b], jb + B * U * period);
                }
            }
        }
    }
};
template <int U, int B, class L> __device__ __forceinline__ GnStream<U, B, L> gn_stream(const GnTask& t, const GnThread& me, L load) { return GnStream<U, B, L>(t, me, load); }
// Whether a second pass loads its first batches before it waits for the sums (no kernel of the chain writes what it loads): 16-bit types,
// whose blocks are few (8 x 211 x 211 x 42 bf16 24.6 -> 23.7 us, 64 x 106 x 106 x 128 bf16 112.8 -> 108.9, backward 188 -> 183).  fp32 loads them
// after that, forward next to the parameters (64 x 106 x 106 x 128 175 -> 172; before the wait 186); backward all in one place: in two parts
// the compiler's code is slower (16 x 106 x 106 x 128 from a checkpoint 64 -> 80).
template <int V> constexpr bool GN_EARLY = V == 8;
template <class F> __device__ __forceinline__ void gn_with_act(int act, F&& f) {
    if (act == SPGT_ACT_SILU) f(std::integral_constant<int, SPGT_ACT_SILU>{});
    else if (act == SPGT_ACT_RELU) f(std::integral_constant<int, SPGT_ACT_RELU>{});
    else if (act == SPGT_ACT_SILU2) f(std::integral_constant<int, SPGT_ACT_SILU2>{});
    else f(std::integral_constant<int, SPGT_ACT_NONE>{});
}

// ---- forward: sums -----------------------------------------------------------------------------------------------------------------
// JOINT: a vector lies in one group (cg a multiple of V, no head), so its V values are one set; else a set per channel.
template <class T, bool JOINT> __global__ void __launch_bounds__(GN_MAX_WORK) gn_stats_kernel(const GnParams p) {
    constexpr int V = Pack<T>::N, S = JOINT ? 1 : V, U = 8;      // vectors to a merge
    extern __shared__ float2 s_set[];                       // [R K S] mean, M2
    __shared__ float one[2 * V];
    __shared__ int one_group[2 * V];
    pdl_launch_next();
    const GnShape& s = p.s;
    const int n_in = blockIdx.x / s.tiles;
    const GnTask t = gn_task<V>(s, p.first + n_in, blockIdx.x - n_in * s.tiles);
    const GnThread me(s);
    const int period = me.period, mine = me.mine, singles = t.head_here + t.tail_here;
    const uint64_t keep = gn_keep();
    const T* x = (const T*)p.x + t.base;
    float mean[S], m2[S], n = 0.0f;
#pragma unroll
    for (int i = 0; i < S; ++i) mean[i] = m2[i] = 0.0f;
    // M vectors: their mean, the squared distances from it, then the merge
    auto take = [&](auto count, const uint4* raw) {
        constexpr int M = decltype(count)::value;
        float2 v[M][V / 2];
#pragma unroll
        for (int u = 0; u < M; ++u) unpack_pairs(raw[u], v[u], T{});
        constexpr float per = JOINT ? (float)(M * V) : (float)M;
        const float total = n + per, fb = __fdividef(per, total), fm = n * fb;
        auto merge = [&](int i, float m, float q) {
            const float d = m - mean[i];
            mean[i] = fmaf(d, fb, mean[i]);
            m2[i] += fmaf(d * fm, d, q);
        };
        if constexpr (JOINT) {
            float2 m = v[0][0], q = pair(0.0f);
#pragma unroll
            for (int u = 0; u < M; ++u)
#pragma unroll
                for (int k = u == 0 ? 1 : 0; k < V / 2; ++k) m = add2(m, v[u][k]);
            const float mm = (m.x + m.y) * (1.0f / per);
            const float2 minus = pair(-mm);
#pragma unroll
            for (int u = 0; u < M; ++u)
#pragma unroll
                for (int k = 0; k < V / 2; ++k) { const float2 d = add2(v[u][k], minus); q = fma2(d, d, q); }
            merge(0, mm, q.x + q.y);
        } else {
#pragma unroll
            for (int k = 0; k < V / 2; ++k) {
                float2 m = v[0][k], q = pair(0.0f);
#pragma unroll
                for (int u = 1; u < M; ++u) m = add2(m, v[u][k]);
                m = mul2(m, pair(1.0f / per));
                const float2 minus = make_float2(-m.x, -m.y);
#pragma unroll
                for (int u = 0; u < M; ++u) { const float2 d = add2(v[u][k], minus); q = fma2(d, d, q); }
                merge(2 * k, m.x, q.x);
                merge(2 * k + 1, m.y, q.y);
            }
        }
        n = total;
    };
    gn_vectors<U, 1>(t, me, [&](int j) { return gn_raw(x + (int64_t)j * V, keep); }, [&](int j, const uint4 (&raw)[U]) {
        if (j + (U - 1) * period < t.left) { take(std::integral_constant<int, U>{}, raw); return; }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u * period < t.left) take(std::integral_constant<int, 1>{}, raw + u);
    });
    if (me.active) {
#pragma unroll
        for (int i = 0; i < S; ++i) s_set[mine * S + i] = make_float2(mean[i], m2[i]);
    }
    if (threadIdx.x < singles) {                            // sets of one
        const int64_t at = gn_single(t, s, threadIdx.x);
        one[threadIdx.x] = to_f32(((const T*)p.x)[t.first + at]);
        one_group[threadIdx.x] = (int)(at % s.C) / s.cg;
    }
    __syncthreads();
    // groups, `lanes` threads each
    const int lane = threadIdx.x & (s.lanes - 1), groups = s.work / s.lanes;
    const int even = t.left == s.iters * period ? s.iters : 0;      // every thread has as many vectors
    const int phase = t.head < s.C ? t.head : t.head % s.C;
    for (int g0 = 0; g0 < s.G; g0 += groups) {
        const int g = g0 + threadIdx.x / s.lanes, per_row = JOINT ? s.cg / V : s.mult * s.cg;
        auto sets = [&](auto&& f) {                         // f(count, set) for this thread's share of the group's sets
            if (g >= s.G) return;
            if constexpr (JOINT) {
                for (int i = lane; i < s.R * per_row; i += s.lanes) {
                    const int r = i / per_row, col = g * per_row + i - r * per_row;
                    f((float)(V * (even ? even : gn_count(t, s, r, col))), s_set[r * s.K + col]);
                }
            } else {
                for (int k = lane; k < per_row; k += s.lanes) {
                    const int m = k / s.cg, c = g * s.cg + k - m * s.cg;
                    const int pos = (c >= phase ? c - phase : c - phase + s.C) + m * s.C, col = pos / V;
                    for (int r = 0; r < s.R; ++r) f((float)(even ? even : gn_count(t, s, r, col)), s_set[r * s.K * V + pos]);
                }
            }
            if (singles > 0 && lane == 0)
                for (int e = 0; e < singles; ++e)
                    if (one_group[e] == g) f(1.0f, make_float2(one[e], 0.0f));
        };
        float cnt = 0.0f, sum = 0.0f, m2 = 0.0f;
        sets([&](float c, float2 e) { cnt += c; sum = fmaf(c, e.x, sum); });
        cnt = lanes_sum(cnt, s.lanes); sum = lanes_sum(sum, s.lanes);
        const float mean = cnt > 0.0f ? sum / cnt : 0.0f;
        sets([&](float c, float2 e) { const float d = e.x - mean; m2 += fmaf(c * d, d, e.y); });
        m2 = lanes_sum(m2, s.lanes);
        if (lane == 0 && g < s.G) p.words[((int64_t)t.n * s.tiles + t.tile) * s.G + g] = make_float2(mean, m2);
    }
    pdl_wait();                                             // (see gn_bwd_sums_kernel)
}

// f(pass, tile, word) for this thread's share of the words of a group of sample n, in order, in two passes with between() in between.
// Up to GN_HELD words are read at a time, and once for both passes if that is all.
constexpr int GN_HELD = 6;
template <class F, class B> __device__ __forceinline__ void gn_words(const GnParams& p, int n, int g, F&& f, B&& between) {
    const GnShape& s = p.s;
    const int lane = threadIdx.x & (s.lanes - 1), tiles = g < s.G ? s.tiles : 0, batch = GN_HELD * s.lanes;
    const float2* at = p.words + (int64_t)n * s.tiles * s.G + g;
    float2 v[GN_HELD];
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
        for (int from = lane; from < tiles; from += batch) {
            if (pass == 0 || s.tiles > batch) {
#pragma unroll
                for (int i = 0; i < GN_HELD; ++i)
                    if (from + i * s.lanes < tiles) v[i] = __ldcg(at + (int64_t)(from + i * s.lanes) * s.G);
            }
#pragma unroll
            for (int i = 0; i < GN_HELD; ++i)
                if (from + i * s.lanes < tiles) f(pass, from + i * s.lanes, v[i]);
        }
        if (pass == 0) between();
    }
}
// What the results of a sample need, for all groups in s_group [G]: pair(g), a group's, on its first lane.
template <class F> __device__ __forceinline__ void gn_groups(const GnShape& s, float2* s_group, F&& pair) {
    const int lane = threadIdx.x & (s.lanes - 1), groups = s.work / s.lanes;
    for (int g0 = 0; g0 < s.G; g0 += groups) {
        const int g = g0 + threadIdx.x / s.lanes;
        const float2 v = pair(g);
        if (lane == 0 && g < s.G) s_group[g] = v;
    }
    __syncthreads();
}
// mean and 1 / sqrt(var + eps)
__device__ __forceinline__ float2 gn_merge_stats(const GnParams& p, const GnTask& t, int g) {
    const GnShape& s = p.s;
    const float total = (float)(s.L / s.C) * (float)s.cg;
    // tiles are whole periods of channels, the first one's head and the last one's end apart
    const int full = s.R * s.iters * s.mult * s.cg, q = t.head / s.C, rest = t.head - q * s.C - g * s.cg;
    const int before = q * s.cg + (rest < 0 ? 0 : rest > s.cg ? s.cg : rest);
    const float end = (float)((s.L / s.C) * s.cg - (int64_t)(s.tiles - 1) * full - before);
    auto count = [&](int k) { return k == s.tiles - 1 ? end + (s.tiles == 1 ? (float)before : 0.0f) : k == 0 ? (float)(full + before) : (float)full; };
    float sum = 0.0f, m2 = 0.0f, mean = 0.0f;
    gn_words(p, t.n, g,
             [&](int pass, int k, float2 v) {
                 if (pass == 0) sum = fmaf(count(k), v.x, sum);
                 else { const float d = v.x - mean; m2 += fmaf(count(k) * d, d, v.y); }
             },
             [&] { mean = lanes_sum(sum, s.lanes) / total; });
    m2 = lanes_sum(m2, s.lanes);
    return make_float2(mean, rsqrtf(m2 / total + p.eps));
}

// A thread's channels, z = (x - mean) a + b, from its groups' statistics stats(group); JOINT: one group.
template <int V, bool JOINT> struct GnChannels {
    static constexpr int S = JOINT ? 1 : V / 2;
    float2 minus[S], a[V / 2], b[V / 2];                    // - mean
    template <class F> __device__ __forceinline__ GnChannels(const GnParams& p, const GnTask& t, const GnThread& me, F&& stats) {
        float rstd = 0.0f;
        if constexpr (JOINT) { const float2 st = stats(me.col * V / p.s.cg); minus[0] = pair(-st.x); rstd = st.y; }
        gn_channels<V>(t, me, p.s, [&](int i, int c, int g) {
            float r = rstd;
            if constexpr (!JOINT) { const float2 st = stats(g); (i & 1 ? minus[i / 2].y : minus[i / 2].x) = -st.x; r = st.y; }
            (i & 1 ? a[i / 2].y : a[i / 2].x) = r * (p.w ? __ldg(p.w + c) : 1.0f);
            (i & 1 ? b[i / 2].y : b[i / 2].x) = p.b ? __ldg(p.b + c) : 0.0f;
        });
    }
    __device__ __forceinline__ float2 minus_mean(int i) const { return minus[JOINT ? 0 : i]; }
};

// ---- forward: y --------------------------------------------------------------------------------------------------------------------
template <class T, bool JOINT, bool KEEP> __global__ void __launch_bounds__(GN_MAX_WORK) gn_apply_kernel(const GnParams p) {
    constexpr int V = Pack<T>::N, U = 6;
    extern __shared__ float2 s_group[];
    pdl_launch_next();
    const GnShape& s = p.s;
    const int n_in = blockIdx.x / s.tiles;
    // (the last tiles first: they are the ones that L2 has surely kept)
    const GnTask t = gn_task<V>(s, p.first + n_in, s.tiles - 1 - (int)(blockIdx.x - n_in * s.tiles));
    const GnThread me(s);
    const uint64_t drop = gn_drop();
    const T* x = (const T*)p.x + t.base;
    auto vectors = gn_stream<U, V == 4 ? 1 : 2>(t, me, [&](int j) { return gn_raw(x + (int64_t)j * V, drop); });
    if constexpr (GN_EARLY<V>) vectors.start();
    pdl_wait();
    gn_groups(s, s_group, [&](int g) { return gn_merge_stats(p, t, g); });
    if constexpr (!GN_EARLY<V>) vectors.start();
    if (t.tile == 0)
        for (int g = threadIdx.x; g < s.G; g += s.work) p.stats[(int64_t)t.n * s.G + g] = s_group[g];
    const GnChannels<V, JOINT> ch(p, t, me, [&](int g) { return s_group[g]; });
    gn_with_act(p.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if (threadIdx.x < t.head_here + t.tail_here) {
            const int64_t at = gn_single(t, s, threadIdx.x);
            const int c = (int)(at % s.C);
            const float2 st = s_group[c / s.cg];
            float z[1] = {fmaf(to_f32(((const T*)p.x)[t.first + at]) - st.x, st.y * (p.w ? p.w[c] : 1.0f), p.b ? p.b[c] : 0.0f)};
            act_values(ACT, z);
            ((T*)p.out)[t.first + at] = from_f32<T>(z[0]);
        }
        vectors.run([&](int j0, const uint4 (&batch)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * me.period;
                if (j >= t.left) break;
                const uint4 raw = batch[u];
                float2 v[V / 2];
                unpack_pairs(raw, v, T{});
                const int64_t o = t.base + (int64_t)j * V;
                // (C a multiple of 32: the lanes that share a block of the checkpoint take part together)
                if constexpr (KEEP) {
                    float x[V];
#pragma unroll
                    for (int i = 0; i < V / 2; ++i) { x[2 * i] = v[i].x; x[2 * i + 1] = v[i].y; }
                    q8_store(p.out_codes, p.out_steps, o, x, (Q8_BLOCK / V == 8 ? 0xffu : 0xfu) << (threadIdx.x & 31 & ~(Q8_BLOCK / V - 1)));
                }
#pragma unroll
                for (int i = 0; i < V / 2; ++i) v[i] = act_value2<ACT>(fma2(add2(v[i], ch.minus_mean(i)), ch.a[i], ch.b[i]));
                __stcs(reinterpret_cast<uint4*>((T*)p.out + o), pack_pairs(v, T{}));
            }
        });
    });
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------
template <class T, bool CODES> __device__ __forceinline__ float gn_load_single(const GnParams& p, int64_t at) {
    if constexpr (CODES) return (float)p.codes[at] * q8_step(p.steps[at >> 5]);
    else return to_f32(((const T*)p.x)[at]);
}
// Vectors in a batch and batches ahead.  Measured with batches of 2, one at a time, and the rest singly / these: 4 x 71 x 71 x 128 fp32 19.4 /
// 16.2 us, 16 x 106 x 106 x 128 fp32 from a checkpoint 70.6 / 64, 8 x 211 x 211 x 44 bf16 from one 46.4 / 36.2.
template <int V> constexpr int GN_BWD_BATCH = V == 4 ? 2 : 6;
template <int V> constexpr int GN_BWD_AHEAD = V == 4 ? 3 : 1;
// A vector of dy with its x, as loaded.
template <int V, bool CODES> struct GnPair { uint4 d; uint4 x; };
template <int V> struct GnPair<V, true> { uint4 d; uint32_t q[V / 4]; uint32_t e; };
template <class T, bool CODES> __device__ __forceinline__ GnPair<Pack<T>::N, CODES> gn_load_pair(const GnParams& p, int64_t at, uint64_t policy) {
    constexpr int V = Pack<T>::N;
    GnPair<V, CODES> r;
    r.d = gn_raw((const T*)p.dy + at, policy);
    if constexpr (CODES) {
        if constexpr (V == 4) {
            asm volatile("ld.global.L2::cache_hint.u32 %0, [%1], %2;" : "=r"(r.q[0]) : "l"(p.codes + at), "l"(policy));
        } else {
            asm volatile("ld.global.L2::cache_hint.v2.u32 {%0, %1}, [%2], %3;" : "=r"(r.q[0]), "=r"(r.q[V / 4 - 1]) : "l"(p.codes + at), "l"(policy));
        }
        r.e = __ldg(p.steps + (at >> 5));
    } else {
        r.x = gn_raw((const T*)p.x + at, policy);
    }
    return r;
}
// x - mean and dy
template <class T, bool CODES, bool JOINT, int V> __device__ __forceinline__ void gn_values(const GnPair<V, CODES>& r, const GnChannels<V, JOINT>& ch, float2 (&x)[V / 2], float2 (&d)[V / 2]) {
    unpack_pairs(r.d, d, T{});
    if constexpr (CODES) {
        const float2 step = pair(q8_step(r.e));
#pragma unroll
        for (int w = 0; w < V / 4; ++w) {
            const uint32_t u = r.q[w] ^ 0x80808080u;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 c = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + 2 * k)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541 + 2 * k)));
                x[2 * w + k] = fma2(add2(c, pair(-8388736.0f)), step, ch.minus_mean(2 * w + k));      // (code * step is exact)
            }
        }
    } else {
        unpack_pairs(r.x, x, T{});
#pragma unroll
        for (int i = 0; i < V / 2; ++i) x[i] = add2(x[i], ch.minus_mean(i));
    }
}

// sums of dz and dz xh of each channel over a tile's pixels, and of w dz and w dz xh of each group
template <class T, bool JOINT, bool CODES> __global__ void __launch_bounds__(GN_MAX_WORK) gn_bwd_sums_kernel(const GnParams p) {
    constexpr int V = Pack<T>::N, U = GN_BWD_BATCH<V>;
    extern __shared__ float2 s_sum[];                       // [R][K V]
    __shared__ float2 one[2 * V];
    __shared__ int one_channel[2 * V];
    pdl_launch_next();
    const GnShape& s = p.s;
    const int n_in = blockIdx.x / s.tiles;
    const GnTask t = gn_task<V>(s, p.first + n_in, blockIdx.x - n_in * s.tiles);
    const GnThread me(s);
    const float2* stats = p.stats + (int64_t)t.n * s.G;
    const int singles = t.head_here + t.tail_here;
    const uint64_t keep = gn_keep();
    float2 A[V / 2], B[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) A[i] = B[i] = pair(0.0f);
    const GnChannels<V, JOINT> ch(p, t, me, [&](int g) { return stats[g]; });
    gn_with_act(p.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if (threadIdx.x < singles) {
            const int64_t at = gn_single(t, s, threadIdx.x);
            const int c = (int)(at % s.C);
            const float2 st = stats[c / s.cg];
            const float xm = gn_load_single<T, CODES>(p, t.first + at) - st.x;
            const float z[1] = {fmaf(xm, st.y * (p.w ? p.w[c] : 1.0f), p.b ? p.b[c] : 0.0f)};
            float d[1] = {to_f32(((const T*)p.dy)[t.first + at])};
            act_slopes(ACT, z, d);
            one[threadIdx.x] = make_float2(d[0], d[0] * xm);
            one_channel[threadIdx.x] = c;
        }
        gn_vectors<U, GN_BWD_AHEAD<V>>(t, me, [&](int j) { return gn_load_pair<T, CODES>(p, t.base + (int64_t)j * V, keep); }, [&](int j0, const GnPair<V, CODES> (&batch)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j0 + u * me.period >= t.left) break;
                const GnPair<V, CODES>& r = batch[u];
                float2 v[V / 2], d[V / 2];
                gn_values<T, CODES, JOINT, V>(r, ch, v, d);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const float2 dz = act_slope2<ACT>(fma2(v[i], ch.a[i], ch.b[i]), d[i]);
                    A[i] = add2(A[i], dz);
                    B[i] = fma2(dz, v[i], B[i]);
                }
            }
        });
    });
    if (me.active) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            s_sum[me.mine * V + 2 * i] = make_float2(A[i].x, B[i].x);
            s_sum[me.mine * V + 2 * i + 1] = make_float2(A[i].y, B[i].y);
        }
    }
    __syncthreads();
    // channels, which go to dw and db, then groups, which dx waits for
    const int phase = t.head < s.C ? t.head : t.head % s.C;
    for (int c = threadIdx.x; c < s.C; c += s.work) {
        float2 sum = make_float2(0.0f, 0.0f);
        float2* own = s_sum + (c >= phase ? c - phase : c - phase + s.C);
        const float2* from = own;
        for (int r = 0; r < s.R; ++r, from += s.K * V)
            for (int m = 0; m < s.mult; ++m) { const float2 v = from[m * s.C]; sum.x += v.x; sum.y += v.y; }
        for (int e = 0; e < singles; ++e)
            if (one_channel[e] == c) { sum.x += one[e].x; sum.y += one[e].y; }
        sum.y *= stats[c / s.cg].y;
        p.chan[((int64_t)t.n * s.tiles + t.tile) * s.C + c] = sum;
        const float w = p.w ? __ldg(p.w + c) : 1.0f;
        *own = make_float2(w * sum.x, w * sum.y);           // (in the place of its first row)
    }
    __syncthreads();
    const int lane = threadIdx.x & (s.lanes - 1), groups = s.work / s.lanes;
    for (int g0 = 0; g0 < s.G; g0 += groups) {
        const int g = g0 + threadIdx.x / s.lanes;
        float c1 = 0.0f, c2 = 0.0f;
        for (int k = lane; k < s.cg && g < s.G; k += s.lanes) { const int c = g * s.cg + k; const float2 v = s_sum[c >= phase ? c - phase : c - phase + s.C]; c1 += v.x; c2 += v.y; }
        c1 = lanes_sum(c1, s.lanes); c2 = lanes_sum(c2, s.lanes);
        if (lane == 0 && g < s.G) p.words[((int64_t)t.n * s.tiles + t.tile) * s.G + g] = make_float2(c1, c2);
    }
    // Nothing here needs the results of the unit before, whose blocks may still be at work; but whoever waits for this launch to end
    // counts on those having ended, too.
    pdl_wait();
}
// means of w dz and w dz xh over a group
__device__ __forceinline__ float2 gn_bwd_merge(const GnParams& p, const GnTask& t, int g) {
    const GnShape& s = p.s;
    const float total = (float)(s.L / s.C) * (float)s.cg;
    float c1 = 0.0f, c2 = 0.0f;
    gn_words(p, t.n, g, [&](int pass, int, float2 v) { if (pass == 0) { c1 += v.x; c2 += v.y; } }, [] {});
    return make_float2(lanes_sum(c1, s.lanes) / total, lanes_sum(c2, s.lanes) / total);
}

// dw and db from all tiles' sums [rows][C], by the blocks of the last launch once they have written their tile: two channels a block, a
// share of the rows to each thread, in a fixed order.  (Backward of 16 x 106 x 106 x 128 from a checkpoint with 1 / 2 / 4 / 8 channels a
// block 69.5 / 70.9 / 75.0 / 82.5 us, of 8 x 211 x 211 x 44 bf16 49.5 / 46.1 / 46.4 / 46.8; in a launch of its own 72.4 and 49.0.)
constexpr int GN_PARAM_COLS = 2;

__device__ __forceinline__ void gn_params(const GnParams& p, float2* part) {
    const GnShape& s = p.s;
    const int lane = threadIdx.x & 31, shares = s.work / GN_PARAM_COLS;
    const int64_t rows = (int64_t)s.N * s.tiles;
    for (int c0 = blockIdx.x * GN_PARAM_COLS; c0 < s.C; c0 += gridDim.x * GN_PARAM_COLS) {
        const int c = c0 + (lane & (GN_PARAM_COLS - 1));
        float2 sum = pair(0.0f);
        if (c < s.C)
#pragma unroll 4
            for (int64_t k = threadIdx.x / GN_PARAM_COLS; k < rows; k += shares) sum = add2(sum, __ldcg(p.chan + k * s.C + c));
#pragma unroll
        for (int o = GN_PARAM_COLS; o < 32; o <<= 1) sum = add2(sum, make_float2(__shfl_xor_sync(0xffffffffu, sum.x, o), __shfl_xor_sync(0xffffffffu, sum.y, o)));
        __syncthreads();
        if (lane < GN_PARAM_COLS) part[(threadIdx.x >> 5) * GN_PARAM_COLS + lane] = sum;
        __syncthreads();
        if (threadIdx.x < GN_PARAM_COLS && c < s.C) {
            for (int k = 1; k < s.work / 32; ++k) sum = add2(sum, part[k * GN_PARAM_COLS + lane]);
            if (p.db) p.db[c] = sum.x;
            if (p.dw) p.dw[c] = sum.y;
        }
    }
}

template <class T, bool JOINT, bool CODES> __global__ void __launch_bounds__(GN_MAX_WORK) gn_bwd_apply_kernel(const GnParams p) {
    constexpr int V = Pack<T>::N, S = JOINT ? 1 : V / 2, U = GN_BWD_BATCH<V>;
    extern __shared__ float2 s_group[];
    pdl_launch_next();
    const GnShape& s = p.s;
    const int n_in = blockIdx.x / s.tiles;
    const GnTask t = gn_task<V>(s, p.first + n_in, s.tiles - 1 - (int)(blockIdx.x - n_in * s.tiles));
    const GnThread me(s);
    const float2* stats = p.stats + (int64_t)t.n * s.G;
    const uint64_t drop = gn_drop();
    auto load = [&](int j) { return gn_load_pair<T, CODES>(p, t.base + (int64_t)j * V, drop); };
    auto vectors = gn_stream<U, GN_BWD_AHEAD<V>>(t, me, load);
    if constexpr (GN_EARLY<V>) vectors.start();
    pdl_wait();
    gn_groups(s, s_group, [&](int g) { return gn_bwd_merge(p, t, g); });
    const GnChannels<V, JOINT> ch(p, t, me, [&](int g) { return stats[g]; });
    float2 k1[S], k2[S];
    if constexpr (JOINT) {
        const int g = me.col * V / s.cg;
        const float2 st = stats[g], k = s_group[g];
        k1[0] = pair(-st.y * k.x); k2[0] = pair(-st.y * st.y * k.y);
    } else {
        gn_channels<V>(t, me, s, [&](int i, int, int g) {
            const float2 st = stats[g], k = s_group[g];
            (i & 1 ? k1[i / 2].y : k1[i / 2].x) = -st.y * k.x;
            (i & 1 ? k2[i / 2].y : k2[i / 2].x) = -st.y * st.y * k.y;
        });
    }
    gn_with_act(p.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if (threadIdx.x < t.head_here + t.tail_here) {
            const int64_t at = gn_single(t, s, threadIdx.x);
            const int c = (int)(at % s.C);
            const float2 st = stats[c / s.cg], k = s_group[c / s.cg];
            const float xm = gn_load_single<T, CODES>(p, t.first + at) - st.x, a = st.y * (p.w ? p.w[c] : 1.0f);
            const float z[1] = {fmaf(xm, a, p.b ? p.b[c] : 0.0f)};
            float d[1] = {to_f32(((const T*)p.dy)[t.first + at])};
            act_slopes(ACT, z, d);
            ((T*)p.out)[t.first + at] = from_f32<T>(fmaf(xm, -st.y * st.y * k.y, fmaf(a, d[0], -st.y * k.x)));
        }
        auto use = [&](int j0, const GnPair<V, CODES> (&batch)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * me.period;
                if (j >= t.left) break;
                const GnPair<V, CODES>& r = batch[u];
                float2 v[V / 2], d[V / 2];
                gn_values<T, CODES, JOINT, V>(r, ch, v, d);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const float2 dz = act_slope2<ACT>(fma2(v[i], ch.a[i], ch.b[i]), d[i]);
                    d[i] = fma2(v[i], k2[JOINT ? 0 : i], fma2(ch.a[i], dz, k1[JOINT ? 0 : i]));
                }
                __stcs(reinterpret_cast<uint4*>((T*)p.out + t.base + (int64_t)j * V), pack_pairs(d, T{}));
            }
        };
        if constexpr (GN_EARLY<V>) vectors.run(use);
        else gn_vectors<U, GN_BWD_AHEAD<V>>(t, me, load, use);
    });
    if (p.last) gn_params(p, s_group);
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------
// tensors: how many both passes read; codes: one of them as a checkpoint (whose workspace is no larger).
static int gn_shape(int N, int64_t P, int C, int G, int dtype, int tensors, bool codes, GnShape& s) {
    if (N < 0 || P < 0 || C <= 0 || G <= 0 || C % G || dtype < SPGT_F32 || dtype > SPGT_F16) return SPGT_ERR_SHAPE;
    s = GnShape{};
    s.V = dtype == SPGT_F32 ? 4 : 8;
    const int value_bytes = codes ? 16 / s.V + 1 : 16 / s.V * tensors;
    int d = s.V;
    while (C % d) d >>= 1;                                  // gcd(C, V): V is a power of two
    s.K = C / d; s.mult = s.V / d;
    if (s.K > GN_MAX_WORK || P > ((int64_t)1 << 40) / C) return SPGT_ERR_SHAPE;
    s.N = N; s.L = P * C; s.C = C; s.G = G; s.cg = C / G;
    s.R = (s.K > 256 ? GN_MAX_WORK : 256) / s.K;
    s.work = ceil_div(s.R * s.K, 32) * 32;
    s.lanes = 32;
    while (s.lanes > 1 && s.lanes * G > s.work) s.lanes >>= 1;
    // Units of 96 MB of what is read: fewer launches against more of it found in L2 (64 x 106 x 106 x 128 fp32: units of 48 / 64 / 96 / 112
    // MB 188 / 179 / 178 / 190 us; 16 samples backward 94 / 100 / 74 / 83).
    const int64_t bytes = s.L * value_bytes, unit = bytes > 0 ? ((int64_t)96 << 20) / bytes : 1;
    const int samples = N > 0 ? N : 1, units = (int)(unit >= samples ? 1 : ceil_div<int64_t>(samples, unit < 1 ? 1 : unit));
    s.unit = ceil_div(samples, units);                      // (units of nearly the same size)
    // As many tiles as blocks run at a time, so that a pass is one wave and its blocks end together; no tile of less than four rows of
    // vectors, nor less than twice the words that a block of the second pass merges.  Vectors of eight values, and the backward pass's pairs,
    // take more registers, and blocks more merging: two blocks to an SM (backward of 16 x 106 x 106 x 128 with 2 / 3 / 4: 64 / 77 / 79 us, 8 x
    // 211 x 211 x 42 bf16 forward 24.6 / 33 / 31; 64 x 106 x 106 x 128 fp32 forward 188 / 180 / 174).
    const int64_t rows = ceil_div<int64_t>(s.L / s.V, (int64_t)s.R * s.K), resident = (int64_t)num_sms() * (s.work > 256 ? 1 : s.V == 8 || tensors == 2 ? 2 : 4);
    int64_t tiles = resident / s.unit;
    while (tiles > 1 && tiles * tiles * 16 * G > bytes) tiles = tiles * 7 / 8;
    if (tiles > rows / 4) tiles = rows / 4;
    if (tiles < 1) tiles = 1;
    s.iters = (int)(rows > tiles ? ceil_div(rows, tiles) : 1);
    tiles = rows > s.iters ? ceil_div<int64_t>(rows, s.iters) : 1;
    if (tiles * samples > 0x7fffffff) return SPGT_ERR_SHAPE;
    s.tiles = (int)tiles;
    return SPGT_OK;
}
template <void (*KERNEL)(const GnParams)> static int gn_launch(GnParams p, int first, size_t smem, cudaStream_t st) {
    p.first = first;
    const int samples = p.s.N - first < p.s.unit ? p.s.N - first : p.s.unit;
    return launch_chained(KERNEL, dim3((unsigned)((int64_t)samples * p.s.tiles)), p.s.work, smem, st, p);
}

}  // namespace spgt

using namespace spgt;

extern "C" size_t spgt_group_norm_workspace_bytes(int N, int64_t P, int C, int G, int dtype) {
    GnShape s;
    if (gn_shape(N, P, C, G, dtype, 1, false, s)) return 0;
    return (size_t)s.N * s.tiles * s.G * sizeof(float2) + 16;
}
extern "C" size_t spgt_group_norm_bwd_workspace_bytes(int N, int64_t P, int C, int G, int dtype) {
    GnShape s;
    if (gn_shape(N, P, C, G, dtype, 2, false, s)) return 0;
    return (size_t)s.N * s.tiles * (s.G + s.C) * sizeof(float2) + 16;
}

extern "C" int spgt_group_norm_fwd(const void* x, const float* w, const float* b, void* y, float* stats, int8_t* codes, uint8_t* steps,
                                   int N, int64_t P, int C, int G, float eps, int act, int dtype, void* workspace, size_t workspace_bytes,
                                   spgt_stream_t stream) {
    GnParams p{};
    if (int e = gn_shape(N, P, C, G, dtype, 1, false, p.s)) return e;
    if (act < SPGT_ACT_NONE || act > SPGT_ACT_SILU2) return SPGT_ERR_SHAPE;
    const cudaStream_t st = (cudaStream_t)stream;
    if (N == 0 || P == 0) {                                 // no pixels: the statistics are zero
        if (N > 0 && stats && cudaMemsetAsync(stats, 0, (size_t)N * G * sizeof(float2), st) != cudaSuccess) return launch_status();
        return SPGT_OK;
    }
    if (!x || !y || !stats || !workspace || !codes != !steps) return SPGT_ERR_NULL;
    if (workspace_bytes < spgt_group_norm_workspace_bytes(N, P, C, G, dtype)) return SPGT_ERR_WORKSPACE;
    if (!aligned16(x) || !aligned16(y) || !aligned16(stats) || !aligned16(workspace) || (codes && !aligned16(codes))) return SPGT_ERR_ALIGN;
    const GnShape& s = p.s;
    p.words = (float2*)workspace;
    p.x = x; p.out = y; p.w = w; p.b = b; p.stats = (float2*)stats; p.eps = eps; p.act = act;
    p.out_codes = codes; p.out_steps = steps;
    const bool joint = s.cg % s.V == 0, keep = codes && C % Q8_BLOCK == 0;
    // (the checkpoint where blocks of 32 values are not whole lanes of the kernel: first, since y may be x)
    if (codes && !keep)
        if (int e = spgt_compress8(x, dtype, SPGT_ACT_NONE, nullptr, codes, steps, N * s.L, stream)) return e;
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        const size_t sets = (size_t)s.R * s.K * (joint ? 1 : s.V) * sizeof(float2), groups = (size_t)G * sizeof(float2);
        ChainScope chain;
        for (int n = 0; n < N; n += s.unit) {
            if (int e = joint ? gn_launch<gn_stats_kernel<T, true>>(p, n, sets, st) : gn_launch<gn_stats_kernel<T, false>>(p, n, sets, st)) return e;
            const int e = keep ? (joint ? gn_launch<gn_apply_kernel<T, true, true>>(p, n, groups, st) : gn_launch<gn_apply_kernel<T, false, true>>(p, n, groups, st))
                               : (joint ? gn_launch<gn_apply_kernel<T, true, false>>(p, n, groups, st) : gn_launch<gn_apply_kernel<T, false, false>>(p, n, groups, st));
            if (e) return e;
        }
        return (int)SPGT_OK;
    });
}

extern "C" int spgt_group_norm_bwd(const void* dy, const void* x, const int8_t* codes, const uint8_t* steps, const float* w, const float* b,
                                   const float* stats, void* dx, float* dw, float* db, int N, int64_t P, int C, int G, int act, int dtype,
                                   void* workspace, size_t workspace_bytes, spgt_stream_t stream) {
    GnParams p{};
    if (int e = gn_shape(N, P, C, G, dtype, 2, codes != nullptr, p.s)) return e;
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
    p.words = (float2*)workspace;
    p.chan = p.words + (int64_t)N * s.tiles * G;
    const bool joint = s.cg % s.V == 0;
    ChainScope chain;
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        const size_t sums = (size_t)s.R * s.K * s.V * sizeof(float2), groups = (size_t)(G > s.work / 32 * GN_PARAM_COLS ? G : s.work / 32 * GN_PARAM_COLS) * sizeof(float2);
        for (int n = 0; n < N; n += s.unit) {
            p.last = n + s.unit >= N && (dw || db);
            int e = joint ? (codes ? gn_launch<gn_bwd_sums_kernel<T, true, true>>(p, n, sums, st) : gn_launch<gn_bwd_sums_kernel<T, true, false>>(p, n, sums, st))
                          : (codes ? gn_launch<gn_bwd_sums_kernel<T, false, true>>(p, n, sums, st) : gn_launch<gn_bwd_sums_kernel<T, false, false>>(p, n, sums, st));
            if (e) return e;
            e = joint ? (codes ? gn_launch<gn_bwd_apply_kernel<T, true, true>>(p, n, groups, st) : gn_launch<gn_bwd_apply_kernel<T, true, false>>(p, n, groups, st))
                      : (codes ? gn_launch<gn_bwd_apply_kernel<T, false, true>>(p, n, groups, st) : gn_launch<gn_bwd_apply_kernel<T, false, false>>(p, n, groups, st));
            if (e) return e;
        }
        return (int)SPGT_OK;
    });
}

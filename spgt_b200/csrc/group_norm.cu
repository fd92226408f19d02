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
// One launch each way.  The work is a list of items, a tile's sums or a tile's results, which blocks take in order through a
// ticket counter; the block that finishes a sample's last sums merges them and raises the sample's flag, and items that need the
// flag wait for it.  An item only waits for items before it in the list, and those are in the hands of blocks that run, so every
// wait ends however few blocks run at a time.  The sums of a unit of samples come one unit before its results: the results'
// reads of x (and dy) then find it in L2 and the waits are over before they begin.
// A warp of its own takes the items and copies their vectors, in chunks of a few rows, into a ring in shared memory, ahead of the
// threads that compute: the latencies of the counters, the statistics and the merges are not the memory's.
#include "lowp.cuh"
#include "tc_common.cuh"

namespace spgt {

constexpr int GN_ROWS = 4;              // rows of vectors in a chunk
constexpr int GN_STAGES = 3;            // chunks in the ring
constexpr int GN_MAX_WORK = 512;        // computing threads, most
constexpr int GN_HEADER = 384;          // barriers, flag and tasks before the ring

struct GnShape {
    int64_t L;                  // values of a sample
    int N, C, G, cg;
    int V, K, mult;             // values per vector, vectors per period, periods of channels in one period of vectors
    int R, iters, tiles;        // vector rows a block takes at once, how many times per tile, tiles per sample
    int work;                   // computing threads; a warp more copies
    int lanes;                  // threads that work on a group together
    int unit, lag;              // samples per unit of the list; units between a unit's sums and its results
    int items;
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
    float2* means;              // [N][G]: means of w dz and w dz xh
    int *ticket, *samples, *count, *flag;   // zero at launch: next item, samples merged; [N] tiles summed, [N] merged
    float *dw, *db;
    float eps;
    int act;
};

// An item as the copying warp hands it to the computing threads, in shared memory.
struct GnTask {
    int64_t base, first;        // offsets of the tile's first vector and of its sample
    int n, tile, left;          // left: vectors of the tile
    int head, head_here, tail_here;      // single values before the sample's first vector; those this tile takes, before and after
    int kind;                   // 0 behind the list's end, 1 sums, 2 results
    int pad;
};
template <int V> __device__ __forceinline__ GnTask gn_task(const GnShape& s, int n, int tile, bool sums) {
    GnTask t;
    t.n = n; t.tile = tile; t.kind = sums ? 1 : 2;
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
// A computing thread's place: in a row of vectors, and in the ring.
struct GnThread {
    int row, col, mine, period;
    bool active;
    int at = 0, item = 0;       // chunks and items taken
    bool alive = true;          // false once a wait gave up: the thread goes on to the block's next barriers without data, and the
                                // block ends together before its next item
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

__device__ int g_gn_status = 0;

// ---- the list of items ---------------------------------------------------------------------------------------------------------
// lag 1: sums of unit 0, then for each unit the next one's sums and its results in turn; lag 0: each unit's sums, then its results
// from the last tile to the first, which are the ones still in L2.
struct GnItem { int n, tile; bool sums; };
__device__ __forceinline__ GnItem gn_item(const GnShape& s, int i) {
    const int full = s.unit * s.tiles, units = (s.N + s.unit - 1) / s.unit;
    auto place = [&](int u, int k, bool sums) {
        const int n = k / s.tiles;
        return GnItem{u * s.unit + n, k - n * s.tiles, sums};
    };
    auto size = [&](int u) { const int left = s.N - u * s.unit; return (left < s.unit ? left : s.unit) * s.tiles; };
    if (s.lag == 0) {
        const int u = i / (2 * full), k = i - u * 2 * full, n = size(u);
        return k < n ? place(u, k, true) : place(u, 2 * n - 1 - k, false);
    }
    if (i < full) return place(0, i, true);                                  // (the first unit is a whole one, or all)
    i -= full;
    const int last = units > 1 ? (units - 2) * 2 * full + full + size(units - 1) : 0;      // where the last unit's results begin
    if (i >= last) return place(units - 1, i - last, false);
    const int u = i / (2 * full), k = i - u * 2 * full, next = size(u + 1);   // results of u, sums of u + 1 in turn
    if (k < 2 * next) return (k & 1) ? place(u, k >> 1, false) : place(u + 1, k >> 1, true);
    return place(u, k - next, false);
}
// ---- the ring -----------------------------------------------------------------------------------------------------------------
struct GnRing {
    uint8_t* smem; uint32_t bars; int stage_bytes;
    GnTask* task;               // [stages + 1] items in order: the one being computed and those that have a chunk in the ring
    volatile int* abort_flag;
    __device__ __forceinline__ uint32_t full(int s) const { return bars + 8u * s; }
    __device__ __forceinline__ uint32_t empty(int s) const { return bars + 8u * (GN_STAGES + s); }
};
// Copying: `bytes` (a multiple of 16, from a 16-byte boundary) of up to two tensors per chunk.
__device__ __forceinline__ void gn_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void gn_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// One thread: takes items and fills the ring with their chunks, of `a` and, if not NULL, `b`.  Ends with the list or with the block's
// abort flag, when what it has copied has arrived.
template <class T> __device__ __forceinline__ void gn_produce(const GnParams& p, const GnRing& r, const T* a, const T* b) {
    constexpr int V = Pack<T>::N;
    const GnShape& s = p.s;
    const int chunk = s.R * s.K * GN_ROWS;
    int issued = 0, st = 0, slot = 0;
    uint32_t phase = 1;
    for (bool more = true; more;) {
        const int i = atomicAdd(p.ticket, 1);
        GnTask t = {};
        if (i < s.items) {
            const GnItem item = gn_item(s, i);
            t = gn_task<V>(s, item.n, item.tile, item.sums);
        } else more = false;
        int j = 0;
        do {                                                                // (a tile without vectors: an empty chunk)
            const int n = t.left - j < chunk ? t.left - j : chunk;
            if (!mbar_wait(r.empty(st), phase, r.abort_flag, 121, &g_gn_status)) { more = false; break; }
            if (j == 0) r.task[slot] = t;
            const uint32_t bytes = (uint32_t)n * 16u, dst = smem_u32(r.smem) + st * r.stage_bytes;
            gn_expect(r.full(st), b ? 2 * bytes : bytes);
            if (bytes) {
                gn_copy(dst, a + t.base + (int64_t)j * V, bytes, r.full(st));
                if (b) gn_copy(dst + chunk * 16, b + t.base + (int64_t)j * V, bytes, r.full(st));
            }
            ++issued;
            if (++st == GN_STAGES) { st = 0; phase ^= 1u; }
            j += chunk;
        } while (j < t.left);
        slot = slot == GN_STAGES ? 0 : slot + 1;
    }
    int ignored = 0;
    for (int k = issued > GN_STAGES ? issued - GN_STAGES : 0; k < issued; ++k)
        mbar_wait(r.full(k % GN_STAGES), (uint32_t)(k / GN_STAGES & 1), &ignored, 122, &g_gn_status);
}
__device__ __forceinline__ bool gn_chunk(const GnRing& r, GnThread& me) {
    if (!mbar_wait(r.full(me.at % GN_STAGES), (uint32_t)(me.at / GN_STAGES & 1), r.abort_flag, 123, &g_gn_status)) me.alive = false;
    return me.alive;
}
__device__ __forceinline__ void gn_free(const GnRing& r, GnThread& me) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(r.empty(me.at % GN_STAGES));
    ++me.at;
}
// barriers of the computing threads
__device__ __forceinline__ void gn_sync(int work) { asm volatile("bar.sync 1, %0;" ::"r"(work) : "memory"); }

__device__ __forceinline__ bool gn_all(bool v, int work) {
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((uint32_t)v), "r"(work) : "memory");
    return all != 0;
}

// One more tile of sample n is summed: whether it was the last.  What the block wrote before is then visible to whoever sees it so.
__device__ __forceinline__ bool gn_last(int* count, int of, int* slot, int work) {
    gn_sync(work);
    if (threadIdx.x == 0) {
        __threadfence();
        *slot = atomicAdd(count, 1) == of - 1;
        __threadfence();
    }
    gn_sync(work);
    return *slot != 0;
}
__device__ __forceinline__ void gn_raise(int* flag, int work) {
    gn_sync(work);
    if (threadIdx.x == 0) {
        __threadfence();
        asm volatile("st.release.gpu.global.s32 [%0], 1;" ::"l"(flag) : "memory");
    }
}
// Waits for a sample's flag, two seconds at most.
__device__ __forceinline__ bool gn_wait(const int* flag, int* slot, volatile int* abort_flag, int work) {
    if (threadIdx.x == 0) {
        int v = 0;
        unsigned long long t0 = 0;
        for (uint32_t i = 0;; ++i) {
            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
            if (v) break;
            __nanosleep(32);
            if ((i & 63u) == 0u) {
                const unsigned long long now = globaltimer_ns();
                if (i == 0u) t0 = now;
                else if (now - t0 > TC_WAIT_LIMIT_NS) { *abort_flag = 120; atomicCAS(&g_gn_status, 0, 120); break; }
            }
        }
        *slot = v;
    }
    gn_sync(work);
    return *slot != 0;
}
__device__ __forceinline__ float2 gn_load2(const float2* p) { return __ldcg(p); }     // written in this launch: never from L1

// ---- forward statistics -----------------------------------------------------------------------------------------------------------
// JOINT: a vector lies in one group (cg a multiple of V, no head), so its V values are one set; else a set per channel.
template <class T, bool JOINT>
__device__ __forceinline__ void gn_stats_tile(const GnParams& p, const GnTask& t, const GnRing& ring, GnThread& me, float2* s_set) {
    constexpr int V = Pack<T>::N, S = JOINT ? 1 : V;        // s_set: [R K S] mean, M2
    __shared__ float s_one[2 * V];
    __shared__ int s_one_group[2 * V];
    const GnShape& s = p.s;
    const int period = me.period, mine = me.mine, singles = t.head_here + t.tail_here;
    if (threadIdx.x < singles) {                            // sets of one
        const int64_t at = gn_single(t, s, threadIdx.x);
        s_one[threadIdx.x] = to_f32(((const T*)p.x)[t.first + at]);
        s_one_group[threadIdx.x] = (int)(at % s.C) / s.cg;
    }
    float mean[S], m2[S], n = 0.0f;
#pragma unroll
    for (int i = 0; i < S; ++i) mean[i] = m2[i] = 0.0f;
    // U vectors: their mean, the squared distances from it, then the merge
    auto take = [&](auto count, const T* x) {
        constexpr int U = decltype(count)::value;
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) load_pack(x + u * period * V, v[u]);
        constexpr float per = JOINT ? (float)(U * V) : (float)U;
        const float total = n + per, fb = __fdividef(per, total), fm = n * fb;
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
    int left = t.left;
    const int all = t.left;
    do {
        if (!gn_chunk(ring, me)) break;
        const T* x = reinterpret_cast<const T*>(ring.smem + me.at % GN_STAGES * ring.stage_bytes) + mine * V;
        if (me.active) {
            if (left >= GN_ROWS * period) take(std::integral_constant<int, GN_ROWS>{}, x);
            else for (int u = 0; u * period + mine < left; ++u) take(std::integral_constant<int, 1>{}, x + u * period * V);
        }
        left -= GN_ROWS * period;
        gn_free(ring, me);
    } while (left > 0);
    if (me.active) {
#pragma unroll
        for (int i = 0; i < S; ++i) s_set[mine * S + i] = make_float2(mean[i], m2[i]);
    }
    gn_sync(s.work);
    // groups, `lanes` threads each
    const int lane = threadIdx.x & (s.lanes - 1), groups = s.work / s.lanes;
    const int even = all == s.iters * period ? s.iters : 0;      // every thread has as many vectors
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
                    if (s_one_group[e] == g) f(1.0f, make_float2(s_one[e], 0.0f));
        };
        float cnt = 0.0f, sum = 0.0f, m2 = 0.0f;
        sets([&](float c, float2 e) { cnt += c; sum = fmaf(c, e.x, sum); });
        cnt = lanes_sum(cnt, s.lanes); sum = lanes_sum(sum, s.lanes);
        const float mean = cnt > 0.0f ? sum / cnt : 0.0f;
        sets([&](float c, float2 e) { const float d = e.x - mean; m2 += fmaf(c * d, d, e.y); });
        m2 = lanes_sum(m2, s.lanes);
        if (lane == 0 && g < s.G) p.partial[((int64_t)t.n * s.tiles + t.tile) * s.G + g] = make_float4(cnt, mean, m2, 0.0f);
    }
}

// a sample's statistics from its tiles'
__device__ __forceinline__ void gn_merge_stats(const GnParams& p, int n) {
    const GnShape& s = p.s;
    const int lane = threadIdx.x & (s.lanes - 1), groups = s.work / s.lanes;
    const float total = (float)(s.L / s.C) * (float)s.cg;
    for (int g0 = 0; g0 < s.G; g0 += groups) {
        const int g = g0 + threadIdx.x / s.lanes, tiles = g < s.G ? s.tiles : 0;
        const float4* e = p.partial + (int64_t)n * s.tiles * s.G + g;
        float sum = 0.0f, m2 = 0.0f;
#pragma unroll 8
        for (int k = lane; k < tiles; k += s.lanes) { const float4 v = __ldcg(e + (int64_t)k * s.G); sum = fmaf(v.x, v.y, sum); }
        const float mean = lanes_sum(sum, s.lanes) / total;
#pragma unroll 8
        for (int k = lane; k < tiles; k += s.lanes) { const float4 v = __ldcg(e + (int64_t)k * s.G); const float d = v.y - mean; m2 += fmaf(v.x * d, d, v.z); }
        m2 = lanes_sum(m2, s.lanes);
        if (lane == 0 && g < s.G) p.stats[(int64_t)n * s.G + g] = make_float2(mean, rsqrtf(m2 / total + p.eps));
    }
}

// A thread's channels: y or dx = a function of x - mean with factors that are the channels' or, JOINT, the group's.
template <int V, bool JOINT> struct GnChannels {
    static constexpr int S = JOINT ? 1 : V;
    float mean[S], a[V], b[V];                              // z = (x - mean) a + b
    __device__ __forceinline__ GnChannels(const GnParams& p, const GnTask& t, const GnThread& me, const float2* stats) {
        float rstd = 0.0f;
        if constexpr (JOINT) { const float2 st = gn_load2(stats + me.col * V / p.s.cg); mean[0] = st.x; rstd = st.y; }
        gn_channels<V>(t, me, p.s, [&](int i, int c, int g) {
            float r = rstd;
            if constexpr (!JOINT) { const float2 st = gn_load2(stats + g); mean[i] = st.x; r = st.y; }
            a[i] = r * (p.w ? __ldg(p.w + c) : 1.0f);
            b[i] = p.b ? __ldg(p.b + c) : 0.0f;
        });
    }
    __device__ __forceinline__ float centred(float x, int i) const { return x - mean[JOINT ? 0 : i]; }
};

// ---- forward: y --------------------------------------------------------------------------------------------------------------------
template <class T, bool JOINT, bool KEEP>
__device__ __forceinline__ void gn_apply_tile(const GnParams& p, const GnTask& t, const GnRing& ring, GnThread& me) {
    constexpr int V = Pack<T>::N;
    const GnShape& s = p.s;
    const float2* stats = p.stats + (int64_t)t.n * s.G;
    if (threadIdx.x < t.head_here + t.tail_here) {
        const int64_t at = gn_single(t, s, threadIdx.x);
        const int c = (int)(at % s.C);
        const float2 st = gn_load2(stats + c / s.cg);
        float z[1] = {fmaf(to_f32(((const T*)p.x)[t.first + at]) - st.x, st.y * (p.w ? p.w[c] : 1.0f), p.b ? p.b[c] : 0.0f)};
        act_values(p.act, z);
        ((T*)p.out)[t.first + at] = from_f32<T>(z[0]);
    }
    const GnChannels<V, JOINT> ch(p, t, me, stats);
    const int period = me.period, mine = me.mine;
    int64_t at = t.base + mine * V;
    int left = t.left;
    do {
        if (!gn_chunk(ring, me)) break;
        const T* x = reinterpret_cast<const T*>(ring.smem + me.at % GN_STAGES * ring.stage_bytes) + mine * V;
        const bool whole = left >= GN_ROWS * period;
#pragma unroll
        for (int u = 0; u < GN_ROWS; ++u) {
            if (me.active && (whole || u * period + mine < left)) {
                float v[V];
                load_pack(x + u * period * V, v);
                const int64_t o = at + u * period * V;
                // (C a multiple of 32: the lanes that share a block of the checkpoint take part together)
                if constexpr (KEEP) q8_store(p.out_codes, p.out_steps, o, v, (Q8_BLOCK / V == 8 ? 0xffu : 0xfu) << (threadIdx.x & 31 & ~(Q8_BLOCK / V - 1)));
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = fmaf(ch.centred(v[i], i), ch.a[i], ch.b[i]);
                act_values(p.act, v);
                store_pack((T*)p.out + o, v);
            }
        }
        at += GN_ROWS * period * V;
        left -= GN_ROWS * period;
        gn_free(ring, me);
    } while (left > 0);
}

// What every block has: the ring, its barriers, and the computing threads' scratch.
template <class T> __device__ __forceinline__ GnRing gn_ring(const GnParams& p, uint8_t* smem, int tensors) {
    GnRing r;
    r.stage_bytes = p.s.R * p.s.K * GN_ROWS * 16 * tensors;
    r.smem = smem + GN_HEADER;
    r.bars = smem_u32(smem);
    r.task = reinterpret_cast<GnTask*>(smem + 64);
    r.abort_flag = reinterpret_cast<volatile int*>(smem + 48);
    if (threadIdx.x == 0) {
        for (int k = 0; k < GN_STAGES; ++k) { mbar_init(r.full(k), 1); mbar_init(r.empty(k), p.s.work >> 5); }
        *r.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    return r;
}

template <class T, bool JOINT, bool KEEP> __global__ void __launch_bounds__(GN_MAX_WORK + 32)
gn_forward_kernel(const GnParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int slot[2];
    const GnShape& s = p.s;
    const GnRing ring = gn_ring<T>(p, smem, 1);
    float2* scratch = reinterpret_cast<float2*>(ring.smem + GN_STAGES * ring.stage_bytes);
    if (threadIdx.x >= s.work) {
        if (threadIdx.x == s.work) gn_produce<T>(p, ring, (const T*)p.x, nullptr);
        return;
    }
    for (GnThread me(s);;) {
        const bool ready = gn_chunk(ring, me);
        if (!gn_all(ready, s.work)) return;
        const GnTask& t = ring.task[me.item++ % (GN_STAGES + 1)];
        if (t.kind == 0) return;
        if (t.kind == 1) {
            const int n = t.n;
            gn_stats_tile<T, JOINT>(p, t, ring, me, scratch);
            if (gn_last(p.count + n, s.tiles, slot, s.work)) {
                gn_merge_stats(p, n);
                gn_raise(p.flag + n, s.work);
            }
        } else {
            if (!gn_wait(p.flag + t.n, slot + 1, ring.abort_flag, s.work)) return;
            gn_apply_tile<T, JOINT, KEEP>(p, t, ring, me);
        }
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------
template <class T, bool CODES> __device__ __forceinline__ float gn_load_single(const GnParams& p, int64_t at) {
    if constexpr (CODES) return (float)p.codes[at] * q8_step(p.steps[at >> 5]);
    else return to_f32(((const T*)p.x)[at]);
}

// f(offset, x, dy) for each of this thread's vectors of a tile.  dy comes through the ring, and x with it; the codes of a checkpoint,
// which need not begin on a 16-byte boundary, are loaded here, a chunk ahead.
template <class T, bool CODES, class F>
__device__ __forceinline__ void gn_bwd_chunks(const GnParams& p, const GnTask& t, const GnRing& ring, GnThread& me, F&& f) {
    constexpr int V = Pack<T>::N, W = V / 4;
    const int period = me.period, mine = me.mine;
    int64_t at = t.base + mine * V;
    int left = t.left;
    uint32_t q[CODES ? GN_ROWS : 1][W];
    uint32_t e[CODES ? GN_ROWS : 1];
    auto fetch = [&](int64_t from, int n) {
#pragma unroll
        for (int u = 0; u < GN_ROWS; ++u)
            if (me.active && u * period + mine < n) {
                const int64_t o = from + u * period * V;
                if constexpr (W == 1) q[u][0] = __ldg(reinterpret_cast<const uint32_t*>(p.codes + o));
                else { const uint2 w = __ldg(reinterpret_cast<const uint2*>(p.codes + o)); q[u][0] = w.x; q[u][W - 1] = w.y; }
                e[u] = __ldg(p.steps + (o >> 5));
            }
    };
    if constexpr (CODES) fetch(at, left);
    do {
        if (!gn_chunk(ring, me)) break;
        const T* d = reinterpret_cast<const T*>(ring.smem + me.at % GN_STAGES * ring.stage_bytes) + mine * V;
        const T* x = d + GN_ROWS * period * V;
        const bool whole = left >= GN_ROWS * period;
#pragma unroll
        for (int u = 0; u < GN_ROWS; ++u) {
            if (me.active && (whole || u * period + mine < left)) {
                float vd[V], vx[V];
                load_pack(d + u * period * V, vd);
                if constexpr (CODES) {
                    const float step = q8_step(e[u]);
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        float four[4];
                        q8_decode(q[u][w], step, four);
#pragma unroll
                        for (int i = 0; i < 4; ++i) vx[4 * w + i] = four[i];
                    }
                } else load_pack(x + u * period * V, vx);
                f(at + u * period * V, vx, vd);
            }
        }
        gn_free(ring, me);
        at += GN_ROWS * period * V;
        left -= GN_ROWS * period;
        if constexpr (CODES) fetch(at, left);
    } while (left > 0);
}

// sums of dz and dz xh of each channel over a tile's pixels
template <class T, bool JOINT, bool CODES>
__device__ __forceinline__ void gn_bwd_sums_tile(const GnParams& p, const GnTask& t, const GnRing& ring, GnThread& me, float2* s_sum) {
    constexpr int V = Pack<T>::N;                           // s_sum: [R][K V]
    __shared__ float2 s_one[2 * V];
    __shared__ int s_one_channel[2 * V];
    const GnShape& s = p.s;
    const float2* stats = p.stats + (int64_t)t.n * s.G;
    const int singles = t.head_here + t.tail_here;
    if (threadIdx.x < singles) {
        const int64_t at = gn_single(t, s, threadIdx.x);
        const int c = (int)(at % s.C);
        const float2 st = stats[c / s.cg];
        const float xm = gn_load_single<T, CODES>(p, t.first + at) - st.x;
        const float z[1] = {fmaf(xm, st.y * (p.w ? p.w[c] : 1.0f), p.b ? p.b[c] : 0.0f)};
        float d[1] = {to_f32(((const T*)p.dy)[t.first + at])};
        act_slopes(p.act, z, d);
        s_one[threadIdx.x] = make_float2(d[0], d[0] * xm);
        s_one_channel[threadIdx.x] = c;
    }
    float A[V], B[V];
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = B[i] = 0.0f;
    const GnChannels<V, JOINT> ch(p, t, me, stats);
    gn_bwd_chunks<T, CODES>(p, t, ring, me, [&](int64_t, float (&v)[V], float (&d)[V]) {
        float z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { v[i] = ch.centred(v[i], i); z[i] = fmaf(v[i], ch.a[i], ch.b[i]); }
        act_slopes(p.act, z, d);
#pragma unroll
        for (int i = 0; i < V; ++i) { A[i] += d[i]; B[i] = fmaf(d[i], v[i], B[i]); }
    });
    if (me.active) {
#pragma unroll
        for (int i = 0; i < V; ++i) s_sum[me.mine * V + i] = make_float2(A[i], B[i]);
    }
    gn_sync(s.work);
    const int phase = t.head < s.C ? t.head : t.head % s.C;
    for (int c = threadIdx.x; c < s.C; c += s.work) {
        float2 sum = make_float2(0.0f, 0.0f);
        const float2* from = s_sum + (c >= phase ? c - phase : c - phase + s.C);
        for (int r = 0; r < s.R; ++r, from += s.K * V)
            for (int m = 0; m < s.mult; ++m) { const float2 v = from[m * s.C]; sum.x += v.x; sum.y += v.y; }
        for (int e = 0; e < singles; ++e)
            if (s_one_channel[e] == c) { sum.x += s_one[e].x; sum.y += s_one[e].y; }
        p.chan[((int64_t)t.n * s.tiles + t.tile) * s.C + c] = make_float2(sum.x, sum.y * stats[c / s.cg].y);
    }
}

// Sums over `count` rows of [count][C]: threads take channels and every `rows`-th row, their sums are added in order; f(channel, sum).
template <class F> __device__ __forceinline__ void gn_column_sums(const float2* v, int count, int C, int work, float2* s_mem, F&& f) {
    const int rows = C >= work ? 1 : work / C;
    for (int c0 = 0; c0 < C; c0 += work) {                  // (one pass unless C is larger than the block)
        const int r = rows == 1 ? 0 : (int)threadIdx.x / C, c = rows == 1 ? c0 + (int)threadIdx.x : (int)threadIdx.x - r * C;
        float2 sum = make_float2(0.0f, 0.0f);
        if (r < rows && c < C)
#pragma unroll 8
            for (int k = r; k < count; k += rows) { const float2 e = __ldcg(v + (int64_t)k * C + c); sum.x += e.x; sum.y += e.y; }
        if (rows > 1) {
            gn_sync(work);
            if (r < rows) s_mem[threadIdx.x] = sum;
            gn_sync(work);
            if (r == 0)
                for (int k = 1; k < rows; ++k) { const float2 e = s_mem[k * C + c]; sum.x += e.x; sum.y += e.y; }
        }
        if (r == 0 && c < C) f(c, sum);
    }
    gn_sync(work);
}
// a sample's sums, and its groups' means
__device__ __forceinline__ void gn_bwd_merge(const GnParams& p, int n, float2* s_mem) {
    const GnShape& s = p.s;
    float2* sums = p.sums + (int64_t)n * s.C;
    gn_column_sums(p.chan + (int64_t)n * s.tiles * s.C, s.tiles, s.C, s.work, s_mem, [&](int c, float2 v) { sums[c] = v; });
    const int lane = threadIdx.x & (s.lanes - 1), groups = s.work / s.lanes;
    const float total = (float)(s.L / s.C) * (float)s.cg;
    for (int g0 = 0; g0 < s.G; g0 += groups) {
        const int g = g0 + threadIdx.x / s.lanes;
        float c1 = 0.0f, c2 = 0.0f;
        for (int k = lane; k < s.cg && g < s.G; k += s.lanes) {
            const int c = g * s.cg + k;
            const float2 v = sums[c];                       // (of this block)
            const float w = p.w ? p.w[c] : 1.0f;
            c1 = fmaf(w, v.x, c1); c2 = fmaf(w, v.y, c2);
        }
        c1 = lanes_sum(c1, s.lanes); c2 = lanes_sum(c2, s.lanes);
        if (lane == 0 && g < s.G) p.means[(int64_t)n * s.G + g] = make_float2(c1 / total, c2 / total);
    }
}

template <class T, bool JOINT, bool CODES>
__device__ __forceinline__ void gn_bwd_apply_tile(const GnParams& p, const GnTask& t, const GnRing& ring, GnThread& me) {
    constexpr int V = Pack<T>::N, S = JOINT ? 1 : V;
    const GnShape& s = p.s;
    const float2* stats = p.stats + (int64_t)t.n * s.G;
    const float2* means = p.means + (int64_t)t.n * s.G;
    if (threadIdx.x < t.head_here + t.tail_here) {
        const int64_t at = gn_single(t, s, threadIdx.x);
        const int c = (int)(at % s.C);
        const float2 st = stats[c / s.cg], k = gn_load2(means + c / s.cg);
        const float xm = gn_load_single<T, CODES>(p, t.first + at) - st.x, a = st.y * (p.w ? p.w[c] : 1.0f);
        const float z[1] = {fmaf(xm, a, p.b ? p.b[c] : 0.0f)};
        float d[1] = {to_f32(((const T*)p.dy)[t.first + at])};
        act_slopes(p.act, z, d);
        ((T*)p.out)[t.first + at] = from_f32<T>(fmaf(xm, -st.y * st.y * k.y, fmaf(a, d[0], -st.y * k.x)));
    }
    const GnChannels<V, JOINT> ch(p, t, me, stats);
    float k1[S], k2[S];
    auto constants = [&](int i, int g) { const float2 st = stats[g], k = gn_load2(means + g); k1[i] = -st.y * k.x; k2[i] = -st.y * st.y * k.y; };
    if constexpr (JOINT) constants(0, me.col * V / s.cg);
    else gn_channels<V>(t, me, s, [&](int i, int, int g) { constants(i, g); });
    gn_bwd_chunks<T, CODES>(p, t, ring, me, [&](int64_t at, float (&v)[V], float (&d)[V]) {
        float z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { v[i] = ch.centred(v[i], i); z[i] = fmaf(v[i], ch.a[i], ch.b[i]); }
        act_slopes(p.act, z, d);
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = fmaf(v[i], k2[JOINT ? 0 : i], fmaf(ch.a[i], d[i], k1[JOINT ? 0 : i]));
        store_pack((T*)p.out + at, d);
    });
}

template <class T, bool JOINT, bool CODES> __global__ void __launch_bounds__(GN_MAX_WORK + 32)
gn_backward_kernel(const GnParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int slot[2];
    const GnShape& s = p.s;
    const GnRing ring = gn_ring<T>(p, smem, CODES ? 1 : 2);
    float2* scratch = reinterpret_cast<float2*>(ring.smem + GN_STAGES * ring.stage_bytes);
    if (threadIdx.x >= s.work) {
        if (threadIdx.x == s.work) gn_produce<T>(p, ring, (const T*)p.dy, CODES ? nullptr : (const T*)p.x);
        return;
    }
    for (GnThread me(s);;) {
        const bool ready = gn_chunk(ring, me);
        if (!gn_all(ready, s.work)) return;
        const GnTask& t = ring.task[me.item++ % (GN_STAGES + 1)];
        if (t.kind == 0) return;
        if (t.kind == 1) {
            const int n = t.n;
            gn_bwd_sums_tile<T, JOINT, CODES>(p, t, ring, me, scratch);
            if (gn_last(p.count + n, s.tiles, slot, s.work)) {
                gn_bwd_merge(p, n, scratch);
                gn_raise(p.flag + n, s.work);
                // the block that merges the last sample adds up the parameters' gradients
                if (gn_last(p.samples, s.N, slot, s.work))
                    gn_column_sums(p.sums, s.N, s.C, s.work, scratch, [&](int c, float2 v) { if (p.db) p.db[c] = v.x; if (p.dw) p.dw[c] = v.y; });
            }
        } else {
            if (!gn_wait(p.flag + t.n, slot + 1, ring.abort_flag, s.work)) return;
            gn_bwd_apply_tile<T, JOINT, CODES>(p, t, ring, me);
        }
    }
}

int gn_status(bool reset) {
    int v = 0;
    if (reset) return cudaMemcpyToSymbol(g_gn_status, &v, sizeof(int)) == cudaSuccess ? SPGT_OK : SPGT_ERR_LAUNCH;
    return cudaMemcpyFromSymbol(&v, g_gn_status, sizeof(int)) == cudaSuccess ? v : SPGT_ERR_LAUNCH;
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------
static int gn_shape(int N, int64_t P, int C, int G, int dtype, GnShape& s, int tensors = 1) {
    if (N < 0 || P < 0 || C <= 0 || G <= 0 || C % G || dtype < SPGT_F32 || dtype > SPGT_F16) return SPGT_ERR_SHAPE;
    s = GnShape{};
    s.V = dtype == SPGT_F32 ? 4 : 8;
    int d = s.V;
    while (C % d) d >>= 1;                                  // gcd(C, V): V is a power of two
    s.K = C / d; s.mult = s.V / d;
    if (s.K > GN_MAX_WORK || P > ((int64_t)1 << 40) / C) return SPGT_ERR_SHAPE;
    s.N = N; s.L = P * C; s.C = C; s.G = G; s.cg = C / G;
    s.R = (s.K > 256 ? GN_MAX_WORK : 256) / s.K;
    s.work = ceil_div(s.R * s.K, 32) * 32;
    s.lanes = 32;
    while (s.lanes > 1 && s.lanes * G > s.work) s.lanes >>= 1;
    // Tiles of up to 16 rows of vectors (64 KB), fewer where that leaves SMs without a tile, more where a sample would have so many
    // that merging them takes long.
    const int64_t rows = ceil_div<int64_t>(s.L / s.V, (int64_t)s.R * s.K);
    int64_t iters = N > 0 ? rows * N / num_sms() / GN_ROWS * GN_ROWS : 1;
    iters = iters < GN_ROWS ? GN_ROWS : iters > 16 ? 16 : iters;
    if (iters < rows / 512) iters = ceil_div<int64_t>(rows / 512, GN_ROWS) * GN_ROWS;
    s.iters = (int)iters;
    const int64_t tiles = rows > iters ? ceil_div<int64_t>(rows, iters) : 1;
    if (tiles * (N > 0 ? N : 1) > 0x30000000) return SPGT_ERR_SHAPE;
    s.tiles = (int)tiles;
    // Units of 24 MB of what is read, which is more than the blocks that run at a time hold; where two units and their results would
    // not stay in L2, each unit's results follow its sums.
    const int64_t bytes = s.L * (16 / s.V) * tensors, unit = bytes > 0 ? ceil_div<int64_t>((int64_t)24 << 20, bytes) : 1;
    s.unit = (int)(unit > (N > 0 ? N : 1) ? (N > 0 ? N : 1) : unit);
    s.lag = s.unit * bytes <= ((int64_t)40 << 20) ? 1 : 0;
    s.items = 2 * N * s.tiles;
    return SPGT_OK;
}


// Workspace: the counters, which a launch finds zero, then what the tiles leave.
static inline size_t gn_counters(int N) { return ((size_t)(2 * (int64_t)N + 4) * sizeof(int) + 15) / 16 * 16; }
static inline int gn_begin(GnParams& p, void* workspace, cudaStream_t st) {
    if (cudaError_t e = cudaMemsetAsync(workspace, 0, gn_counters(p.s.N), st)) { g_last_cuda_error = (int)e; (void)cudaGetLastError(); return SPGT_ERR_LAUNCH; }
    p.ticket = (int*)workspace; p.samples = p.ticket + 1; p.count = p.ticket + 4; p.flag = p.count + p.s.N;
    return SPGT_OK;
}
static inline size_t gn_smem(const GnShape& s, int tensors, int sets) {
    return GN_HEADER + (size_t)s.R * s.K * (GN_STAGES * GN_ROWS * 16 * tensors + sets * sizeof(float2));
}
static inline unsigned gn_grid(const GnShape& s) {
    const int most = num_sms() * 4;
    return (unsigned)(s.items < most ? s.items : most);
}

template <void (*KERNEL)(const GnParams)> static int gn_launch(const GnParams& p, size_t smem, cudaStream_t st) {
    static SmemOptIn configured;
    if (int e = smem_opt_in(KERNEL, smem, configured)) return e;
    KERNEL<<<gn_grid(p.s), p.s.work + 32, smem, st>>>(p);
    return launch_status();
}

}  // namespace spgt

using namespace spgt;

extern "C" size_t spgt_group_norm_workspace_bytes(int N, int64_t P, int C, int G, int dtype) {
    GnShape s;
    if (gn_shape(N, P, C, G, dtype, s)) return 0;
    return gn_counters(N) + (size_t)s.N * s.tiles * s.G * sizeof(float4);
}
extern "C" size_t spgt_group_norm_bwd_workspace_bytes(int N, int64_t P, int C, int G, int dtype) {
    GnShape s;
    if (gn_shape(N, P, C, G, dtype, s)) return 0;
    return gn_counters(N) + (((size_t)s.N * s.tiles + s.N) * s.C + (size_t)N * G) * sizeof(float2);
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
    const GnShape& s = p.s;
    const cudaStream_t st = (cudaStream_t)stream;
    if (int e = gn_begin(p, workspace, st)) return e;
    p.x = x; p.out = y; p.w = w; p.b = b; p.stats = (float2*)stats; p.eps = eps; p.act = act;
    p.partial = (float4*)((char*)workspace + gn_counters(N));
    p.out_codes = codes; p.out_steps = steps;
    const bool joint = s.cg % s.V == 0, keep = codes && C % Q8_BLOCK == 0;
    const size_t smem = gn_smem(s, 1, joint ? 1 : s.V);
    // (the checkpoint where blocks of 32 values are not whole lanes of the kernel: first, since y may be x)
    if (codes && !keep)
        if (int e = spgt_compress8(x, dtype, SPGT_ACT_NONE, nullptr, codes, steps, N * s.L, stream)) return e;
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        if (keep && joint) return gn_launch<gn_forward_kernel<T, true, true>>(p, smem, st);
        if (keep) return gn_launch<gn_forward_kernel<T, false, true>>(p, smem, st);
        if (joint) return gn_launch<gn_forward_kernel<T, true, false>>(p, smem, st);
        return gn_launch<gn_forward_kernel<T, false, false>>(p, smem, st);
    });
}

extern "C" int spgt_group_norm_bwd(const void* dy, const void* x, const int8_t* codes, const uint8_t* steps, const float* w, const float* b,
                                   const float* stats, void* dx, float* dw, float* db, int N, int64_t P, int C, int G, int act, int dtype,
                                   void* workspace, size_t workspace_bytes, spgt_stream_t stream) {
    GnParams p{};
    if (int e = gn_shape(N, P, C, G, dtype, p.s, 2)) return e;
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
    if (int e = gn_begin(p, workspace, st)) return e;
    p.dy = dy; p.x = x; p.codes = codes; p.steps = steps; p.w = w; p.b = b; p.stats = (float2*)stats; p.out = dx; p.dw = dw; p.db = db; p.act = act;
    const GnShape& s = p.s;
    p.sums = (float2*)((char*)workspace + gn_counters(N));
    p.means = p.sums + (int64_t)N * C;
    p.chan = p.means + (int64_t)N * G;
    const bool joint = s.cg % s.V == 0;
    const size_t smem = gn_smem(s, codes ? 1 : 2, s.V);    // (the scratch holds a value per thread of the merges as well)
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        if (joint) return codes ? gn_launch<gn_backward_kernel<T, true, true>>(p, smem, st) : gn_launch<gn_backward_kernel<T, true, false>>(p, smem, st);
        return codes ? gn_launch<gn_backward_kernel<T, false, true>>(p, smem, st) : gn_launch<gn_backward_kernel<T, false, false>>(p, smem, st);
    });
}

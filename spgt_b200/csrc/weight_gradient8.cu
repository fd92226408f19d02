// dW [N, K] = dy^T x  for dy [rows, N] and an 8-bit checkpoint of x [rows, K] (lowp.cuh), with the column sums of dy: weight and bias
// gradient of a dense layer that kept its input in 8 bits.
//
// On the bf16 tensor cores, exactly: a checkpoint's value has seven significant bits and is a bf16 number as it is; dy is the sum of
// three bf16 numbers (fp32: 8 + 8 + 8 bits, cut off, so nothing overflows), two (fp16) or one (bf16).  All products are exact in fp32.
// The sums run over the rows, and row-major blocks of rows are what an MMA takes as MN-major operands: nothing is transposed.  Eight
// warps load blocks of 64 rows, a block ahead, into registers and store them as bf16 parts with the 128-byte swizzle (64 columns of a row
// are a line); per 16 rows one MMA of 128 x 128 per part.  The accumulate step of an MMA truncates, so after every 64 rows the chain
// restarts and its result is added to fp32 registers.  Blocks split the rows; their results are added by a second kernel in order.
//   warps 0-7 load and convert, 8-15 accumulate, 16 issues the MMAs.  Every wait is a bounded mbarrier poll that records a code on expiry.
// Floor: rows (N e + 1.03 K) bytes of HBM.
#include "lowp.cuh"

namespace spgt {

__device__ int g_w8_status = 0;

constexpr int W8_T = 128, W8_ROWS = 64, W8_STAGES = 2, W8_THREADS = 544;
constexpr int W8_HALF = W8_ROWS * 128;                      // 64 columns of a block's rows: lines of 128 bytes
constexpr int W8_PART = 2 * W8_HALF;
constexpr int W8_BAR = 256;

template <class T> struct W8Parts { static constexpr int N = 3; };
template <> struct W8Parts<__half> { static constexpr int N = 2; };
template <> struct W8Parts<__nv_bfloat16> { static constexpr int N = 1; };
template <class T> constexpr int w8_stage = (W8Parts<T>::N + 1) * W8_PART;
template <class T> constexpr int w8_smem = W8_STAGES * w8_stage<T> + W8_BAR;

struct W8Params {
    const void* dy; const int8_t* codes; const uint8_t* steps;
    float *partial, *colpart;           // [split][tile][128][128], [split][row of tiles][128]
    float *dw, *db;
    int N, K, kt, splits;               // kt: tiles along K
    int64_t rows;
};

// Eight consecutive columns of a row, as loaded.
template <class T> struct W8Dy { uint4 v[sizeof(T) == 4 ? 2 : 1]; };
struct W8X { uint2 q; uint32_t e; };

// a 16-byte unit of bf16 from eight fp32 bit patterns' upper halves
__device__ __forceinline__ uint4 w8_upper(const uint32_t (&b)[8]) {
    return make_uint4(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632), __byte_perm(b[4], b[5], 0x7632), __byte_perm(b[6], b[7], 0x7632));
}
// where unit c (of 16, of eight columns) of row r lies in a part
__device__ __forceinline__ uint32_t w8_at(int r, int c) { return (uint32_t)((c >> 3) * W8_HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

__device__ __forceinline__ uint64_t w8_desc(uint32_t smem) {
    // MN-major, 128-byte swizzle: 64-column blocks W8_HALF apart (leading), groups of eight rows 1024 bytes apart (stride)
    return (uint64_t)((smem >> 4) & 0x3fffu) | ((uint64_t)(W8_HALF >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// D[tmem] (+)= A B: M = N = 128, K = 16, bf16 both, both MN-major, fp32 accumulators
__device__ __forceinline__ void w8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
    constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(W8_T >> 3) << 17) | ((uint32_t)(W8_T >> 4) << 24);
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// VEC: N and K are multiples of eight, so eight columns of a row are in or out together and start on a boundary of their size.
template <class T, bool VEC> __global__ void __launch_bounds__(W8_THREADS, 1) weight_gradient8_kernel(const W8Params p) {
    constexpr int P = W8Parts<T>::N, STAGE = w8_stage<T>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem), bars = base + W8_STAGES * STAGE;
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicCAS(&g_w8_status, 0, 130);
        return;
    }
    auto st_full = [&](uint32_t s) { return bars + 8u * s; };             // [2]
    auto st_empty = [&](uint32_t s) { return bars + 8u * (2 + s); };      // [2]
    auto acc_full = [&](uint32_t s) { return bars + 8u * (4 + s); };      // [2]
    auto acc_empty = [&](uint32_t s) { return bars + 8u * (6 + s); };     // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + W8_STAGES * STAGE + 96);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + W8_STAGES * STAGE + 104);
    const int tid = threadIdx.x, warp = (int)tc_uniform(tid >> 5), lane = tid & 31;
    const int tile = blockIdx.y, n0 = tile / p.kt * W8_T, k0 = tile % p.kt * W8_T;
    const int64_t blocks = (p.rows + W8_ROWS - 1) / W8_ROWS, first = blocks * blockIdx.x / p.splits;
    const int mine = (int)(blocks * (blockIdx.x + 1) / p.splits - first);
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) { mbar_init(st_full(s), 256); mbar_init(st_empty(s), 1); mbar_init(acc_full(s), 1); mbar_init(acc_empty(s), 256); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(256) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tc_uniform(*tmem_slot);
    float sums[8] = {};

    if (warp < 8) {
        // ------------------------------------------ load and convert: unit c of rows r0, r0 + 16, ... ------------------------------------------
        const int c = lane & 15, r0 = warp * 2 + (lane >> 4);
        const int nc = n0 + c * 8, kc = k0 + c * 8;         // first column of dy and x
        W8Dy<T> dy[2][4];
        W8X x[2][4];
        auto load = [&](int k, W8Dy<T> (&d)[4], W8X (&v)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t r = (first + k) * W8_ROWS + r0 + 16 * i;
                const bool in = k < mine && r < p.rows;
                const T* from = (const T*)p.dy + r * p.N + nc;
                const int64_t at = r * p.K + kc;
#pragma unroll
                for (int j = 0; j < (int)(sizeof(d[i].v) / 16); ++j) d[i].v[j] = make_uint4(0, 0, 0, 0);
                v[i].q = make_uint2(0, 0); v[i].e = 1;
                if constexpr (VEC) {
                    if (in && nc < p.N) {
#pragma unroll
                        for (int j = 0; j < (int)(sizeof(d[i].v) / 16); ++j) d[i].v[j] = __ldg(reinterpret_cast<const uint4*>(from) + j);
                    }
                    if (in && kc < p.K) {
                        v[i].q = __ldg(reinterpret_cast<const uint2*>(p.codes + at));
                        v[i].e = __ldg(p.steps + (at >> 5));
                    }
                } else if (in) {
                    T* to = reinterpret_cast<T*>(&d[i]);
                    uint8_t* codes = reinterpret_cast<uint8_t*>(&v[i].q);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (nc + j < p.N) to[j] = from[j];
                        if (kc + j < p.K) codes[j] = (uint8_t)p.codes[at + j];
                    }
                    // the steps of the eight values: those of the first and, from `from_second` on, of the next block
                    if (kc < p.K) {
                        const int64_t blocks32 = (p.rows * p.K + 31) >> 5, b = at >> 5;
                        v[i].e = p.steps[b] | (b + 1 < blocks32 ? (uint32_t)p.steps[b + 1] << 8 : 0u) | (uint32_t)(32 - (int)(at & 31)) << 16;
                    }
                }
            }
        };
        auto store = [&](int s, const W8Dy<T> (&d)[4], const W8X (&v)[4]) {
            uint8_t* stage = smem + s * STAGE;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t at = w8_at(r0 + 16 * i, c);
                if constexpr (P == 1) {
                    *reinterpret_cast<uint4*>(stage + at) = d[i].v[0];
                    const uint32_t w[4] = {d[i].v[0].x, d[i].v[0].y, d[i].v[0].z, d[i].v[0].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) { sums[2 * j] += __uint_as_float(w[j] << 16); sums[2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u); }
                } else {
                    float f[8];
                    if constexpr (P == 3) {
                        const uint32_t w[8] = {d[i].v[0].x, d[i].v[0].y, d[i].v[0].z, d[i].v[0].w, d[i].v[P == 3].x, d[i].v[P == 3].y, d[i].v[P == 3].z, d[i].v[P == 3].w};
#pragma unroll
                        for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
                    } else {
                        const uint32_t w[4] = {d[i].v[0].x, d[i].v[0].y, d[i].v[0].z, d[i].v[0].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) { const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[j])); f[2 * j] = g.x; f[2 * j + 1] = g.y; }
                    }
                    uint32_t b[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) { sums[j] += f[j]; b[j] = __float_as_uint(f[j]); }
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        *reinterpret_cast<uint4*>(stage + q * W8_PART + at) = w8_upper(b);
                        if (q + 1 < P) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) {           // the rest; none of an infinity
                                const float h = __uint_as_float(b[j] & 0xffff0000u), g = __uint_as_float(b[j]);
                                b[j] = __float_as_uint(h == g ? 0.0f : g - h);
                            }
                        }
                    }
                }
                float2 y[4];
                const uint32_t w[2] = {v[i].q.x ^ 0x80808080u, v[i].q.y ^ 0x80808080u};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    y[j] = add2(make_float2(__uint_as_float(__byte_perm(w[j >> 1], 0x4b000000u, 0x7540 + 2 * (j & 1))), __uint_as_float(__byte_perm(w[j >> 1], 0x4b000000u, 0x7541 + 2 * (j & 1)))), pair(-8388736.0f));
                if constexpr (VEC) {
                    const float2 step = pair(q8_step(v[i].e));
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = mul2(y[j], step);
                } else {
                    const float s0 = q8_step(v[i].e & 255u), s1 = q8_step(v[i].e >> 8 & 255u);
                    const int second = (int)(v[i].e >> 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        y[j].x = kc + 2 * j < p.K ? y[j].x * (2 * j < second ? s0 : s1) : 0.0f;
                        y[j].y = kc + 2 * j + 1 < p.K ? y[j].y * (2 * j + 1 < second ? s0 : s1) : 0.0f;
                    }
                }
                *reinterpret_cast<uint4*>(stage + P * W8_PART + at) = pack_pairs(y, __nv_bfloat16{});
            }
        };
        load(0, dy[0], x[0]);
        uint32_t s = 0, ph = 1;
        bool alive = true;
        auto step = [&](int k, int cur) {
            load(k + 1, dy[cur ^ 1], x[cur ^ 1]);
            if (!mbar_wait(st_empty(s), ph, abort_flag, 131, &g_w8_status)) { alive = false; return; }
            store(s, dy[cur], x[cur]);
            fence_proxy_async();
            mbar_arrive(st_full(s));
            if (++s == W8_STAGES) { s = 0; ph ^= 1u; }
        };
        for (int k = 0; k < mine && alive; k += 2) {
            step(k, 0);
            if (k + 1 < mine && alive) step(k + 1, 1);
        }
    } else if (warp == 16) {
        // ------------------------------------------ MMA issuer ------------------------------------------
        if (tc_elect()) {
            uint32_t s = 0, ph = 0;
            for (int k = 0; k < mine; ++k) {
                const uint32_t buf = (uint32_t)(k & 1), d = tmem_base + buf * W8_T;
                if (!mbar_wait(acc_empty(buf), (uint32_t)((k >> 1) & 1) ^ 1u, abort_flag, 132, &g_w8_status)) break;
                if (!mbar_wait(st_full(s), ph, abort_flag, 133, &g_w8_status)) break;
                tc_fence_after();
                const uint32_t st = base + s * STAGE;
                const uint64_t a = w8_desc(st), b = w8_desc(st + P * W8_PART);
#pragma unroll
                for (int q = P - 1; q >= 0; --q)            // the smallest parts first
#pragma unroll
                    for (int k16 = 0; k16 < W8_ROWS / 16; ++k16)
                        w8_mma(d, a + q * (W8_PART >> 4) + k16 * 128, b + k16 * 128, q < P - 1 || k16 > 0 ? 1u : 0u);
                tc_commit(st_empty(s));
                tc_commit(acc_full(buf));
                if (++s == W8_STAGES) { s = 0; ph ^= 1u; }
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------ accumulation ------------------------------------------
        const int q = warp & 3, half = (warp - 8) >> 2;     // columns 64 half .. + 63 of this lane's row
        const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
        float acc[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = 0.0f;
        bool alive = true;
        for (int k = 0; k < mine; ++k) {
            const uint32_t buf = (uint32_t)(k & 1);
            if (!mbar_wait(acc_full(buf), (uint32_t)((k >> 1) & 1), abort_flag, 134, &g_w8_status)) { alive = false; break; }
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < 64; j += 16) {
                float v[16];
                tc_ld16(tmem_base + lane_addr + buf * W8_T + half * 64 + j, v);
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[j + e] += v[e];
            }
            tc_fence_before();
            mbar_arrive(acc_empty(buf));
        }
        if (alive) {
            float* out = p.partial + (((int64_t)blockIdx.x * gridDim.y + tile) * W8_T + q * 32 + lane) * W8_T + half * 64;
#pragma unroll
            for (int j = 0; j < 16; ++j) reinterpret_cast<float4*>(out)[j] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(256) : "memory");
    }
    // column sums of dy: 16 threads have a column each; the stages are free
    if (k0 == 0 && p.db) {
        float* part = reinterpret_cast<float*>(smem);
        if (warp < 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) part[(warp * 2 + (lane >> 4)) * W8_T + (lane & 15) * 8 + j] = sums[j];
        }
        __syncthreads();
        if (tid < W8_T) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < 16; ++k) s += part[k * W8_T + tid];
            p.colpart[((int64_t)blockIdx.x * (gridDim.y / p.kt) + tile / p.kt) * W8_T + tid] = s;
        }
    }
}

// dw and db from the splits' results.  Eight threads share a result (four columns of a row, or a column sum): thread g adds results g,
// g + 8, ..., and the eight sums are added in order.
__global__ void __launch_bounds__(256) weight_gradient8_reduce_kernel(const W8Params p, int tiles) {
    __shared__ float4 part[8][32];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c_blocks = tiles * (W8_T * W8_T / 4 / 32);
    pdl_launch_next();
    pdl_wait();
    if ((int)blockIdx.x < c_blocks) {
        const int i = blockIdx.x * 32 + lane;               // of the padded [tiles][128][128 / 4]
        const int c4 = i % (W8_T / 4), r = i / (W8_T / 4) % W8_T, tile = i / (W8_T * W8_T / 4);
        const int row = tile / p.kt * W8_T + r, col = tile % p.kt * W8_T + c4 * 4;
        const bool in = row < p.N && col < p.K;
        const float4* src = reinterpret_cast<const float4*>(p.partial) + i;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in)
#pragma unroll 8
            for (int k = g; k < p.splits; k += 8) {
                const float4 v = __ldca(src + (int64_t)k * tiles * (W8_T * W8_T / 4));
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
        part[g][lane] = s;
        __syncthreads();
        if (g || !in) return;
#pragma unroll
        for (int k = 1; k < 8; ++k) { const float4 v = part[k][lane]; s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; }
        const float o[4] = {s.x, s.y, s.z, s.w};
        float* dst = p.dw + (int64_t)row * p.K + col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.K) dst[e] = o[e];
    } else {
        const int c = (blockIdx.x - c_blocks) * 32 + lane;  // (whole tiles of columns)
        float s = 0.0f;
#pragma unroll 8
        for (int k = g; k < p.splits; k += 8) s += __ldca(p.colpart + (int64_t)k * (tiles / p.kt) * W8_T + c);
        part[g][lane].x = s;
        __syncthreads();
        if (g || c >= p.N) return;
#pragma unroll
        for (int k = 1; k < 8; ++k) s += part[k][lane].x;
        p.db[c] = s;
    }
}

// Blocks that share the rows: one wave over the SMs, at least two blocks of rows each
static int w8_splits(int N, int K, int64_t rows) {
    const int tiles = ceil_div(N, W8_T) * ceil_div(K, W8_T), most = num_sms() / tiles < 1 ? 1 : num_sms() / tiles;
    const int64_t want = ceil_div<int64_t>(rows, W8_ROWS * 2);
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

int w8_status(bool reset) {
    int v = 0;
    if (reset) return cudaMemcpyToSymbol(g_w8_status, &v, sizeof(int)) == cudaSuccess ? SPGT_OK : SPGT_ERR_LAUNCH;
    return cudaMemcpyFromSymbol(&v, g_w8_status, sizeof(int)) == cudaSuccess ? v : SPGT_ERR_LAUNCH;
}

template <class T, bool VEC> static int w8_launch(const W8Params& p, int tiles, cudaStream_t st) {
    static SmemOptIn configured;
    if (int e = smem_opt_in(weight_gradient8_kernel<T, VEC>, w8_smem<T>, configured)) return e;
    ChainScope chain;
    if (int e = launch_chained(weight_gradient8_kernel<T, VEC>, dim3((unsigned)p.splits, (unsigned)tiles), W8_THREADS, w8_smem<T>, st, p)) return e;
    return launch_chained(weight_gradient8_reduce_kernel, dim3((unsigned)(tiles * (W8_T * W8_T / 4 / 32) + (p.db ? tiles / p.kt * (W8_T / 32) : 0))), 256, 0, st, p, tiles);
}

}  // namespace spgt

using namespace spgt;

extern "C" size_t spgt_weight_gradient8_workspace_bytes(int N, int K, int64_t rows) {
    if (N <= 0 || K <= 0 || rows < 0 || N > 4096 || K > 4096 || rows > ((int64_t)1 << 36)) return 0;
    const size_t tiles = (size_t)ceil_div(N, W8_T) * ceil_div(K, W8_T);
    return (size_t)w8_splits(N, K, rows) * (tiles * W8_T + ceil_div(N, W8_T)) * W8_T * sizeof(float);
}

extern "C" int spgt_weight_gradient8(const void* dy, int dtype, const int8_t* codes, const uint8_t* steps, float* dw, float* db, int N, int K,
                                     int64_t rows, void* workspace, size_t workspace_bytes, spgt_stream_t stream) {
    const size_t need = spgt_weight_gradient8_workspace_bytes(N, K, rows);
    if (need == 0 || dtype < SPGT_F32 || dtype > SPGT_F16) return SPGT_ERR_SHAPE;
    if (!dw || !workspace || (rows > 0 && (!dy || !codes || !steps))) return SPGT_ERR_NULL;
    if (workspace_bytes < need) return SPGT_ERR_WORKSPACE;
    if (!aligned16(dy) || !aligned16(codes) || !aligned16(workspace)) return SPGT_ERR_ALIGN;
    const int kt = ceil_div(K, W8_T), tiles = ceil_div(N, W8_T) * kt;
    W8Params p{dy, codes, steps, (float*)workspace, nullptr, dw, db, N, K, kt, w8_splits(N, K, rows), rows};
    p.colpart = p.partial + (size_t)p.splits * tiles * W8_T * W8_T;
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        return N % 8 == 0 && K % 8 == 0 ? w8_launch<T, true>(p, tiles, (cudaStream_t)stream) : w8_launch<T, false>(p, tiles, (cudaStream_t)stream);
    });
}

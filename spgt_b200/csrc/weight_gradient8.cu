// dW [N, K] = dy^T x  for dy [rows, N] and an 8-bit checkpoint of x [rows, K] (lowp.cuh), with the column sums of dy: weight and bias
// gradient of a dense layer that kept its input in 8 bits.
//
// On the bf16 tensor cores, exactly: a checkpoint's value has seven significant bits and is a bf16 number as it is; dy is the sum of
// three bf16 numbers (fp32: 8 + 8 + 8 bits, cut off, so nothing overflows), two (fp16) or one (bf16).  All products are exact in fp32.
// The sums run over the rows, and row-major blocks of rows are what an MMA takes as MN-major operands: nothing is transposed.  Eight
// warps copy blocks of 64 rows ahead and store them as bf16 parts with the 128-byte swizzle (64 columns of a row are a line); per 16 rows
// one MMA of 128 x 128 per part.  The accumulate step of an MMA truncates, so after every 128 rows the chain restarts and its result is
// added to fp32 registers.  Blocks split the rows; their results are added by a second kernel in order.
//   warps 0-7 load and convert, 8-15 accumulate, and the first of those issues the MMAs.  Every wait is a bounded mbarrier poll that records a code on expiry.
// Floor: rows (N e + 1.03 K) bytes of HBM.
#include "lowp.cuh"

namespace spgt {

__device__ int g_w8_status = 0;

constexpr int W8_T = 128, W8_ROWS = 64, W8_STAGES = 2, W8_THREADS = 512, W8_LOADERS = 256;
constexpr int W8_HALF = W8_ROWS * 128;                      // 64 columns of a block's rows: lines of 128 bytes
constexpr int W8_PART = 2 * W8_HALF;
constexpr int W8_BAR = 256, W8_CHAIN = 2;                   // blocks of rows that an accumulator sums

template <class T> struct W8Parts { static constexpr int N = 3; };
template <> struct W8Parts<__half> { static constexpr int N = 2; };
template <> struct W8Parts<__nv_bfloat16> { static constexpr int N = 1; };
template <class T> constexpr int w8_stage = (W8Parts<T>::N + 1) * W8_PART;
// raw values of a block of rows, per loading thread: four units of eight columns of dy, in 16-byte pieces, and of codes
template <class T> constexpr int w8_pieces = 8 * (int)sizeof(T) / 16;
template <class T> constexpr int w8_raw = 4 * W8_LOADERS * (16 * w8_pieces<T> + 8);
template <class T> constexpr int W8_RAWS = sizeof(T) == 4 ? 2 : 4;         // blocks of rows under way
template <class T> constexpr int w8_smem = W8_STAGES * w8_stage<T> + W8_RAWS<T> * w8_raw<T> + W8_BAR;

struct W8Params {
    const void* dy; const int8_t* codes; const uint8_t* steps;
    float *partial, *colpart;           // [split][tile][128][128], [split][row of tiles][128]
    float *dw, *db;
    int N, K, kt, splits;               // kt: tiles along K
    int64_t rows;
};

// x less its upper half, for pairs: exact, of an infinity a NaN
__device__ __forceinline__ float2 w8_rest(float2 x) {
    const float2 up = make_float2(__uint_as_float((__float_as_uint(x.x) & 0xffff0000u) ^ 0x80000000u), __uint_as_float((__float_as_uint(x.y) & 0xffff0000u) ^ 0x80000000u));
    return add2(x, up);
}
__device__ __forceinline__ uint32_t w8_upper(float2 x) { return __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632); }
// a 16-byte unit of bf16 from eight fp32 numbers' upper halves
__device__ __forceinline__ uint4 w8_upper(const float2 (&b)[4]) { return make_uint4(w8_upper(b[0]), w8_upper(b[1]), w8_upper(b[2]), w8_upper(b[3])); }
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
    constexpr int P = W8Parts<T>::N, STAGE = w8_stage<T>, RAWS = W8_RAWS<T>, PIECES = w8_pieces<T>, BAR = W8_STAGES * STAGE + RAWS * w8_raw<T>;
    extern __shared__ __align__(1024) uint8_t smem[];
    pdl_launch_next();                                      // (the second kernel waits for the end of this one)
    const uint32_t base = smem_u32(smem), bars = base + BAR;
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicCAS(&g_w8_status, 0, 130);
        return;
    }
    auto st_full = [&](uint32_t s) { return bars + 8u * s; };             // [2]
    auto st_empty = [&](uint32_t s) { return bars + 8u * (2 + s); };      // [2]
    auto acc_full = [&](uint32_t s) { return bars + 8u * (4 + s); };      // [2]
    auto acc_empty = [&](uint32_t s) { return bars + 8u * (6 + s); };     // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + BAR + 96);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + BAR + 104);
    const int tid = threadIdx.x, warp = (int)tc_uniform(tid >> 5), lane = tid & 31;
    const int tile = blockIdx.y, n0 = tile / p.kt * W8_T, k0 = tile % p.kt * W8_T;
    const int64_t blocks = (p.rows + W8_ROWS - 1) / W8_ROWS, first = blocks * blockIdx.x / p.splits;
    const int mine = (int)(blocks * (blockIdx.x + 1) / p.splits - first);
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) { mbar_init(st_full(s), 256); mbar_init(st_empty(s), 1); mbar_init(acc_full(s), 1); mbar_init(acc_empty(s), 256); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(256) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tc_uniform(*tmem_slot);
    float2 sums[4] = {};                                    // of this thread's columns of dy

    if (warp < 8) {
        // ------------------------------------------ load and convert ------------------------------------------
        // eight values of dy, in P parts, and of x, of row r: x of unit c of eight columns; dy of the same, or, fp32, of columns 4 c .. + 3
        // and 64 + 4 c .. + 3, so that the lanes' 16-byte copies are next to each other
        auto store = [&](uint8_t* stage, int r, int c, float2 (&b)[4], const float2 (&y)[4]) {
            const uint32_t at = w8_at(r, c), at4 = w8_at(r, c >> 1) + (c & 1) * 8;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                if constexpr (P == 3) {
                    *reinterpret_cast<uint2*>(stage + q * W8_PART + at4) = make_uint2(w8_upper(b[0]), w8_upper(b[1]));
                    *reinterpret_cast<uint2*>(stage + q * W8_PART + W8_HALF + at4) = make_uint2(w8_upper(b[2]), w8_upper(b[3]));
                } else {
                    *reinterpret_cast<uint4*>(stage + q * W8_PART + at) = w8_upper(b);
                }
                if (q + 1 < P) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) b[j] = w8_rest(b[j]);
                }
            }
            *reinterpret_cast<uint4*>(stage + P * W8_PART + at) = pack_pairs(y, __nv_bfloat16{});
        };
        uint32_t s = 0, ph = 1;
        if constexpr (VEC) {
            // Unit c of rows r0, r0 + 16, ...: each thread copies what it will convert, RAWS blocks of rows ahead, and only waits for itself.
            const int c = lane & 15, r0 = warp * 2 + (lane >> 4);
            const int nc = n0 + c * (16 / (int)sizeof(T)), kc = k0 + c * 8;       // first column of dy and x
            const bool n_in = nc < p.N, n2_in = PIECES == 2 && nc + 64 < p.N, k_in = kc < p.K;
            uint8_t* raw = smem + W8_STAGES * STAGE + tid * 16;
            uint32_t e[2][4];                               // steps, of this block and the next
            const int64_t row0 = first * W8_ROWS + r0, dy_row = (int64_t)p.N * (int)sizeof(T), left0 = p.rows - row0;
            const uint8_t* dy_at = (const uint8_t*)p.dy + row0 * dy_row + (int64_t)nc * (int)sizeof(T);       // of the block to copy
            const int8_t* codes_at = p.codes + row0 * p.K + kc;
            int64_t copy_left = left0 < (int64_t)mine * W8_ROWS ? left0 : (int64_t)mine * W8_ROWS;          // rows from this thread's first one
            int copy_slot = 0;
            auto copy = [&] {
                uint8_t* to = raw + copy_slot * w8_raw<T>;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = 16 * i < copy_left;
                    const int8_t* codes = in && k_in ? codes_at + 16 * i * p.K : p.codes;
                    cp_async_zfill<16>(to + i * PIECES * (W8_LOADERS * 16), in && n_in ? dy_at + 16 * i * dy_row : (const uint8_t*)p.dy, in && n_in);
                    if constexpr (PIECES == 2)
                        cp_async_zfill<16>(to + (2 * i + 1) * (W8_LOADERS * 16), in && n2_in ? dy_at + 16 * i * dy_row + 256 : (const uint8_t*)p.dy, in && n2_in);
                    cp_async_zfill<8>(to + 4 * PIECES * (W8_LOADERS * 16) + i * (W8_LOADERS * 8) - tid * 8, codes, in && k_in);
                }
                cp_async_commit();
                dy_at += W8_ROWS * dy_row; codes_at += W8_ROWS * p.K; copy_left -= W8_ROWS;
                copy_slot = copy_slot == RAWS - 1 ? 0 : copy_slot + 1;
            };
            int64_t value_at = row0 * p.K + kc, step_left = copy_left;
            auto steps = [&](uint32_t (&v)[4]) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = 1;
                    if (16 * i < step_left && k_in) v[i] = __ldg(p.steps + ((value_at + 16 * i * p.K) >> 5));
                }
                value_at += W8_ROWS * p.K; step_left -= W8_ROWS;
            };
            int slot = 0;
            if (mine > 0) {
#pragma unroll
                for (int k = 0; k < RAWS; ++k) copy();
                steps(e[0]);
            }
            auto step = [&](uint32_t (&now)[4], uint32_t (&next)[4]) {
                steps(next);
                cp_async_wait<RAWS - 1>();
                if (!mbar_wait(st_empty(s), ph, abort_flag, 131, &g_w8_status)) return false;
                const uint8_t* from = raw + slot * w8_raw<T>;
                slot = slot == RAWS - 1 ? 0 : slot + 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 b[4];
                    if constexpr (PIECES == 2) {
                        float2 h[2];
                        unpack_pairs(*reinterpret_cast<const uint4*>(from + 2 * i * (W8_LOADERS * 16)), h, 0.0f);
                        b[0] = h[0]; b[1] = h[1];
                        unpack_pairs(*reinterpret_cast<const uint4*>(from + (2 * i + 1) * (W8_LOADERS * 16)), h, 0.0f);
                        b[2] = h[0]; b[3] = h[1];
                    } else {
                        unpack_pairs(*reinterpret_cast<const uint4*>(from + i * (W8_LOADERS * 16)), b, T{});
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) sums[j] = add2(sums[j], b[j]);
                    const uint2 q = *reinterpret_cast<const uint2*>(from + 4 * PIECES * (W8_LOADERS * 16) + i * (W8_LOADERS * 8) - tid * 8);
                    const uint32_t w[2] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u};
                    const float2 size = pair(q8_step(now[i]));
                    float2 y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t v = w[j >> 1];
                        const float2 code = make_float2(__uint_as_float(__byte_perm(v, 0x4b000000u, 0x7540 + 2 * (j & 1))), __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7541 + 2 * (j & 1))));
                        y[j] = mul2(add2(code, pair(-8388736.0f)), size);
                    }
                    store(smem + s * STAGE, r0 + 16 * i, c, b, y);
                }
                copy();
                fence_proxy_async();
                mbar_arrive(st_full(s));
                if (++s == W8_STAGES) { s = 0; ph ^= 1u; }
                return true;
            };
            for (int k = 0; k < mine; k += 2) {
                if (!step(e[0], e[1])) break;
                if (k + 1 < mine && !step(e[1], e[0])) break;
            }
            cp_async_wait_all();
        } else {
            // Any widths: columns 2 lane, 2 lane + 1 (+ 64) of rows warp, warp + 8, ...  Every load has an address inside its array and
            // is zeroed afterwards where it lies outside the tile, so that no branch keeps the loads of four rows apart.
            int ncol[4], kcol[4];                           // columns from the tile's first, inside the matrix
            bool n_in[4], k_in[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int col = 2 * lane + (j >> 1) * 64 + (j & 1);
                n_in[j] = n0 + col < p.N; k_in[j] = k0 + col < p.K;
                ncol[j] = n_in[j] ? col : 0; kcol[j] = k_in[j] ? col : 0;
            }
            for (int k = 0; k < mine; ++k) {
                float d[2][4][4];
                uint32_t codes[2][4][4], size[2][4][4];
                auto load = [&](int batch) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int64_t r = (first + k) * W8_ROWS + warp + 8 * (4 * batch + i);
                        const bool in = r < p.rows;
                        const int64_t row = in ? r : 0, at = row * p.K + k0;
                        const T* dy = (const T*)p.dy + row * p.N + n0;
                        const int8_t* code = p.codes + at;
                        const uint8_t* step = p.steps + (at >> 5);
                        const int phase = (int)(at & 31);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            d[batch][i][j] = to_f32(__ldg(dy + ncol[j]));
                            codes[batch][i][j] = (uint32_t)(int)__ldg(code + kcol[j]);
                            size[batch][i][j] = __ldg(step + ((phase + kcol[j]) >> 5));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (!in || !n_in[j]) d[batch][i][j] = 0.0f;
                            if (!in || !k_in[j]) { codes[batch][i][j] = 0; size[batch][i][j] = 1; }
                        }
                    }
                };
                load(0);
                if (!mbar_wait(st_empty(s), ph, abort_flag, 131, &g_w8_status)) break;
                uint8_t* stage = smem + s * STAGE;
#pragma unroll
                for (int batch = 0; batch < 2; ++batch) {
                    if (batch == 0) load(1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = warp + 8 * (4 * batch + i);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {       // 64-column half
                            uint8_t* at = stage + w8_at(r, 8 * h + (lane >> 2)) + (lane & 3) * 4;
                            float2 b = make_float2(d[batch][i][2 * h], d[batch][i][2 * h + 1]);
                            sums[h] = add2(sums[h], b);
#pragma unroll
                            for (int q = 0; q < P; ++q, b = w8_rest(b)) *reinterpret_cast<uint32_t*>(at + q * W8_PART) = w8_upper(b);
                            *reinterpret_cast<uint32_t*>(at + P * W8_PART) = pack_pair(
                                make_float2((float)(int)codes[batch][i][2 * h] * q8_step(size[batch][i][2 * h]), (float)(int)codes[batch][i][2 * h + 1] * q8_step(size[batch][i][2 * h + 1])),
                                __nv_bfloat16{});
                        }
                    }
                }
                fence_proxy_async();
                mbar_arrive(st_full(s));
                if (++s == W8_STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else {
        // ------------------------------------------ MMAs and accumulation ------------------------------------------
        const int q = warp & 3, half = (warp - 8) >> 2;     // columns 64 half .. + 63 of this lane's row
        const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
        const int chains = (mine + W8_CHAIN - 1) / W8_CHAIN;
        float acc[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = 0.0f;
        bool alive = true;
        uint32_t s = 0, ph = 0;
        // one thread: the MMAs of a chain's blocks of rows
        auto issue = [&](int chain) {
            const uint32_t buf = (uint32_t)(chain & 1), d = tmem_base + buf * W8_T;
            if (!mbar_wait(acc_empty(buf), (uint32_t)((chain >> 1) & 1) ^ 1u, abort_flag, 132, &g_w8_status)) return;
            const int blocks = mine - chain * W8_CHAIN < W8_CHAIN ? mine - chain * W8_CHAIN : W8_CHAIN;
            for (int k = 0; k < blocks; ++k) {
                if (!mbar_wait(st_full(s), ph, abort_flag, 133, &g_w8_status)) return;
                tc_fence_after();
                const uint32_t st = base + s * STAGE;
                const uint64_t a = w8_desc(st), b = w8_desc(st + P * W8_PART);
#pragma unroll
                for (int part = P - 1; part >= 0; --part)   // the smallest parts first
#pragma unroll
                    for (int k16 = 0; k16 < W8_ROWS / 16; ++k16)
                        w8_mma(d, a + part * (W8_PART >> 4) + k16 * 128, b + k16 * 128, part < P - 1 || k16 > 0 || k > 0 ? 1u : 0u);
                tc_commit(st_empty(s));
                if (++s == W8_STAGES) { s = 0; ph ^= 1u; }
            }
            tc_commit(acc_full(buf));
        };
        if (warp == 8 && chains > 0) {
            if (tc_elect()) issue(0);
            __syncwarp();
        }
        for (int k = 0; k < chains; ++k) {
            // (the next chain's MMAs go first: they fill the other buffer while this one is read)
            if (warp == 8 && k + 1 < chains) {
                if (tc_elect()) issue(k + 1);
                __syncwarp();
            }
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
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(256) : "memory");
    }
    // column sums of dy, of several threads each; the stages are free
    if (k0 == 0 && p.db) {
        float* part = reinterpret_cast<float*>(smem);
        constexpr int SHARES = VEC ? 16 : 8;
        if (warp < 8) {
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < 8; ++j) part[(warp * 2 + (lane >> 4)) * W8_T + (P == 3 ? (lane & 15) * 4 + (j >> 2) * 64 + (j & 3) : (lane & 15) * 8 + j)] = j & 1 ? sums[j / 2].y : sums[j / 2].x;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) part[warp * W8_T + 2 * lane + (j >> 1) * 64 + (j & 1)] = j & 1 ? sums[j / 2].y : sums[j / 2].x;
            }
        }
        __syncthreads();
        if (tid < W8_T) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < SHARES; ++k) s += part[k * W8_T + tid];
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

// dW [N, K] = dy^T x  for dy [rows, N] and an 8-bit checkpoint of x [rows, K] (lowp.cuh), with the column sums of dy: weight and bias
// gradient of a dense layer that kept its input in 8 bits.
//
// On the bf16 tensor cores, exactly: a checkpoint's value has seven significant bits and is a bf16 number as it is; dy is the sum of
// three bf16 numbers (fp32: 8 + 8 + 8 bits, cut off, so nothing overflows), two (fp16) or one (bf16).  All products are exact in fp32.
// The sums run over the rows, and row-major blocks of rows are what an MMA takes as MN-major operands: nothing is transposed.  Sixteen
// warps copy blocks of 32 or 64 rows ahead and store them as bf16 parts with the 128-byte swizzle (64 columns of a row are a line); per 16 rows
// and part one MMA of 128 columns of dy x up to 256 of x: so dy is converted once for all of x.
// The accumulate step of an MMA truncates: the upper parts' sums and the others' have accumulators of their own, and after 1280 rows
// they are added to the block's result in memory.  Error against 64 bits, relative, with normal inputs: 8.8e-8 for 7396 rows and 3.2e-7
// for 179776, a plain fp32 product's 5e-7 and 1.3e-6.
// Blocks split the rows; their results are added by a second kernel in order.
// Bound by shared memory: of 179776 rows, dy 128 columns and x 256 in fp32, 42 us, about 10 are the start, the blocks' partial results and
// their sum; in the rest a multiprocessor takes 38 blocks of 32 rows, some 0.8 us each.  For one of them 24 KB are copied in, 24 read back, 40
// stored as parts and 72 read by the MMAs: 160 KB, 1280 cycles at 128 bytes a cycle, about 0.7 us.  (The memory's bytes take 21 us in all.)
// fp16 35 us, bf16 32; dy 256 columns, x 128: fp32 58; 7396 rows, 128 x 136 bf16: 11, 1024 x 1024 fp32 79, bf16 65.  Widths that are no
// multiples of eight are read value by value, nothing ahead: dy 130, x 250 fp32 165 (the bytes 21); 712336 rows, 1 x 128: 233 (15).
//   Warps 0-15 load and convert, 16-19 write the results, the first of those issues the MMAs, and 20 copies where blocks are runs of
// memory (W8_WHOLE).  Every wait is a bounded mbarrier poll that records a code on expiry.
#include "lowp.cuh"

namespace spgt {

__device__ int g_w8_status = 0;

constexpr int W8_T = 128, W8_THREADS = 640, W8_LOADERS = 512, W8_BAR = 256, W8_CHAIN = 1280;    // rows that an accumulator sums

template <class T> struct W8Parts { static constexpr int N = 3; };
template <> struct W8Parts<__half> { static constexpr int N = 2; };
template <> struct W8Parts<__nv_bfloat16> { static constexpr int N = 1; };
// How the blocks of rows are read.  W8_ANY: any widths.  W8_VEC: N and K are multiples of eight, so eight columns of a row are in or out
// together and start on a boundary of their size.  W8_WHOLE: besides, one tile holds all columns, so that a block is three runs of memory,
// which bulk copies bring, and K is a multiple of 16 (179776 rows, 128 x 256 columns: fp32 41.5 us against 48.7 as W8_VEC, bf16 32.3 against
// 41.8; when dy of 256 columns, x 128, took 64 us as W8_VEC, it took 113 with a copy for each row of dy).
constexpr int W8_ANY = 0, W8_VEC = 1, W8_WHOLE = 2;
// BN: columns of x in a tile, 128 or 256, and with it rows of a block.
template <class T, int BN, int MODE> struct W8 {
    static constexpr int P = W8Parts<T>::N, ROWS = BN == 256 ? 32 : 64;
    static constexpr int HALF = ROWS * 128, PART = 2 * HALF;                   // 64 columns of a block's rows: lines of 128 bytes; 128 columns
    static constexpr int STAGE = (P + BN / W8_T) * PART, STAGES = BN == 256 ? (P == 3 ? 3 : 4) : 5 - P;
    // raw values of a block per loading thread: DU times eight columns of dy, in 16-byte pieces, and XU times eight codes
    static constexpr int PIECES = 8 * (int)sizeof(T) / 16, DU = ROWS / 32, XU = ROWS * BN / (8 * W8_LOADERS);
    static constexpr int RAW_CODES = ROWS * W8_T * (int)sizeof(T), RAW_STEPS = RAW_CODES + ROWS * BN;      // W8_WHOLE: dy, codes and steps as they are
    static constexpr int RAW = MODE == W8_WHOLE ? RAW_STEPS + ROWS * BN / Q8_BLOCK : W8_LOADERS * (16 * PIECES * DU + 8 * XU);
    static constexpr int RAWS = MODE != W8_WHOLE ? (BN == 256 ? (P == 3 ? 3 : 4) : 5 - P) : BN == 256 ? (P == 3 ? 4 : 6) : P == 3 ? 2 : P == 2 ? 3 : 4;
    static constexpr int THREADS = W8_THREADS + (MODE == W8_WHOLE ? 32 : 0);
    static constexpr int BAR = STAGES * STAGE + RAWS * RAW, SMEM = BAR + W8_BAR, CHAIN = W8_CHAIN / ROWS;
    static constexpr int COLUMNS = (P > 1 ? 2 : 1) * BN;                       // of tensor memory: the upper parts' sums, then the others'
    // where unit c (of eight columns) of row r lies in a part
    static __device__ __forceinline__ uint32_t at(int r, int c) { return (uint32_t)((c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }
    // MN-major, 128-byte swizzle: 64-column blocks HALF apart (leading), groups of eight rows 1024 bytes apart (stride)
    static __device__ __forceinline__ uint64_t desc(uint32_t smem) {
        return (uint64_t)((smem >> 4) & 0x3fffu) | ((uint64_t)(HALF >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
    }
    static_assert(SMEM <= 227 * 1024 && 8 * (2 * STAGES + 2) <= 96 && 128 + 8 * 2 * RAWS <= W8_BAR && RAW % 16 == 0, "shared memory budget");
};

struct W8Params {
    const void* dy; const int8_t* codes; const uint8_t* steps;
    float *partial, *colpart;           // [split][tile][BN / 4][128][4], [split][row of tiles][128]
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
// D[tmem] (+)= A B: M = 128, N = BN, K = 16, bf16 both, both MN-major, fp32 accumulators
template <int BN> __device__ __forceinline__ void w8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
    constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(W8_T >> 4) << 24);
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// a run of memory to shared memory, counted by an mbarrier; 16-byte boundaries and sizes
__device__ __forceinline__ void w8_bulk(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

template <class T, int MODE, int BN> __global__ void __launch_bounds__(W8<T, BN, MODE>::THREADS, 1) weight_gradient8_kernel(const W8Params p) {
    using W = W8<T, BN, MODE>;
    constexpr int P = W::P, STAGES = W::STAGES, STAGE = W::STAGE, PIECES = W::PIECES, DU = W::DU, XU = W::XU, RAWS = W::RAWS, ROWS = W::ROWS, HALF = W::HALF, PART = W::PART;
    extern __shared__ __align__(1024) uint8_t smem[];
    pdl_launch_next();                                      // (the second kernel waits for the end of this one)
    const uint32_t base = smem_u32(smem), bars = base + W::BAR;
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicCAS(&g_w8_status, 0, 130);
        return;
    }
    auto st_full = [&](uint32_t s) { return bars + 8u * s; };
    auto st_empty = [&](uint32_t s) { return bars + 8u * (STAGES + s); };
    const uint32_t acc_full = bars + 8u * (2 * STAGES), acc_empty = acc_full + 8u;
    auto raw_full = [&](uint32_t s) { return bars + 128u + 8u * s; };
    auto raw_empty = [&](uint32_t s) { return bars + 128u + 8u * (RAWS + s); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + W::BAR + 96);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + W::BAR + 104);
    const int tid = threadIdx.x, warp = (int)tc_uniform(tid >> 5), lane = tid & 31;
    const int tile = blockIdx.y, n0 = tile / p.kt * W8_T, k0 = tile % p.kt * BN;
    const int64_t blocks = (p.rows + ROWS - 1) / ROWS, first = blocks * blockIdx.x / p.splits;
    const int mine = (int)(blocks * (blockIdx.x + 1) / p.splits - first);
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(st_full(s), W8_LOADERS / 32); mbar_init(st_empty(s), 1); }
        mbar_init(acc_full, 1); mbar_init(acc_empty, 128);
        if constexpr (MODE == W8_WHOLE)
            for (int s = 0; s < RAWS; ++s) { mbar_init(raw_full(s), 1); mbar_init(raw_empty(s), W8_LOADERS / 32); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(W::COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tc_uniform(*tmem_slot);
    float2 sums[4] = {};                                    // of this thread's columns of dy

    if (warp < 16) {
        // ------------------------------------------ load and convert ------------------------------------------
        uint32_t s = 0, ph = 1;
        auto stored = [&] {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(st_full(s));
            if (++s == STAGES) { s = 0; ph ^= 1u; }
        };
        if constexpr (MODE != W8_ANY) {
            // dy: unit c of rows r, r + 32; fp32: columns 4 c .. + 3 and 64 + 4 c .. + 3, so that the lanes' 16-byte accesses are next to each
            // other.  x: unit kc of rows kr, kr + KSTEP.
            constexpr int KSTEP = ROWS / XU;
            const int c = tid & 15, r = tid >> 4, kc = BN == 256 ? tid & 31 : c, kr = BN == 256 ? tid >> 5 : r;
            const int nc = n0 + c * (16 / (int)sizeof(T));
            const bool n_in = nc < p.N, n2_in = PIECES == 2 && nc + 64 < p.N, k_in = k0 + kc * 8 < p.K;
            const int64_t end = (first + mine) * ROWS < p.rows ? (first + mine) * ROWS : p.rows;
            // rows left at the thread's first row of a block
            int dy_left = (int)(end - first * ROWS) - r, x_left = (int)(end - first * ROWS) - kr;
            auto put_dy = [&](uint8_t* stage, int u, const uint4 (&piece)[PIECES]) {
                float2 b[4];
                if constexpr (PIECES == 2) {
                    float2 h[2];
                    unpack_pairs(piece[0], h, 0.0f);
                    b[0] = h[0]; b[1] = h[1];
                    unpack_pairs(piece[PIECES - 1], h, 0.0f);
                    b[2] = h[0]; b[3] = h[1];
                } else {
                    unpack_pairs(piece[0], b, T{});
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) sums[j] = add2(sums[j], b[j]);
                const uint32_t to = PIECES == 2 ? W::at(r + 32 * u, c >> 1) + (c & 1) * 8 : W::at(r + 32 * u, c);
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    if constexpr (PIECES == 2) {
                        *reinterpret_cast<uint2*>(stage + q * PART + to) = make_uint2(w8_upper(b[0]), w8_upper(b[1]));
                        *reinterpret_cast<uint2*>(stage + q * PART + HALF + to) = make_uint2(w8_upper(b[2]), w8_upper(b[3]));
                    } else {
                        *reinterpret_cast<uint4*>(stage + q * PART + to) = w8_upper(b);
                    }
                    if (q + 1 < P) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) b[j] = w8_rest(b[j]);
                    }
                }
            };
            auto put_x = [&](uint8_t* stage, int u, uint2 q, uint32_t e) {
                const uint32_t w[2] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u};
                const float2 scale = pair(q8_step(e));
                float2 y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t v = w[j >> 1];
                    const float2 code = make_float2(__uint_as_float(__byte_perm(v, 0x4b000000u, 0x7540 + 2 * (j & 1))), __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7541 + 2 * (j & 1))));
                    y[j] = mul2(add2(code, pair(-8388736.0f)), scale);
                }
                *reinterpret_cast<uint4*>(stage + P * PART + W::at(kr + KSTEP * u, kc)) = pack_pairs(y, __nv_bfloat16{});
            };
            if constexpr (MODE == W8_WHOLE) {
                // what warp 20 has copied
                const uint32_t dy_row = (uint32_t)p.N * (uint32_t)sizeof(T), dy_at = r * dy_row + nc * (uint32_t)sizeof(T), x_at = (uint32_t)(kr * p.K + kc * 8), x_step = (uint32_t)(KSTEP * p.K);
                uint32_t slot = 0, slot_ph = 0;
                for (int k = 0; k < mine; ++k) {
                    const bool there = mbar_wait(raw_full(slot), slot_ph, abort_flag, 135, &g_w8_status) && mbar_wait(st_empty(s), ph, abort_flag, 131, &g_w8_status);
                    if (!__all_sync(0xffffffffu, there)) break;
                    uint8_t* stage = smem + s * STAGE;
                    const uint8_t* from = smem + STAGES * STAGE + slot * W::RAW;
#pragma unroll
                    for (int u = 0; u < DU; ++u) {
                        uint4 piece[PIECES];
                        const uint8_t* at = from + dy_at + 32u * u * dy_row;
                        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                        piece[0] = n_in && 32 * u < dy_left ? *reinterpret_cast<const uint4*>(at) : zero;
                        if constexpr (PIECES == 2) piece[1] = n2_in && 32 * u < dy_left ? *reinterpret_cast<const uint4*>(at + 256) : zero;
                        put_dy(stage, u, piece);
                    }
#pragma unroll
                    for (int u = 0; u < XU; ++u) {
                        const bool in = k_in && KSTEP * u < x_left;
                        const uint32_t at = x_at + u * x_step;
                        put_x(stage, u, in ? *reinterpret_cast<const uint2*>(from + W::RAW_CODES + at) : make_uint2(0u, 0u), in ? from[W::RAW_STEPS + at / Q8_BLOCK] : 1u);
                    }
                    dy_left -= ROWS; x_left -= ROWS;
                    stored();
                    if (lane == 0) mbar_arrive(raw_empty(slot));
                    if (++slot == RAWS) { slot = 0; slot_ph ^= 1u; }
                }
            } else {
                // Each thread copies what it will convert, RAWS blocks ahead, and only waits for itself.  (A copy of no bytes touches no address.)
                uint8_t* raw = smem + STAGES * STAGE + tid * 16;
                uint8_t* raw_codes = smem + STAGES * STAGE + DU * PIECES * (W8_LOADERS * 16) + tid * 8;
                const int64_t dy_row = (int64_t)p.N * (int)sizeof(T), x_step = (int64_t)KSTEP * p.K;
                const uint8_t* dy_at = (const uint8_t*)p.dy + (first * ROWS + r) * dy_row + (int64_t)nc * (int)sizeof(T);
                int64_t at = (first * ROWS + kr) * p.K + k0 + kc * 8;        // value of x
                uint32_t e[RAWS][XU];                       // the steps are loaded with the copies and held until their block's turn
                auto copy = [&](int slot) {
#pragma unroll
                    for (int u = 0; u < DU; ++u) {
                        const bool in = 32 * u < dy_left;
                        uint8_t* to = raw + slot * W::RAW + u * PIECES * (W8_LOADERS * 16);
                        const uint8_t* from = dy_at + 32 * u * dy_row;
                        cp_async_zfill<16>(to, from, in && n_in);
                        if constexpr (PIECES == 2) cp_async_zfill<16>(to + W8_LOADERS * 16, from + 256, in && n2_in);
                    }
#pragma unroll
                    for (int u = 0; u < XU; ++u) {
                        const bool there = k_in && KSTEP * u < x_left;
                        const int64_t from = at + u * x_step;
                        cp_async_zfill<8>(raw_codes + slot * W::RAW + u * (W8_LOADERS * 8), p.codes + from, there);
                        e[slot][u] = there ? __ldg(p.steps + (from >> 5)) : 1u;
                    }
                    cp_async_commit();
                    dy_left -= ROWS; x_left -= ROWS; dy_at += ROWS * dy_row; at += XU * x_step;
                };
                if (mine > 0) {
#pragma unroll
                    for (int k = 0; k < RAWS; ++k) copy(k);
                }
                auto step = [&](int slot) {
                    cp_async_wait<RAWS - 1>();
                    if (!__all_sync(0xffffffffu, mbar_wait(st_empty(s), ph, abort_flag, 131, &g_w8_status))) return false;
                    uint8_t* stage = smem + s * STAGE;
#pragma unroll
                    for (int u = 0; u < DU; ++u) {
                        uint4 piece[PIECES];
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) piece[i] = *reinterpret_cast<const uint4*>(raw + slot * W::RAW + (u * PIECES + i) * (W8_LOADERS * 16));
                        put_dy(stage, u, piece);
                    }
#pragma unroll
                    for (int u = 0; u < XU; ++u)
                        put_x(stage, u, *reinterpret_cast<const uint2*>(raw_codes + slot * W::RAW + u * (W8_LOADERS * 8)), e[slot][u]);
                    copy(slot);
                    stored();
                    return true;
                };
                bool alive = true;
                for (int k = 0; k < mine && alive; k += RAWS) {
#pragma unroll
                    for (int j = 0; j < RAWS; ++j)
                        if (alive && k + j < mine) alive = step(j);
                }
                cp_async_wait_all();
            }
        } else {
            // Any widths: columns 2 lane, 2 lane + 1 (+ 64, ...) of rows warp, warp + 16, ...  Every load has an address inside its array and is
            // zeroed afterwards where it lies outside the tile, so that no branch keeps the loads apart.
            constexpr int NJ = 4, KJ = BN / 32;
            for (int part = 0; part < mine * (ROWS / 32); ++part) {
                const int k = part / (ROWS / 32), r0 = warp + part % (ROWS / 32) * 32;       // two rows of 32 at a time
                float d[2][NJ];
                uint32_t codes[2][KJ], size[2][KJ];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int64_t r = (first + k) * ROWS + r0 + 16 * i;
                    const bool in = r < p.rows;
                    const int64_t row = in ? r : 0, at = row * p.K + k0;
                    const T* dy = (const T*)p.dy + row * p.N + n0;
                    const int8_t* code = p.codes + at;
                    const uint8_t* step = p.steps + (at >> 5);
                    const int phase = (int)(at & 31), n_left = in ? p.N - n0 : 0, k_left = in ? p.K - k0 : 0;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        const int col = 2 * lane + (j >> 1) * 64 + (j & 1);
                        d[i][j] = to_f32(__ldg(dy + (col < n_left ? col : 0)));
                        if (col >= n_left) d[i][j] = 0.0f;
                    }
#pragma unroll
                    for (int j = 0; j < KJ; ++j) {
                        const int col = 2 * lane + (j >> 1) * 64 + (j & 1), from = col < k_left ? col : 0;
                        codes[i][j] = (uint32_t)(int)__ldg(code + from);
                        size[i][j] = __ldg(step + ((phase + from) >> 5));
                        if (col >= k_left) { codes[i][j] = 0; size[i][j] = 1; }
                    }
                }
                if (r0 < 32 && !__all_sync(0xffffffffu, mbar_wait(st_empty(s), ph, abort_flag, 131, &g_w8_status))) break;
                uint8_t* stage = smem + s * STAGE;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = r0 + 16 * i;
                    const uint32_t to = W::at(r, lane >> 2) + (lane & 3) * 4;
#pragma unroll
                    for (int h = 0; h < NJ / 2; ++h) {      // 64 columns each
                        float2 b = make_float2(d[i][2 * h], d[i][2 * h + 1]);
                        sums[h] = add2(sums[h], b);
#pragma unroll
                        for (int q = 0; q < P; ++q, b = w8_rest(b)) *reinterpret_cast<uint32_t*>(stage + q * PART + h * HALF + to) = w8_upper(b);
                    }
#pragma unroll
                    for (int h = 0; h < KJ / 2; ++h)
                        *reinterpret_cast<uint32_t*>(stage + P * PART + h * HALF + to) = pack_pair(
                            make_float2((float)(int)codes[i][2 * h] * q8_step(size[i][2 * h]), (float)(int)codes[i][2 * h + 1] * q8_step(size[i][2 * h + 1])), __nv_bfloat16{});
                }
                if (r0 + 32 >= ROWS) stored();
            }
        }
    } else if (MODE == W8_WHOLE && warp == 20) {
        // ------------------------------------------ copy (W8_WHOLE) ------------------------------------------
        const uint32_t dy_row = (uint32_t)p.N * (uint32_t)sizeof(T);
        uint32_t slot = 0, ph = 1;
        int k = 0;
        for (; k < mine; ++k) {
            if (!__all_sync(0xffffffffu, mbar_wait(raw_empty(slot), ph, abort_flag, 136, &g_w8_status))) break;
            const int64_t row = (first + k) * ROWS;
            const uint32_t n = (uint32_t)(p.rows - row < ROWS ? p.rows - row : ROWS), codes = n * (uint32_t)p.K;
            const uint32_t steps = (codes + Q8_BLOCK - 1) / Q8_BLOCK, most = steps & ~15u;       // the last block's may end off a boundary
            const uint32_t to = (uint32_t)(STAGES * STAGE) + slot * (uint32_t)W::RAW;
            const uint8_t* from = p.steps + row * p.K / Q8_BLOCK;
            if (most + lane < steps) smem[to + W::RAW_STEPS + most + lane] = from[most + lane];
            __syncwarp();
            if (lane == 0) {
                const uint32_t bar = raw_full(slot);
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n * dy_row + codes + most) : "memory");
                w8_bulk(base + to, (const T*)p.dy + row * p.N, n * dy_row, bar);
                w8_bulk(base + to + W::RAW_CODES, p.codes + row * p.K, codes, bar);
                if (most > 0) w8_bulk(base + to + W::RAW_STEPS, from, most, bar);
            }
            if (++slot == RAWS) { slot = 0; ph ^= 1u; }
        }
        // nothing is in flight when the block ends, come what may
        volatile int none = 0;
        for (int i = k > RAWS ? k - RAWS : 0; i < k; ++i) mbar_wait(raw_full(i % RAWS), (uint32_t)(i / RAWS) & 1u, &none, 136);
    } else {
        // ------------------------------------------ MMAs and results ------------------------------------------
        const int chains = mine > 0 ? (mine + W::CHAIN - 1) / W::CHAIN : 0;
        uint32_t s = 0, ph = 0;
        float* out = p.partial + (((int64_t)blockIdx.x * gridDim.y + tile) * (BN / 4) * W8_T + (warp - 16) * 32 + lane) * 4;
        const uint32_t row = tmem_base + ((uint32_t)((warp - 16) * 32) << 16);
        // one thread: the MMAs of a chain's blocks of rows
        auto issue = [&](int chain) {
            if (!mbar_wait(acc_empty, (uint32_t)(chain & 1) ^ 1u, abort_flag, 132, &g_w8_status)) return;
            tc_fence_after();
            const int n = mine - chain * W::CHAIN < W::CHAIN ? mine - chain * W::CHAIN : W::CHAIN;
            for (int k = 0; k < n; ++k) {
                if (!mbar_wait(st_full(s), ph, abort_flag, 133, &g_w8_status)) return;
                tc_fence_after();
                const uint32_t st = base + s * STAGE;
                const uint64_t a = W::desc(st), b = W::desc(st + P * PART);
#pragma unroll
                for (int part = P - 1; part >= 0; --part)   // the smallest parts first
#pragma unroll
                    for (int k16 = 0; k16 < ROWS / 16; ++k16)
                        w8_mma<BN>(tmem_base + (part ? BN : 0), a + part * (PART >> 4) + k16 * 128, b + k16 * 128,
                                   k > 0 || k16 > 0 || (part > 0 && part < P - 1) ? 1u : 0u);
                tc_commit(st_empty(s));
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
            tc_commit(acc_full);
        };
        bool alive = true;
        for (int k = 0; k < chains && alive; ++k) {
            if (warp == 16) {
                if (tc_elect()) issue(k);
                __syncwarp();
            }
            if (!mbar_wait(acc_full, (uint32_t)(k & 1), abort_flag, 134, &g_w8_status)) { alive = false; break; }
            tc_fence_after();
#pragma unroll 2
            for (int j = 0; j < BN; j += 16) {
                float v[16];
                if constexpr (P > 1) tc_ld16_sum(row + j, BN, v);
                else tc_ld16(row + j, v);
                float4* to = reinterpret_cast<float4*>(out + j * W8_T);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 u = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    if (k > 0) { const float4 w = to[i * W8_T]; u.x += w.x; u.y += w.y; u.z += w.z; u.w += w.w; }
                    to[i * W8_T] = u;
                }
            }
            tc_fence_before();
            mbar_arrive(acc_empty);
        }
        if (chains == 0)                                    // no rows
            for (int j = 0; j < BN; j += 4) *reinterpret_cast<float4*>(out + j * W8_T) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(W::COLUMNS) : "memory");
    }
    // column sums of dy, of several threads each; the stages are free
    if (k0 == 0 && p.db) {
        float* part = reinterpret_cast<float*>(smem);
        constexpr int SHARES = MODE != W8_ANY ? 32 : 16;
        if (warp < 16) {
            if constexpr (MODE != W8_ANY) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    part[(tid >> 4) * W8_T + (PIECES == 2 ? (tid & 15) * 4 + (j >> 2) * 64 + (j & 3) : (tid & 15) * 8 + j)] = j & 1 ? sums[j / 2].y : sums[j / 2].x;
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

// dw and db from the splits' results.  W8_SHARES threads share a result (four columns of a row, or a column sum): thread g adds results g,
// g + W8_SHARES, ..., and their sums are added in order.  (16 threads with ten loads at a time: one round for 148 splits; 8 threads with
// eight took 1.5 us more.)
constexpr int W8_SHARES = 16;
template <int BN> __global__ void __launch_bounds__(32 * W8_SHARES) weight_gradient8_reduce_kernel(const W8Params p, int tiles) {
    __shared__ float4 part[W8_SHARES][32];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c_blocks = tiles * (W8_T * BN / 4 / 32);
    pdl_launch_next();
    pdl_wait();
    if ((int)blockIdx.x < c_blocks) {
        const int i = blockIdx.x * 32 + lane;               // of the padded [tiles][BN / 4][128]
        const int r = i % W8_T, c4 = i / W8_T % (BN / 4), tile = i / (W8_T * BN / 4);
        const int row = tile / p.kt * W8_T + r, col = tile % p.kt * BN + c4 * 4;
        const bool in = row < p.N && col < p.K;
        const float4* src = reinterpret_cast<const float4*>(p.partial) + i;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in)
#pragma unroll 10
            for (int k = g; k < p.splits; k += W8_SHARES) {
                const float4 v = __ldcg(src + (int64_t)k * tiles * (W8_T * BN / 4));
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
        part[g][lane] = s;
        __syncthreads();
        if (g || !in) return;
#pragma unroll
        for (int k = 1; k < W8_SHARES; ++k) { const float4 v = part[k][lane]; s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; }
        const float o[4] = {s.x, s.y, s.z, s.w};
        float* dst = p.dw + (int64_t)row * p.K + col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.K) dst[e] = o[e];
    } else {
        const int c = (blockIdx.x - c_blocks) * 32 + lane;  // (whole tiles of columns)
        float s = 0.0f;
#pragma unroll 10
        for (int k = g; k < p.splits; k += W8_SHARES) s += __ldcg(p.colpart + (int64_t)k * (tiles / p.kt) * W8_T + c);
        part[g][lane].x = s;
        __syncthreads();
        if (g || c >= p.N) return;
#pragma unroll
        for (int k = 1; k < W8_SHARES; ++k) s += part[k][lane].x;
        p.db[c] = s;
    }
}

// Tiles of 128 columns of x where that is all there are, of 256 otherwise: a tile of 128 leaves room for blocks of 64 rows, half as many
// rounds of the pipeline (179776 rows, dy 256 columns, x 128, fp32: 66 us against 77 with blocks of 32), and one of 256 converts dy once
// for all of x (dy 128 columns, x 256: 55 us against 61 as two tiles of 128).
static inline int w8_width(int K) { return K <= W8_T ? W8_T : 2 * W8_T; }
// Blocks that share the rows: one wave over the SMs, at least 128 rows each
static int w8_splits(int N, int K, int64_t rows) {
    const int tiles = ceil_div(N, W8_T) * ceil_div(K, w8_width(K)), most = num_sms() / tiles < 1 ? 1 : num_sms() / tiles;
    const int64_t want = ceil_div<int64_t>(rows, 128);
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

int w8_status(bool reset) {
    int v = 0;
    if (reset) return cudaMemcpyToSymbol(g_w8_status, &v, sizeof(int)) == cudaSuccess ? SPGT_OK : SPGT_ERR_LAUNCH;
    return cudaMemcpyFromSymbol(&v, g_w8_status, sizeof(int)) == cudaSuccess ? v : SPGT_ERR_LAUNCH;
}

template <class T, int MODE, int BN> static int w8_launch(const W8Params& p, int tiles, cudaStream_t st) {
    using W = W8<T, BN, MODE>;
    static SmemOptIn configured;
    if (int e = smem_opt_in(weight_gradient8_kernel<T, MODE, BN>, W::SMEM, configured)) return e;
    ChainScope chain;
    if (int e = launch_chained(weight_gradient8_kernel<T, MODE, BN>, dim3((unsigned)p.splits, (unsigned)tiles), W::THREADS, W::SMEM, st, p)) return e;
    return launch_chained(weight_gradient8_reduce_kernel<BN>, dim3((unsigned)(tiles * (W8_T * BN / 4 / 32) + (p.db ? tiles / p.kt * (W8_T / 32) : 0))), 32 * W8_SHARES, 0, st, p, tiles);
}
template <class T, int BN> static int w8_launch(const W8Params& p, int tiles, cudaStream_t st) {
    if (p.N % 8 || p.K % 8) return w8_launch<T, W8_ANY, BN>(p, tiles, st);
    return tiles == 1 && p.K % 16 == 0 && aligned16(p.steps) ? w8_launch<T, W8_WHOLE, BN>(p, tiles, st) : w8_launch<T, W8_VEC, BN>(p, tiles, st);
}

}  // namespace spgt

using namespace spgt;

extern "C" size_t spgt_weight_gradient8_workspace_bytes(int N, int K, int64_t rows) {
    if (N <= 0 || K <= 0 || rows < 0 || N > 4096 || K > 4096 || rows > ((int64_t)1 << 36)) return 0;
    const size_t tiles = (size_t)ceil_div(N, W8_T) * ceil_div(K, w8_width(K));
    return (size_t)w8_splits(N, K, rows) * (tiles * w8_width(K) + ceil_div(N, W8_T)) * W8_T * sizeof(float);
}

extern "C" int spgt_weight_gradient8(const void* dy, int dtype, const int8_t* codes, const uint8_t* steps, float* dw, float* db, int N, int K,
                                     int64_t rows, void* workspace, size_t workspace_bytes, spgt_stream_t stream) {
    const size_t need = spgt_weight_gradient8_workspace_bytes(N, K, rows);
    if (need == 0 || dtype < SPGT_F32 || dtype > SPGT_F16) return SPGT_ERR_SHAPE;
    if (!dw || !workspace || (rows > 0 && (!dy || !codes || !steps))) return SPGT_ERR_NULL;
    if (workspace_bytes < need) return SPGT_ERR_WORKSPACE;
    if (!aligned16(dy) || !aligned16(codes) || !aligned16(workspace)) return SPGT_ERR_ALIGN;
    const int width = w8_width(K), kt = ceil_div(K, width), tiles = ceil_div(N, W8_T) * kt;
    W8Params p{dy, codes, steps, (float*)workspace, nullptr, dw, db, N, K, kt, w8_splits(N, K, rows), rows};
    p.colpart = p.partial + (size_t)p.splits * tiles * W8_T * width;
    return with_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        return width == W8_T ? w8_launch<T, W8_T>(p, tiles, (cudaStream_t)stream) : w8_launch<T, 2 * W8_T>(p, tiles, (cudaStream_t)stream);
    });
}

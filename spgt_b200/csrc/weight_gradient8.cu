// dW [N, K] = dy^T x  for dy [rows, N] and an 8-bit checkpoint of x [rows, K] (lowp.cuh), with the column sums of dy: weight and bias
// gradient of a dense layer that kept its input in 8 bits.  Blocks split the rows; their partial results are added in a fixed order.
#include "lowp.cuh"

namespace spgt {

constexpr int W8_T = 64, W8_ROWS = 16, W8_THREADS = 256;

struct W8Params {
    const void* dy; const int8_t* codes; const uint8_t* steps;
    float *partial, *colpart;           // [split][N][K], [split][N]
    float *dw, *db;
    int N, K, splits;
    int64_t rows;
};

template <class T> __global__ void __launch_bounds__(W8_THREADS) weight_gradient8_kernel(const W8Params p) {
    __shared__ float a[W8_ROWS][W8_T + 4], x[W8_ROWS][W8_T + 4];
    const int kt = ceil_div(p.K, W8_T), n0 = blockIdx.y / kt * W8_T, k0 = blockIdx.y % kt * W8_T;
    const int64_t r0 = p.rows * blockIdx.x / p.splits, r1 = p.rows * (blockIdx.x + 1) / p.splits;
    const int ty = threadIdx.x / 16 * 4, tx = threadIdx.x % 16 * 4;
    float acc[4][4] = {}, col = 0.0f;
    for (int64_t r = r0; r < r1; r += W8_ROWS) {
        __syncthreads();
        for (int i = threadIdx.x; i < W8_ROWS * W8_T; i += W8_THREADS) {
            const int rr = i / W8_T, c = i % W8_T;
            const bool in = r + rr < r1;
            const int64_t at = (r + rr) * p.K + k0 + c;
            a[rr][c] = in && n0 + c < p.N ? to_f32(((const T*)p.dy)[(r + rr) * p.N + n0 + c]) : 0.0f;
            x[rr][c] = in && k0 + c < p.K ? (float)p.codes[at] * q8_step(p.steps[at >> 5]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int rr = 0; rr < W8_ROWS; ++rr) {
            if (k0 == 0 && threadIdx.x < W8_T) col += a[rr][threadIdx.x];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[rr][ty + i], x[rr][tx + j], acc[i][j]);
        }
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
            if (n0 + ty + i < p.N && k0 + tx + j < p.K) p.partial[((int64_t)blockIdx.x * p.N + n0 + ty + i) * p.K + k0 + tx + j] = acc[i][j];
    if (k0 == 0 && threadIdx.x < W8_T && n0 + threadIdx.x < p.N) p.colpart[(int64_t)blockIdx.x * p.N + n0 + threadIdx.x] = col;
}

__global__ void __launch_bounds__(256) weight_gradient8_reduce_kernel(const W8Params p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, nk = (int64_t)p.N * p.K;
    if (i >= nk + p.N) return;
    const float* src = i < nk ? p.partial + i : p.colpart + (i - nk);
    const int64_t step = i < nk ? nk : p.N;
    float s = 0.0f;
#pragma unroll 4
    for (int k = 0; k < p.splits; ++k) s += src[k * step];
    if (i < nk) p.dw[i] = s;
    else if (p.db) p.db[i - nk] = s;
}

static int w8_splits(int N, int K, int64_t rows) {
    const int64_t tiles = (int64_t)ceil_div(N, W8_T) * ceil_div(K, W8_T), most = ceil_div<int64_t>(4 * num_sms(), tiles), want = ceil_div<int64_t>(rows, 128);
    return (int)(want < most ? want : most);
}

}  // namespace spgt

using namespace spgt;

extern "C" size_t spgt_weight_gradient8_workspace_bytes(int N, int K, int64_t rows) {
    if (N <= 0 || K <= 0 || rows < 0 || N > 16384 || K > 16384) return 0;
    return (size_t)w8_splits(N, K, rows) * ((size_t)N * K + N) * sizeof(float) + 16;
}

extern "C" int spgt_weight_gradient8(const void* dy, int dtype, const int8_t* codes, const uint8_t* steps, float* dw, float* db, int N, int K,
                                     int64_t rows, void* workspace, size_t workspace_bytes, spgt_stream_t stream) {
    const size_t need = spgt_weight_gradient8_workspace_bytes(N, K, rows);
    if (need == 0 || dtype < SPGT_F32 || dtype > SPGT_F16) return SPGT_ERR_SHAPE;
    if (!dw || !workspace || (rows > 0 && (!dy || !codes || !steps))) return SPGT_ERR_NULL;
    if (workspace_bytes < need) return SPGT_ERR_WORKSPACE;
    if (!aligned16(dy) || !aligned16(codes) || !aligned16(workspace)) return SPGT_ERR_ALIGN;
    W8Params p{dy, codes, steps, (float*)workspace, nullptr, dw, db, N, K, w8_splits(N, K, rows), rows};
    p.colpart = p.partial + (size_t)p.splits * N * K;
    if (rows > 0) {
        const int e = with_type(dtype, [&](auto zero) {
            using T = decltype(zero);
            weight_gradient8_kernel<T><<<dim3((unsigned)p.splits, (unsigned)(ceil_div(N, W8_T) * ceil_div(K, W8_T))), W8_THREADS, 0, (cudaStream_t)stream>>>(p);
            return launch_status();
        });
        if (e) return e;
    }
    weight_gradient8_reduce_kernel<<<(unsigned)ceil_div<int64_t>((int64_t)N * K + N, 256), 256, 0, (cudaStream_t)stream>>>(p);
    return launch_status();
}

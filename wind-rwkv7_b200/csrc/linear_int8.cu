// Products in 8 bits of a few rows (generation):  y = act((x w^T) xs ws + bias) + residual,  x [M, K], w [N, K] signed 8-bit.
// Bound by the weight's stream.  A CTA has 16 rows of the weight and all of k, shared out over its warps, one to sixteen: within 64 k a lane has 16 adjacent bytes of two weight
// rows and of each x row, and sums their products, four an instruction.  All requests of a step are under way together.  The sums, 32-bit integers, are joined over the
// lanes that share a weight row and through shared memory over the warps.  Figures, against the tensor-memory form of linear.cu, at int8_rows_fit().
// (With mma.sync m16n8k32 for the products 16 x 2048 -> 50001 took 81 us instead of 22: some 200 cycles an instruction.)
#include "activations.cuh"
#include "mma_bf16.cuh"
#include "wkv7_kernels.h"
#include <type_traits>

namespace wkv7 {
namespace lin {

constexpr int ROWS_WARPS = 16, ROWS_N = 16, ROWS_CHUNK = 64, ROWS_MOST = 2;  // warps of a CTA at most

struct RowsParams {
    const signed char *x, *w;
    LinearEpilogue e;  // xs, ws, bias, residual, y
    long long ldx, ldw;
    int K;
};
// the bytes k .. k + 15 of a row, zeros from `K` on
__device__ __forceinline__ uint4 tail16(const signed char* row, int k, int K) {
    if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < K) w[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float act_of(int a, float x) {
    switch (a) {
        case kActRelu: return act<kActRelu>(x);
        case kActRelu2: return act<kActRelu2>(x);
        case kActTanh: return act<kActTanh>(x);
        case kActSigmoid: return act<kActSigmoid>(x);
        case kActSilu: return act<kActSilu>(x);
        case kActGelu: return act<kActGelu>(x);
        default: return x;
    }
}

// MT: x rows.  STEP: chunks of 64 k that a warp requests at a time
template <int MT, int STEP> __global__ void __launch_bounds__(32 * ROWS_WARPS) int8_rows_kernel(const __grid_constant__ RowsParams p) {
    __shared__ int sums[ROWS_WARPS][MT][ROWS_N];
    const int tid = threadIdx.x, warps = blockDim.x >> 5, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const long long n0 = (long long)blockIdx.x * ROWS_N;
    const int chunks = p.K / ROWS_CHUNK;
    // rows behind the last are the last again, and not stored
    const signed char *w[2], *x[MT];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long long r = n0 + g + 8 * i;
        w[i] = p.w + (r < p.e.cols ? r : p.e.cols - 1) * p.ldw + 16 * t;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = p.x + (i < p.e.rows ? i : p.e.rows - 1) * p.ldx + 16 * t;
    int acc[2][MT] = {};
    stream_order();
    auto products = [&](const uint4& a, const uint4& b, int& s) { s = __dp4a((int)a.x, (int)b.x, __dp4a((int)a.y, (int)b.y, __dp4a((int)a.z, (int)b.z, __dp4a((int)a.w, (int)b.w, s)))); };
    auto step = [&](int c, auto count) {
        constexpr int S = decltype(count)::value;
        uint4 a[S][2], b[S][MT];
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) a[s][i] = __ldcs(reinterpret_cast<const uint4*>(w[i] + (long long)(c + warps * s) * ROWS_CHUNK));
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < MT; ++i) b[s][i] = *reinterpret_cast<const uint4*>(x[i] + (c + warps * s) * ROWS_CHUNK);
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m) products(a[s][i], b[s][m], acc[i][m]);
    };
    int c = warp;
#pragma unroll 1
    for (; c + warps * (STEP - 1) < chunks; c += warps * STEP) step(c, std::integral_constant<int, STEP>{});
#pragma unroll 1
    for (; c < chunks; c += warps) step(c, std::integral_constant<int, 1>{});
    if (p.K % ROWS_CHUNK && warp == warps - 1) {  // what is left of k
        const int k = chunks * ROWS_CHUNK + 16 * t;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint4 b = tail16(x[m] - 16 * t, k, p.K);
#pragma unroll
            for (int i = 0; i < 2; ++i) products(tail16(w[i] - 16 * t, k, p.K), b, acc[i][m]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            int s = acc[i][m];
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            if (t == 0) sums[warp][m][g + 8 * i] = s;
        }
    __syncthreads();
    const LinearEpilogue& e = p.e;
    const int m = tid / ROWS_N, i = tid % ROWS_N;
    const long long col = n0 + i;
    if (m >= e.rows || m >= MT || col >= e.cols) return;
    int s = 0;
    for (int r = 0; r < warps; ++r) s += sums[r][m][i];
    float v = __fmul_rn(__fmul_rn((float)s, e.ws[col]), e.xs[m]);  // (in this order in the other kernels, too)
    if (e.bias) v += e.bias_f32 ? ((const float*)e.bias)[col] : __bfloat162float(((const bf16*)e.bias)[col]);
    v = act_of(e.act, v);
    const long long at = m * e.ldy + col;
    if (e.residual) v += e.y_f32 ? ((const float*)e.residual)[m * e.ldr + col] : __bfloat162float(((const bf16*)e.residual)[m * e.ldr + col]);
    if (e.y_f32) ((float*)e.y)[at] = v;
    else ((bf16*)e.y)[at] = __float2bfloat16_rn(v);
}

}  // namespace lin

// us, in a graph, against the tensor-memory form: 1 x 2048 -> 8192 5.2 / 7.4 (the weight's stream alone 2.6), 1 x 8192 -> 2048 6.6 / 6.9, 1 x 768 -> 768 2.0 / 3.5.  About the cut, one row and two:
// 4096 -> 8192 8.9 / 10.0 and 10.2 / 10.1, 8192 -> 4096 8.7 / 10.2 and 9.9 / 10.3; 8192 -> 8192 15.2 / 15.5 and 17.6 / 15.6, 4096 -> 14336 14.9 / 14.3 and 17.3 / 14.4, 2048 -> 50001 22.2 / 20.4 and
// 25.3 / 20.5.  On the other side of it by themselves: 2560 -> 10240 10.3 / 8.9 (40 chunks for eight warps of four), 14336 -> 4096 12.6 / 14.7, 2 x 8192 -> 2048 8.0 / 7.1.  With more rows the products
// of four take longer than the stream: 4 x 4096 -> 4096 8.9 / 7.8
bool int8_rows_fit(long long rows, long long cols, long long k) { return rows <= lin::ROWS_MOST && cols * k <= 1LL << 25; }

int launch_int8_rows(LinearOperand x, LinearOperand w, long long k, const LinearEpilogue& e, cudaStream_t stream) {
    using namespace lin;
    const RowsParams p{(const signed char*)x.p, (const signed char*)w.p, e, x.ld, w.ld, (int)k};
    const auto kern = e.rows == 1 ? int8_rows_kernel<1, 4> : int8_rows_kernel<2, 4>;
    // warps: a step each
    const long long chunks = (k + ROWS_CHUNK - 1) / ROWS_CHUNK;
    int warps = 1;
    while (warps < ROWS_WARPS && warps * 4 < chunks) warps *= 2;
    return launch(kern, dim3((unsigned)((e.cols + ROWS_N - 1) / ROWS_N)), 32 * warps, 0, stream, p) ? kOk : kLaunchFailed;
}

}  // namespace wkv7

// Rows to 8 bits, and dropout by itself.  Both are bound by memory; dropout of bf16 elements as much by its generator's ten rounds.
#include "norm.cuh"

namespace wkv7 {
namespace norm {

// ---- rows to 8 bits --------------------------------------------------------------------------------------------------------
struct QuantizeKernelParams : QuantizeParams {
    Teams t;
    Lie lx, lq;
};
// NV 0: rows of any length, read twice
template <int NV, bool XF, bool EVEN> __global__ void __launch_bounds__(NV ? threads_most(NV) : 1024) quantize_kernel(const __grid_constant__ QuantizeKernelParams p) {
    __shared__ Room room;
    stream_order();
    constexpr int HELD = NV ? NV : 1;
    const int team = p.t.threads, lane = threadIdx.x % team, K = (int)p.K;
    const long long step = (long long)gridDim.x * p.t.rows;
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const int col0 = first_col(row, K) + 8 * lane;
    const int vectors = NV ? NV : (int)((K + 7 + 8LL * team - 1) / (8LL * team));
    Raw<XF> x[HELD];
    auto ask = [&](long long m) {
        if (m >= p.M) return;
#pragma unroll
        for (int v = 0; v < HELD; ++v) request<XF, EVEN>(x[v], p.x, p.lx, m, col0 + 8 * team * v, K);
    };
    if (NV) ask(row);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * p.t.rows; first < p.M; first += step, row += step) {
        const bool in = row < p.M;
        float f[HELD][8], none = 0.f, top = 0.f;
        auto tops = [&](const Raw<XF>& r, int col, float (&to)[8]) {
            floats<XF>(r, to);
            clear_outside<EVEN>(col, K, to);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_abs(top, to[i]);
        };
        if (NV) {
#pragma unroll
            for (int v = 0; v < HELD; ++v) {
                if (in) complete<XF, EVEN>(x[v], p.x, p.lx, row, col0 + 8 * team * v, K);
                tops(x[v], col0 + 8 * team * v, f[v]);
            }
            ask(row + step);
        } else {
#pragma unroll 4
            for (int v = 0; v < vectors; ++v) {
                const long long col = col0 + 8LL * team * v;
                Raw<XF> r{};
                if (in && col < K) {
                    request<XF, EVEN>(r, p.x, p.lx, row, (int)col, K);
                    complete<XF, EVEN>(r, p.x, p.lx, row, (int)col, K);
                }
                tops(r, (int)(col < K ? col : K), f[0]);
            }
        }
        reduce<false, true>(team, room, turn, none, top);
        turn ^= 1;
        if (!in) continue;
        if (lane == 0) p.scale[row] = Rounder::scale(top, 1.f);
        const Rounder round(top);
#pragma unroll
        for (int v = 0; v < vectors; ++v) {
            const long long col = col0 + 8LL * team * v;
            if (col >= K) break;
            if (!NV) {
                request<XF, EVEN>(x[0], p.x, p.lx, row, (int)col, K);
                complete<XF, EVEN>(x[0], p.x, p.lx, row, (int)col, K);
                floats<XF>(x[0], f[0]);
            }
            store_int8<EVEN>(p.q, p.lq, row, (int)col, K, f[NV ? v : 0], round);
        }
    }
}

// ---- dropout alone ---------------------------------------------------------------------------------------------------------
template <bool XF, int RES> __global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
    constexpr bool RF = RES == 2;
    stream_order();
    const Dropper drop(p.d);
    const Lie lie{8, p.n};  // rows of eight
    const long long step = (long long)gridDim.x * 256 * 8;
    for (long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; at < p.n; at += step) {
        const int live = (int)(p.n - at < 8 ? p.n - at : 8);
        Raw<XF> x;
        Raw<RF> r;
        request<XF, false>(x, p.x, lie, at >> 3, 0, live);
        if (RES) request<RF, false>(r, p.residual, lie, at >> 3, 0, live);
        float f[8];
        complete<XF, false>(x, p.x, lie, at >> 3, 0, live);
        floats<XF>(x, f);
        if (p.d.threshold) drop.apply(at >> 3, f);
        if (RES) {
            float g[8];
            complete<RF, false>(r, p.residual, lie, at >> 3, 0, live);
            floats<RF>(r, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __fadd_rn(g[i], f[i]);
        }
        store<false>(p.y, p.y_f32, lie, at >> 3, 0, live, f);
    }
}

}  // namespace norm

int launch_quantize(const QuantizeParams& a, cudaStream_t stream) {
    using namespace norm;
    QuantizeKernelParams p;
    static_cast<QuantizeParams&>(p) = a;
    const long long pieces = pieces_of(p.K);
    const int nv = pieces > 4 * threads_most(4) ? 0 : vectors_of(p.M, pieces);
    p.t = nv ? teams_of(pieces, nv) : Teams{1024, 1};
    p.lx = lie_of(p.x, p.M, p.K, p.ldx, 16);
    p.lq = lie_of(p.q, p.M, p.K, p.ldq, 8);
#define WKV7_TYPES(nv, even) {quantize_kernel<nv, false, even>, quantize_kernel<nv, true, even>}
    static void (*const kernels[4][2][2])(QuantizeKernelParams) = {{WKV7_TYPES(0, false), WKV7_TYPES(0, true)}, {WKV7_TYPES(1, false), WKV7_TYPES(1, true)},
                                                                   {WKV7_TYPES(2, false), WKV7_TYPES(2, true)}, {WKV7_TYPES(4, false), WKV7_TYPES(4, true)}};
#undef WKV7_TYPES
    const bool even = p.K % 8 == 0 && p.lx.end && p.lq.end;
    const unsigned grid = (unsigned)ctas_of(p.M, p.t, sm_count(), nv == 4 ? 544 : 1024);
    return launch(kernels[nv == 4 ? 3 : nv][even][p.x_f32], dim3(grid), p.t.threads * p.t.rows, 0, stream, p) ? kOk : kLaunchFailed;
}

int launch_dropout(const DropoutParams& p, cudaStream_t stream) {
    using namespace norm;
    static void (*const kernels[2][3])(DropoutParams) = {{dropout_kernel<false, 0>, dropout_kernel<false, 1>, dropout_kernel<false, 2>},
                                                         {dropout_kernel<true, 0>, dropout_kernel<true, 1>, dropout_kernel<true, 2>}};
    const long long want = (p.n + 2047) / 2048, most = (long long)sm_count() * 8;
    return launch(kernels[p.x_f32][p.residual ? 1 + p.r_f32 : 0], dim3((unsigned)(want < most ? want : most)), 256, 0, stream, p) ? kOk : kLaunchFailed;
}

}  // namespace wkv7

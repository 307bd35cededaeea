// Rows to 8 bits, and dropout by itself.  Both are bound by memory, dropout of bf16 elements with its generator's ten rounds only partly behind it.
#include "norm.cuh"

namespace wkv7 {
namespace norm {

// ---- rows to 8 bits --------------------------------------------------------------------------------------------------------
struct QuantizeKernelParams : QuantizeParams {
    Teams t;
    Lie at_x, at_q;
};
// A row stays in registers between its maximum and its integers; NV 0: rows of any length, read twice.  Three operations an element besides the maximum.  us: 8192 x 8192 38 (5.3 TB/s),
// 8192 x 2048 11.9, 8192 x 2049 23.5 (its rows in 8 bits are stored byte by byte), 512 x 65536 37.
template <int NV, bool XF, bool EVEN> __global__ void __launch_bounds__(NV ? threads_most(NV) : 1024) quantize_kernel(const __grid_constant__ QuantizeKernelParams p) {
    __shared__ Room room;
    stream_order();
    constexpr int HELD = NV ? NV : 1, XS = XF ? 4 : 2;
    const int team = p.t.threads, lane = threadIdx.x % team, K = (int)p.K;
    const long long step = (long long)gridDim.x * p.t.rows;
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const int col0 = first_col(row, K) + 8 * lane;
    const Byte* x_at = p.at_x.base + (row * p.at_x.ld + col0) * XS;
    Byte* q_at = (Byte*)p.q + row * p.at_q.ld + col0;
    const long long x_step = step * p.at_x.ld * XS, q_step = step * p.at_q.ld;
    const long long vectors = (K + 7 + 8LL * team - 1) / (8LL * team);
    Raw<XF> x[HELD];
    auto ask = [&](bool in) {
        if (!in) return;
#pragma unroll
        for (int v = 0; v < HELD; ++v) request<XF, EVEN>(x[v], x_at + 8 * team * v * XS, p.at_x.end, col0 + 8 * team * v, K);
    };
    if (NV) ask(row < p.M);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * p.t.rows; first < p.M; first += step) {
        const bool in = row < p.M;
        float f[HELD][8], none = 0.f, top = 0.f;
        auto tops = [&](int col, float (&to)[8]) {
            clear_outside<EVEN>(col, K, to);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_abs(top, to[i]);
        };
        // a piece of a long row
        auto get = [&](long long v, float (&to)[8]) {
            const int col = (int)(col0 + 8 * team * v);
            Raw<XF> r{};
            request<XF, EVEN>(r, x_at + 8 * team * v * XS, p.at_x.end, col, K);
            complete<XF, EVEN>(r, x_at + 8 * team * v * XS, p.at_x.end, col, K);
            floats<XF>(r, to);
        };
        if (NV) {
#pragma unroll
            for (int v = 0; v < HELD; ++v) {
                const int col = col0 + 8 * team * v;
                if (in) complete<XF, EVEN>(x[v], x_at + 8 * team * v * XS, p.at_x.end, col, K);
                floats<XF>(x[v], f[v]);
                tops(col, f[v]);
            }
        } else {
#pragma unroll 4
            for (long long v = 0; v < vectors; ++v) {
                if (col0 + 8 * team * v >= K) break;
                get(v, f[0]);
                tops((int)(col0 + 8 * team * v), f[0]);
            }
        }
        const Byte* const again = x_at;
        x_at += x_step;
        if (NV) ask(row + step < p.M);
        reduce<false, true, false>(team, room, turn, none, top);
        turn ^= 1;
        if (in) {
            if (lane == 0) p.scale[row] = Rounder::scale(top, 1.f);
            const Rounder round(top);
            if (NV) {
#pragma unroll
                for (int v = 0; v < HELD; ++v) store_int8<EVEN>(q_at + 8 * team * v, p.at_q.end, col0 + 8 * team * v, K, f[v], round);
            } else {
                x_at = again;
#pragma unroll 4
                for (long long v = 0; v < vectors; ++v) {
                    const long long col = col0 + 8 * team * v;
                    if (col >= K) break;
                    get(v, f[0]);
                    store_int8<EVEN>(q_at + 8 * team * v, p.at_q.end, (int)col, K, f[0], round);
                }
                x_at += x_step;
            }
        }
        row += step;
        q_at += q_step;
    }
}

// ---- dropout alone ---------------------------------------------------------------------------------------------------------
// Two pieces a thread at a time; the last elements, less than a piece, go one to a thread.  us for 2^26 elements: bf16 63 (4.3 TB/s; traffic alone would be 41, the
// generator's products 32; no pipe is full, ALU 61 %, issue 55 %, heavy FMA 36 %), with a residual 69 (5.8), all in fp32 126 (6.4, the copy rate).
constexpr int DROPOUT_CTAS = 8;  // of an SM, where registers leave room for as many
template <bool XF, int RES, bool LOW> __global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
    constexpr bool RF = RES == 2;
    constexpr int XS = XF ? 4 : 2, RS = RF ? 4 : 2;
    stream_order();
    const Dropper drop(p.d);
    const int ys = p.y_f32 ? 4 : 2;
    const long long pieces = p.n >> 3, step = (long long)gridDim.x * 512;
    auto finish = [&](const Raw<XF>& x, const Raw<RF>& r, long long n) {
        float f[8];
        floats<XF>(x, f);
        drop.template apply<LOW>(n, f);
        if (RES) {
            float g[8];
            floats<RF>(r, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __fadd_rn(g[i], f[i]);
        }
        store<true>((Byte*)p.y + 8 * n * ys, nullptr, p.y_f32, 0, 8, f);
    };
    for (long long n = (long long)blockIdx.x * 512 + threadIdx.x; n < pieces; n += step) {
        Raw<XF> x[2];
        Raw<RF> r[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int there = n + 256 * b < pieces ? 0 : 8;  // (behind the end: not read)
            request<XF, true>(x[b], (const Byte*)p.x + 8 * (n + 256 * b) * XS, nullptr, there, 8);
            if (RES) request<RF, true>(r[b], (const Byte*)p.residual + 8 * (n + 256 * b) * RS, nullptr, there, 8);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
            if (n + 256 * b < pieces) finish(x[b], r[b], n + 256 * b);
    }
    if (blockIdx.x == 0 && threadIdx.x < (p.n & 7)) {
        const long long at = 8 * pieces + threadIdx.x;
        uint32_t c[2][4];
        drop.template words<LOW>(pieces, c);
        uint32_t word = c[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) word = threadIdx.x == i ? c[i / 4][i % 4] : word;
        float f = XF ? ((const float*)p.x)[at] : __bfloat162float(((const bf16*)p.x)[at]);
        f = drop.keeps(word) ? __fmul_rn(f, drop.scale) : 0.f;
        if (RES) f = __fadd_rn(RF ? ((const float*)p.residual)[at] : __bfloat162float(((const bf16*)p.residual)[at]), f);
        if (p.y_f32) ((float*)p.y)[at] = f;
        else ((bf16*)p.y)[at] = __float2bfloat16_rn(f);
    }
}

}  // namespace norm

int launch_quantize(const QuantizeParams& a, cudaStream_t stream) {
    using namespace norm;
    QuantizeKernelParams p;
    static_cast<QuantizeParams&>(p) = a;
    const long long pieces = pieces_of(p.K);
    const int nv = pieces > 4 * threads_most(4) ? 0 : vectors_of(p.M, pieces);
    p.t = nv ? teams_of(pieces, nv, pieces <= 32 * nv ? 256 : 1) : Teams{1024, 1};
    p.at_x = lie_of(p.x, p.M, p.K, p.ldx, p.x_f32 ? 4 : 2);
    p.at_q = lie_of(p.q, p.M, p.K, p.ldq, 1);
#define WKV7_TYPES(nv, even) {quantize_kernel<nv, false, even>, quantize_kernel<nv, true, even>}
    static void (*const kernels[4][2][2])(QuantizeKernelParams) = {{WKV7_TYPES(0, false), WKV7_TYPES(0, true)}, {WKV7_TYPES(1, false), WKV7_TYPES(1, true)},
                                                                   {WKV7_TYPES(2, false), WKV7_TYPES(2, true)}, {WKV7_TYPES(4, false), WKV7_TYPES(4, true)}};
#undef WKV7_TYPES
    const bool even = p.K % 8 == 0 && p.at_x.end && p.at_q.end;
    const unsigned grid = (unsigned)ctas_of(p.M, p.t, sm_count(), nv == 4 ? 544 : 1024);
    return launch(kernels[nv == 4 ? 3 : nv][even][p.x_f32], dim3(grid), p.t.threads * p.t.rows, 0, stream, p) ? kOk : kLaunchFailed;
}

int launch_dropout(const DropoutParams& p, cudaStream_t stream) {
    using namespace norm;
#define WKV7_LOW(xf, res) {dropout_kernel<xf, res, false>, dropout_kernel<xf, res, true>}
    static void (*const kernels[2][3][2])(DropoutParams) = {{WKV7_LOW(false, 0), WKV7_LOW(false, 1), WKV7_LOW(false, 2)}, {WKV7_LOW(true, 0), WKV7_LOW(true, 1), WKV7_LOW(true, 2)}};
#undef WKV7_LOW
    const long long want = (p.n + 4095) / 4096, most = (long long)sm_count() * DROPOUT_CTAS;
    return launch(kernels[p.x_f32][p.residual ? 1 + p.r_f32 : 0][low_counters(p.n)], dim3((unsigned)(want < most ? want : most)), 256, 0, stream, p) ? kOk : kLaunchFailed;
}

}  // namespace wkv7

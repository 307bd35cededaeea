// The residual stream between the mixers: its addition with dropout, its norm, and rows in 8 bits for the products of serving.
//     h = residual + dropout(x)                     rounded to the residual's type: the stream as it is kept
//     y = h r w,  r = 1 / sqrt(mean h^2 + eps)      in x's type, fp32, or 8 bits: q = rint(127 y / a), scale a / 127, a = max |y| of the row
//     dh += r (g - h r^2 mean(g h)),  g = dy w;  dx = dropout'(dh);  dw = sum over the rows of dy h r
// All of it is bound by memory: each element is read once and written once.  A row belongs to a team of threads, eight adjacent elements (NV times) to a thread, so
// that it stays in registers between its sums and its results; CTAs are persistent, hold the weight in registers and request a row's
// elements while they work on the one before.  a does not need r, since max |h r w| = r max |h w|: one reduction serves both.
// Sums are fp32, in an order that the sizes alone decide.
#include "norm.cuh"

namespace wkv7 {
namespace norm {

// CTAs of the most threads that an SM is to hold, and the threads of an SM that the grid is sized for
constexpr int fwd_ctas(int nv) { return nv == 1 ? 4 : 1; }
constexpr int fwd_threads(int nv) { return nv == 1 ? 1024 : nv == 2 ? 512 : 544; }
struct FwdKernelParams : NormFwdParams {
    Teams t;
    Lie lx, lr, ly, lh;
    float inv_d;  // 1 / D
};
// RES: no residual, bf16, fp32.  Of rows that take four pieces a thread nothing is requested ahead and the weight is not held: registers.
template <int NV, bool XF, int RES, bool DROP, bool INT8, bool EVEN> __global__ void __launch_bounds__(threads_most(NV), fwd_ctas(NV)) norm_fwd_kernel(const __grid_constant__ FwdKernelParams p) {
    constexpr bool HELD = NV < 4, RF = RES == 2;
    __shared__ Room room;
    stream_order();
    const int team = p.t.threads, lane = threadIdx.x % team, D = p.D;
    const long long step = (long long)gridDim.x * p.t.rows;
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const int col0 = first_col(row, D) + 8 * lane;
    float w[HELD ? NV : 1][8];
    Raw<XF> x[NV];
    Raw<RF> r[NV];
    auto ask = [&](long long m) {
        if (m >= p.M) return;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            request<XF, EVEN>(x[v], p.x, p.lx, m, col0 + 8 * team * v, D);
            if (RES) request<RF, EVEN>(r[v], p.residual, p.lr, m, col0 + 8 * team * v, D);
        }
    };
    if (HELD) {
        ask(row);
#pragma unroll
        for (int v = 0; v < NV; ++v) weights(p.weight, p.w_f32, col0 + 8 * team * v, D, w[v]);
    }
    const Dropper drop(p.d);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * p.t.rows; first < p.M; first += step, row += step) {  // (the same for all threads: there are barriers within)
        const bool in = row < p.M;
        if (!HELD) ask(row);
        float f[NV][8], sum = 0.f, top = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = col0 + 8 * team * v;
            if (in) complete<XF, EVEN>(x[v], p.x, p.lx, row, col, D);
            floats<XF>(x[v], f[v]);
            if (DROP) drop.apply((unsigned long long)(row * D + col) >> 3, f[v]);
            if (RES) {
                float g[8];
                if (in) complete<RF, EVEN>(r[v], p.residual, p.lr, row, col, D);
                floats<RF>(r[v], g);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] = __fadd_rn(g[i], f[v][i]);  // (not merged with dropout's product: what is kept is the same however it is called)
                if (!RF) unpack8(pack8(f[v]), f[v]);
                if (in) store<EVEN>(p.h, RF, p.lh, row, col, D, f[v]);
            }
            clear_outside<EVEN>(col, D, f[v]);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(f[v][i], f[v][i], sum);
            if (!HELD && INT8) weights(p.weight, p.w_f32, col, D, w[0]);
            if (HELD || INT8)
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= w[HELD ? v : 0][i];
            if (INT8)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max_abs(top, f[v][i]);
        }
        if (HELD) ask(row + step);
        reduce<true, INT8>(team, room, turn, sum, top);
        turn ^= 1;
        const float rstd = rsqrtf(fmaf(sum, p.inv_d, p.eps));
        if (!in) continue;
        if (lane == 0) {
            if (p.rstd) p.rstd[row] = rstd;
            if (INT8) p.scale[row] = Rounder::scale(top, rstd);
        }
        const Rounder round(top);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = col0 + 8 * team * v;
            if (INT8) {
                store_int8<EVEN>((signed char*)p.y, p.ly, row, col, D, f[v], round);
            } else {
                if (!HELD) weights(p.weight, p.w_f32, col, D, w[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= HELD ? rstd : rstd * w[0][i];
                store<EVEN>(p.y, p.y_f32, p.ly, row, col, D, f[v]);
            }
        }
    }
}

}  // namespace norm

int launch_norm_fwd(const NormFwdParams& a, cudaStream_t stream) {
    using namespace norm;
    FwdKernelParams p;
    static_cast<NormFwdParams&>(p) = a;
    const long long pieces = pieces_of(p.D);
    const int nv = vectors_of(p.M, pieces);
    p.t = teams_of(pieces, nv);
    p.inv_d = (float)(1. / p.D);
    const bool int8 = p.scale != nullptr, drop = p.d.threshold != 0;
    p.lx = lie_of(p.x, p.M, p.D, p.ldx, 16);
    p.lr = lie_of(p.residual, p.M, p.D, p.ldr, 16);
    p.lh = lie_of(p.h, p.M, p.D, p.ldh, 16);
    p.ly = lie_of(p.y, p.M, p.D, p.ldy, int8 ? 8 : 16);
    // (rows of four pieces a thread have no EVEN form, only a residual has dropout)
#define WKV7_OUT(nv, xf, res, drop, even) {norm_fwd_kernel<nv, xf, res, drop, false, even>, norm_fwd_kernel<nv, xf, res, drop, true, even>}
#define WKV7_RES(nv, xf, e) \
    {{WKV7_OUT(nv, xf, 0, false, e), WKV7_OUT(nv, xf, 0, false, e)}, {WKV7_OUT(nv, xf, 1, false, e), WKV7_OUT(nv, xf, 1, true, e)}, {WKV7_OUT(nv, xf, 2, false, e), WKV7_OUT(nv, xf, 2, true, e)}}
#define WKV7_EVEN(nv, even) {{WKV7_RES(nv, false, false), WKV7_RES(nv, true, false)}, {WKV7_RES(nv, false, even), WKV7_RES(nv, true, even)}}
    static void (*const kernels[3][2][2][3][2][2])(FwdKernelParams) = {WKV7_EVEN(1, true), WKV7_EVEN(2, true), WKV7_EVEN(4, false)};
#undef WKV7_EVEN
#undef WKV7_RES
#undef WKV7_OUT
    const bool even = p.D % 8 == 0 && p.lx.end && (!p.residual || (p.lr.end && p.lh.end)) && p.ly.end;
    const auto kern = kernels[nv / 2][even][p.x_f32][p.residual ? 1 + p.r_f32 : 0][drop][int8];
    return launch(kern, dim3((unsigned)ctas_of(p.M, p.t, sm_count(), fwd_threads(nv))), p.t.threads * p.t.rows, 0, stream, p) ? kOk : kLaunchFailed;
}

}  // namespace wkv7

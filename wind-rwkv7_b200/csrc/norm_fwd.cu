// The residual stream between the mixers: its addition with dropout, its norm, and rows in 8 bits for the products of serving.
//     h = residual + dropout(x)                     rounded to the residual's type: the stream as it is kept
//     y = h r w,  r = 1 / sqrt(mean h^2 + eps)      in x's type, fp32, or 8 bits: q = rint(127 y / a), scale a / 127, a = max |y| of the row
//     dh += r (g - h r^2 mean(g h)),  g = dy w;  dx = dropout'(dh);  dw = sum over the rows of dy h r
// All of it is bound by memory: each element is read once and written once.  A row belongs to a team of threads, eight adjacent elements (NV times) to a thread, so
// that it stays in registers between its sums and its results; CTAs are persistent, hold the weight in registers and request a row's
// elements while they work on the one before.  a does not need r, since max |h r w| = r max |h w|: one reduction serves both.
// Sums are fp32, in an order that the sizes alone decide.  us, bf16 unless noted: 8192 x 2048 23.5 (5.7 TB/s), with dropout 30.4, 16384 x 4096 with an fp32 stream 136 (5.9 TB/s),
// 65536 x 768 72, 60000 x 1001 with dropout 133, 4096 x 16384 151.
#include "norm.cuh"

namespace wkv7 {
namespace norm {

// Threads of an SM, for which there are registers and the grid is sized.  Two pieces of bf16 without parts fit 96 registers (8192 x 2048 25.1 -> 23.5 us, 65536 x 768 78 -> 72);
// the other forms of two pieces would spill what they have requested (60000 x 1001 with dropout 131 -> 175).  Four pieces: 544 threads, which rows of 16378 to 16383 elements need, leave
// 96 registers, and 39 of the 40 such forms spill, 4 to 836 bytes a thread.
constexpr int fwd_threads(int nv, bool narrow) { return nv == 1 ? 576 : nv == 2 ? narrow ? 640 : 512 : 544; }
struct FwdKernelParams : NormFwdParams {
    Teams t;
    Lie at_x, at_r, at_y, at_h;
    float inv_d;  // 1 / D
    bool low;     // dropout's counters are below 2^32
};
// ---- forward -----------------------------------------------------------------------------------------------------------------
// RES: no residual, bf16, fp32.  Of rows that take four pieces a thread nothing is requested ahead and the weight is not held: registers.
template <int NV, bool XF, int RES, bool DROP, bool INT8, bool EVEN>
__global__ void __launch_bounds__(NV == 1 ? threads_most(1) : fwd_threads(NV, EVEN && !XF && RES != 2), 1) norm_fwd_kernel(const __grid_constant__ FwdKernelParams p) {
    constexpr bool HELD = NV < 4, RF = RES == 2;
    constexpr int XS = XF ? 4 : 2, RS = RF ? 4 : 2;
    __shared__ Room room;
    stream_order();
    const int team = p.t.threads, lane = threadIdx.x % team, D = p.D;
    const long long step = (long long)gridDim.x * p.t.rows;
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const int col0 = first_col(row, D) + 8 * lane, ys = INT8 ? 1 : p.y_f32 ? 4 : 2;
    const Byte* x_at = p.at_x.base + (row * p.at_x.ld + col0) * XS;
    const Byte* r_at = p.at_r.base + (row * p.at_r.ld + col0) * RS;
    Byte* h_at = (Byte*)p.h + (row * p.at_h.ld + col0) * RS;
    Byte* y_at = (Byte*)p.y + (row * p.at_y.ld + col0) * ys;
    const long long x_step = step * p.at_x.ld * XS, r_step = step * p.at_r.ld * RS, h_step = step * p.at_h.ld * RS, y_step = step * p.at_y.ld * ys;
    Piece w[HELD ? NV : 1];
    Raw<XF> x[NV];
    Raw<RF> r[NV];
    auto ask = [&](bool in) {
        if (!in) return;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            request<XF, EVEN>(x[v], x_at + 8 * team * v * XS, p.at_x.end, col0 + 8 * team * v, D);
            if (RES) request<RF, EVEN>(r[v], r_at + 8 * team * v * RS, p.at_r.end, col0 + 8 * team * v, D);
        }
    };
    auto weight = [&](Piece& to, int v) {
        float f[8];
        weights(p.weight, p.w_f32, col0 + 8 * team * v, D, f);
        to.set(f);
    };
    if (HELD) {
        ask(row < p.M);
#pragma unroll
        for (int v = 0; v < NV; ++v) weight(w[HELD ? v : 0], v);
    }
    const Dropper drop(p.d);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * p.t.rows; first < p.M; first += step) {  // (the same for all threads: there are barriers within)
        const bool in = row < p.M;
        if (!HELD) ask(in);
        Piece y[NV];
        uint64_t sums = 0;  // (two zeros)
        float top = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = col0 + 8 * team * v;
            float f[8];
            if (in) complete<XF, EVEN>(x[v], x_at + 8 * team * v * XS, p.at_x.end, col, D);
            floats<XF>(x[v], f);
            if (DROP) drop.apply(p.low, (unsigned long long)(row * D + col) >> 3, f);
            y[v].set(f);
            if (RES) {
                float g[8];
                if (in) complete<RF, EVEN>(r[v], r_at + 8 * team * v * RS, p.at_r.end, col, D);
                floats<RF>(r[v], g);
                Piece res;
                res.set(g);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[v].p[i] = add2(res.p[i], y[v].p[i]);  // (not merged with dropout's product: what is kept is the same however it is called)
                y[v].get(f);
                if (!RF) unpack8(pack8(f), f);
                if (in) store<EVEN>(h_at + 8 * team * v * RS, p.at_h.end, RF, col, D, f);
            }
            clear_outside<EVEN>(col, D, f);
            y[v].set(f);
            if (!HELD && INT8) weight(w[0], v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sums = fma2(y[v].p[i], y[v].p[i], sums);
                if (HELD || INT8) y[v].p[i] = mul2(y[v].p[i], w[HELD ? v : 0].p[i]);
            }
            if (INT8) {
                y[v].get(f);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max_abs(top, f[i]);
            }
        }
        x_at += x_step;
        r_at += r_step;
        if (HELD) ask(row + step < p.M);
        float sum = sum_of(sums);
        reduce<true, INT8, false>(team, room, turn, sum, top);
        turn ^= 1;
        const float rstd = rsqrtf(fmaf(sum, p.inv_d, p.eps));
        if (in) {
            if (lane == 0) {
                if (p.rstd) p.rstd[row] = rstd;
                if (INT8) p.scale[row] = Rounder::scale(top, rstd);
            }
            const Rounder round(top);
            const uint64_t rr = two(rstd, rstd);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float f[8];
                if (!INT8) {
                    if (!HELD) weight(w[0], v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[v].p[i] = mul2(y[v].p[i], HELD ? rr : mul2(rr, w[0].p[i]));
                }
                y[v].get(f);
                if (INT8) store_int8<EVEN>(y_at + 8 * team * v, p.at_y.end, col0 + 8 * team * v, D, f, round);
                else store<EVEN>(y_at + 8 * team * v * ys, p.at_y.end, p.y_f32, col0 + 8 * team * v, D, f);
            }
        }
        row += step;
        h_at += h_step;
        y_at += y_step;
    }
}

}  // namespace norm

int launch_norm_fwd(const NormFwdParams& a, cudaStream_t stream) {
    using namespace norm;
    FwdKernelParams p;
    static_cast<NormFwdParams&>(p) = a;
    const long long pieces = pieces_of(p.D);
    const int nv = vectors_of(p.M, pieces);
    p.t = teams_of(pieces, nv, pieces <= 32 * nv ? 256 : 1);
    p.inv_d = (float)(1. / p.D);
    p.low = low_counters(p.M * p.D);
    const bool int8 = p.scale != nullptr, drop = p.d.threshold != 0;
    p.at_x = lie_of(p.x, p.M, p.D, p.ldx, p.x_f32 ? 4 : 2);
    p.at_r = lie_of(p.residual, p.M, p.D, p.ldr, p.r_f32 ? 4 : 2);
    p.at_h = lie_of(p.h, p.M, p.D, p.ldh, p.r_f32 ? 4 : 2);
    p.at_y = lie_of(p.y, p.M, p.D, p.ldy, int8 ? 1 : p.y_f32 ? 4 : 2);
    // (only a residual has dropout)
#define WKV7_OUT(nv, xf, res, drop, even) {norm_fwd_kernel<nv, xf, res, drop, false, even>, norm_fwd_kernel<nv, xf, res, drop, true, even>}
#define WKV7_RES(nv, xf, e) \
    {{WKV7_OUT(nv, xf, 0, false, e), WKV7_OUT(nv, xf, 0, false, e)}, {WKV7_OUT(nv, xf, 1, false, e), WKV7_OUT(nv, xf, 1, true, e)}, {WKV7_OUT(nv, xf, 2, false, e), WKV7_OUT(nv, xf, 2, true, e)}}
#define WKV7_EVEN(nv) {{WKV7_RES(nv, false, false), WKV7_RES(nv, true, false)}, {WKV7_RES(nv, false, true), WKV7_RES(nv, true, true)}}
    static void (*const kernels[3][2][2][3][2][2])(FwdKernelParams) = {WKV7_EVEN(1), WKV7_EVEN(2), WKV7_EVEN(4)};
#undef WKV7_EVEN
#undef WKV7_RES
#undef WKV7_OUT
    const bool even = p.D % 8 == 0 && p.at_x.end && (!p.residual || (p.at_r.end && p.at_h.end)) && p.at_y.end;
    const auto kern = kernels[nv / 2][even][p.x_f32][p.residual ? 1 + p.r_f32 : 0][drop][int8];
    return launch(kern, dim3((unsigned)ctas_of(p.M, p.t, sm_count(), fwd_threads(nv, even && !p.x_f32 && !(p.residual && p.r_f32)))), p.t.threads * p.t.rows, 0, stream, p) ? kOk : kLaunchFailed;
}

}  // namespace wkv7

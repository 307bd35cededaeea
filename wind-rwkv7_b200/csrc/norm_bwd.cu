// Backward of the residual stream's norm (norm_fwd.cu has the formulas): one pass over the rows, the weight's gradient kept in registers by the threads that have its columns, and
// a second kernel for the CTAs' parts of it.
#include "norm.cuh"

namespace wkv7 {
namespace norm {

// CTAs of the most threads that an SM is to hold, and the threads of an SM that the grid is sized for
constexpr int bwd_ctas(int nv) { return nv == 1 ? 2 : 1; }
constexpr int bwd_threads(int nv) { return nv == 1 ? 768 : nv == 2 ? 512 : 544; }
// ---- backward --------------------------------------------------------------------------------------------------------------
struct BwdKernelParams : NormBwdParams {
    Teams t;
    Lie at_h, at_dy, at_dh, at_dx, at_dr;
    float inv_d;  // 1 / D
};
template <int NV, bool YF, bool HF, bool DROP, bool EVEN> __global__ void __launch_bounds__(threads_most(NV), bwd_ctas(NV)) norm_bwd_kernel(const __grid_constant__ BwdKernelParams p) {
    constexpr bool HELD = NV < 4;
    __shared__ Room room;
    extern __shared__ float sums[];  // [rows of a CTA][D], where it has several
    stream_order();
    const int team = p.t.threads, lane = threadIdx.x % team, D = p.D;
    const long long step = (long long)gridDim.x * p.t.rows;
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const int col0 = first_col(row, D) + 8 * lane;
    float w[HELD ? NV : 1][8], dw[NV][8];
    Raw<HF> h[NV], dh[NV];
    Raw<YF> dy[NV];
    float rstd_next = 0.f;
    auto ask = [&](long long m) {
        if (m >= p.M) return;
        rstd_next = p.rstd[m];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            request<HF, EVEN>(h[v], p.h, p.at_h, m, col0 + 8 * team * v, D);
            request<YF, EVEN>(dy[v], p.dy, p.at_dy, m, col0 + 8 * team * v, D);
            if (p.dh) request<HF, EVEN>(dh[v], p.dh, p.at_dh, m, col0 + 8 * team * v, D);
        }
    };
    if (HELD) ask(row);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if (HELD) weights(p.weight, p.w_f32, col0 + 8 * team * v, D, w[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[v][i] = 0.f;
    }
    const Dropper drop(p.d);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * p.t.rows; first < p.M; first += step, row += step) {
        const bool in = row < p.M;
        if (!HELD) ask(row);
        const float rstd = rstd_next;
        float sum = 0.f, none = 0.f;
        Raw<HF> h_now[NV], dh_now[NV];
        Raw<YF> dy_now[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float f[8], g[8];
            const int col = col0 + 8 * team * v;
            if (in) {
                complete<HF, EVEN>(h[v], p.h, p.at_h, row, col, D);
                complete<YF, EVEN>(dy[v], p.dy, p.at_dy, row, col, D);
                if (p.dh) complete<HF, EVEN>(dh[v], p.dh, p.at_dh, row, col, D);
            }
            h_now[v] = h[v]; dy_now[v] = dy[v]; dh_now[v] = dh[v];
            floats<HF>(h_now[v], f);
            floats<YF>(dy_now[v], g);
            clear_outside<EVEN>(col, D, f);
            clear_outside<EVEN>(col, D, g);
            if (!HELD) weights(p.weight, p.w_f32, col, D, w[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (in) dw[v][i] = fmaf(g[i], f[i] * rstd, dw[v][i]);
                sum = fmaf(g[i] * w[HELD ? v : 0][i], f[i], sum);
            }
        }
        if (HELD) ask(row + step);
        reduce<true, false>(team, room, turn, sum, none);
        turn ^= 1;
        if (!in) continue;
        const float c = sum * p.inv_d * rstd * rstd;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = col0 + 8 * team * v;
            float f[8], g[8], d[8];
            floats<HF>(h_now[v], f);
            floats<YF>(dy_now[v], g);
            clear_outside<EVEN>(col, D, f);
            clear_outside<EVEN>(col, D, g);
            if (!HELD) weights(p.weight, p.w_f32, col, D, w[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = rstd * fmaf(-c, f[i], g[i] * w[HELD ? v : 0][i]);
            if (p.dh) {
                float e[8];
                floats<HF>(dh_now[v], e);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] += e[i];
            }
            if (p.dr) store<EVEN>(p.dr, HF, p.at_dr, row, col, D, d);
            if (p.dx) {
                if (DROP) drop.apply((unsigned long long)(row * D + col) >> 3, d);
                store<EVEN>(p.dx, p.x_f32, p.at_dx, row, col, D, d);
            }
        }
    }
    if (!p.dw) return;
    float* const out = p.partial + (long long)blockIdx.x * p.D;
    float* const mine = p.t.rows == 1 ? out : sums + (threadIdx.x / team) * p.D;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int col = col0 + 8 * team * v + i;
            if (col >= 0 && col < D) mine[col] = dw[v][i];
        }
    if (p.t.rows == 1) return;
    __syncthreads();
    for (int c = threadIdx.x; c < p.D; c += blockDim.x) {
        float s = 0.f;
        for (int r = 0; r < p.t.rows; ++r) s += sums[r * p.D + c];
        out[c] = s;
    }
}
// Sums of the CTAs' parts: 32 columns a CTA, its 32 warps take the parts in turn.
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* partial, float* dw, int D, int parts) {
    stream_order();
    __shared__ float sums[32][33];
    const int x = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float s = 0.f;
    if (c < D)
#pragma unroll 4
        for (int i = r; i < parts; i += 32) s += partial[(long long)i * D + c];
    sums[r][x] = s;
    __syncthreads();
    if (r == 0 && c < D) {
        for (int i = 1; i < 32; ++i) s += sums[i][x];
        dw[c] = s;
    }
}

}  // namespace norm

// The parts of dw: CTAs of the backward.  Sizes alone decide their number, so that the sums are the same on every device.
int norm_bwd_partials(long long M, long long D) {
    using namespace norm;
    const long long pieces = pieces_of(D);
    const int nv = vectors_of(M, pieces);
    return (int)ctas_of(M, teams_of(pieces, nv), 148, bwd_threads(nv));
}

int launch_norm_bwd(const NormBwdParams& a, cudaStream_t stream) {
    using namespace norm;
    BwdKernelParams p;
    static_cast<NormBwdParams&>(p) = a;
    const long long pieces = pieces_of(p.D);
    const int nv = vectors_of(p.M, pieces), parts = norm_bwd_partials(p.M, p.D);
    p.t = teams_of(pieces, nv);
    p.inv_d = (float)(1. / p.D);
    p.at_h = lie_of(p.h, p.M, p.D, p.ldh, 16);
    p.at_dy = lie_of(p.dy, p.M, p.D, p.lddy, 16);
    p.at_dh = lie_of(p.dh, p.M, p.D, p.lddh, 16);
    p.at_dx = lie_of(p.dx, p.M, p.D, p.lddx, 16);
    p.at_dr = lie_of(p.dr, p.M, p.D, p.lddr, 16);
#define WKV7_DROP(nv, yf, hf, even) {norm_bwd_kernel<nv, yf, hf, false, even>, norm_bwd_kernel<nv, yf, hf, true, even>}
#define WKV7_TYPES(nv, e) {{WKV7_DROP(nv, false, false, e), WKV7_DROP(nv, false, true, e)}, {WKV7_DROP(nv, true, false, e), WKV7_DROP(nv, true, true, e)}}
    // (rows of four pieces a thread have no EVEN form)
    static void (*const kernels[3][2][2][2][2])(BwdKernelParams) = {{WKV7_TYPES(1, false), WKV7_TYPES(1, true)}, {WKV7_TYPES(2, false), WKV7_TYPES(2, true)},
                                                                    {WKV7_TYPES(4, false), WKV7_TYPES(4, false)}};
#undef WKV7_TYPES
#undef WKV7_DROP
    const bool even = p.D % 8 == 0 && p.at_h.end && p.at_dy.end && (!p.dh || p.at_dh.end) && (!p.dx || p.at_dx.end) && (!p.dr || p.at_dr.end);
    const auto kern = kernels[nv / 2][even][p.y_f32][p.h_f32][p.d.threshold && p.dx];
    const int smem = p.dw && p.t.rows > 1 ? p.t.rows * p.D * 4 : 0;  // (rows x D <= 256 threads x two pieces: 16 KB)
    if (!launch(kern, dim3((unsigned)parts), p.t.threads * p.t.rows, smem, stream, p)) return kLaunchFailed;
    if (p.dw && !launch(norm_dw_kernel, dim3((unsigned)((p.D + 31) / 32)), 1024, 0, stream, (const float*)p.partial, p.dw, p.D, parts)) return kLaunchFailed;
    return kOk;
}

}  // namespace wkv7

// Backward of the residual stream's norm (norm_fwd.cu has the formulas): one pass over the rows, the weight's gradient kept in registers by the threads that have its columns, and
// a second kernel for the CTAs' parts of it.  Each of h, dy and dh is read once (rows of four pieces a thread: twice), dr and dx are written once.  Bound by memory; with dropout as much
// by its generator.  us: 16384 x 4096 with an fp32 stream 185 (5.8 TB/s), 8192 x 2048 bf16 30.7, with dropout 43.7, 65536 x 768 85, 60000 x 1001 with dropout 198, 4096 x 16384 274.
#include "norm.cuh"

namespace wkv7 {
namespace norm {

// CTAs of the most threads that an SM's registers are shared out to, and the threads of an SM that the grid is sized for
constexpr int bwd_ctas(int nv) { return nv == 1 ? 2 : 1; }
constexpr int bwd_threads(int nv) { return nv == 1 ? 768 : nv == 2 ? 512 : 544; }
// ---- backward --------------------------------------------------------------------------------------------------------------
struct BwdKernelParams : NormBwdParams {
    Teams t;
    Lie at_h, at_dy, at_dh, at_dx, at_dr;
    float inv_d;  // 1 / D
    bool low;     // dropout's counters are below 2^32
};
// HELD: the weight's gradient and the next row are in registers, the weight in shared memory (in registers, too, 100 to 400 bytes a thread would be spilled, among
// them what has been requested, which is then waited for: 16384 x 4096 with an fp32 stream 185 -> 261 us).  Rows of four pieces a thread have the gradient in shared memory
// and are read twice.
template <int NV, bool YF, bool HF, bool DROP, bool EVEN>
__global__ void __launch_bounds__(threads_most(NV), bwd_ctas(NV)) norm_bwd_kernel(const __grid_constant__ BwdKernelParams p) {
    constexpr bool HELD = NV < 4;
    constexpr int HS = HF ? 4 : 2, YS = YF ? 4 : 2, N = HELD ? NV : 1;
    __shared__ Room room;
    extern __shared__ __align__(16) ulonglong2 shared[];  // HELD: the threads' parts of the weight [NV][2][threads], in the end its gradients [rows of a CTA][D]; else gradients
    stream_order();
    const int team = p.t.threads, lane = threadIdx.x % team, D = p.D;
    const long long step = (long long)gridDim.x * p.t.rows;
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const int col0 = first_col(row, D) + 8 * lane;
    const auto piece = [&](const Lie& t, int size, long long m, int v) { return t.base + (m * t.ld + (col0 + 8 * team * v)) * size; };
    const auto mine = [&](int v, int half) -> ulonglong2& { return shared[(2 * v + half) * blockDim.x + threadIdx.x]; };
    const auto from_shared = [&](Piece& to, int v) {
        const ulonglong2 lo = mine(v, 0), hi = mine(v, 1);
        to.p[0] = lo.x; to.p[1] = lo.y; to.p[2] = hi.x; to.p[3] = hi.y;
    };
    const auto to_shared = [&](const Piece& from, int v) {
        mine(v, 0) = make_ulonglong2(from.p[0], from.p[1]);
        mine(v, 1) = make_ulonglong2(from.p[2], from.p[3]);
    };
    const auto weight = [&](Piece& to, int v) {
        float f[8];
        weights(p.weight, p.w_f32, col0 + 8 * team * v, D, f);
        to.set(f);
    };
    Piece dw[N];
    Raw<HF> h[N], dh[N];
    Raw<YF> dy[N];
    float rstd_next = 0.f;
    const auto ask = [&](long long m) {
        if (m >= p.M) return;
        rstd_next = p.rstd[m];
#pragma unroll
        for (int v = 0; v < (HELD ? NV : 0); ++v) {
            const int col = col0 + 8 * team * v, u = HELD ? v : 0;
            request<HF, EVEN>(h[u], piece(p.at_h, HS, m, v), p.at_h.end, col, D);
            request<YF, EVEN>(dy[u], piece(p.at_dy, YS, m, v), p.at_dy.end, col, D);
            if (p.dh) request<HF, EVEN>(dh[u], piece(p.at_dh, HS, m, v), p.at_dh.end, col, D);
        }
    };
    if (HELD) ask(row);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        Piece z;
        if (HELD) {
            weight(z, v);
            to_shared(z, v);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) z.p[i] = 0;  // (two zeros)
        if (HELD) dw[HELD ? v : 0] = z;
        else if (p.dw) to_shared(z, v);
    }
    const Dropper drop(p.d);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * p.t.rows; first < p.M; first += step, row += step) {
        const bool in = row < p.M;
        if (!HELD) ask(row);
        const float rstd = rstd_next;
        const uint64_t rr = two(rstd, rstd);
        uint64_t both = 0;
        Raw<HF> h_now[N], dh_now[N];
        Raw<YF> dy_now[N];
#pragma unroll(HELD ? NV : 2)
        for (int v = 0; v < NV; ++v) {
            const int col = col0 + 8 * team * v, u = HELD ? v : 0;
            if (in) {
                if (!HELD) {
                    request<HF, EVEN>(h[0], piece(p.at_h, HS, row, v), p.at_h.end, col, D);
                    request<YF, EVEN>(dy[0], piece(p.at_dy, YS, row, v), p.at_dy.end, col, D);
                }
                complete<HF, EVEN>(h[u], piece(p.at_h, HS, row, v), p.at_h.end, col, D);
                complete<YF, EVEN>(dy[u], piece(p.at_dy, YS, row, v), p.at_dy.end, col, D);
                if (HELD && p.dh) complete<HF, EVEN>(dh[u], piece(p.at_dh, HS, row, v), p.at_dh.end, col, D);
            }
            if (HELD) {
                h_now[u] = h[u];
                dy_now[u] = dy[u];
                dh_now[u] = dh[u];
            }
            float f[8], g[8];
            floats<HF>(h[u], f);
            floats<YF>(dy[u], g);
            clear_outside<EVEN>(col, D, f);
            clear_outside<EVEN>(col, D, g);
            Piece a, b, w;
            a.set(f);
            b.set(g);
            if (in && p.dw) {
                if (!HELD) from_shared(dw[0], v);
#pragma unroll
                for (int i = 0; i < 4; ++i) dw[u].p[i] = fma2(b.p[i], mul2(a.p[i], rr), dw[u].p[i]);
                if (!HELD) to_shared(dw[0], v);
            }
            if (HELD) from_shared(w, v);
            else weight(w, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) both = fma2(mul2(b.p[i], w.p[i]), a.p[i], both);
        }
        if (HELD) ask(row + step);
        float sum = sum_of(both), none = 0.f;
        reduce<true, false, HELD>(team, room, turn, sum, none);
        turn ^= 1;
        if (!in) continue;
        const float c = -(sum * p.inv_d * rstd * rstd);
        const uint64_t cc = two(c, c);
#pragma unroll(HELD ? NV : 2)
        for (int v = 0; v < NV; ++v) {
            const int col = col0 + 8 * team * v, u = HELD ? v : 0;
            if (!HELD) {
                request<HF, EVEN>(h_now[0], piece(p.at_h, HS, row, v), p.at_h.end, col, D);
                complete<HF, EVEN>(h_now[0], piece(p.at_h, HS, row, v), p.at_h.end, col, D);
                request<YF, EVEN>(dy_now[0], piece(p.at_dy, YS, row, v), p.at_dy.end, col, D);
                complete<YF, EVEN>(dy_now[0], piece(p.at_dy, YS, row, v), p.at_dy.end, col, D);
                if (p.dh) {
                    request<HF, EVEN>(dh_now[0], piece(p.at_dh, HS, row, v), p.at_dh.end, col, D);
                    complete<HF, EVEN>(dh_now[0], piece(p.at_dh, HS, row, v), p.at_dh.end, col, D);
                }
            }
            float f[8], g[8];
            floats<HF>(h_now[u], f);
            floats<YF>(dy_now[u], g);
            Piece a, b, w;
            a.set(f);
            b.set(g);
            if (HELD) from_shared(w, v);
            else weight(w, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) b.p[i] = fma2(cc, a.p[i], mul2(b.p[i], w.p[i]));
            if (p.dh) {
                floats<HF>(dh_now[u], f);
                a.set(f);
#pragma unroll
                for (int i = 0; i < 4; ++i) b.p[i] = fma2(rr, b.p[i], a.p[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) b.p[i] = mul2(rr, b.p[i]);
            }
            b.get(f);
            if (p.dr) store<EVEN>((Byte*)piece(p.at_dr, HS, row, v), p.at_dr.end, HF, col, D, f);
            if (p.dx) {
                if (DROP) drop.apply(p.low, (unsigned long long)(row * D + col) >> 3, f);
                store<EVEN>((Byte*)piece(p.at_dx, p.x_f32 ? 4 : 2, row, v), p.at_dx.end, p.x_f32, col, D, f);
            }
        }
    }
    if (!p.dw) return;
    if (HELD) __syncthreads();  // (the weight is read no more)
    float* const out = p.partial + (long long)blockIdx.x * D;
    float* const sums = reinterpret_cast<float*>(shared);
    float* const to = !HELD || p.t.rows == 1 ? out : sums + (threadIdx.x / team) * D;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float f[8];
        if (!HELD) from_shared(dw[0], v);
        dw[HELD ? v : 0].get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int col = col0 + 8 * team * v + i;
            if (col >= 0 && col < D) to[col] = f[i];
        }
    }
    if (p.t.rows == 1) return;
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
        float s = 0.f;
        for (int r = 0; r < p.t.rows; ++r) s += sums[r * D + c];
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

namespace norm {
// (where all is fp32 two pieces do not fit the registers: such rows of more than 288 pieces spill 84 to 200 bytes a thread)
static int bwd_vectors(long long M, long long pieces, bool wide) { return wide && pieces <= threads_most(1) ? 1 : vectors_of(M, pieces); }
// One CTA an SM where there are rows for as many teams, so that there are few parts of dw; else smaller ones
static Teams bwd_teams(long long M, long long pieces, int nv) {
    Teams t = teams_of(pieces, nv, nv == 1 ? 256 : nv == 2 ? threads_most(nv) : 1);  // (four pieces a thread: teams are CTAs)
    while (t.rows > 1 && (t.rows - 1) * 148LL >= M && t.rows * t.threads > 32) t.rows = (t.rows + 1) / 2;
    while (t.rows * t.threads % 32) t.rows *= 2;
    return t;
}
// The parts of dw: CTAs of the backward.  Sizes and types alone decide their number, so that the sums are the same on every device.
static int parts_of(long long M, long long pieces, int nv) { return (int)ctas_of(M, bwd_teams(M, pieces, nv), 148, bwd_threads(nv)); }
}  // namespace norm

int norm_bwd_partials(long long M, long long D) {
    using namespace norm;
    const long long pieces = pieces_of(D);
    const int a = parts_of(M, pieces, bwd_vectors(M, pieces, false)), b = parts_of(M, pieces, bwd_vectors(M, pieces, true));
    return a > b ? a : b;
}

int launch_norm_bwd(const NormBwdParams& a, cudaStream_t stream) {
    using namespace norm;
    BwdKernelParams p;
    static_cast<NormBwdParams&>(p) = a;
    const long long pieces = pieces_of(p.D);
    const int nv = bwd_vectors(p.M, pieces, p.y_f32 && p.h_f32), parts = parts_of(p.M, pieces, nv);
    p.t = bwd_teams(p.M, pieces, nv);
    p.inv_d = (float)(1. / p.D);
    p.low = low_counters(p.M * p.D);
    p.at_h = lie_of(p.h, p.M, p.D, p.ldh, p.h_f32 ? 4 : 2);
    p.at_dy = lie_of(p.dy, p.M, p.D, p.lddy, p.y_f32 ? 4 : 2);
    p.at_dh = lie_of(p.dh, p.M, p.D, p.lddh, p.h_f32 ? 4 : 2);
    p.at_dx = lie_of(p.dx, p.M, p.D, p.lddx, p.x_f32 ? 4 : 2);
    p.at_dr = lie_of(p.dr, p.M, p.D, p.lddr, p.h_f32 ? 4 : 2);
#define WKV7_DROP(nv, yf, hf, even) {norm_bwd_kernel<nv, yf, hf, false, even>, norm_bwd_kernel<nv, yf, hf, true, even>}
#define WKV7_TYPES(nv, e) {{WKV7_DROP(nv, false, false, e), WKV7_DROP(nv, false, true, e)}, {WKV7_DROP(nv, true, false, e), WKV7_DROP(nv, true, true, e)}}
    static void (*const kernels[3][2][2][2][2])(BwdKernelParams) = {{WKV7_TYPES(1, false), WKV7_TYPES(1, true)}, {WKV7_TYPES(2, false), WKV7_TYPES(2, true)},
                                                                    {WKV7_TYPES(4, false), WKV7_TYPES(4, true)}};
#undef WKV7_TYPES
#undef WKV7_DROP
    const bool even = p.D % 8 == 0 && p.at_h.end && p.at_dy.end && (!p.dh || p.at_dh.end) && (!p.dx || p.at_dx.end) && (!p.dr || p.at_dr.end);
    const auto kern = kernels[nv / 2][even][p.y_f32][p.h_f32][p.d.threshold && p.dx];
    const int threads = p.t.threads * p.t.rows;
    const int smem = threads * nv * 32;  // (the rows' gradients fit, too: rows x D <= threads x 8 nv)
    static thread_local uint32_t allowed[64];
    if (nv == 4 && !allow_smem(kern, allowed, (even ? 8 : 0) | (p.y_f32 ? 4 : 0) | (p.h_f32 ? 2 : 0) | (p.d.threshold && p.dx ? 1 : 0), threads_most(4) * 4 * 32)) return kLaunchFailed;
    if (!launch(kern, dim3((unsigned)parts), threads, smem, stream, p)) return kLaunchFailed;
    if (p.dw && !launch(norm_dw_kernel, dim3((unsigned)((p.D + 31) / 32)), 1024, 0, stream, (const float*)p.partial, p.dw, p.D, parts)) return kLaunchFailed;
    return kOk;
}

}  // namespace wkv7

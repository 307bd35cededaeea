// The residual stream between the mixers: its addition with dropout, its norm, and rows in 8 bits for the products of serving.
//     h = residual + dropout(x)                     rounded to the residual's type: the stream as it is kept
//     y = h r w,  r = 1 / sqrt(mean h^2 + eps)      in x's type, fp32, or 8 bits: q = rint(127 y / a), scale a / 127, a = max |y| of the row
//     dh += r (g - h r^2 mean(g h)),  g = dy w;  dx = dropout'(dh);  dw = sum over the rows of dy h r
// All of it is bound by memory: each element is read once and written once.  A row belongs to a team of threads, eight adjacent elements (NV times) to a thread, so
// that it stays in registers between its sums and its results; CTAs are persistent, hold the weight in registers and request a row's
// elements while they work on the one before.  a does not need r, since max |h r w| = r max |h w|: one reduction serves both.
// Sums are fp32, in an order that the sizes alone decide.
#include "norm.h"
#include "mma_bf16.cuh"
#include "wkv7_kernels.h"

namespace wkv7 {
namespace norm {

// ---- Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) -----------------------
// Ten rounds of two 32 x 32 -> 64 products for four words.  No mask is stored: the backward forms the words again.
struct Dropper {
    uint32_t k0, k1, below;  // kept: word > below (the threshold less one; 2^32 less one drops all)
    float scale;
    __device__ __forceinline__ explicit Dropper(const Dropout& d) : below((uint32_t)(d.threshold - 1)), scale(d.scale) {
        const unsigned long long s = d.where ? *d.where : d.seed;
        k0 = __shfl_sync(0xffffffffu, (uint32_t)s, 0);  // (the same for all lanes, which the compiler cannot see: the rounds' keys then cost the lanes nothing)
        k1 = __shfl_sync(0xffffffffu, (uint32_t)(s >> 32), 0);
    }
    // eight adjacent elements, of which the first is element 8 n
    __device__ __forceinline__ void apply(unsigned long long n, float (&f)[8]) const {
        uint32_t c[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            c[b][0] = (uint32_t)(2 * n) + b;
            c[b][1] = (uint32_t)(n >> 31);
            c[b][2] = c[b][3] = 0;
        }
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            const uint32_t r0 = k0 + i * 0x9E3779B9u, r1 = k1 + i * 0xBB67AE85u;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const unsigned long long x = (unsigned long long)c[b][0] * 0xD2511F53u, y = (unsigned long long)c[b][2] * 0xCD9E8D57u;
                c[b][0] = (uint32_t)(y >> 32) ^ c[b][1] ^ r0;
                c[b][2] = (uint32_t)(x >> 32) ^ c[b][3] ^ r1;
                c[b][1] = (uint32_t)y;
                c[b][3] = (uint32_t)x;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = c[i / 4][i % 4] > below ? __fmul_rn(f[i], scale) : 0.f;
    }
};

// ---- eight adjacent elements of a row ------------------------------------------------------------------------------------
// A thread's elements are 8 n .. 8 n + 7 of the whole tensor, counted row-major: where rows lie back to back they are 16-byte pieces whatever the row's length, and
// they are two counters' words of dropout.  Of a row they are columns col .. col + 7, of which the row's first and last piece may have only a part.
template <bool F32> struct Raw { uint4 w[F32 ? 2 : 1]; };
__device__ __forceinline__ bool whole(int col, int D) { return col >= 0 && col + 8 <= D; }
template <bool F32> __device__ __forceinline__ void request(Raw<F32>& r, const void* base, long long row, int col, int D, bool vec) {
    if (vec && whole(col, D)) {
        const uint4* p = reinterpret_cast<const uint4*>((const unsigned char*)base + (row + col) * (F32 ? 4 : 2));
        r.w[0] = p[0];
        if (F32) r.w[F32] = p[1];
        return;
    }
    uint32_t w[F32 ? 8 : 4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (col + i >= 0 && col + i < D) {
            if (F32) w[F32 ? i : 0] = ((const uint32_t*)base)[row + col + i];
            else w[i / 2] |= (uint32_t)((const uint16_t*)base)[row + col + i] << (16 * (i & 1));
        }
    r.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
    if (F32) r.w[F32] = make_uint4(w[F32 ? 4 : 0], w[F32 ? 5 : 0], w[F32 ? 6 : 0], w[F32 ? 7 : 0]);
}
template <bool F32> __device__ __forceinline__ void floats(const Raw<F32>& r, float (&f)[8]) {
    if (F32) {
        const uint4 a = r.w[0], b = r.w[F32];
        f[0] = __uint_as_float(a.x); f[1] = __uint_as_float(a.y); f[2] = __uint_as_float(a.z); f[3] = __uint_as_float(a.w);
        f[4] = __uint_as_float(b.x); f[5] = __uint_as_float(b.y); f[6] = __uint_as_float(b.z); f[7] = __uint_as_float(b.w);
    } else {
        unpack8(r.w[0], f);
    }
}
__device__ __forceinline__ void store(void* base, bool f32, long long row, int col, int D, bool vec, const float (&f)[8]) {
    if (vec && whole(col, D)) {
        if (f32) {
            float4* p = reinterpret_cast<float4*>((float*)base + row + col);
            p[0] = make_float4(f[0], f[1], f[2], f[3]);
            p[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>((bf16*)base + row + col) = pack8(f);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (col + i >= 0 && col + i < D) {
            if (f32) ((float*)base)[row + col + i] = f[i];
            else ((bf16*)base)[row + col + i] = __float2bfloat16_rn(f[i]);
        }
}
// the weight's, ones without
__device__ __forceinline__ void weights(const void* w, bool f32, int col, int D, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = !w || col + i < 0 || col + i >= D ? 1.f : f32 ? ((const float*)w)[col + i] : __bfloat162float(((const bf16*)w)[col + i]);
}

// ---- a row in 8 bits -------------------------------------------------------------------------------------------------------
// top: the bits of max |y|, a NaN if there is one.  Rows without a magnitude above 2^-100 are zeros with scale 0, a row that holds a NaN or an infinity is
// zeros with a NaN for its scale: so are its products.
constexpr uint32_t TINY_BITS = (127 - 100) << 23, INF_BITS = 0x7f800000u;
__device__ __forceinline__ float max_abs(float top, float f) {  // (a NaN stays)
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(f)));
    return r;
}
// q = rint(v c), c = 127 / a rounded up.  Of bf16 rows that is rint(127 v / a), ties to even: with 8-bit mantissas 127 v / a is n + 1/2 either because v = +-a / 2, where c
// gives 63.5 or a little more and 64 is right; or because 127 divides a's mantissa, where c and v c are exact.  Quotients that are no ties are 2^-17 of their size
// away from one (the numerators differ by a whole step), v c is off by 2^-22.
struct Rounder {
    float c;
    uint32_t mask;
    __device__ __forceinline__ explicit Rounder(float top) {
        const bool live = top > __uint_as_float(TINY_BITS) && top < __uint_as_float(INF_BITS);
        c = live ? __fdiv_ru(127.f, top) : 0.f;
        mask = live ? ~0u : 0u;
    }
    __device__ __forceinline__ uint32_t four(float a, float b, float d, float e) const {
        const float M = 12582912.f;  // 1.5 * 2^23: the sum's low byte is the integer nearest to v c
        const uint32_t x = __float_as_uint(__fadd_rn(__fmul_rn(a, c), M)), y = __float_as_uint(__fadd_rn(__fmul_rn(b, c), M));
        const uint32_t z = __float_as_uint(__fadd_rn(__fmul_rn(d, c), M)), w = __float_as_uint(__fadd_rn(__fmul_rn(e, c), M));
        return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410) & mask;
    }
    __device__ __forceinline__ static float scale(float top, float times) {
        return !(top < __uint_as_float(INF_BITS)) ? __uint_as_float(0x7fc00000u) : top > __uint_as_float(TINY_BITS) ? __fdiv_rn(top * times, 127.f) : 0.f;
    }
};
__device__ __forceinline__ void store_int8(signed char* q, long long row, int col, int D, bool vec, const float (&f)[8], const Rounder& round) {
    const uint32_t w[2] = {round.four(f[0], f[1], f[2], f[3]), round.four(f[4], f[5], f[6], f[7])};
    if (vec && whole(col, D)) {
        *reinterpret_cast<uint2*>(q + row + col) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i >= 0 && col + i < D) q[row + col + i] = (signed char)(w[i / 4] >> (8 * (i & 3)));
    }
}

// ---- teams ---------------------------------------------------------------------------------------------------------------
// A team has a row: a power of two of a warp's threads, or whole warps of a CTA, which then has one row.
struct Teams {
    int threads, rows;  // of a team; of a CTA
};
constexpr int threads_most(int nv) { return nv == 1 ? 288 : nv == 2 ? 512 : 544; }  // (288, 544: rows of 2047 and 16383 elements have up to 257 and 2049 pieces)
// CTAs of so many threads that an SM's registers hold, forward and backward
constexpr int fwd_ctas(int nv) { return nv == 1 ? 4 : 1; }
constexpr int bwd_ctas(int nv) { return nv == 1 ? 2 : 1; }
constexpr int vectors_of(long long pieces) { return pieces <= threads_most(1) ? 1 : pieces <= 2 * threads_most(2) ? 2 : 4; }
constexpr long long pieces_of(long long D) { return D % 8 ? (D + 14) / 8 : D / 8; }
static_assert(pieces_of(NORM_MAX_D) <= 4 * threads_most(4) && pieces_of(NORM_MAX_D - 1) <= 4 * threads_most(4), "a thread has four pieces at most");
constexpr int MAX_WARPS = 32;
// Sum and maximum over a team, in everyone's registers.  room: two of them in turn, so that one barrier a row is enough: before a thread comes to
// write one again all have passed the other's barrier, and so have read this one.
struct Room { float sum[2][MAX_WARPS], top[2][MAX_WARPS]; };
template <bool SUM, bool TOP> __device__ __forceinline__ void reduce(int team, Room& room, int turn, float& sum, float& top) {
    for (int o = (team < 32 ? team : 32) / 2; o; o /= 2) {
        if (SUM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (TOP) top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (team <= 32) return;
    const int warps = team / 32, warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
        if (SUM) room.sum[turn][warp] = sum;
        if (TOP) room.top[turn][warp] = top;
    }
    __syncthreads();
    sum = 0.f;
    for (int i = 0; i < warps; ++i) {
        if (SUM) sum += room.sum[turn][i];
        if (TOP) top = max_abs(top, room.top[turn][i]);
    }
}
// The rows of a team are `step` apart, a multiple of 8 wherever a team has several and rows are no multiple of 8 long: their first pieces then all begin with the same
// column, 0 to -7, and a thread has the same columns of each.
__device__ __forceinline__ int first_col(long long row, int D) { return -(int)((row * D) & 7); }

// ---- forward ---------------------------------------------------------------------------------------------------------------
struct FwdKernelParams : NormFwdParams {
    Teams t;
    bool vec, vec_y;  // x, residual and h (y) by 16-byte pieces (8 bits: 8)
};
// RES: no residual, bf16, fp32.  Of rows that take four pieces a thread nothing is requested ahead and the weight is not held: registers.
template <int NV, bool XF, int RES, bool DROP, bool INT8> __global__ void __launch_bounds__(threads_most(NV), fwd_ctas(NV)) norm_fwd_kernel(const __grid_constant__ FwdKernelParams p) {
    constexpr bool HELD = NV < 4, RF = RES == 2;
    __shared__ Room room;
    stream_order();
    const int team = p.t.threads, lane = threadIdx.x % team;
    const long long step = (long long)gridDim.x * p.t.rows;
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const int col0 = first_col(row, p.D) + 8 * lane;
    float w[HELD ? NV : 1][8];
    Raw<XF> x[NV];
    Raw<RF> r[NV];
    auto ask = [&](long long m) {
        if (m >= p.M) return;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            request<XF>(x[v], p.x, m * p.ldx, col0 + 8 * team * v, p.D, p.vec);
            if (RES) request<RF>(r[v], p.residual, m * p.ldr, col0 + 8 * team * v, p.D, p.vec);
        }
    };
    if (HELD) {
        ask(row);
#pragma unroll
        for (int v = 0; v < NV; ++v) weights(p.weight, p.w_f32, col0 + 8 * team * v, p.D, w[v]);
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
            floats<XF>(x[v], f[v]);
            if (DROP) drop.apply((unsigned long long)(row * p.D + col) >> 3, f[v]);
            if (RES) {
                float g[8];
                floats<RF>(r[v], g);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] = __fadd_rn(g[i], f[v][i]);  // (not merged with dropout's product: what is kept is the same however it is called)
                if (!RF) unpack8(pack8(f[v]), f[v]);
                if (in) store(p.h, RF, row * p.ldh, col, p.D, p.vec, f[v]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(f[v][i], f[v][i], sum);
            if (INT8) {
                if (!HELD) weights(p.weight, p.w_f32, col, p.D, w[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    f[v][i] *= w[HELD ? v : 0][i];
                    top = max_abs(top, f[v][i]);
                }
            }
        }
        if (HELD) ask(row + step);
        reduce<true, INT8>(team, room, turn, sum, top);
        turn ^= 1;
        const float rstd = 1.f / sqrtf(sum / (float)p.D + p.eps);
        if (!in) continue;
        if (lane == 0) {
            if (p.rstd) p.rstd[row] = rstd;
            if (INT8) p.scale[row] = Rounder::scale(top, rstd);
        }
        if (INT8) {
            const Rounder round(top);
#pragma unroll
            for (int v = 0; v < NV; ++v) store_int8((signed char*)p.y, row * p.ldy, col0 + 8 * team * v, p.D, p.vec_y, f[v], round);
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (!HELD) weights(p.weight, p.w_f32, col0 + 8 * team * v, p.D, w[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] = f[v][i] * w[HELD ? v : 0][i] * rstd;
                store(p.y, p.y_f32, row * p.ldy, col0 + 8 * team * v, p.D, p.vec_y, f[v]);
            }
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------
struct BwdKernelParams : NormBwdParams {
    Teams t;
    bool vec;
};
template <int NV, bool YF, bool HF, bool DROP> __global__ void __launch_bounds__(threads_most(NV), bwd_ctas(NV)) norm_bwd_kernel(const __grid_constant__ BwdKernelParams p) {
    constexpr bool HELD = NV < 4;
    __shared__ Room room;
    extern __shared__ float sums[];  // [rows of a CTA][D], where it has several
    stream_order();
    const int team = p.t.threads, lane = threadIdx.x % team;
    const long long step = (long long)gridDim.x * p.t.rows;
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const int col0 = first_col(row, p.D) + 8 * lane;
    float w[HELD ? NV : 1][8], dw[NV][8];
    Raw<HF> h[NV], dh[NV];
    Raw<YF> dy[NV];
    float rstd_next = 0.f;
    auto ask = [&](long long m) {
        if (m >= p.M) return;
        rstd_next = p.rstd[m];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            request<HF>(h[v], p.h, m * p.ldh, col0 + 8 * team * v, p.D, p.vec);
            request<YF>(dy[v], p.dy, m * p.lddy, col0 + 8 * team * v, p.D, p.vec);
            if (p.dh) request<HF>(dh[v], p.dh, m * p.lddh, col0 + 8 * team * v, p.D, p.vec);
        }
    };
    if (HELD) ask(row);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if (HELD) weights(p.weight, p.w_f32, col0 + 8 * team * v, p.D, w[v]);
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
            h_now[v] = h[v]; dy_now[v] = dy[v]; dh_now[v] = dh[v];
            floats<HF>(h_now[v], f);
            floats<YF>(dy_now[v], g);
            if (!HELD) weights(p.weight, p.w_f32, col0 + 8 * team * v, p.D, w[0]);
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
        const float c = sum / (float)p.D * rstd * rstd;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = col0 + 8 * team * v;
            float f[8], g[8], d[8];
            floats<HF>(h_now[v], f);
            floats<YF>(dy_now[v], g);
            if (!HELD) weights(p.weight, p.w_f32, col, p.D, w[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = rstd * fmaf(-c, f[i], g[i] * w[HELD ? v : 0][i]);
            if (p.dh) {
                float e[8];
                floats<HF>(dh_now[v], e);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] += e[i];
            }
            if (p.dr) store(p.dr, HF, row * p.lddr, col, p.D, p.vec, d);
            if (p.dx) {
                if (DROP) drop.apply((unsigned long long)(row * p.D + col) >> 3, d);
                store(p.dx, p.x_f32, row * p.lddx, col, p.D, p.vec, d);
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
            if (col >= 0 && col < p.D) mine[col] = dw[v][i];
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

// ---- rows to 8 bits --------------------------------------------------------------------------------------------------------
struct QuantizeKernelParams : QuantizeParams {
    Teams t;
    bool vec, vec_q;
};
// NV 0: rows of any length, read twice
template <int NV, bool XF> __global__ void __launch_bounds__(NV ? threads_most(NV) : 1024) quantize_kernel(const __grid_constant__ QuantizeKernelParams p) {
    __shared__ Room room;
    stream_order();
    constexpr int HELD = NV ? NV : 1;
    const int team = p.t.threads, lane = threadIdx.x % team, K = (int)p.K;
    const long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const bool in = row < p.M;
    const int col0 = first_col(row, K) + 8 * lane;
    const int vectors = NV ? NV : (int)((p.K + 7 + 8LL * team - 1) / (8LL * team));
    Raw<XF> x[HELD];
    float none = 0.f, top = 0.f;
    auto tops = [&](const Raw<XF>& r) {
        float f[8];
        floats<XF>(r, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max_abs(top, f[i]);
    };
    if (NV) {
#pragma unroll
        for (int v = 0; v < HELD; ++v) {
            x[v] = Raw<XF>{};
            if (in) request<XF>(x[v], p.x, row * p.ldx, col0 + 8 * team * v, K, p.vec);
        }
#pragma unroll
        for (int v = 0; v < HELD; ++v) tops(x[v]);
    } else {
#pragma unroll 4
        for (int v = 0; v < vectors; ++v) {
            const long long col = col0 + 8LL * team * v;
            Raw<XF> r{};
            if (in && col < K) request<XF>(r, p.x, row * p.ldx, (int)col, K, p.vec);
            tops(r);
        }
    }
    reduce<false, true>(team, room, 0, none, top);
    if (!in) return;
    if (lane == 0) p.scale[row] = Rounder::scale(top, 1.f);
    const Rounder round(top);
#pragma unroll
    for (int v = 0; v < vectors; ++v) {
        const long long col = col0 + 8LL * team * v;
        if (col >= K) break;
        if (!NV) request<XF>(x[0], p.x, row * p.ldx, (int)col, K, p.vec);
        float f[8];
        floats<XF>(x[NV ? v : 0], f);
        store_int8(p.q, row * p.ldq, (int)col, K, p.vec_q, f, round);
    }
}

// ---- dropout alone ---------------------------------------------------------------------------------------------------------
template <bool XF, int RES> __global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
    constexpr bool RF = RES == 2;
    stream_order();
    const Dropper drop(p.d);
    const long long step = (long long)gridDim.x * 256 * 8;
    for (long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; at < p.n; at += step) {
        const int live = (int)(p.n - at < 8 ? p.n - at : 8);
        Raw<XF> x;
        Raw<RF> r;
        request<XF>(x, p.x, at, 0, live, true);
        if (RES) request<RF>(r, p.residual, at, 0, live, true);
        float f[8];
        floats<XF>(x, f);
        if (p.d.threshold) drop.apply(at >> 3, f);
        if (RES) {
            float g[8];
            floats<RF>(r, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __fadd_rn(g[i], f[i]);
        }
        store(p.y, p.y_f32, at, 0, live, true, f);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
static bool al(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// whether a tensor's pieces of eight elements lie on boundaries of `bytes`
static bool pieces_lie(const void* p, long long M, long long D, long long ld, int bytes) { return !p || (al(p, bytes) && (M == 1 || ld == D || (D % 8 == 0 && ld % 8 == 0))); }
// teams for rows of D elements, nv pieces to a thread, CTAs of some 256 threads
static Teams teams_of(long long D, int nv) {
    const long long need = (pieces_of(D) + nv - 1) / nv;
    int team = 1;
    if (need <= 32) while (team < need) team *= 2;
    else team = (int)((need + 31) / 32 * 32);
    return Teams{team, team > 32 ? 1 : 256 / team};
}
// CTAs for M rows: as many as SMs hold, and a multiple of 8 where a team has several rows (see first_col)
static long long ctas_of(long long M, const Teams& t, int sms, int threads) {
    const int per_sm = threads / (t.threads * t.rows);
    const long long want = (M + t.rows - 1) / t.rows, most = (long long)sms * (per_sm < 1 ? 1 : per_sm) / 8 * 8;
    return want < most || most == 0 ? want : most;
}
}  // namespace norm

int launch_norm_fwd(const NormFwdParams& a, cudaStream_t stream) {
    using namespace norm;
    FwdKernelParams p;
    static_cast<NormFwdParams&>(p) = a;
    const int nv = vectors_of(pieces_of(p.D));
    p.t = teams_of(p.D, nv);
    const bool int8 = p.scale != nullptr, drop = p.d.threshold != 0;
    p.vec = pieces_lie(p.x, p.M, p.D, p.ldx, 16) && pieces_lie(p.residual, p.M, p.D, p.ldr, 16) && pieces_lie(p.h, p.M, p.D, p.ldh, 16);
    p.vec_y = pieces_lie(p.y, p.M, p.D, p.ldy, int8 ? 8 : 16);
#define WKV7_OUT(nv, xf, res, drop) {norm_fwd_kernel<nv, xf, res, drop, false>, norm_fwd_kernel<nv, xf, res, drop, true>}
#define WKV7_RES(nv, xf) {{WKV7_OUT(nv, xf, 0, false), WKV7_OUT(nv, xf, 0, false)}, {WKV7_OUT(nv, xf, 1, false), WKV7_OUT(nv, xf, 1, true)}, {WKV7_OUT(nv, xf, 2, false), WKV7_OUT(nv, xf, 2, true)}}
    static void (*const kernels[3][2][3][2][2])(FwdKernelParams) = {{WKV7_RES(1, false), WKV7_RES(1, true)}, {WKV7_RES(2, false), WKV7_RES(2, true)}, {WKV7_RES(4, false), WKV7_RES(4, true)}};
#undef WKV7_RES
#undef WKV7_OUT
    const auto kern = kernels[nv / 2][p.x_f32][p.residual ? 1 + p.r_f32 : 0][drop][int8];
    return launch(kern, dim3((unsigned)ctas_of(p.M, p.t, sm_count(), nv == 1 ? 1024 : threads_most(nv))), p.t.threads * p.t.rows, 0, stream, p) ? kOk : kLaunchFailed;
}

// The parts of dw: CTAs of the backward.  Sizes alone decide their number, so that the sums are the same on every device.
int norm_bwd_partials(long long M, long long D) {
    using namespace norm;
    const int nv = vectors_of(pieces_of(D));
    return (int)ctas_of(M, teams_of(D, nv), 148, nv == 1 ? 768 : threads_most(nv));
}

int launch_norm_bwd(const NormBwdParams& a, cudaStream_t stream) {
    using namespace norm;
    BwdKernelParams p;
    static_cast<NormBwdParams&>(p) = a;
    const int nv = vectors_of(pieces_of(p.D)), parts = norm_bwd_partials(p.M, p.D);
    p.t = teams_of(p.D, nv);
    p.vec = pieces_lie(p.h, p.M, p.D, p.ldh, 16) && pieces_lie(p.dy, p.M, p.D, p.lddy, 16) && pieces_lie(p.dh, p.M, p.D, p.lddh, 16) && pieces_lie(p.dx, p.M, p.D, p.lddx, 16) &&
            pieces_lie(p.dr, p.M, p.D, p.lddr, 16);
#define WKV7_DROP(nv, yf, hf) {norm_bwd_kernel<nv, yf, hf, false>, norm_bwd_kernel<nv, yf, hf, true>}
#define WKV7_TYPES(nv) {{WKV7_DROP(nv, false, false), WKV7_DROP(nv, false, true)}, {WKV7_DROP(nv, true, false), WKV7_DROP(nv, true, true)}}
    static void (*const kernels[3][2][2][2])(BwdKernelParams) = {WKV7_TYPES(1), WKV7_TYPES(2), WKV7_TYPES(4)};
#undef WKV7_TYPES
#undef WKV7_DROP
    const auto kern = kernels[nv / 2][p.y_f32][p.h_f32][p.d.threshold && p.dx];
    const int smem = p.dw && p.t.rows > 1 ? p.t.rows * p.D * 4 : 0;  // (rows x D <= 256 threads x 8 elements)
    if (!launch(kern, dim3((unsigned)parts), p.t.threads * p.t.rows, smem, stream, p)) return kLaunchFailed;
    if (p.dw && !launch(norm_dw_kernel, dim3((unsigned)((p.D + 31) / 32)), 1024, 0, stream, (const float*)p.partial, p.dw, p.D, parts)) return kLaunchFailed;
    return kOk;
}

int launch_quantize(const QuantizeParams& a, cudaStream_t stream) {
    using namespace norm;
    QuantizeKernelParams p;
    static_cast<QuantizeParams&>(p) = a;
    const long long pieces = pieces_of(p.K);
    const int nv = pieces > 4 * threads_most(4) ? 0 : vectors_of(pieces);
    p.t = nv ? teams_of(p.K, nv) : Teams{1024, 1};
    p.vec = pieces_lie(p.x, p.M, p.K, p.ldx, 16);
    p.vec_q = pieces_lie(p.q, p.M, p.K, p.ldq, 8);
    const long long grid = (p.M + p.t.rows - 1) / p.t.rows;
    if (grid > 0x7fffffffLL) return kTooLarge;
    static void (*const kernels[4][2])(QuantizeKernelParams) = {{quantize_kernel<0, false>, quantize_kernel<0, true>}, {quantize_kernel<1, false>, quantize_kernel<1, true>},
                                                                {quantize_kernel<2, false>, quantize_kernel<2, true>}, {quantize_kernel<4, false>, quantize_kernel<4, true>}};
    return launch(kernels[nv == 4 ? 3 : nv][p.x_f32], dim3((unsigned)grid), p.t.threads * p.t.rows, 0, stream, p) ? kOk : kLaunchFailed;
}

int launch_dropout(const DropoutParams& p, cudaStream_t stream) {
    using namespace norm;
    static void (*const kernels[2][3])(DropoutParams) = {{dropout_kernel<false, 0>, dropout_kernel<false, 1>, dropout_kernel<false, 2>},
                                                         {dropout_kernel<true, 0>, dropout_kernel<true, 1>, dropout_kernel<true, 2>}};
    const long long want = (p.n + 2047) / 2048, most = (long long)sm_count() * 8;
    return launch(kernels[p.x_f32][p.residual ? 1 + p.r_f32 : 0], dim3((unsigned)(want < most ? want : most)), 256, 0, stream, p) ? kOk : kLaunchFailed;
}

}  // namespace wkv7

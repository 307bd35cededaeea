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
struct Words4 { uint32_t w[4]; };
__device__ __forceinline__ Words4 philox(unsigned long long block, uint32_t k0, uint32_t k1) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = 0, c3 = 0;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Words4{{c0, c1, c2, c3}};
}
struct Dropper {
    uint32_t k0, k1, below;  // kept: word > below (the threshold less one; 2^32 less one drops all)
    float scale;
    __device__ __forceinline__ explicit Dropper(const Dropout& d) : below((uint32_t)(d.threshold - 1)), scale(d.scale) {
        const unsigned long long s = d.where ? *d.where : d.seed;
        k0 = (uint32_t)s;
        k1 = (uint32_t)(s >> 32);
    }
    // eight adjacent elements, of which the first is element `at`
    __device__ __forceinline__ void apply(unsigned long long at, float (&f)[8]) const {
        const Words4 a = philox(at >> 2, k0, k1), b = philox((at >> 2) + 1, k0, k1);
        const int off = (int)(at & 3);
        if (off == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[i] = a.w[i] > below ? __fmul_rn(f[i], scale) : 0.f;
                f[4 + i] = b.w[i] > below ? __fmul_rn(f[4 + i], scale) : 0.f;
            }
        } else {  // (rows whose length is no multiple of four)
            const Words4 c = philox((at >> 2) + 2, k0, k1);
            const uint32_t w[12] = {a.w[0], a.w[1], a.w[2], a.w[3], b.w[0], b.w[1], b.w[2], b.w[3], c.w[0], c.w[1], c.w[2], c.w[3]};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t word = off == 1 ? w[i + 1] : off == 2 ? w[i + 2] : w[i + 3];
                f[i] = word > below ? __fmul_rn(f[i], scale) : 0.f;
            }
        }
    }
};

// ---- eight adjacent elements of a row ------------------------------------------------------------------------------------
struct Raw8 { uint4 lo, hi; };  // bf16: lo alone
__device__ __forceinline__ float load1(const void* base, bool f32, long long at) { return f32 ? ((const float*)base)[at] : __bfloat162float(((const bf16*)base)[at]); }
// live: how many of them there are (0 to 8); the others are zero.  vec: they start on a 16-byte boundary where all eight are there
__device__ __forceinline__ Raw8 request(const void* base, bool f32, long long at, int live, bool vec) {
    Raw8 r;
    r.lo = r.hi = make_uint4(0, 0, 0, 0);
    if (vec && live == 8) {
        const uint4* p = reinterpret_cast<const uint4*>((const unsigned char*)base + at * (f32 ? 4 : 2));
        r.lo = p[0];
        if (f32) r.hi = p[1];
    } else if (f32) {
        uint32_t* w[8] = {&r.lo.x, &r.lo.y, &r.lo.z, &r.lo.w, &r.hi.x, &r.hi.y, &r.hi.z, &r.hi.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live) *w[i] = ((const uint32_t*)base)[at + i];
    } else {
        uint32_t* w[4] = {&r.lo.x, &r.lo.y, &r.lo.z, &r.lo.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live) *w[i / 2] |= (uint32_t)((const uint16_t*)base)[at + i] << (16 * (i & 1));
    }
    return r;
}
__device__ __forceinline__ void floats(const Raw8& r, bool f32, float (&f)[8]) {
    if (f32) {
        f[0] = __uint_as_float(r.lo.x); f[1] = __uint_as_float(r.lo.y); f[2] = __uint_as_float(r.lo.z); f[3] = __uint_as_float(r.lo.w);
        f[4] = __uint_as_float(r.hi.x); f[5] = __uint_as_float(r.hi.y); f[6] = __uint_as_float(r.hi.z); f[7] = __uint_as_float(r.hi.w);
    } else {
        unpack8(r.lo, f);
    }
}
__device__ __forceinline__ void store(void* base, bool f32, long long at, int live, bool vec, const float (&f)[8]) {
    if (vec && live == 8) {
        if (f32) {
            float4* p = reinterpret_cast<float4*>((float*)base + at);
            p[0] = make_float4(f[0], f[1], f[2], f[3]);
            p[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>((bf16*)base + at) = pack8(f);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live) {
                if (f32) ((float*)base)[at + i] = f[i];
                else ((bf16*)base)[at + i] = __float2bfloat16_rn(f[i]);
            }
    }
}
__device__ __forceinline__ int live_of(long long n, long long at) { return at >= n ? 0 : n - at < 8 ? (int)(n - at) : 8; }

// ---- a row in 8 bits -------------------------------------------------------------------------------------------------------
// top: the bits of max |y|, compared as integers, so that NaN is above infinity and neither is lost.  Rows without a magnitude above 2^-100 are zeros with scale
// 0, a row that holds a NaN or an infinity is zeros with a NaN for its scale: so are its products.
constexpr uint32_t TINY_BITS = (127 - 100) << 23, INF_BITS = 0x7f800000u;
struct Rounder {
    float two, a, inv;  // the power of two that brings the maximum to [1, 4), the maximum so brought, its inverse
    bool live;
    __device__ __forceinline__ explicit Rounder(uint32_t top) : live(top > TINY_BITS && top < INF_BITS) {
        const uint32_t e = live ? top >> 23 : 127;
        two = __uint_as_float((e >= 254 ? 1u : 254u - e) << 23);
        a = live ? __uint_as_float(top) * two : 1.f;
        inv = 1.f / a;
    }
    // rint(127 v / a), ties to even.  bf16 rows have ties, 127 v = (n + 1/2) a, and the rounding of 1 / a must not decide them: the remainder 127 v - n a does, which
    // is exact (15 bits less 15 bits)
    __device__ __forceinline__ int operator()(float v) const {
        const float t = 127.f * (v * two);
        float n = rintf(t * inv);
        const float twice = 2.f * fmaf(-n, a, t);
        if (fabsf(twice) > a || (fabsf(twice) == a && ((int)n & 1))) n += copysignf(1.f, twice);
        return live ? (int)n : 0;
    }
    __device__ __forceinline__ static float scale(uint32_t top, float times) {
        return top >= INF_BITS ? __uint_as_float(0x7fc00000u) : top > TINY_BITS ? __fdiv_rn(__uint_as_float(top) * times, 127.f) : 0.f;
    }
};
__device__ __forceinline__ uint32_t top_of(uint32_t top, const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    return top;
}
__device__ __forceinline__ void store_int8(signed char* q, long long at, int live, bool vec, const float (&f)[8], const Rounder& round) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i / 4] |= (uint32_t)(round(f[i]) & 255) << (8 * (i & 3));
    if (vec && live == 8) {
        *reinterpret_cast<uint2*>(q + at) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live) q[at + i] = (signed char)(w[i / 4] >> (8 * (i & 3)));
    }
}

// ---- teams ---------------------------------------------------------------------------------------------------------------
// A team has a row: a power of two of a warp's threads, or whole warps of a CTA, which then has one row.
struct Teams {
    int threads, rows;  // of a team; of a CTA
};
constexpr int vectors_of(long long D) { return D <= 2048 ? 1 : D <= 8192 ? 2 : 4; }
constexpr int threads_most(int nv) { return nv == 1 ? 256 : 512; }
constexpr int per_sm(int nv) { return nv == 1 ? 4 : nv == 2 ? 2 : 1; }  // CTAs of the persistent kernels
static_assert(NORM_MAX_D <= 8 * 4 * threads_most(4), "a thread has four vectors at most");
constexpr int MAX_WARPS = 32;
// Sum and maximum over a team, in everyone's registers.  room: two of them in turn, so that one barrier a row is enough: before a thread comes to
// write one again all have passed the other's barrier, and so have read this one.
struct Room { float sum[2][MAX_WARPS]; uint32_t top[2][MAX_WARPS]; };
template <bool TOP> __device__ __forceinline__ void reduce(int team, Room& room, int turn, float& sum, uint32_t& top) {
    for (int o = (team < 32 ? team : 32) / 2; o; o /= 2) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (TOP) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (team <= 32) return;
    const int warps = team / 32, warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
        room.sum[turn][warp] = sum;
        if (TOP) room.top[turn][warp] = top;
    }
    __syncthreads();
    sum = 0.f;
    for (int i = 0; i < warps; ++i) {
        sum += room.sum[turn][i];
        if (TOP) top = max(top, room.top[turn][i]);
    }
}

// ---- forward ---------------------------------------------------------------------------------------------------------------
struct FwdKernelParams : NormFwdParams {
    Teams t;
    bool vec;  // rows start on 16-byte boundaries (q: 8)
};
template <int NV, bool DROP, bool INT8> __global__ void __launch_bounds__(threads_most(NV), per_sm(NV)) norm_fwd_kernel(const __grid_constant__ FwdKernelParams p) {
    __shared__ Room room;
    stream_order();
    const int team = p.t.threads, lane = threadIdx.x % team;
    const long long step = (long long)gridDim.x * p.t.rows;
    float w[NV][8];
    int live[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int col = 8 * (lane + team * v);
        live[v] = live_of(p.D, col);
        if (p.weight) floats(request(p.weight, p.w_f32, col, live[v], p.vec), p.w_f32, w[v]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) w[v][i] = 1.f;
    }
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    Raw8 x[NV], r[NV];
    auto ask = [&](long long m) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = 8 * (lane + team * v), n = m < p.M ? live[v] : 0;
            x[v] = request(p.x, p.x_f32, m * p.ldx + col, n, p.vec);
            if (p.residual) r[v] = request(p.residual, p.r_f32, m * p.ldr + col, n, p.vec);
        }
    };
    ask(row);
    const Dropper drop(p.d);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * p.t.rows; first < p.M; first += step, row += step) {  // (the same for all threads: there are barriers within)
        const bool in = row < p.M;
        float f[NV][8], sum = 0.f;
        uint32_t top = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = 8 * (lane + team * v);
            floats(x[v], p.x_f32, f[v]);
            if (DROP) drop.apply((unsigned long long)row * p.D + col, f[v]);
            if (p.residual) {
                float g[8];
                floats(r[v], p.r_f32, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] = __fadd_rn(g[i], f[v][i]);  // (not merged with dropout's product: what is kept is the same however it is called)
                if (!p.r_f32) unpack8(pack8(f[v]), f[v]);
                if (in) store(p.h, p.r_f32, row * p.ldh + col, live[v], p.vec, f[v]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(f[v][i], f[v][i], sum);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[v][i] *= w[v][i];
            if (INT8) top = top_of(top, f[v]);
        }
        ask(row + step);
        reduce<INT8>(team, room, turn, sum, top);
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
            for (int v = 0; v < NV; ++v) store_int8((signed char*)p.y, row * p.ldy + 8 * (lane + team * v), live[v], p.vec, f[v], round);
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= rstd;
                store(p.y, p.y_f32, row * p.ldy + 8 * (lane + team * v), live[v], p.vec, f[v]);
            }
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------
struct BwdKernelParams : NormBwdParams {
    Teams t;
    bool vec;
};
template <int NV, bool DROP> __global__ void __launch_bounds__(threads_most(NV), per_sm(NV)) norm_bwd_kernel(const __grid_constant__ BwdKernelParams p) {
    __shared__ Room room;
    extern __shared__ float sums[];  // [rows of a CTA][D], where it has several
    stream_order();
    const int team = p.t.threads, lane = threadIdx.x % team;
    const long long step = (long long)gridDim.x * p.t.rows;
    float w[NV][8], dw[NV][8];
    int live[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int col = 8 * (lane + team * v);
        live[v] = live_of(p.D, col);
        if (p.weight) floats(request(p.weight, p.w_f32, col, live[v], p.vec), p.w_f32, w[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!p.weight) w[v][i] = 1.f;
            dw[v][i] = 0.f;
        }
    }
    long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    Raw8 h[NV], dy[NV], dh[NV];
    float rstd_next = 0.f;
    auto ask = [&](long long m) {
        if (m < p.M) rstd_next = p.rstd[m];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = 8 * (lane + team * v), n = m < p.M ? live[v] : 0;
            h[v] = request(p.h, p.h_f32, m * p.ldh + col, n, p.vec);
            dy[v] = request(p.dy, p.y_f32, m * p.lddy + col, n, p.vec);
            if (p.dh) dh[v] = request(p.dh, p.h_f32, m * p.lddh + col, n, p.vec);
        }
    };
    ask(row);
    const Dropper drop(p.d);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * p.t.rows; first < p.M; first += step, row += step) {
        const bool in = row < p.M;
        const float rstd = rstd_next;
        float f[NV][8], g[NV][8], sum = 0.f;
        Raw8 more[NV];
        uint32_t none = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            floats(h[v], p.h_f32, f[v]);
            floats(dy[v], p.y_f32, g[v]);
            more[v] = dh[v];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (in) dw[v][i] = fmaf(g[v][i], f[v][i] * rstd, dw[v][i]);
                g[v][i] *= w[v][i];
                sum = fmaf(g[v][i], f[v][i], sum);
            }
        }
        ask(row + step);
        reduce<false>(team, room, turn, sum, none);
        turn ^= 1;
        if (!in) continue;
        const float c = sum / (float)p.D * rstd * rstd;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int col = 8 * (lane + team * v);
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = rstd * fmaf(-c, f[v][i], g[v][i]);
            if (p.dh) {
                float e[8];
                floats(more[v], p.h_f32, e);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] += e[i];
            }
            if (p.dr) store(p.dr, p.h_f32, row * p.lddr + col, live[v], p.vec, d);
            if (p.dx) {
                if (DROP) drop.apply((unsigned long long)row * p.D + col, d);
                store(p.dx, p.x_f32, row * p.lddx + col, live[v], p.vec, d);
            }
        }
    }
    if (!p.dw) return;
    float* const out = p.partial + (long long)blockIdx.x * p.D;
    if (p.t.rows == 1) {
#pragma unroll
        for (int v = 0; v < NV; ++v) store(out, true, 8 * (lane + team * v), live[v], p.D % 4 == 0, dw[v]);
        return;
    }
    float* mine = sums + (threadIdx.x / team) * p.D;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live[v]) mine[8 * (lane + team * v) + i] = dw[v][i];
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
    bool vec;
};
// NV 0: rows of any length, read twice
template <int NV> __global__ void __launch_bounds__(NV ? threads_most(NV) : 1024) quantize_kernel(const __grid_constant__ QuantizeKernelParams p) {
    __shared__ Room room;
    stream_order();
    constexpr int HELD = NV ? NV : 1;
    const int team = p.t.threads, lane = threadIdx.x % team;
    const long long row = (long long)blockIdx.x * p.t.rows + threadIdx.x / team;
    const bool in = row < p.M;
    const int vectors = NV ? NV : (int)((p.K + 8LL * team - 1) / (8LL * team));
    float f[HELD][8], none = 0.f;
    uint32_t top = 0;
    auto get = [&](int v, float (&to)[8]) {
        const long long col = 8LL * (lane + (long long)team * v);
        floats(request(p.x, p.x_f32, row * p.ldx + col, in ? live_of(p.K, col) : 0, p.vec), p.x_f32, to);
    };
    if (NV) {
        Raw8 x[HELD];
#pragma unroll
        for (int v = 0; v < HELD; ++v) {
            const long long col = 8LL * (lane + (long long)team * v);
            x[v] = request(p.x, p.x_f32, row * p.ldx + col, in ? live_of(p.K, col) : 0, p.vec);
        }
#pragma unroll
        for (int v = 0; v < HELD; ++v) {
            floats(x[v], p.x_f32, f[v]);
            top = top_of(top, f[v]);
        }
    } else {
#pragma unroll 4
        for (int v = 0; v < vectors; ++v) {
            get(v, f[0]);
            top = top_of(top, f[0]);
        }
    }
    reduce<true>(team, room, 0, none, top);
    if (!in) return;
    if (lane == 0) p.scale[row] = Rounder::scale(top, 1.f);
    const Rounder round(top);
#pragma unroll
    for (int v = 0; v < vectors; ++v) {
        const long long col = 8LL * (lane + (long long)team * v);
        if (!NV) get(v, f[0]);
        store_int8(p.q, row * p.ldq + col, live_of(p.K, col), p.vec, f[NV ? v : 0], round);
    }
}

// ---- dropout alone ---------------------------------------------------------------------------------------------------------
template <bool RES> __global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
    stream_order();
    const Dropper drop(p.d);
    const long long step = (long long)gridDim.x * 256 * 8;
    for (long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; at < p.n; at += step) {
        const int live = live_of(p.n, at);
        const Raw8 x = request(p.x, p.x_f32, at, live, true);
        Raw8 r;
        if (RES) r = request(p.residual, p.r_f32, at, live, true);
        float f[8];
        floats(x, p.x_f32, f);
        if (p.d.threshold) drop.apply(at, f);
        if (RES) {
            float g[8];
            floats(r, p.r_f32, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __fadd_rn(g[i], f[i]);
        }
        store(p.y, p.y_f32, at, live, true, f);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
static bool al(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// teams for rows of D elements, nv vectors of eight to a thread, CTAs of about 256 threads
static Teams teams_of(long long D, int nv) {
    const long long need = (D + 8 * nv - 1) / (8 * nv);
    int team = 1;
    if (need <= 32) while (team < need) team *= 2;
    else team = (int)((need + 31) / 32 * 32);
    return Teams{team, team >= 256 || team > 32 ? 1 : 256 / team};
}
// CTAs that fill the device where `per` of the largest fit an SM
static long long places(int sms, int per, int most, const Teams& t) { return (long long)sms * per * (most / (t.threads * t.rows)); }
}  // namespace norm

int launch_norm_fwd(const NormFwdParams& a, cudaStream_t stream) {
    using namespace norm;
    FwdKernelParams p;
    static_cast<NormFwdParams&>(p) = a;
    const int nv = vectors_of(p.D);
    p.t = teams_of(p.D, nv);
    const bool int8 = p.scale != nullptr, drop = p.d.threshold != 0;
    const auto ok = [&](const void* q, long long ld) { return !q || (al(q, 16) && (p.M == 1 || ld % 8 == 0)); };
    p.vec = ok(p.x, p.ldx) && ok(p.residual, p.ldr) && ok(p.h, p.ldh) && ok(p.weight, 0) && (int8 ? al(p.y, 8) && (p.M == 1 || p.ldy % 8 == 0) : ok(p.y, p.ldy));
#define WKV7_FWD(nv) {{norm_fwd_kernel<nv, false, false>, norm_fwd_kernel<nv, false, true>}, {norm_fwd_kernel<nv, true, false>, norm_fwd_kernel<nv, true, true>}}
    static void (*const kernels[3][2][2])(FwdKernelParams) = {WKV7_FWD(1), WKV7_FWD(2), WKV7_FWD(4)};
#undef WKV7_FWD
    const auto kern = kernels[nv / 2][drop][int8];
    const int threads = p.t.threads * p.t.rows;
    const long long want = (p.M + p.t.rows - 1) / p.t.rows, most = places(sm_count(), per_sm(nv), threads_most(nv), p.t);
    return launch(kern, dim3((unsigned)(want < most ? want : most)), threads, 0, stream, p) ? kOk : kLaunchFailed;
}

// The parts of dw: CTAs of the backward.  Sizes alone decide their number, so that the sums are the same on every device.
int norm_bwd_partials(long long M, long long D) {
    using namespace norm;
    const int nv = vectors_of(D);
    const Teams t = teams_of(D, nv);
    const long long want = (M + t.rows - 1) / t.rows, most = places(148, per_sm(nv), threads_most(nv), t);
    return (int)(want < most ? want : most);
}

int launch_norm_bwd(const NormBwdParams& a, cudaStream_t stream) {
    using namespace norm;
    BwdKernelParams p;
    static_cast<NormBwdParams&>(p) = a;
    const int nv = vectors_of(p.D), parts = norm_bwd_partials(p.M, p.D);
    p.t = teams_of(p.D, nv);
    const auto ok = [&](const void* q, long long ld) { return !q || (al(q, 16) && (p.M == 1 || ld % 8 == 0)); };
    p.vec = ok(p.h, p.ldh) && ok(p.dy, p.lddy) && ok(p.dh, p.lddh) && ok(p.dx, p.lddx) && ok(p.dr, p.lddr) && ok(p.weight, 0);
    static void (*const kernels[3][2])(BwdKernelParams) = {{norm_bwd_kernel<1, false>, norm_bwd_kernel<1, true>}, {norm_bwd_kernel<2, false>, norm_bwd_kernel<2, true>},
                                                           {norm_bwd_kernel<4, false>, norm_bwd_kernel<4, true>}};
    const auto kern = kernels[nv / 2][p.d.threshold && p.dx];
    const int smem = p.dw && p.t.rows > 1 ? p.t.rows * p.D * 4 : 0;  // (rows x D <= 256 threads x 8 elements)
    if (!launch(kern, dim3((unsigned)parts), p.t.threads * p.t.rows, smem, stream, p)) return kLaunchFailed;
    if (p.dw && !launch(norm_dw_kernel, dim3((unsigned)((p.D + 31) / 32)), 1024, 0, stream, (const float*)p.partial, p.dw, p.D, parts)) return kLaunchFailed;
    return kOk;
}

int launch_quantize(const QuantizeParams& a, cudaStream_t stream) {
    using namespace norm;
    QuantizeKernelParams p;
    static_cast<QuantizeParams&>(p) = a;
    const int nv = p.K > NORM_MAX_D ? 0 : vectors_of(p.K);
    p.t = nv ? teams_of(p.K, nv) : Teams{1024, 1};
    p.vec = al(p.x, 16) && al(p.q, 8) && (p.M == 1 || (p.ldx % 8 == 0 && p.ldq % 8 == 0));
    const long long grid = (p.M + p.t.rows - 1) / p.t.rows;
    if (grid > 0x7fffffffLL) return kTooLarge;
    const auto kern = nv == 0 ? quantize_kernel<0> : nv == 1 ? quantize_kernel<1> : nv == 2 ? quantize_kernel<2> : quantize_kernel<4>;
    return launch(kern, dim3((unsigned)grid), p.t.threads * p.t.rows, 0, stream, p) ? kOk : kLaunchFailed;
}

int launch_dropout(const DropoutParams& p, cudaStream_t stream) {
    using namespace norm;
    const auto kern = p.residual ? dropout_kernel<true> : dropout_kernel<false>;
    const long long want = (p.n + 2047) / 2048, most = (long long)sm_count() * 8;
    return launch(kern, dim3((unsigned)(want < most ? want : most)), 256, 0, stream, p) ? kOk : kLaunchFailed;
}

}  // namespace wkv7

// What the kernels of the residual stream share: dropout's generator, rows by pieces of eight elements, rows in 8 bits, teams of threads.
#pragma once
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
// they are two counters' words of dropout.  Of a row they are columns col .. col + 7, of which the row's first and last piece may have only a part: it is read whole, where
// the tensor has it whole, and the rest is put to zero.  What is not read so, a tensor's last part of a piece and layouts without such pieces, is read element by
// element where it is used, not where it is requested: a request is a load and nothing else, which nothing waits for.
// EVEN: all tensors lie in pieces and rows are a multiple of 8 long, so that there are no parts.
template <bool F32> struct Raw { uint4 w[F32 ? 2 : 1]; };
struct Lie {   // how a tensor's pieces lie
    long long ld, end;  // elements from row to row; behind the last one; 0: by single elements
};
__device__ __forceinline__ bool whole(int col, int D) { return col >= 0 && col + 8 <= D; }
__device__ __forceinline__ bool any(int col, int D) { return col > -8 && col < D; }
template <bool F32, bool EVEN> __device__ __forceinline__ void request(Raw<F32>& r, const void* base, const Lie& t, long long row, int col, int D) {
    const long long at = row * t.ld + col;
    if (EVEN ? col < D : any(col, D) && at + 8 <= t.end) {
        const uint4* p = reinterpret_cast<const uint4*>((const unsigned char*)base + at * (F32 ? 4 : 2));
        r.w[0] = p[0];
        if (F32) r.w[F32] = p[1];
    }
}
__device__ __forceinline__ void put(uint4& u, int i, uint32_t v) {
    u.x |= i == 0 ? v : 0u; u.y |= i == 1 ? v : 0u; u.z |= i == 2 ? v : 0u; u.w |= i == 3 ? v : 0u;
}
// what was requested, complete
template <bool F32, bool EVEN> __device__ __forceinline__ void complete(Raw<F32>& r, const void* base, const Lie& t, long long row, int col, int D) {
    const long long at = row * t.ld + col;
    if (EVEN || !any(col, D) || at + 8 <= t.end) return;
    r = Raw<F32>{};
#pragma unroll 1
    for (int i = col < 0 ? -col : 0; i < 8 && col + i < D; ++i) {
        if (F32) {
            const uint32_t v = ((const uint32_t*)base)[at + i];
            put(r.w[0], i, v);
            put(r.w[F32], i - 4, v);
        } else {
            put(r.w[0], i >> 1, (uint32_t)((const uint16_t*)base)[at + i] << (16 * (i & 1)));
        }
    }
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
// (EVEN: behind the row)
template <bool EVEN> __device__ __forceinline__ void clear_outside(int col, int D, float (&f)[8]) {
    if (EVEN ? col < D : whole(col, D)) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = !EVEN && col + i >= 0 && col + i < D ? f[i] : 0.f;
}
__device__ __forceinline__ float element(const float (&f)[8], int i) {
    const float a = i & 1 ? f[1] : f[0], b = i & 1 ? f[3] : f[2], c = i & 1 ? f[5] : f[4], d = i & 1 ? f[7] : f[6];
    return i & 4 ? i & 2 ? d : c : i & 2 ? b : a;
}
template <bool EVEN> __device__ __forceinline__ void store(void* base, bool f32, const Lie& t, long long row, int col, int D, const float (&f)[8]) {
    const long long at = row * t.ld + col;
    if (EVEN ? col < D : whole(col, D) && t.end) {
        if (f32) {
            float4* p = reinterpret_cast<float4*>((float*)base + at);
            p[0] = make_float4(f[0], f[1], f[2], f[3]);
            p[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>((bf16*)base + at) = pack8(f);
        }
    } else if (!EVEN) {
#pragma unroll 1
        for (int i = col < 0 ? -col : 0; i < 8 && col + i < D; ++i) {
            if (f32) ((float*)base)[at + i] = element(f, i);
            else ((bf16*)base)[at + i] = __float2bfloat16_rn(element(f, i));
        }
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
template <bool EVEN> __device__ __forceinline__ void store_int8(signed char* q, const Lie& t, long long row, int col, int D, const float (&f)[8], const Rounder& round) {
    const uint32_t lo = round.four(f[0], f[1], f[2], f[3]), hi = round.four(f[4], f[5], f[6], f[7]);
    const long long at = row * t.ld + col;
    if (EVEN ? col < D : whole(col, D) && t.end) {
        *reinterpret_cast<uint2*>(q + at) = make_uint2(lo, hi);
    } else if (!EVEN) {
#pragma unroll 1
        for (int i = col < 0 ? -col : 0; i < 8 && col + i < D; ++i) q[at + i] = (signed char)((i & 4 ? hi : lo) >> (8 * (i & 3)));
    }
}

// ---- teams ---------------------------------------------------------------------------------------------------------------
// A team has a row: a power of two of a warp's threads, or whole warps of a CTA, which then has one row.
struct Teams {
    int threads, rows;  // of a team; of a CTA
};
constexpr int threads_most(int nv) { return nv == 1 ? 288 : nv == 2 ? 512 : 544; }  // (288, 544: rows of 2047 and 16383 elements have up to 257 and 2049 pieces)
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

// ---- host ------------------------------------------------------------------------------------------------------------------
// Pieces of a thread.  One where there are few rows, whose time is latency; two where there are many: what a team does once a row is then half a piece's share.
inline int vectors_of(long long M, long long pieces) {
    if (pieces > 2 * threads_most(2)) return 4;
    return pieces <= threads_most(1) && M <= 2 * 148 ? 1 : 2;
}
inline bool al(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// bytes: of a piece of eight elements that is read or written at once, at most 16
inline Lie lie_of(const void* p, long long M, long long D, long long ld, int bytes) {
    const bool pieces = al(p, bytes) && (M == 1 || ld == D || (D % 8 == 0 && ld % 8 == 0));
    return Lie{ld, pieces ? (M - 1) * ld + D : 0};
}
// teams for rows of `pieces` pieces, nv to a thread, CTAs of some 256 threads
inline Teams teams_of(long long pieces, int nv) {
    const long long need = (pieces + nv - 1) / nv;
    int team = 1;
    if (need <= 32) while (team < need) team *= 2;
    else team = (int)((need + 31) / 32 * 32);
    return Teams{team, team > 32 ? 1 : 256 / team};
}
// CTAs for M rows: as many as SMs hold, and a multiple of 8 where a team has several rows (see first_col)
inline long long ctas_of(long long M, const Teams& t, int sms, int threads) {
    const int per_sm = threads / (t.threads * t.rows);
    const long long want = (M + t.rows - 1) / t.rows, most = (long long)sms * (per_sm < 1 ? 1 : per_sm) / 8 * 8;
    return want < most || most == 0 ? want : most;
}

}  // namespace norm
}  // namespace wkv7

// What the kernels of the residual stream share: dropout's generator, rows by pieces of eight elements, rows in 8 bits, teams of threads.
#pragma once
#include "norm.h"
#include "mma_bf16.cuh"
#include "wkv7_kernels.h"

namespace wkv7 {
namespace norm {

// ---- Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) -----------------------
// Ten rounds of two 32 x 32 -> 64 products for four words.  No mask is stored: the backward forms the words again.  36 products
// for a piece of eight, at four cycles each in a quarter of an SM, come to 63800 cycles for 2^26 elements: 32 us at 1965 MHz, computed, beside 41 of traffic in bf16.
struct Dropper {
    uint32_t k0, k1, from;  // kept: word >= from
    bool none;              // all dropped, the threshold is 2^32
    float scale;
    __device__ __forceinline__ explicit Dropper(const Dropout& d) : from((uint32_t)d.threshold), none(d.threshold >> 32 != 0), scale(d.scale) {
        const unsigned long long s = d.where ? *d.where : d.seed;
        k0 = __shfl_sync(0xffffffffu, (uint32_t)s, 0);  // (the same for all lanes, which the compiler cannot see)
        k1 = __shfl_sync(0xffffffffu, (uint32_t)(s >> 32), 0);
    }
    // the eight words of counters 2 n and 2 n + 1.  LOW: both are below 2^32, so that the second round's first product is the same for all
    template <bool LOW> __device__ __forceinline__ void words(unsigned long long n, uint32_t (&c)[2][4]) const {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            c[b][0] = (uint32_t)(2 * n) + b;
            c[b][1] = LOW ? 0u : (uint32_t)(n >> 31);
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
    }
    __device__ __forceinline__ bool keeps(uint32_t word) const { return word >= from && !none; }
    // eight adjacent elements, of which the first is element 8 n
    template <bool LOW> __device__ __forceinline__ void apply(unsigned long long n, float (&f)[8]) const {
        uint32_t c[2][4];
        words<LOW>(n, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = keeps(c[i / 4][i % 4]) ? __fmul_rn(f[i], scale) : 0.f;
    }
    __device__ __forceinline__ void apply(bool low, unsigned long long n, float (&f)[8]) const {
        if (low) apply<true>(n, f);
        else apply<false>(n, f);
    }
};
inline bool low_counters(long long elements) { return elements <= 1LL << 34; }

// ---- two fp32 operations an instruction ------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// a piece as four pairs
struct Piece {
    uint64_t p[4];
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = two(f[2 * i], f[2 * i + 1]);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) split(p[i], f[2 * i], f[2 * i + 1]);
    }
};
__device__ __forceinline__ float sum_of(uint64_t s) {
    float a, b;
    split(s, a, b);
    return a + b;
}

// ---- eight adjacent elements of a row ------------------------------------------------------------------------------------
// A thread's elements are 8 n .. 8 n + 7 of the whole tensor, counted row-major: where rows lie back to back they are 16-byte pieces whatever the row's length, and
// they are two counters' words of dropout.  Of a row they are columns col .. col + 7, of which the row's first and last piece may have only a part: it is read whole, where
// the tensor has it whole, and the rest is put to zero.  What is not read so, a tensor's last part of a piece and layouts without such pieces, is read element by
// element where it is used, not where it is requested: a request is a load and nothing else, which nothing waits for.
// EVEN: all tensors lie in pieces and rows are a multiple of 8 long, so that there are no parts.
using Byte = unsigned char;
template <bool F32> struct Raw { uint4 w[F32 ? 2 : 1]; };
struct Lie {          // how a tensor lies
    const Byte* base;
    const Byte* end;  // behind its last element; null: not in 16-byte pieces
    long long ld;     // elements from row to row
};
__device__ __forceinline__ bool whole(int col, int D) { return col >= 0 && col + 8 <= D; }
__device__ __forceinline__ bool any(int col, int D) { return col > -8 && col < D; }
// at: of the piece's first element
template <bool F32, bool EVEN> __device__ __forceinline__ void request(Raw<F32>& r, const Byte* at, const Byte* end, int col, int D) {
    if (EVEN ? col < D : any(col, D) && at + (F32 ? 32 : 16) <= end) {
        r.w[0] = reinterpret_cast<const uint4*>(at)[0];
        if (F32) r.w[F32] = reinterpret_cast<const uint4*>(at)[1];
    }
}
__device__ __forceinline__ void put(uint4& u, int i, uint32_t v) {
    u.x |= i == 0 ? v : 0u; u.y |= i == 1 ? v : 0u; u.z |= i == 2 ? v : 0u; u.w |= i == 3 ? v : 0u;
}
// what was requested, complete
template <bool F32, bool EVEN> __device__ __forceinline__ void complete(Raw<F32>& r, const Byte* at, const Byte* end, int col, int D) {
    if (EVEN || !any(col, D) || at + (F32 ? 32 : 16) <= end) return;
    r = Raw<F32>{};
#pragma unroll 1
    for (int i = col < 0 ? -col : 0; i < 8 && col + i < D; ++i) {
        if (F32) {
            const uint32_t v = reinterpret_cast<const uint32_t*>(at)[i];
            put(r.w[0], i, v);
            put(r.w[F32], i - 4, v);
        } else {
            put(r.w[0], i >> 1, (uint32_t)reinterpret_cast<const uint16_t*>(at)[i] << (16 * (i & 1)));
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
// Elements lo .. hi - 1 of a piece, of which one end is the piece's own: three stores at most, of one, two and four elements.  W: words of four elements.
template <typename T1, typename T2, typename T4> __device__ __forceinline__ void store_part(Byte* at, int lo, int hi, const T1 (&e)[8], const T2 (&two)[4], const T4 (&four)[2]) {
    T1* const p1 = reinterpret_cast<T1*>(at);
    if (hi == 8) {
        if (lo & 1) p1[lo] = lo & 4 ? lo & 2 ? e[7] : e[5] : lo & 2 ? e[3] : e[1];
        const int l2 = (lo + 1) & 6;
        if (l2 & 2) *reinterpret_cast<T2*>(p1 + l2) = l2 & 4 ? two[3] : two[1];
        if (lo <= 4) *reinterpret_cast<T4*>(p1 + 4) = four[1];
    } else {
        if (hi & 4) *reinterpret_cast<T4*>(p1) = four[0];
        if (hi & 2) *reinterpret_cast<T2*>(p1 + (hi & 4)) = hi & 4 ? two[2] : two[0];
        if (hi & 1) p1[hi & 6] = hi & 4 ? hi & 2 ? e[6] : e[4] : hi & 2 ? e[2] : e[0];
    }
}
__device__ __forceinline__ float element(const float (&f)[8], int i) {
    const float a = i & 1 ? f[1] : f[0], b = i & 1 ? f[3] : f[2], c = i & 1 ? f[5] : f[4], d = i & 1 ? f[7] : f[6];
    return i & 4 ? i & 2 ? d : c : i & 2 ? b : a;
}
template <bool EVEN> __device__ __forceinline__ void store(Byte* at, const Byte* end, bool f32, int col, int D, const float (&f)[8]) {
    if (EVEN ? col < D : whole(col, D) && end) {
        if (f32) {
            reinterpret_cast<float4*>(at)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(at)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>(at) = pack8(f);
        }
    } else if (!EVEN && any(col, D)) {
        const int lo = col < 0 ? -col : 0, hi = D - col < 8 ? D - col : 8;
        if (!end || (lo && hi < 8)) {
#pragma unroll 1
            for (int i = lo; i < hi; ++i) {
                if (f32) reinterpret_cast<float*>(at)[i] = element(f, i);
                else reinterpret_cast<bf16*>(at)[i] = __float2bfloat16_rn(element(f, i));
            }
        } else if (f32) {
            const float2 two[4] = {{f[0], f[1]}, {f[2], f[3]}, {f[4], f[5]}, {f[6], f[7]}};
            const float4 four[2] = {make_float4(f[0], f[1], f[2], f[3]), make_float4(f[4], f[5], f[6], f[7])};
            store_part<float, float2, float4>(at, lo, hi, f, two, four);
        } else {
            const uint4 u = pack8(f);
            const uint16_t e[8] = {(uint16_t)u.x, (uint16_t)(u.x >> 16), (uint16_t)u.y, (uint16_t)(u.y >> 16), (uint16_t)u.z, (uint16_t)(u.z >> 16), (uint16_t)u.w, (uint16_t)(u.w >> 16)};
            const uint32_t two[4] = {u.x, u.y, u.z, u.w};
            const uint2 four[2] = {make_uint2(u.x, u.y), make_uint2(u.z, u.w)};
            store_part<uint16_t, uint32_t, uint2>(at, lo, hi, e, two, four);
        }
    }
}
// the weight's, ones without
__device__ __forceinline__ void weights(const void* w, bool f32, int col, int D, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = !w || col + i < 0 || col + i >= D ? 1.f : f32 ? ((const float*)w)[col + i] : __bfloat162float(((const bf16*)w)[col + i]);
}

// ---- a row in 8 bits -------------------------------------------------------------------------------------------------------
// top: max |y|, a NaN if there is one.  Rows without a magnitude above 2^-100 are zeros with scale 0, a row that holds a NaN or an infinity is
// zeros with a NaN for its scale: so are its products.
constexpr uint32_t TINY_BITS = (127 - 100) << 23, INF_BITS = 0x7f800000u;
__device__ __forceinline__ float max_abs(float top, float f) {  // (a NaN stays)
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(f)));
    return r;
}
// q = rint(v c), c the least number that is not below 127 / a.  Of bf16 rows that is rint(127 v / a), ties to even: with 8-bit mantissas 127 v / a is n + 1/2 either because
// v = +-a / 2, where v c is 63.5 or a little more and 64 is right; or because 127 divides a's mantissa, where c and v c are exact.  Quotients that are no ties are 2^-17 of
// their size away from one (the numerators differ by a whole step), v c is off by 2^-22.
struct Rounder {
    float c;
    uint32_t mask;
    __device__ __forceinline__ explicit Rounder(float top) {
        const bool live = top > __uint_as_float(TINY_BITS) && top < __uint_as_float(INF_BITS);
        const float q = 127.f / top;
        c = live ? fmaf(-q, top, 127.f) > 0.f ? __uint_as_float(__float_as_uint(q) + 1) : q : 0.f;  // (the remainder is exact)
        mask = live ? ~0u : 0u;
    }
    __device__ __forceinline__ uint32_t four(float a, float b, float d, float e) const {
        // 1.5 * 2^23: the sum's low byte is the integer nearest to v c.  (The product is rounded by itself: merged into the sum it would be, too, in effect.)
        const uint64_t M = two(12582912.f, 12582912.f), cc = two(c, c);
        float x, y, z, w;
        split(add2(mul2(two(a, b), cc), M), x, y);
        split(add2(mul2(two(d, e), cc), M), z, w);
        return __byte_perm(__byte_perm(__float_as_uint(x), __float_as_uint(y), 0x0040), __byte_perm(__float_as_uint(z), __float_as_uint(w), 0x0040), 0x5410) & mask;
    }
    __device__ __forceinline__ static float scale(float top, float times) {
        return !(top < __uint_as_float(INF_BITS)) ? __uint_as_float(0x7fc00000u) : top > __uint_as_float(TINY_BITS) ? __fdiv_rn(top * times, 127.f) : 0.f;
    }
};
// (pieces of 8 bytes)
template <bool EVEN> __device__ __forceinline__ void store_int8(Byte* at, const Byte* end, int col, int D, const float (&f)[8], const Rounder& round) {
    const uint32_t lo = round.four(f[0], f[1], f[2], f[3]), hi = round.four(f[4], f[5], f[6], f[7]);
    if (EVEN ? col < D : whole(col, D) && end) {
        *reinterpret_cast<uint2*>(at) = make_uint2(lo, hi);
    } else if (!EVEN && whole(col, D)) {  // (rows of x lie back to back, those in 8 bits on boundaries: pieces of the one are not pieces of the other)
#pragma unroll
        for (int i = 0; i < 8; ++i) at[i] = (Byte)((i & 4 ? hi : lo) >> (8 * (i & 3)));
    } else if (!EVEN) {
#pragma unroll 1
        for (int i = col < 0 ? -col : 0; i < 8 && col + i < D; ++i) at[i] = (Byte)((i & 4 ? hi : lo) >> (8 * (i & 3)));
    }
}

// ---- teams ---------------------------------------------------------------------------------------------------------------
// A team has a row: a power of two of a warp's threads, or whole warps.
struct Teams {
    int threads, rows;  // of a team; of a CTA
};
constexpr int threads_most(int nv) { return nv == 1 ? 288 : nv == 2 ? 512 : 544; }  // (288, 544: rows of 2047 and 16383 elements have up to 257 and 2049 pieces)
constexpr long long pieces_of(long long D) { return D % 8 ? (D + 14) / 8 : D / 8; }
static_assert(pieces_of(NORM_MAX_D) <= 4 * threads_most(4) && pieces_of(NORM_MAX_D - 1) <= 4 * threads_most(4), "a thread has four pieces at most");
constexpr int MAX_WARPS = 32;
// Sum and maximum over a team, in everyone's registers.  room: two of them in turn, so that one barrier a row is enough: before a thread comes to
// write one again all have passed the other's barrier, and so have read this one.
struct Room { float sum[2][MAX_WARPS], top[2][MAX_WARPS]; };  // [turn][warp of the CTA]
template <bool SUM, bool TOP> __device__ __forceinline__ void butterfly(int n, float& sum, float& top) {
#pragma unroll
    for (int o = 16; o; o /= 2)
        if (o < n) {
            if (SUM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (TOP) top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
}
// SEVERAL: a CTA has several teams of more than a warp, each with a barrier of its own.  (A kernel that names barriers by number takes all 16 of a CTA's, and an SM
// has room for few such CTAs: teams of 64 threads, one a CTA, 65536 x 768 78 -> 116 us.)
template <bool SUM, bool TOP, bool SEVERAL> __device__ __forceinline__ void reduce(int team, Room& room, int turn, float& sum, float& top) {
    butterfly<SUM, TOP>(team, sum, top);
    if (team <= 32) return;
    const int warps = team / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, of = SEVERAL ? threadIdx.x / team : 0;
    if (lane == 0) {
        if (SUM) room.sum[turn][warp] = sum;
        if (TOP) room.top[turn][warp] = top;
    }
    if (SEVERAL) asm volatile("barrier.sync %0, %1;" ::"r"(1 + of), "r"(team) : "memory");
    else __syncthreads();
    if (SUM) sum = lane < warps ? room.sum[turn][of * warps + lane] : 0.f;
    if (TOP) top = lane < warps ? room.top[turn][of * warps + lane] : 0.f;
    butterfly<SUM, TOP>(32, sum, top);
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
// size: of an element; pieces of eight lie on boundaries of 16 bytes, of 8 in 8 bits
inline Lie lie_of(const void* p, long long M, long long D, long long ld, int size) {
    const bool pieces = p && al(p, size == 1 ? 8 : 16) && (M == 1 || ld == D || (D % 8 == 0 && ld % 8 == 0));
    return Lie{(const Byte*)p, pieces ? (const Byte*)p + ((M - 1) * ld + D) * size : nullptr, ld};
}
// teams for rows of `pieces` pieces, nv to a thread; CTAs of `threads` threads at most, of one team where it has more
inline Teams teams_of(long long pieces, int nv, int threads) {
    const long long need = (pieces + nv - 1) / nv;
    int team = 1;
    if (need <= 32) while (team < need) team *= 2;
    else team = (int)((need + 31) / 32 * 32);
    return Teams{team, team < threads ? threads / team : 1};
}
// CTAs for M rows: as many as SMs hold, and a multiple of 8 where a team has several rows (see first_col)
inline long long ctas_of(long long M, const Teams& t, int sms, int threads) {
    const int per_sm = threads / (t.threads * t.rows);
    const long long want = (M + t.rows - 1) / t.rows, most = (long long)sms * (per_sm < 1 ? 1 : per_sm) / 8 * 8;
    return want < most || most == 0 ? want : most;
}

}  // namespace norm
}  // namespace wkv7

// Dense products with their epilogue:  y = act(x w^T + bias) + residual, and the products of its backward.
//     x [M, K], w [N, K] (an nn.Linear weight), bf16;  fp32 accumulation in tensor memory;  y bf16 or fp32
//     dz = dy act'(z),  dx = dz w,  dw = dz^T x,  dbias = sum of dz over the rows
// All three are one form, out[i, j] = sum_k P[i, k] Q[j, k]: an operand whose k is contiguous in memory is read K-major, one whose index is (w in
// dx; dz and x in dw) as it lies, MN-major, so that nothing is transposed in memory.
//
// linear_pair_kernel, for large products: persistent pairs of CTAs, a tile of 256 x BN per pair (each CTA holds 128 rows of P and half of the
// tile's Q rows; one thread of the pair issues tcgen05.mma.cta_group::2), two accumulators, so that eight warps empty one while the
// other is filled.  Bound by the tensor cores (active 88 % of the time, 8192 x 8192 x 2048 in 171 to 176 us, 1.6 PFLOP/s) and, in long programs, by the power cap.
// linear_tile_kernel, for the rest: one tile of 128 x NT a CTA, the sum over k split over a cluster of up to eight CTAs, which add their
// parts through distributed shared memory in a fixed order (each part is sent: fetching it, 24 x 8192 x 2048 took 32 us instead of 12).  Few rows (decoding): the
// weight is P and the rows of x are Q, so that a CTA streams 128 weight rows against all of x.  Bound by the weight's stream: 16 x 2048 x 50001 in 37 us, 5.7 TB/s.
#include <cuda.h>
#include <cstring>

#include "linear.h"
#include "mma_bf16.cuh"
#include "wkv7_kernels.h"

namespace wkv7 {
namespace lin {

constexpr int BM = 128, BK = 64;
constexpr int MAXSTAGES = 12;
// A wait for an accumulator lasts for a whole sum.  2^21 k blocks (k = 2^27) at 0.35 us are 0.7 s; the limit is 1.1 s.
constexpr long long SUM_LIMIT = ACROSS_HANDOFF_LIMIT;
constexpr int MAX_KBLOCKS = 1 << 21;

// ---- activations -----------------------------------------------------------------------------------------
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid_f(float x) { return rcp_mufu(1.f + ex2_approx(-LOG2E * x)); }
__device__ __forceinline__ float tanh_f(float x) {
    // (1 - e) / (1 + e), e = exp(-2 |x|): relative error 2e-6 from |x| = 0.1 on; the series' first four terms below (next one: 2e-10)
    const float t = fabsf(x), e = ex2_approx(-2.f * LOG2E * t), x2 = x * x;
    const float big = copysignf((1.f - e) * rcp_mufu(1.f + e), x);
    const float small = x * (1.f + x2 * (-1.f / 3.f + x2 * (2.f / 15.f - x2 * (17.f / 315.f))));
    return t < 0.1f ? small : big;
}
constexpr float GELU_C = 1.5957691216057308f;  // 2 sqrt(2 / pi): gelu(x) = x sigmoid(GELU_C (x + 0.044715 x^3))
__device__ __forceinline__ float gelu_s(float x) { return sigmoid_f(GELU_C * x * (1.f + 0.044715f * x * x)); }
__device__ __forceinline__ float sqrt_f(float x) {  // relative error 2^-23
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float relu_f(float x) { return x < 0.f ? 0.f : x; }  // (a NaN stays one)

template <int ACT> __device__ __forceinline__ float act(float x) {
    switch (ACT) {
        case kActRelu: return relu_f(x);
        case kActRelu2: { const float r = relu_f(x); return r * r; }
        case kActTanh: return tanh_f(x);
        case kActSigmoid: return sigmoid_f(x);
        case kActSilu: return x * sigmoid_f(x);
        case kActGelu: return x * gelu_s(x);
        default: return x;
    }
}
// act'(z); FROM_Y: of relu and relu2 from their values, 2 sqrt(y) for 2 relu(z)
template <int ACT, bool FROM_Y> __device__ __forceinline__ float act_grad(float z) {
    switch (ACT) {
        case kActRelu: return z <= 0.f ? 0.f : 1.f;
        case kActRelu2: return FROM_Y ? 2.f * sqrt_f(z) : 2.f * relu_f(z);
        case kActTanh: { const float e = ex2_approx(-2.f * LOG2E * fabsf(z)), r = rcp_mufu(1.f + e); return 4.f * e * r * r; }
        case kActSigmoid: { const float e = ex2_approx(-LOG2E * fabsf(z)), r = rcp_mufu(1.f + e); return e * r * r; }  // (s (1 - s) would be 0 from z = 17 on)
        case kActSilu: { const float s = sigmoid_f(z); return s * (1.f + z * (1.f - s)); }  // (beside a 1 what 1 - s loses does not count; nor in gelu')
        case kActGelu: {
            z = z > 64.f ? 64.f : z < -64.f ? -64.f : z;  // (1 and 0 long before; z^3 would leave fp32's range)
            const float s = gelu_s(z);
            return s + z * s * (1.f - s) * GELU_C * (1.f + 3.f * 0.044715f * z * z);
        }
        default: return 1.f;
    }
}

// ---- epilogue --------------------------------------------------------------------------------------------
struct Epi : LinearEpilogue {
    bool vec;       // rows of y start and end on 16-byte boundaries (bulk stores clip in steps of 16 bytes), those of the residual start there
    bool bias_vec;  // so does the bias
};
__device__ __forceinline__ void load8g(const void* base, bool f32, long long at, float (&f)[8]) {
    if (f32) {
        const float4 a = *reinterpret_cast<const float4*>((const float*)base + at), b = *reinterpret_cast<const float4*>((const float*)base + at + 4);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
        unpack8(*reinterpret_cast<const uint4*>((const bf16*)base + at), f);
    }
}
// the same in two steps, for several rows requested at once
struct Words8 { uint4 lo, hi; };
__device__ __forceinline__ Words8 request8(const void* base, bool f32, long long at) {
    const uint4* p = reinterpret_cast<const uint4*>((const unsigned char*)base + at * (f32 ? 4 : 2));
    Words8 w;
    w.lo = p[0];
    w.hi = f32 ? p[1] : w.lo;
    return w;
}
__device__ __forceinline__ void floats8(const Words8& w, bool f32, float (&f)[8]) {
    if (f32) {
        f[0] = __uint_as_float(w.lo.x); f[1] = __uint_as_float(w.lo.y); f[2] = __uint_as_float(w.lo.z); f[3] = __uint_as_float(w.lo.w);
        f[4] = __uint_as_float(w.hi.x); f[5] = __uint_as_float(w.hi.y); f[6] = __uint_as_float(w.hi.z); f[7] = __uint_as_float(w.hi.w);
    } else {
        unpack8(w.lo, f);
    }
}
__device__ __forceinline__ float load1g(const void* base, bool f32, long long at) {
    return f32 ? ((const float*)base)[at] : __bfloat162float(((const bf16*)base)[at]);
}
__device__ __forceinline__ void store_z1(const Epi& e, long long row, long long col, float v) {
    if (e.z_f32) ((float*)e.z)[row * e.ldz + col] = v;
    else ((bf16*)e.z)[row * e.ldz + col] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ void store8g(void* base, bool f32, long long at, const float (&f)[8]) {
    if (f32) {
        *reinterpret_cast<float4*>((float*)base + at) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>((float*)base + at + 4) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        *reinterpret_cast<uint4*>((bf16*)base + at) = pack8(f);
    }
}
// the bias of eight adjacent columns
__device__ __forceinline__ void bias8(const Epi& e, long long col, float (&f)[8]) {
    if (e.bias_vec && col + 8 <= e.cols) {
        load8g(e.bias, e.bias_f32, col, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = col + i < e.cols ? load1g(e.bias, e.bias_f32, col + i) : 0.f;
    }
}
// eight adjacent columns of a row, from the accumulator to memory; bias already added
template <int ACT> __device__ __forceinline__ void finish8(const Epi& e, long long row, long long col, float (&f)[8]) {
    const int live = (int)(e.cols - col < 8 ? e.cols - col : 8);
    if (e.z) store8g(e.z, e.z_f32, row * e.ldz + col, f);  // (ldz is a multiple of 8: room for all eight)
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = act<ACT>(f[i]);
    if (e.vec && live == 8) {
        if (e.residual) {
            float r[8];
            load8g(e.residual, e.y_f32, row * e.ldr + col, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += r[i];
        }
        store8g(e.y, e.y_f32, row * e.ldy + col, f);
        return;
    }
    if (e.residual) {  // (all of it is read before anything is stored: y may be the residual, so the compiler keeps them in order)
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = i < live ? load1g(e.residual, e.y_f32, row * e.ldr + col + i) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += r[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < live) {
            if (e.y_f32) ((float*)e.y)[row * e.ldy + col + i] = f[i];
            else ((bf16*)e.y)[row * e.ldy + col + i] = __float2bfloat16_rn(f[i]);
        }
}
// A block of 32 x 32 results to memory by a bulk tensor store, which clips it: a lane has a row of it, or (TURNED) a column.  `turn`: which half of the
// staging area is next (bf16; fp32 takes all of it); it is written again when the store that reads it has.  `all`: wait for all stores, where halves do not alternate.
template <bool TURNED> __device__ __forceinline__ void bulk_store_block(float* staging, const CUtensorMap* map, bool f32, bool all, const float (&v)[32], int lane, int& turn, long long col0, long long row0) {
    unsigned char* to = reinterpret_cast<unsigned char*>(staging) + (f32 ? 0 : 2048 * turn);
    if (lane == 0) {
        if (f32 || all) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        else asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    }
    __syncwarp();
    if (f32) {  // rows of 128 bytes, piece u of row r at u ^ (r % 8)
        if (TURNED) {
#pragma unroll
            for (int c = 0; c < 32; ++c) *reinterpret_cast<float*>(to + c * 128 + (((lane >> 2) ^ (c & 7)) << 4) + (lane & 3) * 4) = v[c];
        } else {
#pragma unroll
            for (int u = 0; u < 8; ++u) *reinterpret_cast<float4*>(to + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
        }
    } else {    // rows of 64 bytes, piece u of row r at u ^ (r / 2 % 4)
        if (TURNED) {
#pragma unroll
            for (int c = 0; c < 32; ++c) *reinterpret_cast<bf16*>(to + c * 64 + (((lane >> 3) ^ (c >> 1 & 3)) << 4) + (lane & 7) * 2) = __float2bfloat16_rn(v[c]);
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                *reinterpret_cast<uint4*>(to + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4)) = make_uint4(pack_bf16x2(v[8 * u], v[8 * u + 1]), pack_bf16x2(v[8 * u + 2], v[8 * u + 3]),
                                                                                                   pack_bf16x2(v[8 * u + 4], v[8 * u + 5]), pack_bf16x2(v[8 * u + 6], v[8 * u + 7]));
        }
        turn ^= 1;
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"((int)col0), "r"((int)row0), "r"(smem_u32(to)) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}

// The same for two bf16 blocks side by side, a lane a row: one wait and one fence for both.
__device__ __forceinline__ void bulk_store_two(float* staging, const CUtensorMap* map, const float (&v)[2][32], int lane, long long col0, long long row0) {
    unsigned char* to = reinterpret_cast<unsigned char*>(staging);
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < 4; ++u)
            *reinterpret_cast<uint4*>(to + 2048 * h + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4)) =
                make_uint4(pack_bf16x2(v[h][8 * u], v[h][8 * u + 1]), pack_bf16x2(v[h][8 * u + 2], v[h][8 * u + 3]),
                           pack_bf16x2(v[h][8 * u + 4], v[h][8 * u + 5]), pack_bf16x2(v[h][8 * u + 6], v[h][8 * u + 7]));
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                         ::"l"(map), "r"((int)col0 + 32 * h), "r"((int)row0), "r"(smem_u32(to + 2048 * h)) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}
// Two blocks side by side, wholly among the columns and all bf16: one block's latencies are spent on the other.
template <int ACT, typename Sums> __device__ __forceinline__ void finish_rows_two(const Epi& e, const CUtensorMap* Y, const CUtensorMap* Z, float* mine, int lane, long long row0, long long col0,
                                                                                 Sums sums) {
    const bool in = row0 + lane < e.rows;
    const long long at = (row0 + lane) * e.ldr + col0;
    uint4 res[8];
    if (e.residual && in)
#pragma unroll
        for (int c = 0; c < 8; ++c) res[c] = *reinterpret_cast<const uint4*>((const bf16*)e.residual + at + 8 * c);
    float v[2][32];
    sums(v);
    if (e.bias)
#pragma unroll
        for (int c = 0; c < 64; c += 8) {
            float f[8];
            bias8(e, col0 + c, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c / 32][c % 32 + i] += f[i];
        }
    if (e.z) bulk_store_two(mine, Z, v, lane, col0, row0);
#pragma unroll
    for (int c = 0; c < 64; ++c) v[c / 32][c % 32] = act<ACT>(v[c / 32][c % 32]);
    if (e.residual && in)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            float f[8];
            unpack8(res[c], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c / 4][8 * (c % 4) + i] += f[i];
        }
    bulk_store_two(mine, Y, v, lane, col0, row0);
}
// A warp's block of 32 x 32, a lane a column of y; the sums come by sums(v).  Rows that are not aligned are stored, 32 adjacent elements an instruction, as they lie.
template <int ACT, typename Sums> __device__ __forceinline__ void finish_cols(const Epi& e, const CUtensorMap* Y, const CUtensorMap* Z, float* mine, bool mixed, int lane, int& turn,
                                                                             long long row0, long long col0, Sums sums) {
    const long long col = col0 + lane;
    const bool in = col < e.cols;
    const int rows = (int)(e.rows - row0 < 32 ? e.rows - row0 : 32);
    float v[32];
    const float bias = e.bias && in ? load1g(e.bias, e.bias_f32, col) : 0.f;
    sums(v);
    if (e.bias)
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] += bias;
    if (e.z) {
        if (e.vec) {
            bulk_store_block<true>(mine, Z, e.z_f32, mixed, v, lane, turn, col0, row0);
        } else {
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (in && c < rows) store_z1(e, row0 + c, col, v[c]);
        }
    }
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] = act<ACT>(v[c]);
#pragma unroll
    for (int half = 0; half < 32; half += 16) {
        if (e.residual) {  // (sixteen rows of it before they are stored: y may be the residual, so the compiler keeps them in order)
            float res[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) res[c] = in && half + c < rows ? load1g(e.residual, e.y_f32, (row0 + half + c) * e.ldr + col) : 0.f;
#pragma unroll
            for (int c = 0; c < 16; ++c) v[half + c] += res[c];
        }
        if (e.vec) continue;
#pragma unroll
        for (int c = half; c < half + 16; ++c)
            if (in && c < rows) {
                if (e.y_f32) ((float*)e.y)[(row0 + c) * e.ldy + col] = v[c];
                else ((bf16*)e.y)[(row0 + c) * e.ldy + col] = __float2bfloat16_rn(v[c]);
            }
    }
    if (e.vec) bulk_store_block<true>(mine, Y, e.y_f32, mixed, v, lane, turn, col0, row0);
}
// a block of which each lane has a row, turned so that each has a column
__device__ __forceinline__ void turn_block(float* mine, int lane, float (&v)[32]) {
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 8; ++u)  // 16-byte unit u of row r at u ^ (r % 8)
        *reinterpret_cast<float4*>(mine + lane * 32 + ((u ^ (lane & 7)) << 2)) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] = mine[c * 32 + (((lane >> 2) ^ (c & 7)) << 2) + (lane & 3)];
}
// A warp's block of 32 x 32, a lane a row of y: the sums come by sums(v), residual and bias are applied as they lie.
template <int ACT, typename Sums> __device__ __forceinline__ void finish_rows(const Epi& e, const CUtensorMap* Y, const CUtensorMap* Z, float* mine, bool mixed, int lane, int& turn,
                                                                             long long row0, long long col0, Sums sums) {
    const bool whole = row0 + lane < e.rows && col0 + 32 <= e.cols;
    const long long at = (row0 + lane) * e.ldr + col0;
    Words8 res[4];
    if (e.residual && whole)
#pragma unroll
        for (int c = 0; c < 4; ++c) res[c] = request8(e.residual, e.y_f32, at + 8 * c);
    float v[32];
    sums(v);
    if (e.bias)
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
            float f[8];
            bias8(e, col0 + c, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c + i] += f[i];
        }
    if (e.z) bulk_store_block<false>(mine, Z, e.z_f32, mixed, v, lane, turn, col0, row0);
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] = act<ACT>(v[c]);
    if (e.residual) {
        if (whole) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float f[8];
                floats8(res[c], e.y_f32, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * c + i] += f[i];
            }
        } else if (row0 + lane < e.rows) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (col0 + c < e.cols) v[c] += load1g(e.residual, e.y_f32, at + c);
        }
    }
    bulk_store_block<false>(mine, Y, e.y_f32, mixed, v, lane, turn, col0, row0);
}

// ---- tensor core and copy helpers --------------------------------------------------------------------------
// shared-memory descriptors of 128-byte-swizzled operands.  K-major: 128-byte rows of 64 k, groups of 8 rows 1024 bytes apart.  MN-major: [k][64
// indices] boxes, 8 k rows = 1024 bytes, the next 64 indices in the next box of 64 k (8192 bytes).
__device__ __forceinline__ uint64_t desc_of(uint32_t saddr, bool mn) {
    const uint64_t lbo = mn ? (8192 >> 4) : 1;
    return (uint64_t)((saddr >> 4) & 0x3fff) | (lbo << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// fp32 accumulate, bf16 operands
__host__ __device__ constexpr uint32_t idesc_of(int m, int n, bool p_mn, bool q_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((p_mn ? 1u : 0u) << 15) | ((q_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void tmem_ld32(uint32_t ta, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]),"=r"(v[1]),"=r"(v[2]),"=r"(v[3]),"=r"(v[4]),"=r"(v[5]),"=r"(v[6]),"=r"(v[7]),"=r"(v[8]),"=r"(v[9]),"=r"(v[10]),"=r"(v[11]),"=r"(v[12]),"=r"(v[13]),"=r"(v[14]),"=r"(v[15]),
                   "=r"(v[16]),"=r"(v[17]),"=r"(v[18]),"=r"(v[19]),"=r"(v[20]),"=r"(v[21]),"=r"(v[22]),"=r"(v[23]),"=r"(v[24]),"=r"(v[25]),"=r"(v[26]),"=r"(v[27]),"=r"(v[28]),"=r"(v[29]),"=r"(v[30]),"=r"(v[31])
                 : "r"(ta));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t ta, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]),"=r"(v[1]),"=r"(v[2]),"=r"(v[3]),"=r"(v[4]),"=r"(v[5]),"=r"(v[6]),"=r"(v[7]),"=r"(v[8]),"=r"(v[9]),"=r"(v[10]),"=r"(v[11]),"=r"(v[12]),"=r"(v[13]),"=r"(v[14]),"=r"(v[15])
                 : "r"(ta));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// ---- tiles of 128 x NT, k split over a cluster ---------------------------------------------------------------
struct TileParams {
    CUtensorMap P, Q, Y, Z;  // Y, Z: as the pairs'
    Epi e;
    int p_mn, q_mn, nt, kblocks, splits, stages, accs, swap, direct, outer, p_tiles;  // swap: P runs over the columns of y, Q over its rows
    uint32_t tmem_cols;
    // outer > 1: each tile has that many clusters, which leave their sums in memory; of the CTAs that have the same rows of a tile the last to arrive adds them, in
    // their order, and finishes
    float* sums;        // [outer][tile][128][nt]
    unsigned* arrived;  // [tile][rank], zero
};
struct TileCtrl {
    uint64_t full[MAXSTAGES], empty[MAXSTAGES], accum, drain;
    uint32_t tmem_base;
    volatile int abort, zero;
    int last;
};
static_assert(sizeof(TileCtrl) <= 1024, "the KB ahead of the ring");
constexpr int TILE_THREADS = 192;  // warps 0-3: accumulator rows, warp 4: copies, warp 5: products; all six: the result
constexpr int P_BYTES = BM * 128;
__host__ __device__ constexpr int q_bytes(int nt) { return nt * 128; }  // a multiple of 1024 from 8 rows on
// Accumulator rows in shared memory, nt + 4 floats apart: rows r .. r + 7 start on different groups of four banks.  Each CTA of a cluster has 128 / splits rows
// of the tile to finish and a place for every CTA's part of them.
__host__ __device__ constexpr int part_pitch(int nt) { return nt + 4; }
__host__ __device__ constexpr int part_bytes(int nt) { return BM * part_pitch(nt) * 4; }

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }

template <int ACT> __global__ void __launch_bounds__(TILE_THREADS, 3) linear_tile_kernel(const __grid_constant__ TileParams p, int* status) {
    extern __shared__ unsigned char smem_dyn[];
    TileCtrl* ctrl = reinterpret_cast<TileCtrl*>(smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u));
    unsigned char* sm = reinterpret_cast<unsigned char*>(ctrl) + 1024;
    const int stage_bytes = P_BYTES + q_bytes(p.nt);
    // the parts have a place of their own where other CTAs write to it, which may be done with their share of k before this one
    float* parts = reinterpret_cast<float*>(p.splits > 1 ? sm + p.stages * stage_bytes : sm);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int rank = blockIdx.x % p.splits;
    const long long tile = blockIdx.x / p.splits / p.outer;
    const int cluster = blockIdx.x / p.splits % p.outer;
    const int p0 = (int)(tile % p.p_tiles) * BM, q0 = (int)(tile / p.p_tiles) * p.nt;
    const int share = cluster * p.splits + rank, shares = p.splits * p.outer;
    const int lo = (int)((long long)p.kblocks * share / shares), hi = (int)((long long)p.kblocks * (share + 1) / shares);

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) { mbar_init(&ctrl->full[s], 1); mbar_init(&ctrl->empty[s], 1); }
        mbar_init(&ctrl->accum, 1); mbar_init(&ctrl->drain, 1);
        ctrl->abort = 0; ctrl->zero = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4 && elect_one()) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&p.P) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&p.Q) : "memory");
    }
    if (warp == 0) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctrl->tmem_base)), "r"(p.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = ctrl->tmem_base;
    if (p.splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for before the first write to another CTA)
    stream_order();

    if (warp == 4) {
        if (elect_one()) {
            int s = 0, round = 0, issued = 0;
            for (int kb = lo; kb < hi; ++kb) {
                if (round > 0 && !mbar_wait_bounded<true>(&ctrl->empty[s], (round - 1) & 1, &ctrl->abort, status)) break;
                const uint32_t bar = smem_u32(&ctrl->full[s]), dst = smem_u32(sm + s * stage_bytes);
                expect_tx(&ctrl->full[s], (uint32_t)stage_bytes);
                auto load = [&](const CUtensorMap* m, uint32_t to, int x, int y) {
                    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                                 ::"r"(to), "l"(m), "r"(bar), "r"(x), "r"(y) : "memory");
                };
                if (p.p_mn) { load(&p.P, dst, p0, kb * BK); load(&p.P, dst + 8192, p0 + 64, kb * BK); }
                else load(&p.P, dst, kb * BK, p0);
                if (p.q_mn) for (int b = 0; b < p.nt; b += 64) load(&p.Q, dst + P_BYTES + b * 128, q0 + b, kb * BK);
                else load(&p.Q, dst + P_BYTES, kb * BK, q0);
                ++issued;
                if (++s == p.stages) { s = 0; ++round; }
            }
            for (int i = 0; i < p.stages; ++i) mbar_landed(&ctrl->full[i], (issued + p.stages - 1 - i) / p.stages, &ctrl->zero, status);
        }
        __syncwarp();
    } else if (warp == 5) {
        if (elect_one()) {
            const uint32_t idesc = idesc_of(BM, p.nt, p.p_mn, p.q_mn);
            const uint64_t step_p = p.p_mn ? 2048 >> 4 : 2, step_q = p.q_mn ? 2048 >> 4 : 2;  // 16 k
            int s = 0, round = 0, a = 0;
            for (int kb = lo; kb < hi; ++kb) {
                mbar_wait_bounded<false>(&ctrl->full[s], round & 1, &ctrl->abort, status);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t da = desc_of(smem_u32(sm + s * stage_bytes), p.p_mn), db = desc_of(smem_u32(sm + s * stage_bytes + P_BYTES), p.q_mn);
#pragma unroll
                for (int ks = 0; ks < BK / 16; ++ks)
                    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                                 ::"r"(tmem + a * p.nt), "l"(da + ks * step_p), "l"(db + ks * step_q), "r"(idesc), "r"((kb >= lo + p.accs || ks > 0) ? 1u : 0u) : "memory");
                asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&ctrl->empty[s])) : "memory");
                if (++s == p.stages) { s = 0; ++round; }
                if (++a == p.accs) a = 0;
            }
            asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&ctrl->accum)) : "memory");
            if (ctrl->abort) {  // the later waits fell through: wait for what was issued before tensor memory is released
                asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&ctrl->drain)) : "memory");
                mbar_wait_bounded<false>(&ctrl->drain, 0, &ctrl->zero, status);
            }
        }
        __syncwarp();
    }
    __syncwarp();
    if (warp < 4) {
        mbar_wait_bounded<true>(&ctrl->accum, 0, &ctrl->abort, status, SUM_LIMIT);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (p.splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();  // the ring, where the result goes, is read no more, and its last copies have landed
    const int pitch = part_pitch(p.nt), rows = BM / p.splits;
    if (p.direct) {
        // nothing to join: from the accumulator to the result
        if (warp < 4 && !ctrl->abort) {
            const Epi& e = p.e;
            const bool mixed = e.z && e.z_f32 != e.y_f32;
            float* mine = parts + warp * 1024;
            const uint32_t acc = tmem + ((uint32_t)(32 * warp) << 16);
            int turn = 0;
#pragma unroll 1
            for (int c = 0; c < p.nt; c += 32) {
                auto sums = [&](float (&v)[32]) {
                    tmem_ld32(acc + c, reinterpret_cast<uint32_t(&)[32]>(v));
                    for (int a = 1; a < min(p.accs, hi - lo); ++a) {
                        float u[32];
                        tmem_ld32(acc + a * p.nt + c, reinterpret_cast<uint32_t(&)[32]>(u));
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] += u[i];
                    }
                };
                // (blocks two by two, as the pairs have them, would take 190 registers and more: one CTA an SM)
                const int row0 = p0 + 32 * warp, col0 = q0 + c;
                if (row0 >= e.rows || col0 >= e.cols) continue;
                if (e.vec) finish_rows<ACT>(e, &p.Y, &p.Z, mine, mixed, lane, turn, row0, col0, sums);
                else finish_cols<ACT>(e, &p.Y, &p.Z, mine, mixed, lane, turn, row0, col0, [&](float (&v)[32]) { sums(v); turn_block(mine, lane, v); });
            }
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();
        if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
        return;
    }
    if (warp < 4) {
        // a lane has a row of the accumulators and sends it to the CTA that finishes it
        const int row = 32 * warp + lane;
        const uint32_t to = map_rank(smem_u32(parts + (rank * rows + row % rows) * pitch), row / rows);
#pragma unroll 1
        for (int c = 0; c < p.nt; c += 16) {
            uint32_t v[16];
            tmem_ld16(tmem + ((uint32_t)(32 * warp) << 16) + c, v);
            for (int a = 1; a < min(p.accs, hi - lo); ++a) {
                uint32_t u[16];
                tmem_ld16(tmem + ((uint32_t)(32 * warp) << 16) + a * p.nt + c, u);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(u[i]));
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (c + i) * 4), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]) : "memory");
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (p.splits > 1) cluster_sync();
    else __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");

    // this CTA's rows of the tile: the parts are added in the order of their ranks
    if (ctrl->abort) return;
    const Epi& e = p.e;
    const int r0 = rank * rows;
    if (p.swap) {  // a thread has four of Q's indices, lanes run along P, i.e. along a row of y
        for (int u = tid; u < rows * (p.nt / 4); u += TILE_THREADS) {
            const int i = u % rows, j = u / rows * 4;
            const long long col = p0 + r0 + i;
            if (col >= e.cols || q0 + j >= e.rows) continue;
            float4 x = ld4(parts + i * pitch + j);
            for (int r = 1; r < p.splits; ++r) {
                const float4 y = ld4(parts + (r * rows + i) * pitch + j);
                x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
            }
            const float bias = e.bias ? load1g(e.bias, e.bias_f32, col) : 0.f;
            const float f[4] = {x.x + bias, x.y + bias, x.z + bias, x.w + bias};
            float res[4] = {};
            if (e.residual)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (q0 + j + q < e.rows) res[q] = load1g(e.residual, e.y_f32, (long long)(q0 + j + q) * e.ldr + col);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const long long row = q0 + j + q;
                if (row >= e.rows) break;
                if (e.z) store_z1(e, row, col, f[q]);
                const float v = act<ACT>(f[q]) + res[q];
                if (e.y_f32) ((float*)e.y)[row * e.ldy + col] = v;
                else ((bf16*)e.y)[row * e.ldy + col] = __float2bfloat16_rn(v);
            }
        }
    } else {
        const int per_row = p.nt / 8, units = rows * per_row;
        const long long plane = (long long)gridDim.x / shares * BM * p.nt;
        float* const mine = p.sums + (tile * BM + r0) * p.nt;
        auto joined = [&](int u, float (&f)[8]) {  // the cluster's parts
            const int i = u / per_row, j = 8 * (u % per_row);
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = 0.f;
            for (int r = 0; r < p.splits; ++r) {
                const float* x = parts + (r * rows + i) * pitch + j;
                const float4 a = ld4(x), b = ld4(x + 4);
                f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w; f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
            }
        };
        if (p.outer > 1) {
            for (int u = tid; u < units; u += TILE_THREADS) {
                float f[8];
                joined(u, f);
                float4* to = reinterpret_cast<float4*>(mine + cluster * plane + 8 * u);
                __stcg(to, make_float4(f[0], f[1], f[2], f[3]));
                __stcg(to + 1, make_float4(f[4], f[5], f[6], f[7]));
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) ctrl->last = atomicAdd(p.arrived + tile * p.splits + rank, 1u) == (unsigned)p.outer - 1;
            __syncthreads();
            if (!ctrl->last) return;
            __threadfence();
        }
        for (int u = tid; u < units; u += TILE_THREADS) {
            const int i = u / per_row, j = 8 * (u % per_row);
            const long long row = p0 + r0 + i, col = q0 + j;
            if (row >= e.rows || col >= e.cols) continue;
            float f[8];
            if (p.outer > 1) {
#pragma unroll
                for (int q = 0; q < 8; ++q) f[q] = 0.f;
#pragma unroll 4
                for (int c = 0; c < p.outer; ++c) {
                    const float4* x = reinterpret_cast<const float4*>(mine + c * plane + 8 * u);
                    const float4 a = __ldcg(x), b = __ldcg(x + 1);
                    f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w; f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
                }
            } else {
                joined(u, f);
            }
            if (e.bias) {
                float bias[8];
                bias8(e, col, bias);
#pragma unroll
                for (int q = 0; q < 8; ++q) f[q] += bias[q];
            }
            finish8<ACT>(e, row, col, f);
        }
    }
}

// ---- pairs of CTAs, persistent ------------------------------------------------------------------------------------
// A pair takes every pairs-th tile.  What is left when the tiles no longer fill all pairs (`whole` is a multiple of their number) is cut along k, `splits` units
// to a tile, so that the last round takes a part of a tile's time: each unit writes its sums to the workspace, and of the warps that do so for one block of a tile the
// last to arrive adds all parts, in their order, and finishes the block.  Nobody waits for another.
struct PairParams {
    CUtensorMap P, Q, Y, Z;  // Y, Z: boxes of 32 x 32 for the results' bulk stores, where rows of y are aligned
    Epi e;
    int p_mn, q_mn, bn, kblocks, p_tiles, q_tiles, swap, splits;  // swap: P runs over the columns of y, Q over its rows
    long long tiles, whole;
    float4* parts;         // [units of the cut tiles][CTA of the pair][warp][block][8][lane]
    unsigned* arrived;     // [cut tiles][CTA][warp], zero
};
constexpr int PAIR_STAGES = 6, PAIR_THREADS = 384;  // warp 0: copies, 1: products, 4-11: epilogue
constexpr int PAIR_P = BM * 128, PAIR_Q = 128 * 128, PAIR_STAGE = PAIR_P + PAIR_Q;
constexpr int PAIR_STAGING = 32 * 32 * 4;  // a block of 32 x 32 in fp32, or two in bf16, per epilogue warp
constexpr int BAND = 8;                    // tile rows of 256 that are walked together, column by column, so that concurrent tiles share operands in L2
constexpr int PART_BLOCKS = 4;             // blocks of 32 columns a warp has of a tile at most
constexpr int PART_F4 = 2 * 8 * PART_BLOCKS * 8 * 32;  // float4 of a unit
struct PairCtrl {
    uint64_t full[PAIR_STAGES], empty[PAIR_STAGES], accum_full[2], accum_empty[2], drain;
    uint32_t tmem_base;
    volatile int abort, zero;
};
constexpr int PAIR_SMEM = 1024 + PAIR_STAGES * PAIR_STAGE + 8 * PAIR_STAGING + (int)sizeof(PairCtrl);
static_assert(PAIR_SMEM <= 232448, "shared memory of a CTA");

// the n-th piece of work of a pair
struct PairWork {
    int pi, qi, lo, hi;  // tile, k blocks
    int unit, cut;       // of a cut tile: unit among all, and which of the cut tiles; -1: a whole one
};
__device__ __forceinline__ bool pair_work(const PairParams& p, int n, PairWork& w) {
    const long long pairs = gridDim.x >> 1, pair = blockIdx.x >> 1;
    long long t = n * pairs + pair;
    w.lo = 0; w.hi = p.kblocks; w.unit = w.cut = -1;
    if (t >= p.whole) {
        const long long u = t - p.whole;  // (whole is a multiple of the number of pairs)
        if (u >= (p.tiles - p.whole) * p.splits) return false;
        const int part = (int)(u % p.splits);
        t = p.whole + u / p.splits;
        if (p.splits > 1) {
            w.unit = (int)u;
            w.cut = (int)(t - p.whole);
            w.lo = (int)((long long)p.kblocks * part / p.splits);
            w.hi = (int)((long long)p.kblocks * (part + 1) / p.splits);
        }
    }
    const long long per_band = (long long)BAND * p.q_tiles;
    const int band = (int)(t / per_band), rows = min(BAND, p.p_tiles - band * BAND);
    const int r = (int)(t - band * per_band);
    w.pi = band * BAND + r % rows;
    w.qi = r / rows;
    return true;
}

__global__ void __launch_bounds__(256) linear_zero_kernel(unsigned* p, int n) {
    stream_order();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

template <int ACT> __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1) linear_pair_kernel(const __grid_constant__ PairParams p, int* status) {
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* sm = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    unsigned char* staging = sm + PAIR_STAGES * PAIR_STAGE;
    PairCtrl* ctrl = reinterpret_cast<PairCtrl*>(staging + 8 * PAIR_STAGING);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t rank = cluster_rank();

    if (tid == 0) {
        for (int s = 0; s < PAIR_STAGES; ++s) { mbar_init(&ctrl->full[s], 1); mbar_init(&ctrl->empty[s], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&ctrl->accum_full[i], 1); mbar_init(&ctrl->accum_empty[i], 16); }
        mbar_init(&ctrl->drain, 1);
        ctrl->abort = 0; ctrl->zero = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for behind the rest of the preparation)
    if (warp == 3 && elect_one()) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&p.P) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&p.Q) : "memory");
    }
    if (warp == 2) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctrl->tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the other CTA's barriers are set up
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = ctrl->tmem_base;
    stream_wait();

    PairWork w;
    if (warp == 0) {
        if (elect_one()) {
            const int half = p.bn / 2;
            const uint32_t q_tx = p.q_mn ? (uint32_t)((half + 63) / 64) * 8192u : (uint32_t)half * 128u;
            int s = 0, round = 0;
            long long issued = 0;
            bool going = true;
            for (int n = 0; going && pair_work(p, n, w); ++n) {
                const int p0 = w.pi * 2 * BM + (int)rank * BM, q0 = w.qi * p.bn + (int)rank * half;
                for (int kb = w.lo; kb < w.hi; ++kb) {
                    if (round > 0 && !mbar_wait_bounded<true>(&ctrl->empty[s], (round - 1) & 1, &ctrl->abort, status)) { going = false; break; }
                    // both CTAs' copies count at the first CTA's barrier, whose thread issues the products
                    if (rank == 0) expect_tx(&ctrl->full[s], 2 * (PAIR_P + q_tx));
                    const uint32_t bar = map_rank(smem_u32(&ctrl->full[s]), 0), dst = smem_u32(sm + s * PAIR_STAGE);
                    auto load = [&](const CUtensorMap* m, uint32_t to, int x, int y) {
                        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
                                     ::"r"(to), "l"(m), "r"(bar), "r"(x), "r"(y) : "memory");
                    };
                    if (p.p_mn) { load(&p.P, dst, p0, kb * BK); load(&p.P, dst + 8192, p0 + 64, kb * BK); }
                    else load(&p.P, dst, kb * BK, p0);
                    if (p.q_mn) for (int b = 0; b < half; b += 64) load(&p.Q, dst + PAIR_P + b * 128, q0 + b, kb * BK);
                    else load(&p.Q, dst + PAIR_P, kb * BK, q0);
                    ++issued;
                    if (++s == PAIR_STAGES) { s = 0; ++round; }
                }
            }
            stream_release();
            // this CTA's copies have landed when the products that read them are done, of which both CTAs hear
            for (int i = 0; i < PAIR_STAGES; ++i) {
                const long long n = (issued + PAIR_STAGES - 1 - i) / PAIR_STAGES;
                if (n > 0) mbar_wait_bounded<true>(&ctrl->empty[i], (uint32_t)(n - 1) & 1, &ctrl->zero, status);
            }
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        if (elect_one()) {
            const uint32_t idesc = idesc_of(2 * BM, p.bn, p.p_mn, p.q_mn);
            const uint64_t step_p = p.p_mn ? 2048 >> 4 : 2, step_q = p.q_mn ? 2048 >> 4 : 2;
            auto commit = [](uint64_t* bar) {
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
            };
            int s = 0, round = 0;
            for (int n = 0; pair_work(p, n, w); ++n) {
                const int buf = n & 1;
                if (n >= 2) mbar_wait_bounded<false>(&ctrl->accum_empty[buf], ((n >> 1) - 1) & 1, &ctrl->abort, status);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t acc = tmem + buf * 256;
                for (int kb = w.lo; kb < w.hi; ++kb) {
                    mbar_wait_bounded<false>(&ctrl->full[s], round & 1, &ctrl->abort, status);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t da = desc_of(smem_u32(sm + s * PAIR_STAGE), p.p_mn), db = desc_of(smem_u32(sm + s * PAIR_STAGE + PAIR_P), p.q_mn);
#pragma unroll
                    for (int ks = 0; ks < BK / 16; ++ks)
                        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                                     ::"r"(acc), "l"(da + ks * step_p), "l"(db + ks * step_q), "r"(idesc), "r"((kb > w.lo || ks > 0) ? 1u : 0u) : "memory");
                    commit(&ctrl->empty[s]);
                    if (++s == PAIR_STAGES) { s = 0; ++round; }
                }
                commit(&ctrl->accum_full[buf]);
            }
            if (ctrl->abort) {
                commit(&ctrl->drain);
                mbar_wait_bounded<false>(&ctrl->drain, 0, &ctrl->zero, status);
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // Warps 4-7 take the first half of the tile's Q indices, 8-11 the second; a warp reads the 32 accumulator rows that it may, 32 columns at a time: a lane has
        // a row of y (swap: a column).  Bias, activation and residual are applied as it lies; the block leaves through shared memory by a bulk tensor store,
        // whose swizzle (16-byte pieces, xor of the row) spares bank conflicts.  That is 16 wavefronts of shared memory a block of bf16: the operands'
        // copies and products need all but an eighth of its bandwidth.  (Through shared memory in fp32 and out by 16-byte stores: 64 and the stores'.)
        // Where rows of y are not aligned the block is turned there in fp32, so that a lane has a column.
        const int quarter = warp & 3, side = (warp - 4) >> 2;
        float* mine = reinterpret_cast<float*>(staging + (warp - 4) * PAIR_STAGING);
        int turn = 0;
        const Epi& e = p.e;
        const bool two = e.vec && !p.swap && !e.y_f32 && !(e.z && e.z_f32);  // blocks go two by two
        const bool mixed = two || (e.z && e.z_f32 != e.y_f32);               // stores do not take the staging area's halves in turn
        const int blocks = p.bn / 32, b0 = side ? (blocks + 1) / 2 : 0, b1 = side ? blocks : (blocks + 1) / 2;
        for (int n = 0; pair_work(p, n, w); ++n) {
            const int buf = n & 1;
            if (e.residual) {  // on its way to L2 while the products go on: a lane's row of a block, 64 or 128 bytes
                for (int b = b0; b < b1; ++b) {
                    const long long q0 = (long long)w.qi * p.bn + 32 * b, first = (long long)w.pi * 2 * BM + rank * BM + 32 * quarter;
                    const long long row = (p.swap ? q0 : first) + lane, col = p.swap ? first : q0;
                    if (row < e.rows && col < e.cols) asm volatile("prefetch.global.L2 [%0];" ::"l"((const unsigned char*)e.residual + (row * e.ldr + col) * (e.y_f32 ? 4 : 2)));
                }
            }
            mbar_wait_bounded<true>(&ctrl->accum_full[buf], (n >> 1) & 1, &ctrl->abort, status, SUM_LIMIT);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (ctrl->abort) break;
            const long long p0 = (long long)w.pi * 2 * BM + rank * BM + 32 * quarter;
            const uint32_t acc = tmem + buf * 256 + ((uint32_t)(32 * quarter) << 16);
            auto emptied = [&] {  // the accumulator may be filled again (no memory is handed over: a release would wait for all of this warp's stores, 1600 cycles)
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(map_rank(smem_u32(&ctrl->accum_empty[buf]), 0)) : "memory");
            };
            float4* parts = nullptr;
            if (w.cut >= 0) {  // this unit's sums to memory; the last of the tile's units goes on
                parts = p.parts + ((rank * 8 + warp - 4) * PART_BLOCKS) * 256 + lane;
                float4* to = parts + (long long)w.unit * PART_F4;
#pragma unroll 1
                for (int b = b0; b < b1; ++b) {
                    uint32_t v[32];
                    tmem_ld32(acc + 32 * b, v);
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        __stcg(to + (b - b0) * 256 + u * 32, make_float4(__uint_as_float(v[4 * u]), __uint_as_float(v[4 * u + 1]), __uint_as_float(v[4 * u + 2]), __uint_as_float(v[4 * u + 3])));
                }
                emptied();
                __threadfence();
                __syncwarp();
                unsigned before = 0;
                if (lane == 0) before = atomicAdd(p.arrived + (w.cut * 2 + rank) * 8 + warp - 4, 1u);
                if (__shfl_sync(0xffffffffu, before, 0) != (unsigned)p.splits - 1) continue;
                __threadfence();
                parts += (long long)w.cut * p.splits * PART_F4;
            }
#pragma unroll 1
            for (int b = b0; b < b1; ++b) {
                const long long q0 = (long long)w.qi * p.bn + 32 * b;
                const long long row0 = p.swap ? q0 : p0, col0 = p.swap ? p0 : q0;
                if (two && !parts && b + 1 < b1 && row0 < e.rows && col0 + 64 <= e.cols) {
                    finish_rows_two<ACT>(e, &p.Y, &p.Z, mine, lane, row0, col0, [&](float (&v)[2][32]) {
                        tmem_ld32(acc + 32 * b, reinterpret_cast<uint32_t(&)[32]>(v[0]));
                        tmem_ld32(acc + 32 * b + 32, reinterpret_cast<uint32_t(&)[32]>(v[1]));
                        if (b + 1 == b1 - 1) emptied();
                    });
                    ++b;
                    continue;
                }
                auto sums = [&](float (&v)[32]) {
                    if (parts) {
                        const float4* from = parts + (b - b0) * 256;
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0.f;
#pragma unroll 2
                        for (int c = 0; c < p.splits; ++c, from += PART_F4) {
                            float4 x[8];
#pragma unroll
                            for (int u = 0; u < 8; ++u) x[u] = __ldcg(from + u * 32);
#pragma unroll
                            for (int u = 0; u < 8; ++u) { v[4 * u] += x[u].x; v[4 * u + 1] += x[u].y; v[4 * u + 2] += x[u].z; v[4 * u + 3] += x[u].w; }
                        }
                    } else {
                        tmem_ld32(acc + 32 * b, reinterpret_cast<uint32_t(&)[32]>(v));
                        if (b == b1 - 1) emptied();
                    }
                };
                if (row0 >= e.rows || col0 >= e.cols) {
                    if (b == b1 - 1 && !parts) emptied();
                    continue;
                }
                if (p.swap) finish_cols<ACT>(e, &p.Y, &p.Z, mine, mixed, lane, turn, row0, col0, sums);
                else if (e.vec) finish_rows<ACT>(e, &p.Y, &p.Z, mine, mixed, lane, turn, row0, col0, sums);
                else finish_cols<ACT>(e, &p.Y, &p.Z, mine, mixed, lane, turn, row0, col0, [&](float (&v)[32]) { sums(v); turn_block(mine, lane, v); });
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // shared memory must outlive the stores' reads
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();  // all that arrives at the other CTA's barriers has arrived, and neither reads the accumulators any more
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---- dz and the bias' gradient ---------------------------------------------------------------------------------
// A CTA has 256 columns (8 adjacent ones a thread) of a chunk of rows, four rows of a thread requested at a time (104 to 220 bytes of a thread's 80 registers'
// worth are spilled in the bf16 forms, for three CTAs an SM).  Bound by DRAM: 8192 x 8192, relu2, 403 MB in 65 us.  Column sums go through memory chunk by chunk, so that they are the same from call to call.
constexpr int DZ_COLS = 256, DZ_THREADS = 256;
struct DzParams : LinearDz {
    long long rows_per;
    bool vec;  // rows of dy and saved start on 16-byte boundaries
};
// WIDE: dy or saved is in fp32 (which of them, is looked up)
template <int ACT, bool FROM_Y, bool WIDE> __global__ void __launch_bounds__(DZ_THREADS, WIDE ? 2 : 3) linear_dz_kernel(const __grid_constant__ DzParams p) {
    stream_order();
    __shared__ float sums[8][DZ_COLS + 4];
    const int g = threadIdx.x & 31, r = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * DZ_COLS + 8 * g;
    const long long lo = blockIdx.y * p.rows_per, hi = lo + p.rows_per < p.M ? lo + p.rows_per : p.M;
    float acc[8] = {};
    if (col < p.N) {
        auto row = [&](long long m, float (&d)[8], const float (&z)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (ACT) d[i] = __fmul_rn(d[i], act_grad<ACT, FROM_Y>(z[i]));  // (not merged into the sum: dbias is the same whether dz is wanted or not)
                acc[i] += d[i];
            }
            if (p.dz) *reinterpret_cast<uint4*>((bf16*)p.dz + m * p.ldz + col) = pack8(d);  // (ldz is a multiple of 8)
        };
        const bool dy_f32 = WIDE && p.dy_f32, z_f32 = WIDE && p.saved_f32;
        // rows a thread has requested at a time; behind the chunk's end the last one again, not stored and not summed
        constexpr int AHEAD = 4, EDGE = 2;
        if (p.vec && col + 8 <= p.N) {
            for (long long m = lo + r; m < hi; m += 8 * AHEAD) {
                Words8 dw[AHEAD], zw[AHEAD];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    const long long n = m + 8 * a < hi ? m + 8 * a : m;
                    dw[a] = request8(p.dy, dy_f32, n * p.lddy + col);
                    if (ACT) zw[a] = request8(p.saved, z_f32, n * p.lds + col);
                }
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    float d[8], z[8];
                    floats8(dw[a], dy_f32, d);
                    if (ACT) floats8(zw[a], z_f32, z);
                    if (m + 8 * a < hi) row(m + 8 * a, d, z);
                }
            }
        } else {
            for (long long m = lo + r; m < hi; m += 8 * EDGE) {
                float d[EDGE][8], z[EDGE][8];
#pragma unroll
                for (int a = 0; a < EDGE; ++a) {
                    const long long n = m + 8 * a < hi ? m + 8 * a : m;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const long long c = col + i < p.N ? col + i : p.N - 1;  // (columns behind the last: that one again, and zero)
                        d[a][i] = load1g(p.dy, dy_f32, n * p.lddy + c);
                        if (ACT) z[a][i] = load1g(p.saved, z_f32, n * p.lds + c);
                    }
                }
#pragma unroll
                for (int a = 0; a < EDGE; ++a) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (col + i >= p.N) d[a][i] = 0.f;
                    if (m + 8 * a < hi) row(m + 8 * a, d[a], z[a]);
                }
            }
        }
    }
    if (!p.dbias) return;
    *reinterpret_cast<float4*>(&sums[r][8 * g]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    *reinterpret_cast<float4*>(&sums[r][8 * g + 4]) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    __syncthreads();
    const long long c = (long long)blockIdx.x * DZ_COLS + threadIdx.x;
    if (c < p.N) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += sums[i][threadIdx.x];
        p.partial[blockIdx.y * p.N + c] = s;
    }
}
__global__ void __launch_bounds__(256) linear_dbias_kernel(const float* partial, float* dbias, long long N, int chunks) {
    stream_order();
    __shared__ float sums[8][33];
    const int x = threadIdx.x & 31, r = threadIdx.x >> 5;
    const long long c = (long long)blockIdx.x * 32 + x;
    float s = 0.f;
    if (c < N)
        for (int i = r; i < chunks; i += 8) s += partial[i * N + c];
    sums[r][x] = s;
    __syncthreads();
    if (r == 0 && c < N) {
        for (int i = 1; i < 8; ++i) s += sums[i][x];
        dbias[c] = s;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    return fn;
}
// box_rows: indices of a K-major box; an MN-major one is 64 indices x 64 k
static bool encode(CUtensorMap* m, const LinearOperand& o, long long n, long long k, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)(o.mn ? n : k), (cuuint64_t)(o.mn ? k : n)};
    const cuuint64_t strides[1] = {(cuuint64_t)o.ld * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)(o.mn ? BK : box_rows)};
    const cuuint32_t es[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// results: boxes of 32 columns x 32 rows
static bool encode_out(CUtensorMap* m, const void* p, bool f32, long long rows, long long cols, long long ld) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * (f32 ? 4 : 2)};
    const cuuint32_t box[2] = {32, 32}, es[2] = {1, 1};
    return fn(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static bool encode_results(const Epi& e, CUtensorMap* Y, CUtensorMap* Z) {
    return encode_out(Y, e.y, e.y_f32, e.rows, e.cols, e.ldy) && (!e.z || encode_out(Z, e.z, e.z_f32, e.rows, e.cols, e.ldz));
}

static thread_local uint32_t smem_allowed[64];
template <typename P> struct Kernels { void (*k[kActs])(P, int*); };
#define WKV7_PER_ACT(kernel) {{kernel<kActNone>, kernel<kActRelu>, kernel<kActRelu2>, kernel<kActTanh>, kernel<kActSigmoid>, kernel<kActSilu>, kernel<kActGelu>}}
static const Kernels<TileParams> tile_kernels = WKV7_PER_ACT(linear_tile_kernel);
static const Kernels<PairParams> pair_kernels = WKV7_PER_ACT(linear_pair_kernel);

static int run_tile(LinearOperand a, LinearOperand b, long long na, long long nb, long long k, const Epi& e, bool swap, int nt, int splits, int outer, void* workspace, int* status,
                    cudaStream_t stream) {
    const auto kern = tile_kernels.k[e.act];
    if (!allow_smem(kern, smem_allowed, e.act, 227 * 1024)) return kLaunchFailed;
    TileParams p;
    memset(&p, 0, sizeof(p));
    if (!encode(&p.P, a, na, k, BM) || !encode(&p.Q, b, nb, k, nt)) return kLaunchFailed;
    p.e = e;
    p.p_mn = a.mn; p.q_mn = b.mn; p.nt = nt; p.swap = swap;
    p.outer = outer;
    p.direct = !swap && splits == 1 && outer == 1;
    if (p.direct && e.vec && !encode_results(e, &p.Y, &p.Z)) return kLaunchFailed;
    p.kblocks = (int)((k + BK - 1) / BK);
    p.splits = splits;
    p.p_tiles = (int)((na + BM - 1) / BM);
    const long long tiles = p.p_tiles * ((nb + nt - 1) / nt), grid = tiles * splits * outer;
    if (grid > 0x7fffffffLL) return kTooLarge;
    if (outer > 1) {
        p.sums = (float*)workspace;
        p.arrived = (unsigned*)((char*)workspace + tiles * outer * BM * nt * 4);
        if (!launch(linear_zero_kernel, dim3((unsigned)((tiles * splits + 255) / 256)), 256, 0, stream, p.arrived, (int)(tiles * splits))) return kLaunchFailed;
    }
    const int stage = P_BYTES + q_bytes(nt), part = part_bytes(nt), most = (p.kblocks + splits * outer - 1) / (splits * outer);
    // Two CTAs share an SM where there are more than SMs, and in clusters of four and eight of narrow tiles (they do not find whole free SMs everywhere)
    // and three where the tiles of a wide weight then all run at once (16 x 2048 x 50001: 41 -> 37 us)
    const int per_sm = splits == 1 && nt <= 32 && grid > 2 * sm_count() ? 3 : grid > sm_count() || (splits > 2 && nt <= 64) ? 2 : 1;
    const int room = 227 * 1024 / per_sm - 1024 - 2048 - (splits > 1 ? part : 0);  // (the system has a KB of each CTA's)
    p.stages = room / stage;
    if (p.stages < 2) p.stages = 2;
    if (p.stages > MAXSTAGES) p.stages = MAXSTAGES;
    if (p.stages > most) p.stages = most;
    // Products of one accumulator follow one another with its rounding, which cuts: the error of a long sum grows with its length, as it does in the library's products
    // (fp32 results of 2048 x 2048: 2.1e-6 at K = 2048, 9.1e-6 at 8192, 7.6e-5 at 65536, nearly all of it towards zero; the library's the same).  Where tensor
    // memory has room k blocks go to several accumulators in turn, which are added in the end (16 rows, K = 2048: 1e-7; 333 x 512: 2.3e-7, at K = 8192 1e-6).
    p.accs = 128 / nt;
    if (p.accs > most) p.accs = most;
    p.tmem_cols = 32;
    while ((int)p.tmem_cols < nt * p.accs) p.tmem_cols *= 2;
    const int ring = splits > 1 ? p.stages * stage + part : p.stages * stage > part ? p.stages * stage : part;
    return launch_clusters(kern, dim3((unsigned)grid), TILE_THREADS, 2048 + ring, splits, stream, p, status) ? kOk : kLaunchFailed;
}

static long long pairs_of_sms() { const int n = sm_count() / 2; return n > 0 ? n : 1; }  // (asked for sizes without a device, too)
// How a product is cut into tiles of 256 x bn for the pairs.
struct PairPlan {
    int bn, splits;
    bool swap;
    long long tiles, whole;
    double time;  // in k blocks of a tile of 256 x 256
};
static PairPlan plan_pair(long long rows, long long cols, int kblocks, bool can_swap, bool can_split) {
    const long long pairs = pairs_of_sms();
    PairPlan best{};
    for (int swap = 0; swap <= (can_swap ? 1 : 0); ++swap)
        for (int bn = 256; bn >= 128; bn -= 32) {
            const long long np = swap ? cols : rows, nq = swap ? rows : cols;
            PairPlan x{bn, 1, swap != 0, ((np + 255) / 256) * ((nq + bn - 1) / bn), 0, 0.};
            x.whole = x.tiles / pairs * pairs;
            const long long left = x.tiles - x.whole;
            // a k block of a tile of 256 x bn, relative to bn = 256 and its width: narrow tiles wait for operands (8192 x 8192 x 2048, us: 256 175, 224 180 to 187,
            // 192 196 to 211, 128 233 to 282; columns of y along P, where the tiles are not square, is a little better: 64-byte pieces that fill whole lines)
            static constexpr double factor[5] = {1.45, 1.22, 1.12, 1.05, 1.};
            const double each = factor[bn / 32 - 4] * (bn / 256.) * (swap ? 1.01 : bn < 256 ? 1.04 : 1.);
            // the last round: as it is, or cut, which costs 8 k blocks' time and 8 for each part that is written and read (8192 x 2048, K = 8192: 202 -> 184 us)
            double last = left ? kblocks : 0;
            if (left && can_split)
                for (int c = 2; c <= 8 && left * c <= pairs; ++c) {
                    const double cut = (kblocks + c - 1) / c + 8 + 8 * c;
                    if (cut < last) { last = cut; x.splits = c; }
                }
            x.time = ((double)(x.whole / pairs) * kblocks + last) * each;
            if (!best.bn || x.time < best.time) best = x;
        }
    return best;
}
static size_t pair_ws(const PairPlan& x) { return x.splits > 1 ? (size_t)(x.tiles - x.whole) * ((size_t)x.splits * PART_F4 * 16 + 64) : 0; }

static int run_pair(LinearOperand rows, LinearOperand cols, long long k, const Epi& e, const PairPlan& x, void* workspace, int* status, cudaStream_t stream) {
    const auto kern = pair_kernels.k[e.act];
    if (!allow_smem(kern, smem_allowed, 16 + e.act, PAIR_SMEM)) return kLaunchFailed;
    PairParams p;
    memset(&p, 0, sizeof(p));
    const LinearOperand &a = x.swap ? cols : rows, &b = x.swap ? rows : cols;
    const long long na = x.swap ? e.cols : e.rows, nb = x.swap ? e.rows : e.cols;
    if (!encode(&p.P, a, na, k, BM) || !encode(&p.Q, b, nb, k, x.bn / 2)) return kLaunchFailed;
    if (e.vec && !encode_results(e, &p.Y, &p.Z)) return kLaunchFailed;
    p.e = e;
    p.p_mn = a.mn; p.q_mn = b.mn; p.bn = x.bn; p.swap = x.swap; p.splits = x.splits;
    p.kblocks = (int)((k + BK - 1) / BK);
    p.p_tiles = (int)((na + 2 * BM - 1) / (2 * BM));
    p.q_tiles = (int)((nb + x.bn - 1) / x.bn);
    p.tiles = x.tiles; p.whole = x.whole;
    if (x.splits > 1) {
        const int cut = (int)(x.tiles - x.whole);
        p.parts = (float4*)workspace;
        p.arrived = (unsigned*)((char*)workspace + (size_t)cut * x.splits * PART_F4 * 16);
        if (!launch(linear_zero_kernel, dim3((cut * 16 + 255) / 256), 256, 0, stream, p.arrived, cut * 16)) return kLaunchFailed;
    }
    const long long pairs = pairs_of_sms(), units = x.whole + (x.tiles - x.whole) * x.splits;
    const unsigned grid = 2 * (unsigned)(units < pairs ? units : pairs);
    return launch_clusters(kern, dim3(grid), PAIR_THREADS, PAIR_SMEM, 1, stream, p, status) ? kOk : kLaunchFailed;
}

// Which kernel, and its shape
struct Plan {
    bool pair, swap;
    int nt, splits, outer;  // of tiles of 128 x nt
    PairPlan x;
};
static Plan make_plan(long long rows, long long cols, long long k, bool rows_mn, bool can_split) {
    const int kblocks = (int)((k + BK - 1) / BK), sms = sm_count();
    Plan p{};
    p.outer = 1;
    auto split = [&](long long tiles, int most, int places) {  // CTAs of one tile: as many as there are places for
        int s = 1;
        while (s < most && 2 * s <= kblocks && tiles * s * 2 <= places) s *= 2;
        return s;
    };
    if (rows <= 64 && !rows_mn) {
        p.swap = true;
        p.nt = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
        // us, shared out over 1, 2, 4 and 8 CTAs a tile, two an SM: 1 x 2048 x 8192 12, 9.8, 9.7, 15; 1 x 8192 x 2048 37, 19, 12.7, 10; 1 x 2560 x 10240 14, 12.4, 17, -;
        // 16 x 2048 x 50001 42, 46, -, -; 64 x 2048 x 2048 (parts of 34 KB) -, 11, 8.7, 9.1
        p.splits = split((cols + BM - 1) / BM, p.nt == 64 ? 4 : 8, 2 * sms);
        return p;
    }
    // In us: pairs 7 and 0.3 for a k block of 256 x 256; tiles of 128 x 128 and 128 x 64, one after the other on an SM, 6 (1.5 more to join parts) and 0.27 or 0.2 for
    // a k block, which is what their operands take from L2.
    // (Not looked at where they would be fewer than eight: planning takes the host a us.)
    double best = 1e30;
    if (((rows + 255) / 256) * ((cols + 127) / 128) >= 8) {
        p.x = plan_pair(rows, cols, kblocks, true, can_split);
        best = 7. + 0.3 * p.x.time;
        p.pair = true;
    }
    for (int nt = 128; nt >= 64; nt /= 2) {
        const long long tiles = ((rows + BM - 1) / BM) * ((cols + nt - 1) / nt);
        // (clusters of four with an SM to each CTA do not use all SMs: 36 of them ran in two rounds)
        int s = split(tiles, nt == 128 ? 4 : 8, sms);
        if (nt == 128 && s == 4 && tiles * s > sms - sms / 8) s = 2;
        // few tiles and a long sum (the gradient of a narrow weight): several clusters to a tile, 16 k blocks or more to each CTA
        long long outer = can_split ? sms / (tiles * s) : 1;
        if (outer > kblocks / (16 * s)) outer = kblocks / (16 * s);
        if (outer > 32) outer = 32;
        if (outer < 2) outer = 1;
        const double rounds = (double)((tiles * s * outer + sms - 1) / (sms > 0 ? sms : 1));
        const double t = 6. + (s > 1 ? 1.5 : 0.) + (outer > 1 ? 4. + 0.15 * outer : 0.) + rounds * ((kblocks + s * outer - 1) / (s * outer)) * (nt == 128 ? 0.27 : 0.2);
        if (t < best) { best = t; p.pair = false; p.nt = nt; p.splits = s; p.outer = (int)outer; }
    }
    return p;
}

}  // namespace lin

size_t linear_workspace_bytes(long long rows, long long cols, long long k, bool rows_mn) {
    const lin::Plan p = lin::make_plan(rows, cols, k, rows_mn, true);
    if (p.pair) return lin::pair_ws(p.x);
    const long long tiles = ((rows + lin::BM - 1) / lin::BM) * ((cols + p.nt - 1) / p.nt);
    return p.outer > 1 ? (size_t)tiles * ((size_t)p.outer * lin::BM * p.nt * 4 + (size_t)p.splits * 4) : 0;
}

int launch_linear(LinearOperand rows, LinearOperand cols, long long k, const LinearEpilogue& ep, void* workspace, int* status, cudaStream_t stream) {
    using namespace lin;
    Epi e;
    static_cast<LinearEpilogue&>(e) = ep;
    const int per16 = ep.y_f32 ? 4 : 8;
    e.vec = al16(ep.y) && ep.ldy % per16 == 0 && ep.cols % per16 == 0 && (!ep.residual || (al16(ep.residual) && ep.ldr % per16 == 0));
    e.bias_vec = al16(ep.bias);
    if ((k + BK - 1) / BK > MAX_KBLOCKS) return kTooLarge;
    const Plan p = make_plan(ep.rows, ep.cols, k, rows.mn, workspace != nullptr);
    if (p.pair) return run_pair(rows, cols, k, e, p.x, workspace, status, stream);
    if (p.swap) return run_tile(cols, rows, ep.cols, ep.rows, k, e, true, p.nt, p.splits, 1, nullptr, status, stream);
    return run_tile(rows, cols, ep.rows, ep.cols, k, e, false, p.nt, p.splits, p.outer, workspace, status, stream);
}

int linear_dz_chunks(long long M, long long N) {
    // CTAs of at least 64 rows, some four to each of 148 SMs
    const long long cols = (N + lin::DZ_COLS - 1) / lin::DZ_COLS;
    long long c = (4 * 148 + cols - 1) / cols;
    const long long most = (M + 63) / 64;
    if (c > most) c = most;
    return (int)(c < 1 ? 1 : c);
}

int launch_linear_dz(const LinearDz& d, cudaStream_t stream) {
    using namespace lin;
    DzParams p;
    static_cast<LinearDz&>(p) = d;
    const int chunks = linear_dz_chunks(d.M, d.N);
    p.rows_per = (d.M + chunks - 1) / chunks;
    p.vec = al16(d.dy) && d.lddy % (d.dy_f32 ? 4 : 8) == 0 && (!d.act || (al16(d.saved) && d.lds % (d.saved_f32 ? 4 : 8) == 0));
    const int cols = (int)((d.N + DZ_COLS - 1) / DZ_COLS);
#define WKV7_DZ(act, from_y) {linear_dz_kernel<act, from_y, false>, linear_dz_kernel<act, from_y, true>}
    static void (*const kern[kActs][2])(DzParams) = {WKV7_DZ(kActNone, false), WKV7_DZ(kActRelu, false), WKV7_DZ(kActRelu2, false), WKV7_DZ(kActTanh, false),
                                                     WKV7_DZ(kActSigmoid, false), WKV7_DZ(kActSilu, false), WKV7_DZ(kActGelu, false)};
    const bool wide = d.dy_f32 || (d.act && d.saved_f32);
    // (relu's derivative is the same function of its value as of its argument)
    const auto k = d.from_y && d.act == kActRelu2 ? linear_dz_kernel<kActRelu2, true, false> : kern[d.act][wide];
    if (!launch(k, dim3(cols, chunks), DZ_THREADS, 0, stream, p)) return kLaunchFailed;
    if (d.dbias && !launch(linear_dbias_kernel, dim3((unsigned)((d.N + 31) / 32)), 256, 0, stream, (const float*)d.partial, d.dbias, d.N, chunks)) return kLaunchFailed;
    return kOk;
}

}  // namespace wkv7

// Beam search next to the decode step: the selection over beams and vocabulary, and the reordering of the states that attn_step keeps.
//
// Selection: score(w, v) = s_w + (l_wv - lse_w), lse_w = log sum_v exp(l_wv); the k best of the W V candidates, equal scores by the lowest w V + v.
// One pass over the logits (beam_scan_kernel) leaves the maximum of every segment of 256 logits and, for every few segments, the sum of exp(l - max);
// nothing else is done per logit.  Bound by DRAM and the start and end of the rows' parts: 64 x 16 x 65536 bf16, 134 MB in 30 to 31 us, 4.3 TB/s (torch's sum of
// 205 MB runs at the same rate); with a quarter of the beams ended 101 MB in 26.  The exponential unit, 16 a cycle and SM, would allow 15 us.
// The second kernel (beam_pick_kernel), a CTA per sequence, needs few logits more: the k best candidates lie in the k segments with the best maxima
// (any other candidate is behind those k maxima).  It finds a threshold t that some k to 2k segments reach, as a rule, reads those again, and
// orders the few candidates that reach t: 10 000 cycles, a chain of latencies (normalisers 3500, threshold and lists 2500, logits 3000, order 1000).  Scores are
// compared in 64 bits: what beams' scores are off by is the sums' own error (4e-7 at most and 4e-8 to 1e-7 in the mean over 592 rows of 65536, at maxima of 13 to 1e6).  t is a lower bound in 32 bits, less what roundings may have added, so nothing that
// belongs to the best is lost.

#include "beam.h"
#include "mma_bf16.cuh"
#include "wkv7_kernels.h"

namespace wkv7 {
namespace beam {

constexpr int SEG = 256;  // logits of a segment: eight a lane
constexpr int SCAN_WARPS = 4;
constexpr float LOWEST = -3.402823466e38f, NEG_INF = -__builtin_huge_valf(), POS_INF = __builtin_huge_valf();

// floats in the order of their values, as unsigned numbers
__device__ __forceinline__ uint32_t ordered(float x) {
    const int i = __float_as_int(x);
    return (uint32_t)i ^ (i < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }
// NaN and +inf rule a candidate out, as -inf does
__device__ __forceinline__ float sane(float x) { return x < POS_INF ? x : NEG_INF; }

// Logits [at, at + 8) of a row, -inf behind its end.
template <bool F32> __device__ __forceinline__ void load_edge(const void* base, long long row, int at, int V, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = at + i < V ? (F32 ? ((const float*)base)[row + at + i] : __bfloat162float(((const bf16*)base)[row + at + i])) : NEG_INF;
}
// 16 bytes of logits (eight, or four in fp32) out of whole 16-byte words, `skip` bytes into the first.  A row may lie on any element's boundary; every lane then
// still has the same logits whatever the alignment, so that equal rows give equal sums.
template <bool F32, bool ALIGNED> __device__ __forceinline__ void take(const unsigned char* b, int skip, float* f) {
    const uint4 w = *reinterpret_cast<const uint4*>(b);
    uint32_t o[4] = {w.x, w.y, w.z, w.w};
    if (!ALIGNED) {
        const uint4 v = *reinterpret_cast<const uint4*>(b + 16);
        const uint32_t x[8] = {w.x, w.y, w.z, w.w, v.x, v.y, v.z, v.w};
        const int words = skip >> 2, bits = (skip & 3) * 8;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (words == c) {  // (the same for the whole row)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = F32 ? x[i + c] : __funnelshift_r(x[i + c], x[i + c + 1 < 8 ? i + c + 1 : 7], bits);
            }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (F32) {
            f[i] = __uint_as_float(o[i]);
        } else {
            f[2 * i] = __uint_as_float(o[i] << 16);
            f[2 * i + 1] = __uint_as_float(o[i] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ float warp_max(float x) {  // (a NaN is passed over)
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max8(const float (&f)[8]) { return fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7]))); }
constexpr float LOG2E = 1.4426950408889634f;
constexpr int AHEAD = 2, DEPTH = 4;  // segments that are worked, and requested, together (a batch); batches of the ring

// A part of a row (segments [first, last)) by a warp, AHEAD segments at a time: their maxima, the part's (m) and the lane's share of sum exp(l - m), formed
// as 2^((l - m) LOG2E).  The difference comes first: it is right for logits of any magnitude (rows masked with -1e9 or the type's lowest value among them), where
// l LOG2E and m LOG2E would each be rounded to their own magnitude.
// The logits come by asynchronous copies into a ring of the warp's own, DEPTH - 1 batches ahead: what a warp has requested takes no registers.
// CAREFUL: NaN and +inf are ruled out one by one; without it such a part's s is a NaN.
template <bool F32, bool ALIGNED> __host__ __device__ constexpr int stage_bytes() { return AHEAD * SEG * (F32 ? 4 : 2) + (ALIGNED ? 0 : 16); }
template <bool F32, bool ALIGNED, bool CAREFUL> __device__ __forceinline__ void scan_part(const BeamParams& p, long long row, int first, int last, float* seg_max, unsigned char* ring, int lane, float& m, float& s) {
    constexpr int SIZE = F32 ? 4 : 2, STAGE = stage_bytes<F32, ALIGNED>(), BATCH = AHEAD * SEG * SIZE;
    const unsigned char* at = (const unsigned char*)p.logits + row * SIZE;
    const int skip = (int)(reinterpret_cast<uintptr_t>(at) & 15);
    at -= skip;
    // whether a batch's words lie within the row (those of an unaligned one reach up to a word further on both sides)
    auto within = [&](int g) { return !CAREFUL && g < last && (ALIGNED || g > 0) && (long long)(g + AHEAD) * SEG + (ALIGNED ? 0 : 8) <= p.V; };
    auto request = [&](int g, int stage) {
        if (within(g)) {
            const unsigned char* from = at + (long long)g * SEG * SIZE;
            unsigned char* to = ring + stage * STAGE;
#pragma unroll
            for (int i = 0; i < BATCH / 512; ++i) cp_async16(to + 512 * i + 16 * lane, from + 512 * i + 16 * lane);
            if (!ALIGNED && lane == 0) cp_async16(to + BATCH, from + BATCH);
        }
        cp_async_commit();
    };
    m = NEG_INF;
    F2 sum = f2(0.f, 0.f);
    int stage = 0;
    if (!CAREFUL)
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) request(first + i * AHEAD, i);
#pragma unroll 1
    for (int g0 = first; g0 < last; g0 += AHEAD) {
        float f[AHEAD][8], top[AHEAD];
        if (!CAREFUL) {
            cp_async_wait<DEPTH - 2>();
            __syncwarp();  // the batch is there for all lanes, and all have taken the one before it
            request(g0 + (DEPTH - 1) * AHEAD, stage ? stage - 1 : DEPTH - 1);
        }
        if (within(g0)) {
            const unsigned char* b = ring + stage * STAGE;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (F32) {  // any eight of the segment's logits will do: two groups of four, without bank conflicts
                    take<true, ALIGNED>(b + i * 1024 + 16 * lane, skip, f[i]);
                    take<true, ALIGNED>(b + i * 1024 + 512 + 16 * lane, skip, f[i] + 4);
                } else {
                    take<false, ALIGNED>(b + i * 512 + 16 * lane, skip, f[i]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) load_edge<F32>(p.logits, row, (g0 + i) * SEG + 8 * lane, p.V, f[i]);
        }
        if (!CAREFUL && ++stage == DEPTH) stage = 0;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (CAREFUL) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[i][e] = sane(f[i][e]);
            }
            top[i] = warp_max(max8(f[i]));
        }
        if (lane == 0) {  // (segments come in fours)
#pragma unroll
            for (int i = 0; i < AHEAD; i += 2) *reinterpret_cast<float2*>(seg_max + g0 + i) = make_float2(top[i], top[i + 1]);
        }
        float most = m;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) most = fmaxf(most, top[i]);
        // (from -inf itself a difference would be a NaN)
        const float c = fmaxf(most, LOWEST), old = ex2_approx((fmaxf(m, LOWEST) - c) * LOG2E);
        const F2 minus = f2(-c, -c), log2e = f2(LOG2E, LOG2E);
        sum = mul2(sum, f2(old, old));
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const F2 x = mul2(add2(f2(f[i][e], f[i][e + 1]), minus), log2e);
                sum = add2(sum, f2(ex2_approx(x.x), ex2_approx(x.y)));
            }
        m = most;
    }
    s = sum.x + sum.y;
}

template <bool F32, bool ALIGNED> __global__ void __launch_bounds__(32 * SCAN_WARPS) beam_scan_kernel(const __grid_constant__ BeamParams p) {
    extern __shared__ __align__(16) unsigned char rings[];
    stream_order();
    const int lane = threadIdx.x & 31;
    unsigned char* ring = rings + (threadIdx.x >> 5) * (DEPTH * stage_bytes<F32, ALIGNED>());
    const long long unit = (long long)blockIdx.x * SCAN_WARPS + (threadIdx.x >> 5);
    if (unit >= (long long)p.B * p.W * p.parts) return;
    const long long r = unit / p.parts;
    const int part = (int)(unit - r * p.parts), first = part * p.per_part, last = min(first + p.per_part, p.segments);
    const long long row = r / p.W * p.sb + r % p.W * p.sw;
    float* seg_max = p.seg_max + r * p.segments;
    float m = NEG_INF, s = 0.f;
    if (p.finished && p.finished[r]) {  // goes on with eos alone, at no cost
        for (int g = first; g < last; ++g) {
            const bool here = p.eos >= g * SEG && p.eos < (g + 1) * SEG;
            if (here) { m = 0.f; s = lane == 0 ? 1.f : 0.f; }
            if (lane == 0) seg_max[g] = here ? 0.f : NEG_INF;
        }
    } else {
        scan_part<F32, ALIGNED, false>(p, row, first, last, seg_max, ring, lane, m, s);
        // (a NaN, which maxima pass over, is in some lane's sum; +inf makes one there, as inf - inf)
        if (__any_sync(0xffffffffu, s != s)) scan_part<F32, false, true>(p, row, first, last, seg_max, ring, lane, m, s);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) {
        p.part[2 * unit] = m;
        p.part[2 * unit + 1] = s;
    }
}

// SEGS segments and LIST candidates above the threshold fit; up to RANKED candidates each finds its own place (n / 32 squared steps of a warp), beyond that the best
// are taken out one by one (k rounds of the CTA).
constexpr int PICK_THREADS = 1024, SEGS = 512, LIST = 2 * PICK_THREADS, RANKED = 320;
struct Pick {
    double top[BEAM_MAX_W], logz[BEAM_MAX_W], base[BEAM_MAX_W];  // a beam's largest logit, log sum exp(l - top), score
    double bar[BEAM_MAX_W];                                      // the threshold, less what a score in 64 bits may be off by
    float offset[BEAM_MAX_W], least[BEAM_MAX_W];                 // about base - top - logz; the least logit that may reach the threshold
    double score[LIST];
    uint32_t index[LIST];
    int2 segs[SEGS];       // beam, segment
    uint32_t group[128];   // the best of each group of threads
    unsigned char fin[BEAM_MAX_W];
    double best_score[32];
    uint32_t best_index[32];
    double out_score[BEAM_MAX_K];
    uint32_t out_index[BEAM_MAX_K];
    int nsegs, n, count[32];
    float t;
    unsigned char ruled_out[2 * BEAM_MAX_K];
};
__device__ __forceinline__ bool better(double a, uint32_t i, double b, uint32_t j) { return a > b || (a == b && i < j); }
__device__ __forceinline__ double score_of(const Pick& q, int w, float l) { return l == NEG_INF ? (double)NEG_INF : q.base[w] + (((double)l - q.top[w]) - q.logz[w]); }

// eight adjacent candidates of beam w: their logits, as far as they count
__device__ __forceinline__ void logits8(const BeamParams& p, const Pick& q, long long seq, int w, int at, float (&f)[8]) {
    if (q.fin[w]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = at + i == p.eos ? 0.f : NEG_INF;
        return;
    }
    const long long row = seq * p.sb + w * p.sw;
    if (p.f32) load_edge<true>(p.logits, row, at, p.V, f);
    else load_edge<false>(p.logits, row, at, p.V, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = sane(f[i]);
}

// the k best of q.score[0 .. n), n <= LIST, in order, to the front; all threads.  Each round takes the best that is left.
// (All have read their part of the list before the first barrier.)
__device__ __forceinline__ void keep_best(Pick& q, int n, int k) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    double s[2];
    uint32_t ix[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = tid + e * PICK_THREADS;
        s[e] = i < n ? q.score[i] : (double)NEG_INF;
        ix[e] = i < n ? q.index[i] : 0xffffffffu;
    }
    const int m = n < k ? n : k;
    for (int round = 0; round < m; ++round) {
        double b = s[0];
        uint32_t j = ix[0];
        if (better(s[1], ix[1], b, j)) { b = s[1]; j = ix[1]; }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const double ob = __shfl_xor_sync(0xffffffffu, b, d);
            const uint32_t oj = __shfl_xor_sync(0xffffffffu, j, d);
            if (better(ob, oj, b, j)) { b = ob; j = oj; }
        }
        if (lane == 0) { q.best_score[warp] = b; q.best_index[warp] = j; }
        __syncthreads();
        if (warp == 0) {
            b = q.best_score[lane]; j = q.best_index[lane];
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                const double ob = __shfl_xor_sync(0xffffffffu, b, d);
                const uint32_t oj = __shfl_xor_sync(0xffffffffu, j, d);
                if (better(ob, oj, b, j)) { b = ob; j = oj; }
            }
            if (lane == 0) { q.out_score[round] = b; q.out_index[round] = j; }
        }
        __syncthreads();
        const uint32_t taken = q.out_index[round];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (ix[e] == taken) { s[e] = (double)NEG_INF; ix[e] = 0xffffffffu; }
    }
    if (tid < m) { q.score[tid] = q.out_score[tid]; q.index[tid] = q.out_index[tid]; }
    __syncthreads();
}

// a CTA per sequence
__global__ void __launch_bounds__(PICK_THREADS, 1) beam_pick_kernel(const __grid_constant__ BeamParams p) {
    __shared__ Pick q;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long seq = blockIdx.x, row0 = seq * p.W;
    const int k = p.k;
    if (tid == 0) { q.nsegs = 0; q.n = 0; }
    if (tid < BEAM_MAX_K) { q.out_score[tid] = (double)NEG_INF; q.out_index[tid] = tid; }  // (a candidate that there is: k is W V at most)
    if (tid < 128) q.group[tid] = 0;
    stream_order();
    // a thread has every 1024th of the sequence's segments; their maxima are requested here and used behind the normalisers
    const int total = p.W * p.segments;
    const float* const seg_max = p.seg_max + row0 * p.segments;
    constexpr int HELD = 4;
    float held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = tid + i * PICK_THREADS < total ? seg_max[tid + i * PICK_THREADS] : NEG_INF;
    // the beams' normalisers, a warp each: the parts' sums joined in 64 bits, in a fixed order
    for (int w = warp; w < p.W; w += 32) {
        const float2* part = reinterpret_cast<const float2*>(p.part) + (row0 + w) * p.parts;
        const float2 mine = lane < p.parts ? part[lane] : make_float2(NEG_INF, 0.f);
        const float base = p.scores[row0 + w];
        const unsigned char fin = p.finished ? p.finished[row0 + w] : 0;
        float m = mine.x;
        for (int i = lane + 32; i < p.parts; i += 32) m = fmaxf(m, part[i].x);
        m = warp_max(m);
        double s = mine.x == NEG_INF ? 0. : (double)mine.y * (double)ex2_approx((mine.x - m) * LOG2E);
        for (int i = lane + 32; i < p.parts; i += 32)
            if (part[i].x != NEG_INF) s += (double)part[i].y * (double)ex2_approx((part[i].x - m) * LOG2E);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) {
            // (kept apart: in a row of the type's lowest values their sum would lose logz.  A row without a candidate has none that would read them.)
            const double logz = m == NEG_INF ? 0. : log(s);
            q.top[w] = m == NEG_INF ? 0. : (double)m;
            q.logz[w] = logz;
            q.base[w] = (double)sane(base);
            q.offset[w] = m == NEG_INF ? NEG_INF : fminf((float)(((double)sane(base) - logz) - (double)m), 3.402823466e38f);
            q.fin[w] = fin;
        }
    }
    __syncthreads();
    // A threshold that k candidates reach at least: the k-th best of the bests of 32, 64 or 128 groups of segments, two of them or more for each of the k.  A
    // group has segments of all beams (the best candidates are often of a few), so that some 1.4 k segments reach it as a rule.  The segments' scores in
    // 32 bits here, less what the roundings may have added.  Candidates at -inf are left to the end; where fewer than k groups have others t is -inf, since a score may lie
    // a little below fp32's lowest value and still be rounded to it.
    auto at_least = [&](int w, float l) {
        const float s = l + q.offset[w];
        return s == NEG_INF ? 0u : ordered(s - 2.4e-7f * (fabsf(l) + fabsf(q.offset[w])));
    };
    auto each_segment = [&](auto f) {  // f(beam, segment, maximum)
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int c = tid + i * PICK_THREADS, w = c / p.segments;
            if (c < total) f(w, c - w * p.segments, held[i]);
        }
        for (int c = tid + HELD * PICK_THREADS; c < total; c += PICK_THREADS) f(c / p.segments, c % p.segments, seg_max[c]);
    };
    uint32_t best = 0;
    each_segment([&](int w, int, float l) { best = max(best, at_least(w, l)); });
    const int groups = k <= 16 ? 32 : k <= 32 ? 64 : 128;
    atomicMax(&q.group[tid & (groups - 1)], best);
    __syncthreads();
    for (int g = warp; g < groups; g += 32) {  // a group's place among them
        const uint32_t mine = q.group[g];
        int ahead = 0;
        for (int i = lane; i < groups; i += 32) ahead += __popc(__ballot_sync(0xffffffffu, q.group[i] > mine || (q.group[i] == mine && i < g)));
        if (ahead == k - 1 && lane == 0) q.t = mine ? unordered(mine) : NEG_INF;
    }
    __syncthreads();
    // the segments that reach t, and their candidates that do
    auto list = [&] {
        // score >= t is l >= (t - base + logz) + top, less a little for the roundings on the way (a NaN, which nothing reaches, for a beam at -inf where t is)
        if (tid < p.W) {
            const double t = q.t, l = ((t - q.base[tid]) + q.logz[tid]) + q.top[tid];
            const double off = 1e-15 * (fabs(t) + fabs(q.base[tid]) + 64.);
            q.least[tid] = __double2float_rd(l - (off + 1e-15 * fabs(q.top[tid])));
            q.bar[tid] = t - off;  // (score_of takes l - top first, which is exact where it matters)
        }
        __syncthreads();
        // (that is in the logits' steps, in which all of a beam that is masked with -1e9 are near t: segments that pass are looked at once more in 64 bits)
        each_segment([&](int w, int g, float l) {
            if (l >= q.least[w] && l > NEG_INF && score_of(q, w, l) >= q.bar[w]) {
                const int i = atomicAdd(&q.nsegs, 1);
                if (i < SEGS) q.segs[i] = make_int2(w, g);
            }
        });
        __syncthreads();
        const int nsegs = q.nsegs;
        if (nsegs > SEGS) return false;
        for (int i = warp; i < nsegs; i += 32) {
            const int w = q.segs[i].x, at = q.segs[i].y * SEG + 8 * lane;
            float l[8];
            logits8(p, q, seq, w, at, l);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (l[e] >= q.least[w] && (float)score_of(q, w, l[e]) > NEG_INF) {
                    const int j = atomicAdd(&q.n, 1);
                    if (j < LIST) { q.score[j] = score_of(q, w, l[e]); q.index[j] = w * p.V + at + e; }
                }
        }
        __syncthreads();
        return q.n <= LIST;
    };
    bool listed = list();
    if (!listed) {
        // Too many: the groups' threshold is the exact one only as far as the best segments lie in different groups.  (A mask of the type's lowest value that leaves a few
        // tokens puts them in a few segments.)  The exact one, bit by bit, and once more.
        uint32_t t = 0;
        if (tid < 32) q.count[tid] = 0;
        for (int bit = 31; bit >= 0; --bit) {
            __syncthreads();
            const uint32_t trial = t | 1u << bit;
            int c = 0;
            each_segment([&](int w, int, float l) { c += at_least(w, l) >= trial; });
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0 && c) atomicAdd(&q.count[bit], c);
            __syncthreads();
            if (q.count[bit] >= k) t = trial;
        }
        __syncthreads();
        if (tid == 0) { q.t = t ? unordered(t) : NEG_INF; q.nsegs = 0; q.n = 0; }
        __syncthreads();
        listed = list();
    }
    int n = listed ? q.n : 0;
    if (listed && n <= RANKED) {
        // each candidate's place is the number of better ones
        for (int c = warp; c < n; c += 32) {
            const double s = q.score[c];
            const uint32_t ix = q.index[c];
            int place = 0;
            for (int i = lane; i < (n + 31) / 32 * 32; i += 32) place += __popc(__ballot_sync(0xffffffffu, i < n && better(q.score[i], q.index[i], s, ix)));
            if (place < k && lane == 0) { q.out_score[place] = s; q.out_index[place] = ix; }
        }
        n = min(n, k);
    } else if (listed) {
        keep_best(q, n, k);
        n = min(n, k);
    } else {
        // Many equal or nearly equal ones: all that reach t in order, into a list whose first `kept` are the k best so far.  A candidate joins it only if it
        // is better than the last of those, which one of equal score behind it is not.  The list is thinned out when it might not take another step's.
        __syncthreads();
        if (tid == 0) q.n = 0;
        __syncthreads();
        int kept = 0, filled = 0;
        constexpr int STEP = PICK_THREADS / 8;  // threads whose eight candidates each join in one step: 1024 at most
        for (long long c0 = 0; c0 < (long long)total * (SEG / 8); c0 += PICK_THREADS) {
            const long long c = c0 + tid;
            const int g = (int)(c / (SEG / 8)), w = g < total ? g / p.segments : 0, at = (g - w * p.segments) * SEG + 8 * (int)(c % (SEG / 8));
            const float l = g < total ? seg_max[g] : NEG_INF;
            float f[8];
            uint32_t mask = 0;
            auto joins = [&](int e) {
                const double s = score_of(q, w, f[e]);
                return f[e] >= q.least[w] && (float)s > NEG_INF && (kept < k || better(s, (uint32_t)(w * p.V + at + e), q.score[k - 1], q.index[k - 1]));
            };
            if (l >= q.least[w] && l > NEG_INF) {
                logits8(p, q, seq, w, at, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) mask |= joins(e) ? 1u << e : 0u;
            }
            if (!__syncthreads_or(mask != 0)) continue;
            for (int step = 0; step < PICK_THREADS; step += STEP) {
                if (mask && tid >= step && tid < step + STEP) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((mask >> e & 1) && joins(e)) {
                            const int j = atomicAdd(&q.n, 1);
                            q.score[j] = score_of(q, w, f[e]);
                            q.index[j] = (uint32_t)(w * p.V + at + e);
                        }
                }
                __syncthreads();
                filled = q.n;
                if (filled > LIST - PICK_THREADS) {
                    keep_best(q, filled, k);
                    filled = kept = min(filled, k);
                    if (tid == 0) q.n = kept;
                }
                __syncthreads();
            }
        }
        keep_best(q, filled, k);
        n = min(filled, k);
    }
    __syncthreads();
    if (n < k) {
        // the rest at -inf, the lowest of them: there are k at least among the first 2 k candidates
        const int look = min(2 * k, (int)min((long long)2 * BEAM_MAX_K, (long long)p.W * p.V));
        if (tid < look) {
            const int w = tid / p.V, v = tid - w * p.V;
            float l;
            if (q.fin[w]) l = v == p.eos ? 0.f : NEG_INF;
            else {
                const long long at = seq * p.sb + w * p.sw + v;
                l = sane(p.f32 ? ((const float*)p.logits)[at] : __bfloat162float(((const bf16*)p.logits)[at]));
            }
            q.ruled_out[tid] = (float)score_of(q, w, l) == NEG_INF;
        }
        __syncthreads();
        if (tid == 0)
            for (int i = 0, j = n; j < k && i < look; ++i)
                if (q.ruled_out[i]) { q.out_score[j] = (double)NEG_INF; q.out_index[j++] = i; }
        __syncthreads();
    }
    if (tid < k) {
        const uint32_t ix = q.out_index[tid];
        const int w = ix / p.V, v = ix - w * p.V;
        const long long o = seq * k + tid;
        p.out_scores[o] = (float)q.out_score[tid];
        p.parents[o] = w;
        p.tokens[o] = v;
        if (p.finished) p.out_finished[o] = q.fin[w] || v == p.eos;
    }
}

// ---- reordering ------------------------------------------------------------------------------------------------
// Row (b, j) of dst := row (b, parents[b, j]) of src.  A thread has one column of 16 bytes (or as many as the rows' sizes and places allow) in all rows of a
// sequence: it reads what it will write before it writes, so that src and dst may be the same.  In place, rows that stay are left alone.  Bound by DRAM: 16 x 8 rows of 6.3 MB
// in 36 tensors, 80 of 128 rows moving, 57 read: 875 MB in 137 to 146 us, 6.0 to 6.4 TB/s.
template <typename U, int K> __device__ __forceinline__ void move_column(const unsigned char* src, unsigned char* dst, long long sp, long long dp, const int* from, int k) {
    U v[K];
#pragma unroll
    for (int j = 0; j < K; ++j)
        if (j < k && from[j] >= 0) v[j] = *reinterpret_cast<const U*>(src + from[j] * sp);
#pragma unroll
    for (int j = 0; j < K; ++j)
        if (j < k) {
            if (from[j] == -2) *reinterpret_cast<U*>(dst + j * dp) = U{};
            else if (from[j] >= 0) *reinterpret_cast<U*>(dst + j * dp) = v[j];
        }
}
constexpr int RE_THREADS = 256;
struct ReorderLaunch : ReorderParams {
    int first[REORDER_MAX + 1];         // CTAs of the tensors before each
    unsigned char unit[REORDER_MAX];    // bytes that a thread moves at once
};
template <int K> __global__ void __launch_bounds__(RE_THREADS) reorder_kernel(const __grid_constant__ ReorderLaunch p) {
    __shared__ int from[K];
    stream_order();
    int t = 0, hi = p.count;
    while (hi - t > 1) {
        const int mid = (t + hi) / 2;
        if (p.first[mid] <= (int)blockIdx.x) t = mid;
        else hi = mid;
    }
    const int unit = p.unit[t];
    const long long units = p.row_bytes[t] / unit;
    const int per_seq = (int)((units + RE_THREADS - 1) / RE_THREADS), tile = blockIdx.x - p.first[t], b = tile / per_seq;
    const bool inplace = p.src[t] == p.dst[t];
    if (threadIdx.x < p.k) {
        const long long at = (long long)b * p.k + threadIdx.x;
        const long long f = p.idx64 ? ((const int64_t*)p.parents)[at] : ((const int32_t*)p.parents)[at];
        int use = (int)f;  // -1: nothing to do, -2: zeros
        if (f < 0 || f >= p.W) {
            use = inplace ? -1 : p.keep ? (int)threadIdx.x : -2;
            *reinterpret_cast<volatile int*>(p.status) = (int)kBadIndex;
            __threadfence_system();
        } else if (inplace && f == (long long)threadIdx.x) {
            use = -1;
        }
        from[threadIdx.x] = use;
    }
    __syncthreads();
    const long long u = (long long)(tile - b * per_seq) * RE_THREADS + threadIdx.x;
    if (u >= units) return;
    const unsigned char* src = (const unsigned char*)p.src[t] + (long long)b * p.W * p.src_pitch[t] + u * unit;
    unsigned char* dst = (unsigned char*)p.dst[t] + (long long)b * p.k * p.dst_pitch[t] + u * unit;
    if (unit == 16) {
        if (K <= 32) {
            move_column<uint4, K>(src, dst, p.src_pitch[t], p.dst_pitch[t], from, p.k);
        } else {  // two halves: 64 rows of 16 bytes would not fit the registers
            move_column<uint2, K>(src, dst, p.src_pitch[t], p.dst_pitch[t], from, p.k);
            move_column<uint2, K>(src + 8, dst + 8, p.src_pitch[t], p.dst_pitch[t], from, p.k);
        }
    } else if (unit == 4) {
        move_column<uint32_t, K>(src, dst, p.src_pitch[t], p.dst_pitch[t], from, p.k);
    } else {
        move_column<unsigned char, K>(src, dst, p.src_pitch[t], p.dst_pitch[t], from, p.k);
    }
}

}  // namespace beam

// ---- host ------------------------------------------------------------------------------------------------------
static void beam_plan(long long B, long long W, long long V, int& segments, int& per_part, int& parts) {
    segments = (int)((V + beam::SEG - 1) / beam::SEG + 3) / 4 * 4;  // (those behind the row's end hold -inf)
    // a warp takes four segments, or eight, where that still gives every place on the SMs (148, 32 warps each) two
    per_part = B * W * segments / 16 >= 2 * 148 * 32 ? 16 : B * W * segments / 8 >= 2 * 148 * 32 ? 8 : 4;
    parts = (segments + per_part - 1) / per_part;
}
size_t beam_workspace_bytes(long long B, long long W, long long V) {
    int segments, per_part, parts;
    beam_plan(B, W, V, segments, per_part, parts);
    return (size_t)(B * W) * (segments + 2 * (size_t)parts) * 4;
}
int launch_beam_select(BeamParams p, void* workspace, cudaStream_t stream) {
    beam_plan(p.B, p.W, p.V, p.segments, p.per_part, p.parts);
    p.seg_max = (float*)workspace;
    p.part = p.seg_max + (long long)p.B * p.W * p.segments;
    const long long units = (long long)p.B * p.W * p.parts, ctas = (units + beam::SCAN_WARPS - 1) / beam::SCAN_WARPS;
    if (ctas > 0x7fffffffLL) return kTooLarge;
    const uintptr_t size = p.f32 ? 4 : 2;
    const bool aligned = (((uintptr_t)p.logits | p.sb * size | p.sw * size) & 15) == 0;
    auto scan = p.f32 ? aligned ? beam::beam_scan_kernel<true, true> : beam::beam_scan_kernel<true, false>
                      : aligned ? beam::beam_scan_kernel<false, true> : beam::beam_scan_kernel<false, false>;
    const int stage = p.f32 ? aligned ? beam::stage_bytes<true, true>() : beam::stage_bytes<true, false>()
                            : aligned ? beam::stage_bytes<false, true>() : beam::stage_bytes<false, false>();
    const int smem = beam::SCAN_WARPS * beam::DEPTH * stage;
    static thread_local uint32_t smem_allowed[64];
    if (!allow_smem(scan, smem_allowed, 2 * p.f32 + aligned, smem)) return kLaunchFailed;
    if (!launch(scan, dim3((unsigned)ctas), 32 * beam::SCAN_WARPS, smem, stream, p)) return kLaunchFailed;
    return launch(beam::beam_pick_kernel, dim3((unsigned)p.B), beam::PICK_THREADS, 0, stream, p) ? kOk : kLaunchFailed;
}

int launch_reorder(const ReorderParams& r, cudaStream_t stream) {
    beam::ReorderLaunch p;
    static_cast<ReorderParams&>(p) = r;
    long long ctas = 0;
    for (int t = 0; t < r.count; ++t) {
        const unsigned long long bits = (unsigned long long)(uintptr_t)r.src[t] | (uintptr_t)r.dst[t] | r.row_bytes[t] | r.src_pitch[t] | r.dst_pitch[t];
        p.unit[t] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
        p.first[t] = (int)ctas;
        const long long units = r.row_bytes[t] / p.unit[t];
        ctas += (units + beam::RE_THREADS - 1) / beam::RE_THREADS * r.B;
        if (ctas > 0x7fffffffLL) return kTooLarge;
    }
    p.first[r.count] = (int)ctas;
    if (!ctas) return kOk;
    auto kern = r.k <= 4 ? beam::reorder_kernel<4> : r.k <= 8 ? beam::reorder_kernel<8> : r.k <= 16 ? beam::reorder_kernel<16> : r.k <= 32 ? beam::reorder_kernel<32> : beam::reorder_kernel<64>;
    return launch(kern, dim3((unsigned)ctas), beam::RE_THREADS, 0, stream, p) ? kOk : kLaunchFailed;
}

}  // namespace wkv7

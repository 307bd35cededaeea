// Beam search next to the decode step: the selection over beams and vocabulary, and the reordering of the states that attn_step keeps.
//
// Selection: score(w, v) = s_w + (l_wv - lse_w), lse_w = log sum_v exp(l_wv); the k best of the W V candidates, equal scores by the lowest w V + v.
// One pass over the logits (beam_scan_kernel) leaves the maximum of every segment of 256 logits and, for every few segments, the sum of exp(l - max);
// nothing else is done per logit, so that it runs at DRAM speed (the exponential unit's bound, 16 a cycle and SM, is 3/4 of it for bf16).
// The second kernel, a CTA per sequence, needs few logits more: the k best candidates lie in the k segments with the best maxima
// (any other candidate is behind those k maxima).  It finds a threshold t for which some k to 2k segments qualify, reads those again, and
// orders the few candidates that reach t.  Scores are compared in 64 bits: a rounded one decides between beams only where they are closer than
// the sums' own error (3e-7).  t is compared with scores rounded to 32 bits, which keeps their order, so nothing that belongs to the best is lost.
#include "beam.h"
#include "mma_bf16.cuh"
#include "wkv7_kernels.h"

namespace wkv7 {
namespace beam {

constexpr int SEG = 256;  // logits of a segment: eight a lane
constexpr int SCAN_WARPS = 8;
constexpr float NEG_INF = -__builtin_huge_valf(), POS_INF = __builtin_huge_valf();

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
// The same as whole 16-byte words, of which the logits start `skip` bytes into the first.  A row may lie on any element's boundary; every lane then still
// has the same logits whatever the alignment, so that equal rows give equal sums.  Words that reach beyond the row are not read: false.
template <bool F32, bool ALIGNED> struct Raw {
    static constexpr int WORDS = (F32 ? 2 : 1) + (ALIGNED ? 0 : 1);
    uint4 w[WORDS];
    __device__ __forceinline__ bool load(const void* base, long long row, int at, int V) {
        const int size = F32 ? 4 : 2;
        const unsigned char *start = (const unsigned char*)base + row * size, *end = start + (long long)V * size, *p = start + (long long)at * size;
        p -= reinterpret_cast<uintptr_t>(p) & 15;
        if (p < start || p + 16 * WORDS > end) return false;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
        return true;
    }
    __device__ __forceinline__ void take(int skip, float (&f)[8]) const {
        uint32_t x[4 * WORDS], o[F32 ? 8 : 4];
#pragma unroll
        for (int i = 0; i < WORDS; ++i) { x[4 * i] = w[i].x; x[4 * i + 1] = w[i].y; x[4 * i + 2] = w[i].z; x[4 * i + 3] = w[i].w; }
        constexpr int N_ = F32 ? 8 : 4;
        if (ALIGNED) {
#pragma unroll
            for (int i = 0; i < N_; ++i) o[i] = x[i];
        } else {
            const int words = skip >> 2, bits = (skip & 3) * 8;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (words == c) {  // (the same for the whole row)
#pragma unroll
                    for (int i = 0; i < N_; ++i) o[i] = F32 ? x[i + c] : __funnelshift_r(x[i + c], x[i + c + 1 < 4 * WORDS ? i + c + 1 : i + c], bits);
                }
        }
        if (F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(o[i % N_]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(o[i] << 16); f[2 * i + 1] = __uint_as_float(o[i] & 0xffff0000u); }
        }
    }
};
__device__ __forceinline__ float warp_max(float x) { return unordered(__reduce_max_sync(0xffffffffu, ordered(x))); }

// A warp per part of a row (per_part segments), four segments' words requested at once.
template <bool F32, bool ALIGNED> __global__ void __launch_bounds__(32 * SCAN_WARPS) beam_scan_kernel(const __grid_constant__ BeamParams p) {
    stream_order();
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * SCAN_WARPS + (threadIdx.x >> 5);
    if (unit >= (long long)p.B * p.W * p.parts) return;
    const long long r = unit / p.parts;
    const int part = (int)(unit - r * p.parts), first = part * p.per_part, last = min(first + p.per_part, p.segments);
    const long long row = r / p.W * p.sb + r % p.W * p.sw;
    const int skip = (int)((reinterpret_cast<uintptr_t>(p.logits) + row * (F32 ? 4 : 2)) & 15);
    float* seg_max = p.seg_max + r * p.segments;
    float m = NEG_INF, s = 0.f;
    if (p.finished && p.finished[r]) {  // goes on with eos alone, at no cost
        for (int g = first; g < last; ++g) {
            const bool here = p.eos >= g * SEG && p.eos < (g + 1) * SEG;
            if (here) { m = 0.f; s = lane == 0 ? 1.f : 0.f; }
            if (lane == 0) seg_max[g] = here ? 0.f : NEG_INF;
        }
    } else {
        constexpr int AHEAD = 4;
        for (int g0 = first; g0 < last; g0 += AHEAD) {
            Raw<F32, ALIGNED> raw[AHEAD];
            bool whole[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) whole[i] = g0 + i < last && raw[i].load(p.logits, row, (g0 + i) * SEG + 8 * lane, p.V);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (g0 + i >= last) break;
                float f[8];
                if (whole[i]) raw[i].take(skip, f);
                else load_edge<F32>(p.logits, row, (g0 + i) * SEG + 8 * lane, p.V, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = sane(f[e]);
                const float top = warp_max(fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7]))));
                if (lane == 0) seg_max[g0 + i] = top;
                if (top > m) {  // (the warp's maximum: all lanes take the same way)
                    s *= ex2_approx((m - top) * 1.4426950408889634f);
                    m = top;
                }
                if (m == NEG_INF) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e) s += ex2_approx((f[e] - m) * 1.4426950408889634f);
            }
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) {
        p.part[2 * unit] = m;
        p.part[2 * unit + 1] = s;
    }
}

constexpr int PICK_THREADS = 1024, CAP = 256, LIST = PICK_THREADS + BEAM_MAX_K;
struct Pick {
    double top[BEAM_MAX_W], logz[BEAM_MAX_W], base[BEAM_MAX_W];  // a beam's largest logit, log sum exp(l - top), score
    double score[LIST];
    uint32_t index[LIST];
    uint32_t segs[CAP];
    unsigned char fin[BEAM_MAX_W];
    double best_score[32];
    uint32_t best_index[32];
    double out_score[BEAM_MAX_K];
    uint32_t out_index[BEAM_MAX_K];
    int nsegs, n, kept;
    unsigned char ruled_out[2 * BEAM_MAX_K];
};
__device__ __forceinline__ bool better(double a, uint32_t i, double b, uint32_t j) { return a > b || (a == b && i < j); }
__device__ __forceinline__ double score_of(const Pick& q, int w, float l) { return l == NEG_INF ? (double)NEG_INF : q.base[w] + (((double)l - q.top[w]) - q.logz[w]); }

// eight adjacent candidates of beam w: their scores
__device__ __forceinline__ void scores8(const BeamParams& p, const Pick& q, long long seq, int w, int at, double (&s)[8]) {
    float f[8];
    if (q.fin[w]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = at + i == p.eos ? 0.f : NEG_INF;
    } else {
        const long long row = seq * p.sb + w * p.sw;
        if (p.f32) load_edge<true>(p.logits, row, at, p.V, f);
        else load_edge<false>(p.logits, row, at, p.V, f);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = score_of(q, w, sane(f[i]));
}

// the k best of q.score[0 .. n), n <= LIST, in order, to the front; all threads.  Each round takes the best that is left.
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
    const int k = p.k, total = p.W * p.segments;
    stream_order();
    if (tid == 0) { q.nsegs = 0; q.n = 0; }
    // the beams' normalisers, a warp each: the parts' sums joined in 64 bits, in a fixed order
    for (int w = warp; w < p.W; w += 32) {
        const float* part = p.part + 2 * (row0 + w) * p.parts;
        float m = NEG_INF;
        for (int i = lane; i < p.parts; i += 32) m = fmaxf(m, part[2 * i]);
        m = warp_max(m);
        double s = 0.;
        for (int i = lane; i < p.parts; i += 32)
            if (part[2 * i] != NEG_INF) s += (double)part[2 * i + 1] * exp((double)part[2 * i] - (double)m);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) {
            // (kept apart: in a row of the type's lowest values their sum would lose logz.  A row without a candidate has none that would read them.)
            q.top[w] = (double)m;
            q.logz[w] = log(s);
            q.base[w] = (double)sane(p.scores[row0 + w]);
            q.fin[w] = p.finished ? p.finished[row0 + w] : 0;
        }
    }
    __syncthreads();
    // the best segment of each thread's, rounded to 32 bits
    uint32_t best = 0;
    for (int g = tid; g < total; g += PICK_THREADS) best = max(best, ordered((float)score_of(q, g / p.segments, p.seg_max[row0 * p.segments + g])));
    // the largest t that k threads reach, bit by bit; fewer steps where somewhat more than k do.  Candidates at -inf are left to the end.
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
        const int c = __syncthreads_count(best >= (t | bit));
        if (c >= k) t |= bit;
        if (c >= k && c <= 2 * k) break;
    }
    t = max(t, ordered(NEG_INF) + 1);
    for (int g = tid; g < total; g += PICK_THREADS)
        if (ordered((float)score_of(q, g / p.segments, p.seg_max[row0 * p.segments + g])) >= t) {
            const int i = atomicAdd(&q.nsegs, 1);
            if (i < CAP) q.segs[i] = g;
        }
    __syncthreads();
    const int nsegs = q.nsegs;
    if (nsegs <= CAP) {
        for (int i = warp; i < nsegs; i += 32) {
            const int w = q.segs[i] / p.segments, at = (q.segs[i] - w * p.segments) * SEG + 8 * lane;
            double s[8];
            scores8(p, q, seq, w, at, s);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (ordered((float)s[e]) >= t) {
                    const int j = atomicAdd(&q.n, 1);
                    if (j < CAP) { q.score[j] = s[e]; q.index[j] = w * p.V + at + e; }
                }
        }
        __syncthreads();
    }
    int n = q.n;
    if (nsegs <= CAP && n <= CAP) {
        // each candidate's place is the number of better ones
        if (tid < n) {
            const double s = q.score[tid];
            const uint32_t ix = q.index[tid];
            int place = 0;
            for (int i = 0; i < n; ++i) place += better(q.score[i], q.index[i], s, ix);
            if (place < k) { q.out_score[place] = s; q.out_index[place] = ix; }
        }
        n = min(n, k);
    } else {
        // many equal or nearly equal ones: all segments that reach t in order, with the k best so far at the front of the list; a candidate joins it only if it
        // is better than the last of those, which one of equal score behind it is not
        __syncthreads();
        if (tid == 0) q.n = 0;
        __syncthreads();
        int kept = 0;
        for (long long c0 = 0; c0 < (long long)p.W * p.segments * (SEG / 8); c0 += PICK_THREADS / 8) {
            // 128 threads' worth of eight candidates: 1024 at most join at once
            if (tid < PICK_THREADS / 8) {
                const long long c = c0 + tid;
                const int g = (int)(c / (SEG / 8));
                if (g < total) {
                    const int w = g / p.segments, at = (g - w * p.segments) * SEG + 8 * (int)(c % (SEG / 8));
                    if (ordered((float)score_of(q, w, p.seg_max[row0 * p.segments + g])) >= t) {
                        double s[8];
                        scores8(p, q, seq, w, at, s);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t ix = (uint32_t)(w * p.V + at + e);
                            if (ordered((float)s[e]) >= t && (kept < k || better(s[e], ix, q.score[k - 1], q.index[k - 1]))) {
                                const int j = kept + atomicAdd(&q.n, 1);
                                q.score[j] = s[e];
                                q.index[j] = ix;
                            }
                        }
                    }
                }
            }
            __syncthreads();
            const int fresh = q.n;
            __syncthreads();
            if (fresh) {
                if (tid == 0) q.n = 0;
                keep_best(q, kept + fresh, k);
                kept = min(kept + fresh, k);
            }
        }
        if (tid < kept) { q.out_score[tid] = q.score[tid]; q.out_index[tid] = q.index[tid]; }
        n = kept;
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
// sequence: it reads what it will write before it writes, so that src and dst may be the same.  In place, rows that stay are left alone.  Bound by DRAM.
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
            use = inplace ? -1 : -2;
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
    segments = (int)((V + beam::SEG - 1) / beam::SEG);
    // a warp takes up to eight segments, fewer while the SMs (148, 32 warps each) are not full of warps
    const long long all = B * W * segments;
    per_part = 8;
    while (per_part > 1 && all / per_part < 148 * 32) per_part /= 2;
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
    if (!launch(scan, dim3((unsigned)ctas), 32 * beam::SCAN_WARPS, 0, stream, p)) return kLaunchFailed;
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

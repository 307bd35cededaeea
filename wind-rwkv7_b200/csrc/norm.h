// Interface between the C ABI (capi.cu) and the residual stream's kernels: norm, dropout, rows to 8 bits (norm_fwd.cu, norm_bwd.cu, norm.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace wkv7 {

// Which elements are dropped.  Element i, counted in row-major order, has word i % 4 of Philox4x32-10 with counter i / 4 and key `seed`; it is kept where that
// is >= threshold.
struct Dropout {
    unsigned long long threshold;     // round(p 2^32), 0: none is dropped
    float scale;                      // of what is kept, 1 / (1 - p)
    unsigned long long seed;
    const unsigned long long* where;  // device memory that holds the seed, or null
};

struct DropoutParams {
    const void *x, *residual;  // residual: or null
    void* y;
    long long n;
    Dropout d;
    bool x_f32, r_f32, y_f32;
};
int launch_dropout(const DropoutParams& p, cudaStream_t stream);

constexpr long long NORM_MAX_D = 16384;
struct NormFwdParams {
    const void *x, *residual, *weight;  // residual, weight: or null
    void *y, *h;                        // h: null without a residual
    float *rstd, *scale;                // rstd: or null; scale: of y in 8 bits, else null
    long long M, ldx, ldr, ldy, ldh;
    int D;
    float eps;
    Dropout d;
    bool x_f32, r_f32, w_f32, y_f32;    // h has the residual's type
};
int launch_norm_fwd(const NormFwdParams& p, cudaStream_t stream);

struct NormBwdParams {
    const void *h, *weight, *dy, *dh;  // weight, dh: or null
    const float* rstd;
    void *dx, *dr;                     // either or null
    float *dw, *partial;               // or null; partial: norm_bwd_partials(M, D) x D floats at most
    long long M, ldh, lddy, lddh, lddx, lddr;
    int D;
    Dropout d;
    bool h_f32, w_f32, y_f32, x_f32;   // dy has y's type, dx x's, dh and dr have h's
};
int norm_bwd_partials(long long M, long long D);
int launch_norm_bwd(const NormBwdParams& p, cudaStream_t stream);

struct QuantizeParams {
    const void* x;
    signed char* q;
    float* scale;
    long long M, K, ldx, ldq;
    bool x_f32;
};
int launch_quantize(const QuantizeParams& p, cudaStream_t stream);

}  // namespace wkv7

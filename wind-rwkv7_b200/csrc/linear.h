// Interface between the C ABI (capi.cu) and the dense products with their epilogue (linear.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace wkv7 {

enum LinearAct : int { kActNone = 0, kActRelu = 1, kActRelu2 = 2, kActTanh = 3, kActSigmoid = 4, kActSilu = 5, kActGelu = 6, kActs = 7 };

// what happens to a product between the accumulator and memory
struct LinearEpilogue {
    const void* bias;      // [cols] or null
    const void* residual;  // [rows, cols], of y's type, or null
    void* y;               // [rows, cols]
    void* z;               // [rows, ldz] bf16 or fp32, the argument of the activation, or null
    long long ldr, ldy, ldz, rows, cols;
    int act;
    bool bias_f32, y_f32, z_f32;
    const float *xs = nullptr, *ws = nullptr;  // operands in 8 bits: the rows' and the columns' scales, [rows] and [cols]; null: bf16 operands
};

// y[rows, cols] = epilogue(sum_k P[i, k] Q[j, k]); an operand is [index, k] with k contiguous, or (`_mn`) [k, index] with the index contiguous
struct LinearOperand {
    const void* p;
    long long ld;
    bool mn;
};
// 8-bit operands (epilogues with scales): K-major, rows a multiple of 16 bytes apart, k < 2^17 (a sum of 2^17 products of -128 leaves 32 bits), no z.
// workspace: linear_workspace_bytes() bytes (rows_mn: the rows' operand is [k, index]), or null: no tile is cut along k
size_t linear_workspace_bytes(long long rows, long long cols, long long k, bool rows_mn, bool i8 = false);
int launch_linear(LinearOperand rows, LinearOperand cols, long long k, const LinearEpilogue& e, void* workspace, int* status, cudaStream_t stream);

// products in 8 bits of few rows (linear_int8.cu): whether they are done so, and the launch
bool int8_rows_fit(long long rows, long long cols, long long k);
int launch_int8_rows(LinearOperand x, LinearOperand w, long long k, const LinearEpilogue& e, cudaStream_t stream);

// dz = dy act'(saved) as bf16 [M, ldz] (not written where dz is null) and dbias = column sums of dz (or null; then of dz before its rounding)
struct LinearDz {
    const void *dy, *saved;
    void* dz;
    float *dbias, *partial;  // partial: linear_dz_chunks(M, N) x N floats, where dbias is wanted
    long long M, N, lddy, lds, ldz;
    int act;
    bool dy_f32, saved_f32, from_y;     // from_y: `saved` is the activation's value, not its argument
};
int linear_dz_chunks(long long M, long long N);
int launch_linear_dz(const LinearDz& p, cudaStream_t stream);

}  // namespace wkv7

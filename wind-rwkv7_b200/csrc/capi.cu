// extern "C" entry points of libwkv7_sm100.so (declared in include/wkv7_sm100.h): host-side
// validation, the per-device status word, and dispatch to the kernel launchers.
#include <atomic>
#include <cmath>
#include <cstdlib>
#include "../../include/wkv7_sm100.h"
#include "wkv7_kernels.h"
#include "ddlerp.h"
#include "expand_loras.h"
#include "linear.h"
#include "beam.h"
#include "norm.h"

#include <mutex>

// Scratch for wkv7_attn_ln_bwd_static: lives in the library's device image, one copy on every GPU
// that loads the library, until the process exits.  Only its ADDRESS ON THE DEVICE may be given
// to a kernel; in host code the name is a host-side stand-in, so the address is fetched once
// per device with cudaGetSymbolAddress (see static_scratch()).
static __device__ __align__(256) float g_attn_ln_static_scratch[WKV7_STATIC_SCRATCH_BYTES / sizeof(float)];

namespace {

// The status word that a kernel's bounded wait writes when it gives up: a managed variable, part of the library's
// image (nothing is allocated at run time), one per process, readable by the host while kernels run (concurrent
// managed access), so that wkv7_peek_status() is a plain load that synchronises nothing.  The page stays on the host
// side unless a kernel reports an error.
__managed__ int g_status_word = 0;

int* status_ptr() {
    static int* word = [] {
        int* p = nullptr;
        if (cudaGetSymbolAddress((void**)&p, g_status_word) != cudaSuccess) p = nullptr;
        return p;
    }();
    return word;
}

// Device address of g_attn_ln_static_scratch on the current device, looked up on the first call
// for that device and cached.  Returns nullptr if the lookup fails.
float* static_scratch() {
    constexpr int kMaxDevices = 64;
    static float* cache[kMaxDevices] = {};
    static std::mutex mu;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
    std::lock_guard<std::mutex> lock(mu);
    if (!cache[dev]) {
        float* ptr = nullptr;
        if (cudaGetSymbolAddress((void**)&ptr, g_attn_ln_static_scratch) != cudaSuccess) return nullptr;
        cache[dev] = ptr;
    }
    return cache[dev];
}

// Forward implementation for bf16 attn (see wkv7_set_fwd_impl in the header): 0 = warp-MMA kernel,
// +-2..4 = tcgen05 kernel with 3..5 slots (attn_ln: 4), negative: operands not rounded.
bool valid_fwd_impl(int x) { return x == 0 || (x >= 2 && x <= 4) || (x <= -2 && x >= -4); }
std::atomic<int>& fwd_impl() {
    static std::atomic<int> v([] {
        const char* e = std::getenv("WKV7_FWD_TC");
        if (!e) return 4;
        const int x = std::atoi(e);
        return valid_fwd_impl(x) ? x : 0;
    }());
    return v;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_common(int64_t B, int64_t T, int64_t H, int64_t N, int64_t sb, int64_t st, int64_t sh, int io_dtype) {
    if (B < 0 || T < 0 || H < 0 || N <= 0) return wkv7::kBadShape;
    if (N != wkv7::N) return wkv7::kBadHeadSize;
    if (io_dtype != WKV7_BF16 && io_dtype != WKV7_F32 && io_dtype != WKV7_F32_TF32) return wkv7::kBadDtype;
    const int64_t per16 = io_dtype == WKV7_BF16 ? 8 : 4;  // elements per 16 bytes
    if (sb % per16 || st % per16 || sh % per16) return wkv7::kBadAlign;
    if (sb < 0 || st < 0 || sh < 0) return wkv7::kBadShape;
    // entries that all lie in one place: outputs cannot, and a tensor map has no such stride
    if ((B > 1 && sb == 0) || (T > 1 && st == 0) || (H > 1 && sh == 0)) return wkv7::kBadShape;
    if (B * H > 0x7fffffffLL) return wkv7::kTooLarge;
    // the kernels address checkpoint records through 32-bit row coordinates of their tensor maps (80 rows of 64 floats
    // per record)
    if (B * H > 0 && (T + wkv7::L - 1) / wkv7::L > (0x7fffffffLL / (wkv7::CK_FLOATS / wkv7::N)) / (B * H)) return wkv7::kTooLarge;
    return wkv7::kOk;
}

}  // namespace

namespace wkv7 {
int sm_count() {
    constexpr int kMaxDevices = 64;
    static std::atomic<int> cache[kMaxDevices];
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    int n = cache[dev].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        cache[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

WorkSplit plan_work(long long chains, long long per_chain, int per_sm, unsigned* flags) {
    long long ctas = chains, per_cta = per_chain;
    const long long slots = (long long)sm_count() * per_sm;
    if (flags && slots > 0 && slots * sizeof(unsigned) <= WORK_FLAG_BYTES && chains > slots) {
        ctas = slots;
        per_cta = (chains * per_chain + slots - 1) / slots;
        ctas = (chains * per_chain + per_cta - 1) / per_cta;  // no empty ranges
    } else {
        flags = nullptr;
    }
    return WorkSplit{(int)ctas, (int)per_cta, (int)per_chain, (int)(chains * per_chain), flags};
}
}  // namespace wkv7

extern "C" {

const char* wkv7_status_string(int status) {
    switch (status) {
        case WKV7_OK: return "ok";
        case WKV7_ERR_SHAPE: return "bad shape: negative or inconsistent dimensions";
        case WKV7_ERR_HEAD_SIZE: return "unsupported head size: only N == 64 is built";
        case WKV7_ERR_CHUNK: return "ddlerp, expand_loras: C must be a multiple of 64";
        case WKV7_ERR_ALIGN: return "pointer or stride breaks 16-byte row alignment";
        case WKV7_ERR_DTYPE: return "unknown io_dtype";
        case WKV7_ERR_NULL: return "a required pointer is null";
        case WKV7_ERR_LAUNCH: return "CUDA launch failed";
        case WKV7_ERR_TOO_LARGE: return "B*H exceeds the grid limit, or B*H*ceil(T/16) checkpoint records exceed 32-bit row addressing";
        case WKV7_ERR_DEVICE_TIMEOUT: return "a bounded device-side wait ran out";
        case WKV7_ERR_STATIC_SCRATCH: return "problem needs more than WKV7_STATIC_SCRATCH_BYTES of built-in scratch (B*3*H*N*4 bytes); use wkv7_attn_ln_bwd with a caller-provided workspace";
        case WKV7_ERR_INDEX: return "wkv7_reorder: a parent beam that does not exist";
        default: return "unknown status";
    }
}

int64_t wkv7_checkpoint_bytes(int64_t B, int64_t T, int64_t H, int64_t N) {
    if (B < 0 || T < 0 || H < 0 || N < 0) return 0;
    if (N != wkv7::N) return 0;
    return B * H * ((T + wkv7::L - 1) / wkv7::L) * (int64_t)wkv7::CK_FLOATS * (int64_t)sizeof(float);
}

__device__ long long g_selftest_cycles[4];

int wkv7_selftest_bounded_wait(int64_t limit_cycles, int64_t* cycles_out, void* stream) {
    if (limit_cycles <= 0 || limit_cycles > (1LL << 28)) return WKV7_ERR_SHAPE;
    int* status = status_ptr();
    long long* cyc = nullptr;
    if (!status || cudaGetSymbolAddress((void**)&cyc, g_selftest_cycles) != cudaSuccess) return WKV7_ERR_LAUNCH;
    int rc = wkv7::launch_bounded_wait_selftest(limit_cycles, status, cyc, (cudaStream_t)stream);
    if (rc) return rc;
    if (cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess) return WKV7_ERR_LAUNCH;
    if (cycles_out) {
        long long h[4];
        if (cudaMemcpy(h, cyc, sizeof(h), cudaMemcpyDeviceToHost) != cudaSuccess) return WKV7_ERR_LAUNCH;
        for (int i = 0; i < 4; ++i) cycles_out[i] = h[i];
    }
    return wkv7_device_status();
}

int wkv7_set_fwd_impl(int impl) {
    if (!valid_fwd_impl(impl)) return WKV7_ERR_SHAPE;
    fwd_impl().store(impl, std::memory_order_relaxed);
    return WKV7_OK;
}

int wkv7_get_fwd_impl(void) { return fwd_impl().load(std::memory_order_relaxed); }

int wkv7_device_status(void) {
    int* w = status_ptr();
    if (!w) return WKV7_ERR_LAUNCH;
    if (cudaDeviceSynchronize() != cudaSuccess) return WKV7_ERR_LAUNCH;  // every stream of the current device, non-blocking ones too
    return __atomic_exchange_n(w, 0, __ATOMIC_ACQ_REL);                  // read and clear in one step
}

int wkv7_peek_status(void) {
    int* w = status_ptr();
    return w ? __atomic_load_n(w, __ATOMIC_ACQUIRE) : WKV7_ERR_LAUNCH;
}

static int fwd_common(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                      const void* g, const float* params, bool ln, float eps, const float* s0, void* y, float* sT,
                      float* ckpt, int64_t B, int64_t T, int64_t H, int64_t N, int64_t sb, int64_t st, int64_t sh,
                      int io_dtype, void* workspace, void* stream) {
    int rc = check_common(B, T, H, N, sb, st, sh, io_dtype);
    if (rc) return rc;
    if (B == 0 || H == 0) return WKV7_OK;
    if (T == 0) {  // nothing to scan: the state passes through
        if (sT) {
            size_t bytes = (size_t)B * H * N * N * sizeof(float);
            cudaError_t e = s0 ? cudaMemcpyAsync(sT, s0, bytes, cudaMemcpyDeviceToDevice, (cudaStream_t)stream)
                               : cudaMemsetAsync(sT, 0, bytes, (cudaStream_t)stream);
            if (e != cudaSuccess) return WKV7_ERR_LAUNCH;
        }
        return WKV7_OK;
    }
    if (!r || !w || !k || !v || !a || !b || !y || (ln && (!g || !params))) return WKV7_ERR_NULL;
    const void* ptrs[] = {r, w, k, v, a, b, y, g, s0, sT, ckpt, params, workspace};
    for (const void* p : ptrs)
        if (p && !aligned16(p)) return WKV7_ERR_ALIGN;
    wkv7::FwdParams p{};
    p.r = r; p.w = w; p.k = k; p.v = v; p.a = a; p.b = b; p.g = g; p.params = params;
    p.s0 = s0; p.y = y; p.sT = sT; p.ckpt = ckpt;
    p.B = B; p.T = T; p.H = H;
    p.st = wkv7::Strides{sb, st, sh};
    p.eps = eps;
    p.flags = (unsigned*)workspace;
    p.status = status_ptr();
    if (!p.status) return WKV7_ERR_LAUNCH;
    if (io_dtype == WKV7_BF16) {
        const int impl = fwd_impl().load(std::memory_order_relaxed);
        if (impl) return wkv7::launch_fwd_tc(p, impl, ln, (cudaStream_t)stream);
    }
    return wkv7::launch_fwd(p, io_dtype, ln, (cudaStream_t)stream);
}

int wkv7_fwd(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
             const float* s0, void* y, float* sT, float* ckpt, int64_t B, int64_t T, int64_t H, int64_t N,
             int64_t stride_b, int64_t stride_t, int64_t stride_h, int io_dtype, void* stream) {
    return fwd_common(r, w, k, v, a, b, nullptr, nullptr, false, 0.f, s0, y, sT, ckpt, B, T, H, N, stride_b, stride_t,
                      stride_h, io_dtype, nullptr, stream);
}

size_t wkv7_workspace_bytes(void) { return wkv7::WORK_FLAG_BYTES; }

static int64_t bwd_scratch_bytes(int64_t B, int64_t T, int64_t H, int64_t N, int io_dtype, bool ln) {
    if (B < 0 || T < 0 || H < 0 || N != wkv7::N) return 0;
    if (io_dtype == WKV7_BF16) return (int64_t)wkv7::bwd_workspace_bytes(B, T, H, ln);
    return (int64_t)(io_dtype == WKV7_F32 && !ln ? wkv7::bwd32_workspace_bytes(B, T, H) : wkv7::WORK_FLAG_BYTES);
}
int64_t wkv7_bwd_ws_bytes(int64_t B, int64_t T, int64_t H, int64_t N, int io_dtype) { return bwd_scratch_bytes(B, T, H, N, io_dtype, false); }
int64_t wkv7_attn_ln_bwd_ws_bytes(int64_t B, int64_t T, int64_t H, int64_t N, int io_dtype) { return bwd_scratch_bytes(B, T, H, N, io_dtype, true); }

int wkv7_fwd_ws(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                const float* s0, void* y, float* sT, float* ckpt, int64_t B, int64_t T, int64_t H, int64_t N,
                int64_t stride_b, int64_t stride_t, int64_t stride_h, int io_dtype, void* workspace, void* stream) {
    return fwd_common(r, w, k, v, a, b, nullptr, nullptr, false, 0.f, s0, y, sT, ckpt, B, T, H, N, stride_b, stride_t,
                      stride_h, io_dtype, workspace, stream);
}

int64_t wkv7_fwd_time_split_workspace_bytes(int64_t B, int64_t H, int64_t nseg) {
    return B < 0 || H < 0 || nseg < 0 ? 0 : (int64_t)wkv7::time_split_workspace_bytes(B, H, (int)nseg);
}

int wkv7_fwd_time_split(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                        const float* s0, void* y, float* sT, int64_t B, int64_t T, int64_t H, int64_t N, int64_t nseg,
                        int64_t stride_t, void* workspace, void* stream) {
    int rc = check_common(B, T, H, N, T * stride_t, stride_t, N, WKV7_BF16);
    if (rc) return rc;
    if (nseg < 2 || nseg > 4096 || T % nseg != 0) return WKV7_ERR_SHAPE;
    if (B == 0 || H == 0 || T == 0) return WKV7_ERR_SHAPE;
    if (!r || !w || !k || !v || !a || !b || !y || !workspace) return WKV7_ERR_NULL;
    const void* ptrs[] = {r, w, k, v, a, b, y, s0, sT, workspace};
    for (const void* p : ptrs)
        if (p && !aligned16(p)) return WKV7_ERR_ALIGN;
    if (B * nseg * H > 0x7fffffff) return WKV7_ERR_TOO_LARGE;
    const int impl = fwd_impl().load(std::memory_order_relaxed);
    wkv7::FwdParams p{};
    p.r = r; p.w = w; p.k = k; p.v = v; p.a = a; p.b = b; p.s0 = s0; p.y = y; p.sT = sT;
    p.B = B; p.T = T; p.H = H;
    p.st = wkv7::Strides{T * stride_t, stride_t, N};
    p.flags = (unsigned*)workspace;
    p.status = status_ptr();
    if (!p.status) return WKV7_ERR_LAUNCH;
    return wkv7::launch_fwd_time_split(p, (int)nseg, impl ? impl : 4, (cudaStream_t)stream);
}

int wkv7_step(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b, const float* s0,
              void* y, float* sT, int64_t B, int64_t T, int64_t H, int64_t N, int64_t stride_b, int64_t stride_t,
              int64_t stride_h, int io_dtype, void* stream) {
    int rc = check_common(B, T, H, N, stride_b, stride_t, stride_h, io_dtype);
    if (rc) return rc;
    if (B == 0 || H == 0) return WKV7_OK;
    if (T == 0) {
        if (sT && sT != s0) {
            size_t bytes = (size_t)B * H * N * N * sizeof(float);
            cudaError_t e = s0 ? cudaMemcpyAsync(sT, s0, bytes, cudaMemcpyDeviceToDevice, (cudaStream_t)stream)
                               : cudaMemsetAsync(sT, 0, bytes, (cudaStream_t)stream);
            if (e != cudaSuccess) return WKV7_ERR_LAUNCH;
        }
        return WKV7_OK;
    }
    if (!r || !w || !k || !v || !a || !b || !y) return WKV7_ERR_NULL;
    const void* ptrs[] = {r, w, k, v, a, b, y, s0, sT};
    for (const void* q : ptrs)
        if (q && !aligned16(q)) return WKV7_ERR_ALIGN;
    wkv7::StepParams p{};
    p.r = r; p.w = w; p.k = k; p.v = v; p.a = a; p.b = b; p.s0 = s0; p.y = y; p.sT = sT;
    p.B = B; p.T = T; p.H = H;
    p.st = wkv7::Strides{stride_b, stride_t, stride_h};
    p.status = status_ptr();
    return wkv7::launch_step(p, io_dtype == WKV7_BF16 ? 0 : 1, (cudaStream_t)stream);
}

int wkv7_attn_ln_fwd(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                     const void* g, const float* params, const float* s0, void* y, float* sT, float* ckpt, float eps,
                     int64_t B, int64_t T, int64_t H, int64_t N, int64_t stride_b, int64_t stride_t, int64_t stride_h,
                     int io_dtype, void* stream) {
    return fwd_common(r, w, k, v, a, b, g, params, true, eps, s0, y, sT, ckpt, B, T, H, N, stride_b, stride_t,
                      stride_h, io_dtype, nullptr, stream);
}

int wkv7_attn_ln_fwd_ws(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                        const void* g, const float* params, const float* s0, void* y, float* sT, float* ckpt, float eps,
                        int64_t B, int64_t T, int64_t H, int64_t N, int64_t stride_b, int64_t stride_t, int64_t stride_h,
                        int io_dtype, void* workspace, void* stream) {
    return fwd_common(r, w, k, v, a, b, g, params, true, eps, s0, y, sT, ckpt, B, T, H, N, stride_b, stride_t,
                      stride_h, io_dtype, workspace, stream);
}

static int bwd_common(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                      const void* g, const float* params, bool ln, float eps, const void* dy, const float* ckpt,
                      const float* dsT, const float* sT, void* dr, void* dw, void* dk, void* dv, void* da, void* db,
                      void* dg, float* dparams, float* dparams_ws, float* ds0, int64_t B, int64_t T, int64_t H, int64_t N,
                      int64_t stride_b, int64_t stride_t, int64_t stride_h, int io_dtype, void* workspace, void* stream) {
    int rc = check_common(B, T, H, N, stride_b, stride_t, stride_h, io_dtype);
    if (rc) return rc;
    if (B == 0 || H == 0) return WKV7_OK;
    if (T == 0) {
        if (ln && dparams) {
            if (cudaMemsetAsync(dparams, 0, (size_t)3 * H * N * sizeof(float), (cudaStream_t)stream) != cudaSuccess)
                return WKV7_ERR_LAUNCH;
        }
        if (ds0) {
            size_t bytes = (size_t)B * H * N * N * sizeof(float);
            cudaError_t e = dsT ? cudaMemcpyAsync(ds0, dsT, bytes, cudaMemcpyDeviceToDevice, (cudaStream_t)stream)
                                : cudaMemsetAsync(ds0, 0, bytes, (cudaStream_t)stream);
            if (e != cudaSuccess) return WKV7_ERR_LAUNCH;
        }
        return WKV7_OK;
    }
    if (!r || !w || !k || !v || !a || !b || !dy || !ckpt || !dr || !dw || !dk || !dv || !da || !db) return WKV7_ERR_NULL;
    if (dsT && !sT) return WKV7_ERR_NULL;
    if (ln && (!g || !params || !dg || !dparams || !dparams_ws)) return WKV7_ERR_NULL;
    const void* ptrs[] = {r, w, k, v, a, b, dy, ckpt, dsT, sT, dr, dw, dk, dv, da, db, ds0, g, params, dg, dparams, dparams_ws, workspace};
    for (const void* p : ptrs)
        if (p && !aligned16(p)) return WKV7_ERR_ALIGN;
    wkv7::BwdParams p{};
    p.r = r; p.w = w; p.k = k; p.v = v; p.a = a; p.b = b; p.dy = dy;
    p.ckpt = ckpt; p.dsT = dsT; p.sT = sT;
    p.g = g; p.params = params; p.dg = dg; p.dparams = dparams; p.dparams_ws = dparams_ws; p.eps = eps;
    p.dr = dr; p.dw = dw; p.dk = dk; p.dv = dv; p.da = da; p.db = db; p.ds0 = ds0;
    p.B = B; p.T = T; p.H = H;
    p.st = wkv7::Strides{stride_b, stride_t, stride_h};
    p.flags = (unsigned*)workspace;
    p.status = status_ptr();
    if (!p.status) return WKV7_ERR_LAUNCH;
    return wkv7::launch_bwd(p, io_dtype, ln, (cudaStream_t)stream);
}

int wkv7_bwd(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
             const void* dy, const float* ckpt, const float* dsT, const float* sT, void* dr, void* dw, void* dk,
             void* dv, void* da, void* db, float* ds0, int64_t B, int64_t T, int64_t H, int64_t N, int64_t stride_b,
             int64_t stride_t, int64_t stride_h, int io_dtype, void* stream) {
    return bwd_common(r, w, k, v, a, b, nullptr, nullptr, false, 0.f, dy, ckpt, dsT, sT, dr, dw, dk, dv, da, db, nullptr,
                      nullptr, nullptr, ds0, B, T, H, N, stride_b, stride_t, stride_h, io_dtype, nullptr, stream);
}

int wkv7_bwd_ws(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                const void* dy, const float* ckpt, const float* dsT, const float* sT, void* dr, void* dw, void* dk,
                void* dv, void* da, void* db, float* ds0, int64_t B, int64_t T, int64_t H, int64_t N, int64_t stride_b,
                int64_t stride_t, int64_t stride_h, int io_dtype, void* workspace, void* stream) {
    return bwd_common(r, w, k, v, a, b, nullptr, nullptr, false, 0.f, dy, ckpt, dsT, sT, dr, dw, dk, dv, da, db, nullptr,
                      nullptr, nullptr, ds0, B, T, H, N, stride_b, stride_t, stride_h, io_dtype, workspace, stream);
}

int64_t wkv7_attn_ln_bwd_workspace_bytes(int64_t B, int64_t H, int64_t N) {
    if (B < 0 || H < 0 || N < 0) return 0;
    return B * 3 * H * N * (int64_t)sizeof(float);
}

int wkv7_attn_ln_bwd(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                     const void* g, const float* params, const void* dy, const float* ckpt, const float* dsT,
                     const float* sT, void* dr, void* dw, void* dk, void* dv, void* da, void* db, void* dg,
                     float* dparams, float* workspace, float* ds0, float eps, int64_t B, int64_t T, int64_t H,
                     int64_t N, int64_t stride_b, int64_t stride_t, int64_t stride_h, int io_dtype, void* stream) {
    return bwd_common(r, w, k, v, a, b, g, params, true, eps, dy, ckpt, dsT, sT, dr, dw, dk, dv, da, db, dg, dparams,
                      workspace, ds0, B, T, H, N, stride_b, stride_t, stride_h, io_dtype, nullptr, stream);
}

int wkv7_attn_ln_bwd_ws(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                        const void* g, const float* params, const void* dy, const float* ckpt, const float* dsT,
                        const float* sT, void* dr, void* dw, void* dk, void* dv, void* da, void* db, void* dg,
                        float* dparams, float* dparams_workspace, float* ds0, float eps, int64_t B, int64_t T, int64_t H,
                        int64_t N, int64_t stride_b, int64_t stride_t, int64_t stride_h, int io_dtype, void* workspace, void* stream) {
    return bwd_common(r, w, k, v, a, b, g, params, true, eps, dy, ckpt, dsT, sT, dr, dw, dk, dv, da, db, dg, dparams,
                      dparams_workspace, ds0, B, T, H, N, stride_b, stride_t, stride_h, io_dtype, workspace, stream);
}

int wkv7_attn_ln_bwd_static(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                            const void* g, const float* params, const void* dy, const float* ckpt, const float* dsT,
                            const float* sT, void* dr, void* dw, void* dk, void* dv, void* da, void* db, void* dg,
                            float* dparams, float* ds0, float eps, int64_t B, int64_t T, int64_t H, int64_t N,
                            int64_t stride_b, int64_t stride_t, int64_t stride_h, int io_dtype, void* stream) {
    if (B < 0 || H < 0 || N < 0) return WKV7_ERR_SHAPE;
    if (wkv7_attn_ln_bwd_workspace_bytes(B, H, N) > (int64_t)WKV7_STATIC_SCRATCH_BYTES) return WKV7_ERR_STATIC_SCRATCH;
    float* scratch = static_scratch();
    if (!scratch) return WKV7_ERR_LAUNCH;
    return bwd_common(r, w, k, v, a, b, g, params, true, eps, dy, ckpt, dsT, sT, dr, dw, dk, dv, da, db, dg, dparams,
                      scratch, ds0, B, T, H, N, stride_b, stride_t, stride_h, io_dtype, nullptr, stream);
}

int wkv7_proj_gemm_group_ld(int count, const void* const* A, const void* const* W, void* const* C, const int64_t* N, const int64_t* K,
                            const int64_t* lda, const int64_t* tanh_from, const int64_t* tanh_to, int64_t M, void* stream) {
    if (count < 1 || count > WKV7_PROJ_LD_MAX || M < 0) return WKV7_ERR_SHAPE;
    for (int i = 0; i < count; ++i) {
        if (K[i] <= 0 || lda[i] < K[i] || N[i] <= 0 || tanh_from[i] < 0 || tanh_to[i] < tanh_from[i] || tanh_to[i] > N[i]) return WKV7_ERR_SHAPE;
        if (N[i] % 8 != 0 || K[i] % 8 != 0 || lda[i] % 8 != 0) return WKV7_ERR_ALIGN;   // 16-byte rows for the bulk tensor loads and the stores
        if (M > 0x7fffffffLL || N[i] > 0x7fffffffLL || lda[i] > 0x7fffffffLL || (M + 127) / 128 > 65535) return WKV7_ERR_TOO_LARGE;
        if (M == 0) continue;
        if (!A[i] || !W[i] || !C[i]) return WKV7_ERR_NULL;
        if (!aligned16(A[i]) || !aligned16(W[i]) || !aligned16(C[i])) return WKV7_ERR_ALIGN;
    }
    if (M == 0) return WKV7_OK;
    int* status = status_ptr();
    if (!status) return WKV7_ERR_LAUNCH;
    return wkv7::launch_proj_gemm(count, A, W, C, N, K, lda, tanh_from, tanh_to, M, status, (cudaStream_t)stream);
}

int wkv7_proj_gemm_group(int count, const void* const* A, const void* const* W, void* const* C, const int64_t* N, const int64_t* tanh_from,
                         const int64_t* tanh_to, int64_t M, int64_t K, void* stream) {
    if (count < 1 || count > WKV7_PROJ_MAX) return WKV7_ERR_SHAPE;
    int64_t k[WKV7_PROJ_MAX];
    for (int i = 0; i < count; ++i) k[i] = K;
    return wkv7_proj_gemm_group_ld(count, A, W, C, N, k, k, tanh_from, tanh_to, M, stream);
}

int wkv7_proj_gemm(const void* A, const void* W, void* C, int64_t M, int64_t N, int64_t K, int64_t tanh_from,
                   int64_t tanh_to, void* stream) {
    return wkv7_proj_gemm_group(1, &A, &W, &C, &N, &tanh_from, &tanh_to, M, K, stream);
}

static_assert(WKV7_PROJ_LD_MAX == wkv7::PROJ_MAX && WKV7_PROJ_MAX <= wkv7::PROJ_MAX, "mirrored constants");

static_assert(WKV7_ACT_NONE == wkv7::kActNone && WKV7_ACT_RELU == wkv7::kActRelu && WKV7_ACT_RELU2 == wkv7::kActRelu2 && WKV7_ACT_TANH == wkv7::kActTanh &&
              WKV7_ACT_SIGMOID == wkv7::kActSigmoid && WKV7_ACT_SILU == wkv7::kActSilu && WKV7_ACT_GELU == wkv7::kActGelu, "mirrored constants");

static int linear_check(const void* x, const void* w, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int act, int flags, int known_flags) {
    if (M < 0 || N <= 0 || K <= 0 || ldx < K || ldw < K || act < 0 || act >= wkv7::kActs || (flags & ~known_flags)) return WKV7_ERR_SHAPE;
    if (K % 8 != 0 || ldx % 8 != 0 || ldw % 8 != 0) return WKV7_ERR_ALIGN;  // 16-byte rows for the bulk tensor copies
    // coordinates of the copies are 32 bits wide (tiles overhang by up to 255), strides of the maps 40
    constexpr int64_t most = 0x7fffffffLL - 256;
    if (M > most || N > most || K > most || ldx > most || ldw > most) return WKV7_ERR_TOO_LARGE;
    if (M == 0) return WKV7_OK;
    if (!x || !w) return WKV7_ERR_NULL;
    return aligned16(x) && aligned16(w) ? WKV7_OK : WKV7_ERR_ALIGN;
}

int wkv7_linear_fwd(const void* x, const void* w, const void* bias, const void* residual, void* y, void* z, int64_t M, int64_t N, int64_t K,
                    int64_t ldx, int64_t ldw, int64_t ldr, int64_t ldy, int64_t ldz, int act, int flags, void* workspace, void* stream) {
    int rc = linear_check(x, w, M, N, K, ldx, ldw, act, flags, WKV7_LINEAR_F32_OUT | WKV7_LINEAR_F32_BIAS | WKV7_LINEAR_F32_Z);
    if (rc) return rc;
    const int64_t n8 = (N + 7) / 8 * 8;
    if (ldy < N || (residual && ldr < N) || (z && ldz < n8)) return WKV7_ERR_SHAPE;
    if ((z && (ldz % 8 != 0 || !aligned16(z))) || !aligned16(workspace)) return WKV7_ERR_ALIGN;
    if (M == 0) return WKV7_OK;
    if (!y) return WKV7_ERR_NULL;
    const uintptr_t ysize = flags & WKV7_LINEAR_F32_OUT ? 4 : 2, bsize = flags & WKV7_LINEAR_F32_BIAS ? 4 : 2;
    if ((uintptr_t)y % ysize || (uintptr_t)residual % ysize || (uintptr_t)bias % bsize) return WKV7_ERR_ALIGN;
    int* status = status_ptr();
    if (!status) return WKV7_ERR_LAUNCH;
    const wkv7::LinearEpilogue e{bias, residual, y, z, ldr, ldy, ldz, M, N, act, bsize == 4, ysize == 4, (flags & WKV7_LINEAR_F32_Z) != 0};
    return wkv7::launch_linear({x, ldx, false}, {w, ldw, false}, K, e, workspace, status, (cudaStream_t)stream);
}

int64_t wkv7_linear_fwd_workspace_bytes(int64_t M, int64_t N, int64_t K) { return M <= 0 || N <= 0 || K <= 0 ? 0 : (int64_t)wkv7::linear_workspace_bytes(M, N, K, false); }

static int64_t linear_dz_bytes(int64_t M, int64_t N) { return (M * ((N + 7) / 8 * 8) * 2 + 15) / 16 * 16; }

// dz, the chunks' sums for dbias, and the scratch of the two products, which follow one another
static int64_t linear_sums_bytes(int64_t M, int64_t N) { return ((int64_t)wkv7::linear_dz_chunks(M, N) * N * 4 + 15) / 16 * 16; }
int64_t wkv7_linear_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const size_t a = wkv7::linear_workspace_bytes(M, K, N, false), b = wkv7::linear_workspace_bytes(N, K, M, true);
    return linear_dz_bytes(M, N) + linear_sums_bytes(M, N) + (int64_t)(a > b ? a : b);
}

int wkv7_linear_bwd(const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw, float* dbias, int64_t M, int64_t N, int64_t K,
                    int64_t ldx, int64_t ldw, int64_t lds, int64_t lddy, int act, int flags, void* workspace, void* stream) {
    int rc = linear_check(x, w, M, N, K, ldx, ldw, act, flags, WKV7_LINEAR_F32_OUT | WKV7_LINEAR_FROM_Y | WKV7_LINEAR_F32_Z);
    if (rc) return rc;
    const bool from_y = flags & WKV7_LINEAR_FROM_Y, f32 = flags & WKV7_LINEAR_F32_OUT, z32 = flags & WKV7_LINEAR_F32_Z;
    if (from_y && ((act != WKV7_ACT_RELU && act != WKV7_ACT_RELU2) || f32 || z32)) return WKV7_ERR_SHAPE;
    if (lddy < N || (act && lds < N)) return WKV7_ERR_SHAPE;
    cudaStream_t s = (cudaStream_t)stream;
    if (M == 0) {  // sums over nothing
        if ((dw && cudaMemsetAsync(dw, 0, (size_t)N * K * 2, s) != cudaSuccess) || (dbias && cudaMemsetAsync(dbias, 0, (size_t)N * 4, s) != cudaSuccess)) return WKV7_ERR_LAUNCH;
        return WKV7_OK;
    }
    if (!dy || !workspace || (act && !saved)) return WKV7_ERR_NULL;
    if (!aligned16(workspace) || (dx && !aligned16(dx)) || (dw && !aligned16(dw)) || (uintptr_t)dbias % 4 || (uintptr_t)dy % (f32 ? 4 : 2) || (act && (uintptr_t)saved % (z32 ? 4 : 2)))
        return WKV7_ERR_ALIGN;
    int* status = status_ptr();
    if (!status) return WKV7_ERR_LAUNCH;
    // without an activation a bf16 dy whose rows the bulk copies can read is dz
    const bool as_is = !act && !f32 && aligned16(dy) && lddy % 8 == 0;
    wkv7::LinearOperand dz{dy, lddy, false};
    if (!as_is || dbias) {
        if (!as_is) dz = wkv7::LinearOperand{workspace, (N + 7) / 8 * 8, false};
        if (dbias || ((dx || dw) && !as_is)) {
            const wkv7::LinearDz d{dy, saved, as_is || !(dx || dw) ? nullptr : workspace, dbias, (float*)((char*)workspace + linear_dz_bytes(M, N)), M, N, lddy, lds,
                                   (N + 7) / 8 * 8, act, f32, z32, from_y};
            rc = wkv7::launch_linear_dz(d, s);
            if (rc) return rc;
        }
    }
    void* const scratch = (char*)workspace + linear_dz_bytes(M, N) + linear_sums_bytes(M, N);
    if (dx) {
        const wkv7::LinearEpilogue e{nullptr, nullptr, dx, nullptr, 0, K, 0, M, K, 0, false, false, false};
        rc = wkv7::launch_linear(dz, {w, ldw, true}, N, e, scratch, status, s);
        if (rc) return rc;
    }
    if (dw) {
        const wkv7::LinearEpilogue e{nullptr, nullptr, dw, nullptr, 0, K, 0, N, K, 0, false, false, false};
        rc = wkv7::launch_linear({dz.p, dz.ld, true}, {x, ldx, true}, M, e, scratch, status, s);
    }
    return rc;
}

int64_t wkv7_linear_int8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    return M <= 0 || N <= 0 || K <= 0 ? 0 : (int64_t)wkv7::linear_workspace_bytes(M, N, K, false, true);
}

int wkv7_linear_int8(const void* x, const float* xs, const void* w, const float* ws, const void* bias, const void* residual, void* y, int64_t M, int64_t N, int64_t K,
                     int64_t ldx, int64_t ldw, int64_t ldr, int64_t ldy, int act, int flags, void* workspace, void* stream) {
    if (M < 0 || N <= 0 || K <= 0 || ldx < K || ldw < K || act < 0 || act >= wkv7::kActs || (flags & ~(WKV7_LINEAR_F32_OUT | WKV7_LINEAR_F32_BIAS))) return WKV7_ERR_SHAPE;
    if (ldy < N || (residual && ldr < N)) return WKV7_ERR_SHAPE;
    if (ldx % 16 != 0 || ldw % 16 != 0) return WKV7_ERR_ALIGN;
    constexpr int64_t most = 0x7fffffffLL - 256;  // as wkv7_linear_fwd
    if (M > most || N > most || K >= 1 << 17 || ldx > most || ldw > most) return WKV7_ERR_TOO_LARGE;
    if (M == 0) return WKV7_OK;
    if (!x || !w || !xs || !ws || !y) return WKV7_ERR_NULL;
    const uintptr_t ysize = flags & WKV7_LINEAR_F32_OUT ? 4 : 2, bsize = flags & WKV7_LINEAR_F32_BIAS ? 4 : 2;
    if (!aligned16(x) || !aligned16(w) || !aligned16(workspace) || (uintptr_t)xs % 4 || (uintptr_t)ws % 4 || (uintptr_t)y % ysize || (uintptr_t)residual % ysize ||
        (uintptr_t)bias % bsize)
        return WKV7_ERR_ALIGN;
    int* status = status_ptr();
    if (!status) return WKV7_ERR_LAUNCH;
    const wkv7::LinearEpilogue e{bias, residual, y, nullptr, ldr, ldy, 0, M, N, act, bsize == 4, ysize == 4, false, xs, ws};
    return wkv7::launch_linear({x, ldx, false}, {w, ldw, false}, K, e, workspace, status, (cudaStream_t)stream);
}

int wkv7_quantize(const void* x, void* q, float* scale, int64_t M, int64_t K, int64_t ldx, int64_t ldq, int flags, void* stream) {
    if (M < 0 || K <= 0 || ldx < K || ldq < K || (flags & ~WKV7_X_F32)) return WKV7_ERR_SHAPE;
    if (K > 1 << 30) return WKV7_ERR_TOO_LARGE;
    if (M == 0) return WKV7_OK;
    if (!x || !q || !scale) return WKV7_ERR_NULL;
    if ((uintptr_t)x % (flags & WKV7_X_F32 ? 4 : 2) || (uintptr_t)scale % 4) return WKV7_ERR_ALIGN;
    return wkv7::launch_quantize({x, (signed char*)q, scale, M, K, ldx, ldq, (flags & WKV7_X_F32) != 0}, (cudaStream_t)stream);
}

static_assert(WKV7_NORM_MAX_D == wkv7::NORM_MAX_D, "mirrored constants");

// false: no probability
static bool dropout_of(double p, uint64_t seed, const void* seed_ptr, wkv7::Dropout* d) {
    if (!(p >= 0. && p <= 1.)) return false;
    *d = wkv7::Dropout{(unsigned long long)std::nearbyint(p * 4294967296.), p < 1. ? (float)(1. / (1. - p)) : 0.f, seed, (const unsigned long long*)seed_ptr};
    return true;
}

int wkv7_rms_norm_fwd(const void* x, const void* residual, const void* weight, void* y, void* h, float* rstd, float* scale, int64_t M, int64_t D,
                      int64_t ldx, int64_t ldr, int64_t ldy, int64_t ldh, float eps, double p, uint64_t seed, const void* seed_ptr, int flags, void* stream) {
    wkv7::NormFwdParams n{};
    const bool int8 = flags & WKV7_Y_INT8;
    if (M < 0 || D <= 0 || ldx < D || ldy < D || (residual && (ldr < D || ldh < D)) || !(eps >= 0.f) || (flags & ~(WKV7_X_F32 | WKV7_R_F32 | WKV7_W_F32 | WKV7_Y_F32 | WKV7_Y_INT8)) ||
        (int8 && (flags & WKV7_Y_F32)) || !dropout_of(p, seed, seed_ptr, &n.d))
        return WKV7_ERR_SHAPE;
    if (D > WKV7_NORM_MAX_D) return WKV7_ERR_TOO_LARGE;
    if (M == 0) return WKV7_OK;
    if (p > 0. && !residual) return WKV7_ERR_SHAPE;
    if (!x || !y || !residual != !h || int8 != (scale != nullptr)) return WKV7_ERR_NULL;
    const auto size = [&](int f) -> uintptr_t { return flags & f ? 4 : 2; };
    if ((uintptr_t)x % size(WKV7_X_F32) || (uintptr_t)residual % size(WKV7_R_F32) || (uintptr_t)h % size(WKV7_R_F32) || (uintptr_t)weight % size(WKV7_W_F32) ||
        (!int8 && (uintptr_t)y % size(WKV7_Y_F32)) || (uintptr_t)rstd % 4 || (uintptr_t)scale % 4 || (uintptr_t)seed_ptr % 8)
        return WKV7_ERR_ALIGN;
    n.x = x; n.residual = residual; n.weight = weight; n.y = y; n.h = h; n.rstd = rstd; n.scale = scale;
    n.M = M; n.ldx = ldx; n.ldr = ldr; n.ldy = ldy; n.ldh = ldh; n.D = (int)D; n.eps = eps;
    n.x_f32 = flags & WKV7_X_F32; n.r_f32 = flags & WKV7_R_F32; n.w_f32 = flags & WKV7_W_F32; n.y_f32 = flags & WKV7_Y_F32;
    return wkv7::launch_norm_fwd(n, (cudaStream_t)stream);
}

int64_t wkv7_rms_norm_bwd_workspace_bytes(int64_t M, int64_t D) {
    return M <= 0 || D <= 0 || D > WKV7_NORM_MAX_D ? 0 : (int64_t)wkv7::norm_bwd_partials(M, D) * D * 4;
}

int wkv7_rms_norm_bwd(const void* h, const float* rstd, const void* weight, const void* dy, const void* dh, void* dx, void* dr, float* dw, int64_t M, int64_t D,
                      int64_t ldh, int64_t lddy, int64_t lddh, int64_t lddx, int64_t lddr, double p, uint64_t seed, const void* seed_ptr, int flags, void* workspace,
                      void* stream) {
    wkv7::NormBwdParams n{};
    if (M < 0 || D <= 0 || ldh < D || lddy < D || (dh && lddh < D) || (dx && lddx < D) || (dr && lddr < D) || (flags & ~(WKV7_X_F32 | WKV7_R_F32 | WKV7_W_F32 | WKV7_Y_F32)) ||
        !dropout_of(p, seed, seed_ptr, &n.d))
        return WKV7_ERR_SHAPE;
    if (D > WKV7_NORM_MAX_D) return WKV7_ERR_TOO_LARGE;
    if (M == 0) return dw && cudaMemsetAsync(dw, 0, (size_t)D * 4, (cudaStream_t)stream) != cudaSuccess ? WKV7_ERR_LAUNCH : WKV7_OK;  // a sum over nothing
    if (!h || !rstd || !dy || (dw && !workspace)) return WKV7_ERR_NULL;
    const auto size = [&](int f) -> uintptr_t { return flags & f ? 4 : 2; };
    if ((uintptr_t)h % size(WKV7_R_F32) || (uintptr_t)dh % size(WKV7_R_F32) || (uintptr_t)dr % size(WKV7_R_F32) || (uintptr_t)dx % size(WKV7_X_F32) ||
        (uintptr_t)weight % size(WKV7_W_F32) || (uintptr_t)dy % size(WKV7_Y_F32) || (uintptr_t)rstd % 4 || (uintptr_t)dw % 4 || !aligned16(workspace) || (uintptr_t)seed_ptr % 8)
        return WKV7_ERR_ALIGN;
    n.h = h; n.weight = weight; n.dy = dy; n.dh = dh; n.rstd = rstd; n.dx = dx; n.dr = dr; n.dw = dw; n.partial = (float*)workspace;
    n.M = M; n.ldh = ldh; n.lddy = lddy; n.lddh = lddh; n.lddx = lddx; n.lddr = lddr; n.D = (int)D;
    n.h_f32 = flags & WKV7_R_F32; n.w_f32 = flags & WKV7_W_F32; n.y_f32 = flags & WKV7_Y_F32; n.x_f32 = flags & WKV7_X_F32;
    return wkv7::launch_norm_bwd(n, (cudaStream_t)stream);
}

int wkv7_dropout(const void* x, const void* residual, void* y, int64_t n, double p, uint64_t seed, const void* seed_ptr, int flags, void* stream) {
    wkv7::DropoutParams d{};
    if (n < 0 || (flags & ~(WKV7_X_F32 | WKV7_R_F32 | WKV7_Y_F32)) || !dropout_of(p, seed, seed_ptr, &d.d)) return WKV7_ERR_SHAPE;
    if (n == 0) return WKV7_OK;
    if (!x || !y) return WKV7_ERR_NULL;
    if (!aligned16(x) || !aligned16(residual) || !aligned16(y) || (uintptr_t)seed_ptr % 8) return WKV7_ERR_ALIGN;
    d.x = x; d.residual = residual; d.y = y; d.n = n;
    d.x_f32 = flags & WKV7_X_F32; d.r_f32 = flags & WKV7_R_F32; d.y_f32 = flags & WKV7_Y_F32;
    return wkv7::launch_dropout(d, (cudaStream_t)stream);
}

static_assert(WKV7_ERR_INDEX == wkv7::kBadIndex, "mirrored constants");

static int beam_check(int64_t B, int64_t W, int64_t V, int64_t k) {
    if (B < 0 || W < 1 || V < 1 || k < 1 || W > wkv7::BEAM_MAX_W || k > wkv7::BEAM_MAX_K) return WKV7_ERR_SHAPE;
    if (V > 1 << 30 || W * V > 0x7fffffffLL || B > 0x7fffffffLL / wkv7::BEAM_MAX_W) return WKV7_ERR_TOO_LARGE;
    return k <= W * V ? WKV7_OK : WKV7_ERR_SHAPE;
}

int64_t wkv7_beam_select_workspace_bytes(int64_t B, int64_t W, int64_t V) {
    return beam_check(B, W, V, 1) || B == 0 ? 0 : (int64_t)wkv7::beam_workspace_bytes(B, W, V);
}

int wkv7_beam_select(const void* logits, const float* scores, const void* finished, float* out_scores, int64_t* parents, int64_t* tokens,
                     void* out_finished, int64_t B, int64_t W, int64_t V, int64_t k, int64_t eos, int64_t stride_b, int64_t stride_w, int logits_f32,
                     void* workspace, void* stream) {
    int rc = beam_check(B, W, V, k);
    if (rc) return rc;
    if (stride_b < 0 || stride_w < 0 || (finished && (eos < 0 || eos >= V))) return WKV7_ERR_SHAPE;
    if (B == 0) return WKV7_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens || !workspace || (finished && !out_finished)) return WKV7_ERR_NULL;
    if ((uintptr_t)logits % (logits_f32 ? 4 : 2) || (uintptr_t)scores % 4 || (uintptr_t)out_scores % 4 || (uintptr_t)parents % 8 || (uintptr_t)tokens % 8 || !aligned16(workspace))
        return WKV7_ERR_ALIGN;
    wkv7::BeamParams p{};
    p.logits = logits; p.scores = scores; p.finished = (const unsigned char*)finished;
    p.out_scores = out_scores; p.parents = parents; p.tokens = tokens; p.out_finished = (unsigned char*)out_finished;
    p.sb = stride_b; p.sw = stride_w;
    p.B = (int)B; p.W = (int)W; p.V = (int)V; p.k = (int)k; p.eos = (int)eos; p.f32 = logits_f32 != 0;
    return wkv7::launch_beam_select(p, workspace, (cudaStream_t)stream);
}

int wkv7_reorder(int count, const void* const* src, void* const* dst, const int64_t* row_bytes, const int64_t* src_pitch, const int64_t* dst_pitch,
                 const void* parents, int flags, int64_t B, int64_t W, int64_t k, void* stream) {
    const bool parents_i32 = flags & WKV7_REORDER_I32, keep = flags & WKV7_REORDER_KEEP;
    if ((flags & ~(WKV7_REORDER_I32 | WKV7_REORDER_KEEP)) || (keep && k != W)) return WKV7_ERR_SHAPE;
    if (count < 0 || B < 0 || W < 1 || k < 1 || W > wkv7::BEAM_MAX_W || k > wkv7::BEAM_MAX_K) return WKV7_ERR_SHAPE;
    if (B > 0x7fffffffLL / wkv7::BEAM_MAX_W) return WKV7_ERR_TOO_LARGE;
    for (int i = 0; i < count; ++i) {
        if (row_bytes[i] < 0 || src_pitch[i] < row_bytes[i] || dst_pitch[i] < row_bytes[i]) return WKV7_ERR_SHAPE;
        if (B == 0 || row_bytes[i] == 0) continue;
        if (!src[i] || !dst[i]) return WKV7_ERR_NULL;
        if (src[i] == dst[i] && (k != W || src_pitch[i] != dst_pitch[i])) return WKV7_ERR_SHAPE;
    }
    if (B == 0 || count == 0) return WKV7_OK;
    if (!parents) return WKV7_ERR_NULL;
    if ((uintptr_t)parents % (parents_i32 ? 4 : 8)) return WKV7_ERR_ALIGN;
    int* status = status_ptr();
    if (!status) return WKV7_ERR_LAUNCH;
    for (int from = 0; from < count; from += wkv7::REORDER_MAX) {
        wkv7::ReorderParams p{};
        p.parents = parents; p.idx64 = !parents_i32; p.keep = keep;
        p.B = (int)B; p.W = (int)W; p.k = (int)k; p.status = status;
        for (int i = from; i < count && i < from + wkv7::REORDER_MAX; ++i) {
            if (row_bytes[i] == 0) continue;
            const int j = p.count++;
            p.src[j] = src[i]; p.dst[j] = dst[i];
            p.row_bytes[j] = row_bytes[i]; p.src_pitch[j] = src_pitch[i]; p.dst_pitch[j] = dst_pitch[i];
        }
        const int rc = p.count ? wkv7::launch_reorder(p, (cudaStream_t)stream) : WKV7_OK;
        if (rc) return rc;
    }
    return WKV7_OK;
}

static int ddlerp_check(int64_t B, int64_t T, int64_t C, int64_t D) {
    if (B < 0 || T < 0 || C <= 0 || D <= 0) return WKV7_ERR_SHAPE;
    if (C % 64 != 0) return WKV7_ERR_CHUNK;
    if (D != 16 && D != 32 && D != 64) return WKV7_ERR_SHAPE;  // rank 128: the backward's resident L and R blocks exceed shared memory
    return WKV7_OK;
}

int wkv7_ddlerp_fwd(const void* x, const void* alpha, const void* L, const void* R, const void* beta, void* m, void* y,
                    int64_t B, int64_t T, int64_t C, int64_t D, void* stream) {
    int rc = ddlerp_check(B, T, C, D);
    if (rc) return rc;
    if (B == 0 || T == 0) return WKV7_OK;
    const void* ptrs[] = {x, alpha, L, R, beta, m, y};
    for (const void* q : ptrs) {
        if (!q) return WKV7_ERR_NULL;
        if (!aligned16(q)) return WKV7_ERR_ALIGN;
    }
    wkv7::DdlerpFwdParams p{x, alpha, L, R, beta, m, y, B * T, T, C, (int)D};
    return wkv7::launch_ddlerp_fwd(p, (cudaStream_t)stream);
}

size_t wkv7_ddlerp_fwd_tc_workspace_bytes(int64_t C, int64_t D) {
    if (C <= 0 || D <= 0) return 0;
    return wkv7::ddlerp_fwd_tc_workspace_bytes(C, (int)D);
}

int wkv7_ddlerp_fwd_tc(const void* x, const void* alpha, const void* L, const void* R, const void* beta, void* m, void* y,
                       void* workspace, int64_t B, int64_t T, int64_t C, int64_t D, void* stream) {
    int rc = ddlerp_check(B, T, C, D);
    if (rc) return rc;
    if (B == 0 || T == 0) return WKV7_OK;
    const void* ptrs[] = {x, alpha, L, R, beta, m, y, workspace};
    for (const void* q : ptrs) {
        if (!q) return WKV7_ERR_NULL;
        if (!aligned16(q)) return WKV7_ERR_ALIGN;
    }
    int* status = status_ptr();
    if (!status) return WKV7_ERR_LAUNCH;
    wkv7::DdlerpFwdParams p{x, alpha, L, R, beta, m, y, B * T, T, C, (int)D};
    return wkv7::launch_ddlerp_fwd_tc(p, workspace, status, (cudaStream_t)stream);
}

static int ddlerp_bwd_any(const void* x, const void* alpha, const void* L, const void* R, const void* beta, const void* m,
                          const void* dy0, const void* dy1, const void* dy2, const void* dy3, void* dpre_workspace, void* dx,
                          float* dalpha, float* dL, float* dR, float* dbeta, void* workspace, bool tc, int64_t B, int64_t T, int64_t C,
                          int64_t D, void* stream) {
    int rc = ddlerp_check(B, T, C, D);
    if (rc) return rc;
    if (tc && (!workspace || !aligned16(workspace))) return workspace ? WKV7_ERR_ALIGN : WKV7_ERR_NULL;
    const void* ptrs[] = {x, alpha, L, R, beta, m, dy0, dy1, dy2, dy3, dpre_workspace, dx, dalpha, dL, dR, dbeta};
    for (const void* q : ptrs) {
        if (!q) return WKV7_ERR_NULL;
        if (!aligned16(q)) return WKV7_ERR_ALIGN;
    }
    wkv7::DdlerpBwdParams p{};
    p.x = x; p.alpha = alpha; p.L = L; p.R = R; p.beta = beta; p.m = m;
    p.dy[0] = dy0; p.dy[1] = dy1; p.dy[2] = dy2; p.dy[3] = dy3;
    p.dpre = dpre_workspace; p.dx = dx; p.dalpha = dalpha; p.dL = dL; p.dR = dR; p.dbeta = dbeta;
    p.rows = B * T; p.T = T; p.C = C; p.D = (int)D;
    if (B == 0 || T == 0) {  // parameter gradients of an empty batch are zero
        cudaStream_t s = (cudaStream_t)stream;
        if (cudaMemsetAsync(dalpha, 0, sizeof(float) * C, s) != cudaSuccess || cudaMemsetAsync(dbeta, 0, sizeof(float) * 4 * C, s) != cudaSuccess ||
            cudaMemsetAsync(dR, 0, sizeof(float) * 4 * C * D, s) != cudaSuccess || cudaMemsetAsync(dL, 0, sizeof(float) * 4 * D * C, s) != cudaSuccess)
            return WKV7_ERR_LAUNCH;
        return WKV7_OK;
    }
    if (!tc) return wkv7::launch_ddlerp_bwd(p, (cudaStream_t)stream);
    int* status = status_ptr();
    if (!status) return WKV7_ERR_LAUNCH;
    return wkv7::launch_ddlerp_bwd_tc(p, workspace, status, (cudaStream_t)stream);
}

int wkv7_ddlerp_bwd(const void* x, const void* alpha, const void* L, const void* R, const void* beta, const void* m,
                    const void* dy0, const void* dy1, const void* dy2, const void* dy3, void* dpre_workspace, void* dx,
                    float* dalpha, float* dL, float* dR, float* dbeta, int64_t B, int64_t T, int64_t C, int64_t D,
                    void* stream) {
    return ddlerp_bwd_any(x, alpha, L, R, beta, m, dy0, dy1, dy2, dy3, dpre_workspace, dx, dalpha, dL, dR, dbeta, nullptr, false, B, T, C, D, stream);
}

size_t wkv7_ddlerp_bwd_tc_workspace_bytes(int64_t C, int64_t D) {
    if (C <= 0 || D <= 0) return 0;
    return wkv7::ddlerp_bwd_tc_workspace_bytes(C, (int)D);
}

int wkv7_ddlerp_bwd_tc(const void* x, const void* alpha, const void* L, const void* R, const void* beta, const void* m,
                       const void* dy0, const void* dy1, const void* dy2, const void* dy3, void* dpre_workspace, void* dx,
                       float* dalpha, float* dL, float* dR, float* dbeta, void* workspace, int64_t B, int64_t T, int64_t C, int64_t D,
                       void* stream) {
    return ddlerp_bwd_any(x, alpha, L, R, beta, m, dy0, dy1, dy2, dy3, dpre_workspace, dx, dalpha, dL, dR, dbeta, workspace, true, B, T, C, D, stream);
}

static int loras_check(int64_t B, int64_t T, int64_t C, int64_t D) {
    if (B < 0 || T < 0 || C <= 0 || D <= 0) return WKV7_ERR_SHAPE;
    if (C % 64 != 0) return WKV7_ERR_CHUNK;
    if (D != 16 && D != 32 && D != 64 && D != 128) return WKV7_ERR_SHAPE;
    return WKV7_OK;
}

// row pitches of the rank-D tensors: null = D each
static bool loras_pitches(const int64_t* ld, int64_t D, long long (&out)[4]) {
    for (int i = 0; i < 4; ++i) {
        out[i] = ld ? ld[i] : D;
        if (out[i] < D || out[i] % 8 != 0) return false;
    }
    return true;
}

int wkv7_expand_loras_fwd(const void* w_in, const void* k_in, const void* z_in, const void* a_in, const void* ma_in,
                          const void* mk_in, const void* Wz, const void* Wa, const void* Wma, const void* Wmk,
                          const void* w_bias, const void* a_bias, const void* ma_bias, const void* mk_bias, void* w_out,
                          void* k_out, void* kk_out, void* b_out, int64_t B, int64_t T, int64_t C, int64_t D, void* stream) {
    return wkv7_expand_loras_fwd_ld(w_in, k_in, z_in, a_in, ma_in, mk_in, nullptr, Wz, Wa, Wma, Wmk, w_bias, a_bias, ma_bias, mk_bias,
                                    w_out, k_out, kk_out, b_out, B, T, C, D, stream);
}

int wkv7_expand_loras_fwd_ld(const void* w_in, const void* k_in, const void* z_in, const void* a_in, const void* ma_in,
                             const void* mk_in, const int64_t* ld, const void* Wz, const void* Wa, const void* Wma, const void* Wmk,
                             const void* w_bias, const void* a_bias, const void* ma_bias, const void* mk_bias, void* w_out,
                             void* k_out, void* kk_out, void* b_out, int64_t B, int64_t T, int64_t C, int64_t D, void* stream) {
    int rc = loras_check(B, T, C, D);
    if (rc) return rc;
    if (B == 0 || T == 0) return WKV7_OK;
    const void* ptrs[] = {w_in, k_in, z_in, a_in, ma_in, mk_in, Wz, Wa, Wma, Wmk, w_bias, a_bias, ma_bias, mk_bias, w_out, k_out, kk_out, b_out};
    for (const void* q : ptrs) {
        if (!q) return WKV7_ERR_NULL;
        if (!aligned16(q)) return WKV7_ERR_ALIGN;
    }
    wkv7::LorasParams p{};
    p.w_in = w_in; p.k_in = k_in; p.lin[0] = z_in; p.lin[1] = a_in; p.lin[2] = ma_in; p.lin[3] = mk_in;
    p.W[0] = Wz; p.W[1] = Wa; p.W[2] = Wma; p.W[3] = Wmk;
    p.w_bias = w_bias; p.bias[0] = a_bias; p.bias[1] = ma_bias; p.bias[2] = mk_bias;
    p.w_out = w_out; p.k_out = k_out; p.kk_out = kk_out; p.b_out = b_out;
    p.rows = B * T; p.C = C; p.D = (int)D;
    if (!loras_pitches(ld, D, p.ld)) return WKV7_ERR_ALIGN;
    return wkv7::launch_loras_fwd(p, (cudaStream_t)stream);
}

int64_t wkv7_expand_loras_bwd_workspace_bytes(int64_t B, int64_t T, int64_t C, int64_t D) {
    if (B < 0 || T < 0 || C < 0 || D < 0) return 0;
    return 4 * B * T * (C / 64) * D * 2;
}

int wkv7_expand_loras_bwd(const void* w_in, const void* k_in, const void* z_in, const void* a_in, const void* ma_in,
                          const void* mk_in, const void* Wz, const void* Wa, const void* Wma, const void* Wmk,
                          const void* w_bias, const void* a_bias, const void* ma_bias, const void* mk_bias,
                          const void* dw_out, const void* dk_out, const void* dkk_out, const void* db_out, void* dw_in,
                          void* dk_in, void* dz_in, void* da_in, void* dma_in, void* dmk_in, float* dWz, float* dWa,
                          float* dWma, float* dWmk, float* dw_bias, float* da_bias, float* dma_bias, float* dmk_bias,
                          void* workspace, int64_t B, int64_t T, int64_t C, int64_t D, void* stream) {
    return wkv7_expand_loras_bwd_ld(w_in, k_in, z_in, a_in, ma_in, mk_in, nullptr, Wz, Wa, Wma, Wmk, w_bias, a_bias, ma_bias, mk_bias,
                                    dw_out, dk_out, dkk_out, db_out, dw_in, dk_in, dz_in, da_in, dma_in, dmk_in, nullptr,
                                    dWz, dWa, dWma, dWmk, dw_bias, da_bias, dma_bias, dmk_bias, workspace, B, T, C, D, stream);
}

int wkv7_expand_loras_bwd_ld(const void* w_in, const void* k_in, const void* z_in, const void* a_in, const void* ma_in,
                             const void* mk_in, const int64_t* ld, const void* Wz, const void* Wa, const void* Wma, const void* Wmk,
                             const void* w_bias, const void* a_bias, const void* ma_bias, const void* mk_bias,
                             const void* dw_out, const void* dk_out, const void* dkk_out, const void* db_out, void* dw_in,
                             void* dk_in, void* dz_in, void* da_in, void* dma_in, void* dmk_in, const int64_t* ld_grad,
                             float* dWz, float* dWa, float* dWma, float* dWmk, float* dw_bias, float* da_bias, float* dma_bias,
                             float* dmk_bias, void* workspace, int64_t B, int64_t T, int64_t C, int64_t D, void* stream) {
    int rc = loras_check(B, T, C, D);
    if (rc) return rc;
    const void* ptrs[] = {w_in, k_in, z_in, a_in, ma_in, mk_in, Wz, Wa, Wma, Wmk, w_bias, a_bias, ma_bias, mk_bias,
                          dw_out, dk_out, dkk_out, db_out, dw_in, dk_in, dz_in, da_in, dma_in, dmk_in,
                          dWz, dWa, dWma, dWmk, dw_bias, da_bias, dma_bias, dmk_bias, workspace};
    for (const void* q : ptrs) {
        if (!q) return WKV7_ERR_NULL;
        if (!aligned16(q)) return WKV7_ERR_ALIGN;
    }
    wkv7::LorasParams p{};
    p.w_in = w_in; p.k_in = k_in; p.lin[0] = z_in; p.lin[1] = a_in; p.lin[2] = ma_in; p.lin[3] = mk_in;
    p.W[0] = Wz; p.W[1] = Wa; p.W[2] = Wma; p.W[3] = Wmk;
    p.w_bias = w_bias; p.bias[0] = a_bias; p.bias[1] = ma_bias; p.bias[2] = mk_bias;
    p.dw_out = dw_out; p.dk_out = dk_out; p.dkk_out = dkk_out; p.db_out = db_out;
    p.dw_in = dw_in; p.dk_in = dk_in; p.dlin[0] = dz_in; p.dlin[1] = da_in; p.dlin[2] = dma_in; p.dlin[3] = dmk_in;
    p.dW[0] = dWz; p.dW[1] = dWa; p.dW[2] = dWma; p.dW[3] = dWmk;
    p.dw_bias = dw_bias; p.dbias[0] = da_bias; p.dbias[1] = dma_bias; p.dbias[2] = dmk_bias;
    p.partial = workspace;
    p.rows = B * T; p.C = C; p.D = (int)D;
    if (!loras_pitches(ld, D, p.ld) || !loras_pitches(ld_grad, D, p.ldg)) return WKV7_ERR_ALIGN;
    return wkv7::launch_loras_bwd(p, (cudaStream_t)stream);
}

int wkv7_cast(const void* const* src, void* const* dst, const int64_t* numel, const int* kind, int count, void* stream) {
    if (count < 0 || count > WKV7_CAST_MAX) return WKV7_ERR_SHAPE;
    wkv7::CastParams p{};
    for (int i = 0; i < count; ++i) {
        if (numel[i] < 0 || kind[i] < 0 || kind[i] > 2) return WKV7_ERR_SHAPE;
        if (numel[i] == 0) continue;
        if (!src[i] || !dst[i]) return WKV7_ERR_NULL;
        if (numel[i] % 8 != 0 || !aligned16(src[i]) || !aligned16(dst[i])) return WKV7_ERR_ALIGN;
        p.src[p.count] = src[i]; p.dst[p.count] = dst[i]; p.numel[p.count] = numel[i]; p.kind[p.count] = kind[i];
        ++p.count;
    }
    return p.count ? wkv7::launch_cast(p, (cudaStream_t)stream) : WKV7_OK;
}

}  // extern "C"

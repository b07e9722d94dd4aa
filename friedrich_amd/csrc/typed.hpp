// typed.hpp -- what the operators over 64-, 32- and 16-bit data share: element types, staging of host operands, workspaces that a
// captured stream may keep, and the bracket around their C entry points.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <new>

#include "fr_internal.hpp"

namespace fr {

// the type that sums and states are held in: 64 bits for f64 data, 32 bits for everything narrower
template <typename T>
struct Wide {
    using type = float;
};
template <>
struct Wide<double> {
    using type = double;
};
template <typename T>
using wide_t = typename Wide<T>::type;

__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__hip_bfloat16 v)
{
    unsigned short b;
    __builtin_memcpy(&b, &v, 2);
    return __uint_as_float((unsigned)b << 16);
}

// one rounding, to nearest even, where a result leaves for 16-bit memory
template <typename T>
__device__ __forceinline__ T narrow(wide_t<T> v);
template <>
__device__ __forceinline__ double narrow<double>(double v) { return v; }
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ __hip_bfloat16 narrow<__hip_bfloat16>(float v)
{
    const __bf16 b = (__bf16)v;  // (v_cvt_pk_bf16_f32)
    __hip_bfloat16 r;
    __builtin_memcpy(&r, &b, 2);
    return r;
}

// E neighbouring elements from any address of that element's alignment
template <typename T, int E>
struct __attribute__((packed, aligned(sizeof(T)))) Run {
    T v[E];
};
template <typename T, int E>
__device__ __forceinline__ Run<T, E> load_run(const T* p)
{
    Run<T, E> r;
    __builtin_memcpy(&r, __builtin_assume_aligned(p, sizeof(T)), sizeof(r));
    return r;
}
template <typename T, int E>
__device__ __forceinline__ void store_run(T* p, const Run<T, E>& r)
{
    __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), &r, sizeof(r));
}
inline int64_t dtype_size(int dtype) { return dtype == FR_F64 ? 8 : dtype == FR_F32 ? 4 : 2; }
inline int64_t wide_size(int dtype) { return dtype == FR_F64 ? 8 : 4; }

// the capture that the call's stream is in, 0 if none: there is no allocation, no copy to or from pageable memory and no wait in one
unsigned long long stream_capture(fr_ctx* ctx);

// A workspace for one call.  Eager calls take it from the context's pool and give it back (the pool is stream-ordered).  A captured
// call takes it out of the pool for as long as the context lives: a graph is replayed on any stream, next to other graphs and to eager calls
// of the context, so nobody else may be handed the same bytes.  Only later calls of the same capture on the same stream, which its replays
// run one after the other, use it again.
struct OpWorkspace {
    fr_ctx* ctx;
    void* p = nullptr;
    int kept = -1;  // its place in ctx->captured
    explicit OpWorkspace(fr_ctx* c) : ctx(c) {}
    OpWorkspace(const OpWorkspace&) = delete;
    ~OpWorkspace()
    {
        if (kept >= 0)
            ctx->captured[kept].busy = false;
        else if (p)
            ws_put(ctx, p);
    }
    int get(size_t bytes);
};

// `lines` stretches of `line` contiguous elements of `elem` bytes, `ld` elements apart, made available on the device: device memory in
// place, host memory through a workspace.  The layouts of fr_layout differ only in which axis is contiguous.
struct Operand {
    fr_ctx* ctx;
    char* dev = nullptr;
    int64_t ld = 0;
    explicit Operand(fr_ctx* c) : ctx(c), ws(c) {}
    Operand(const Operand&) = delete;
    // host data that will be written back starts as what the caller's memory holds: places that a kernel leaves alone stay as they are
    int stage(const void* p, int64_t line, int64_t lines, int64_t ld, int64_t elem, const char* name, bool output = false);
    int commit();  // host outputs: copy back (waits)
    template <typename T>
    T* as() const
    {
        return (T*)dev;
    }

private:
    OpWorkspace ws;
    char* host = nullptr;
    int64_t host_ld = 0, line_ = 0, lines_ = 0, elem_ = 0;
};

// 64-bit words that no kernel has written yet, between workgroups that pass results on (not hipMemsetAsync: such nodes of a captured graph
// have given wrong results on replays)
constexpr unsigned long long kUnset = ~0ull;
int launch_unset(fr_ctx* ctx, unsigned long long* p, int64_t n);

// The contiguous axis first: (line, lines) of a rows x cols matrix in a layout
inline int stage_matrix(Operand& o, int layout, const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t elem, const char* name, bool output = false)
{
    return layout == FR_LAYOUT_ROWMAJOR ? o.stage(p, cols, rows, ld, elem, name, output) : o.stage(p, rows, cols, ld, elem, name, output);
}

// The current device is the context's during a call and the caller's again afterwards.
struct DeviceScope {
    int before = -1;
    int enter(fr_ctx* ctx)
    {
        FR_HIP(ctx, hipGetDevice(&before));
        if (before == ctx->device) {
            before = -1;
            return FR_OK;
        }
        FR_HIP(ctx, hipSetDevice(ctx->device));
        return FR_OK;
    }
    ~DeviceScope()
    {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// body of a C entry point: the context's lock, its device, and no exception across the boundary
template <class F>
int op_entry(fr_ctx* ctx, F&& body)
{
    if (!ctx) return FR_INVALID_ARGUMENT;
    try {
        FR_LOCK(ctx);
        DeviceScope dev;
        FR_TRY(dev.enter(ctx));
        FR_TRY(lost_waits(ctx));  // (of an earlier call whose results stayed on the device)
        return body();
    } catch (const std::bad_alloc&) {
        return FR_OUT_OF_MEMORY;
    } catch (...) {
        return FR_HIP_ERROR;
    }
}

}  // namespace fr

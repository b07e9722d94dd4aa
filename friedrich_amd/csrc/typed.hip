// typed.hip -- host side of typed.hpp: operands and workspaces of the operators over 64-, 32- and 16-bit data.
#include "typed.hpp"

namespace fr {

unsigned long long stream_capture(fr_ctx* ctx)
{
    if (!ctx->stream) return 0;  // the null stream cannot be captured
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(ctx->stream, &st, &id) != hipSuccess) {
        (void)hipGetLastError();
        return 0;
    }
    return st == hipStreamCaptureStatusNone ? 0 : id + 1;
}

__global__ __launch_bounds__(256) void unset_kernel(unsigned long long* p, int64_t n)
{
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) p[i] = kUnset;
}

int launch_unset(fr_ctx* ctx, unsigned long long* p, int64_t n)
{
    const int64_t blocks = (n + 255) / 256;
    hipLaunchKernelGGL(unset_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, ctx->ls, p, n);
    FR_HIP(ctx, hipGetLastError());
    return FR_OK;
}

int OpWorkspace::get(size_t bytes)
{
    const unsigned long long id = stream_capture(ctx);
    if (!id) {
        p = ws_get(ctx, bytes);
        return p ? FR_OK : FR_OUT_OF_MEMORY;
    }
    for (size_t i = 0; i < ctx->captured.size(); ++i) {
        CapturedBuf& b = ctx->captured[i];
        if (b.id != id || b.stream != ctx->stream || b.busy || b.cap < bytes) continue;
        b.busy = true;
        p = b.p;
        kept = (int)i;
        return FR_OK;
    }
    DevBuf* best = nullptr;
    for (DevBuf& b : ctx->pool)
        if (b.p && !b.in_use && b.cap >= bytes && (!best || b.cap < best->cap)) best = &b;
    // (kept for good: of about the size asked for, as an eager call takes and leaves one -- ws_get)
    if (!best || best->cap > bytes * 2 + (1u << 20))
        return set_err(ctx, FR_OUT_OF_MEMORY,
                       "a captured call needs a workspace of %zu bytes and cannot allocate it: run the calls once outside the capture before each capture", bytes);
    ctx->captured.push_back({best->p, best->cap, id, ctx->stream, true});
    kept = (int)ctx->captured.size() - 1;
    p = best->p;
    best->in_use = true;
    return FR_OK;
}

int Operand::stage(const void* p, int64_t line, int64_t lines, int64_t ld_, int64_t elem, const char* name, bool output)
{
    if (line < 0 || lines < 0) return set_err(ctx, FR_SHAPE, "%s: negative extent (%lld x %lld)", name, (long long)line, (long long)lines);
    if (line == 0 || lines == 0) return FR_OK;
    if (!p) return set_err(ctx, FR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (lines > 1 && ld_ < line) return set_err(ctx, FR_SHAPE, "%s: leading dimension %lld below %lld", name, (long long)ld_, (long long)line);
    if ((uintptr_t)p % (uintptr_t)elem) return set_err(ctx, FR_INVALID_ARGUMENT, "%s: not aligned to its %lld-byte elements", name, (long long)elem);
    ld = lines > 1 ? ld_ : line;
    hipPointerAttribute_t a;
    const bool known = hipPointerGetAttributes(&a, p) == hipSuccess;
    if (!known) (void)hipGetLastError();  // pageable host memory
    if (known && a.type == hipMemoryTypeDevice) {
        if (a.device != ctx->device) return set_err(ctx, FR_INVALID_ARGUMENT, "%s: lives on device %d, the context on device %d", name, a.device, ctx->device);
        dev = (char*)const_cast<void*>(p);
        return FR_OK;
    }
    if (stream_capture(ctx)) return set_err(ctx, FR_INVALID_ARGUMENT, "%s: host memory in a captured call", name);
    ld = line;
    FR_TRY(ws.get((size_t)(elem * line * lines)));
    dev = (char*)ws.p;
    line_ = line, lines_ = lines, elem_ = elem, host_ld = lines > 1 ? ld_ : line;
    FR_HIP(ctx, hipMemcpy2DAsync(dev, (size_t)(line * elem), p, (size_t)(host_ld * elem), (size_t)(line * elem), (size_t)lines, hipMemcpyHostToDevice, ctx->stream));
    FR_HIP(ctx, hipStreamSynchronize(ctx->stream));  // the caller's memory is free when the call returns
    if (output) host = (char*)const_cast<void*>(p);
    return FR_OK;
}

int Operand::commit()
{
    if (!host) return FR_OK;
    FR_HIP(ctx, hipMemcpy2DAsync(host, (size_t)(host_ld * elem_), dev, (size_t)(line_ * elem_), (size_t)(line_ * elem_), (size_t)lines_, hipMemcpyDeviceToHost, ctx->stream));
    FR_HIP(ctx, hipStreamSynchronize(ctx->stream));
    return lost_waits(ctx);
}

}  // namespace fr

// kk_ops.hip -- the C entries of the operators over an 8-bit cache: checks, the context's device, the launch.
// They enqueue on the caller's stream, allocate nothing and touch nothing of the context but its device.
#include <cstdio>
#include <new>

#include "kk_host.h"
#include "kk_kv.h"

namespace kk {
namespace {

constexpr char kTooLarge[] = "the batch is too large for one launch";

int refuse(char* err, size_t errlen, int code, const std::string& m) {
    if (err && errlen) std::snprintf(err, errlen, "%s", m.c_str());
    return code;
}

int status(char* err, size_t errlen, hipError_t rc) {
    if (rc == hipSuccess) return KK_OK;
    return refuse(err, errlen, rc == hipErrorOutOfMemory ? KK_ERR_OOM : KK_ERR_HIP, hipGetErrorString(rc));
}

// The context's device for one call; the caller's current one afterwards.
struct OnDevice {
    int was = -1;
    hipError_t rc;
    explicit OnDevice(int device) {
        rc = hipGetDevice(&was);
        if (rc == hipSuccess && was != device)
            rc = hipSetDevice(device);
        else
            was = -1;
    }
    ~OnDevice() {
        if (was >= 0) (void)hipSetDevice(was);
    }
};

template <class F>
int entry(const kk_ctx* ctx, char* err, size_t errlen, F&& f) {
    if (!ctx) return refuse(err, errlen, KK_ERR_INVALID, "null context");
    OnDevice on(ctx_device(ctx));
    if (on.rc != hipSuccess) return status(err, errlen, on.rc);
    return status(err, errlen, f());
}

// The messages are std::strings: a failed allocation is a status like any other.
template <class F>
auto no_throw(char* err, size_t errlen, F&& f) -> decltype(f()) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        if (err && errlen) std::snprintf(err, errlen, "host allocation failed");
        return KK_ERR_OOM;
    } catch (...) {
        return KK_ERR_INVALID;
    }
}

bool empty(const kk_kv_batch& b) { return b.n == 0 || b.rows == 0 || b.max_new == 0; }

}  // namespace
}  // namespace kk

using namespace kk;

extern "C" {

int kk_qk_norm_rope(kk_ctx* ctx, const kk_norm_rope* args, void* stream, char* err, size_t errlen) {
    return no_throw(err, errlen, [&] {
        const std::string e = norm_rope_error(args);
        if (!e.empty()) return refuse(err, errlen, KK_ERR_INVALID, e);
        return entry(ctx, err, errlen, [&] {
            if (args->rows == 0 || args->q_heads + args->k_heads == 0) return hipSuccess;
            return launch_norm_rope(*args, ctx_cus(ctx), (hipStream_t)stream);
        });
    });
}

static int kv_copy(bool write, kk_ctx* ctx, const kk_kv_cache* cache, const kk_kv_batch* batch, const kk_kv_rows* rows,
                   void* stream, char* err, size_t errlen) {
    return no_throw(err, errlen, [&] {
        std::string e = kv_batch_error(cache, batch);
        if (e.empty() && !(rows && empty(*batch))) e = kv_rows_error(rows);
        if (!e.empty()) return refuse(err, errlen, KK_ERR_INVALID, e);
        return entry(ctx, err, errlen, [&] {
            if (empty(*batch)) return hipSuccess;
            return (write ? launch_kv_write : launch_kv_read)(*cache, *batch, *rows, (hipStream_t)stream);
        });
    });
}

int kk_kv_write(kk_ctx* ctx, const kk_kv_cache* cache, const kk_kv_batch* batch, const kk_kv_rows* rows, void* stream,
                char* err, size_t errlen) {
    return kv_copy(true, ctx, cache, batch, rows, stream, err, errlen);
}

int kk_kv_read(kk_ctx* ctx, const kk_kv_cache* cache, const kk_kv_batch* batch, const kk_kv_rows* rows, void* stream,
               char* err, size_t errlen) {
    return kv_copy(false, ctx, cache, batch, rows, stream, err, errlen);
}

int64_t kk_kv_attention_workspace(kk_ctx* ctx, const kk_kv_cache* cache, const kk_kv_batch* batch,
                                  const kk_kv_attention_args* args, char* err, size_t errlen) {
    return no_throw(err, errlen, [&]() -> int64_t {
        const std::string e = kv_attention_error(cache, batch, args);
        if (!e.empty()) return refuse(err, errlen, KK_ERR_INVALID, e);
        if (!ctx) return refuse(err, errlen, KK_ERR_INVALID, "null context");
        if (empty(*batch)) return 0;
        const AttnPlan p = attention_plan(*cache, *batch, *args, ctx_cus(ctx));
        if (!attention_fits(p, *batch, args->heads, cache->heads)) return refuse(err, errlen, KK_ERR_INVALID, kTooLarge);
        return p.ws_bytes;
    });
}

int kk_kv_attention(kk_ctx* ctx, const kk_kv_cache* cache, const kk_kv_batch* batch, const kk_kv_attention_args* args,
                    void* stream, char* err, size_t errlen) {
    return no_throw(err, errlen, [&] {
        const std::string e = kv_attention_error(cache, batch, args);
        if (!e.empty()) return refuse(err, errlen, KK_ERR_INVALID, e);
        if (!ctx) return refuse(err, errlen, KK_ERR_INVALID, "null context");
        if (empty(*batch)) return (int)KK_OK;
        const AttnPlan p = attention_plan(*cache, *batch, *args, ctx_cus(ctx));
        if (!attention_fits(p, *batch, args->heads, cache->heads)) return refuse(err, errlen, KK_ERR_INVALID, kTooLarge);
        if (p.ws_bytes && (!args->workspace || args->workspace_bytes < (size_t)p.ws_bytes || (uintptr_t)args->workspace % 16))
            return refuse(err, errlen, KK_ERR_INVALID,
                          "the workspace is null, not 16-byte aligned or smaller than " + std::to_string(p.ws_bytes) + " bytes");
        return entry(ctx, err, errlen, [&] { return launch_kv_attention(*cache, *batch, *args, p, (hipStream_t)stream); });
    });
}

}  // extern "C"

// What the Backend-style entry points (linalg_core::Backend's operators and those beside them)
// share: the error that a check throws, its mapping to lg_core_error, the stream of a call.
#pragma once

#include "lg_internal.h"

namespace lg {

struct TensorErr {
    lg_core_error code;
    std::string message;
};

[[noreturn]] inline void core_fail(lg_core_error code, const std::string& msg) { throw TensorErr{code, msg}; }

// Runs `body` (checks, then launches) with the entry points' error mapping: check failures
// return their code; device failures return UnsupportedDevice with the HIP message.
template <typename F>
lg_core_error run_op(F&& body) {
    try {
        body();
        clear_last_error();
        return LG_CORE_OK;
    } catch (const TensorErr& e) {
        set_last_error(e.message);
        return e.code;
    } catch (const Failure& f) {
        set_last_error(f.message);
        return LG_CORE_UNSUPPORTED_DEVICE;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return LG_CORE_UNSUPPORTED_DEVICE;
    } catch (...) {
        set_last_error("internal error: unknown exception");
        return LG_CORE_UNSUPPORTED_DEVICE;
    }
}

inline hipStream_t device_stream(lg_ctx* ctx, void* stream) {
    if (ctx == nullptr) core_fail(LG_CORE_UNSUPPORTED_DEVICE, "null context");
    set_device(ctx);
    return pick_stream(ctx, stream);
}

template <typename T>
T* dev(const lg_tensor* t) {
    return static_cast<T*>(t->base);
}

}  // namespace lg

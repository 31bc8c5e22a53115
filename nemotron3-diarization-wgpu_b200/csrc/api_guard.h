// The C ABI's exception boundary: every entry point runs its body in guarded(), which
// turns exceptions into n3d_status codes and sets this thread's n3d_last_error().
#pragma once

#include <new>
#include <string>

#include "../../include/n3d.h"
#include "n3d_internal.h"

namespace n3d {

std::string& last_error();  // this thread's message (api.cpp)

template <class F>
n3d_status guarded(F&& f) {
    try {
        f();
        last_error().clear();
        return N3D_OK;
    } catch (const Error& e) {
        last_error() = e.what();
        return (n3d_status)e.status;
    } catch (const std::bad_alloc&) {
        last_error() = "out of host memory";
        return N3D_ERR_GPU;
    } catch (const std::exception& e) {
        last_error() = e.what();
        return N3D_ERR_GPU;
    }
}

inline void arg_check(bool ok, const char* what) {
    if (!ok) throw Error(N3D_ERR_INVALID_ARGUMENT, what);
}

}  // namespace n3d

// How every C entry point reports: the message to the caller's buffer and jc_last_error(), C++
// exceptions caught and turned into errors.
#pragma once
#include <algorithm>
#include <cstring>
#include <exception>
#include <string>
#include <type_traits>

#include "jc_internal.h"

namespace jc {

inline void report(char *err, size_t len, const std::string &msg) {
    jc::set_error(msg);
    if (!err || len == 0) return;
    const size_t n = std::min(msg.size(), len - 1);
    std::memcpy(err, msg.data(), n);
    err[n] = 0;
}

template <typename F>
auto guarded(char *err, size_t len, F &&f) -> decltype(f()) {
    try {
        return f();
    } catch (const std::exception &ex) {
        report(err, len, std::string("julia-cuda: exception: ") + ex.what());
    } catch (...) {
        report(err, len, "julia-cuda: unknown exception");
    }
    // Failure: -1 for the int-returning entry points, NULL for the pointer-returning ones.
    if constexpr (std::is_same_v<decltype(f()), int>)
        return -1;
    else
        return decltype(f())();
}

}  // namespace jc

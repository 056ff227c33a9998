// Text of the last error of a call without a handle, one per host thread.
#pragma once

namespace moe {
constexpr int THREAD_ERROR_BYTES = 512;
inline char* thread_error() {
    static thread_local char text[THREAD_ERROR_BYTES] = "";
    return text;
}
}  // namespace moe

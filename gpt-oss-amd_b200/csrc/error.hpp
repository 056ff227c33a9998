// Text of the last error of the calls without a handle.
//
// The stand-alone operators are called from many threads at once: the text of one that fails belongs to its thread.
// The others (create and the functions around it) may be called in one thread and asked about in another: their text
// is every thread's.  A thread reads the later one of its own and the common one.
#pragma once
#include <cstdio>
#include <mutex>

namespace moe {

constexpr int ERROR_BYTES = 512;

struct ErrorText {
    char text[ERROR_BYTES] = "";
    unsigned long long at = 0;  // failed calls before it
};

struct CommonError {
    std::mutex mutex;
    ErrorText last;
    unsigned long long failed = 0;
};

inline CommonError& common_error() {
    static CommonError c;
    return c;
}

inline ErrorText& thread_error() {
    static thread_local ErrorText e;
    return e;
}

inline void set_thread_error(const char* text) {
    ErrorText& e = thread_error();
    snprintf(e.text, sizeof(e.text), "%s", text);
    CommonError& c = common_error();
    std::lock_guard<std::mutex> lock(c.mutex);
    e.at = ++c.failed;
}

inline void set_common_error(const char* text) {
    CommonError& c = common_error();
    std::lock_guard<std::mutex> lock(c.mutex);
    snprintf(c.last.text, sizeof(c.last.text), "%s", text);
    c.last.at = ++c.failed;
}

// Valid until the thread's next call.
inline const char* last_error() {
    ErrorText& e = thread_error();
    CommonError& c = common_error();
    std::lock_guard<std::mutex> lock(c.mutex);
    if (c.last.at > e.at)
        e = c.last;
    return e.text;
}

}  // namespace moe

// What the translation units of the C ABI share: the thread's error text and
// the library's scratch of a stream. Internal header: not installed.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <string>

namespace ofh {

// Sets ofh_last_error() and returns the code.
int api_error(int code, const std::string& msg);

// Scratch that the library owns, held from acquire() until the call's launches
// are queued: release() then, or the destructor on an error path.
class ScratchLease {
public:
    ScratchLease() = default;
    ScratchLease(const ScratchLease&) = delete;
    ScratchLease& operator=(const ScratchLease&) = delete;
    ~ScratchLease();
    // fits = false, and nothing held: a stream under capture whose buffer is too small.
    int acquire(size_t bytes, hipStream_t stream, bool& fits);
    int release();
    void* ptr = nullptr;

private:
    hipStream_t stream_ = nullptr;
    void* shared_ = nullptr;
    bool locked_ = false;
};

}  // namespace ofh

// The device of an operator's call: checks of its pointers and its stream.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

namespace qwen_hip {

// Makes the device that holds `anchor` current for the rest of the scope.
// Every pointer given is refused unless a kernel on that device can use it
// (std::runtime_error, with `owner` in its message).
class OpDevice {
public:
    OpDevice(const void* anchor, const char* what, const char* owner, hipStream_t stream);
    ~OpDevice();
    OpDevice(const OpDevice&) = delete;
    OpDevice& operator=(const OpDevice&) = delete;
    void check(const void* pointer, const char* what, unsigned alignment = 4) const;

private:
    const char* owner_;
    int device_ = 0, before_ = 0;
};

// An argument of a call. Arrays that are written overlap no others, but for
// the one that is only read whose place they may take, from its start.
struct OpArray {
    const char* name;
    const void* at;
    size_t bytes;
    bool needed, written;
    unsigned alignment = 4;
    const void* in_place_of = nullptr;
};
// Null and overlapping arguments are refused; no device is needed.
void check_arrays(const OpArray* arrays, int count);

// Whether two arrays of `bytes` have nothing in common.
bool apart(const void* a, size_t a_bytes, const void* b, size_t b_bytes);

}  // namespace qwen_hip

// The device of an operator's call: checks of its pointers and its stream.
#include "op_device.hpp"

#include <cstdint>

#include "qwen_common.hpp"

namespace qwen_hip {

namespace {
void hip_check(hipError_t e) {
    if (e != hipSuccess) throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e));
}

// Where a pointer's memory lies, refusing what no kernel can use.
hipPointerAttribute_t attributes(const void* p, const char* what) {
    hipPointerAttribute_t a{};
    if (hipPointerGetAttributes(&a, p) != hipSuccess || a.type == hipMemoryTypeUnregistered) {
        (void)hipGetLastError();
        throw std::runtime_error(std::string("Not device memory: ") + what);
    }
    return a;
}
}  // namespace

OpDevice::OpDevice(const void* anchor, const char* what, const char* owner, hipStream_t stream) : owner_(owner) {
    // The runtime's handles 1 and 2 stand for streams and point to none: asked for the device of 1, it ends the
    // process.
    require(stream != hipStreamLegacy && stream != hipStreamPerThread,
            "The stream must be NULL or a stream that was created");
    device_ = attributes(anchor, what).device;
    hip_check(hipGetDevice(&before_));
    if (stream) {
        hipDevice_t of = 0;
        hip_check(hipStreamGetDevice(stream, &of));
        if (of != device_) throw std::runtime_error(std::string("The stream belongs to another device than ") + owner_);
    }
    if (before_ != device_) hip_check(hipSetDevice(device_));
}

OpDevice::~OpDevice() {
    if (before_ != device_) (void)hipSetDevice(before_);
}

void OpDevice::check(const void* p, const char* what, unsigned alignment) const {
    // (Messages are put together where they are needed: a call has many arguments.)
    if (!p) throw std::runtime_error(std::string("Null argument: ") + what);
    if (reinterpret_cast<uintptr_t>(p) % alignment != 0)
        throw std::runtime_error(std::string("Not aligned to ") + std::to_string(alignment) + " bytes: " + what);
    const hipPointerAttribute_t a = attributes(p, what);
    if (a.type == hipMemoryTypeDevice && a.device != device_)
        throw std::runtime_error(std::string("On another device than ") + owner_ + ": " + what);
}

void check_arrays(const OpArray* arrays, int count) {
    for (int i = 0; i < count; ++i)
        if (!arrays[i].at && arrays[i].needed) throw std::runtime_error(std::string("Null argument: ") + arrays[i].name);
    for (int i = 0; i < count; ++i) {
        const OpArray& a = arrays[i];
        if (!a.written || !a.at) continue;
        for (int j = 0; j < count; ++j) {
            const OpArray& b = arrays[j];
            if (j == i || !b.at || (a.at == b.at && a.in_place_of == b.at && !b.written)) continue;
            if (!apart(a.at, a.bytes, b.at, b.bytes))
                throw std::runtime_error(std::string(a.name) + " overlaps " + b.name);
        }
    }
}

bool apart(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y ? y - x >= a_bytes : x - y >= b_bytes;
}

}  // namespace qwen_hip

// Stands in for the library's runtime where the source of operators on device arrays is compiled for the host, kernels and all, and run
// there (host_hip/hip/hip_runtime.h); contexts are numbers that are not zero.
#include <exception>
#include <functional>
#include <string>

#include "../../include/adhip.h"

namespace {
std::string last;
}

namespace host_hip {
bool last_first = false;
}
extern "C" void host_last_workgroup_first(int yes) { host_hip::last_first = yes; }

namespace adhip {
int context_guarded(adhip_ctx* ctx, const std::function<void()>& f) {
    if (!ctx) return 2;
    try {
        f();
        return 0;
    } catch (const std::exception& e) {
        last = e.what();
    }
    return 2;
}
}  // namespace adhip

extern "C" const char* adhip_last_error(adhip_ctx*) { return last.c_str(); }
extern "C" void* adhip_stream(adhip_ctx*) { return nullptr; }

// 16 bits of a float, to the nearest, ties to even: what the host's compiler calls for the conversion.
extern "C" __bf16 __truncsfbf2(float x) {
    unsigned w = __builtin_bit_cast(unsigned, x);
    if (x == x) w += 0x7fff + (w >> 16 & 1);
    else w |= 1u << 22;
    return __builtin_bit_cast(__bf16, (unsigned short)(w >> 16));
}

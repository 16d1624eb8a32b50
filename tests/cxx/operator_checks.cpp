// What stands in for the runtime where the host side of the operators on device arrays is looked at without a GPU: calls that
// would launch a kernel are noted, contexts are numbers that are not zero.  Linked with csrc/{adamw,gradients,layer_norm,recurrence}.hip,
// compiled for the host alone.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <functional>
#include <string>
#include <vector>

#include "../../include/adhip.h"

namespace {
std::string last;
struct Launch {
    uint32_t x, y, z, threads;
};
std::vector<Launch> launches;
}  // namespace

namespace adhip {
int context_guarded(adhip_ctx* ctx, const std::function<void()>& f) {
    if (!ctx) return 2;
    try {
        f();
        return 0;
    } catch (const std::exception& e) {
        last = e.what();
    } catch (...) {
        last = "unknown error";
    }
    return 2;
}
}  // namespace adhip

extern "C" {
const char* adhip_last_error(adhip_ctx*) { return last.c_str(); }
void* adhip_stream(adhip_ctx*) { return nullptr; }
int adhip_alloc(adhip_ctx*, size_t, void**) { return 2; }
int adhip_free(adhip_ctx*, void*) { return 2; }
int adhip_copy_in(adhip_ctx*, void*, const void*, size_t) { return 2; }
int adhip_copy_out(adhip_ctx*, void*, const void*, size_t) { return 2; }
int adhip_sync(adhip_ctx*) { return 2; }
int adhip_program_buffer(adhip_program*, const char*, void**, const uint64_t**, size_t*) { return 2; }
int adhip_attention_workspace(adhip_ctx*, const adhip_attention_args*, int, size_t*) { return 2; }
int adhip_attention(adhip_ctx*, const adhip_attention_args*, void*) { return 2; }
int adhip_attention_backward(adhip_ctx*, const adhip_attention_args*, void*) { return 2; }
int adhip_rotary(adhip_ctx*, const adhip_rotary_args*, void*) { return 2; }

hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t, hipStream_t) {
    launches.push_back({grid.x, grid.y, grid.z, block.x * block.y * block.z});
    return hipSuccess;
}
// Notes of the launches since the last call, four numbers each; returns how many there were.
int noted_launches(uint32_t* out, int room) {
    const int n = (int)launches.size();
    for (int i = 0; i < n && i < room; ++i) {
        out[4 * i] = launches[i].x, out[4 * i + 1] = launches[i].y, out[4 * i + 2] = launches[i].z, out[4 * i + 3] = launches[i].threads;
    }
    launches.clear();
    return n;
}
// Kernels compiled for the host alone have no device code to register.
void** __hipRegisterFatBinary(const void*) { static void* none; return &none; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}
void __hipRegisterVar(void**, void*, char*, const char*, int, size_t, int, int) {}
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*) { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "an error"; }
}

// What a hand-written kernel's source needs of HIP to be compiled for the host and run there, workgroup by workgroup in the order of
// their numbers, or in the opposite one: on its include path this file stands in for the real one.  The threads of a workgroup are contexts of one thread of the
// host; those of a wavefront go from one exchange between lanes to the next together, and wavefronts from barrier to barrier.
#pragma once
#include <ucontext.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <memory>
#include <vector>

#define __global__
#define __device__
#define __forceinline__ inline
#define __shared__ static  // (one workgroup at a time)
#define __launch_bounds__(...)

typedef void* hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
inline const char* hipGetErrorString(hipError_t) { return "an error"; }

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x = 1, unsigned y = 1, unsigned z = 1) : x(x), y(y), z(z) {}
};
struct alignas(8) float2 {
    float x, y;
};
inline float2 make_float2(float x, float y) { return {x, y}; }
struct alignas(16) float4 {
    float x, y, z, w;
};
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }

inline dim3 threadIdx, blockIdx, blockDim, gridDim;

namespace host_hip {

struct Thread {
    ucontext_t at;
    enum { kRuns, kLanes, kBarrier, kDone } state;
    unsigned turn;  // of the two places that exchanges alternate between
};
inline Thread* current;
inline ucontext_t scheduler;
inline std::vector<Thread> threads;
inline std::vector<std::unique_ptr<char[]>> stacks;
inline std::vector<int> lanes[2];  // what each thread put in
inline const std::function<void()>* body;

inline void leave(decltype(Thread::state) how) {
    current->state = how;
    swapcontext(&current->at, &scheduler);
}
inline void begin() {
    (*body)();
    current->state = Thread::kDone;
}

// What the 64 threads of the caller's wavefront put in.
inline const int* exchange(int mine) {
    const unsigned place = current->turn++ & 1;
    lanes[place][threadIdx.x] = mine;
    leave(Thread::kLanes);
    return &lanes[place][threadIdx.x & ~63u];
}

inline void run_workgroup(unsigned n) {
    constexpr size_t kStack = 1 << 16;
    threads.resize(n);
    for (auto& l : lanes) l.assign(n, 0);
    while (stacks.size() < n) stacks.emplace_back(new char[kStack]);
    for (unsigned i = 0; i < n; ++i) {
        getcontext(&threads[i].at);
        threads[i].at.uc_stack.ss_sp = stacks[i].get();
        threads[i].at.uc_stack.ss_size = kStack;
        threads[i].at.uc_link = &scheduler;
        threads[i].state = Thread::kRuns;
        threads[i].turn = 0;
        makecontext(&threads[i].at, begin, 0);
    }
    for (bool goes_on = true; goes_on;) {
        goes_on = false;
        for (unsigned wave = 0; wave < n; wave += 64)  // each as far as its next barrier
            for (;;) {
                unsigned met[4] = {};
                for (unsigned i = wave; i < wave + 64; ++i) {
                    Thread& t = threads[i];
                    if (t.state == Thread::kRuns || t.state == Thread::kLanes) {
                        current = &t;
                        threadIdx.x = i;
                        t.state = Thread::kRuns;
                        swapcontext(&scheduler, &t.at);
                    }
                    ++met[t.state];
                }
                if (met[Thread::kLanes] && met[Thread::kLanes] != 64) {
                    fprintf(stderr, "an exchange between some lanes of a wavefront\n");
                    abort();
                }
                if (!met[Thread::kLanes]) break;
            }
        unsigned met[4] = {};
        for (Thread& t : threads) ++met[t.state];
        if (met[Thread::kBarrier] && met[Thread::kDone]) {
            fprintf(stderr, "a barrier that some threads do not come to\n");
            abort();
        }
        if (met[Thread::kBarrier]) {
            goes_on = true;
            for (Thread& t : threads) t.state = Thread::kRuns;
        }
    }
}

extern bool last_first;  // the order of workgroups

inline hipError_t run(const std::function<void()>& kernel, dim3 grid, dim3 block) {
    body = &kernel;
    gridDim = grid, blockDim = block;
    for (uint64_t i = 0, n = (uint64_t)grid.x * grid.y; i < n; ++i) {
        const uint64_t at = last_first ? n - 1 - i : i;
        blockIdx = dim3((unsigned)(at % grid.x), (unsigned)(at / grid.x), 0);
        run_workgroup(block.x);
    }
    return hipSuccess;
}

struct Two {
    int v[2];
    int operator[](int i) const { return v[i]; }
};
// Where a lane's value comes from under those controls of the data-parallel primitives that kernels here use.
inline int from_lane(int x, int control) {
    const int* all = exchange(x);
    const int lane = (int)(threadIdx.x & 63);
    if (control < 0x100) return all[(lane & ~3) | (control >> 2 * (lane & 3) & 3)];  // any of four lanes
    if (control == 0x140) return all[lane ^ 15];                                    // sixteen mirrored
    if (control == 0x141) return all[lane ^ 7];                                     // eight mirrored
    fprintf(stderr, "control 0x%x is not known here\n", control);
    abort();
}
inline Two swap_lanes(int x, unsigned off) {
    const int* all = exchange(x);
    return {{all[(threadIdx.x & 63) & ~off], all[(threadIdx.x & 63) | off]}};
}

}  // namespace host_hip

// (in the one place that launches, the kernel and its arguments are in reach)
#define hipLaunchKernel(function, grid, block, at, lds, stream) ((void)at, host_hip::run([&] { kernel(args...); }, grid, block))

inline void __syncthreads() { host_hip::leave(host_hip::Thread::kBarrier); }
inline uint64_t __ballot(bool x) {
    const int* all = host_hip::exchange(x);
    uint64_t r = 0;
    for (int i = 0; i < 64; ++i) r |= (uint64_t)(all[i] != 0) << i;
    return r;
}
inline float __shfl_xor(float x, int off) {
    const int* all = host_hip::exchange(__builtin_bit_cast(int, x));
    return __builtin_bit_cast(float, all[(threadIdx.x & 63) ^ off]);
}
inline double __shfl_xor(double x, int off) {
    const uint64_t w = __builtin_bit_cast(uint64_t, x), low = (unsigned)host_hip::exchange((int)w)[(threadIdx.x & 63) ^ off];
    return __builtin_bit_cast(double, low | (uint64_t)(unsigned)host_hip::exchange((int)(w >> 32))[(threadIdx.x & 63) ^ off] << 32);
}
inline int atomicMin(int* a, int x) { const int was = *a; *a = x < was ? x : was; return was; }
inline int atomicMax(int* a, int x) { const int was = *a; *a = x > was ? x : was; return was; }
template <class T>
inline T min(T a, T b) { return b < a ? b : a; }
template <class T>
inline T max(T a, T b) { return a < b ? b : a; }
inline float __uint_as_float(unsigned x) { return __builtin_bit_cast(float, x); }

#define __builtin_amdgcn_readfirstlane(x) (x)  // asked for what all lanes share
#define __builtin_amdgcn_s_waitcnt(x) ((void)0)
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_rcpf(x) (1.f / (x))
#define __builtin_amdgcn_update_dpp(old, x, control, rows, banks, bound) host_hip::from_lane(x, control)
#define __builtin_amdgcn_permlane16_swap(a, b, ...) host_hip::swap_lanes(a, 16)
#define __builtin_amdgcn_permlane32_swap(a, b, ...) host_hip::swap_lanes(a, 32)

// Host-side checks and small device helpers that the operators on device arrays share.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>
#include <type_traits>

#include "common.hpp"
#include "runtime.hpp"

namespace adhip {

// What a launch holds: fewer than 2^32 threads in each dimension.  Of more, the runtime says nothing and the hardware sees the
// remainder.
inline bool fits_launch(int64_t blocks, unsigned threads) { return blocks <= (int64_t)(0xffffffffu / threads); }

// Queues a kernel; an error is the launch's own, not one that another call of the process has left behind.
template <class... P>
void launch(const char* op, void (*kernel)(P...), dim3 grid, unsigned threads, hipStream_t stream, const std::common_type_t<P>&... args) {
    void* at[] = {(void*)&args...};
    ADHIP_CHECK(fits_launch(grid.x, threads), "%s: %u blocks are too many for a launch", op, grid.x);
    const hipError_t e = hipLaunchKernel((const void*)kernel, grid, dim3(threads), at, 0, stream);
    if (e != hipSuccess) throw Error(strf("%s: the launch failed: %s", op, hipGetErrorString(e)));
}

inline int type_bytes(int type) { return type == ADHIP_BF16 ? 2 : type == ADHIP_E4M3 ? 1 : 4; }
inline const char* type_name(int type) {
    static const char* const names[] = {"f32", "bf16", "int32", "e4m3"};
    return type >= 0 && type < 4 ? names[type] : "unknown";
}

inline std::string array_str(const adhip_array& a) {
    std::string s = std::string(type_name(a.type)) + " [";
    for (int i = 0; i < a.rank && i < 4; ++i) s += (i ? ", " : "") + std::to_string(a.dims[i]);
    return s + "]";
}

// `a` has this type (-1: any) and rank, and extents that are not negative.  Returns how many elements it has.
inline int64_t check_shape(const char* op, const char* name, const adhip_array& a, int type, int rank) {
    ADHIP_CHECK(a.rank == rank, "%s: %s has %d dims, %d are wanted", op, name, (int)a.rank, rank);
    ADHIP_CHECK(type < 0 || a.type == type, "%s: %s is %s, %s is wanted", op, name, type_name(a.type), type_name(type));
    int64_t count = 1;
    for (int i = 0; i < rank; ++i) {
        ADHIP_CHECK(a.dims[i] >= 0, "%s: %s has a negative extent: %s", op, name, array_str(a).c_str());
        ADHIP_CHECK(!__builtin_mul_overflow(count, a.dims[i], &count) && count < (int64_t(1) << 60), "%s: %s is too large: %s", op, name,
                    array_str(a).c_str());
    }
    return count;
}

// The same, and it is given, with a memory extent that fits 2^62 bytes.
inline void check_array(const char* op, const char* name, const adhip_array& a, int type, int rank) {
    const int64_t count = check_shape(op, name, a, type, rank);
    int64_t span = 0;
    for (int i = 0; i < rank; ++i) {
        ADHIP_CHECK(a.strides[i] >= 0, "%s: %s has a negative stride", op, name);
        int64_t far = 0;
        ADHIP_CHECK(!__builtin_mul_overflow(a.dims[i] > 0 ? a.dims[i] - 1 : 0, a.strides[i], &far) && !__builtin_add_overflow(span, far, &span) &&
                        span < (int64_t(1) << 60),
                    "%s: the strides of %s reach too far", op, name);
    }
    ADHIP_CHECK(a.data || count == 0, "%s: %s is missing", op, name);
    ADHIP_CHECK((uintptr_t)a.data % (size_t)type_bytes(a.type) == 0, "%s: %s is not aligned to its type", op, name);
}

inline void check_dims(const char* op, const char* name, const adhip_array& a, std::initializer_list<int64_t> want) {
    int i = 0;
    bool same = a.rank == (int)want.size();
    for (int64_t w : want) same = same && a.dims[i++] == w;
    if (same) return;
    std::string s;
    for (int64_t w : want) s += (s.empty() ? "" : ", ") + std::to_string(w);
    throw Error(strf("%s: %s is %s, [%s] is wanted", op, name, array_str(a).c_str(), s.c_str()));
}

// The last dim is packed (an extent of 1 has no stride to speak of).
inline void check_packed_rows(const char* op, const char* name, const adhip_array& a) {
    const int last = a.rank - 1;
    ADHIP_CHECK(a.strides[last] == 1 || a.dims[last] <= 1, "%s: the last stride of %s is %lld, 1 is wanted", op, name,
                (long long)a.strides[last]);
}

// No two elements of an output share memory: with the dims in the order of their strides, each stride passes what the
// dims below it reach.
inline void check_distinct(const char* op, const char* name, const adhip_array& a) {
    int order[4];
    for (int i = 0; i < a.rank; ++i) {
        if (a.dims[i] == 0) return;
        int j = i;
        for (; j > 0 && a.strides[order[j - 1]] > a.strides[i]; --j) order[j] = order[j - 1];
        order[j] = i;
    }
    int64_t reach = 0;
    for (int i = 0; i < a.rank; ++i) {
        const int d = order[i];
        if (a.dims[d] <= 1) continue;
        ADHIP_CHECK(a.strides[d] > reach, "%s: elements of %s share memory", op, name);
        reach += (a.dims[d] - 1) * a.strides[d];
    }
}

// The largest power of two, at most `most`, that divides an array's address and all its strides but the last (extents of
// one aside), in elements: how many elements a lane may take at once from a multiple of it.
inline int vector_elements(const adhip_array& a, int most) {
    int v = most;
    const int w = type_bytes(a.type);
    while (v > 1 && (uintptr_t)a.data % (size_t)(v * w)) v /= 2;
    for (int i = 0; i + 1 < a.rank; ++i)
        while (v > 1 && a.dims[i] > 1 && a.strides[i] % v) v /= 2;
    return v;
}

// ---- device side ----------------------------------------------------------------------------------------------------

typedef __bf16 bf16;

template <class T, int N>
struct __attribute__((aligned(sizeof(T) * N))) Pack {
    T v[N];
};

}  // namespace adhip

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

// The last cache before memory.  A call whose arrays pass it together leaves nothing there for the next one; written past it, its results
// cost no room for what is still to be read, and the next call finds no lines that have to be written back first.
constexpr int64_t kLastCache = 256 << 20;  // bytes

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

// Whether two arrays of packed rows share memory: whether a row of one and a row of the other are less than a row apart.  The distance of
// rows is a sum over the dims' strides, each times an index (a difference of two, where both arrays have the stride); the search goes
// from the largest stride on and leaves out what the smaller ones cannot make up for, so distinct elements leave it one or two ways at each.
// Where thousands of ways (of arrays that interleave under unlike strides) do not tell, none is found.
class SharedMemory {
    using Wide = __int128;  // (two arrays may reach 2^62 bytes each)
    struct Term {
        Wide stride, least, most;
    } terms[8];
    int n = 0, ways = 1 << 13;
    Wide below, above;  // rows meet at distances between the two

    void add(int64_t stride, int64_t least, int64_t most) {
        if (stride == 0) return;
        int i = 0;
        while (i < n && terms[i].stride > stride) ++i;
        if (i < n && terms[i].stride == stride) {
            terms[i].least += least, terms[i].most += most;
            return;
        }
        for (int j = n++; j > i; --j) terms[j] = terms[j - 1];
        terms[i] = {stride, least, most};
    }
    static Wide reach(const adhip_array& a) {
        int64_t r = a.dims[a.rank - 1];
        for (int d = 0; d + 1 < a.rank; ++d) r += (a.dims[d] - 1) * a.strides[d];
        return r;
    }
    static Wide floor_div(Wide a, Wide b) { return a / b - (a % b < 0); }
    bool meets(int i, Wide at) {
        Wide least = 0, most = 0;
        for (int j = i; j < n; ++j) least += terms[j].least * terms[j].stride, most += terms[j].most * terms[j].stride;
        if (--ways < 0 || at + least >= above || at + most <= below) return false;
        if (i == n) return true;
        const Term t = terms[i];
        least -= t.least * t.stride, most -= t.most * t.stride;
        const Wide from = floor_div(below - at - most, t.stride) + 1, to = -floor_div(at + least - above, t.stride) - 1;
        for (Wide k = from > t.least ? from : t.least; k <= (to < t.most ? to : t.most) && ways > 0; ++k)
            if (meets(i + 1, at + k * t.stride)) return true;
        return false;
    }

public:
    bool found = false;
    SharedMemory(const adhip_array& a, const adhip_array& b) {
        const int64_t aw = type_bytes(a.type), bw = type_bytes(b.type);
        for (const adhip_array* x : {&a, &b})
            for (int d = 0; d < x->rank; ++d)
                if (x->dims[d] == 0) return;
        const Wide at = (Wide)(uintptr_t)b.data - (Wide)(uintptr_t)a.data;
        above = a.dims[a.rank - 1] * aw, below = -(Wide)(b.dims[b.rank - 1] * bw);
        if (at >= reach(a) * aw || -at >= reach(b) * bw) return;  // (as a rule)
        for (int d = 0; d + 1 < b.rank; ++d)
            if (b.dims[d] > 1) add(b.strides[d] * bw, 0, b.dims[d] - 1);
        for (int d = 0; d + 1 < a.rank; ++d)
            if (a.dims[d] > 1) add(a.strides[d] * aw, 1 - a.dims[d], 0);
        found = meets(0, at);
    }
};

// What may be written where it is read, element by element, or apart from it: an input and an output of one shape and type.
inline void check_in_place(const char* op, const char* in_name, const adhip_array& in, const char* out_name, const adhip_array& out) {
    bool same = in.data == out.data;
    for (int d = 0; d < in.rank; ++d) same = same && (in.strides[d] == out.strides[d] || in.dims[d] <= 1);
    ADHIP_CHECK(same || !SharedMemory(in, out).found, "%s: %s and %s share memory, but not element by element", op, out_name, in_name);
}

// Two outputs.
inline void check_apart(const char* op, const char* a_name, const adhip_array& a, const char* b_name, const adhip_array& b) {
    ADHIP_CHECK(!SharedMemory(a, b).found, "%s: %s and %s share memory", op, a_name, b_name);
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

// 16 bytes that begin at any element: global memory takes such accesses, at the cost of one more line where they cross one.
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[N];
};

// 4, 8 and 16 bytes written past the caches, to addresses that are aligned to two.
typedef unsigned Word4 __attribute__((aligned(2)));
typedef unsigned Word8 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned Word16 __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void store_past(Word4* to, unsigned w) { __builtin_nontemporal_store(w, to); }
__device__ __forceinline__ void store_past(Word8* to, Word8 w) { __builtin_nontemporal_store(w, to); }
__device__ __forceinline__ void store_past(Word16* to, Word16 w) { __builtin_nontemporal_store(w, to); }

}  // namespace adhip

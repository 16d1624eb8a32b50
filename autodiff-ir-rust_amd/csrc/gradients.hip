// The norm over all gradients of a step and clipping by it (Pascanu et al. 2013): norm = |grad_scale| sqrt(sum g^2), factor =
// norm <= limit ? 1 : limit / norm, clipped gradients g grad_scale factor.  The norm and the factor stay on the device: the
// clipping pass, or AdamW, reads the factor from there, and no stream waits for the host.
//
// Memory bounds it: one read of every gradient for the norm, and one more read and a write to clip, which cannot begin before
// the norm is known.  Squares are added in 64 bits, whose exponents hold the squares of all f32 numbers and whose sums lose
// nothing that counts; the vector units have the time (three instructions an element).  Each workgroup leaves one partial sum
// and a last workgroup adds them in the order of their numbers, so the same gradients give the same bits.
// 38 M gradients in f32: squares 26 us (5.8 TB/s), norm 4.7, products 46 (6.6 TB/s, a part of them from the last cache).
#include "operators.hpp"

#include <algorithm>
#include <cmath>
#include <vector>

#pragma clang fp contract(off)

namespace adhip {
namespace {

constexpr int kTensors = 128;    // of a launch: their descriptors stay within 4 KiB of kernel arguments
constexpr int kThreads = 256;
constexpr int kChunk = 8192;     // elements of a workgroup
constexpr int kSmall = 1024;     // elements of a wavefront where one workgroup does everything,
constexpr int kSmallChunks = 64; // and how many such chunks there may be
constexpr int64_t kBlocks = 0xffffffffu / kThreads;  // workgroups of a launch: it holds fewer than 2^32 threads

struct GradientLaunch {
    const void* g[kTensors];
    void* out[kTensors];
    int64_t count[kTensors];
    unsigned first[kTensors + 1];                            // the workgroup that begins each tensor
    unsigned bf16s[kTensors / 32];                           // bit i: tensor i is bf16
    int n;
    float grad_scale;
    const float* factor;
    double* partial;  // of the launch's first workgroup
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int off = 32; off; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

// The sum over a workgroup's threads, in the same order every time; thread 0 has it.
template <int THREADS>
__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[THREADS / 64];
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) x += part[i];
    return x;
}

// The tensor that a workgroup belongs to.
__device__ __forceinline__ int tensor_of(const GradientLaunch& a, unsigned block) {
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.first[mid] <= block) lo = mid;
        else hi = mid;
    }
    return lo;
}

// THREADS with consecutive numbers share a chunk, in packs of 16 bytes that begin at any element: the address, which for views of odd sizes in one
// buffer is anything, decides over no bit (38 M in bf16 off an aligned address: clipped in 47 us as aligned, and 61 by single elements).
template <class T, int THREADS>
__device__ __forceinline__ double square_chunk(const T* g, int64_t begin, int64_t end) {
    constexpr int V = 16 / sizeof(T);
    double s[2] = {0, 0};
    int64_t i = begin + (int64_t)(threadIdx.x % THREADS) * V;
    // whole packs, four of them under way
    constexpr int U = 4;
    for (; i + (U - 1) * THREADS * V + V <= end; i += U * THREADS * V) {
        Loose<T, V> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = *(const Loose<T, V>*)(g + i + u * THREADS * V);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const double x = (float)r[u].v[k];
                s[k & 1] = __builtin_fma(x, x, s[k & 1]);
            }
    }
    for (; i < end; i += THREADS * V)
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (i + k < end) {
                const double x = (float)g[i + k];
                s[0] = __builtin_fma(x, x, s[0]);
            }
    return s[0] + s[1];
}

template <int THREADS, int CHUNK>
__device__ __forceinline__ double squares_of(const GradientLaunch& a, unsigned chunk) {
    const int t = tensor_of(a, chunk);
    const int64_t begin = (int64_t)(chunk - a.first[t]) * CHUNK, end = min(begin + CHUNK, a.count[t]);
    return a.bf16s[t >> 5] >> (t & 31) & 1 ? square_chunk<bf16, THREADS>((const bf16*)a.g[t], begin, end)
                                           : square_chunk<float, THREADS>((const float*)a.g[t], begin, end);
}

__global__ __launch_bounds__(kThreads) void gradient_squares_kernel(const GradientLaunch a) {
    const double sum = block_sum<kThreads>(squares_of<kThreads, kChunk>(a, blockIdx.x));
    if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

__device__ __forceinline__ float clip_factor(double norm, double limit) { return norm <= limit ? 1.f : (float)(limit / norm); }

constexpr int kFinish = 1024;

struct Norm {
    double grad_scale, limit;
    float *norm, *factor;
    __device__ __forceinline__ float put(double squares) const {
        const double length = sqrt(squares) * fabs(grad_scale);
        const float f = clip_factor(length, limit);
        if (threadIdx.x == 0) {
            *norm = (float)length;
            if (factor) *factor = f;
        }
        return f;
    }
};

__global__ __launch_bounds__(kFinish) void gradient_norm_kernel(const double* partial, int64_t n, const Norm norm) {
    double s = 0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < n; i += kFinish) s += partial[i];
    norm.put(block_sum<kFinish>(s));
}

// PAST: written past the caches, which hold what is read again instead.
template <class T, int THREADS, bool PAST>
__device__ __forceinline__ void scale_chunk(const T* g, T* out, int64_t begin, int64_t end, float scale) {
    constexpr int V = 16 / sizeof(T);
    int64_t i = begin + (int64_t)(threadIdx.x % THREADS) * V;
    constexpr int U = 4;
    for (; i + (U - 1) * THREADS * V + V <= end; i += U * THREADS * V) {
        Loose<T, V> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = *(const Loose<T, V>*)(g + i + u * THREADS * V);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < V; ++k) r[u].v[k] = (T)((float)r[u].v[k] * scale);
            Word16 w;  // (as one store of 16 bytes)
            __builtin_memcpy(&w, &r[u], sizeof w);
            if (PAST) store_past((Word16*)(out + i + u * THREADS * V), w);
            else *(Word16*)(out + i + u * THREADS * V) = w;
        }
    }
    for (; i < end; i += THREADS * V)
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (i + k < end) out[i + k] = (T)((float)g[i + k] * scale);
}

template <int THREADS, int CHUNK, bool PAST>
__device__ __forceinline__ void scale_of(const GradientLaunch& a, unsigned chunk, float scale) {
    const int t = tensor_of(a, chunk);
    // in place, a scale of one leaves every number as it is
    if (scale == 1.f && a.out[t] == a.g[t]) return;
    const int64_t begin = (int64_t)(chunk - a.first[t]) * CHUNK, end = min(begin + CHUNK, a.count[t]);
    if (a.bf16s[t >> 5] >> (t & 31) & 1) scale_chunk<bf16, THREADS, PAST>((const bf16*)a.g[t], (bf16*)a.out[t], begin, end, scale);
    else scale_chunk<float, THREADS, PAST>((const float*)a.g[t], (float*)a.out[t], begin, end, scale);
}

template <bool PAST>
__global__ __launch_bounds__(kThreads) void gradient_scale_kernel(const GradientLaunch a) {
    scale_of<kThreads, kChunk, PAST>(a, blockIdx.x, a.grad_scale * *a.factor);
}

// Gradients of little more than nothing: norm, factor and, with CLIP, what is made of them in one launch of one workgroup, a chunk a
// wavefront.
template <bool CLIP>
__global__ __launch_bounds__(kFinish) void gradient_small_kernel(const GradientLaunch a, const Norm norm) {
    const unsigned chunks = a.first[a.n], wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    double s = 0;
    for (unsigned i = wave; i < chunks; i += kFinish / 64) s += squares_of<64, kSmall>(a, i);
    const float factor = norm.put(block_sum<kFinish>(s));
    if (CLIP)
        for (unsigned i = wave; i < chunks; i += kFinish / 64) scale_of<64, kSmall, false>(a, i, a.grad_scale * factor);
}

int64_t blocks_of(int64_t count) { return (count + kChunk - 1) / kChunk; }

// Workgroups of all tensors: one partial sum each.
int64_t check_tensors(const char* op, const adhip_gradients_args& g) {
    ADHIP_CHECK(g.n_tensors >= 0 && (g.tensors || g.n_tensors == 0), "%s: no tensors", op);
    int64_t blocks = 0;
    for (int64_t i = 0; i < g.n_tensors; ++i) {
        const adhip_gradient& t = g.tensors[i];
        ADHIP_CHECK(t.type == ADHIP_F32 || t.type == ADHIP_BF16, "%s: gradient %lld is %s, f32 or bf16 is wanted", op, (long long)i, type_name((int)std::min<int64_t>(std::max<int64_t>(t.type, -1), 4)));
        ADHIP_CHECK(t.count >= 0 && t.count < (int64_t(1) << 48), "%s: gradient %lld has %lld elements", op, (long long)i, (long long)t.count);
        blocks += blocks_of(t.count);
        ADHIP_CHECK(blocks < (int64_t(1) << 40), "%s: too many elements", op);
    }
    return blocks;
}

// (a factor that nobody asked for has its place behind the partial sums)
size_t workspace_of(int64_t blocks) { return (size_t)(blocks + 1) * sizeof(double); }

void gradients(const char* op, const adhip_gradients_args& g, bool clip, hipStream_t stream) {
    const int64_t blocks = check_tensors(op, g);
    ADHIP_CHECK(g.limit > 0, "%s: limit %g is not above zero", op, g.limit);
    ADHIP_CHECK(std::isfinite((float)g.grad_scale), "%s: grad_scale must be finite", op);
    ADHIP_CHECK(g.norm && (uintptr_t)g.norm % 4 == 0 && (uintptr_t)g.factor % 4 == 0, "%s: norm is missing, or norm or factor is not aligned to its type", op);
    ADHIP_CHECK(g.workspace && (uintptr_t)g.workspace % 8 == 0 && g.workspace_bytes >= workspace_of(blocks),
                "%s: the workspace has %zu bytes, %zu are wanted, aligned to 8", op, g.workspace ? g.workspace_bytes : (size_t)0, workspace_of(blocks));
    for (int64_t i = 0; i < g.n_tensors; ++i) {
        const adhip_gradient& t = g.tensors[i];
        const size_t w = (size_t)type_bytes((int)t.type);
        ADHIP_CHECK(t.count == 0 || (t.g && (t.out || !clip)), "%s: an array of gradient %lld is missing", op, (long long)i);
        ADHIP_CHECK((uintptr_t)t.g % w == 0 && (!clip || (uintptr_t)t.out % w == 0), "%s: an array of gradient %lld is not aligned to its type", op,
                    (long long)i);
    }
    if (clip) {  // a gradient that is listed twice would be scaled twice, at once; one where another is written may be read too late
        struct Span {
            uintptr_t begin, end;
            int64_t i;
        };
        const auto span = [&](const void* a, int64_t i) {
            return Span{(uintptr_t)a, (uintptr_t)a + (uintptr_t)g.tensors[i].count * type_bytes((int)g.tensors[i].type), i};
        };
        std::vector<Span> outs;
        for (int64_t i = 0; i < g.n_tensors; ++i)
            if (g.tensors[i].count) outs.push_back(span(g.tensors[i].out, i));
        std::sort(outs.begin(), outs.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
        for (size_t k = 1; k < outs.size(); ++k) ADHIP_CHECK(outs[k].begin >= outs[k - 1].end, "%s: two clipped gradients share memory", op);
        for (int64_t i = 0; i < g.n_tensors; ++i) {
            if (g.tensors[i].count == 0) continue;
            const Span in = span(g.tensors[i].g, i);
            // (the first of them that ends behind the gradient's begin; its own, in place, is the only one that it meets)
            const auto out = std::partition_point(outs.begin(), outs.end(), [&](const Span& o) { return o.end <= in.begin; });
            ADHIP_CHECK(out == outs.end() || out->begin >= in.end || (out->i == i && out->begin == in.begin),
                        "%s: gradient %lld lies where another clipped one is written", op, (long long)i);
        }
    }
    double* const partial = (double*)g.workspace;
    float* const factor = g.factor || !clip ? g.factor : (float*)(partial + blocks);
    const Norm norm = {g.grad_scale, g.limit, g.norm, factor};
    // Descriptors of as many tensors as a launch holds, in chunks of `chunk` elements; `flush` launches them.
    auto each_launch = [&](int64_t chunk, auto&& flush) {
        GradientLaunch a = {};
        a.grad_scale = (float)g.grad_scale;
        a.factor = factor;
        a.partial = partial;
        auto done = [&] {
            flush(a);
            a.partial += a.first[a.n];
            a.n = 0;
            a.first[0] = 0;
            for (unsigned& bits : a.bf16s) bits = 0;
        };
        for (int64_t i = 0; i < g.n_tensors; ++i) {
            const adhip_gradient& t = g.tensors[i];
            // (a tensor that passes what a launch holds goes on in the next)
            for (int64_t at = 0; at < t.count;) {
                if (a.n == kTensors || a.first[a.n] == kBlocks) done();
                const int64_t own = std::min<int64_t>((t.count - at + chunk - 1) / chunk, kBlocks - a.first[a.n]), width = type_bytes((int)t.type);
                a.g[a.n] = (const char*)t.g + at * width;
                a.out[a.n] = clip ? (char*)t.out + at * width : nullptr;
                a.count[a.n] = std::min(t.count - at, own * chunk);
                if (t.type == ADHIP_BF16) a.bf16s[a.n >> 5] |= 1u << (a.n & 31);
                at += own * chunk;
                ++a.n;
                a.first[a.n] = a.first[a.n - 1] + (unsigned)own;
            }
        }
        if (a.n) done();
    };
    // One launch where there is little: a call on 65536 elements takes 11 us with one workgroup and 17 with three launches, one on
    // 262144 takes 33 and 17.
    int64_t tensors = 0, small_chunks = 0, bytes = 0;
    for (int64_t i = 0; i < g.n_tensors; ++i) {
        const adhip_gradient& t = g.tensors[i];
        tensors += t.count > 0;
        small_chunks += (t.count + kSmall - 1) / kSmall;
        bytes += t.count * type_bytes((int)t.type) * (t.out == t.g ? 1 : 2);
    }
    if (tensors > 0 && tensors <= kTensors && small_chunks <= kSmallChunks) {
        each_launch(kSmall, [&](const GradientLaunch& a) {
            launch(op, clip ? gradient_small_kernel<true> : gradient_small_kernel<false>, 1, kFinish, stream, a, norm);
        });
        return;
    }
    each_launch(kChunk, [&](const GradientLaunch& a) { launch(op, gradient_squares_kernel, a.first[a.n], kThreads, stream, a); });
    launch(op, gradient_norm_kernel, 1, kFinish, stream, partial, blocks, norm);
    // Where the last cache does not hold gradients and what is made of them, what is written goes past it, and the gradients are still
    // there when they are read again.  38 M in f32: 76 us instead of 91.
    const bool past = bytes > kLastCache;
    if (clip)
        each_launch(kChunk, [&](const GradientLaunch& a) {
            launch(op, past ? gradient_scale_kernel<true> : gradient_scale_kernel<false>, a.first[a.n], kThreads, stream, a);
        });
}

}  // namespace
}  // namespace adhip

extern "C" {

int adhip_gradient_norm_workspace(adhip_ctx* ctx, const adhip_gradients_args* args, size_t* bytes) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args && bytes, "adhip_gradient_norm_workspace: no arguments");
        *bytes = adhip::workspace_of(adhip::check_tensors("adhip_gradient_norm_workspace", *args));
    });
}

int adhip_gradient_norm(adhip_ctx* ctx, const adhip_gradients_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_gradient_norm: no arguments");
        adhip::gradients("adhip_gradient_norm", *args, false, (hipStream_t)stream);
    });
}

int adhip_clip_gradients(adhip_ctx* ctx, const adhip_gradients_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_clip_gradients: no arguments");
        adhip::gradients("adhip_clip_gradients", *args, true, (hipStream_t)stream);
    });
}
}

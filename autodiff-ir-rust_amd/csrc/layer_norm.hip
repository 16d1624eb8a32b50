// Layer norm (Ba et al. 2016), and without the mean RMS norm (Zhang and Sennrich 2019), of the rows of an array, with the
// residual that is added on the way; the backward pass with the sums over rows that are the weights' gradients.
//
// Memory bounds it: a row is read once, stays in the registers of the lanes that share it (16, 64, 256 or 1024 of them, up to 16
// elements each), and its results are written once.  Mean and squared deviations are two sums one after the other over those
// registers, so a mean that is large against the deviations costs no bits.  In the backward pass a lane keeps the same columns of all
// rows that it meets, so the weights' gradients add up in its registers; a workgroup adds its lanes' sums in LDS, and a small second
// kernel the workgroups', always in the same order.
#include "operators.hpp"

#include <algorithm>
#include <cmath>

namespace adhip {
namespace {

constexpr int kElements = 16;      // of a row that a lane holds
constexpr int kGradThreads = 1024;
constexpr int kGradBlocks = 256;   // a compute unit each: more would leave more partial sums of the weights' gradients
constexpr int64_t kMostSize = 1024 * kElements;

struct Place {
    int64_t s[3];  // strides of the dims that number the rows
};

struct NormParams {
    const void *x, *added, *weight, *bias, *out_grad, *total_grad;
    void *total, *out, *x_grad;
    float *stats, *part;
    Place x_at, added_at, total_at, out_at, out_grad_at, total_grad_at, x_grad_at;
    unsigned rows, n1, n2;  // row number (i0 n1 + i1) n2 + i2
    int size, padded;       // padded: of a row of partial sums
    float eps, centered;    // centered: 1 or 0
};

struct RowIndex {
    int64_t i0, i1, i2;
    __device__ __forceinline__ RowIndex(const NormParams& p, unsigned row) {
        if (p.n1 == 1 && p.n2 == 1) {
            i0 = row, i1 = i2 = 0;
        } else {
            const unsigned r = row / p.n2;
            i0 = r / p.n1, i1 = r % p.n1, i2 = row % p.n2;
        }
    }
    __device__ __forceinline__ int64_t at(const Place& p) const { return i0 * p.s[0] + i1 * p.s[1] + i2 * p.s[2]; }
};

// 16 bytes that begin at any element: global memory takes such accesses, at the cost of one more line where they cross one.
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[N];
};

// V elements of a row from e on; zeros behind its end.
template <class T, int V>
__device__ __forceinline__ void load_row(const void* row, int64_t at, int e, int size, float (&f)[V]) {
    const T* x = (const T*)row + at + e;
    if (e + V <= size) {
        const Loose<T, V> r = *(const Loose<T, V>*)x;
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = (float)r.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = e + k < size ? (float)x[k] : 0.f;
    }
}

template <class T, int V>
__device__ __forceinline__ void store_row(void* row, int64_t at, int e, int size, const float (&f)[V]) {
    T* x = (T*)row + at + e;
    if (e + V <= size) {
        Loose<T, V> r;
#pragma unroll
        for (int k = 0; k < V; ++k) r.v[k] = (T)f[k];
        *(Loose<T, V>*)x = r;
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (e + k < size) x[k] = (T)f[k];
    }
}

template <int CTRL>
__device__ __forceinline__ float add_from(float x) {
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// The sum over 16 lanes or the wavefront's 64, in all of them and the same in all of them: partners exchange, so both add the same two.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x) {
    x = add_from<0xb1>(x);   // the other of a pair
    x = add_from<0x4e>(x);   // the other pair of four
    x = add_from<0x141>(x);  // eight lanes mirrored
    x = add_from<0x140>(x);  // sixteen
    if (LANES >= 64) {
        const int i = __builtin_bit_cast(int, x);
        const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
        const int s = __builtin_bit_cast(int, __builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]));
        const auto h = __builtin_amdgcn_permlane32_swap(s, s, false, false);
        x = __builtin_bit_cast(float, (int)h[0]) + __builtin_bit_cast(float, (int)h[1]);
    }
    return x;
}

// Sums of a and b over the lanes of a row.  More than a wavefront meet in LDS, in one of two places by turns: between a
// place's readers and its next writers stands the other place's barrier.
template <int LANES, int THREADS>
struct RowSums {
    static constexpr int kWaves = THREADS / 64, kOfRow = LANES / 64;
    int turn = 0;
    __device__ __forceinline__ void operator()(float& a, float& b) {
        a = lanes_sum<LANES>(a);
        b = lanes_sum<LANES>(b);
        if constexpr (LANES > 64) {
            __shared__ float2 parts[2][kWaves];
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) parts[turn][wave] = make_float2(a, b);
            __syncthreads();
            const int first = wave / kOfRow * kOfRow;
            a = b = 0;
#pragma unroll
            for (int i = 0; i < kOfRow; ++i) {
                const float2 s = parts[turn][first + i];
                a += s.x;
                b += s.y;
            }
            turn ^= 1;
        }
    }
};

template <class T, class W, int LANES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_kernel(const NormParams p) {
    constexpr int kThreads = LANES < 256 ? 256 : LANES, V = 16 / sizeof(T), C = kElements / V;
    const int lane = threadIdx.x % LANES;
    RowSums<LANES, kThreads> sums;
    const float per = 1.f / (float)p.size;
    for (unsigned row = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES; row < p.rows; row += gridDim.x * (kThreads / LANES)) {
        const RowIndex index(p, row);
        float x[C][V];
#pragma unroll
        for (int c = 0; c < C; ++c) load_row<T, V>(p.x, index.at(p.x_at), (c * LANES + lane) * V, p.size, x[c]);
        if (p.added) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int e = (c * LANES + lane) * V;
                float y[V];
                load_row<T, V>(p.added, index.at(p.added_at), e, p.size, y);
                // rounded to the arrays' type as it is kept: what is normed here is what the backward pass reads
#pragma unroll
                for (int k = 0; k < V; ++k) x[c][k] = (float)(T)(x[c][k] + y[k]);
                store_row<T, V>(p.total, index.at(p.total_at), e, p.size, x[c]);
            }
        }
        float sum = 0, none = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) sum += x[c][k];
        float mean = 0;
        if (p.centered != 0.f) {
            sums(sum, none);
            mean = sum * per;
        }
        float squares = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                x[c][k] = (c * LANES + lane) * V + k < p.size ? x[c][k] - mean : 0.f;
                squares = __builtin_fmaf(x[c][k], x[c][k], squares);
            }
        none = 0;
        sums(squares, none);
        const float root = 1.f / sqrtf(squares * per + p.eps);
        if (p.stats && lane == 0) *(float2*)(p.stats + 2 * (int64_t)row) = make_float2(mean, root);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = (c * LANES + lane) * V;
            float w[V];
#pragma unroll
            for (int k = 0; k < V; ++k) x[c][k] *= root;
            if (p.weight) {
                load_row<W, V>(p.weight, 0, e, p.size, w);
#pragma unroll
                for (int k = 0; k < V; ++k) x[c][k] *= w[k];
            }
            if (p.bias) {
                load_row<W, V>(p.bias, 0, e, p.size, w);
#pragma unroll
                for (int k = 0; k < V; ++k) x[c][k] += w[k];
            }
            store_row<T, V>(p.out, index.at(p.out_at), e, p.size, x[c]);
        }
    }
}

// With n the normed row and u = out_grad weight:
//     x_grad = root (u - mean(u) - n mean(u n)) + total_grad      (without the mean of u where the norm takes no mean)
//     weight_grad = sum over rows of out_grad n,  bias_grad = sum over rows of out_grad
template <class T, class W, int LANES, bool SUMS>
__global__ __launch_bounds__(kGradThreads) void norm_backward_kernel(const NormParams p) {
    constexpr int V = 16 / sizeof(T), C = kElements / V, kRows = kGradThreads / LANES;
    const int lane = threadIdx.x % LANES;
    RowSums<LANES, kGradThreads> sums;
    const float per = 1.f / (float)p.size;
    float dw[C][V] = {}, db[C][V] = {};
    // (all lanes of a workgroup go round equally often: they meet at barriers)
    for (unsigned first = blockIdx.x * kRows; first < p.rows; first += gridDim.x * kRows) {
        const unsigned row = first + threadIdx.x / LANES;
        const bool there = row < p.rows;
        const RowIndex index(p, there ? row : 0);
        float n[C][V], u[C][V];
        float mean = 0, root = 0;
        if (there) {
            const float2 s = *(const float2*)(p.stats + 2 * (int64_t)row);
            mean = s.x, root = s.y;
        }
        float sum = 0, along = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = (c * LANES + lane) * V, size = there ? p.size : 0;
            float w[V];
            load_row<T, V>(p.x, index.at(p.x_at), e, size, n[c]);
            load_row<T, V>(p.out_grad, index.at(p.out_grad_at), e, size, u[c]);
            if (p.weight) {
                load_row<W, V>(p.weight, 0, e, p.size, w);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) w[k] = 1.f;
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                n[c][k] = (n[c][k] - mean) * root;
                if (SUMS) {
                    dw[c][k] = __builtin_fmaf(u[c][k], n[c][k], dw[c][k]);
                    db[c][k] += u[c][k];
                }
                u[c][k] *= w[k];
                sum += u[c][k];
                along = __builtin_fmaf(u[c][k], n[c][k], along);
            }
        }
        sums(sum, along);
        sum *= per * p.centered;
        along *= per;
        if (there) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int e = (c * LANES + lane) * V;
#pragma unroll
                for (int k = 0; k < V; ++k) u[c][k] = root * (u[c][k] - sum - n[c][k] * along);
                if (p.total_grad) {
                    float g[V];
                    load_row<T, V>(p.total_grad, index.at(p.total_grad_at), e, p.size, g);
#pragma unroll
                    for (int k = 0; k < V; ++k) u[c][k] += g[k];
                }
                store_row<T, V>(p.x_grad, index.at(p.x_grad_at), e, p.size, u[c]);
            }
        }
    }
    if constexpr (SUMS) {
        // The rows' sums of one workgroup: of a wavefront's groups of 16 lanes by exchange, of wavefronts (or of the sets of them
        // that share rows) pairwise in LDS.  Lane `lane` of the first of them is left with the columns that it had all along.
        if constexpr (LANES == 16) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    for (float* s : {&dw[c][k], &db[c][k]}) {
                        *s += __shfl_xor(*s, 16);
                        *s += __shfl_xor(*s, 32);
                    }
                }
        }
        if constexpr (LANES < kGradThreads) {
            constexpr int kSet = LANES < 64 ? 64 : LANES, kSets = kGradThreads / kSet;
            __shared__ float meet[kSets / 2][kElements][kSet];
            const int set = threadIdx.x / kSet, at = threadIdx.x % kSet;
            for (int half = kSets / 2; half >= 1; half /= 2)
                for (auto* s : {&dw, &db}) {
                    __syncthreads();
                    if (set >= half && set < 2 * half)
#pragma unroll
                        for (int c = 0; c < C; ++c)
#pragma unroll
                            for (int k = 0; k < V; ++k) meet[set - half][c * V + k][at] = (*s)[c][k];
                    __syncthreads();
                    if (set < half)
#pragma unroll
                        for (int c = 0; c < C; ++c)
#pragma unroll
                            for (int k = 0; k < V; ++k) (*s)[c][k] += meet[set][c * V + k][at];
                }
        }
        if (threadIdx.x < LANES)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int e = (c * LANES + lane) * V;
                float* part = p.part + (int64_t)blockIdx.x * 2 * p.padded;
                store_row<float, V>(part, 0, e, p.size, dw[c]);
                store_row<float, V>(part, p.padded, e, p.size, db[c]);
            }
    }
}

// Sums of the workgroups' partial sums: 64 columns a workgroup, 16 of its threads a column and each every 16th part.
__global__ __launch_bounds__(256) void norm_sums_kernel(const float* part, int parts, int size, int padded, void* weight_grad, void* bias_grad,
                                                        bool weight_bf16, bool bias_bf16) {
    const bool bias = blockIdx.y != 0;
    void* out = bias ? bias_grad : weight_grad;
    if (!out) return;
    const int column = blockIdx.x * 64 + (threadIdx.x & 15) * 4, first = threadIdx.x >> 4;
    float4 s = make_float4(0, 0, 0, 0);
    if (column < size) {
        const float* from = part + (bias ? padded : 0) + column;
#pragma unroll 4
        for (int i = first; i < parts; i += 16) {
            const float4 x = *(const float4*)(from + (int64_t)i * 2 * padded);
            s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
        }
    }
    __shared__ float4 meet[256];
    meet[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < 64) {
        const int at = threadIdx.x, col = blockIdx.x * 64 + at;
        float sum = 0;
        for (int i = 0; i < 16; ++i) sum += ((const float*)&meet[i * 16 + at / 4])[at & 3];
        if (col < size) {
            if (bias ? bias_bf16 : weight_bf16) ((bf16*)out)[col] = (bf16)sum;
            else ((float*)out)[col] = sum;
        }
    }
}

// Lanes that share a row.
int lanes_of(int64_t size) { return size <= 16 * kElements ? 16 : size <= 64 * kElements ? 64 : size <= 256 * kElements ? 256 : 1024; }

int padded_of(int64_t size) { return (int)((size + 3) / 4 * 4); }

int64_t grad_blocks(int64_t rows, int64_t size) {
    const int64_t at_once = kGradThreads / lanes_of(size);
    return std::min<int64_t>((rows + at_once - 1) / at_once, kGradBlocks);
}

size_t workspace_of(int64_t rows, int64_t size) { return (size_t)grad_blocks(rows, size) * 2 * (size_t)padded_of(size) * sizeof(float); }

template <class T, class W, bool SUMS>
void launch_backward(const char* op, const NormParams& p, unsigned blocks, hipStream_t stream) {
    const int lanes = lanes_of(p.size);
    launch(op, lanes == 16 ? norm_backward_kernel<T, W, 16, SUMS> : lanes == 64 ? norm_backward_kernel<T, W, 64, SUMS>
               : lanes == 256 ? norm_backward_kernel<T, W, 256, SUMS> : norm_backward_kernel<T, W, 1024, SUMS>, blocks, kGradThreads, stream, p);
}

template <class T, class W>
void launch_norm(const char* op, const NormParams& p, bool backward, bool sums, unsigned blocks, hipStream_t stream) {
    if (backward) {
        if (sums) launch_backward<T, W, true>(op, p, blocks, stream);
        else launch_backward<T, W, false>(op, p, blocks, stream);
        return;
    }
    const int lanes = lanes_of(p.size), threads = std::max(256, lanes);
    const int64_t at_once = threads / lanes;
    // (more rows than a launch holds go round)
    const int64_t all = std::min<int64_t>((p.rows + at_once - 1) / at_once, 0xffffffffu / threads);
    launch(op, lanes == 16 ? norm_kernel<T, W, 16> : lanes == 64 ? norm_kernel<T, W, 64> : lanes == 256 ? norm_kernel<T, W, 256> : norm_kernel<T, W, 1024>,
           (unsigned)all, threads, stream, p);
}

struct Named {
    const char* name;
    const adhip_array* a;
    Place* at;
    bool output;
};

// The rows of x: of an array of 2 to 4 dims whose last one is normed.
int64_t check_rows(const char* op, const adhip_array& x) {
    ADHIP_CHECK(x.type == ADHIP_F32 || x.type == ADHIP_BF16, "%s: x is %s, f32 or bf16 is wanted", op, type_name(x.type));
    ADHIP_CHECK(x.rank >= 2 && x.rank <= 4, "%s: x has %d dims, 2 to 4 are wanted", op, (int)x.rank);
    const int64_t count = check_shape(op, "x", x, x.type, x.rank), size = x.dims[x.rank - 1];
    ADHIP_CHECK(size >= 1 && size <= kMostSize, "%s: rows of %lld elements, 1 to %lld are wanted", op, (long long)size, (long long)kMostSize);
    const int64_t rows = count / size;
    ADHIP_CHECK(rows < (int64_t(1) << 31), "%s: %lld rows are too many for one call", op, (long long)rows);
    return rows;
}

void check_vector(const char* op, const char* name, const adhip_array& a, int64_t size, bool output) {
    ADHIP_CHECK(a.type == ADHIP_F32 || a.type == ADHIP_BF16, "%s: %s is %s, f32 or bf16 is wanted", op, name, type_name(a.type));
    check_array(op, name, a, a.type, 1);
    check_dims(op, name, a, {size});
    check_packed_rows(op, name, a);
}

void layer_norm(const char* op, const adhip_layer_norm_args& g, bool backward, hipStream_t stream) {
    const int64_t rows = check_rows(op, g.x), size = g.x.dims[g.x.rank - 1];
    const int lead = g.x.rank - 1;
    NormParams p = {};
    const bool adds = !backward && (g.added.data || g.total.data);
    Named arrays[4];
    int n = 0;
    arrays[n++] = {"x", &g.x, &p.x_at, false};
    if (backward) {
        arrays[n++] = {"out_grad", &g.out_grad, &p.out_grad_at, false};
        if (g.total_grad.data) arrays[n++] = {"total_grad", &g.total_grad, &p.total_grad_at, false};
        arrays[n++] = {"x_grad", &g.x_grad, &p.x_grad_at, true};
    } else {
        if (adds) arrays[n++] = {"added", &g.added, &p.added_at, false}, arrays[n++] = {"total", &g.total, &p.total_at, true};
        arrays[n++] = {"out", &g.out, &p.out_at, true};
    }
    for (int i = 0; i < n; ++i) {
        const adhip_array& a = *arrays[i].a;
        check_array(op, arrays[i].name, a, g.x.type, g.x.rank);
        for (int d = 0; d <= lead; ++d)
            ADHIP_CHECK(a.dims[d] == g.x.dims[d], "%s: %s is %s, the shape of x %s is wanted", op, arrays[i].name, array_str(a).c_str(), array_str(g.x).c_str());
        check_packed_rows(op, arrays[i].name, a);
        if (arrays[i].output) check_distinct(op, arrays[i].name, a);
    }
    // weights: of x's type or f32, both alike
    const int w_type = g.weight.data ? g.weight.type : g.bias.data && !backward ? g.bias.type : ADHIP_F32;
    if (g.weight.data) check_vector(op, "weight", g.weight, size, false);
    if (g.bias.data && !backward) check_vector(op, "bias", g.bias, size, false);
    ADHIP_CHECK(w_type == ADHIP_F32 || w_type == g.x.type, "%s: weight and bias are %s, f32 or the type of x is wanted", op, type_name(w_type));
    ADHIP_CHECK(backward || !g.weight.data || !g.bias.data || g.weight.type == g.bias.type, "%s: weight is %s and bias %s, one type is wanted", op,
                type_name(g.weight.type), type_name(g.bias.type));
    ADHIP_CHECK((float)g.eps > 0 && std::isfinite((float)g.eps), "%s: eps %g is not above zero", op, g.eps);
    // statistics: packed pairs
    if (backward || g.stats.data) {
        check_array(op, "stats", g.stats, ADHIP_F32, g.x.rank);
        int64_t packed = 2;
        bool fits = g.stats.dims[lead] == 2 && (g.stats.strides[lead] == 1);
        for (int d = lead - 1; d >= 0; packed *= g.x.dims[d--])
            fits = fits && g.stats.dims[d] == g.x.dims[d] && (g.stats.strides[d] == packed || g.stats.dims[d] <= 1 || rows == 0);
        ADHIP_CHECK(fits, "%s: stats is %s, two packed numbers for each row of x are wanted", op, array_str(g.stats).c_str());
        ADHIP_CHECK((uintptr_t)g.stats.data % 8 == 0, "%s: stats is not aligned to 8 bytes", op);
    }
    const bool sums = backward && (g.weight_grad.data || g.bias_grad.data);
    if (backward) {
        if (g.weight_grad.data) check_vector(op, "weight_grad", g.weight_grad, size, true);
        if (g.bias_grad.data) check_vector(op, "bias_grad", g.bias_grad, size, true);
        ADHIP_CHECK(!sums || rows == 0 || (g.workspace && (uintptr_t)g.workspace % 16 == 0 && g.workspace_bytes >= workspace_of(rows, size)),
                    "%s: the workspace has %zu bytes, %zu are wanted, aligned to 16", op, g.workspace ? g.workspace_bytes : (size_t)0, workspace_of(rows, size));
    }
    p.rows = (unsigned)rows;
    p.size = (int)size;
    p.padded = padded_of(size);
    p.eps = (float)g.eps;
    p.centered = g.centered ? 1.f : 0.f;
    p.x = g.x.data;
    p.weight = g.weight.data;
    p.stats = (float*)g.stats.data;
    if (backward) {
        p.out_grad = g.out_grad.data;
        p.total_grad = g.total_grad.data;
        p.x_grad = g.x_grad.data;
        p.part = (float*)g.workspace;
    } else {
        p.bias = g.bias.data;
        p.added = adds ? g.added.data : nullptr;
        p.total = g.total.data;
        p.out = g.out.data;
    }
    // The dims that number the rows, from the last one on: two are one where every array's strides allow it.
    int64_t dims[3] = {1, 1, 1}, used = 0;
    for (int d = lead - 1; d >= 0; --d) {
        bool joins = used > 0;
        for (int i = 0; i < n && joins; ++i) joins = arrays[i].a->strides[d] == arrays[i].at->s[used - 1] * dims[used - 1];
        if (g.x.dims[d] == 1 && used > 0) continue;
        if (joins) {
            dims[used - 1] *= g.x.dims[d];
            continue;
        }
        dims[used] = g.x.dims[d];
        for (int i = 0; i < n; ++i) arrays[i].at->s[used] = arrays[i].a->strides[d];
        ++used;
    }
    // (found from the last dim on; numbered from the first)
    for (int i = 0; i < n; ++i) {
        const Place found = *arrays[i].at;
        for (int d = 0; d < 3; ++d) arrays[i].at->s[d] = d < used ? found.s[used - 1 - d] : 0;
    }
    p.n1 = used >= 2 ? (unsigned)dims[used - 2] : 1;
    p.n2 = used >= 3 ? (unsigned)dims[used - 3] : 1;

    if (rows > 0) {
        const unsigned blocks = (unsigned)grad_blocks(rows, size);
        if (g.x.type == ADHIP_F32) launch_norm<float, float>(op, p, backward, sums, blocks, stream);
        else if (w_type == ADHIP_F32) launch_norm<bf16, float>(op, p, backward, sums, blocks, stream);
        else launch_norm<bf16, bf16>(op, p, backward, sums, blocks, stream);
    }
    if (sums)
        launch(op, norm_sums_kernel, dim3((unsigned)((size + 63) / 64), 2), 256, stream, (const float*)g.workspace, rows > 0 ? (int)grad_blocks(rows, size) : 0,
               (int)size, p.padded, g.weight_grad.data, g.bias_grad.data, g.weight_grad.type == ADHIP_BF16, g.bias_grad.type == ADHIP_BF16);
}

}  // namespace
}  // namespace adhip

extern "C" {

int adhip_layer_norm_workspace(adhip_ctx* ctx, const adhip_layer_norm_args* args, size_t* bytes) {
    return adhip::context_guarded(ctx, [&] {
        const char* op = "adhip_layer_norm_workspace";
        ADHIP_CHECK(args && bytes, "%s: no arguments", op);
        *bytes = adhip::workspace_of(adhip::check_rows(op, args->x), args->x.dims[args->x.rank - 1]);
    });
}

int adhip_layer_norm(adhip_ctx* ctx, const adhip_layer_norm_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_layer_norm: no arguments");
        adhip::layer_norm("adhip_layer_norm", *args, false, (hipStream_t)stream);
    });
}

int adhip_layer_norm_backward(adhip_ctx* ctx, const adhip_layer_norm_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_layer_norm_backward: no arguments");
        adhip::layer_norm("adhip_layer_norm_backward", *args, true, (hipStream_t)stream);
    });
}
}

// Layer norm (Ba et al. 2016), and without the mean RMS norm (Zhang and Sennrich 2019), of the rows of an array, with the
// residual that is added on the way; the backward pass with the sums over rows that are the weights' gradients.
//
// Memory bounds it: a row is read once, stays in the registers of the lanes that share it (16 of them, or 1 to 16 whole wavefronts, up to 16
// elements each), and its results are written once.  Mean and squared deviations are two sums one after the other over those
// registers, so a mean that is large against the deviations costs them its own rounding alone.  In the backward pass a lane keeps the same columns of all
// rows that it meets, so the weights' gradients add up in its registers; a workgroup adds its lanes' sums in LDS, and a small second
// kernel the workgroups', always in the same order.
// 16384 rows of 4096 in bf16 with a residual: forward 92 us (5.9 TB/s), backward 107 (5.0) and 5 for the last sums; 131072 rows of 128: 15, 19
// and 4; 3001 rows of 1023 in f32 with a residual: 14.5, 15.7 and 3.8, and 10.8 and 14.6 from the last cache.  Results past the caches gain nothing here.
#include "operators.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace adhip {
namespace {

constexpr int kElements = 16;          // of a row that a lane holds at most
constexpr int kThreads = 256;          // of a workgroup that rows of one wavefront and less share
constexpr int kWaves = 16;             // of a row at most, and of a workgroup of the backward pass
constexpr int kGradBlocks = 256;       // a compute unit each: twice as many leave twice the partial sums (202 us become 208)
constexpr int64_t kMostSize = kWaves * 64 * kElements;

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
    int waves, groups;      // wavefronts that share a row, and rows that a workgroup has at once
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

// Where a pack of V elements that begins at `at` lies.  In rows that do not fill their lanes (FULL) one that would pass the end is moved
// back to it: its first `skip` elements belong to another lane, all V to a lane behind the end.  So every lane makes the same loads, with
// no branch between them, and rows of at least V elements are wanted.
template <int V, bool FULL>
struct Spot {
    int e, skip;
    __device__ __forceinline__ Spot(int at, int size) : e(FULL ? at : min(at, size - V)), skip(FULL ? 0 : at - e) {}
    __device__ __forceinline__ bool has(int k) const { return FULL || k >= skip; }
};

template <class T, int V, bool FULL>
__device__ __forceinline__ void load_row(const void* row, int64_t at, const Spot<V, FULL>& spot, float (&f)[V]) {
    const Loose<T, V> r = *(const Loose<T, V>*)((const T*)row + at + spot.e);
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = spot.has(k) ? (float)r.v[k] : 0.f;
}

template <class T, int V, bool FULL>
__device__ __forceinline__ void store_row(void* row, int64_t at, const Spot<V, FULL>& spot, const float (&f)[V]) {
    T* x = (T*)row + at + spot.e;
    if (FULL || spot.skip == 0) {
        Loose<T, V> r;
#pragma unroll
        for (int k = 0; k < V; ++k) r.v[k] = (T)f[k];
        if constexpr (V == 1) {
            *(Loose<T, V>*)x = r;
        } else {  // (as one store of 16 bytes)
            Word16 w;
            static_assert(sizeof r == sizeof w, "a lane's pack");
            __builtin_memcpy(&w, &r, sizeof w);
            *(Word16*)x = w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (spot.has(k)) x[k] = (T)f[k];
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

// The lanes of a row: 16 of a wavefront, or all of 1 to 16 wavefronts.
template <int LANES>
struct Team {
    int waves, wave, group, lane;  // lane: of the row's
    int turn = 0;
    __device__ __forceinline__ Team(const NormParams& p) {
        waves = p.waves;
        wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        if (LANES == 64) {
            group = waves == 1 ? wave : wave / waves;
            lane = (wave - group * waves) * 64 + (threadIdx.x & 63);
        } else {
            group = threadIdx.x / LANES;
            lane = threadIdx.x % LANES;
        }
    }
    __device__ __forceinline__ int lanes() const { return LANES == 64 ? waves * 64 : LANES; }
    // Sums of a and b over the row.  Those of several wavefronts meet in LDS, in one of two places by turns: between a place's
    // readers and its next writers stands the other place's barrier.
    __device__ __forceinline__ void sum(float& a, float& b) {
        a = lanes_sum<LANES>(a);
        b = lanes_sum<LANES>(b);
        if (LANES < 64 || waves == 1) return;
        __shared__ float2 parts[2][kWaves];
        if ((threadIdx.x & 63) == 0) parts[turn][wave] = make_float2(a, b);
        __syncthreads();
        a = b = 0;
        for (int i = 0; i < waves; ++i) {
            const float2 s = parts[turn][group * waves + i];
            a += s.x;
            b += s.y;
        }
        turn ^= 1;
    }
};

// A workgroup takes several rows one after the other: the next one, whose loads no branch divides, is asked for as soon as this one is in
// other registers, and weight and bias stay in registers.
template <class T, class W, int V, int LANES, int C, bool FULL, bool ADDS>
__global__ __launch_bounds__(LANES == 64 ? kWaves * 64 : kThreads) void norm_kernel(const NormParams p) {
    Team<LANES> team(p);
    const int lanes = team.lanes();
    const float per = 1.f / (float)p.size;
    const auto spot = [&](int c) { return Spot<V, FULL>((c * lanes + team.lane) * V, p.size); };
    struct Row {
        Loose<T, V> x[C], added[ADDS ? C : 1];
    } raw;
    const auto ask = [&](unsigned row) {
        const RowIndex index(p, row);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            raw.x[c] = *(const Loose<T, V>*)((const T*)p.x + index.at(p.x_at) + spot(c).e);
            if (ADDS) raw.added[c] = *(const Loose<T, V>*)((const T*)p.added + index.at(p.added_at) + spot(c).e);
        }
    };
    const unsigned step = gridDim.x * p.groups;
    ask(min(blockIdx.x * p.groups + team.group, p.rows - 1));
    Loose<W, V> weight[C], bias[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (p.weight) weight[c] = *(const Loose<W, V>*)((const W*)p.weight + spot(c).e);
        if (p.bias) bias[c] = *(const Loose<W, V>*)((const W*)p.bias + spot(c).e);
    }
    // (all lanes of a workgroup go round equally often: they meet at barriers)
    for (unsigned first = blockIdx.x * p.groups; first < p.rows; first += step) {
        const unsigned row = min(first + team.group, p.rows - 1);
        const bool there = first + team.group < p.rows;  // (a row too many reads the last one, and writes nothing)
        const RowIndex index(p, row);
        float x[C][V], added[ADDS ? C : 1][V];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                x[c][k] = spot(c).has(k) ? (float)raw.x[c].v[k] : 0.f;
                if (ADDS) added[c][k] = spot(c).has(k) ? (float)raw.added[c].v[k] : 0.f;
            }
        ask(min(first + step + team.group, p.rows - 1));
        if (ADDS) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                // rounded to the arrays' type as it is kept: what is normed here is what the backward pass reads
#pragma unroll
                for (int k = 0; k < V; ++k) x[c][k] = (float)(T)(x[c][k] + added[c][k]);
                if (there) store_row<T>(p.total, index.at(p.total_at), spot(c), x[c]);
            }
        }
        float sum = 0, none = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) sum += x[c][k];
        float mean = 0;
        if (p.centered != 0.f) {
            team.sum(sum, none);
            mean = sum * per;
        }
        float squares = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                x[c][k] = spot(c).has(k) ? x[c][k] - mean : 0.f;
                squares = __builtin_fmaf(x[c][k], x[c][k], squares);
            }
        none = 0;
        team.sum(squares, none);
        const float root = 1.f / sqrtf(squares * per + p.eps);
        if (!there) continue;
        if (p.stats && team.lane == 0) *(float2*)(p.stats + 2 * (int64_t)row) = make_float2(mean, root);
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int k = 0; k < V; ++k) x[c][k] *= root;
            if (p.weight)
#pragma unroll
                for (int k = 0; k < V; ++k) x[c][k] *= (float)weight[c].v[k];
            if (p.bias)
#pragma unroll
                for (int k = 0; k < V; ++k) x[c][k] += (float)bias[c].v[k];
            store_row<T>(p.out, index.at(p.out_at), spot(c), x[c]);
        }
    }
}

// With n the normed row and u = out_grad weight:
//     x_grad = root (u - mean(u) - n mean(u n)) + total_grad      (without the mean of u where the norm takes no mean)
//     weight_grad = sum over rows of out_grad n,  bias_grad = sum over rows of out_grad
// The next row is asked for as soon as this one is in other registers (AHEAD); loads without a branch are loads that the compiler can
// count, so it waits for those of this row alone.
template <class T, class W, int V, int LANES, int C, bool FULL, bool SUMS, bool ADDS>
__global__ __launch_bounds__(kWaves * 64) void norm_backward_kernel(const NormParams p) {
    Team<LANES> team(p);
    const int lanes = team.lanes();
    const float per = 1.f / (float)p.size;
    float dw[C][V] = {}, db[C][V] = {};
    struct Row {
        Loose<T, V> x[C], d[C], more[ADDS ? C : 1];
        float2 stats;
    } raw;
    const auto spot = [&](int c) { return Spot<V, FULL>((c * lanes + team.lane) * V, p.size); };
    const auto ask = [&](Row& r, unsigned row) {
        const RowIndex index(p, row);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            r.x[c] = *(const Loose<T, V>*)((const T*)p.x + index.at(p.x_at) + spot(c).e);
            r.d[c] = *(const Loose<T, V>*)((const T*)p.out_grad + index.at(p.out_grad_at) + spot(c).e);
            if (ADDS) r.more[c] = *(const Loose<T, V>*)((const T*)p.total_grad + index.at(p.total_grad_at) + spot(c).e);
        }
        r.stats = *(const float2*)(p.stats + 2 * (int64_t)row);
    };
    const unsigned step = gridDim.x * p.groups;
    constexpr bool AHEAD = FULL || C * V <= 8;  // (of others the registers do not hold two rows; 12001 of 1030 in f32: 62 us, and 73 without)
    if (AHEAD) ask(raw, min(blockIdx.x * p.groups + team.group, p.rows - 1));
    // (all lanes of a workgroup go round equally often: they meet at barriers)
    for (unsigned first = blockIdx.x * p.groups; first < p.rows; first += step) {
        const unsigned row = first + team.group;
        const bool there = row < p.rows;
        const RowIndex index(p, there ? row : 0);
        float n[C][V], u[C][V], more[ADDS ? C : 1][V], w[C][V];
        if (!AHEAD) ask(raw, min(row, p.rows - 1));
        // (a row that is not there read the last one, or what x_grad put in its place, and must not show in the sums)
        const float mean = there ? raw.stats.x : 0.f, root = there ? raw.stats.y : 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                // what does not count has n = 0, whatever mean and root are
                const bool counts = there && spot(c).has(k);
                n[c][k] = counts ? (float)raw.x[c].v[k] : mean;
                u[c][k] = counts ? (float)raw.d[c].v[k] : 0.f;
                if (ADDS) more[c][k] = (float)raw.more[c].v[k];
            }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (p.weight) {
                load_row<W>(p.weight, 0, spot(c), w[c]);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) w[c][k] = 1.f;
            }
        }
        if (AHEAD) ask(raw, min(row + step, p.rows - 1));
        float sum = 0, along = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                n[c][k] = (n[c][k] - mean) * root;
                if (SUMS) {
                    dw[c][k] = __builtin_fmaf(u[c][k], n[c][k], dw[c][k]);
                    db[c][k] += u[c][k];
                }
                u[c][k] *= w[c][k];
                sum += u[c][k];
                along = __builtin_fmaf(u[c][k], n[c][k], along);
            }
        team.sum(sum, along);
        sum *= per * p.centered;
        along *= per;
        if (there) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
#pragma unroll
                for (int k = 0; k < V; ++k) u[c][k] = root * (u[c][k] - sum - n[c][k] * along);
                if (ADDS)
#pragma unroll
                    for (int k = 0; k < V; ++k) u[c][k] += more[c][k];
                store_row<T>(p.x_grad, index.at(p.x_grad_at), spot(c), u[c]);
            }
        }
    }
    if constexpr (SUMS) {
        // The sums of a workgroup: those of a wavefront's groups of 16 lanes by exchange, then all that have the same columns in LDS,
        // one after the other; all columns at once, behind one barrier (3001 rows of 1023 in f32, both passes: 35 us; a pack's columns at a time 38).
        __shared__ float meet[2 * C * kWaves * 64 * V];
        const int across = LANES == 64 ? lanes * V : LANES * V, rows = LANES == 64 ? p.groups : kWaves;
        const int mine = LANES == 64 ? team.group : team.wave;
        float* const part = p.part + (int64_t)blockIdx.x * 2 * p.padded;
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float s[V];
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    s[k] = which ? db[c][k] : dw[c][k];
                    if (LANES == 16) {
                        s[k] += __shfl_xor(s[k], 16);
                        s[k] += __shfl_xor(s[k], 32);
                    }
                }
                if (LANES == 64 || (threadIdx.x & 63) < LANES)
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        if (spot(c).has(k)) meet[(mine * 2 + which) * C * across + spot(c).e + k] = s[k];
            }
        __syncthreads();
        const int columns = C * across;
        for (int which = 0; which < 2; ++which)
            for (int i = threadIdx.x; i < columns; i += blockDim.x) {
                float sum = 0;
                for (int r = 0; r < rows; ++r) sum += meet[(r * 2 + which) * columns + i];
                if (i < p.size) part[which * p.padded + i] = sum;
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

// How rows are shared out: 16 lanes each, or 1 to 16 wavefronts; packs of 16 bytes a lane; whether rows fill their lanes.
struct Share {
    int lanes, packs, waves, groups, grad_groups;
    bool full, narrow;  // narrow: rows shorter than a pack, an element a lane
    Share(int type, int64_t size) {
        const int v = 16 / type_bytes(type);
        narrow = size < v;
        // One pack where the lanes hold a row so, two otherwise, and four of f32 where 16 wavefronts of two do not.  With fewer elements a lane
        // more rows are under way: 30001 rows of 250 in f32, both passes: 55 us, and 71 by 16 lanes of four packs; 32072 rows of 500 in bf16:
        // 17, and 22 with two.  With one pack a lane, more wavefronts meet in longer rows: 20001 rows of 3001 in bf16: 79 us, and 59 with two.
        lanes = size <= 16 * 2 * v ? 16 : 64;
        packs = size <= lanes * v ? 1 : size <= kWaves * 64 * 2 * v ? 2 : 4;
        full = false;
        // Two packs a lane, or one, that rows fill exactly.  Of bf16 rather one: two, and a residual's gradient, pass the registers (16384 rows
        // of 4096, both passes: 202 us with one, 242 with two).  Of f32 rather two, which halve the wavefronts that have to meet (8192
        // rows: 206 with two, 226 with one).
        for (int i : {0, 1}) {
            const int c = type == ADHIP_BF16 ? 2 - i : 1 + i;
            const int64_t unit = (int64_t)lanes * v * c;
            if (lanes == 16 ? size == unit : size % unit == 0 && size / unit <= kWaves) packs = c, full = true;
        }
        waves = lanes == 16 ? 1 : (int)((size + 64 * v * packs - 1) / (64 * v * packs));
        groups = lanes == 16 ? kThreads / 16 : std::max(1, kThreads / 64 / waves);
        grad_groups = lanes == 16 ? kWaves * 4 : kWaves / waves;
    }
    int threads(bool backward) const { return lanes == 16 ? (backward ? kWaves * 64 : kThreads) : (backward ? grad_groups : groups) * waves * 64; }
};

int padded_of(int64_t size) { return (int)((size + 3) / 4 * 4); }

int64_t grad_blocks(int type, int64_t rows, int64_t size) {
    const int64_t at_once = Share(type, size).grad_groups;
    return std::min<int64_t>((rows + at_once - 1) / at_once, kGradBlocks);
}

size_t workspace_of(int type, int64_t rows, int64_t size) { return (size_t)grad_blocks(type, rows, size) * 2 * (size_t)padded_of(size) * sizeof(float); }

template <class T, class W, int V, int LANES, int C, bool FULL>
void launch_norm(const char* op, const NormParams& p, const Share& share, bool backward, bool sums, unsigned blocks, hipStream_t stream) {
    const unsigned threads = (unsigned)share.threads(backward);
    if (!backward)
        launch(op, p.added ? norm_kernel<T, W, V, LANES, C, FULL, true> : norm_kernel<T, W, V, LANES, C, FULL, false>, blocks, threads, stream, p);
    else if (sums && p.total_grad)
        launch(op, norm_backward_kernel<T, W, V, LANES, C, FULL, true, true>, blocks, threads, stream, p);
    else if (sums)
        launch(op, norm_backward_kernel<T, W, V, LANES, C, FULL, true, false>, blocks, threads, stream, p);
    else if (p.total_grad)
        launch(op, norm_backward_kernel<T, W, V, LANES, C, FULL, false, true>, blocks, threads, stream, p);
    else
        launch(op, norm_backward_kernel<T, W, V, LANES, C, FULL, false, false>, blocks, threads, stream, p);
}

template <auto X>
using Is = std::integral_constant<decltype(X), X>;

template <class T, class W>
void launch_norm(const char* op, const NormParams& p, const Share& share, bool backward, bool sums, unsigned blocks, hipStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const auto go = [&](auto lanes, auto packs, auto full) {
        launch_norm<T, W, V, lanes(), packs(), full()>(op, p, share, backward, sums, blocks, stream);
    };
    const auto with_lanes = [&](auto lanes) {
        if (share.full && share.packs == 1) return go(lanes, Is<1>(), Is<true>());
        if (share.full) return go(lanes, Is<2>(), Is<true>());
        if (share.packs == 1) return go(lanes, Is<1>(), Is<false>());
        if constexpr (lanes() == 64 && V == 4)
            if (share.packs == 4) return go(lanes, Is<4>(), Is<false>());
        go(lanes, Is<2>(), Is<false>());
    };
    if (share.narrow) launch_norm<T, W, 1, 16, 1, false>(op, p, share, backward, sums, blocks, stream);
    else if (share.lanes == 16) with_lanes(Is<16>());
    else with_lanes(Is<64>());
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

void check_vector(const char* op, const char* name, const adhip_array& a, int64_t size) {
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
    ADHIP_CHECK(!adds || rows == 0 || g.total.data != g.out.data, "%s: total and out are one array", op);
    for (int i = 0; i < n; ++i)
        for (int j = i + 1; j < n; ++j) {
            const Named &a = arrays[i], &b = arrays[j];  // (inputs come first)
            if (b.output && !a.output) check_in_place(op, a.name, *a.a, b.name, *b.a);
            else if (b.output) check_apart(op, a.name, *a.a, b.name, *b.a);
        }
    // weights: of x's type or f32, both alike
    const int w_type = g.weight.data ? g.weight.type : g.bias.data && !backward ? g.bias.type : ADHIP_F32;
    if (g.weight.data) check_vector(op, "weight", g.weight, size);
    if (g.bias.data && !backward) check_vector(op, "bias", g.bias, size);
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
    bool one_sum = false;  // one array for both holds bias_grad: nobody writes weight_grad there before or after it
    if (backward) {
        if (g.weight_grad.data) check_vector(op, "weight_grad", g.weight_grad, size);
        if (g.bias_grad.data) check_vector(op, "bias_grad", g.bias_grad, size);
        if (g.weight_grad.data && g.bias_grad.data) {
            const char *w = (const char*)g.weight_grad.data, *b = (const char*)g.bias_grad.data;
            one_sum = w == b && g.weight_grad.type == g.bias_grad.type;
            ADHIP_CHECK(one_sum || w + size * type_bytes(g.weight_grad.type) <= b || b + size * type_bytes(g.bias_grad.type) <= w,
                        "%s: weight_grad and bias_grad share memory", op);
        }
        ADHIP_CHECK(!sums || rows == 0 || (g.workspace && (uintptr_t)g.workspace % 16 == 0 && g.workspace_bytes >= workspace_of(g.x.type, rows, size)),
                    "%s: the workspace has %zu bytes, %zu are wanted, aligned to 16", op, g.workspace ? g.workspace_bytes : (size_t)0, workspace_of(g.x.type, rows, size));
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
        const Share share(g.x.type, size);
        p.waves = share.waves;
        p.groups = backward ? share.grad_groups : share.groups;
        // A forward workgroup takes several rows, two at least where there are more than the chip has at once, in four times as many workgroups
        // as it holds, and eight times with a residual (16384 rows of 4096 in bf16: 52 us, with a residual 96; the other way round 56 and 98; a
        // row each 76 and 98).
        const int64_t each = (rows + p.groups - 1) / p.groups, at_once = 256 * 2048 / share.threads(false);
        const int64_t rounds = std::max<int64_t>((each - 1) / (at_once * (adds ? 8 : 4)) + 1, each > 2 * at_once ? 2 : 1);
        const int64_t all = (each + rounds - 1) / rounds;
        const unsigned blocks = (unsigned)(backward ? grad_blocks(g.x.type, rows, size) : all);
        if (g.x.type == ADHIP_F32) launch_norm<float, float>(op, p, share, backward, sums, blocks, stream);
        else if (w_type == ADHIP_F32) launch_norm<bf16, float>(op, p, share, backward, sums, blocks, stream);
        else launch_norm<bf16, bf16>(op, p, share, backward, sums, blocks, stream);
    }
    if (sums)
        launch(op, norm_sums_kernel, dim3((unsigned)((size + 63) / 64), 2), 256, stream, (const float*)g.workspace, rows > 0 ? (int)grad_blocks(g.x.type, rows, size) : 0,
               (int)size, p.padded, one_sum ? nullptr : g.weight_grad.data, g.bias_grad.data, g.weight_grad.type == ADHIP_BF16, g.bias_grad.type == ADHIP_BF16);
}

}  // namespace
}  // namespace adhip

extern "C" {

int adhip_layer_norm_workspace(adhip_ctx* ctx, const adhip_layer_norm_args* args, size_t* bytes) {
    return adhip::context_guarded(ctx, [&] {
        const char* op = "adhip_layer_norm_workspace";
        ADHIP_CHECK(args && bytes, "%s: no arguments", op);
        const int64_t rows = adhip::check_rows(op, args->x);
        *bytes = adhip::workspace_of(args->x.type, rows, args->x.dims[args->x.rank - 1]);
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

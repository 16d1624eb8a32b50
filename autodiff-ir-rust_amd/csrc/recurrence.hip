// A gated linear recurrence over the positions of a sequence, each channel by itself (as in the quasi-recurrent network of
// Bradbury et al. 2016 and the minimal gated unit of Zhou et al. 2016):
//     h[t] = a[t] h[t-1] + b[t],   a = sigmoid(gate), b = (1 - a) x,   or  a = gate, b = x  where gates are factors
// and backwards, with l[t] the gradient that reaches h[t] altogether:
//     l[t] = out_grad[t] + a[t+1] l[t+1];   gradient of b: l[t], of a: l[t] h[t-1].
//
// Memory bounds it.  One step is the map h -> A h + B, and two maps one after the other are such a map again (Blelloch 1990), so
// a workgroup takes a tile of positions at once: a thread composes the maps of its K consecutive ones, threads of a wavefront and
// wavefronts of the workgroup exchange theirs, and each thread then walks its positions again from the state that it now
// knows, out of registers.  From tile to tile only the state is carried, so inputs are read once.  The backward pass needs the
// states again: the forward pass leaves one every 256 positions, from which a tile of them is recomputed beside the gradients,
// instead of reading all outputs, which are rounded.
#include "operators.hpp"

#include <algorithm>
#include <cmath>

namespace adhip {
namespace {

constexpr int kBlock = ADHIP_RECURRENCE_BLOCK;  // positions between states that are kept
constexpr int kWaves = 8, kThreads = kWaves * 64;
constexpr int kLanes = 16;                      // of a row of channels: four positions' threads a wavefront
constexpr int kSteps = 8;                       // consecutive positions of a thread
constexpr int kTile = kThreads / kLanes * kSteps;
static_assert(kTile == kBlock, "a tile of the backward pass begins at a state that is kept");
constexpr unsigned kAll = (1u << kSteps) - 1;

struct Rows {
    int64_t b, t;  // strides of batch and positions
};

struct RecurrenceParams {
    const void *x, *gates, *out_grad;
    void *out, *x_grad, *gates_grad;
    const float *initial, *final_grad;
    float *states, *final, *initial_grad;
    const int *lengths, *documents;
    Rows x_at, gates_at, out_at, out_grad_at, x_grad_at, gates_grad_at, states_at, documents_at;
    int64_t initial_b, final_b, final_grad_b, initial_grad_b, lengths_b;
    int length, channels, groups;  // groups: of channels that a workgroup takes
};

// Elements that begin at any of their own addresses: global memory takes such accesses.
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[N];
};

// 1 / (1 + exp(-g)) and 1 / (1 + exp(g)), each to its own last bits.
template <class T>
__device__ __forceinline__ void sigmoids(float g, float& a, float& rest) {
    constexpr float kLog2 = 1.44269504f;
    float y = -fabsf(g);
    float e;
    if (sizeof(T) == 4) {
        y = y < -150.f ? -150.f : y;  // (infinities have no remainder; a NaN stays one)
        const float t = y * kLog2;
        const float low = __builtin_fmaf(y, 1.92596299e-8f, __builtin_fmaf(y, kLog2, -t));
        e = __builtin_amdgcn_exp2f(t);
        e = __builtin_fmaf(e, low * 0.693147181f, e);
    } else {
        e = __builtin_amdgcn_exp2f(y * kLog2);  // (|g| 2^-24 off, far below what is kept of a result)
    }
    const float r = __builtin_amdgcn_rcpf(1.f + e), s = e * r;
    a = g < 0.f ? s : r;
    rest = g < 0.f ? r : s;
}

// The map h -> a h + b of a state, and the factor of two maps one after the other.  A factor of zero drops what was there and a
// state of zero takes any factor, also where the other one has grown beyond all numbers.  States of sigmoid gates are means
// of what was put in and their factors at most 1: always finite, and zero times such a number is zero by itself.
template <bool FACTORS>
__device__ __forceinline__ float onward(float a, float h, float b) {
    const float r = __builtin_fmaf(a, h, b);
    return FACTORS && (a == 0.f || h == 0.f) ? b : r;
}
template <bool FACTORS>
__device__ __forceinline__ float together(float a, float b) {
    return FACTORS && (a == 0.f || b == 0.f) ? 0.f : a * b;
}

// Which of K positions from t on count (live), and where the state before is dropped (cut); positions from `count` on pass it on.
struct Marks {
    unsigned live, cut;
    int count;
    __device__ __forceinline__ Marks(const RecurrenceParams& p, int64_t b, int t, int length) {
        count = min(max(length - t, 0), kSteps);
        live = (1u << count) - 1;
        cut = 0;
        if (p.documents && count > 0) {
            const int* d = p.documents + b * p.documents_at.b;
            int before = d[(int64_t)(t > 0 ? t - 1 : t) * p.documents_at.t];
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
                if (k < count) {
                    const int here = d[(int64_t)(t + k) * p.documents_at.t];
                    if (here < 0) live &= ~(1u << k);
                    if (here < 0 || here != before) cut |= 1u << k;
                    before = here;
                }
        }
    }
    __device__ __forceinline__ bool plain() const { return live == kAll && cut == 0; }
};

// K positions of V channels; zeros where there are none.
template <class T, int V>
struct Steps {
    Loose<T, V> r[kSteps];
    __device__ __forceinline__ void load(const void* from, const Rows& at, int64_t b, int t, int c, int length, int channels) {
        const T* x = (const T*)from + b * at.b + (int64_t)t * at.t + c;
        if (t + kSteps <= length && c + V <= channels) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) r[k] = *(const Loose<T, V>*)(x + k * at.t);
        } else {
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) r[k].v[v] = t + k < length && c + v < channels ? x[k * at.t + v] : (T)0.f;
        }
    }
    __device__ __forceinline__ void store(void* to, const Rows& at, int64_t b, int t, int c, int length, int channels) const {
        T* x = (T*)to + b * at.b + (int64_t)t * at.t + c;
        if (t + kSteps <= length && c + V <= channels) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) *(Loose<T, V>*)(x + k * at.t) = r[k];
        } else {
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (t + k < length && c + v < channels) x[k * at.t + v] = r[k].v[v];
        }
    }
};

template <int V>
__device__ __forceinline__ void load_state(const float* from, int64_t at, int c, int channels, float (&h)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = from && c + v < channels ? from[at + c + v] : 0.f;
}
template <int V>
__device__ __forceinline__ void store_state(float* to, int64_t at, int c, int channels, const float (&h)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (c + v < channels) to[at + c + v] = h[v];
}

// The maps of a thread's positions.
template <class T, int V, bool FACTORS>
__device__ __forceinline__ void maps(const Steps<T, V>& x, const Steps<T, V>& g, const Marks& m, float (&a)[kSteps][V], float (&b)[kSteps][V]) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float in = (float)x.r[k].v[v];
            if (FACTORS) {
                a[k][v] = (float)g.r[k].v[v];
                b[k][v] = in;
            } else {
                float rest;
                sigmoids<T>((float)g.r[k].v[v], a[k][v], rest);
                b[k][v] = rest * in;
            }
        }
    if (!m.plain())
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                a[k][v] = m.cut >> k & 1 ? 0.f : k < m.count ? a[k][v] : 1.f;
                b[k][v] = m.live >> k & 1 ? b[k][v] : 0.f;
            }
}

// The exchange between the four threads of a wavefront that have the same channels: composes A h + B of the threads before this
// one (behind it where BACK), and of all four.
template <bool FACTORS, bool BACK>
__device__ __forceinline__ void across(int lane, float& A, float& B, float& preA, float& preB) {
    preA = 1, preB = 0;
#pragma unroll
    for (int off = kLanes; off < 64; off *= 2) {
        const float otherA = __shfl_xor(A, off), otherB = __shfl_xor(B, off);
        if (((lane & off) != 0) != BACK) {
            preB = onward<FACTORS>(preA, otherB, preB);
            preA = together<FACTORS>(preA, otherA);
            B = onward<FACTORS>(A, otherB, B);
        } else {
            B = onward<FACTORS>(otherA, B, otherB);
        }
        A = together<FACTORS>(A, otherA);
    }
}

template <class T, int V, bool FACTORS>
__global__ __launch_bounds__(kThreads) void recurrence_kernel(const RecurrenceParams p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), slot = (lane & (kLanes - 1)) * V;
    const int64_t batch = blockIdx.x / (unsigned)p.groups;
    const int c = (int)(blockIdx.x % (unsigned)p.groups) * kLanes * V + slot;
    const int length = p.lengths ? min(max(p.lengths[batch * p.lengths_b], 0), p.length) : p.length;
    const int own = (wave * 4 + lane / kLanes) * kSteps;  // this thread's positions in a tile
    __shared__ float2 parts[2][kWaves][kLanes * V];       // (by turns: the other one's barrier stands between readers and writers)
    float carry[V];
    load_state<V>(p.initial, batch * p.initial_b, c, p.channels, carry);
    Steps<T, V> x, g, next_x, next_g;
    x.load(p.x, p.x_at, batch, own, c, length, p.channels);
    g.load(p.gates, p.gates_at, batch, own, c, length, p.channels);
    int turn = 0;
    for (int begin = 0; begin < p.length; begin += kTile, turn ^= 1) {
        const int t = begin + own;
        if (begin + kTile < p.length) {
            next_x.load(p.x, p.x_at, batch, t + kTile, c, length, p.channels);
            next_g.load(p.gates, p.gates_at, batch, t + kTile, c, length, p.channels);
        }
        const Marks m(p, batch, t, length);
        float a[kSteps][V], b[kSteps][V], A[V], B[V], preA[V], preB[V], h[V];
        maps<T, V, FACTORS>(x, g, m, a, b);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            A[v] = 1, B[v] = 0;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                A[v] = together<FACTORS>(A[v], a[k][v]);
                B[v] = onward<FACTORS>(a[k][v], B[v], b[k][v]);
            }
            across<FACTORS, false>(lane, A[v], B[v], preA[v], preB[v]);
            if (lane < kLanes) parts[turn][wave][slot + v] = make_float2(A[v], B[v]);
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 part = parts[turn][w][slot + v];
                if (w == wave) h[v] = carry[v];
                carry[v] = onward<FACTORS>(part.x, carry[v], part.y);
            }
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = onward<FACTORS>(preA[v], h[v], preB[v]);
        if (p.states && own == 0) store_state<V>(p.states, batch * p.states_at.b + (int64_t)(t / kBlock) * p.states_at.t, c, p.channels, h);
        Steps<T, V> o;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = onward<FACTORS>(a[k][v], h[v], b[k][v]);
                o.r[k].v[v] = (T)(m.live >> k & 1 ? h[v] : 0.f);
            }
        o.store(p.out, p.out_at, batch, t, c, p.length, p.channels);
        x = next_x;
        g = next_g;
    }
    if (p.final && own == 0) store_state<V>(p.final, batch * p.final_b, c, p.channels, carry);
}

template <class T, int V, bool FACTORS>
__global__ __launch_bounds__(kThreads) void recurrence_backward_kernel(const RecurrenceParams p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), slot = (lane & (kLanes - 1)) * V;
    const int64_t batch = blockIdx.x / (unsigned)p.groups;
    const int c = (int)(blockIdx.x % (unsigned)p.groups) * kLanes * V + slot;
    const int length = p.lengths ? min(max(p.lengths[batch * p.lengths_b], 0), p.length) : p.length;
    const int own = (wave * 4 + lane / kLanes) * kSteps;
    __shared__ float2 parts[2][kWaves][kLanes * V];
    __shared__ float back_parts[2][kWaves][kLanes * V];
    float carry[V];  // the gradient of the state behind the tile
    load_state<V>(p.final_grad, batch * p.final_grad_b, c, p.channels, carry);
    int turn = 0;
    for (int begin = (p.length - 1) / kTile * kTile; begin >= 0 && p.length > 0; begin -= kTile, turn ^= 1) {
        const int t = begin + own;
        Steps<T, V> x, g, d;
        x.load(p.x, p.x_at, batch, t, c, length, p.channels);
        g.load(p.gates, p.gates_at, batch, t, c, length, p.channels);
        d.load(p.out_grad, p.out_grad_at, batch, t, c, length, p.channels);
        float state[V];
        load_state<V>(p.states, batch * p.states_at.b + (int64_t)(begin / kBlock) * p.states_at.t, c, p.channels, state);
        const Marks m(p, batch, t, length);
        float a[kSteps][V], b[kSteps][V], A[V], B[V], preA[V], preB[V], back[V], behindA[V], behindB[V], h[V], l[V];
        maps<T, V, FACTORS>(x, g, m, a, b);
        if (m.live != kAll)
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) d.r[k].v[v] = m.live >> k & 1 ? d.r[k].v[v] : (T)0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            A[v] = 1, B[v] = 0, back[v] = 0;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                A[v] = together<FACTORS>(A[v], a[k][v]);
                B[v] = onward<FACTORS>(a[k][v], B[v], b[k][v]);
            }
#pragma unroll
            for (int k = kSteps - 1; k >= 0; --k) back[v] = onward<FACTORS>(a[k][v], back[v] + (float)d.r[k].v[v], 0.f);
            float again = A[v];
            across<FACTORS, false>(lane, A[v], B[v], preA[v], preB[v]);
            across<FACTORS, true>(lane, again, back[v], behindA[v], behindB[v]);
            if (lane < kLanes) {
                parts[turn][wave][slot + v] = make_float2(A[v], B[v]);
                back_parts[turn][wave][slot + v] = back[v];
            }
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = state[v];
#pragma unroll
            for (int w = 0; w < kWaves - 1; ++w) {
                const float2 part = parts[turn][w][slot + v];
                if (w < wave) h[v] = onward<FACTORS>(part.x, h[v], part.y);
            }
#pragma unroll
            for (int w = kWaves - 1; w >= 0; --w) {
                if (w == wave) l[v] = carry[v];
                carry[v] = onward<FACTORS>(parts[turn][w][slot + v].x, carry[v], back_parts[turn][w][slot + v]);
            }
            h[v] = onward<FACTORS>(preA[v], h[v], preB[v]);
            l[v] = onward<FACTORS>(behindA[v], l[v], behindB[v]);
        }
        // forwards: b becomes the state before each position (what the factor is multiplied with)
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float before = h[v];
                h[v] = onward<FACTORS>(a[k][v], h[v], b[k][v]);
                b[k][v] = m.cut >> k & 1 ? 0.f : before;
            }
        // backwards
#pragma unroll
        for (int k = kSteps - 1; k >= 0; --k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float here = l[v] + (float)d.r[k].v[v], in = (float)x.r[k].v[v];
                l[v] = onward<FACTORS>(a[k][v], here, 0.f);
                float dx = here, dg = here * b[k][v];
                if (!FACTORS) {
                    float own_a, rest;
                    sigmoids<T>((float)g.r[k].v[v], own_a, rest);
                    dx = here * rest;
                    dg = dx * (b[k][v] - in) * own_a;
                }
                const bool live = m.live >> k & 1;
                x.r[k].v[v] = (T)(live ? dx : 0.f);
                g.r[k].v[v] = (T)(live ? dg : 0.f);
            }
        x.store(p.x_grad, p.x_grad_at, batch, t, c, p.length, p.channels);
        g.store(p.gates_grad, p.gates_grad_at, batch, t, c, p.length, p.channels);
    }
    if (p.initial_grad && own == 0) store_state<V>(p.initial_grad, batch * p.initial_grad_b, c, p.channels, carry);
}

template <class T, int V>
void launch_recurrence(const char* op, const RecurrenceParams& p, bool backward, bool factors, int64_t blocks, hipStream_t stream) {
    launch(op, backward ? (factors ? recurrence_backward_kernel<T, V, true> : recurrence_backward_kernel<T, V, false>)
                        : (factors ? recurrence_kernel<T, V, true> : recurrence_kernel<T, V, false>), (unsigned)blocks, kThreads, stream, p);
}

// Shape and type of x: [batch, length, channels].
void check_x(const char* op, const adhip_array& x) {
    ADHIP_CHECK(x.type == ADHIP_F32 || x.type == ADHIP_BF16, "%s: x is %s, f32 or bf16 is wanted", op, type_name(x.type));
    check_shape(op, "x", x, x.type, 3);
    for (int d = 0; d < 3; ++d)
        ADHIP_CHECK(x.dims[d] < (int64_t(1) << 30), "%s: x is %s, extents below 2^30 are wanted", op, array_str(x).c_str());
}

// An array of x's shape.
Rows check_like(const char* op, const char* name, const adhip_array& a, const adhip_array& x, bool output) {
    check_array(op, name, a, x.type, 3);
    check_dims(op, name, a, {x.dims[0], x.dims[1], x.dims[2]});
    check_packed_rows(op, name, a);
    if (output) check_distinct(op, name, a);
    return {a.strides[0], a.strides[1]};
}

// f32 [batch, channels], which need not be given.
int64_t check_state(const char* op, const char* name, const adhip_array& a, const adhip_array& x, bool output) {
    if (!a.data) return 0;
    check_array(op, name, a, ADHIP_F32, 2);
    check_dims(op, name, a, {x.dims[0], x.dims[2]});
    check_packed_rows(op, name, a);
    if (output) check_distinct(op, name, a);
    return a.strides[0];
}

void recurrence(const char* op, const adhip_recurrence_args& g, bool backward, hipStream_t stream) {
    check_x(op, g.x);
    const int64_t batch = g.x.dims[0], length = g.x.dims[1], channels = g.x.dims[2];
    RecurrenceParams p = {};
    p.x_at = check_like(op, "x", g.x, g.x, false);
    p.gates_at = check_like(op, "gates", g.gates, g.x, false);
    if (backward) {
        p.out_grad_at = check_like(op, "out_grad", g.out_grad, g.x, false);
        p.x_grad_at = check_like(op, "x_grad", g.x_grad, g.x, true);
        p.gates_grad_at = check_like(op, "gates_grad", g.gates_grad, g.x, true);
        p.final_grad_b = check_state(op, "final_grad", g.final_grad, g.x, false);
        p.initial_grad_b = check_state(op, "initial_grad", g.initial_grad, g.x, true);
    } else {
        p.out_at = check_like(op, "out", g.out, g.x, true);
        p.initial_b = check_state(op, "initial", g.initial, g.x, false);
        p.final_b = check_state(op, "final", g.final, g.x, true);
    }
    if (backward || g.states.data) {
        check_array(op, "states", g.states, ADHIP_F32, 3);
        check_dims(op, "states", g.states, {batch, (length + kBlock - 1) / kBlock, channels});
        check_packed_rows(op, "states", g.states);
        if (!backward) check_distinct(op, "states", g.states);
        p.states_at = {g.states.strides[0], g.states.strides[1]};
    }
    if (g.lengths.data) {
        check_array(op, "lengths", g.lengths, ADHIP_I32, 1);
        check_dims(op, "lengths", g.lengths, {batch});
        p.lengths_b = g.lengths.strides[0];
    }
    if (g.documents.data) {
        check_array(op, "documents", g.documents, ADHIP_I32, 2);
        check_dims(op, "documents", g.documents, {batch, length});
        p.documents_at = {g.documents.strides[0], g.documents.strides[1]};
    }
    p.x = g.x.data, p.gates = g.gates.data, p.lengths = (const int*)g.lengths.data, p.documents = (const int*)g.documents.data;
    p.states = (float*)g.states.data;
    if (backward) {
        p.out_grad = g.out_grad.data, p.x_grad = g.x_grad.data, p.gates_grad = g.gates_grad.data;
        p.final_grad = (const float*)g.final_grad.data, p.initial_grad = (float*)g.initial_grad.data;
    } else {
        p.out = g.out.data, p.initial = (const float*)g.initial.data, p.final = (float*)g.final.data;
    }
    p.length = (int)length;
    p.channels = (int)channels;
    const int v = g.x.type == ADHIP_BF16 ? 2 : 1;
    p.groups = (int)((channels + kLanes * v - 1) / (kLanes * v));
    const int64_t blocks = batch * p.groups;
    ADHIP_CHECK(fits_launch(blocks, kThreads), "%s: %lld sequences of %lld channels are too many for one call", op, (long long)batch, (long long)channels);
    if (blocks == 0) return;
    if (g.x.type == ADHIP_BF16) launch_recurrence<bf16, 2>(op, p, backward, g.factors != 0, blocks, stream);
    else launch_recurrence<float, 1>(op, p, backward, g.factors != 0, blocks, stream);
}

}  // namespace
}  // namespace adhip

extern "C" {

int adhip_recurrence_workspace(adhip_ctx* ctx, const adhip_recurrence_args* args, int backward, size_t* bytes) {
    return adhip::context_guarded(ctx, [&] {
        const char* op = "adhip_recurrence_workspace";
        ADHIP_CHECK(args && bytes, "%s: no arguments", op);
        adhip::check_x(op, args->x);
        *bytes = 0;
    });
}

int adhip_recurrence(adhip_ctx* ctx, const adhip_recurrence_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_recurrence: no arguments");
        adhip::recurrence("adhip_recurrence", *args, false, (hipStream_t)stream);
    });
}

int adhip_recurrence_backward(adhip_ctx* ctx, const adhip_recurrence_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_recurrence_backward: no arguments");
        adhip::recurrence("adhip_recurrence_backward", *args, true, (hipStream_t)stream);
    });
}
}

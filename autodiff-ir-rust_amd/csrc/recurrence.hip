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
//
// 2 x 8192 positions of 4096 channels in bf16: forward 108 us, backward 179 (3.8 TB/s; in this pattern, 64 bytes of rows 8 KB apart, two
// arrays copied into a third take 107, three into two 186), of 4032 channels 90 and 151; 4 x 2048 of 4096 in f32, 128 bytes of a row: 80 and 134 (5.0 TB/s).  One position of
// 256 x 8192 channels: 12 us.  A compute unit with one workgroup of wide rows takes 5.0 us for a tile of 256 positions of 64 channels from memory and 4.1 from the last
// cache (4 x 2049 of 2560 in bf16, factors: 45 and 37 us): its vector units issue 61 % of the latter's cycles, 25 instructions an element.
#include "operators.hpp"

#include <algorithm>
#include <cmath>
#include <utility>

namespace adhip {
namespace {

constexpr int kBlock = ADHIP_RECURRENCE_BLOCK;  // positions between states that are kept
constexpr int kTile = kBlock;                   // positions that a workgroup takes at once: a tile begins at a state that is kept
constexpr int kSteps = 8;                       // consecutive positions of a thread
// A workgroup takes rows of LANES times 4 bytes of channels; as many threads of each lane share the positions of a tile.
template <int LANES>
struct Team {
    static constexpr int kThreads = kTile / kSteps * LANES, kWaves = kThreads / 64, kSpread = 64 / LANES;
    // A sequence shorter than a tile takes no more wavefronts than it has positions for.
    static int threads(int length) { return std::min(kThreads, (std::max(length, 1) + kSteps * kSpread - 1) / (kSteps * kSpread) * 64); }
};
constexpr unsigned kAll = (1u << kSteps) - 1;
constexpr int kNarrow = 16, kWide = 32;         // lanes of a row of channels
constexpr int kFull = 256;                      // workgroups that give every compute unit one

struct Rows {
    int64_t b, t;  // strides of batch and positions
};

struct RecurrenceParams {
    const void *x, *gates, *out_grad;
    void *out, *x_grad, *gates_grad;
    const float *initial, *final_grad;
    float *states, *final, *initial_grad;
    const int *lengths, *documents;
    float2* carry;  // [ranges, batch, channels]: what a range does to a state (to a gradient); one place holds what all begin with
    Rows x_at, gates_at, out_at, out_grad_at, x_grad_at, gates_grad_at, states_at, documents_at;
    int64_t initial_b, final_b, final_grad_b, initial_grad_b, lengths_b;
    int length, channels, groups;  // groups: of channels that a workgroup takes
    int batch, ranges, tiles;      // of positions, and tiles of a range
    bool past;                     // results go past the caches
    bool near;                     // neighbouring workgroups share cache lines
};

// Operand of a wait for all memory operations of a wavefront, and of nothing else.
constexpr int kNoneUnderWay = 0x0f70;

// 4 bytes of channels, beginning at any element: global memory takes such accesses.
template <class T>
constexpr int kPack = 4 / sizeof(T);
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Word {
    unsigned w;
};

template <class T>
__device__ __forceinline__ void unpack(unsigned w, float (&f)[kPack<T>]) {
    if constexpr (sizeof(T) == 4) {
        f[0] = __uint_as_float(w);
    } else {
        f[0] = __uint_as_float(w << 16);
        f[1] = __uint_as_float(w & 0xffff0000u);
    }
}
template <class T>
__device__ __forceinline__ unsigned pack(const float (&f)[kPack<T>]) {
    union {
        T v[kPack<T>];
        unsigned w;
    } u;
#pragma unroll
    for (int v = 0; v < kPack<T>; ++v) u.v[v] = (T)f[v];
    return u.w;
}

// a = 1 / (1 + exp(-g)) and rest = 1 / (1 + exp(g)), each to its own last bits.
template <class T>
__device__ __forceinline__ void sigmoids(float g, float& a, float& rest) {
    constexpr float kLog2 = 1.44269504f;
    if constexpr (sizeof(T) == 4) {
        float y = -fabsf(g);
        y = y < -150.f ? -150.f : y;  // (infinities have no remainder; a NaN stays one)
        const float t = y * kLog2;
        const float low = __builtin_fmaf(y, 1.92596299e-8f, __builtin_fmaf(y, kLog2, -t));
        float e = __builtin_amdgcn_exp2f(t);
        e = __builtin_fmaf(e, low * 0.693147181f, e);
        const float r = __builtin_amdgcn_rcpf(1.f + e), s = e * r;
        a = g < 0.f ? s : r;
        rest = g < 0.f ? r : s;
    } else {
        // The exponent is |g| 2^-24 off, far below what is kept of a result.  Below -83 a gate counts as -83 (a = 2^-120), whose
        // exponential still has a reciprocal.
        const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g * -kLog2, 120.f));
        a = __builtin_amdgcn_rcpf(1.f + e);
        rest = e * a;
    }
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

// The same with the factor of one position, which is finite: a comparison that serves both (4 x 2049 positions of 2560 channels in bf16,
// factors: forward 48 us, with the other two 51; both passes 146 and 158).
template <bool FACTORS>
__device__ __forceinline__ float step(float a, float h, float b) {
    const float r = __builtin_fmaf(a, h, b);
    return FACTORS && a == 0.f ? b : r;
}
template <bool FACTORS>
__device__ __forceinline__ float grown(float A, float a) {
    const float r = A * a;
    return FACTORS && a == 0.f ? 0.f : r;
}

// Which of K positions from t on count (live), and where the state before is dropped (cut); positions from `count` on pass it on.
struct Marks {
    unsigned live, cut;
    int count;
    __device__ __forceinline__ bool plain() const { return live == kAll && cut == 0; }
};

// Documents of a wavefront's positions: every lane looks at one of them and at the one before it, and all are told (each thread at its own
// eight: 16 x 1000 positions of 4000 channels in f32, both passes: 494 us; so 453).
template <int LANES>
struct Documents {
    static constexpr int kPositions = 64 / LANES * kSteps;
    int here, before;
    // Which of a wavefront's positions a lane looks at.
    static __device__ __forceinline__ int looked_at(int lane) { return lane % kPositions; }
    __device__ __forceinline__ void load(const RecurrenceParams& p, int64_t b, int t) {
        const int* from = p.documents + b * p.documents_at.b;
        here = from[(int64_t)min(t, p.length - 1) * p.documents_at.t];
        before = from[(int64_t)min(max(t - 1, 0), p.length - 1) * p.documents_at.t];
    }
    __device__ __forceinline__ Marks marks(int lane, int count) const {
        const int shift = lane / LANES * kSteps;
        const unsigned all = (1u << count) - 1, none = (unsigned)(__ballot(here < 0) >> shift), other = (unsigned)(__ballot(here < 0 || here != before) >> shift);
        return {all & ~none, all & other, count};
    }
};

// An address that all lanes share stays in scalar registers; folded into the lanes' own it would take two registers of each.
template <class P>
__device__ __forceinline__ P* row_of(P* p) {
    asm("" : "+s"(p));
    return p;
}

// K positions of a pack of channels.
template <class T>
struct Steps {
    unsigned w[kSteps];
};

// Where a workgroup and a thread of it are.
template <class T, int LANES>
struct Seat {
    static constexpr int V = kPack<T>;
    int lane, wave, slot, base, c, own, range, first, tiles, length;
    int64_t batch, state;  // state: of the channels in [batch, channels]
    bool lone;
    __device__ __forceinline__ Seat(const RecurrenceParams& p) {
        lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), slot = (lane & (LANES - 1)) * V;
        // Workgroups go to the eight dies in turn: of 256, which run at a time, neighbours of a row, whose channels share cache lines,
        // go to one die, and together they cover whole rows (2 x 8192 positions of 4096 channels in bf16, both passes: 285 us, and 319 without; 8191
        // of 1000 in f32 104 and 125).  Where rows of workgroups are whole lines there is nothing to share (4 x 2048 of 4096 in f32: 224 us so, 214
        // without).
        unsigned at = blockIdx.x;
        if (p.near) {
            const unsigned window = at / kFull * kFull, of = at % kFull, die = min(gridDim.x - window, (unsigned)kFull) / 8;
            at = window + of % 8 * die + of / 8;
        }
        const unsigned group = at % (unsigned)p.groups;
        at /= (unsigned)p.groups;
        batch = at % (unsigned)p.batch;
        range = (int)(at / (unsigned)p.batch);
        // Packs that would pass the row's end begin before it: their lanes compute what a neighbour in their wavefront computes too, bit
        // for bit.  A lone last channel has no neighbour here, but in another workgroup, which may already have written there.
        base = (int)group * LANES * V;
        lone = base + V > p.channels;
        c = lone ? base : min(base + slot, p.channels - V);
        own = (wave * Team<LANES>::kSpread + lane / LANES) * kSteps;
        first = range * p.tiles * kTile;
        tiles = min(p.tiles, (p.length - first + kTile - 1) / kTile);
        length = p.lengths ? min(max(p.lengths[batch * p.lengths_b], 0), p.length) : p.length;
        state = batch * p.channels + c;
    }
    // (a launch has a multiple of eight workgroups)
    __device__ __forceinline__ bool there(int ranges) const { return range < ranges; }
    // Tiles of this range that have positions of the sequence.
    __device__ __forceinline__ int used() const { return min((max(length - first, 0) + kTile - 1) / kTile, tiles); }
};

// An array's tiles as seen by a thread: uniform addresses of positions, and this thread's own bytes from there.  Whole tiles, tiles
// that end within and lone channels make the same number of loads, without a branch between them, so that the compiler knows
// how many are under way and waits for those that it needs alone.
template <class T>
struct Side {
    char* tile;
    int64_t step;
    unsigned off, lane;
    template <int LANES>
    __device__ __forceinline__ Side(const void* p, const Rows& at, const Seat<T, LANES>& seat)
        : tile((char*)p + (seat.batch * at.b + (int64_t)seat.first * at.t + seat.base) * (int64_t)sizeof(T)), step(at.t * (int64_t)sizeof(T)),
          off((unsigned)seat.own * (unsigned)step), lane((unsigned)(seat.c - seat.base) * (unsigned)sizeof(T)) {}
    // Tile i, of which `rows` positions are there (those behind are read as the last one), or where `there` says that there is none,
    // bytes of its beginning that cost next to nothing.
    template <int LANES>
    __device__ __forceinline__ void load(Steps<T>& s, const Seat<T, LANES>& seat, int i, int rows, bool there) const {
        const char* from = tile + (int64_t)i * kTile * step;
        if (rows >= kTile && !seat.lone) {
            const unsigned at = there ? off + lane : 0;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) s.w[k] = ((const Word<T>*)(row_of(from + k * step) + at))->w;
        } else if (!seat.lone) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
                s.w[k] = ((const Word<T>*)(from + ((unsigned)min(seat.own + k, rows - 1) * (unsigned)step + lane)))->w;
        } else {
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
                s.w[k] = *(const unsigned short*)(from + (unsigned)min(seat.own + k, rows - 1) * (unsigned)step);
        }
    }
    template <int LANES>
    __device__ __forceinline__ void store(const Steps<T>& s, const Seat<T, LANES>& seat, int i, int rows, bool past) const {
        char* to = tile + (int64_t)i * kTile * step;
        if (rows >= kTile && !seat.lone) {
            if (LANES == kWide && past) {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) store_past((Word4*)(row_of(to + k * step) + (off + lane)), s.w[k]);
            } else {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) ((Word<T>*)(row_of(to + k * step) + (off + lane)))->w = s.w[k];
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
            if (seat.own + k < rows) {
                char* at = to + ((unsigned)(seat.own + k) * (unsigned)step + lane);
                if (seat.lone) *(unsigned short*)at = (unsigned short)s.w[k];
                else ((Word<T>*)at)->w = s.w[k];
            }
        // Stores that only some ways make would have the compiler wait for those of whole tiles too: it sees here that none is left.
        __builtin_amdgcn_s_waitcnt(kNoneUnderWay);
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

// The maps of a thread's positions as they are, and with marks.
template <class T, bool FACTORS>
__device__ __forceinline__ void maps(const Steps<T>& x, const Steps<T>& g, float (&a)[kSteps][kPack<T>], float (&b)[kSteps][kPack<T>]) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        float in[kPack<T>], gate[kPack<T>];
        unpack<T>(x.w[k], in);
        unpack<T>(g.w[k], gate);
#pragma unroll
        for (int v = 0; v < kPack<T>; ++v) {
            if (FACTORS) {
                a[k][v] = gate[v];
                b[k][v] = in[v];
            } else {
                float rest;
                sigmoids<T>(gate[v], a[k][v], rest);
                b[k][v] = rest * in[v];
            }
        }
    }
}
template <int V>
__device__ __forceinline__ void mark(const Marks& m, float (&a)[kSteps][V], float (&b)[kSteps][V]) {
    if (m.plain()) return;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            a[k][v] = m.cut >> k & 1 ? 0.f : k < m.count ? a[k][v] : 1.f;
            b[k][v] = m.live >> k & 1 ? b[k][v] : 0.f;
        }
}
template <class T>
__device__ __forceinline__ void hide(const Marks& m, Steps<T>& s) {
    if (m.live == kAll) return;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) s.w[k] = m.live >> k & 1 ? s.w[k] : 0;
}

// What the lanes of each two neighbouring groups of OFF (16 or 32) hold, in the lanes of both: the lower group's, the upper one's.  (Through
// LDS, as a shuffle goes: 141 us instead of 134 for both passes of 4 x 2049 positions of 2560 channels in bf16, factors.)
template <int OFF>
__device__ __forceinline__ void both(float x, float& low, float& high) {
    const int i = __builtin_bit_cast(int, x);
    if constexpr (OFF == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
        low = __builtin_bit_cast(float, (int)r[0]), high = __builtin_bit_cast(float, (int)r[1]);
    } else {
        static_assert(OFF == 32, "rows of 16 lanes, or halves");
        const auto r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
        low = __builtin_bit_cast(float, (int)r[0]), high = __builtin_bit_cast(float, (int)r[1]);
    }
}

// The exchange between the threads of a wavefront that have the same channels: composes A h + B of the threads before this
// one (behind it where BACK), and of all of them.
template <int OFF, bool FACTORS, bool BACK>
__device__ __forceinline__ void across(int lane, float& A, float& B, float& preA, float& preB) {
    float lowA, highA, lowB, highB;
    both<OFF>(A, lowA, highA);
    both<OFF>(B, lowB, highB);
    const float firstA = BACK ? highA : lowA, firstB = BACK ? highB : lowB, thenA = BACK ? lowA : highA, thenB = BACK ? lowB : highB;
    const bool second = ((lane & OFF) != 0) != BACK;
    const float b = onward<FACTORS>(preA, firstB, preB), a = together<FACTORS>(preA, firstA);
    preB = second ? b : preB;
    preA = second ? a : preA;
    B = onward<FACTORS>(thenA, firstB, thenB);
    A = together<FACTORS>(firstA, thenA);
    if constexpr (OFF < 32) across<OFF * 2, FACTORS, BACK>(lane, A, B, preA, preB);
}

// A state carried over whole ranges, from `r` on up to, but not, `end`.  The maps are loaded eight at once: there may be many.
template <class T, int LANES, bool FACTORS>
__device__ __forceinline__ void over_ranges(const RecurrenceParams& p, const Seat<T, LANES>& seat, int r, int end, int way, float (&h)[kPack<T>]) {
    constexpr int kAtOnce = 8;
    const int64_t range = (int64_t)p.batch * p.channels;
    while (r != end) {
        float2 m[kAtOnce][kPack<T>];
        const int n = min(abs(end - r), kAtOnce);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
            for (int v = 0; v < kPack<T>; ++v) m[i][v] = p.carry[(r + way * min(i, n - 1)) * range + seat.state + (seat.lone ? 0 : v)];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
            for (int v = 0; v < kPack<T>; ++v)
                if (i < n) h[v] = onward<FACTORS>(m[i][v].x, h[v], m[i][v].y);
        r += way * n;
    }
}

// The range whose map nobody asks for: the last one's, and backwards the first one's.  Its place holds the state (the gradient) that all begin
// with, put aside before any range writes: final may be initial and initial_grad final_grad, and the range that writes them may be done
// before another one begins.
template <bool BACK>
__device__ __forceinline__ int64_t aside(const RecurrenceParams& p) {
    return BACK ? 0 : (int64_t)(p.ranges - 1) * p.batch * p.channels;
}

// The state before a range's first position, and backwards the gradient behind its last one.
template <class T, int LANES, bool FACTORS, bool BACK>
__device__ __forceinline__ void first_state(const RecurrenceParams& p, const Seat<T, LANES>& seat, const float* given, int64_t given_b,
                                            float (&h)[kPack<T>]) {
    constexpr int V = kPack<T>;
    if (p.ranges == 1) return load_state<V>(given, seat.batch * given_b, seat.c, p.channels, h);
    float2 kept[V];
#pragma unroll
    for (int v = 0; v < V; ++v) kept[v] = p.carry[aside<BACK>(p) + seat.state + (seat.lone ? 0 : v)];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = kept[v].y;
    over_ranges<T, LANES, FACTORS>(p, seat, BACK ? p.ranges - 1 : 0, seat.range, BACK ? -1 : 1, h);
}

// A state carried over the maps of whole wavefronts, from `w` on up to, but not, `end`, four loads at once.  `map` reads one.  A wavefront
// goes over those before it alone, and of a pack's two channels a thread over one: with all of both, where 16 wavefronts share wide rows,
// a third of all instructions (4 x up to 2049 positions of 2560 channels: 41 us, with all 44; 256 x 16 of 1024, both passes: 40 and 48).
template <bool FACTORS, class M>
__device__ __forceinline__ float over_waves(int w, int end, int way, float h, M&& map) {
    constexpr int kAtOnce = 4;
    while (w != end) {
        float2 m[kAtOnce];
        const int n = min(abs(end - w), kAtOnce);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) m[i] = map(w + way * min(i, n - 1));
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (i < n) h = onward<FACTORS>(m[i].x, h, m[i].y);
        w += way * n;
    }
    return h;
}

// Of the threads of a wavefront that have the same two channels one half carries states over wavefronts for the one, the other half for
// the other: this gives both to both.
template <int LANES>
__device__ __forceinline__ void share(float at, float (&h)[2]) { both<LANES>(at, h[0], h[1]); }
template <int LANES>
__device__ __forceinline__ void share(float at, float (&h)[1]) { h[0] = at; }

template <class T, int LANES, bool FACTORS, bool DOCS>
__global__ __launch_bounds__(Team<LANES>::kThreads) void recurrence_kernel(const RecurrenceParams p) {
    constexpr int V = kPack<T>, kWaves = Team<LANES>::kWaves;
    const Seat<T, LANES> seat(p);
    if (!seat.there(p.ranges)) return;
    const int lane = seat.lane, wave = seat.wave, slot = seat.slot;
    __shared__ float2 parts[2][kWaves][LANES * V];  // (by turns: the other one's barrier stands between readers and writers)
    __shared__ float carried[2][LANES * V];         // the state before a tile: who needs it reads it, and the last wavefront leaves the next one
    const int waves = blockDim.x / 64, pick = lane / LANES % V;
    float carry[V];
    first_state<T, LANES, FACTORS, false>(p, seat, p.initial, p.initial_b, carry);
    if (seat.own == 0)
#pragma unroll
        for (int v = 0; v < V; ++v) carried[0][slot + v] = carry[v];
    int turn = 0;
    // From the maps of a tile to its states, and the state behind it.
    auto states = [&](const float (&a)[kSteps][V], const float (&b)[kSteps][V], int begin, Steps<T>& o) {
        float A[V], B[V], preA[V], preB[V], h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            A[v] = a[0][v], B[v] = b[0][v];
#pragma unroll
            for (int k = 1; k < kSteps; ++k) {
                A[v] = grown<FACTORS>(A[v], a[k][v]);
                B[v] = step<FACTORS>(a[k][v], B[v], b[k][v]);
            }
            preA[v] = 1, preB[v] = 0;
            across<LANES, FACTORS, false>(lane, A[v], B[v], preA[v], preB[v]);
            if (lane < LANES) parts[turn][wave][slot + v] = make_float2(A[v], B[v]);
        }
        __syncthreads();
        const float at = over_waves<FACTORS>(0, wave, 1, carried[turn][slot + pick], [&](int w) { return parts[turn][w][slot + pick]; });
        if (wave == waves - 1 && lane < LANES * V) {
            const float2 part = parts[turn][wave][slot + pick];
            carried[turn ^ 1][slot + pick] = onward<FACTORS>(part.x, at, part.y);
        }
        share<LANES>(at, h);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = onward<FACTORS>(preA[v], h[v], preB[v]);
        turn ^= 1;
        if (p.states && seat.own == 0) store_state<V>(p.states, seat.batch * p.states_at.b + (int64_t)(begin / kBlock) * p.states_at.t, seat.c, p.channels, h);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = step<FACTORS>(a[k][v], h[v], b[k][v]);
            o.w[k] = pack<T>(h);
        }
    };
    const Side<T> x_side(p.x, p.x_at, seat), g_side(p.gates, p.gates_at, seat), o_side(p.out, p.out_at, seat);
    struct Tile {
        Steps<T> x, g;
        Documents<LANES> documents;
    };
    const int used = seat.used();
    auto load = [&](Tile& s, int i) {
        const bool there = i < used;
        i = min(i, used - 1);
        const int begin = seat.first + i * kTile;
        x_side.load(s.x, seat, i, p.length - begin, there);
        g_side.load(s.g, seat, i, p.length - begin, there);
        if (DOCS) s.documents.load(p, seat.batch, begin + wave * Documents<LANES>::kPositions + Documents<LANES>::looked_at(lane));
    };
    Tile one;
    if (used > 0) load(one, 0);
    for (int i = 0; i < used; ++i) {
        const int begin = seat.first + i * kTile, count = min(max(seat.length - begin - seat.own, 0), kSteps);
        float a[kSteps][V], b[kSteps][V];
        maps<T, FACTORS>(one.x, one.g, a, b);
        Marks m = {(1u << count) - 1, 0, count};
        if (DOCS) m = one.documents.marks(lane, count);
        mark<V>(m, a, b);
        load(one, i + 1);
        Steps<T> o;
        states(a, b, begin, o);
        hide(m, o);
        o_side.store(o, seat, i, p.length - begin, p.past);
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = carried[turn][slot + v];
    for (int i = used; i < seat.tiles; ++i) {  // behind the sequence
        const int begin = seat.first + i * kTile;
        if (p.states && seat.own == 0)
            store_state<V>(p.states, seat.batch * p.states_at.b + (int64_t)(begin / kBlock) * p.states_at.t, seat.c, p.channels, carry);
        Steps<T> o = {};
        o_side.store(o, seat, i, p.length - begin, p.past);
    }
    if (p.final && seat.own == 0 && seat.range == p.ranges - 1) store_state<V>(p.final, seat.batch * p.final_b, seat.c, p.channels, carry);
}

template <class T, int LANES, bool FACTORS, bool DOCS>
__global__ __launch_bounds__(Team<LANES>::kThreads) void recurrence_backward_kernel(const RecurrenceParams p) {
    constexpr int V = kPack<T>, kWaves = Team<LANES>::kWaves;
    const Seat<T, LANES> seat(p);
    if (!seat.there(p.ranges)) return;
    const int lane = seat.lane, wave = seat.wave, slot = seat.slot;
    __shared__ float2 parts[2][kWaves][LANES * V];
    __shared__ float back_parts[2][kWaves][LANES * V];
    __shared__ float carried[2][LANES * V];  // the gradient of the state behind a tile, as forwards
    const int waves = blockDim.x / 64, pick = lane / LANES % V;
    float carry[V];
    first_state<T, LANES, FACTORS, true>(p, seat, p.final_grad, p.final_grad_b, carry);
    if (seat.own == 0)
#pragma unroll
        for (int v = 0; v < V; ++v) carried[0][slot + v] = carry[v];
    int turn = 0;
    // From a tile's inputs to the gradients of x and gates, in their places.  `more` is called as soon as the inputs are in
    // other registers.  What one instruction makes of them again (b = rest x, with wide rows, whose threads have 128 registers, also the
    // halves of a pack) is not kept from the first walk to the second.
    auto gradients = [&](Steps<T>& x, Steps<T>& g, Steps<T>& d, const float (&state)[V], const Marks& m, auto&& more) {
        float a[kSteps][V], rest[kSteps][V], A[V], B[V], preA[V], preB[V], back[V], behindA[V], behindB[V], h[V], l[V];
        hide(m, x);
        hide(m, d);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            float f[V];
            unpack<T>(g.w[k], f);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (FACTORS) a[k][v] = f[v];
                else sigmoids<T>(f[v], a[k][v], rest[k][v]);
            }
        }
        if (!m.plain())
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    a[k][v] = m.cut >> k & 1 ? 0.f : k < m.count ? a[k][v] : 1.f;
                    if (!FACTORS) rest[k][v] = m.live >> k & 1 ? rest[k][v] : 0.f;
                }
        Steps<T> in = x, gate = g, out_grad = d;
        more();
        auto put_in = [&](int k, float (&b)[V]) {
            unpack<T>(in.w[k], b);
#pragma unroll
            for (int v = 0; v < V; ++v) b[v] = FACTORS ? b[v] : rest[k][v] * b[v];
        };
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1, B[v] = 0, back[v] = 0;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            float b[V];
            put_in(k, b);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A[v] = grown<FACTORS>(A[v], a[k][v]);
                B[v] = step<FACTORS>(a[k][v], B[v], b[v]);
            }
        }
#pragma unroll
        for (int k = kSteps - 1; k >= 0; --k) {
            float f[V];
            unpack<T>(out_grad.w[k], f);
#pragma unroll
            for (int v = 0; v < V; ++v) back[v] = step<FACTORS>(a[k][v], back[v] + f[v], 0.f);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float again = A[v];
            preA[v] = behindA[v] = 1, preB[v] = behindB[v] = 0;
            across<LANES, FACTORS, false>(lane, A[v], B[v], preA[v], preB[v]);
            across<LANES, FACTORS, true>(lane, again, back[v], behindA[v], behindB[v]);
            if (lane < LANES) {
                parts[turn][wave][slot + v] = make_float2(A[v], B[v]);
                back_parts[turn][wave][slot + v] = back[v];
            }
        }
        __syncthreads();
        const int mine = slot + pick;
        const float before = over_waves<FACTORS>(0, wave, 1, pick ? state[V - 1] : state[0], [&](int w) { return parts[turn][w][mine]; });
        const float behind = over_waves<FACTORS>(waves - 1, wave, -1, carried[turn][mine],
                                                 [&](int w) { return make_float2(parts[turn][w][mine].x, back_parts[turn][w][mine]); });
        if (wave == 0 && lane < LANES * V) carried[turn ^ 1][mine] = onward<FACTORS>(parts[turn][0][mine].x, behind, back_parts[turn][0][mine]);
        share<LANES>(before, h);
        share<LANES>(behind, l);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = onward<FACTORS>(preA[v], h[v], preB[v]);
            l[v] = onward<FACTORS>(behindA[v], l[v], behindB[v]);
        }
        turn ^= 1;
        if constexpr (LANES == kWide)  // (unpacked again from here on)
#pragma unroll
            for (int k = 0; k < kSteps; ++k) asm volatile("" : "+v"(in.w[k]), "+v"(out_grad.w[k]));
        // forwards: what a factor's change is worth, the state before (less x, which a gate that is not a factor takes as much from)
        float worth[kSteps][V];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            float f[V];
            unpack<T>(in.w[k], f);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float before = DOCS && (m.cut >> k & 1) ? 0.f : h[v];
                worth[k][v] = FACTORS ? before : before - f[v];
                h[v] = step<FACTORS>(a[k][v], h[v], FACTORS ? f[v] : rest[k][v] * f[v]);
            }
        }
        // backwards
#pragma unroll
        for (int k = kSteps - 1; k >= 0; --k) {
            float dx[V], dg[V], ds[V], own[V];
            unpack<T>(out_grad.w[k], ds);
#pragma unroll
            for (int v = 0; v < V; ++v) own[v] = a[k][v];
            if (DOCS && !FACTORS && (m.cut >> k & 1)) {  // where the state before was dropped, the gate still weighs x
                float gs[V], again;
                unpack<T>(gate.w[k], gs);
#pragma unroll
                for (int v = 0; v < V; ++v) sigmoids<T>(gs[v], own[v], again);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float here = l[v] + ds[v];
                l[v] = step<FACTORS>(a[k][v], here, 0.f);
                dx[v] = FACTORS ? here : here * rest[k][v];
                dg[v] = FACTORS ? here * worth[k][v] : dx[v] * worth[k][v] * own[v];
            }
            x.w[k] = pack<T>(dx);
            g.w[k] = pack<T>(dg);
        }
        hide(m, x);
        hide(m, g);
    };
    const Side<T> x_side(p.x, p.x_at, seat), g_side(p.gates, p.gates_at, seat), d_side(p.out_grad, p.out_grad_at, seat);
    const Side<T> dx_side(p.x_grad, p.x_grad_at, seat), dg_side(p.gates_grad, p.gates_grad_at, seat);
    struct Tile {
        Steps<T> x, g, d;
        float state[V];
        Documents<LANES> documents;
    };
    const int used = seat.used();
    auto load = [&](Tile& s, int i) {
        const bool there = i >= 0;
        i = max(i, 0);
        const int begin = seat.first + i * kTile;
        x_side.load(s.x, seat, i, p.length - begin, there);
        g_side.load(s.g, seat, i, p.length - begin, there);
        d_side.load(s.d, seat, i, p.length - begin, there);
        const float* state = p.states + seat.batch * p.states_at.b + (int64_t)(begin / kBlock) * p.states_at.t + seat.c;
#pragma unroll
        for (int v = 0; v < V; ++v) s.state[v] = state[seat.lone ? 0 : v];
        if (DOCS) s.documents.load(p, seat.batch, begin + wave * Documents<LANES>::kPositions + Documents<LANES>::looked_at(lane));
    };
    for (int i = seat.tiles - 1; i >= used; --i) {  // behind the sequence
        const Steps<T> none = {};
        dx_side.store(none, seat, i, p.length - seat.first - i * kTile, p.past);
        dg_side.store(none, seat, i, p.length - seat.first - i * kTile, p.past);
    }
    Tile one;
    if (used > 0) load(one, used - 1);
    for (int i = used - 1; i >= 0; --i) {
        const int begin = seat.first + i * kTile, count = min(max(seat.length - begin - seat.own, 0), kSteps);
        Marks m = {(1u << count) - 1, 0, count};
        if (DOCS) m = one.documents.marks(lane, count);
        Tile next;
        gradients(one.x, one.g, one.d, one.state, m, [&] { load(next, i - 1); });
        dx_side.store(one.x, seat, i, p.length - begin, p.past);
        dg_side.store(one.g, seat, i, p.length - begin, p.past);
        one = next;
    }
    if (!p.initial_grad || seat.range != 0) return;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = carried[turn][slot + v];
    if (seat.own == 0) store_state<V>(p.initial_grad, seat.batch * p.initial_grad_b, seat.c, p.channels, carry);
}

// What each range of positions does to the state before it (to the gradient behind it where BACK): the map of all its positions.  A
// thread goes through its share of them by itself, and all meet once.
template <class T, int LANES, bool FACTORS, bool DOCS, bool BACK>
__global__ __launch_bounds__(Team<LANES>::kThreads) void recurrence_range_kernel(const RecurrenceParams p) {
    constexpr int V = kPack<T>, kWaves = Team<LANES>::kWaves;
    const Seat<T, LANES> seat(p);
    if (!seat.there(p.ranges - 1)) return;
    const int range = seat.range + BACK;  // the last one has none behind it, the first one none before it
    const int first = range * p.tiles * kTile + seat.own * p.tiles;  // this thread's first position, of tiles * kSteps
    const bool whole = !seat.lone && (range + 1) * p.tiles * kTile <= p.length;
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1, B[v] = 0;
    auto compose = [&](const Steps<T>& x, const Steps<T>& g, const Marks& m) {
        float a[kSteps][V], b[kSteps][V];
        maps<T, FACTORS>(x, g, a, b);
        if (BACK) {
            // b is the gradient that joins here: what comes before it is all that is scaled, h -> a (h + d)
            Steps<T> d = x;
            hide(m, d);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) unpack<T>(d.w[k], b[k]);
        }
        if (!m.plain()) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    a[k][v] = m.cut >> k & 1 ? 0.f : k < m.count ? a[k][v] : 1.f;
                    if (!BACK) b[k][v] = m.live >> k & 1 ? b[k][v] : 0.f;
                }
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int k = BACK ? kSteps - 1 - i : i;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                B[v] = BACK ? step<FACTORS>(a[k][v], B[v] + b[k][v], 0.f) : step<FACTORS>(a[k][v], B[v], b[k][v]);
                A[v] = grown<FACTORS>(A[v], a[k][v]);
            }
        }
    };
    const Rows other_at = BACK ? p.out_grad_at : p.x_at;
    const char* other = (const char*)(BACK ? p.out_grad : p.x) + (seat.batch * other_at.b + seat.c) * (int64_t)sizeof(T);
    const char* gates = (const char*)p.gates + (seat.batch * p.gates_at.b + seat.c) * (int64_t)sizeof(T);
    const int64_t other_step = other_at.t * (int64_t)sizeof(T), gates_step = p.gates_at.t * (int64_t)sizeof(T);
    auto load = [&](Steps<T>& s, const char* from, int64_t step, int t) {
        if (whole) {
            from += t * step;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) s.w[k] = ((const Word<T>*)(from + k * step))->w;
        } else {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const char* at = from + min(t + k, p.length - 1) * step;
                s.w[k] = seat.lone ? *(const unsigned short*)at : ((const Word<T>*)at)->w;
            }
        }
    };
    // What lies before the last position where the state is dropped (behind the first one, backwards) does not show in the range's map: a
    // wavefront without others passes on what it gets, as one behind the sequence does (both passes of 32768 positions of 2048 channels in f32 with
    // documents of 700: 644 us, and 709 if it reads them all; with one document alone looking for them costs 5 us).
    const int begin = range * p.tiles * kTile, mine = seat.wave * Team<LANES>::kSpread * kSteps * p.tiles;
    bool shows = begin + mine < seat.length;
    if (DOCS) {
        __shared__ int edge;
        if (threadIdx.x == 0) edge = BACK ? p.length : -1;
        __syncthreads();
        const int* documents = p.documents + seat.batch * p.documents_at.b;
        for (int t = begin + threadIdx.x; t < min(begin + p.tiles * kTile, seat.length); t += Team<LANES>::kThreads) {
            const int here = documents[t * p.documents_at.t], before = documents[max(t - 1, 0) * p.documents_at.t];
            if (here < 0 || here != before) BACK ? atomicMin(&edge, t) : atomicMax(&edge, t);
        }
        __syncthreads();
        const int at = __builtin_amdgcn_readfirstlane(edge) - begin - mine;
        shows = shows && (BACK ? at >= 0 : at < Team<LANES>::kSpread * kSteps * p.tiles);
    }
    for (int i = 0; i < p.tiles && shows; ++i) {
        const int t = first + (BACK ? p.tiles - 1 - i : i) * kSteps, count = min(max(seat.length - t, 0), kSteps);
        Steps<T> x, g;
        load(x, other, other_step, t);
        load(g, gates, gates_step, t);
        Marks m = {(1u << count) - 1, 0, count};
        if (DOCS) {
            Documents<LANES> d;
            const int at = Documents<LANES>::looked_at(seat.lane);  // of as many positions, but those of each thread are `tiles` as far apart
            d.load(p, seat.batch, t - seat.own * p.tiles + (seat.wave * Team<LANES>::kSpread + at / kSteps) * kSteps * p.tiles + at % kSteps);
            m = d.marks(seat.lane, count);
        }
        compose(x, g, m);
    }
    __shared__ float2 parts[kWaves][LANES * V];
    float preA = 1, preB = 0;  // (of no use here)
#pragma unroll
    for (int v = 0; v < V; ++v) {
        across<LANES, FACTORS, BACK>(seat.lane, A[v], B[v], preA, preB);
        if (seat.lane < LANES) parts[seat.wave][seat.slot + v] = make_float2(A[v], B[v]);
    }
    __syncthreads();
    if (seat.own != 0) return;
    if (seat.range == 0) {
        float given[V];
        load_state<V>(BACK ? p.final_grad : p.initial, seat.batch * (BACK ? p.final_grad_b : p.initial_b), seat.c, p.channels, given);
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (seat.c + v < p.channels) p.carry[aside<BACK>(p) + seat.state + v] = make_float2(0, given[v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float a = 1, b = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float2 part = parts[BACK ? kWaves - 1 - i : i][seat.slot + v];
            b = onward<FACTORS>(part.x, b, part.y);
            a = together<FACTORS>(a, part.x);
        }
        if (seat.c + v < p.channels) p.carry[(int64_t)range * p.batch * p.channels + seat.state + v] = make_float2(a, b);
    }
}

// Few positions, as a decoder takes them one by one: a lane goes through those of its channels by itself.  A lone last channel belongs to
// one lane alone (in place, a pack of two would read what its neighbour may already have written).
template <class T, bool FACTORS>
__global__ __launch_bounds__(256) void recurrence_step_kernel(const RecurrenceParams p) {
    constexpr int V = kPack<T>;
    const unsigned packs = (unsigned)((p.channels + V - 1) / V);
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, batch = at / packs;
    if (batch >= p.batch) return;
    const int c = (int)(at - batch * packs) * V;
    const bool lone = c + V > p.channels;
    const int length = p.lengths ? min(max(p.lengths[batch * p.lengths_b], 0), p.length) : p.length;
    const auto address = [&](const void* from, const Rows& rows, int t) { return (char*)from + (batch * rows.b + t * rows.t + c) * (int64_t)sizeof(T); };
    Steps<T> x = {}, g = {};
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
        if (k < p.length) {
            const char *from = address(p.x, p.x_at, k), *gate = address(p.gates, p.gates_at, k);
            x.w[k] = lone ? *(const unsigned short*)from : ((const Word<T>*)from)->w;
            g.w[k] = lone ? *(const unsigned short*)gate : ((const Word<T>*)gate)->w;
        }
    float h[V];
    load_state<V>(p.initial, batch * p.initial_b, c, p.channels, h);
    if (p.states) store_state<V>(p.states, batch * p.states_at.b, c, p.channels, h);
    Marks m = {(1u << length) - 1, 0, length};
    if (p.documents) {
        const int* from = p.documents + batch * p.documents_at.b;
        int before = from[0];
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
            if (k < length) {
                const int here = from[k * p.documents_at.t];
                m.live &= ~((unsigned)(here < 0) << k);
                m.cut |= (unsigned)(here < 0 || here != before) << k;
                before = here;
            }
    }
    float a[kSteps][V], b[kSteps][V];
    maps<T, FACTORS>(x, g, a, b);
    mark<V>(m, a, b);
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
        if (k < p.length) {
            float o[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = step<FACTORS>(a[k][v], h[v], b[k][v]);
                o[v] = m.live >> k & 1 ? h[v] : 0.f;
            }
            char* to = address(p.out, p.out_at, k);
            const unsigned w = pack<T>(o);
            if (lone) *(unsigned short*)to = (unsigned short)w;
            else ((Word<T>*)to)->w = w;
        }
    if (p.final) store_state<V>(p.final, batch * p.final_b, c, p.channels, h);
}

// Wide rows bring whole cache lines: a tenth and more, forward and backward in f32.  The backward pass of bf16, and that of documents, does not fit
// the 128 registers that their 1024 threads have: 16 x 1000 positions of 4000 channels in bf16 with documents 275 us wide and 184 narrow.
constexpr bool wide_pays(int type, bool backward, bool documents) { return !backward || (type == ADHIP_F32 && !documents); }

template <class T, int LANES, bool FACTORS, bool DOCS>
void launch_recurrence(const char* op, const RecurrenceParams& p, bool backward, hipStream_t stream) {
    const unsigned threads = (unsigned)Team<LANES>::threads(p.length);
    const auto blocks = [&](int ranges) { return (unsigned)(((int64_t)p.groups * p.batch * ranges + 7) / 8 * 8); };
    if (!backward) {
        if (p.ranges > 1) launch(op, recurrence_range_kernel<T, LANES, FACTORS, DOCS, false>, blocks(p.ranges - 1), Team<LANES>::kThreads, stream, p);
        launch(op, recurrence_kernel<T, LANES, FACTORS, DOCS>, blocks(p.ranges), threads, stream, p);
    }
    if constexpr (LANES == kNarrow || wide_pays(sizeof(T) == 4 ? ADHIP_F32 : ADHIP_BF16, true, DOCS))
        if (backward) {
            if (p.ranges > 1) launch(op, recurrence_range_kernel<T, LANES, FACTORS, DOCS, true>, blocks(p.ranges - 1), Team<LANES>::kThreads, stream, p);
            launch(op, recurrence_backward_kernel<T, LANES, FACTORS, DOCS>, blocks(p.ranges), threads, stream, p);
        }
}

template <class T, int LANES>
void launch_recurrence(const char* op, const RecurrenceParams& p, bool backward, bool factors, hipStream_t stream) {
    if (factors && p.documents) launch_recurrence<T, LANES, true, true>(op, p, backward, stream);
    else if (factors) launch_recurrence<T, LANES, true, false>(op, p, backward, stream);
    else if (p.documents) launch_recurrence<T, LANES, false, true>(op, p, backward, stream);
    else launch_recurrence<T, LANES, false, false>(op, p, backward, stream);
}

// How channels are cut into rows and positions into ranges.  Compute units left without a workgroup are given ranges of positions, at
// the price of a kernel that reads them before (8191 positions of 1000 channels in f32, forward and backward: 185 us in one range, 107 in four), of
// two tiles or more each.  Rows are wide where narrow ones would give some compute units two workgroups (4 x 2049 of 2560 in bf16: 56 us
// narrow, 44 wide; 2 x 8192 of 4096, where they give each one: 285 narrow, 328 wide), and where there are ranges of four
// tiles and more to make up for them (the first example in eight: 103 us; 4096 positions of 1024 channels in bf16, two tiles each, forward: 16 narrow, 20 wide).
struct Cut {
    int lanes, groups, tiles, ranges;  // tiles: of a range
    Cut(const adhip_array& x, bool wide) {
        const int64_t v = 4 / type_bytes(x.type), channels = x.dims[2], batch = std::max<int64_t>(x.dims[0], 1);
        const int64_t all = (x.dims[1] + kTile - 1) / kTile;
        const auto blocks = [&](int lanes) { return std::max<int64_t>((channels + lanes * v - 1) / (lanes * v) * batch, 1); };
        const bool many = blocks(kNarrow) > kFull, long_ranges = 2 * blocks(kNarrow) <= kFull && all * blocks(kWide) >= 4 * kFull;
        lanes = wide && (many || long_ranges) ? kWide : kNarrow;
        groups = (int)((channels + lanes * v - 1) / (lanes * v));
        const int64_t want = std::max<int64_t>(1, std::min<int64_t>(kFull / blocks(lanes), all / 2));
        tiles = (int)std::max<int64_t>(1, (all + want - 1) / want);
        ranges = (int)std::max<int64_t>(1, (all + tiles - 1) / tiles);
    }
    size_t workspace(const adhip_array& x) const { return ranges == 1 ? 0 : (size_t)ranges * (size_t)x.dims[0] * (size_t)x.dims[2] * sizeof(float2); }
};

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
    return {a.strides[0], a.dims[1] > 1 ? a.strides[1] : 0};  // (one position alone is not apart from any)
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

// What is written takes the place of an input, element by element, or shares no memory with any.
void check_shared(const char* op, const adhip_recurrence_args& g, bool backward) {
    const auto in_place = [&](const char* in_name, const adhip_array& in, const char* out_name, const adhip_array& out) {
        if (in.data && out.data) check_in_place(op, in_name, in, out_name, out);
    };
    if (backward) {
        ADHIP_CHECK(g.x.dims[1] == 0 || g.x_grad.data != g.gates_grad.data, "%s: x_grad and gates_grad are one array", op);
        for (const auto& [out_name, out] : {std::pair("x_grad", &g.x_grad), std::pair("gates_grad", &g.gates_grad)}) {
            in_place("x", g.x, out_name, *out);
            in_place("gates", g.gates, out_name, *out);
            in_place("out_grad", g.out_grad, out_name, *out);
        }
        check_apart(op, "x_grad", g.x_grad, "gates_grad", g.gates_grad);
        in_place("final_grad", g.final_grad, "initial_grad", g.initial_grad);
    } else {
        in_place("x", g.x, "out", g.out);
        in_place("gates", g.gates, "out", g.out);
        in_place("initial", g.initial, "final", g.final);
    }
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
    for (const Rows* at : {&p.x_at, &p.gates_at, &p.out_at, &p.out_grad_at, &p.x_grad_at, &p.gates_grad_at})
        ADHIP_CHECK(at->t <= (1 << 21), "%s: positions %lld elements apart, at most 2^21 are wanted", op, (long long)at->t);
    const Cut cut(g.x, wide_pays(g.x.type, backward, g.documents.data != nullptr));
    p.length = (int)length;
    p.channels = (int)channels;
    p.batch = (int)batch;
    p.groups = cut.groups;
    p.ranges = cut.ranges;
    p.tiles = cut.tiles;
    const int64_t blocks = batch * p.groups;
    const bool factors = g.factors != 0, wide = cut.lanes == kWide;
    const auto whole_lines = [&](const adhip_array& a) {
        const int64_t w = type_bytes(a.type);
        return (uintptr_t)a.data % 128 == 0 && a.strides[0] * w % 128 == 0 && a.strides[1] * w % 128 == 0;
    };
    p.near = !wide || !whole_lines(g.x) || !whole_lines(g.gates);
    // (4 x 2048 positions of 4096 channels in f32, both passes: 215 us past the caches, 232 through them.  Half lines, as narrow rows write them,
    // cost a quarter more traffic past the caches, at the same time.)
    p.past = wide && (backward ? 5 : 3) * batch * length * channels * type_bytes(g.x.type) > kLastCache;
    if (!backward && length >= 1 && length <= kSteps) {
        const int64_t v = 4 / type_bytes(g.x.type), lanes = batch * ((channels + v - 1) / v);
        ADHIP_CHECK(fits_launch((lanes + 255) / 256, 256), "%s: %lld sequences of %lld channels are too many for one call", op, (long long)batch, (long long)channels);
        if (lanes == 0) return;
        check_shared(op, g, backward);
        launch(op, g.x.type == ADHIP_BF16 ? (factors ? recurrence_step_kernel<bf16, true> : recurrence_step_kernel<bf16, false>)
                                          : (factors ? recurrence_step_kernel<float, true> : recurrence_step_kernel<float, false>),
               (unsigned)((lanes + 255) / 256), 256, stream, p);
        return;
    }
    ADHIP_CHECK(fits_launch(blocks * cut.ranges + 8, (unsigned)(wide ? Team<kWide>::threads(p.length) : Team<kNarrow>::threads(p.length))), "%s: %lld sequences of %lld channels are too many for one call", op, (long long)batch, (long long)channels);
    if (blocks == 0) return;
    ADHIP_CHECK(cut.workspace(g.x) == 0 || (g.workspace && (uintptr_t)g.workspace % 16 == 0 && g.workspace_bytes >= cut.workspace(g.x)),
                "%s: the workspace has %zu bytes, %zu are wanted, aligned to 16", op, g.workspace ? g.workspace_bytes : (size_t)0, cut.workspace(g.x));
    check_shared(op, g, backward);
    p.carry = (float2*)g.workspace;
    if (g.x.type == ADHIP_BF16 && wide) launch_recurrence<bf16, kWide>(op, p, backward, factors, stream);
    else if (g.x.type == ADHIP_BF16) launch_recurrence<bf16, kNarrow>(op, p, backward, factors, stream);
    else if (wide) launch_recurrence<float, kWide>(op, p, backward, factors, stream);
    else launch_recurrence<float, kNarrow>(op, p, backward, factors, stream);
}

}  // namespace
}  // namespace adhip

extern "C" {

int adhip_recurrence_workspace(adhip_ctx* ctx, const adhip_recurrence_args* args, int backward, size_t* bytes) {
    return adhip::context_guarded(ctx, [&] {
        const char* op = "adhip_recurrence_workspace";
        ADHIP_CHECK(args && bytes, "%s: no arguments", op);
        adhip::check_x(op, args->x);
        *bytes = std::max(adhip::Cut(args->x, true).workspace(args->x), adhip::Cut(args->x, false).workspace(args->x));
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

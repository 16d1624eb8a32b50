// Attention on device arrays: what its kernels share.
//
// All heads that share a key head are worked on together: row r = i G + g of key head c is query i of head c G + g, so that
// a tile of rows reads its keys once for the whole group and the gradients of keys and values sum over the group by
// themselves.
//
// Every product is a tile of 32 x 32 on the matrix cores, contracted 16 at a time: A[i = lane % 32][k], B[k][j = lane % 32],
// where a lane holds k = 8 (lane / 32) .. + 7, and C[8 g + 4 (lane / 32) + e][lane % 32] in its register 4 g + e.  The order of
// k is free as long as A and B agree, so registers 8 s .. 8 s + 7 of a C tile are, as they stand, the B operand of a product
// over its rows 16 s .. + 15: scores become the operand of the next product without leaving their lanes.  Its A operand
// takes rows 16 s + 4 (lane / 32) + {0..3, 8..11} of the column lane % 32: the transposing reads of LDS for 16-bit
// types, single words for 32-bit ones.
#pragma once
#include "operators.hpp"

namespace adhip {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRange = 32;  // positions that share an entry of the document ranges

struct Tensor {
    const void* data;
    int64_t b, l, h;  // strides in elements
    int vec;          // rows begin at multiples of 16 bytes and hold whole pieces of 16 bytes
};

struct Params {
    Tensor q, k, v, out, dout, dq, dk, dv;  // out: written by the forward kernels, read by the backward ones
    Tensor q3, k3, v3, dout3;               // f32 in parts: three planes of bf16, q_plane or k_plane elements apart,
    int64_t q_plane, k_plane;               // rows of D3 features, the last of them zeros
    int D3;
    float* lse;
    int64_t lse_b, lse_l, lse_h;
    const float* slopes;
    int64_t slope_stride;
    const int *lengths, *prefix, *qdoc, *kdoc;
    int64_t lengths_s, prefix_s, qdoc_b, qdoc_l, kdoc_b, kdoc_l;
    const int2 *qrange, *krange;  // the range of documents of every kRange positions (document_range)
    int qranges, kranges;         // entries of a sequence
    int B, Lq, Lk, Hk, G, D, R;   // R = Lq G rows
    float scale, cap;
    int causal, window;
    int tiles, splits;            // row tiles (or key tiles); ranges that the keys (or rows) are split into
    float *part, *part_ml;        // forward, split: [split][b][c][row][D], [..][row][2]
    float* stats;                 // backward, [2][b][head][query]: lse log2 e (+inf: sees nothing), -delta
    float *part_dq, *part_dk, *part_dv;  // backward, split: [split] of what the gradients are, packed [b][c][row or key][D]
    int dq_splits, dk_splits;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Ways to multiply: the type of arrays (IO) and of elements in LDS (E), the operand as loaded (Raw) and as multiplied.
//   bf16   one instruction for 16 of k
//   float  FP32 matrix cores, eight instructions of 64 cycles each
//   Parts  f32 as the sum of three bf16 parts (24 bits: exactly), six products of parts on the bf16 matrix cores, what is
//          left out being 2^-24 of the product: 192 cycles instead of 512.  Tiles hold three planes of parts, which a kernel
//          of its own has made of the arrays, once for all workgroups.
//   Split  the same with f32 in LDS, split where an operand is read: for keys that are read by one wavefront only.
// Infinities lose their sign in the parts' products: where one is seen, the result is NaN.
struct Parts {};
struct Split {};
struct Frag3 {
    bf16x8 p[3];
};
template <class X>
struct Matrix;
template <>
struct Matrix<bf16> {
    typedef bf16 IO;
    typedef bf16 E;
    typedef bf16x8 Raw;
    typedef bf16x8 Frag;
    static constexpr int kChunk = 8, kPlanes = 1;  // elements of 16 bytes; tiles that make one
    static constexpr bool kAside = true;           // (keep_aside)
    static constexpr bool kFine = false;           // (tanh_of)
    static __device__ __forceinline__ Frag operand(const Raw& x) { return x; }
    static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Matrix<float> {
    typedef float IO;
    typedef float E;
    typedef f32x8 Raw;
    typedef f32x8 Frag;
    static constexpr int kChunk = 4, kPlanes = 1;
    static constexpr bool kAside = false;  // used where sums fill that half
    static constexpr bool kFine = true;
    static __device__ __forceinline__ Frag operand(const Raw& x) { return x; }
    static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};
struct MatrixInParts {
    typedef float IO;
    typedef f32x8 Raw;
    typedef Frag3 Frag;
    static constexpr bool kAside = true, kFine = true;
    static __device__ __forceinline__ Frag operand(const Raw& x) {
        Frag f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bf16 hi = (bf16)x[e];
            const float r = x[e] - (float)hi;
            const bf16 mid = (bf16)r;
            f.p[0][e] = hi;
            f.p[1][e] = mid;
            f.p[2][e] = (bf16)(r - (float)mid);
        }
        return f;
    }
    // the smallest products first
    static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
    }
};
template <>
struct Matrix<Parts> : MatrixInParts {
    typedef bf16 E;
    static constexpr int kChunk = 8, kPlanes = 3;
};
template <>
struct Matrix<Split> : MatrixInParts {
    typedef float E;
    static constexpr int kChunk = 4, kPlanes = 1;
};

// Tiles in LDS: rows of DP features in pieces of 16 bytes, whose places within a row are exchanged by an exclusive or
// with bits of the row's number.  16 rows at one piece (an operand whose rows are rows of the tile) then lie in all 64
// banks, and so do 4 rows at four pieces (the transposing reads): 230 and 200 bytes a clock, where rows padded by 16 bytes
// give the first 230 and the second 62, unpadded ones 16 and less.  The exchange costs one instruction an address, and
// pieces keep places of 16 bytes, so that loads can go to LDS without passing through registers.
template <class E, int DP>
struct Lds {
    static constexpr int kPieces = DP * (int)sizeof(E) / 16;
    static constexpr int kPlaces = kPieces == 12 ? 16 : kPieces;  // the exchange wants a power of two in each row
    static constexpr int kPitch = kPlaces * 16;                   // bytes
    static __device__ __forceinline__ constexpr int swap(int row) {
        if (kPlaces % 16 == 0) return (row & 3) << 2 | (row >> 2 & 3);
        if (kPlaces % 8 == 0) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
        return row >> 2 & 3;
    }
    static constexpr int kSwapped = kPlaces % 16 == 0 ? 15 : kPlaces % 8 == 0 ? 7 : 3;  // bits of a piece's number that are
    static __device__ __forceinline__ constexpr int at(int row, int piece) { return row * kPitch + (piece ^ swap(row)) * 16; }
    // From the address of (row, piece) to that of (row + rows, piece + pieces), where neither addition carries: the exchange is
    // linear in the bits.
    static __device__ __forceinline__ constexpr unsigned step(unsigned from, int rows, int pieces) {
        return (from ^ (unsigned)((swap(rows) ^ pieces) & kSwapped) * 16u) + (unsigned)((pieces & ~kSwapped) * 16 + rows * kPitch);
    }
};

// Addresses in LDS as numbers
template <class V>
__device__ __forceinline__ V lds_read(unsigned at) {
    return *(__attribute__((address_space(3))) const V*)(uintptr_t)at;
}
__device__ __forceinline__ unsigned lds_address(const void* p) { return (unsigned)(uintptr_t)p; }  // (it ends in the offset)

// Where a lane's part of an operand begins in a tile: the operand's other parts are an exclusive or and a fixed offset away.
// `here` keeps the compiler from computing all of them ahead of a loop, where they would fill registers.
__device__ __forceinline__ unsigned here(unsigned x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// Holds an operand that stays in the half of the registers that only matrix instructions reach, where one wavefront has all
// of a SIMD's: the other half is left to sums and scores, which vector instructions work on.
__device__ __forceinline__ void keep_aside(bf16x8& f) {
    f32x4 x = __builtin_bit_cast(f32x4, f);
    asm volatile("" : "+a"(x));
    f = __builtin_bit_cast(bf16x8, x);
}
__device__ __forceinline__ void keep_aside(f32x8& f) { asm volatile("" : "+a"(f)); }
__device__ __forceinline__ void keep_aside(Frag3& f) {
#pragma unroll
    for (int i = 0; i < 3; ++i) keep_aside(f.p[i]);
}

// A (or B) operand whose rows are rows of a tile of ROWS rows: rows row0 .. + 31 (row0 a multiple of 16), features 16 step ..
// + 15; `from`: the tile's address + rows_lane()
template <class X, int DP>
__device__ __forceinline__ unsigned rows_lane(int lane) {
    typedef typename Matrix<X>::E E;
    return (unsigned)Lds<E, DP>::at(lane & 31, (lane >> 5) * (int)sizeof(E) / 2);
}
template <class X, int DP, int ROWS>
__device__ __forceinline__ typename Matrix<X>::Frag rows_frag(unsigned from, int row0, int step) {
    typedef Matrix<X> M;
    typedef Lds<typename M::E, DP> L;
    if constexpr (sizeof(typename M::E) == 2) {
        typename M::Frag f;
#pragma unroll
        for (int i = 0; i < M::kPlanes; ++i) ((f32x4*)&f)[i] = lds_read<f32x4>(L::step(from, row0 + i * ROWS, 2 * step));
        return f;
    } else {
        typename M::Raw f;
#pragma unroll
        for (int i = 0; i < 2; ++i) ((f32x4*)&f)[i] = lds_read<f32x4>(L::step(from, row0, 4 * step + i));
        return M::operand(f);
    }
}

// A operand whose rows are features d0 .. + 31 of the tile and whose k are its rows k0 .. + 15 (a multiple of 16), in the order
// of C's registers; `from`: the tile's address + cols_lane()
template <class X, int DP>
__device__ __forceinline__ unsigned cols_lane(int lane) {
    typedef typename Matrix<X>::E E;
    if (sizeof(E) == 2)
        return (unsigned)Lds<E, DP>::at(4 * (lane >> 5) + ((lane & 15) >> 2), (lane >> 4 & 1) * 2 + (lane >> 1 & 1)) + 8 * (lane & 1);
    return (unsigned)Lds<E, DP>::at(4 * (lane >> 5), (lane & 31) >> 2) + 4 * (lane & 3);
}
template <class X, int DP, int ROWS>
__device__ __forceinline__ typename Matrix<X>::Frag cols_frag(unsigned from, int k0, int d0) {
    typedef Matrix<X> M;
    typedef Lds<typename M::E, DP> L;
    if constexpr (sizeof(typename M::E) == 2) {
        typedef __attribute__((address_space(3))) s16x4* Ptr;
        typename M::Frag f;
#pragma unroll
        for (int i = 0; i < M::kPlanes; ++i) {
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(uintptr_t)L::step(from, k0 + i * ROWS, d0 / 8));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(uintptr_t)L::step(from, k0 + 8 + i * ROWS, d0 / 8));
            ((s16x8*)&f)[i] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return f;
    } else {
        typename M::Raw r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = lds_read<float>(L::step(from, k0 + (e & 3) + 2 * (e & 4), d0 / 4));
        return M::operand(r);
    }
}

// registers 8 s .. + 7 of a C tile as a B operand.  Probabilities and score gradients are rounded to the operands' type
// here, as the matrix cores take them; sums of probabilities are taken before.  In bf16 that makes the error of a result 0.0023
// to 0.0024 of its norm, 0.0017 of which is the rounding of the result itself; two parts would take these products twice.
__device__ __forceinline__ void to_frag(const f32x16& c, int s, bf16x8& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (bf16)c[8 * s + e];
}
__device__ __forceinline__ void to_frag(const f32x16& c, int s, f32x8& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c[8 * s + e];
}
__device__ __forceinline__ void to_frag(const f32x16& c, int s, Frag3& f) {
    f32x8 x;
    to_frag(c, s, x);
    f = MatrixInParts::operand(x);
}

// 16 bytes of a row of D features from d on; what lies behind the row's end is zero.  VEC: rows begin at multiples of 16
// bytes and hold whole pieces of 16 bytes; otherwise element by element.
template <bool VEC, class T>
__device__ __forceinline__ uint4 load_chunk(const T* row, int d, int D) {
    uint4 r = {0, 0, 0, 0};
    if (VEC) {
        if (d < D) r = *(const uint4*)(row + d);
    } else {
        T t[Matrix<T>::kChunk];
#pragma unroll
        for (int e = 0; e < Matrix<T>::kChunk; ++e) t[e] = d + e < D ? row[d + e] : (T)0.f;
        r = *(uint4*)t;
    }
    return r;
}

// the stationary operand of a product: eight features of one row of an array
template <bool VEC, class T>
__device__ __forceinline__ typename Matrix<T>::Raw load_frag(const T* row, int d, int D, bool valid) {
    typename Matrix<T>::Raw f;
    uint4* u = (uint4*)&f;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(f) / 16); ++i)
        u[i] = valid ? load_chunk<VEC>(row, d + i * Matrix<T>::kChunk, D) : uint4{0, 0, 0, 0};
    return f;
}

// Four features of a row from registers, in the array's type
template <class T>
__device__ __forceinline__ void store4(T* row, int d, int D, int vec, const float (&f)[4]) {
    if (vec) {
        if (d < D) {
            Pack<T, 4> p;
#pragma unroll
            for (int e = 0; e < 4; ++e) p.v[e] = (T)f[e];
            *(Pack<T, 4>*)(row + d) = p;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < D) row[d + e] = (T)f[e];
    }
}

// tanh(x) from y = 2 x log2 e: what a capped score takes, in units of the cap.  To about 1.5e-7; FINE, for f32, also in
// relation to small values, where scores mostly lie: by the series below 0.3, 5e-8 of the value.
template <bool FINE>
__device__ __forceinline__ float tanh_of(float y) {
    const float e = __builtin_amdgcn_exp2f(y), far = __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
    if (!FINE) return far;
    const float x = y * (0.5f * kLn2), t = x * x;
    const float near = __builtin_fmaf(
        x * t, __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), x);
    return t < 0.09f ? near : far;
}

// The larger (the sum) of a lane's value and that of the lane 32 away, in both.
__device__ __forceinline__ float max_of_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// row of register i of a C tile
__device__ __forceinline__ constexpr int c_row(int i) { return 8 * (i >> 2) + (i & 3); }

// How raw products become scores in units of log 2: tanh(raw bend) where they are capped, then times unit, then the
// distance's part.
struct Scoring {
    float bend, unit;  // 2 log2 e scale / cap; cap log2 e, or scale log2 e
    __device__ __forceinline__ explicit Scoring(const Params& p)
        : bend(p.cap > 0.f ? 2.f * kLog2e * p.scale / p.cap : 0.f), unit((p.cap > 0.f ? p.cap : p.scale) * kLog2e) {}
};

// Positions that a query sees: j < n and (j < prefix or lo <= j <= hi).  lo and hi by the query's own position.
struct Band {
    int below, above;  // lo = at - below, hi = at + above; where there is no limit, more than any position
    __device__ __forceinline__ explicit Band(const Params& p) {
        constexpr int kAll = 1 << 30;
        below = p.window ? p.window - 1 : kAll;
        above = p.causal ? 0 : below;
    }
};

// What a lane's row sees of a run of keys, by the run's ends: a wavefront whose rows all see everything skips the masks, one
// whose rows each see all or nothing takes one choice a row.  Rows that matter to nobody (`idle`: behind the last one, of no
// document) see everything, so that they keep no wavefront from that; their results are replaced at the end.
struct Sight {
    int lo, hi, pre, doc;  // hi below the sequence's end
    bool idle;
    __device__ __forceinline__ bool all(int first, int last, bool documents, int2 theirs) const {
        return idle || (((lo <= first && last <= hi) || last < pre) && (!documents || (theirs.x == doc && theirs.y == doc)));
    }
    __device__ __forceinline__ bool none(int first, int last, bool documents, int2 theirs) const {
        return ((last < lo || first > hi) && first >= pre) || (documents && (doc < (theirs.x < 0 ? ~theirs.x : theirs.x) || doc > theirs.y));
    }
    __device__ __forceinline__ bool sees(int j) const { return (unsigned)(j - lo) <= (unsigned)(hi - lo) || j < pre; }
};

__device__ __forceinline__ int sequence_length(const Params& p, int b) {
    const int n = p.lengths ? p.lengths[b * p.lengths_s] : p.Lk;
    return min(max(n, 0), p.Lk);
}

// Smallest and largest document (of those from 0 on) of some positions: x, y; x is its complement, and so negative, where
// some of the positions belong to none.
__device__ __forceinline__ int2 document_range(const int2* ranges, int first, int last) {
    int2 r = {0x7fffffff, -1};
    int none = 0;
    for (int i = first / kRange; i <= last / kRange; ++i) {
        const int2 x = ranges[i];
        none |= x.x;
        r.x = min(r.x, x.x < 0 ? ~x.x : x.x);
        r.y = max(r.y, x.y);
    }
    if (none < 0) r.x = ~r.x;
    return r;
}
__device__ __forceinline__ bool documents_meet(int2 a, int2 b) {
    return (a.x < 0 ? ~a.x : a.x) <= b.y && (b.x < 0 ? ~b.x : b.x) <= a.y;
}

// Walks the tiles begin .. stop - 1 that a block needs, 64 candidates at a time: each lane decides on one, all wavefronts
// alike.  Of those needed, split s of S takes numbers s, s + S, ..: the splits' shares are even whatever the masks leave.
// needed(tile, documents) also tells the smallest and largest document of the tile (where there are any).
struct Tile {
    int t;           // -1: none
    int2 documents;
};
template <class Needed>
struct Tiles {
    const Needed& needed;
    int base, end, split, splits, lane, seen = 0;
    unsigned long long mask = 0;
    int2 documents = {0, 0};
    __device__ __forceinline__ Tiles(const Needed& f, int begin, int stop, int split_, int splits_, int lane_)
        : needed(f), base(begin - 64), end(stop), split(split_), splits(splits_), lane(lane_) {}
    __device__ __forceinline__ Tile next() {
        while (!mask) {
            if (base + 64 >= end) return {-1, {0, 0}};
            base += 64;
            const bool mine = base + lane < end && needed(base + lane, documents);
            mask = __ballot(mine);
            if (splits > 1) {
                const int number = seen + __popcll(mask & ((1ull << lane) - 1));
                seen += __popcll(mask);
                mask = __ballot(mine && number % splits == split);
            }
        }
        const int i = __builtin_ctzll(mask);
        mask &= mask - 1;
        return {base + i, {__builtin_amdgcn_readlane(documents.x, i), __builtin_amdgcn_readlane(documents.y, i)}};
    }
};

// A ring of BUFS tiles in LDS: the oldest is worked on while the others are under way.  `start(tile, buffer)` begins a
// tile's loads, of which the last LOADS of each wavefront are its own; `landed(tile, buffer)` runs when it is there and all
// wavefronts have come.  A load takes one to two microseconds from other memory than the L2, as long as the products of a
// tile where a compute unit has few wavefronts: then two and three tiles under way are worth their LDS (causal, 2 x 4096 x 16
// heads of 128, one under way and waited for as a whole: 175 us forward, 676 backward; so: 166, 559).
template <int BUFS, int LOADS, class Walk, class Start>
struct Ring {
    Walk& walk;
    const Start& start;
    Tile queue[BUFS];  // queue[0]: the one worked on
    int buf = 0;       // its place
    __device__ __forceinline__ Ring(Walk& w, const Start& s) : walk(w), start(s) {
        queue[0] = walk.next();
        if (BUFS > 1 && queue[0].t >= 0) start(queue[0], 0);
#pragma unroll
        for (int i = 1; i < BUFS - 1; ++i) {
            queue[i] = queue[i - 1].t >= 0 ? walk.next() : Tile{-1, {0, 0}};
            if (queue[i].t >= 0) start(queue[i], i);
        }
    }
    // waits for queue[0], then begins one more
    __device__ __forceinline__ bool ready() {
        if (queue[0].t < 0) return false;
        if (BUFS == 1) {
            __syncthreads();
            start(queue[0], 0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            return true;
        }
        if (BUFS > 2 && queue[BUFS > 2 ? BUFS - 2 : 0].t >= 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((BUFS - 2) * LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        return true;
    }
    __device__ __forceinline__ void more() {
        if (BUFS == 1) return;
        Tile& last = queue[BUFS - 1];
        last = BUFS == 2 || queue[BUFS > 2 ? BUFS - 2 : 0].t >= 0 ? walk.next() : Tile{-1, {0, 0}};
        if (last.t >= 0) start(last, buf == 0 ? BUFS - 1 : buf - 1);
    }
    __device__ __forceinline__ void pop() {
        if (BUFS == 1) {
            queue[0] = walk.next();
            return;
        }
#pragma unroll
        for (int i = 0; i + 1 < BUFS; ++i) queue[i] = queue[i + 1];
        buf = buf + 1 == BUFS ? 0 : buf + 1;
    }
};

// What a workgroup works on.  Workgroups are given out in the order of their numbers, to the eight dies in turn: numbers run
// over key heads and sequences first, so that a key head stays on as few dies as their count allows (one, where it is a
// multiple of eight) and its keys in their L2, and over tiles from the longest walk to the shortest, so that the short ones
// fill the end.
struct Place {
    int tile, split, c, b;
    __device__ __forceinline__ Place(const Params& p, int splits) {
        unsigned id = blockIdx.x;
        const unsigned pairs = p.Hk * p.B, pair = id % pairs;
        id /= pairs;
        b = pair / p.Hk;
        c = pair % p.Hk;
        split = id % splits;
        tile = id / splits;
    }
};

// A load of 16 (or 4) bytes a lane that writes LDS by itself: lane i's go to `to` + 16 i (4 i), from `base` (of the whole wavefront) and the
// lane's offset; an offset behind the resource's end gives zeros.  It stands here as the instruction because the compiler
// orders every later read of LDS behind the one it knows of, and so would wait for a tile that is not needed before the
// next step; the ring above waits and has a barrier where it is.  No vector register is written, so none can be written late.
// A descriptor's word may come straight from v_readfirstlane, whose result a memory instruction may read five wait states later:
// the compiler sees to that between its own instructions, here s_nop 4 does.  m0, where the instruction finds its place in LDS, is
// an operand, so that the compiler knows it to be in use.
template <int BYTES>
__device__ __forceinline__ void load_to_lds(const void* base, unsigned offset, char* to) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const uintptr_t a = (uintptr_t)base;
    const u32x4 source = {(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a),
                          (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)) & 0xffffu, 0x7fffffffu, 0x00020000u};
    const unsigned lds = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)to);  // an address in LDS ends in its offset
    static_assert(BYTES == 16 || BYTES == 4, "widths of these loads");
    if (BYTES == 16) asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(lds), "v"(offset), "s"(source) : "memory");
    else asm volatile("s_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"{m0}"(lds), "v"(offset), "s"(source) : "memory");
}
// Copies of tiles from an array's rows (a fixed stride apart) into LDS by a workgroup of NT threads: ROWS rows of DP
// features.  Where rows allow it (VEC) the loads write LDS themselves, 16 bytes a lane, in the order of the tile's places;
// which piece of which row that is decides each lane's address.  A place without a piece (behind the head's features or
// the last row) is read at an offset behind the resource's end, which gives zeros.  Other rows take the way through
// registers, element by element.
template <class T, int DP, int ROWS, int NT, bool VEC>
struct Copy {
    typedef Lds<T, DP> L;
    static constexpr int kTotal = ROWS * L::kPlaces, kEach = (kTotal + NT - 1) / NT;
    static constexpr unsigned kNowhere = 0xffffffffu;
    static_assert(kTotal % 64 == 0, "whole wavefronts copy");
    static constexpr int kLoads = VEC ? kTotal / NT : 0;  // that every wavefront issues at least
    unsigned offset[kEach];
    int wave;
    static __device__ __forceinline__ int row(int c, int tid) { return (tid + c * NT) / L::kPlaces; }
    __device__ __forceinline__ Copy(int64_t stride, int D, int tid) : wave(__builtin_amdgcn_readfirstlane(tid >> 6)) {
        if (!VEC) return;
#pragma unroll
        for (int c = 0; c < kEach; ++c) {
            const int i = row(c, tid), piece = (tid + c * NT) % L::kPlaces ^ L::swap(i), d = piece * Matrix<T>::kChunk;
            offset[c] = d < D ? (unsigned)(i * stride + d) * (unsigned)sizeof(T) : kNowhere;
        }
    }
    // from: the first row; rows: how many there are (at least one)
    __device__ __forceinline__ void start(char* tile, const T* from, int64_t stride, int rows, int D, int tid) const {
        if (VEC) {
            const bool whole = rows >= ROWS;
#pragma unroll
            for (int c = 0; c < kEach; ++c) {
                if (kTotal % NT != 0 && (wave * 64 + c * NT) >= kTotal) break;
                const unsigned o = whole || row(c, tid) < rows ? offset[c] : kNowhere;
                load_to_lds<16>(from, o, tile + (wave * 64 + c * NT) * 16);
            }
        } else {
#pragma unroll 1
            for (int at = tid; at < kTotal; at += NT) {
                const int i = at / L::kPlaces, d = (at % L::kPlaces ^ L::swap(i)) * Matrix<T>::kChunk;
                T t[Matrix<T>::kChunk];
#pragma unroll
                for (int e = 0; e < Matrix<T>::kChunk; ++e) t[e] = i < rows && d + e < D ? from[i * stride + d + e] : (T)0.f;
                *(uint4*)(tile + at * 16) = *(uint4*)t;
            }
        }
    }
    // rows for which none(row) holds become zeros; behind the copy and a barrier
    template <class None>
    static __device__ __forceinline__ void clear(char* tile, const None& none, int tid) {
#pragma unroll 1
        for (int at = tid; at < kTotal; at += NT)
            if (none(at / L::kPlaces)) *(uint4*)(tile + at * 16) = uint4{0, 0, 0, 0};
    }
};

// ROWS values of 4 bytes, a fixed stride apart, into LDS; zeros behind `count`.  By the first wavefronts; a register is not
// waited for, so the loads that come after stay under way.
template <int ROWS>
__device__ __forceinline__ void copy_words(char* to, const void* from, int64_t stride, int count, int tid, int wave) {
    static_assert(ROWS % 32 == 0, "half wavefronts");
    const bool mine = tid < ROWS;
    if (wave * 64 < ROWS && mine) load_to_lds<4>(from, tid < count ? (unsigned)(tid * stride) * 4u : 0xffffffffu, to + wave * 256);
}

// Tiles of keys and values on their way from memory to LDS: shared by the kernels that own rows.  Keys behind the sequence, of
// no document, or between the prefix and the first query's window are zero, whatever the arrays hold there.
template <class X, int DP, class C, bool VEC>
struct KeyTiles {
    typedef Matrix<X> M;
    typedef typename M::E E;
    typedef Copy<E, DP, C::BK, C::NT, VEC || M::kPlanes == 3> S;
    static_assert(C::NT >= C::BK, "one thread a key for the documents");
    static constexpr int kPlane = C::BK * Lds<E, DP>::kPitch, kTile = M::kPlanes * kPlane;
    static constexpr int kBytes = C::kBufs * (2 * kTile + C::BK * 4);
    static constexpr int kLoads = 2 * M::kPlanes * S::kLoads;
    const Params& p;
    const Tensor &kt, &vt;
    const E *kb, *vb;
    const int* kd;
    char* lds;
    int n, prefix, window, tid, D;  // window: where the first query's begins
    S k, v;
    __device__ __forceinline__ KeyTiles(const Params& p_, int b, int c, int n_, int prefix_, const Band& band, int tid_, char* lds_)
        : p(p_), kt(M::kPlanes == 3 ? p_.k3 : p_.k), vt(M::kPlanes == 3 ? p_.v3 : p_.v), lds(lds_), n(n_), prefix(prefix_),
          window(n_ - p_.Lq - band.below), tid(tid_), D(M::kPlanes == 3 ? p_.D3 : p_.D), k(kt.l, D, tid_), v(vt.l, D, tid_) {
        kb = (const E*)kt.data + b * kt.b + c * kt.h;
        vb = (const E*)vt.data + b * vt.b + c * vt.h;
        kd = p.kdoc ? p.kdoc + b * p.kdoc_b : nullptr;
    }
    __device__ __forceinline__ char* keys(int buf) const { return lds + buf * 2 * kTile; }
    __device__ __forceinline__ char* values(int buf) const { return lds + buf * 2 * kTile + kTile; }
    __device__ __forceinline__ char* docs(int buf) const { return lds + C::kBufs * 2 * kTile + buf * C::BK * 4; }
    __device__ __forceinline__ void operator()(const Tile& tile, int buf) const {
        const int64_t j0 = (int64_t)tile.t * C::BK;
        const int left = n - (int)j0;
        if (kd) copy_words<C::BK>(docs(buf), kd + j0 * p.kdoc_l, p.kdoc_l, left, tid, k.wave);
#pragma unroll
        for (int i = 0; i < M::kPlanes; ++i) k.start(keys(buf) + i * kPlane, kb + i * p.k_plane + j0 * kt.l, kt.l, left, D, tid);
#pragma unroll
        for (int i = 0; i < M::kPlanes; ++i) v.start(values(buf) + i * kPlane, vb + i * p.k_plane + j0 * vt.l, vt.l, left, D, tid);
    }
    // a tile that has arrived and holds keys of no document or in front of every window
    __device__ __forceinline__ void clean(const Tile& tile, int buf) const {
        const int j0 = tile.t * C::BK;
        const bool strays = kd && tile.documents.x < 0, early = j0 < window && j0 + C::BK > prefix;
        if (!strays && !early) return;
        const int* of = (const int*)docs(buf);
#pragma unroll 1
        for (int i = 0; i < 2 * M::kPlanes; ++i)
            S::clear(keys(buf) + i * kPlane, [&](int r) { return (strays && of[r] < 0) || (j0 + r >= prefix && j0 + r < window); }, tid);
        __syncthreads();
    }
};

// What is taken in parts (more than a token's worth of rows of f32, at most 128 features), and its features there.
inline bool in_parts(int type, int D, bool few_rows) { return type == ADHIP_F32 && D <= 128 && !few_rows; }
// Rows of a workgroup of the forward kernels
constexpr int forward_rows(int type, int D, bool few_rows) { return few_rows ? 32 : type == ADHIP_F32 && D > 64 && D <= 128 ? 256 : 128; }
inline int parts_size(int D) { return (D + 7) / 8 * 8; }

// DP: the head's features, rounded up to what the kernels are built for
inline int padded_size(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

// one per type, in files of their own
void forward_bf16(const Params& p, bool few_rows, hipStream_t stream);
void forward_f32(const Params& p, bool few_rows, hipStream_t stream);
void backward_bf16(const Params& p, hipStream_t stream);
void backward_f32(const Params& p, hipStream_t stream);
void backward_f32_wide(const Params& p, hipStream_t stream);

}  // namespace attn
}  // namespace adhip

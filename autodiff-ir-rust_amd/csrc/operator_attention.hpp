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
// types, single words for 32-bit ones.  bf16 takes one instruction (32x32x16), f32 eight (32x32x2), with the same layouts.
#pragma once
#include "operators.hpp"

namespace adhip {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRange = 32;  // positions that share an entry of the document ranges

struct Tensor {
    const void* data;
    int64_t b, l, h;  // strides in elements
    int vec;          // 16 bytes can be read at a time
};

struct Params {
    Tensor q, k, v, out, dout, dq, dk, dv;  // out: written by the forward kernels, read by the backward ones
    float* lse;
    int64_t lse_b, lse_l, lse_h;
    const float* slopes;
    int64_t slope_stride;
    const int *lengths, *prefix, *qdoc, *kdoc;
    int64_t lengths_s, prefix_s, qdoc_b, qdoc_l, kdoc_b, kdoc_l;
    const int2 *qrange, *krange;  // smallest and largest document (of those >= 0) of every kRange positions
    int qranges, kranges;         // entries of a sequence
    int B, Lq, Lk, Hk, G, D, R;   // R = Lq G rows
    float scale, cap;
    int causal, window;
    int tiles, splits;            // row tiles (or key tiles); ranges that the keys (or rows) are split into
    float *part, *part_ml;        // forward, split: [split][b][c][row][D], [..][row][2]
    float* delta;                 // backward: [b][c][row]
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <class T>
struct Matrix;
template <>
struct Matrix<bf16> {
    typedef bf16x8 Frag;
    static constexpr int kChunk = 8;  // elements of 16 bytes
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Matrix<float> {
    typedef f32x8 Frag;
    static constexpr int kChunk = 4;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

template <class T, int DP>
struct Lds {
    // 16 bytes behind every row: eight rows of a fragment start in different banks
    static constexpr int kPitch = DP + 16 / (int)sizeof(T);
};

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// A (or B) operand whose rows are rows of the tile: rows row0 .. + 31, features 16 step .. + 15
template <class T, int DP>
__device__ __forceinline__ typename Matrix<T>::Frag rows_frag(const T* tile, int row0, int step, int lane) {
    return *(const typename Matrix<T>::Frag*)(tile + (row0 + (lane & 31)) * Lds<T, DP>::kPitch + step * 16 + (lane >> 5) * 8);
}

// A operand whose rows are features d0 .. + 31 of the tile and whose k are its rows k0 .. + 15, in the order of C's registers
template <int DP>
__device__ __forceinline__ bf16x8 cols_frag(const bf16* tile, int k0, int d0, int lane) {
    typedef __attribute__((address_space(3))) s16x4* Ptr;
    const bf16* a = tile + (k0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * Lds<bf16, DP>::kPitch + d0 + (lane & 16) + 4 * (lane & 3);
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)a);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(a + 8 * Lds<bf16, DP>::kPitch));
    const s16x8 r = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, r);
}
template <int DP>
__device__ __forceinline__ f32x8 cols_frag(const float* tile, int k0, int d0, int lane) {
    const float* a = tile + (k0 + 4 * (lane >> 5)) * Lds<float, DP>::kPitch + d0 + (lane & 31);
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        r[e] = a[e * Lds<float, DP>::kPitch];
        r[e + 4] = a[(e + 8) * Lds<float, DP>::kPitch];
    }
    return r;
}

// registers 8 s .. + 7 of a C tile as a B operand.  Probabilities and score gradients are rounded to the operands' type
// here, as the matrix cores take them; sums of probabilities are taken before.
__device__ __forceinline__ void to_frag(const f32x16& c, int s, bf16x8& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (bf16)c[8 * s + e];
}
__device__ __forceinline__ void to_frag(const f32x16& c, int s, f32x8& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c[8 * s + e];
}

// 16 bytes of a row of D features from d on; what lies behind the row's end is zero
template <class T>
__device__ __forceinline__ uint4 load_chunk(const T* row, int d, int D, int vec) {
    uint4 r = {0, 0, 0, 0};
    if (vec) {
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
template <class T>
__device__ __forceinline__ typename Matrix<T>::Frag load_frag(const T* row, int d, int D, int vec, bool valid) {
    typename Matrix<T>::Frag f;
    uint4* u = (uint4*)&f;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(f) / 16); ++i)
        u[i] = valid ? load_chunk(row, d + i * Matrix<T>::kChunk, D, vec) : uint4{0, 0, 0, 0};
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

// tanh to about 2e-7 of one: what a capped score takes, in units of the cap
__device__ __forceinline__ float tanh_of(float x) {
    const float e = __builtin_amdgcn_exp2f(x * (2.f * kLog2e));
    return 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
}

// Scores in units of log 2 from raw products, without masks; `bent` gets tanh where scores are capped.
// far: position of the query minus key of register 0 (or key minus position: only its magnitude counts), step: +1 / -1 per row
struct Scoring {
    float scale2, cap_in, cap_out;  // scale log2 e; scale / cap, cap log2 e
    __device__ __forceinline__ explicit Scoring(const Params& p)
        : scale2(p.scale * kLog2e), cap_in(p.cap > 0.f ? p.scale / p.cap : 0.f), cap_out(p.cap * kLog2e) {}
};

// row of register i of a C tile
__device__ __forceinline__ constexpr int c_row(int i) { return 8 * (i >> 2) + (i & 3); }

// Positions that a query sees: j < n and (j < prefix or lo <= j <= hi).  lo and hi by the query's own position.
struct Band {
    int below, above;  // lo = at - below, hi = at + above; where there is no limit, more than any position
    __device__ __forceinline__ explicit Band(const Params& p) {
        constexpr int kAll = 1 << 30;
        below = p.window ? p.window - 1 : kAll;
        above = p.causal ? 0 : below;
    }
};

__device__ __forceinline__ int sequence_length(const Params& p, int b) {
    const int n = p.lengths ? p.lengths[b * p.lengths_s] : p.Lk;
    return min(max(n, 0), p.Lk);
}

// smallest and largest document of positions first .. last from the table of ranges
__device__ __forceinline__ int2 document_range(const int2* ranges, int first, int last) {
    int2 r = {0x7fffffff, -1};
    for (int i = first / kRange; i <= last / kRange; ++i) {
        const int2 x = ranges[i];
        r.x = min(r.x, x.x);
        r.y = max(r.y, x.y);
    }
    return r;
}

// Walks the tiles that a block needs, 64 candidates at a time: each lane decides on one, all wavefronts alike.
template <class Needed>
struct Tiles {
    const Needed& needed;
    int base, end;
    unsigned long long mask = 0;
    __device__ __forceinline__ Tiles(const Needed& f, int begin, int stop) : needed(f), base(begin - 64), end(stop) {}
    // the next tile, or -1
    __device__ __forceinline__ int next(int lane) {
        while (!mask) {
            base += 64;
            if (base >= end) return -1;
            const int t = base + lane;
            mask = __ballot(t < end && needed(t));
        }
        const int t = base + __builtin_ctzll(mask);
        mask &= mask - 1;
        return t;
    }
};

// Consecutive workgroups go to the eight dies in turn; this gives each die a run of consecutive numbers instead, so that
// tiles that share keys share an L2.  The grid is rounded up to a multiple of eight; numbers from `total` on do nothing.
__device__ __forceinline__ int by_die(int block, int total) {
    const int each = (total + 7) / 8;
    return (block & 7) * each + (block >> 3);
}
inline unsigned die_grid(int64_t total) { return (unsigned)((total + 7) / 8 * 8); }

// The tile that a workgroup copies from an array's rows into LDS: NT threads, ROWS rows of DP features.
template <class T, int DP, int ROWS, int NT>
struct Stage {
    static constexpr int kPerRow = DP / Matrix<T>::kChunk;
    static constexpr int kChunks = (ROWS * kPerRow + NT - 1) / NT;
    static constexpr bool kEven = ROWS * kPerRow % NT == 0;
    uint4 r[kChunks];
    // row(i) gives the address of tile row i, or null for a row of zeros
    template <class Row>
    __device__ __forceinline__ void load(const Row& row, int D, int vec, int tid) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int at = tid + c * NT, i = at / kPerRow, d = at % kPerRow * Matrix<T>::kChunk;
            r[c] = uint4{0, 0, 0, 0};
            if (kEven || i < ROWS) {
                const T* x = row(i);
                if (x) r[c] = load_chunk(x, d, D, vec);
            }
        }
    }
    __device__ __forceinline__ void store(T* tile, int tid) const {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int at = tid + c * NT, i = at / kPerRow, d = at % kPerRow * Matrix<T>::kChunk;
            if (kEven || i < ROWS) *(uint4*)(tile + i * Lds<T, DP>::kPitch + d) = r[c];
        }
    }
};

// DP: the head's features, rounded up to what the kernels are built for
inline int padded_size(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

// one per type, in files of their own
void forward_bf16(const Params& p, bool few_rows, hipStream_t stream);
void forward_f32(const Params& p, bool few_rows, hipStream_t stream);
void backward_bf16(const Params& p, hipStream_t stream);
void backward_f32(const Params& p, hipStream_t stream);

}  // namespace attn
}  // namespace adhip

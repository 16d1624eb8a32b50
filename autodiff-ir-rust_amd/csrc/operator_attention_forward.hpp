// Attention forward: softmax in one pass over the keys with a running maximum and sum (Milakov and Gimelshein 2018; Dao et
// al. 2022), the scores never leave the registers.
//
// A wavefront owns 32 rows and multiplies keys by rows (S^T = K Q^T) and values by probabilities (O^T = V^T P^T), so that a
// lane holds one row of the softmax, 16 keys of every 32: its maximum takes one exchange between the lane's halves, its
// sum none until the end, and its rescaling is one factor a lane.
//
// WQ wavefronts along the rows, WK along the keys of a tile of BK.  Many rows: four wavefronts own 128 rows and share each
// tile of keys.  Few rows (one token a sequence): four wavefronts share 32 rows and split each tile of keys, the keys are
// split over workgroups beside that, and the parts are joined, with their maxima and sums, in LDS and by a second kernel.
//
// Measured, causal, clocks risen: bf16 2 x 4096 positions of 16 heads on 4 of 128 156 us (880 TFLOP/s), with capped scores 203 (680:
// tanh takes as many vector cycles as the softmax); 8 heads of 64 62 us (550), of 256 224 (613); f32 2 x 2048, 8 heads of 128 127 us
// (135, parts and join counted).  Matrix instructions and exponentials bound it, half of the one running beside the other.  Tokens: 8
// sequences of 8192 to 16384 keys, 8 key heads of 128 in bf16, 86 to 89 us, 4.5 to 4.7 TB/s, and 5 for the join; row sums read 6.5, with more
// than one tile under way.
#pragma once
#include <algorithm>

#include "operator_attention.hpp"

namespace adhip {
namespace attn {

// BUFS: tiles of keys in LDS; with two, one is under way while the other is worked on.
// WAVES: wavefronts of a SIMD that registers must leave room for.
template <int DP, int WQ_, int WK_, int BK_, int BUFS, int WAVES_>
struct ForwardConfig {
    static constexpr int WQ = WQ_, WK = WK_, BK = BK_, kBufs = BUFS, WAVES = WAVES_;
    static constexpr int NT = 64 * WQ * WK, BQ = 32 * WQ, KB = BK / (32 * WK);
    static constexpr int kMerge = WK > 1 ? WK * 32 * (DP + 4) * 4 + WK * 64 * 4 : 0;
};

template <class X, int DP, bool VEC, class C>
__global__ __launch_bounds__(C::NT, C::WAVES) void forward_kernel(const Params p) {
    typedef Matrix<X> M;
    typedef typename M::IO T;
    typedef typename M::Frag Frag;
    typedef KeyTiles<X, DP, C, VEC> Keys;
    __shared__ __attribute__((aligned(1024))) char lds[Keys::kBytes > C::kMerge ? Keys::kBytes : C::kMerge];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = wave % C::WQ, wk = wave / C::WQ;

    // this workgroup's tile of rows (the last ones see most keys), range of keys, key head and sequence
    const Place place(p, p.splits);
    const int tile = p.tiles - 1 - place.tile, split = place.split, c = place.c, b = place.b;

    const int n = sequence_length(p, b), offset = n - p.Lq;
    const int prefix = p.prefix ? min(max(p.prefix[b * p.prefix_s], 0), n) : 0;
    const Band band(p);
    // the running maximum wants a positive unit: the scale's sign goes to the queries
    const float sign = p.scale < 0.f ? -1.f : 1.f;
    const Scoring sc(p);
    const float unit = p.slopes || p.scale == 0.f ? 1.f : p.cap > 0.f ? sc.unit : sign * sc.unit;
    const int row0 = tile * C::BQ, row1 = min(row0 + C::BQ, p.R) - 1;
    const int first = row0 / p.G, last = row1 / p.G;  // tokens of the tile

    // the lane's row
    const int row = row0 + wq * 32 + (lane & 31);
    const bool valid = row < p.R;
    const int token = valid ? row / p.G : 0, head = c * p.G + (valid ? row - token * p.G : 0);
    const int at = token + offset;
    const int doc = p.qdoc && valid ? p.qdoc[b * p.qdoc_b + token * p.qdoc_l] : 0;
    const bool blind = doc < 0;  // of no document
    const Sight sight = {at - band.below, min(at + band.above, n - 1), prefix, doc, !valid || blind};
    const float slope = p.slopes && valid ? p.slopes[head * p.slope_stride] * kLog2e : 0.f;

    Frag qf[DP / 16];
    {
        const T* q = (const T*)p.q.data + b * p.q.b + token * p.q.l + head * p.q.h;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            typename M::Raw x = load_frag<VEC>(q, s * 16 + half * 8, p.D, valid && p.scale != 0.f);
            if (sign < 0.f)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = -x[e];
            qf[s] = M::operand(x);
            if (C::WAVES == 1 && M::kAside) keep_aside(qf[s]);
        }
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[d] = zero16();
    float m = -__builtin_inff(), l = 0.f;

    // tiles of keys that some row of this workgroup sees
    const int hi_all = last + offset + band.above, lo_all = first + offset - band.below;
    const int t_first = prefix > 0 ? 0 : max(lo_all, 0) / C::BK, t_stop = (min(n, max(hi_all + 1, prefix)) + C::BK - 1) / C::BK;
    const int2* const kr = p.krange ? p.krange + (int64_t)b * p.kranges : nullptr;
    int2 mine = {0, 0};
    if (kr) mine = document_range(p.qrange + (int64_t)b * p.qranges, first, last);
    auto needed = [&](int t, int2& theirs) {
        const int j0 = t * C::BK, j1 = min(j0 + C::BK, n) - 1;
        if (j0 >= prefix && (j0 > hi_all || j1 < lo_all)) return false;
        if (!kr) return true;
        theirs = document_range(kr, j0, j1);
        return documents_meet(mine, theirs);
    };
    // the lane's place in the wavefront's keys of a tile
    const unsigned k_lane = rows_lane<X, DP>(lane) + wk * C::KB * 32 * Lds<typename M::E, DP>::kPitch;
    const unsigned v_lane = cols_lane<X, DP>(lane) + wk * C::KB * 32 * Lds<typename M::E, DP>::kPitch;
    typedef Tiles<decltype(needed)> Walk;
    Walk walk(needed, t_first, t_stop, split, p.splits, lane);
    const Keys kt(p, b, c, n, prefix, band, tid, lds);
    Ring<C::kBufs, Keys::kLoads, Walk, Keys> ring(walk, kt);
    for (; ring.ready(); ring.pop()) {
        const int buf = ring.buf, t = ring.queue[0].t;
        kt.clean(ring.queue[0], buf);
        ring.more();
        const unsigned ks = here(lds_address(kt.keys(buf)) + k_lane), vs = here(lds_address(kt.values(buf)) + v_lane);
        const int* docs = (const int*)kt.docs(buf);
        const int2 theirs = ring.queue[0].documents;
        f32x16 s[C::KB];
#pragma unroll
        for (int x = 0; x < C::KB; ++x) {
            s[x] = zero16();
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) s[x] = M::mma(rows_frag<X, DP, C::BK>(ks, x * 32, k), qf[k], s[x]);
        }
        const int j0 = t * C::BK + wk * C::KB * 32, jl = j0 + 4 * half;  // register i of s[x] has key jl + 32 x + c_row(i)
        if (p.cap > 0.f) {
#pragma unroll
            for (int x = 0; x < C::KB; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[x][i] = tanh_of<M::kFine>(s[x][i] * (sign * sc.bend));
        }
        if (p.slopes) {
            const float inner = p.cap > 0.f ? sc.unit : sign * sc.unit;
#pragma unroll
            for (int x = 0; x < C::KB; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[x][i] = s[x][i] * inner - slope * fabsf((float)(at - jl - 32 * x - c_row(i)));
        }
        const int j1 = j0 + 32 * C::KB - 1;
        const bool all = sight.all(j0, j1, kt.kd, theirs);
        if (!__all(all)) {
            if (__all(all || sight.none(j0, j1, kt.kd, theirs))) {
#pragma unroll
                for (int x = 0; x < C::KB; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[x][i] = all ? s[x][i] : -__builtin_inff();
            } else {
#pragma unroll
                for (int x = 0; x < C::KB; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[x][i] = sight.sees(jl + 32 * x + c_row(i)) ? s[x][i] : -__builtin_inff();
                if (kt.kd) {
#pragma unroll
                    for (int x = 0; x < C::KB; ++x)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const int4 of = *(const int4*)(docs + (wk * C::KB + x) * 32 + 4 * half + c_row(i));
                            s[x][i] = of.x == doc ? s[x][i] : -__builtin_inff();
                            s[x][i + 1] = of.y == doc ? s[x][i + 1] : -__builtin_inff();
                            s[x][i + 2] = of.z == doc ? s[x][i + 2] : -__builtin_inff();
                            s[x][i + 3] = of.w == doc ? s[x][i + 3] : -__builtin_inff();
                        }
                }
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int x = 0; x < C::KB; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[x][i]);
        top = max_of_halves(top);
        // The sums are rescaled when the maximum has grown by more than 2^8, not at each of its first, small steps: they and
        // the probabilities have the same relative precision below that as below one.
        if (__any(top * unit > m * unit + 8.f)) {
            const float m_new = fmaxf(m, top), a = m_new == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * unit);
            l *= a;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= a;
            m = m_new;
        }
        const float base = m == -__builtin_inff() ? 0.f : m * unit;
#pragma unroll
        for (int x = 0; x < C::KB; ++x) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[x][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i], unit, -base));
                l += s[x][i];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag f;
                to_frag(s[x], h, f);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) o[d] = M::mma(cols_frag<X, DP, C::BK>(vs, x * 32 + 16 * h, d * 32), f, o[d]);
            }
        }
    }
    l = sum_of_halves(l);
    m *= unit;
    if (__any(blind)) {
        l = blind ? 0.f : l;
        m = blind ? -__builtin_inff() : m;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = blind ? 0.f : o[d][i];
    }

    const int64_t rows_before = (((int64_t)split * p.B + b) * p.Hk + c) * p.R;
    if (C::WK == 1) {
        if (!valid) return;
        if (p.splits > 1) {
            float* part = p.part + (rows_before + row) * p.D;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float f[4] = {o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
                    store4(part, d * 32 + 8 * g + 4 * half, p.D, (p.D & 3) == 0, f);
                }
            if (half == 0) {
                p.part_ml[(rows_before + row) * 2] = m;
                p.part_ml[(rows_before + row) * 2 + 1] = l;
            }
            return;
        }
        const float r = l > 0.f || l != l ? 1.f / l : 0.f;
        T* out = (T*)p.out.data + b * p.out.b + token * p.out.l + head * p.out.h;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float f[4] = {o[d][4 * g] * r, o[d][4 * g + 1] * r, o[d][4 * g + 2] * r, o[d][4 * g + 3] * r};
                store4(out, d * 32 + 8 * g + 4 * half, p.D, p.out.vec, f);
            }
        if (half == 0) p.lse[b * p.lse_b + token * p.lse_l + head * p.lse_h] = (m + __builtin_amdgcn_logf(l)) * kLn2;
        return;
    }
    // join the wavefronts' parts: every one scales its own to the common maximum, then all add up
    __syncthreads();
    float* const so = (float*)lds;                                // [WK][32][DP + 4]
    float* const sm = so + C::WK * 32 * (DP + 4);                 // [WK][32] maxima, [WK][32] sums
    if (half == 0) sm[wk * 32 + lane] = m;
    __syncthreads();
    float all = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < C::WK; ++w) all = fmaxf(all, sm[w * 32 + (lane & 31)]);
    const float a = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - all);
    if (half == 0) sm[C::WK * 32 + wk * 32 + lane] = l * a;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float* to = so + (wk * 32 + (lane & 31)) * (DP + 4) + d * 32 + 8 * g + 4 * half;
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] = o[d][4 * g + e] * a;
        }
    __syncthreads();
    for (int i = tid; i < 32 * (DP / 4); i += C::NT) {
        const int rr = i / (DP / 4), d = i % (DP / 4) * 4, gr = row0 + rr;
        if (gr >= p.R) break;
        float f[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f, mm = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < C::WK; ++w) {
            const float* from = so + (w * 32 + rr) * (DP + 4) + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] += from[e];
            sum += sm[C::WK * 32 + w * 32 + rr];
            mm = fmaxf(mm, sm[w * 32 + rr]);
        }
        if (p.splits > 1) {
            store4(p.part + (rows_before + gr) * p.D, d, p.D, (p.D & 3) == 0, f);
            if (d == 0) {
                p.part_ml[(rows_before + gr) * 2] = mm;
                p.part_ml[(rows_before + gr) * 2 + 1] = sum;
            }
            continue;
        }
        const int tk = gr / p.G, hd = c * p.G + gr - tk * p.G;
        const float r = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] *= r;
        store4((T*)p.out.data + b * p.out.b + tk * p.out.l + hd * p.out.h, d, p.D, p.out.vec, f);
        if (d == 0) p.lse[b * p.lse_b + tk * p.lse_l + hd * p.lse_h] = (mm + __builtin_amdgcn_logf(sum)) * kLn2;
    }
}

// Joins up to eight ranges of keys, as many rows have them: a thread four features of a row.  All its loads are under way
// together: they are what it takes (four ranges of 2048 x 8 heads of 128: 14 us in f32, 17 by the kernel below).
constexpr int kFewRanges = 8;
template <class T>
__global__ __launch_bounds__(256) void join_few_kernel(const Params p) {
    const unsigned pieces = (p.D + 3) / 4, rows = p.B * p.Hk * p.R, item = blockIdx.x * 256 + threadIdx.x, at = item / pieces;
    if (at >= rows) return;
    const int d = (int)(item - at * pieces) * 4;
    const bool vec = p.D % 4 == 0;
    f32x4 x[kFewRanges];
    float2 ml[kFewRanges];
#pragma unroll
    for (int s = 0; s < kFewRanges; ++s) {
        if (s >= p.splits) break;
        const int64_t row = (int64_t)s * rows + at;
        ml[s] = *(const float2*)(p.part_ml + row * 2);
        const float* from = p.part + row * p.D + d;
        if (vec) x[s] = *(const f32x4*)from;
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) x[s][e] = d + e < p.D ? from[e] : 0.f;
    }
    float m = -__builtin_inff(), sum = 0.f, f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kFewRanges; ++s)
        if (s < p.splits) m = fmaxf(m, ml[s].x);
    const float base = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int s = 0; s < kFewRanges; ++s)
        if (s < p.splits) {
            const float w = __builtin_amdgcn_exp2f(ml[s].x - base);
            sum += ml[s].y * w;
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] += x[s][e] * w;
        }
    const unsigned bc = at / (unsigned)p.R;
    const int row = (int)(at - bc * p.R), b = (int)(bc / p.Hk), c = (int)bc - b * p.Hk, token = row / p.G, head = c * p.G + row - token * p.G;
    const float over = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] *= over;
    store4((T*)p.out.data + b * p.out.b + token * p.out.l + head * p.out.h, d, p.D, p.out.vec, f);
    if (d == 0) p.lse[b * p.lse_b + token * p.lse_l + head * p.lse_h] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

// Joins more of them.  A row takes `pieces` threads of four features for each of `groups` runs of ranges, which are
// added up in LDS: with one wavefront a row that walked its ranges one after the other, the join of 64 ranges took longer
// than the attention before it.
struct JoinShape {
    int pieces, groups, rows;  // rows of a workgroup
    JoinShape(int D, int splits) : pieces((D + 3) / 4), groups(1) {
        // as many runs as ranges leave four each for, and threads allow
        while (groups * 8 <= splits && pieces * groups * 2 <= 256) groups *= 2;
        rows = std::min(256 / (pieces * groups), 2048 / splits);
    }
};
struct JoinPlace {
    int row, group, d;
    bool mine;  // (some threads behind the last row are left over)
    __host__ __device__ JoinPlace(const JoinShape& j, int rows, int tid)
        : row(tid / (j.pieces * j.groups)), group(tid / j.pieces - row * j.groups), d((tid % j.pieces) * 4), mine(row < rows) {}
    // the thread that adds up its own sum and those of the groups behind it, every `pieces` threads
    __host__ __device__ bool adds() const { return mine && group == 0; }
};
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const Params p, const JoinShape j) {
    __shared__ float ml[2 * 2048];
    __shared__ f32x4 sums[256];
    const int64_t rows = (int64_t)p.B * p.Hk * p.R, row0 = (int64_t)blockIdx.x * j.rows;
    const int tid = threadIdx.x, here_rows = (int)min((int64_t)j.rows, rows - row0);
    for (int i = tid; i < here_rows * p.splits; i += 256) {
        const int r = i / p.splits, s = i - r * p.splits;
        const float2 x = *(const float2*)(p.part_ml + (s * rows + row0 + r) * 2);
        ml[2 * i] = x.x;
        ml[2 * i + 1] = x.y;
    }
    __syncthreads();
    const JoinPlace place(j, here_rows, tid);
    const int r = place.row, d = place.d;
    const int64_t at = row0 + r;
    float m = -__builtin_inff(), sum = 0.f;
    f32x4 f = {0.f, 0.f, 0.f, 0.f};
    if (place.mine) {
        const float* of = ml + 2 * r * p.splits;
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s) m = fmaxf(m, of[2 * s]);
        const float base = m == -__builtin_inff() ? 0.f : m;
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s) sum += of[2 * s + 1] * __builtin_amdgcn_exp2f(of[2 * s] - base);
        const bool vec = (p.D & 3) == 0;
#pragma unroll 4
        for (int s = place.group; s < p.splits; s += j.groups) {
            const float w = __builtin_amdgcn_exp2f(of[2 * s] - base);
            const float* x = p.part + (s * rows + at) * p.D + d;
            if (vec) {
                const f32x4 y = *(const f32x4*)x;
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] += y[e] * w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] += d + e < p.D ? x[e] * w : 0.f;
            }
        }
    }
    if (j.groups > 1) {
        sums[tid] = f;
        __syncthreads();
        if (!place.adds()) return;
        for (int i = 1; i < j.groups; ++i) {
            const f32x4 y = sums[tid + i * j.pieces];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] += y[e];
        }
    }
    if (!place.mine) return;
    const int64_t bc = at / p.R;
    const int row = (int)(at - bc * p.R), c = (int)(bc % p.Hk), token = row / p.G, head = c * p.G + row - token * p.G;
    const int64_t b = bc / p.Hk;
    const float over = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const float y[4] = {f[0] * over, f[1] * over, f[2] * over, f[3] * over};
    store4((T*)p.out.data + b * p.out.b + token * p.out.l + head * p.out.h, d, p.D, p.out.vec, y);
    if (d == 0) p.lse[b * p.lse_b + token * p.lse_l + head * p.lse_h] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <class T>
void launch_join(const Params& p, hipStream_t stream) {
    const int pieces = (p.D + 3) / 4;
    // (keys are split where there are at most 1024 workgroups: 32 bits hold all numbers)
    if (p.splits <= kFewRanges) {
        launch("adhip_attention", join_few_kernel<T>, (unsigned)(((int64_t)p.B * p.Hk * p.R * pieces + 255) / 256), 256, stream, p);
        return;
    }
    const JoinShape j(p.D, p.splits);
    launch("adhip_attention", join_kernel<T>, (unsigned)(((int64_t)p.B * p.Hk * p.R + j.rows - 1) / j.rows), 256, stream, p, j);
}

// Bytes of a row of a tile decide how many keys a tile has and how many tiles LDS holds: 64 keys where tiles leave room for
// the workgroups that registers allow, 32 else, and as many tiles as then fit.  (Heads of 256, one workgroup a compute unit: 2 x
// 4096 x 8 heads 220 us with four tiles of 32.)
template <class X, int DP>
struct ForwardMany {
    static constexpr int kRow = DP * (int)sizeof(typename Matrix<X>::E);
    typedef ForwardConfig<DP, 4, 1, kRow <= 256 ? 64 : 32, kRow <= 128 ? 3 : kRow <= 384 ? 2 : kRow <= 512 ? 4 : 2,
                          kRow <= 128 ? 3 : kRow <= 384 ? 2 : 1> C;
};
// In parts: two workgroups of four wavefronts up to 64 features, one of eight above, so that a SIMD always has two and one's
// matrix instructions run beside the other's splitting and exponentials.  (2048 x 8 heads of 128, forward and backward: 415 us, with
// four wavefronts above 64 as well 537.)
template <int DP>
struct ForwardMany<Parts, DP> {
    typedef ForwardConfig<DP, forward_rows(ADHIP_F32, DP, false) / 32, 1, 32, 3, 2> C;
};
template <class X, int DP>
struct ForwardFew {
    static constexpr int kRow = DP * (int)sizeof(typename Matrix<X>::E);
    // as many wavefronts along the keys as LDS holds tiles for twice
    static constexpr int WK = kRow <= 256 ? 4 : kRow <= 512 ? 2 : 1;
    typedef ForwardConfig<DP, 1, WK, 32 * WK, 2, 1> C;
};

template <class X, int DP, class C>
void launch_forward(const Params& p, hipStream_t stream) {
    const unsigned grid = (unsigned)((int64_t)p.tiles * p.splits * p.Hk * p.B);
    const bool vec = p.q.vec && p.k.vec && p.v.vec;
    launch("adhip_attention", vec ? forward_kernel<X, DP, true, C> : forward_kernel<X, DP, false, C>, grid, C::NT, stream, p);
    if (p.splits > 1) launch_join<typename Matrix<X>::IO>(p, stream);
}

// Many: what multiplies where rows fill workgroups; Few: where they do not
template <class Many, class Few, int DP>
void launch_forward(const Params& p, bool few_rows, hipStream_t stream) {
    if (few_rows) launch_forward<Few, DP, typename ForwardFew<Few, DP>::C>(p, stream);
    else launch_forward<Many, DP, typename ForwardMany<Many, DP>::C>(p, stream);
}

}  // namespace attn
}  // namespace adhip

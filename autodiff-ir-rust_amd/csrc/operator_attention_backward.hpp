// Attention backward.  With p = exp(z - lse), dp = dout.v, delta = dout.out and  ds = p (dp - delta) (1 - (z_cap / cap)^2):
//     dq = scale ds k,   dk = scale ds^T q,   dv = p^T dout.
//
// Two kernels, each of which computes the scores again: one owns rows and walks the keys (dq, and delta on the way), one
// owns keys and walks the rows of all heads that share them (dk, dv).  That is seven products where one kernel with dq in
// atomic additions would take five, but nothing is added in an order that changes from run to run, dq takes no memory in
// f32, and heads that share keys add up in registers.
//
// Where there are too few workgroups for the card, or too few for the uneven work of a causal mask to even out, each walk
// is split and the parts are added, in order, by a third kernel.
//
// delta is taken from out as the caller kept it, in bf16 rounded once: beside the roundings of p and ds it adds 0.0001 to the 0.0024
// (norm of the error over the norm) of dq and dk, up to 0.0008 where few keys weigh.  The exact one would take out in more bits, or
// a pass of its own over the scores.
//
// Measured, causal, capped, clocks risen, bf16 2 x 4096 positions of 16 heads on 4 of 128: dq 259 us (795 TFLOP/s over its three
// products), dk and dv 360 (765 over four), adding two parts 15; 8 heads of 64 without a cap 187 us in all; f32 2 x 2048, 8 heads of
// 128 402 us in all.  Bounded like the forward pass by matrix instructions and exponentials, in f32 up to 128 features also by splitting
// what one wavefront a SIMD has nothing to run beside.  f32, 256 features: 2373 us on the FP32 matrix cores, where two of four
// SIMDs have no wavefront (two of them fill LDS), registers spill and every load is waited for.
#pragma once
#include <algorithm>

#include "operator_attention.hpp"

namespace adhip {
namespace attn {

// ---- dq: the forward kernel's walk ------------------------------------------------------------------------------------

template <int BK_, int BUFS, int WAVES_>
struct QueryConfig {
    static constexpr int BK = BK_, kBufs = BUFS, WAVES = WAVES_, NT = 256, BQ = 128, KB = BK / 32;
};

template <class X, int DP, bool VEC, class C>
__global__ __launch_bounds__(C::NT, C::WAVES) void query_gradient_kernel(const Params p) {
    typedef Matrix<X> M;
    typedef typename M::IO T;
    typedef typename M::Frag Frag;
    typedef KeyTiles<X, DP, C, VEC> Keys;
    __shared__ __attribute__((aligned(1024))) char lds[Keys::kBytes];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    const Place place(p, p.dq_splits);
    const int tile = p.tiles - 1 - place.tile, split = place.split, c = place.c, b = place.b;  // the last ones see most keys

    const int n = sequence_length(p, b), offset = n - p.Lq;
    const int prefix = p.prefix ? min(max(p.prefix[b * p.prefix_s], 0), n) : 0;
    const Band band(p);
    const Scoring sc(p);
    const float unit = p.slopes ? 1.f : sc.unit;
    const int row0 = tile * C::BQ, row1 = min(row0 + C::BQ, p.R) - 1;
    const int first = row0 / p.G, last = row1 / p.G;

    const int row = row0 + wave * 32 + (lane & 31);
    bool valid = row < p.R;
    const int token = valid ? row / p.G : 0, head = c * p.G + (valid ? row - token * p.G : 0);
    const int at = token + offset;
    const int doc = p.qdoc && valid ? p.qdoc[b * p.qdoc_b + token * p.qdoc_l] : 0;
    const float slope = p.slopes && valid ? p.slopes[head * p.slope_stride] * kLog2e : 0.f;
    const float lse = valid ? p.lse[b * p.lse_b + token * p.lse_l + head * p.lse_h] : -__builtin_inff();
    const bool inside = valid;
    // a row that sees nothing has no gradient, whatever dout holds there
    if (lse == -__builtin_inff()) valid = false;
    const Sight sight = {at - band.below, min(at + band.above, n - 1), prefix, doc, !valid};
    const float lse2 = lse * kLog2e;

    Frag qf[DP / 16], df[DP / 16];
    float delta = 0.f;
    {
        const T* q = (const T*)p.q.data + b * p.q.b + token * p.q.l + head * p.q.h;
        const T* d = (const T*)p.dout.data + b * p.dout.b + token * p.dout.l + head * p.dout.h;
        const T* o = (const T*)p.out.data + b * p.out.b + token * p.out.l + head * p.out.h;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            qf[s] = M::operand(load_frag<VEC>(q, s * 16 + half * 8, p.D, valid));
            const typename M::Raw x = load_frag<VEC>(d, s * 16 + half * 8, p.D, valid), y = load_frag<VEC>(o, s * 16 + half * 8, p.D, valid);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta += (float)x[e] * (float)y[e];
            df[s] = M::operand(x);
            if (C::WAVES == 1 && M::kAside) {
                keep_aside(qf[s]);
                keep_aside(df[s]);
            }
        }
    }
    delta = sum_of_halves(delta);
    if (inside && half == 0 && split == 0) {
        float* const to = p.stats + ((int64_t)b * p.Hk * p.G + head) * p.Lq + token;
        to[0] = valid ? lse2 : __builtin_inff();  // p = exp2(z - inf) = 0
        to[(int64_t)p.B * p.Hk * p.G * p.Lq] = -delta;
    }
    f32x16 dq[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dq[d] = zero16();

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
    const unsigned r_lane = rows_lane<X, DP>(lane), c_lane = cols_lane<X, DP>(lane);
    typedef Tiles<decltype(needed)> Walk;
    Walk walk(needed, t_first, t_stop, split, p.dq_splits, lane);
    const Keys kt(p, b, c, n, prefix, band, tid, lds);
    Ring<C::kBufs, Keys::kLoads, Walk, Keys> ring(walk, kt);
    for (; ring.ready(); ring.pop()) {
        const int buf = ring.buf, t = ring.queue[0].t;
        kt.clean(ring.queue[0], buf);
        ring.more();
        const unsigned kr_at = here(lds_address(kt.keys(buf)) + r_lane), vr_at = here(lds_address(kt.values(buf)) + r_lane);
        const unsigned kc_at = here(lds_address(kt.keys(buf)) + c_lane);
        const int* docs = (const int*)kt.docs(buf);
        const int2 theirs = ring.queue[0].documents;
#pragma unroll
        for (int x = 0; x < C::KB; ++x) {
            const int key0 = x * 32;
            f32x16 s = zero16(), g;
#pragma unroll
            for (int i = 0; i < 16; ++i) g[i] = -delta;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) s = M::mma(rows_frag<X, DP, C::BK>(kr_at, key0, k), qf[k], s);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) g = M::mma(rows_frag<X, DP, C::BK>(vr_at, key0, k), df[k], g);
            const int j0 = t * C::BK + key0, jl = j0 + 4 * half;
            const bool all = sight.all(j0, j0 + 31, kt.kd, theirs);
            if (p.cap > 0.f) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = tanh_of<M::kFine>(s[i] * sc.bend);
                    g[i] *= 1.f - s[i] * s[i];
                }
            }
            if (p.slopes) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = s[i] * sc.unit - slope * fabsf((float)(at - jl - c_row(i)));
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], unit, -lse2)) * g[i];
            if (!__all(all)) {
                if (__all(all || sight.none(j0, j0 + 31, kt.kd, theirs))) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = all ? s[i] : 0.f;
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = sight.sees(jl + c_row(i)) ? s[i] : 0.f;
                    if (kt.kd) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const int4 of = *(const int4*)(docs + key0 + 4 * half + c_row(i));
                            s[i] = of.x == doc ? s[i] : 0.f;
                            s[i + 1] = of.y == doc ? s[i + 1] : 0.f;
                            s[i + 2] = of.z == doc ? s[i + 2] : 0.f;
                            s[i + 3] = of.w == doc ? s[i + 3] : 0.f;
                        }
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag f;
                to_frag(s, h, f);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) dq[d] = M::mma(cols_frag<X, DP, C::BK>(kc_at, key0 + 16 * h, d * 32), f, dq[d]);
            }
        }
    }
    if (!inside) return;
    if (__any(!valid)) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) dq[d][i] = valid ? dq[d][i] : 0.f;
    }
    float* const part = p.dq_splits > 1 ? p.part_dq + ((((int64_t)split * p.B + b) * p.Hk + c) * p.R + row) * p.D : nullptr;
    T* const out = (T*)p.dq.data + b * p.dq.b + token * p.dq.l + head * p.dq.h;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float f[4] = {dq[d][4 * g] * p.scale, dq[d][4 * g + 1] * p.scale, dq[d][4 * g + 2] * p.scale, dq[d][4 * g + 3] * p.scale};
            if (part) store4(part, d * 32 + 8 * g + 4 * half, p.D, (p.D & 3) == 0, f);
            else store4(out, d * 32 + 8 * g + 4 * half, p.D, p.dq.vec, f);
        }
}

// ---- dk, dv -------------------------------------------------------------------------------------------------------------

// KG wavefronts own 32 keys each, RG of them share the keys and take every RG-th 32 rows of a tile of BR.
// K_LDS, V_LDS: the keys or values are read from LDS, where the two sums leave no registers for them.
template <class X, int DP, int KG_, int RG_, int BUFS, bool K_LDS_, bool V_LDS_, int WAVES_>
struct KeyConfig {
    static constexpr int KG = KG_, RG = RG_, BR = 32 * RG, kBufs = BUFS, NT = 64 * KG * RG, BKEYS = 32 * KG, WAVES = WAVES_;
    static constexpr bool K_LDS = K_LDS_, V_LDS = V_LDS_;
    static constexpr int kPlanes = Matrix<X>::kPlanes, kPitch = Lds<typename Matrix<X>::E, DP>::kPitch;
    static constexpr int kTile = kPlanes * BR * kPitch, kOwn = BKEYS * kPitch;
    static_assert(kPlanes == 1 || (!K_LDS && !V_LDS), "keys and values in parts stay in registers");
    static constexpr int kRows = kBufs * 2 * kTile + (K_LDS ? kOwn : 0) + (V_LDS ? kOwn : 0);
    static constexpr int kLoop = kRows + kBufs * BR * 3 * 4;  // of each row: log-sum, -delta, document
    static constexpr int kMerge = RG > 1 ? (RG - 1) * BKEYS * (DP + 4) * 4 : 0;
    static constexpr int kBytes = kLoop > kMerge ? kLoop : kMerge;
};

template <class X, int DP, bool VEC, class C>
__global__ __launch_bounds__(C::NT, C::WAVES) void key_gradient_kernel(const Params p) {
    typedef Matrix<X> M;
    typedef typename M::IO T;
    typedef typename M::E E;
    typedef typename M::Frag Frag;
    typedef Lds<E, DP> L;
    __shared__ __attribute__((aligned(1024))) char lds[C::kBytes];
    char* const k_own = lds + C::kBufs * 2 * C::kTile;
    char* const v_own = k_own + (C::K_LDS ? C::kOwn : 0);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave % C::KG, rg = wave / C::KG;

    const Place place(p, p.dk_splits);
    const int tile = place.tile, split = place.split, c = place.c, b = place.b;  // the first ones are seen by most rows

    const int n = sequence_length(p, b), offset = n - p.Lq;
    const int prefix = p.prefix ? min(max(p.prefix[b * p.prefix_s], 0), n) : 0;
    const Band band(p);
    const Scoring sc(p);
    const float unit = p.slopes ? 1.f : sc.unit;
    const int key_first = tile * C::BKEYS, key_last = min(key_first + C::BKEYS, n) - 1;
    const int key = key_first + kg * 32 + (lane & 31);
    const int doc = p.kdoc && key < n ? p.kdoc[b * p.kdoc_b + key * p.kdoc_l] : 0;
    const bool valid = key < n && doc >= 0;
    // rows at positions from .. to see this key, all up to the last one, at n - 1, where it is in the prefix: rows behind the last
    // one fill up a tile, and a slope below zero would make infinite probabilities of their distances
    // (a key that no row may see sees everything here, so that it keeps no wavefront from the short way; its gradients are
    // replaced at the end)
    constexpr int kFar = 1 << 29;  // more than any position
    const bool free = !valid || key < prefix;
    const int from = free ? -kFar : key - band.above, to = !valid ? kFar : min(free ? kFar : key + band.below, n - 1);

    Frag kf[C::K_LDS ? 1 : DP / 16], vf[C::V_LDS ? 1 : DP / 16];
    {
        const T* k = (const T*)p.k.data + b * p.k.b + key * p.k.l + c * p.k.h;
        const T* v = (const T*)p.v.data + b * p.v.b + key * p.v.l + c * p.v.h;
        constexpr int N = sizeof(typename M::Raw) / 16;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const typename M::Raw x = load_frag<VEC>(k, s * 16 + half * 8, p.D, valid), y = load_frag<VEC>(v, s * 16 + half * 8, p.D, valid);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int at = L::at(kg * 32 + (lane & 31), (2 * s + half) * N + i);
                if (C::K_LDS && rg == 0) *(uint4*)(k_own + at) = ((const uint4*)&x)[i];
                if (C::V_LDS && rg == 0) *(uint4*)(v_own + at) = ((const uint4*)&y)[i];
            }
            if (!C::K_LDS) {
                kf[s] = M::operand(x);
                if (C::WAVES == 1 && M::kAside) keep_aside(kf[s]);
            }
            if (!C::V_LDS) {
                vf[s] = M::operand(y);
                if (C::WAVES == 1 && M::kAside) keep_aside(vf[s]);
            }
        }
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dk[d] = zero16(), dv[d] = zero16();

    // Tiles of rows: BR queries of one head of the group.  Those that some key's band reaches, `len` a head, are numbered
    // head by head.
    const int i_first = key_first < prefix ? 0 : max(key_first - band.above - offset, 0);
    const int i_last = key_first < prefix ? p.Lq - 1 : min(key_last + band.below - offset, p.Lq - 1);
    const int t_first = i_first / C::BR, len = key_last >= key_first && i_last >= i_first ? i_last / C::BR + 1 - t_first : 0;
    const int2* const qr = p.qrange ? p.qrange + (int64_t)b * p.qranges : nullptr;
    int2 mine = {0, 0};
    if (qr && len > 0) mine = document_range(p.krange + (int64_t)b * p.kranges, key_first, key_last);
    auto needed = [&](int u, int2& theirs) {
        if (!qr) return true;
        const int i0 = (t_first + u % len) * C::BR;
        theirs = document_range(qr, i0, min(i0 + C::BR, p.Lq) - 1);
        return documents_meet(mine, theirs);
    };
    const unsigned r_lane = rows_lane<X, DP>(lane), c_lane = cols_lane<X, DP>(lane);
    typedef Tiles<decltype(needed)> Walk;
    Walk walk(needed, 0, len * p.G, split, p.dk_splits, lane);

    constexpr bool kParts = M::kPlanes == 3;
    typedef Copy<E, DP, C::BR, C::NT, VEC || kParts> Rows;
    const Tensor &tq = kParts ? p.q3 : p.q, &tg = kParts ? p.dout3 : p.dout;
    const int D = kParts ? p.D3 : p.D;
    const Rows copy_q(tq.l, D, tid), copy_g(tg.l, D, tid);
    static_assert(C::NT >= C::BR, "one thread a row for what rows have beside features");
    auto start = [&](const Tile& tile, int buf) {
        const int g = tile.t / len, i0 = (t_first + tile.t - g * len) * C::BR, h = c * p.G + g, left = p.Lq - i0;
        char* const to_q = lds + buf * 2 * C::kTile;
        char* const of = lds + C::kRows + buf * 3 * C::BR * 4;
        const float* const stats = p.stats + ((int64_t)b * p.Hk * p.G + h) * p.Lq + i0;
        copy_words<C::BR>(of, stats, 1, left, tid, wave);
        copy_words<C::BR>(of + C::BR * 4, stats + (int64_t)p.B * p.Hk * p.G * p.Lq, 1, left, tid, wave);
        if (p.qdoc) copy_words<C::BR>(of + 2 * C::BR * 4, p.qdoc + b * p.qdoc_b + i0 * p.qdoc_l, p.qdoc_l, left, tid, wave);
#pragma unroll
        for (int i = 0; i < M::kPlanes; ++i)
            copy_q.start(to_q + i * C::BR * L::kPitch, (const E*)tq.data + i * p.q_plane + b * tq.b + i0 * tq.l + h * tq.h, tq.l, left, D, tid);
#pragma unroll
        for (int i = 0; i < M::kPlanes; ++i)
            copy_g.start(to_q + C::kTile + i * C::BR * L::kPitch, (const E*)tg.data + i * p.q_plane + b * tg.b + i0 * tg.l + h * tg.h, tg.l, left, D, tid);
    };
    // A row that sees nothing is zero, whatever the arrays hold there.  (Rows behind the last one came as zeros, and no key sees
    // them.)
    auto clean = [&](int buf) {
        const float* const of = (const float*)(lds + C::kRows + buf * 3 * C::BR * 4);
        if (!__any(of[lane % C::BR] == __builtin_inff())) return;
        char* const q = lds + buf * 2 * C::kTile;
#pragma unroll 1
        for (int i = 0; i < 2 * M::kPlanes; ++i)
            Rows::clear(q + i * C::BR * L::kPitch, [&](int r) { return of[r] == __builtin_inff(); }, tid);
        __syncthreads();
    };
    static_assert(C::BR <= 64, "a wavefront looks over a tile's rows at once");

    Ring<C::kBufs, 2 * M::kPlanes * Rows::kLoads, Walk, decltype(start)> ring(walk, start);
    for (; ring.ready(); ring.pop()) {
        const int buf = ring.buf, t = ring.queue[0].t;
        clean(buf);
        ring.more();
        const int q0 = rg * 32;
        const unsigned tile_at = lds_address(lds) + buf * 2 * C::kTile + q0 * L::kPitch;
        const unsigned rows_at = here(tile_at + r_lane), cols_at = here(tile_at + c_lane);  // of q; of dout kTile behind
        const unsigned own_at = here(lds_address(k_own) + kg * 32 * L::kPitch + r_lane);
        // what the rows of registers 4 g .. have, array BR + 8 g + e: the log-sum, -delta, the document
        const float* of = (const float*)(lds + C::kRows + buf * 3 * C::BR * 4) + q0 + 4 * half;
        {
            const int g_of = t / len, first_at = (t_first + t - g_of * len) * C::BR + q0 + offset;
            const int2 theirs = ring.queue[0].documents;
            const bool all = from <= first_at && first_at + 31 <= to && (!p.qdoc || !valid || (theirs.x == doc && theirs.y == doc));
            f32x16 s = zero16();
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                s = M::mma(rows_frag<X, DP, C::BR>(rows_at, 0, k), C::K_LDS ? rows_frag<X, DP, C::BKEYS>(own_at, 0, k) : kf[C::K_LDS ? 0 : k], s);
            f32x16 g;
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 x = *(const f32x4*)(of + C::BR + c_row(i));
#pragma unroll
                for (int e = 0; e < 4; ++e) g[i + e] = x[e];
            }
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                g = M::mma(rows_frag<X, DP, C::BR>(rows_at, M::kPlanes * C::BR, k), C::V_LDS ? rows_frag<X, DP, C::BKEYS>(own_at, C::K_LDS ? C::BKEYS : 0, k) : vf[C::V_LDS ? 0 : k], g);
            if (p.cap > 0.f) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = tanh_of<M::kFine>(s[i] * sc.bend);
                    g[i] *= 1.f - s[i] * s[i];
                }
            }
            if (p.slopes) {
                const float slope = p.slopes[(c * p.G + g_of) * p.slope_stride] * kLog2e;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = s[i] * sc.unit - slope * fabsf((float)(first_at + 4 * half + c_row(i) - key));
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 lse = *(const f32x4*)(of + c_row(i));
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + e], unit, -lse[e]));
            }
            if (!__all(all)) {
                const bool none = first_at > to || first_at + 31 < from ||
                                  (p.qdoc && (doc < (theirs.x < 0 ? ~theirs.x : theirs.x) || doc > theirs.y));
                if (__all(all || none)) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = all ? s[i] : 0.f, g[i] = all ? g[i] : 0.f;
                } else {
                    const int rel = first_at + 4 * half - from;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const bool sees = (unsigned)(rel + c_row(i)) <= (unsigned)(to - from);
                        s[i] = sees ? s[i] : 0.f;
                        g[i] = sees ? g[i] : 0.f;
                    }
                    if (p.qdoc) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const int4 x = *(const int4*)(of + 2 * C::BR + c_row(i));
                            s[i] = x.x == doc ? s[i] : 0.f, g[i] = x.x == doc ? g[i] : 0.f;
                            s[i + 1] = x.y == doc ? s[i + 1] : 0.f, g[i + 1] = x.y == doc ? g[i + 1] : 0.f;
                            s[i + 2] = x.z == doc ? s[i + 2] : 0.f, g[i + 2] = x.z == doc ? g[i + 2] : 0.f;
                            s[i + 3] = x.w == doc ? s[i + 3] : 0.f, g[i + 3] = x.w == doc ? g[i + 3] : 0.f;
                        }
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag f;
                to_frag(s, h, f);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) dv[d] = M::mma(cols_frag<X, DP, C::BR>(cols_at, M::kPlanes * C::BR + 16 * h, d * 32), f, dv[d]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] *= g[i];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag f;
                to_frag(s, h, f);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) dk[d] = M::mma(cols_frag<X, DP, C::BR>(cols_at, 16 * h, d * 32), f, dk[d]);
            }
        }
    }
    if (C::RG > 1) {
        // the wavefronts that share keys add up, one sum after the other
        float* const mine_f = (float*)lds + (kg * 32 + (lane & 31)) * (DP + 4) + 4 * half;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
            if (rg > 0) {
#pragma unroll
                for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        f32x4 x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = which ? dv[d][4 * g + e] : dk[d][4 * g + e];
                        *(f32x4*)(mine_f + (rg - 1) * C::BKEYS * (DP + 4) + d * 32 + 8 * g) = x;
                    }
            }
            __syncthreads();
            if (rg == 0) {
#pragma unroll
                for (int r = 0; r < C::RG - 1; ++r)
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const f32x4 x = *(const f32x4*)(mine_f + r * C::BKEYS * (DP + 4) + d * 32 + 8 * g);
#pragma unroll
                            for (int e = 0; e < 4; ++e) (which ? dv[d] : dk[d])[4 * g + e] += x[e];
                        }
            }
        }
        if (rg > 0) return;
    }
    if (key >= p.Lk) return;
    if (__any(!valid)) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) dk[d][i] = valid ? dk[d][i] : 0.f, dv[d][i] = valid ? dv[d][i] : 0.f;
    }
    const int64_t part_at = ((((int64_t)split * p.B + b) * p.Hk + c) * p.Lk + key) * p.D;
    T* ko = (T*)p.dk.data + b * p.dk.b + key * p.dk.l + c * p.dk.h;
    T* vo = (T*)p.dv.data + b * p.dv.b + key * p.dv.l + c * p.dv.h;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = d * 32 + 8 * g + 4 * half;
            const float f[4] = {dk[d][4 * g] * p.scale, dk[d][4 * g + 1] * p.scale, dk[d][4 * g + 2] * p.scale, dk[d][4 * g + 3] * p.scale};
            const float e[4] = {dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]};
            if (p.dk_splits > 1) {
                store4(p.part_dk + part_at, at, p.D, (p.D & 3) == 0, f);
                store4(p.part_dv + part_at, at, p.D, (p.D & 3) == 0, e);
            } else {
                store4(ko, at, p.D, p.dk.vec, f);
                store4(vo, at, p.D, p.dv.vec, e);
            }
        }
}

// Adds the parts of split walks, in their order: [splits][B][Hk][rows][D] to arrays [B, rows / G, Hk G, D].  A thread four
// features of a row, all gradients in one launch.  (Walks are split where there are fewer than 65536 rows: 32 bits hold all
// numbers.)
struct PartsToAdd {
    const float* part;
    Tensor out;
    unsigned splits, rows, G;
};
struct AllPartsToAdd {
    PartsToAdd of[3];
};
template <class T>
__global__ __launch_bounds__(256) void add_parts_kernel(const AllPartsToAdd all, unsigned B, unsigned Hk, int D) {
    const PartsToAdd& j = all.of[blockIdx.y];
    const unsigned pieces = (D + 3) / 4, total = B * Hk * j.rows, at = blockIdx.x * 256 + threadIdx.x, row = at / pieces;
    if (row >= total) return;
    const int d = (int)(at - row * pieces) * 4;
    const float* from = j.part + (int64_t)row * D + d;
    const int64_t step = (int64_t)total * D;
    f32x4 f = {0.f, 0.f, 0.f, 0.f};
    if (D % 4 == 0) {
#pragma unroll 4
        for (unsigned s = 0; s < j.splits; ++s) {
            const f32x4 x = *(const f32x4*)(from + s * step);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] += x[e];
        }
    } else {
        for (unsigned s = 0; s < j.splits; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] += d + e < D ? from[s * step + e] : 0.f;
    }
    const unsigned bc = row / j.rows, r = row - bc * j.rows, i = r / j.G, b = bc / Hk, head = (bc - b * Hk) * j.G + r - i * j.G;
    const float y[4] = {f[0], f[1], f[2], f[3]};
    store4((T*)j.out.data + b * j.out.b + i * j.out.l + head * j.out.h, d, D, j.out.vec, y);
}

// Rows and their gradients stay in registers; two workgroups a compute unit up to 128 features in bf16.
template <class X, int DP>
struct QueryChoice {
    static constexpr int kRow = DP * (int)sizeof(typename Matrix<X>::E);
    typedef QueryConfig<kRow <= 256 ? 64 : 32, kRow <= 128 ? 3 : kRow <= 256 ? 2 : kRow <= 512 ? 4 : kRow <= 768 ? 2 : 1,
                        kRow <= 256 && sizeof(typename Matrix<X>::E) == 2 ? 2 : 1> C;
};
template <int DP>
struct QueryChoice<Parts, DP> { typedef QueryConfig<32, 3, DP <= 64 ? 2 : 1> C; };
// Keys and values in registers where the sums leave room for them, one wavefront a SIMD where they do not leave room for two.
// Two take 8 wavefronts that share a tile of rows: causal training of 2 x 4096 x 16 heads on 4 of 128, capped, took 893 us in
// all with two a SIMD, 1037 with one.
template <class X, int DP>
struct KeyChoice { typedef KeyConfig<X, DP, 4, 1, 2, false, false, 1> C; };
template <int DP>
struct KeyChoice<Parts, DP> { typedef KeyConfig<Parts, DP, 4, 1, 3, false, false, DP <= 32 ? 2 : 1> C; };
template <>
struct KeyChoice<bf16, 32> { typedef KeyConfig<bf16, 32, 4, 2, 2, false, false, 2> C; };
template <>
struct KeyChoice<bf16, 64> { typedef KeyConfig<bf16, 64, 4, 2, 2, false, false, 2> C; };
template <>
struct KeyChoice<bf16, 96> { typedef KeyConfig<bf16, 96, 4, 2, 2, false, true, 2> C; };
template <>
struct KeyChoice<bf16, 128> { typedef KeyConfig<bf16, 128, 4, 2, 2, true, true, 2> C; };
template <>
struct KeyChoice<bf16, 256> { typedef KeyConfig<bf16, 256, 4, 1, 2, false, true, 1> C; };
template <>
struct KeyChoice<float, 192> { typedef KeyConfig<float, 192, 2, 1, 1, false, true, 1> C; };
template <>
struct KeyChoice<float, 256> { typedef KeyConfig<float, 256, 2, 1, 1, false, true, 1> C; };

template <class T>
void add_parts(const Params& p, hipStream_t stream) {
    AllPartsToAdd all;
    unsigned n = 0, most = 0;
    auto add = [&](const float* part, const Tensor& out, int splits, int rows, int G) {
        all.of[n++] = {part, out, (unsigned)splits, (unsigned)rows, (unsigned)G};
        most = std::max(most, (unsigned)rows);
    };
    if (p.dq_splits > 1) add(p.part_dq, p.dq, p.dq_splits, p.R, p.G);
    if (p.dk_splits > 1) {
        add(p.part_dk, p.dk, p.dk_splits, p.Lk, 1);
        add(p.part_dv, p.dv, p.dk_splits, p.Lk, 1);
    }
    if (n == 0) return;
    const unsigned items = p.B * p.Hk * most * ((p.D + 3) / 4);
    launch("adhip_attention_backward", add_parts_kernel<T>, dim3((items + 255) / 256, n), 256, stream, all, (unsigned)p.B, (unsigned)p.Hk, p.D);
}

template <class X, int DP>
void launch_backward(const Params& p, hipStream_t stream) {
    typedef typename Matrix<X>::IO T;
    typedef typename QueryChoice<X, DP>::C Q;
    typedef typename KeyChoice<X, DP>::C K;
    Params x = p;
    const bool vec = p.q.vec && p.k.vec && p.v.vec && p.out.vec && p.dout.vec;
    x.tiles = (p.R + Q::BQ - 1) / Q::BQ;
    unsigned grid = (unsigned)((int64_t)x.tiles * p.dq_splits * p.Hk * p.B);
    const char* const op = "adhip_attention_backward";
    if (grid > 0) launch(op, vec ? query_gradient_kernel<X, DP, true, Q> : query_gradient_kernel<X, DP, false, Q>, grid, Q::NT, stream, x);
    x.tiles = (p.Lk + K::BKEYS - 1) / K::BKEYS;
    grid = (unsigned)((int64_t)x.tiles * p.dk_splits * p.Hk * p.B);
    if (grid > 0) launch(op, vec ? key_gradient_kernel<X, DP, true, K> : key_gradient_kernel<X, DP, false, K>, grid, K::NT, stream, x);
    add_parts<T>(p, stream);
}

}  // namespace attn
}  // namespace adhip

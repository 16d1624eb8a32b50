// Attention backward.  With p = exp(z - lse), dp = dout.v, delta = dout.out and  ds = p (dp - delta) (1 - (z_cap / cap)^2):
//     dq = scale ds k,   dk = scale ds^T q,   dv = p^T dout.
//
// Two kernels, each of which computes the scores again: one owns rows and walks the keys (dq, and delta on the way), one
// owns keys and walks the rows of all heads that share them (dk, dv).  That is seven products where one kernel with dq in
// atomic additions would take five, but nothing is added in an order that changes from run to run, dq takes no memory in
// f32, and heads that share keys add up in registers.
#pragma once
#include "operator_attention.hpp"

namespace adhip {
namespace attn {

// ---- dq: the forward kernel's walk ------------------------------------------------------------------------------------

template <class T, int DP, int BK_, int AHEAD_>
struct QueryConfig {
    static constexpr int BK = BK_, AHEAD = AHEAD_, NT = 256, BQ = 128, KB = BK / 32;
    static constexpr int kTile = BK * Lds<T, DP>::kPitch, kBufs = AHEAD == 2 ? 2 : 1;
    static constexpr int kBytes = kBufs * (2 * kTile * (int)sizeof(T) + BK * 4);
};

template <class T, int DP, class C>
__global__ __launch_bounds__(C::NT) void query_gradient_kernel(const Params p) {
    typedef Matrix<T> M;
    typedef typename M::Frag Frag;
    __shared__ __attribute__((aligned(16))) char lds[C::kBytes];
    T* const ks = (T*)lds;
    T* const vs = ks + C::kBufs * C::kTile;
    int* const docs = (int*)(vs + C::kBufs * C::kTile);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    const int total = p.tiles * p.Hk * p.B;
    int id = by_die(blockIdx.x, total);
    if (id >= total) return;
    const int tile = p.tiles - 1 - id % p.tiles;
    id /= p.tiles;
    const int c = id % p.Hk, b = id / p.Hk;

    const int n = sequence_length(p, b), offset = n - p.Lq;
    const int prefix = p.prefix ? min(max(p.prefix[b * p.prefix_s], 0), n) : 0;
    const Band band(p);
    const Scoring sc(p);
    const int row0 = tile * C::BQ, row1 = min(row0 + C::BQ, p.R) - 1;
    const int first = row0 / p.G, last = row1 / p.G;

    const int row = row0 + wave * 32 + (lane & 31);
    bool valid = row < p.R;
    const int token = valid ? row / p.G : 0, head = c * p.G + (valid ? row - token * p.G : 0);
    const int at = token + offset;
    int lo = at - band.below, hi = at + band.above, pre = prefix;
    const int doc = p.qdoc && valid ? p.qdoc[b * p.qdoc_b + token * p.qdoc_l] : 0;
    const float slope = p.slopes && valid ? p.slopes[head * p.slope_stride] * kLog2e : 0.f;
    const float lse = valid ? p.lse[b * p.lse_b + token * p.lse_l + head * p.lse_h] : -__builtin_inff();
    const bool inside = valid;
    // a row that sees nothing has no gradient, whatever dout holds there
    if (lse == -__builtin_inff()) valid = false;
    if (!valid || doc < 0) lo = 1, hi = 0, pre = 0;
    const float lse2 = lse * kLog2e;

    Frag qf[DP / 16], df[DP / 16];
    float delta = 0.f;
    {
        const T* q = (const T*)p.q.data + b * p.q.b + token * p.q.l + head * p.q.h;
        const T* d = (const T*)p.dout.data + b * p.dout.b + token * p.dout.l + head * p.dout.h;
        const T* o = (const T*)p.out.data + b * p.out.b + token * p.out.l + head * p.out.h;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            qf[s] = load_frag(q, s * 16 + half * 8, p.D, p.q.vec, valid);
            df[s] = load_frag(d, s * 16 + half * 8, p.D, p.dout.vec, valid);
            const Frag of = load_frag(o, s * 16 + half * 8, p.D, p.out.vec, valid);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta += (float)df[s][e] * (float)of[e];
        }
    }
    delta += __shfl_xor(delta, 32);
    if (inside && half == 0) p.delta[((int64_t)b * p.Hk + c) * p.R + row] = delta;
    f32x16 dq[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dq[d] = zero16();

    const int hi_all = last + offset + band.above, lo_all = first + offset - band.below;
    const int2* const kr = p.krange ? p.krange + (int64_t)b * p.kranges : nullptr;
    int2 mine = {0, 0};
    if (kr) mine = document_range(p.qrange + (int64_t)b * p.qranges, first, last);
    auto needed = [&](int t) {
        const int j0 = t * C::BK, j1 = min(j0 + C::BK, n) - 1;
        if (j0 >= prefix && (j0 > hi_all || j1 < lo_all)) return false;
        if (!kr) return true;
        const int2 theirs = document_range(kr, j0, j1);
        return theirs.x <= mine.y && mine.x <= theirs.y;
    };
    Tiles<decltype(needed)> tiles(needed, 0, (n + C::BK - 1) / C::BK);

    const T* const kb = (const T*)p.k.data + b * p.k.b + c * p.k.h;
    const T* const vb = (const T*)p.v.data + b * p.v.b + c * p.v.h;
    const int* const kd = p.kdoc ? p.kdoc + b * p.kdoc_b : nullptr;
    Stage<T, DP, C::BK, C::NT> sk, sv;
    int sd = 0;
    auto used = [&](int j) { return j < n && !(kd && kd[j * p.kdoc_l] < 0); };
    auto load_k = [&](int j0) { sk.load([&](int i) { return used(j0 + i) ? kb + (j0 + i) * p.k.l : (const T*)nullptr; }, p.D, p.k.vec, tid); };
    auto load_v = [&](int j0) { sv.load([&](int i) { return used(j0 + i) ? vb + (j0 + i) * p.v.l : (const T*)nullptr; }, p.D, p.v.vec, tid); };
    auto load_d = [&](int j0) { if (kd && tid < C::BK) sd = j0 + tid < n ? kd[(j0 + tid) * p.kdoc_l] : -1; };
    auto load = [&](int t) {
        load_k(t * C::BK);
        load_v(t * C::BK);
        load_d(t * C::BK);
    };
    static_assert(C::NT >= C::BK, "one thread a key for the documents");
    auto store_d = [&](int buf) { if (kd && tid < C::BK) docs[buf * C::BK + tid] = sd; };
    auto store = [&](int buf) {
        sk.store(ks + buf * C::kTile, tid);
        sv.store(vs + buf * C::kTile, tid);
        store_d(buf);
    };

    int t = tiles.next(lane), buf = 0;
    if (C::AHEAD == 2) {
        if (t >= 0) {
            load(t);
            store(0);
        }
        __syncthreads();
    }
    while (t >= 0) {
        const int next = tiles.next(lane);
        if (C::AHEAD == 2) {
            if (next >= 0) load(next);
        } else {
            __syncthreads();
            load_k(t * C::BK);
            sk.store(ks, tid);
            load_v(t * C::BK);
            sv.store(vs, tid);
            load_d(t * C::BK);
            store_d(0);
            __syncthreads();
        }
        const T* kt = ks + buf * C::kTile;
        const T* vt = vs + buf * C::kTile;
        const int* dt = docs + buf * C::BK;
#pragma unroll
        for (int x = 0; x < C::KB; ++x) {
            const int key0 = x * 32;
            f32x16 s = zero16(), g = zero16();
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) s = M::mma(rows_frag<T, DP>(kt, key0, k, lane), qf[k], s);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) g = M::mma(rows_frag<T, DP>(vt, key0, k, lane), df[k], g);
            const int j0 = t * C::BK + key0, jl = j0 + 4 * half;
            const bool masked = kd || !__all(j0 + 31 < n && ((lo <= j0 && j0 + 31 <= hi) || j0 + 31 < pre));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float z, bend = 1.f;
                if (p.cap > 0.f) {
                    const float y = tanh_of(s[i] * sc.cap_in);
                    z = y * sc.cap_out;
                    bend = 1.f - y * y;
                } else {
                    z = s[i] * sc.scale2;
                }
                if (p.slopes) z -= slope * fabsf((float)(at - jl - c_row(i)));
                const float w = __builtin_amdgcn_exp2f(z - lse2);
                float ds = w * (g[i] - delta) * bend;
                if (masked) {
                    const int j = jl + c_row(i);
                    bool sees = j < n && (j < pre || (lo <= j && j <= hi));
                    if (kd) sees = sees && dt[key0 + 4 * half + c_row(i)] == doc;
                    ds = sees ? ds : 0.f;
                }
                s[i] = ds;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag f;
                to_frag(s, h, f);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) dq[d] = M::mma(cols_frag<DP>(kt, key0 + 16 * h, d * 32, lane), f, dq[d]);
            }
        }
        if (C::AHEAD == 2) {
            buf ^= 1;
            if (next >= 0) store(buf);
            __syncthreads();
        }
        t = next;
    }
    if (!inside) return;
    T* out = (T*)p.dq.data + b * p.dq.b + token * p.dq.l + head * p.dq.h;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float f[4] = {dq[d][4 * g] * p.scale, dq[d][4 * g + 1] * p.scale, dq[d][4 * g + 2] * p.scale, dq[d][4 * g + 3] * p.scale};
            store4(out, d * 32 + 8 * g + 4 * half, p.D, p.dq.vec, f);
        }
}

// ---- dk, dv -------------------------------------------------------------------------------------------------------------

// NW wavefronts own 32 keys each and walk tiles of BR rows.  V_LDS: the values are read from LDS, where registers hold no
// more than keys and two sums.
template <class T, int DP, int NW_, int BR_, int AHEAD_, bool V_LDS_>
struct KeyConfig {
    static constexpr int NW = NW_, BR = BR_, AHEAD = AHEAD_, NT = 64 * NW, BKEYS = 32 * NW;
    static constexpr bool V_LDS = V_LDS_;
    static constexpr int kTile = BR * Lds<T, DP>::kPitch, kBufs = AHEAD == 2 ? 2 : 1;
    static constexpr int kValues = V_LDS ? BKEYS * Lds<T, DP>::kPitch : 0;
    static constexpr int kBytes = (kBufs * 2 * kTile + kValues) * (int)sizeof(T) + kBufs * BR * 5 * 4;
};

template <class T, int DP, class C>
__global__ __launch_bounds__(C::NT) void key_gradient_kernel(const Params p) {
    typedef Matrix<T> M;
    typedef typename M::Frag Frag;
    __shared__ __attribute__((aligned(16))) char lds[C::kBytes];
    T* const qs = (T*)lds;                       // [bufs][BR][pitch]
    T* const gs = qs + C::kBufs * C::kTile;      // dout
    T* const vs = gs + C::kBufs * C::kTile;      // [BKEYS][pitch] where V_LDS
    float* const rows = (float*)(vs + C::kValues);  // [bufs][5][BR]: lse, delta, position, slope, document
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    const int total = p.tiles * p.Hk * p.B;
    int id = by_die(blockIdx.x, total);
    if (id >= total) return;
    const int tile = id % p.tiles;  // the first ones, which most rows see, first
    id /= p.tiles;
    const int c = id % p.Hk, b = id / p.Hk;

    const int n = sequence_length(p, b), offset = n - p.Lq;
    const int prefix = p.prefix ? min(max(p.prefix[b * p.prefix_s], 0), n) : 0;
    const Band band(p);
    const Scoring sc(p);
    const int key_first = tile * C::BKEYS, key_last = min(key_first + C::BKEYS, n) - 1;
    const int key = key_first + wave * 32 + (lane & 31);
    const int doc = p.kdoc && key < n ? p.kdoc[b * p.kdoc_b + key * p.kdoc_l] : 0;
    const bool valid = key < n && doc >= 0;
    // rows at positions from .. to see this key (limits of the sequence aside), all rows where it is in the prefix
    int from = key - band.above, to = key + band.below;
    if (key < prefix) from = -0x7fffffff, to = 0x7fffffff;
    if (!valid) from = 1, to = 0;

    Frag kf[DP / 16], vf[C::V_LDS ? 1 : DP / 16];
    {
        const T* k = (const T*)p.k.data + b * p.k.b + key * p.k.l + c * p.k.h;
        const T* v = (const T*)p.v.data + b * p.v.b + key * p.v.l + c * p.v.h;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            kf[s] = load_frag(k, s * 16 + half * 8, p.D, p.k.vec, valid);
            const Frag f = load_frag(v, s * 16 + half * 8, p.D, p.v.vec, valid);
            if (C::V_LDS) *(Frag*)(vs + (wave * 32 + (lane & 31)) * Lds<T, DP>::kPitch + s * 16 + half * 8) = f;
            else vf[s] = f;
        }
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dk[d] = zero16(), dv[d] = zero16();

    const int2* const qr = p.qrange ? p.qrange + (int64_t)b * p.qranges : nullptr;
    int2 mine = {0, 0};
    if (qr && key_last >= key_first) mine = document_range(p.krange + (int64_t)b * p.kranges, key_first, key_last);
    auto needed = [&](int t) {
        const int i0 = t * C::BR / p.G, i1 = (min((t + 1) * C::BR, p.R) - 1) / p.G;
        if (key_first >= prefix && (i1 + offset < key_first - band.above || i0 + offset > key_last + band.below)) return false;
        if (!qr) return true;
        const int2 theirs = document_range(qr, i0, i1);
        return theirs.x <= mine.y && mine.x <= theirs.y;
    };
    Tiles<decltype(needed)> tiles(needed, 0, key_last >= key_first ? (p.R + C::BR - 1) / C::BR : 0);

    const T* const qb = (const T*)p.q.data + b * p.q.b + (int64_t)c * p.G * p.q.h;
    const T* const gb = (const T*)p.dout.data + b * p.dout.b + (int64_t)c * p.G * p.dout.h;
    const float* const lb = p.lse + b * p.lse_b + (int64_t)c * p.G * p.lse_h;
    const float* const eb = p.delta + ((int64_t)b * p.Hk + c) * p.R;
    Stage<T, DP, C::BR, C::NT> sq, sg;
    float r_lse = 0.f, r_delta = 0.f, r_slope = 0.f;
    int r_at = 0, r_doc = 0;
    // the row's log-sum, or -inf where it sees nothing: such rows are zero, whatever the arrays hold there
    auto row_lse = [&](int r, int i, int g) { return r < p.R ? lb[i * p.lse_l + g * p.lse_h] : -__builtin_inff(); };
    auto load_q = [&](int r0) {
        sq.load([&](int x) {
            const int r = r0 + x, i = r / p.G, g = r - i * p.G;
            return row_lse(r, i, g) != -__builtin_inff() ? qb + i * p.q.l + g * p.q.h : (const T*)nullptr;
        }, p.D, p.q.vec, tid);
    };
    auto load_g = [&](int r0) {
        sg.load([&](int x) {
            const int r = r0 + x, i = r / p.G, g = r - i * p.G;
            return row_lse(r, i, g) != -__builtin_inff() ? gb + i * p.dout.l + g * p.dout.h : (const T*)nullptr;
        }, p.D, p.dout.vec, tid);
    };
    static_assert(C::NT >= C::BR, "one thread a row for what rows have beside features");
    auto load_r = [&](int r0) {
        if (tid >= C::BR) return;
        const int r = r0 + tid, i = r / p.G, g = r - i * p.G;
        const float x = row_lse(r, i, g);
        const bool some = x != -__builtin_inff();
        r_lse = some ? x * kLog2e : __builtin_inff();  // p = exp2(z - inf) = 0
        r_delta = some ? eb[r] : 0.f;
        r_at = i + offset;
        r_slope = p.slopes && some ? p.slopes[(c * p.G + g) * p.slope_stride] * kLog2e : 0.f;
        r_doc = p.qdoc && some ? p.qdoc[b * p.qdoc_b + i * p.qdoc_l] : -1;
    };
    auto store_r = [&](int buf) {
        if (tid >= C::BR) return;
        float* to_rows = rows + buf * 5 * C::BR + tid;
        to_rows[0] = r_lse;
        to_rows[C::BR] = r_delta;
        to_rows[2 * C::BR] = __int_as_float(r_at);
        to_rows[3 * C::BR] = r_slope;
        to_rows[4 * C::BR] = __int_as_float(r_doc);
    };

    int t = tiles.next(lane), buf = 0;
    if (C::AHEAD == 2) {
        if (t >= 0) {
            load_q(t * C::BR);
            load_g(t * C::BR);
            load_r(t * C::BR);
            sq.store(qs, tid);
            sg.store(gs, tid);
            store_r(0);
        }
        __syncthreads();
    }
    while (t >= 0) {
        const int next = tiles.next(lane);
        if (C::AHEAD == 2) {
            if (next >= 0) {
                load_q(next * C::BR);
                load_g(next * C::BR);
                load_r(next * C::BR);
            }
        } else {
            __syncthreads();
            load_q(t * C::BR);
            sq.store(qs, tid);
            load_g(t * C::BR);
            sg.store(gs, tid);
            load_r(t * C::BR);
            store_r(0);
            __syncthreads();
        }
        const T* qt = qs + buf * C::kTile;
        const T* gt = gs + buf * C::kTile;
        const float* rt = rows + buf * 5 * C::BR;
#pragma unroll
        for (int x = 0; x < C::BR / 32; ++x) {
            const int q0 = x * 32, first_at = (t * C::BR + q0) / p.G + offset, last_at = (t * C::BR + q0 + 31) / p.G + offset;
            const bool masked = p.qdoc || !__all(from <= first_at && last_at <= to);
            f32x16 s = zero16();
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) s = M::mma(rows_frag<T, DP>(qt, q0, k, lane), kf[k], s);
            f32x16 bend;
            const float* own = rt + q0 + 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float z;
                if (p.cap > 0.f) {
                    const float y = tanh_of(s[i] * sc.cap_in);
                    z = y * sc.cap_out;
                    bend[i] = 1.f - y * y;
                } else {
                    z = s[i] * sc.scale2;
                    bend[i] = 1.f;
                }
                const int at = __float_as_int(own[2 * C::BR + c_row(i)]);
                if (p.slopes) z -= own[3 * C::BR + c_row(i)] * fabsf((float)(at - key));
                float w = __builtin_amdgcn_exp2f(z - own[c_row(i)]);
                if (masked) {
                    bool sees = from <= at && at <= to;
                    if (p.qdoc) sees = sees && __float_as_int(own[4 * C::BR + c_row(i)]) == doc;
                    w = sees ? w : 0.f;
                    bend[i] = sees ? bend[i] : 0.f;
                }
                s[i] = w;
            }
            f32x16 g = zero16();
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                if (C::V_LDS) g = M::mma(rows_frag<T, DP>(gt, q0, k, lane), rows_frag<T, DP>(vs, wave * 32, k, lane), g);
                else g = M::mma(rows_frag<T, DP>(gt, q0, k, lane), vf[C::V_LDS ? 0 : k], g);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag f;
                to_frag(s, h, f);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) dv[d] = M::mma(cols_frag<DP>(gt, q0 + 16 * h, d * 32, lane), f, dv[d]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = s[i] * (g[i] - own[C::BR + c_row(i)]) * bend[i];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag f;
                to_frag(s, h, f);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) dk[d] = M::mma(cols_frag<DP>(qt, q0 + 16 * h, d * 32, lane), f, dk[d]);
            }
        }
        if (C::AHEAD == 2) {
            buf ^= 1;
            if (next >= 0) {
                sq.store(qs + buf * C::kTile, tid);
                sg.store(gs + buf * C::kTile, tid);
                store_r(buf);
            }
            __syncthreads();
        }
        t = next;
    }
    if (key >= p.Lk) return;
    T* ko = (T*)p.dk.data + b * p.dk.b + key * p.dk.l + c * p.dk.h;
    T* vo = (T*)p.dv.data + b * p.dv.b + key * p.dv.l + c * p.dv.h;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float f[4] = {dk[d][4 * g] * p.scale, dk[d][4 * g + 1] * p.scale, dk[d][4 * g + 2] * p.scale, dk[d][4 * g + 3] * p.scale};
            const float e[4] = {dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]};
            store4(ko, d * 32 + 8 * g + 4 * half, p.D, p.dk.vec, f);
            store4(vo, d * 32 + 8 * g + 4 * half, p.D, p.dv.vec, e);
        }
}

template <class T, int DP>
struct BackwardConfig {
    static constexpr int kRowBytes = DP * (int)sizeof(T);
    typedef QueryConfig<T, DP, sizeof(T) == 2 ? 64 : 32, kRowBytes <= 512 ? 2 : 0> Q;
    typedef KeyConfig<T, DP, kRowBytes <= 512 ? 4 : 2, 32, kRowBytes <= 512 ? 2 : 0, (kRowBytes > 512)> K;
};

template <class T, int DP>
void launch_backward(const Params& p, hipStream_t stream) {
    typedef typename BackwardConfig<T, DP>::Q Q;
    typedef typename BackwardConfig<T, DP>::K K;
    Params x = p;
    x.tiles = (p.R + Q::BQ - 1) / Q::BQ;
    if (x.tiles > 0) query_gradient_kernel<T, DP, Q><<<die_grid((int64_t)x.tiles * p.Hk * p.B), Q::NT, 0, stream>>>(x);
    check_launch("adhip_attention_backward");
    x.tiles = (p.Lk + K::BKEYS - 1) / K::BKEYS;
    if (x.tiles > 0) key_gradient_kernel<T, DP, K><<<die_grid((int64_t)x.tiles * p.Hk * p.B), K::NT, 0, stream>>>(x);
    check_launch("adhip_attention_backward");
}

template <class T>
void backward(const Params& p, hipStream_t stream) {
    switch (padded_size(p.D)) {
        case 32: return launch_backward<T, 32>(p, stream);
        case 64: return launch_backward<T, 64>(p, stream);
        case 96: return launch_backward<T, 96>(p, stream);
        case 128: return launch_backward<T, 128>(p, stream);
        case 192: return launch_backward<T, 192>(p, stream);
        case 256: return launch_backward<T, 256>(p, stream);
    }
}

}  // namespace attn
}  // namespace adhip

// AdamW (Loshchilov and Hutter 2019) over many tensors in one launch, states in 32 bits or, after Dettmers et al. 2022, in
// 8 bits with a scale for each block of 256 elements.
//
// Memory bounds it: every element's parameter, gradient and two moments are read once and the first and the last two
// written once (28 bytes in 32 bits, 10 with bf16 and 8-bit states).  A wavefront takes blocks of 256 elements, four a
// lane, so that a block's largest element is one reduction over its lanes; UNITS blocks are loaded before the first is
// used.  The tensors' addresses travel as kernel arguments: nothing is copied to the device before the launch.
// 38 M elements in 32 bits: 191 us, 5.5 TB/s; 17.7 M in bf16 with 8-bit states: 44 us, 4.1 TB/s, where the correctly rounded
// divisions and roots take as long as memory.
//
// Eight bits are e4m3 numbers (three bits of mantissa, 2^-9 .. 448) times the block's scale.  The second moment is held
// as its root, which halves the range it spans, and never becomes zero by rounding: the first moment is divided by that
// root, and a root of zero beside a first moment that is none would throw the parameter by |m| / eps.
//
// The arithmetic is the written formula's, each operation rounded by itself (no contraction), so that a code is the same
// wherever it is computed.
#include "operators.hpp"

#include <cmath>

#pragma clang fp contract(off)

namespace adhip {
namespace {

constexpr int kTensors = 32;           // of a launch: their descriptors stay within 4 KiB of kernel arguments
constexpr int kBlock = ADHIP_ADAMW_BLOCK;
constexpr int kUnits = 4;              // blocks of 256 that a wavefront has under way
constexpr int kChunk = 4 * kUnits * kBlock;  // elements of a workgroup (four wavefronts)
constexpr uint64_t kBlocks = 0xffffffffu / 256;  // workgroups of a launch: it holds fewer than 2^32 threads

struct AdamwLaunch {
    adhip_adamw_tensor t[kTensors];
    unsigned first[kTensors + 1];  // the workgroup that begins each tensor
    int n;
    unsigned aligned;              // bit i: every array of tensor i can be read four elements at once
    float grad_scale, beta1, grow1, beta2, grow2, root_scale, eps, keep, rate;
};

template <class T>
__device__ __forceinline__ void load4(const T* x, int64_t i, int64_t n, bool whole, float (&f)[4]) {
    if (whole) {
        const Pack<T, 4> r = *(const Pack<T, 4>*)(x + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = (float)r.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = i + k < n ? (float)x[i + k] : 0.f;
    }
}

template <class T>
__device__ __forceinline__ void store4(T* x, int64_t i, int64_t n, bool whole, const float (&f)[4]) {
    if (whole) {
        Pack<T, 4> r;
#pragma unroll
        for (int k = 0; k < 4; ++k) r.v[k] = (T)f[k];
        *(Pack<T, 4>*)(x + i) = r;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) x[i + k] = (T)f[k];
    }
}

// codes of four e4m3 numbers
__device__ __forceinline__ void decode4(unsigned c, float (&f)[4]) {
    f[0] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
    f[1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1);
    f[2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2);
    f[3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3);
}
__device__ __forceinline__ unsigned encode4(const float (&f)[4]) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], c, true);
}

// The largest of a wavefront's values, in all lanes: within 16 lanes by rotations, then by exchanges of rows.
template <int CTRL>
__device__ __forceinline__ unsigned max_with(unsigned x) {
    return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ unsigned wave_max(unsigned x) {
    x = max_with<0xb1>(x);   // the other of a pair
    x = max_with<0x4e>(x);   // the other pair of four
    x = max_with<0x124>(x);  // four and eight lanes round
    x = max_with<0x128>(x);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(r[0], r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(h[0], h[1]);
}

// The scale of a block from its values: their largest magnitude, by the bits, so that a NaN is the largest of all.
__device__ __forceinline__ float block_scale(const float (&f)[4]) {
    unsigned most = __float_as_uint(0x1p-100f);
#pragma unroll
    for (int k = 0; k < 4; ++k) most = max(most, __float_as_uint(f[k]) & 0x7fffffffu);
    return __uint_as_float(wave_max(most)) * (1.f / 448.f);
}

// x / scale for the four values of a lane, rounded correctly: from the scale's reciprocal, with one correction by the exact
// remainder (Markstein 1990); a scale that is not finite takes the divisions.
__device__ __forceinline__ void over_scale(const float (&x)[4], float scale, float (&q)[4]) {
    if (scale < __builtin_inff()) {
        const float r = 1.f / scale;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float y = x[k] * r;
            q[k] = __builtin_fmaf(__builtin_fmaf(-y, scale, x[k]), r, y);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = x[k] / scale;
    }
}

// A wavefront's blocks of a tensor.  WHOLE: all of them are there and can be read four elements at once; then no load waits
// for a choice, and all are under way together.
template <class PT, class GT, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void adamw_blocks(const AdamwLaunch& a, const adhip_adamw_tensor& t, bool aligned, int64_t unit0, int lane) {
    const int64_t n = t.count;
    float p[kUnits][4], g[kUnits][4], m[kUnits][4], v[kUnits][4];
    unsigned mc[kUnits], vc[kUnits];
    float ms[kUnits], vs[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t at = (unit0 + u) * kBlock + lane * 4;
        if (!WHOLE && (unit0 + u) * kBlock >= n) break;
        const bool whole = WHOLE || (aligned && at + 4 <= n);
        load4((const PT*)t.p, at, n, whole, p[u]);
        load4((const GT*)t.g, at, n, whole, g[u]);
        if (EIGHT) {
            mc[u] = ((const unsigned*)t.m)[(unit0 + u) * 64 + lane];
            vc[u] = ((const unsigned*)t.v)[(unit0 + u) * 64 + lane];
            ms[u] = t.m_scale[unit0 + u];
            vs[u] = t.v_scale[unit0 + u];
        } else {
            load4((const float*)t.m, at, n, whole, m[u]);
            load4((const float*)t.v, at, n, whole, v[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t at = (unit0 + u) * kBlock + lane * 4;
        if (!WHOLE && (unit0 + u) * kBlock >= n) return;
        const bool whole = WHOLE || (aligned && at + 4 <= n);
        float root[4];
        if (EIGHT) {
            decode4(mc[u], m[u]);
            decode4(vc[u], v[u]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (EIGHT) {
                m[u][k] *= ms[u];
                const float r = v[u][k] * vs[u];
                v[u][k] = r * r;
            }
            const float x = g[u][k] * a.grad_scale;
            m[u][k] = m[u][k] * a.beta1 + x * a.grow1;
            v[u][k] = v[u][k] * a.beta2 + x * x * a.grow2;
            root[k] = sqrtf(v[u][k]);
            const float under = root[k] * a.root_scale + a.eps;
            p[u][k] = p[u][k] * a.keep - m[u][k] / under * a.rate;
        }
        store4((PT*)t.p_out, at, n, whole, p[u]);
        if (EIGHT) {
            // what lies behind the tensor's end stays zero
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (at + k >= n) m[u][k] = root[k] = 0.f;
            const float m_scale = block_scale(m[u]), v_scale = block_scale(root);
            float c[4];
            over_scale(m[u], m_scale, c);
            ((unsigned*)t.m_out)[(unit0 + u) * 64 + lane] = encode4(c);
            over_scale(root, v_scale, c);
#pragma unroll
            for (int k = 0; k < 4; ++k) c[k] = root[k] > 0.f ? (c[k] < 0x1p-9f ? 0x1p-9f : c[k]) : root[k];
            ((unsigned*)t.v_out)[(unit0 + u) * 64 + lane] = encode4(c);
            if (lane == 0) {
                t.m_scale_out[unit0 + u] = m_scale;
                t.v_scale_out[unit0 + u] = v_scale;
            }
        } else {
            store4((float*)t.m_out, at, n, whole, m[u]);
            store4((float*)t.v_out, at, n, whole, v[u]);
        }
    }
}

template <class PT, class GT, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwLaunch a) {
    int i = 0;
    while (i + 1 < a.n && blockIdx.x >= a.first[i + 1]) ++i;
    const adhip_adamw_tensor t = a.t[i];
    const bool aligned = a.aligned >> i & 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t unit0 = (int64_t)(blockIdx.x - a.first[i]) * (kChunk / kBlock) + wave * kUnits;
    if (aligned && (unit0 + kUnits) * kBlock <= t.count) adamw_blocks<PT, GT, EIGHT, true>(a, t, aligned, unit0, lane);
    else adamw_blocks<PT, GT, EIGHT, false>(a, t, aligned, unit0, lane);
}

template <bool EIGHT>
void launch_adamw(const char* op, const AdamwLaunch& a, int p_type, int g_type, unsigned blocks, hipStream_t stream) {
    if (p_type == ADHIP_F32 && g_type == ADHIP_F32) launch(op, adamw_kernel<float, float, EIGHT>, blocks, 256, stream, a);
    else if (p_type == ADHIP_F32) launch(op, adamw_kernel<float, bf16, EIGHT>, blocks, 256, stream, a);
    else if (g_type == ADHIP_F32) launch(op, adamw_kernel<bf16, float, EIGHT>, blocks, 256, stream, a);
    else launch(op, adamw_kernel<bf16, bf16, EIGHT>, blocks, 256, stream, a);
}

bool aligned_to(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

void adamw(const adhip_adamw_args& g, hipStream_t stream) {
    const char* op = "adhip_adamw";
    ADHIP_CHECK(g.p_type == ADHIP_F32 || g.p_type == ADHIP_BF16, "%s: parameters are %s, f32 or bf16 is wanted", op, type_name(g.p_type));
    ADHIP_CHECK(g.g_type == ADHIP_F32 || g.g_type == ADHIP_BF16, "%s: gradients are %s, f32 or bf16 is wanted", op, type_name(g.g_type));
    ADHIP_CHECK(g.state_type == ADHIP_F32 || g.state_type == ADHIP_E4M3, "%s: states are %s, f32 or e4m3 is wanted", op, type_name(g.state_type));
    ADHIP_CHECK(g.n_tensors >= 0 && (g.tensors || g.n_tensors == 0), "%s: no tensors", op);
    ADHIP_CHECK(g.step >= 1, "%s: step %d: the first step is 1", op, (int)g.step);
    ADHIP_CHECK(g.beta1 >= 0 && g.beta1 < 1 && g.beta2 >= 0 && g.beta2 < 1, "%s: betas %g and %g are not in [0, 1)", op, g.beta1, g.beta2);
    ADHIP_CHECK(g.eps >= 0 && std::isfinite(g.eps) && std::isfinite(g.rate) && std::isfinite(g.decay) && std::isfinite(g.grad_scale),
                "%s: eps must not be negative, and eps, rate, decay and grad_scale finite", op);
    const bool eight = g.state_type == ADHIP_E4M3;
    const size_t pw = (size_t)type_bytes(g.p_type), gw = (size_t)type_bytes(g.g_type);
    for (int64_t i = 0; i < g.n_tensors; ++i) {
        const adhip_adamw_tensor& t = g.tensors[i];
        const long long at = (long long)i;
        ADHIP_CHECK(t.count >= 0 && t.count <= (int64_t)kBlocks * kChunk, "%s: tensor %lld has %lld elements", op, at, (long long)t.count);
        if (t.count == 0) continue;
        ADHIP_CHECK(t.p && t.g && t.m && t.v && t.p_out && t.m_out && t.v_out, "%s: an array of tensor %lld is missing", op, at);
        ADHIP_CHECK(!eight || (t.m_scale && t.v_scale && t.m_scale_out && t.v_scale_out), "%s: a scale array of tensor %lld is missing", op, at);
        ADHIP_CHECK(aligned_to(t.p, pw) && aligned_to(t.p_out, pw) && aligned_to(t.g, gw), "%s: an array of tensor %lld is not aligned to its type", op, at);
        // codes are read four at once: a block of them begins at a multiple of four
        for (const void* s : {t.m, t.v, (const void*)t.m_out, (const void*)t.v_out, (const void*)t.m_scale, (const void*)t.v_scale,
                              (const void*)t.m_scale_out, (const void*)t.v_scale_out})
            ADHIP_CHECK(aligned_to(s, 4), "%s: a state array of tensor %lld is not aligned to 4 bytes", op, at);
    }
    AdamwLaunch a = {};
    a.grad_scale = (float)g.grad_scale;
    a.beta1 = (float)g.beta1;
    a.grow1 = (float)(1.0 - g.beta1);
    a.beta2 = (float)g.beta2;
    a.grow2 = (float)(1.0 - g.beta2);
    a.root_scale = (float)(1.0 / std::sqrt(1.0 - std::pow(g.beta2, g.step)));
    a.eps = (float)g.eps;
    a.keep = (float)(1.0 - g.rate * g.decay);
    a.rate = (float)(g.rate / (1.0 - std::pow(g.beta1, g.step)));
    uint64_t blocks = 0;
    auto flush = [&] {
        if (a.n == 0) return;
        if (eight) launch_adamw<true>(op, a, g.p_type, g.g_type, (unsigned)blocks, stream);
        else launch_adamw<false>(op, a, g.p_type, g.g_type, (unsigned)blocks, stream);
        a.n = 0;
        a.aligned = 0;
        blocks = 0;
    };
    for (int64_t i = 0; i < g.n_tensors; ++i) {
        const adhip_adamw_tensor& t = g.tensors[i];
        if (t.count == 0) continue;
        const uint64_t own = (uint64_t)((t.count + kChunk - 1) / kChunk);
        if (a.n == kTensors || blocks + own > kBlocks) flush();
        a.t[a.n] = t;
        a.first[a.n] = (unsigned)blocks;
        bool whole = aligned_to(t.p, 4 * pw) && aligned_to(t.p_out, 4 * pw) && aligned_to(t.g, 4 * gw);
        if (!eight)
            for (const void* s : {t.m, t.v, (const void*)t.m_out, (const void*)t.v_out}) whole = whole && aligned_to(s, 16);
        if (whole) a.aligned |= 1u << a.n;
        ++a.n;
        blocks += own;
        a.first[a.n] = (unsigned)blocks;
    }
    flush();
}

}  // namespace
}  // namespace adhip

extern "C" int adhip_adamw(adhip_ctx* ctx, const adhip_adamw_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_adamw: no arguments");
        adhip::adamw(*args, (hipStream_t)stream);
    });
}

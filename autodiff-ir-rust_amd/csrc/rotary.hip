// Rotary positions (Su et al. 2021): the features of a head in pairs, each pair turned by the angle that the position and
// the pair give.  Cosines and sines come from tables, so a scaled table serves longer contexts and the angles have the
// precision that the table was made with.
//
// One read and one write of the heads' features bounds it; the arithmetic is nothing.  A lane owns V pairs of a token and
// turns them in up to U heads: their cosines and sines are loaded once, and 2 U loads are under way before the first is
// used.  V is as large as 16 bytes, the number of pairs and the arrays' alignment allow.
#include "operators.hpp"

namespace adhip {
namespace {

struct RotaryArray {
    const void* x;
    void* out;
    int64_t xb, xl, xh, ob, ol, oh;  // strides of batch, length and heads
    int heads, groups;               // groups of U heads
};

struct RotaryParams {
    RotaryArray a[2];
    const float *cos, *sin;
    const int* positions;
    int64_t pb, pl;   // strides of positions
    int64_t rows;     // of the tables
    unsigned tokens, length;
    int size, pairs;
    unsigned chunks, turned;  // chunks of V pairs or V copied features of a head; the first `turned` are pairs
    unsigned items;           // lanes that a token takes: chunks * groups of both arrays
    unsigned per_block;       // tokens of a block (1 where a token takes several)
    float sign;
};

template <class T, int V, int U, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
    unsigned item = blockIdx.y * 256 + threadIdx.x, token = blockIdx.x;
    if (p.per_block > 1) {
        const unsigned t = item / p.items;
        if (t >= p.per_block) return;
        item -= t * p.items;
        token = token * p.per_block + t;
    }
    if (item >= p.items || token >= p.tokens) return;
    const unsigned group = item / p.chunks, chunk = item - group * p.chunks;
    const bool second = group >= (unsigned)p.a[0].groups;
    const RotaryArray& a = second ? p.a[1] : p.a[0];
    const int h0 = (int)(second ? group - p.a[0].groups : group) * U;
    const unsigned b = token / p.length, l = token - b * p.length;
    const T* x = (const T*)a.x + b * a.xb + l * a.xl + h0 * a.xh;
    T* o = (T*)a.out + b * a.ob + l * a.ol + h0 * a.oh;
    const int n = min(U, a.heads - h0);
    typedef Pack<T, V> P;
    if (chunk >= p.turned) {
        const int at = 2 * p.pairs + (int)(chunk - p.turned) * V;
        P r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u < n) r[u] = *(const P*)(x + u * a.xh + at);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u < n) *(P*)(o + u * a.oh + at) = r[u];
        return;
    }
    const int pair = (int)chunk * V;
    const int i0 = INTERLEAVED ? 2 * pair : pair, i1 = INTERLEAVED ? 2 * pair + V : pair + p.pairs;
    P r0[U], r1[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n) {
            r0[u] = *(const P*)(x + u * a.xh + i0);
            r1[u] = *(const P*)(x + u * a.xh + i1);
        }
    const int64_t row = p.positions[b * p.pb + l * p.pl];
    constexpr int W = V < 4 ? V : 4;
    float c[V], s[V];
    if (row >= 0 && row < p.rows) {
#pragma unroll
        for (int i = 0; i < V; i += W) {
            *(Pack<float, W>*)&c[i] = *(const Pack<float, W>*)(p.cos + row * p.pairs + pair + i);
            *(Pack<float, W>*)&s[i] = *(const Pack<float, W>*)(p.sin + row * p.pairs + pair + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = s[i] = __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] *= p.sign;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u >= n) break;
        if (INTERLEAVED) {
            T f[2 * V];
            *(P*)f = r0[u];
            *(P*)(f + V) = r1[u];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float x0 = (float)f[2 * i], x1 = (float)f[2 * i + 1];
                f[2 * i] = (T)(x0 * c[i] - x1 * s[i]);
                f[2 * i + 1] = (T)(x0 * s[i] + x1 * c[i]);
            }
            r0[u] = *(P*)f;
            r1[u] = *(P*)(f + V);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float x0 = (float)r0[u].v[i], x1 = (float)r1[u].v[i];
                r0[u].v[i] = (T)(x0 * c[i] - x1 * s[i]);
                r1[u].v[i] = (T)(x0 * s[i] + x1 * c[i]);
            }
        }
        *(P*)(o + u * a.oh + i0) = r0[u];
        *(P*)(o + u * a.oh + i1) = r1[u];
    }
}

template <class T, int V, int U>
void launch_rotary(const RotaryParams& p, bool interleaved, dim3 grid, hipStream_t stream) {
    if (interleaved) rotary_kernel<T, V, U, true><<<grid, 256, 0, stream>>>(p);
    else rotary_kernel<T, V, U, false><<<grid, 256, 0, stream>>>(p);
}

template <class T, int V>
void launch_rotary(const RotaryParams& p, int u, bool interleaved, dim3 grid, hipStream_t stream) {
    if (u == 4) launch_rotary<T, V, 4>(p, interleaved, grid, stream);
    else launch_rotary<T, V, 1>(p, interleaved, grid, stream);
}

void rotary(const adhip_rotary_args& g, hipStream_t stream) {
    const char* op = "adhip_rotary";
    const int type = g.x.type;
    ADHIP_CHECK(type == ADHIP_F32 || type == ADHIP_BF16, "%s: x is %s, f32 or bf16 is wanted", op, type_name(type));
    check_array(op, "x", g.x, type, 4);
    check_array(op, "out", g.out, type, 4);
    check_array(op, "cos", g.cos, ADHIP_F32, 2);
    check_array(op, "sin", g.sin, ADHIP_F32, 2);
    check_array(op, "positions", g.positions, ADHIP_I32, 2);
    const int64_t batch = g.x.dims[0], length = g.x.dims[1], size = g.x.dims[3], pairs = g.cos.dims[1];
    const bool two = g.second.data != nullptr || g.second_out.data != nullptr;
    check_dims(op, "out", g.out, {batch, length, g.x.dims[2], size});
    check_dims(op, "sin", g.sin, {g.cos.dims[0], pairs});
    check_dims(op, "positions", g.positions, {batch, length});
    ADHIP_CHECK(pairs >= 1 && 2 * pairs <= size, "%s: %lld pairs do not fit heads of %lld features", op, (long long)pairs, (long long)size);
    for (const adhip_array* t : {&g.cos, &g.sin}) {
        check_packed_rows(op, "the table", *t);
        ADHIP_CHECK(t->strides[0] == pairs || t->dims[0] <= 1, "%s: the rows of the tables must be packed", op);
    }
    check_packed_rows(op, "x", g.x);
    check_packed_rows(op, "out", g.out);
    check_distinct(op, "out", g.out);
    if (two) {
        check_array(op, "second", g.second, type, 4);
        check_array(op, "second_out", g.second_out, type, 4);
        check_dims(op, "second", g.second, {batch, length, g.second.dims[2], size});
        check_dims(op, "second_out", g.second_out, {batch, length, g.second.dims[2], size});
        check_packed_rows(op, "second", g.second);
        check_packed_rows(op, "second_out", g.second_out);
        check_distinct(op, "second_out", g.second_out);
    }
    // extents that 32 bits hold, offsets that take 64
    const int64_t tokens = batch * length, heads = g.x.dims[2] + (two ? g.second.dims[2] : 0);
    ADHIP_CHECK(tokens < (int64_t(1) << 31) && size <= (1 << 20) && heads * size < (int64_t(1) << 31),
                "%s: %lld tokens of %lld x %lld features are too many for one call", op, (long long)tokens, (long long)heads, (long long)size);
    if (tokens == 0 || heads == 0) return;

    // elements that a lane takes at once: 16 bytes, fewer where pairs, tail or alignment are not multiples of it
    int v = 16 / type_bytes(type);
    for (const adhip_array* t : {&g.x, &g.out, two ? &g.second : &g.x, two ? &g.second_out : &g.out}) v = vector_elements(*t, v);
    while (v > 1 && (pairs % v || (size - 2 * pairs) % v)) v /= 2;
    const int w = v < 4 ? v : 4;
    if ((uintptr_t)g.cos.data % (size_t)(4 * w) || (uintptr_t)g.sin.data % (size_t)(4 * w)) v = 1;
    RotaryParams p = {};
    const adhip_array* in[2] = {&g.x, &g.second};
    const adhip_array* to[2] = {&g.out, &g.second_out};
    p.turned = (unsigned)(pairs / v);
    p.chunks = p.turned + (unsigned)((size - 2 * pairs) / v);
    // Four heads a lane once that still leaves every compute unit eight wavefronts of lanes; below, one head a lane is
    // the shorter way (a token of 8 + 8 heads: one wavefront's trip to memory instead of four in a row).
    const int u = tokens * heads * p.chunks >= int64_t(4) * 256 * 8 * 64 ? 4 : 1;
    for (int i = 0; i < (two ? 2 : 1); ++i) {
        RotaryArray& a = p.a[i];
        a.x = in[i]->data;
        a.out = to[i]->data;
        a.xb = in[i]->strides[0], a.xl = in[i]->strides[1], a.xh = in[i]->strides[2];
        a.ob = to[i]->strides[0], a.ol = to[i]->strides[1], a.oh = to[i]->strides[2];
        a.heads = (int)in[i]->dims[2];
        a.groups = (a.heads + u - 1) / u;
    }
    p.cos = (const float*)g.cos.data;
    p.sin = (const float*)g.sin.data;
    p.positions = (const int*)g.positions.data;
    p.pb = g.positions.strides[0], p.pl = g.positions.strides[1];
    p.rows = g.cos.dims[0];
    p.tokens = (unsigned)tokens;
    p.length = (unsigned)length;
    p.size = (int)size;
    p.pairs = (int)pairs;
    p.items = p.chunks * (unsigned)(p.a[0].groups + p.a[1].groups);
    p.per_block = p.items < 256 ? 256 / p.items : 1;
    p.sign = g.inverse ? -1.f : 1.f;
    const dim3 grid((unsigned)((tokens + p.per_block - 1) / p.per_block), (p.items + 255) / 256);
    ADHIP_CHECK(grid.y < 65536, "%s: heads of %lld x %lld features are too many for one call", op, (long long)heads, (long long)size);
    const bool il = g.interleaved != 0;
    if (type == ADHIP_BF16) {
        if (v == 8) launch_rotary<bf16, 8>(p, u, il, grid, stream);
        else if (v == 4) launch_rotary<bf16, 4>(p, u, il, grid, stream);
        else if (v == 2) launch_rotary<bf16, 2>(p, u, il, grid, stream);
        else launch_rotary<bf16, 1>(p, u, il, grid, stream);
    } else {
        if (v == 4) launch_rotary<float, 4>(p, u, il, grid, stream);
        else if (v == 2) launch_rotary<float, 2>(p, u, il, grid, stream);
        else launch_rotary<float, 1>(p, u, il, grid, stream);
    }
    check_launch(op);
}

}  // namespace
}  // namespace adhip

extern "C" int adhip_rotary(adhip_ctx* ctx, const adhip_rotary_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_rotary: no arguments");
        adhip::rotary(*args, (hipStream_t)stream);
    });
}

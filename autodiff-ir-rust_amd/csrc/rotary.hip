// Rotary positions (Su et al. 2021): the features of a head in pairs, each pair turned by the angle that the position and
// the pair give.  Cosines and sines come from tables, so a scaled table serves longer contexts and the angles have the
// precision that the table was made with.
//
// One read and one write of the heads' features bounds it; the arithmetic is nothing.  A lane turns V pairs of one head (or
// copies V features); V is as large as 16 bytes, the number of pairs and the arrays' alignment allow.  Four heads a lane,
// with the cosines and sines loaded once for all, were no faster on long sequences (16384 tokens of 32 + 8 heads of 128 in
// bf16: 60 us, 5.7 TB/s, either way) and slower on short ones, where lanes in number hide the way to memory: 3003 tokens of
// 8 + 8 heads of 80, half of them turned, in f32, 20 us with four heads and 8 with one.
#include "operators.hpp"

#include <algorithm>

namespace adhip {
namespace {

struct RotaryArray {
    const void* x;
    void* out;
    int64_t xb, xl, xh, ob, ol, oh;  // strides of batch, length and heads
    int heads;
};

struct RotaryParams {
    RotaryArray a[2];
    const float *cos, *sin;
    const int* positions;
    int64_t pb, pl;   // strides of positions
    int64_t rows;     // of the tables
    unsigned tokens, length;
    int pairs;
    unsigned turned, copied;  // chunks of V pairs and of V copied features of a head
    unsigned turns, items;    // lanes that a token takes: `turns` for its pairs, the others for copies
    unsigned per_block;       // tokens of a block (1 where a token takes several)
    float sign;
};

template <class T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
    unsigned item = blockIdx.y * 256 + threadIdx.x, token = blockIdx.z * gridDim.x + blockIdx.x;
    if (p.per_block > 1) {
        const unsigned t = item / p.items;
        if (t >= p.per_block) return;
        item -= t * p.items;
        token = token * p.per_block + t;
    }
    if (item >= p.items || token >= p.tokens) return;
    // (pairs first, of all heads: a wavefront has one of the two to do)
    const bool copies = item >= p.turns;
    const unsigned of = copies ? p.copied : p.turned, at_item = copies ? item - p.turns : item;
    const unsigned number = at_item / of, chunk = at_item - number * of;
    const bool second = number >= (unsigned)p.a[0].heads;
    // field by field: an index by lane would send every lane to the kernel's arguments in memory
    const RotaryArray &one = p.a[0], &two = p.a[1];
    const RotaryArray a = {second ? two.x : one.x,   second ? two.out : one.out, second ? two.xb : one.xb, second ? two.xl : one.xl,
                           second ? two.xh : one.xh, second ? two.ob : one.ob,   second ? two.ol : one.ol, second ? two.oh : one.oh,
                           0};
    const int64_t h = second ? number - one.heads : number;
    const unsigned b = token / p.length, l = token - b * p.length;
    const T* x = (const T*)a.x + b * a.xb + l * a.xl + h * a.xh;
    T* o = (T*)a.out + b * a.ob + l * a.ol + h * a.oh;
    typedef Pack<T, V> P;
    if (copies) {
        const int at = 2 * p.pairs + (int)chunk * V;
        *(P*)(o + at) = *(const P*)(x + at);
        return;
    }
    const int pair = (int)chunk * V;
    const int i0 = INTERLEAVED ? 2 * pair : pair, i1 = INTERLEAVED ? 2 * pair + V : pair + p.pairs;
    P r0 = *(const P*)(x + i0), r1 = *(const P*)(x + i1);
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
    if (INTERLEAVED) {
        T f[2 * V];
        *(P*)f = r0;
        *(P*)(f + V) = r1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float x0 = (float)f[2 * i], x1 = (float)f[2 * i + 1];
            f[2 * i] = (T)(x0 * c[i] - x1 * s[i]);
            f[2 * i + 1] = (T)(x0 * s[i] + x1 * c[i]);
        }
        r0 = *(P*)f;
        r1 = *(P*)(f + V);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float x0 = (float)r0.v[i], x1 = (float)r1.v[i];
            r0.v[i] = (T)(x0 * c[i] - x1 * s[i]);
            r1.v[i] = (T)(x0 * s[i] + x1 * c[i]);
        }
    }
    *(P*)(o + i0) = r0;
    *(P*)(o + i1) = r1;
}

template <class T, int V>
void launch_rotary(const char* op, const RotaryParams& p, bool interleaved, dim3 grid, hipStream_t stream) {
    launch(op, interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>, grid, 256, stream, p);
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
    p.copied = (unsigned)((size - 2 * pairs) / v);
    for (int i = 0; i < (two ? 2 : 1); ++i) {
        RotaryArray& a = p.a[i];
        a.x = in[i]->data;
        a.out = to[i]->data;
        a.xb = in[i]->strides[0], a.xl = in[i]->strides[1], a.xh = in[i]->strides[2];
        a.ob = to[i]->strides[0], a.ol = to[i]->strides[1], a.oh = to[i]->strides[2];
        a.heads = (int)in[i]->dims[2];
    }
    p.cos = (const float*)g.cos.data;
    p.sin = (const float*)g.sin.data;
    p.positions = (const int*)g.positions.data;
    p.pb = g.positions.strides[0], p.pl = g.positions.strides[1];
    p.rows = g.cos.dims[0];
    p.tokens = (unsigned)tokens;
    p.length = (unsigned)length;
    p.pairs = (int)pairs;
    p.turns = p.turned * (unsigned)(p.a[0].heads + p.a[1].heads);
    p.items = p.turns + p.copied * (unsigned)(p.a[0].heads + p.a[1].heads);
    p.per_block = p.items < 256 ? 256 / p.items : 1;
    p.sign = g.inverse ? -1.f : 1.f;
    // 2^23 blocks in a row of the grid, so that it holds fewer than 2^32 threads
    const int64_t across = (tokens + p.per_block - 1) / p.per_block;
    const dim3 grid((unsigned)std::min<int64_t>(across, 1 << 23), (p.items + 255) / 256, (unsigned)((across + (1 << 23) - 1) >> 23));
    ADHIP_CHECK(grid.y < 65536, "%s: heads of %lld x %lld features are too many for one call", op, (long long)heads, (long long)size);
    const bool il = g.interleaved != 0;
    if (type == ADHIP_BF16) {
        if (v == 8) launch_rotary<bf16, 8>(op, p, il, grid, stream);
        else if (v == 4) launch_rotary<bf16, 4>(op, p, il, grid, stream);
        else if (v == 2) launch_rotary<bf16, 2>(op, p, il, grid, stream);
        else launch_rotary<bf16, 1>(op, p, il, grid, stream);
    } else {
        if (v == 4) launch_rotary<float, 4>(op, p, il, grid, stream);
        else if (v == 2) launch_rotary<float, 2>(op, p, il, grid, stream);
        else launch_rotary<float, 1>(op, p, il, grid, stream);
    }
}

}  // namespace
}  // namespace adhip

extern "C" int adhip_rotary(adhip_ctx* ctx, const adhip_rotary_args* args, void* stream) {
    return adhip::context_guarded(ctx, [&] {
        ADHIP_CHECK(args, "adhip_rotary: no arguments");
        adhip::rotary(*args, (hipStream_t)stream);
    });
}

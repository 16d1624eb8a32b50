// Attention on device arrays: checks of arguments, workspace, the choice of kernels.
#include "operator_attention.hpp"

#include <algorithm>
#include <cmath>

namespace adhip {
namespace {

using attn::Params;

// Smallest and largest document of every kRange positions, so that a tile whose documents cannot meet is passed over
// without a look at its positions: a wavefront for two entries.  (8191 positions: 5 us, most of it the launch.)
__global__ __launch_bounds__(256) void document_ranges_kernel(const int* q, int64_t qb, int64_t ql, int Lq, int2* qr, int qn, const int* k,
                                                              int64_t kb, int64_t kl, int Lk, int2* kr, int kn) {
    const int blocks = (qn + kn + 7) / 8, lane = threadIdx.x & 31;
    const int64_t b = blockIdx.x / blocks;
    const int entry = (int)(blockIdx.x - b * blocks) * 8 + (threadIdx.x >> 5);
    const bool of_keys = entry >= qn;
    const int e = of_keys ? entry - qn : entry;
    if (of_keys && e >= kn) return;
    const int i = e * attn::kRange + lane;
    const bool there = i < (of_keys ? Lk : Lq);
    const int d = !there ? -1 : max(of_keys ? k[b * kb + i * kl] : q[b * qb + i * ql], -1);
    int lo = d >= 0 ? d : 0x7fffffff, hi = d, none = there && d < 0;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        lo = min(lo, __shfl_xor(lo, s));
        hi = max(hi, __shfl_xor(hi, s));
        none |= __shfl_xor(none, s);
    }
    if (lane == 0) (of_keys ? kr + (int64_t)b * kn : qr + (int64_t)b * qn)[e] = int2{none ? ~lo : lo, hi};
}

// Arrays [B, L, H, D] of f32 as three bf16 parts: planes [B, L, H, D3], the features behind D zeros.  A thread a piece of 8:
// memory bounds it (k and v, 2048 x 8 heads of 128: 8 us, q, k, v and dout 14).
struct PartsJob {
    attn::Tensor in;
    bf16* out;
    int64_t rows;  // B L H
    int L, H;
};
struct PartsJobs {
    PartsJob job[4];
};
__global__ __launch_bounds__(256) void parts_kernel(const PartsJobs jobs, int D, int D3) {
    const PartsJob j = jobs.job[blockIdx.y];
    const int pieces = D3 / 8;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / pieces, plane = j.rows * D3;
    if (row >= j.rows) return;
    const int d = (int)(at - row * pieces) * 8, h = (int)(row % j.H);
    const int64_t bl = row / j.H, b = bl / j.L;
    const float* x = (const float*)j.in.data + b * j.in.b + (bl - b * j.L) * j.in.l + h * j.in.h;
    attn::f32x8 f;
    if (j.in.vec && d + 8 <= D) {
        ((float4*)&f)[0] = *(const float4*)(x + d);
        ((float4*)&f)[1] = *(const float4*)(x + d + 4);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = d + e < D ? x[d + e] : 0.f;
    }
    const attn::Frag3 p = attn::MatrixInParts::operand(f);
#pragma unroll
    for (int i = 0; i < 3; ++i) *(attn::bf16x8*)(j.out + i * plane + row * D3 + d) = p.p[i];
}

attn::Tensor tensor_of(const adhip_array& a) {
    const int chunk = 16 / type_bytes(a.type);
    attn::Tensor t = {a.data, a.strides[0], a.strides[1], a.strides[2], 0};
    // (a tile's offsets, up to 128 rows, are to fit 31 bits)
    t.vec = vector_elements(a, chunk) == chunk && a.dims[3] % chunk == 0 && (a.dims[1] <= 1 || a.strides[1] < (int64_t(1) << 31) / 4 / 128 - 256);
    return t;
}

size_t rounded(size_t n) { return (n + 255) & ~size_t(255); }

// How a call is cut up, and where its workspace's parts begin.
struct Layout {
    bool few_rows;
    int row_tile, tiles, splits, dq_splits, dk_splits;
    size_t qrange, krange, part, part_ml, stats, part_dq, part_dk, part_dv, q3, k3, v3, dout3, bytes;
    bool parts;
};

constexpr int kUnits = 256;  // compute units

// A kind of walk: workgroups of `own` rows (or keys), each of which goes over keys (or rows) in tiles of `step`.
struct Walks {
    int64_t blocks;     // workgroups with one range each
    int own, step;
    int room;           // workgroups that registers and LDS of a compute unit hold
    double across;      // keys (rows) in all, and what it counts for each key: 1, or G where rows are walked
    int times;
    double part_bytes;  // what a range more takes of memory
};

// How many ranges (at most `most`) such walks are split into where rows fill workgroups: the smallest sum of two times, in us.
//   walk  a workgroup's tiles, and one more for its beginning and end, at `pair` ps for a row and a key, as measured for the
//         forward kernels with one workgroup a compute unit (bf16 64 features 140, 128 180, 192 350, 256 380; f32 464, 464 with
//         eight wavefronts, -, 1760).  Workgroups that share a compute unit finish 1.4 (two) and 1.8 (three) times as much.
//         Where all walks are equally long, the compute unit with the most workgroups decides; where a causal mask makes them
//         uneven, given out from the longest, it is the longest walk or the average load, whichever is more, and a little of
//         the other.  Documents, which end walks where they fall, are not looked at: the more ranges of the mask alone even them out too
//         (8191 positions, 8 heads of 64, eight draws of documents of 1200 on average, forward and backward: 192 to 350 us;
//         with the ranges of short walks, mostly one, 197 to 422).
//   join  0.36 us a MB of parts, written and read again, and 6 us for the launch and the parts' ends
// Over 32 shapes (300 to 8192 positions, bf16 64 to 256 features, f32 64 to 256) the choice is within 1 % of the best number in
// the mean, for the backward walks within 2 % over 34; as many ranges as fill the card alone were 17 and 9 % off (8 x 300
// positions of 16 heads of 128 forward: 18 us, 37 with the two ranges that the card had room for).
int ranges(const adhip_attention_args& g, const Walks& w, bool causal, int64_t window, int most) {
    const int64_t Lq = g.q.dims[1], D = g.q.dims[3], Lk = g.k.dims[1];
    const int DP = attn::padded_size((int)D);
    const double pair = g.q.type != ADHIP_F32 ? 70 + 1.15 * DP : DP > 128 ? 7. * DP : (100 + 5. * DP) / (w.own == 256 ? 1.5 : 1.);
    const double tile = pair * w.own * w.step * 1e-6;
    // what the longest walk and the mean one go over
    double longest = w.across, mean = causal ? std::max(1. - Lq / (2. * std::max<double>((double)Lk, 1)), 0.5) * w.across : w.across;
    if (window > 0) {
        longest = std::min(longest, ((causal ? 1. : 2.) * (double)window + (double)w.own * w.times / (double)(g.q.dims[2] / g.k.dims[2])) * w.times);
        mean = std::min(mean, longest);
    }
    const bool even = mean > 0.75 * longest;
    double best = 0;
    int choice = 1;
    for (int s = 1; s <= most && (s == 1 || ((double)s * w.step * 2 <= w.across + w.step && s * w.blocks <= 4 * kUnits)); s += 1 + s / 8) {
        const double walk = (std::ceil(longest / w.step / s) + 1) * tile, workgroups = (double)(w.blocks * s);
        const double each = std::ceil(workgroups / kUnits), faster = 1 + 0.4 * (std::min<double>(each, w.room) - 1);
        double time = each * walk / faster;
        if (!even) {
            const double load = workgroups / kUnits * (mean / w.step / s + 1) * tile / faster;
            time = std::max(walk, load) + 0.05 * std::min(walk, load);
        }
        if (s > 1) time += 6 + 0.36e-6 * s * w.part_bytes;
        if (s == 1 || time < best) best = time, choice = s;
    }
    return choice;
}
// for a call, and the most that a call on arrays of these shapes takes, whatever its masks
struct Ranges {
    int now = 1, most = 1;
    Ranges() {}
    Ranges(const adhip_attention_args& g, const Walks& w) {
        if (w.blocks <= 0) return;
        most = std::max(ranges(g, w, false, 0, 256), ranges(g, w, true, 0, 256));
        now = ranges(g, w, g.causal != 0, g.window, most);
    }
};

Layout layout_of(const adhip_attention_args& g, bool backward) {
    Layout y = {};
    const int64_t B = g.q.dims[0], Lq = g.q.dims[1], H = g.q.dims[2], D = g.q.dims[3], Lk = g.k.dims[1], Hk = g.k.dims[2];
    const int64_t R = Hk > 0 ? Lq * (H / Hk) : 0;
    // One wavefront's 32 columns hold all rows of a key head: the wavefronts of a workgroup go along the keys.
    y.few_rows = R <= 32;
    y.row_tile = attn::forward_rows(g.q.type, attn::padded_size((int)D), y.few_rows);
    y.tiles = (int)((R + y.row_tile - 1) / y.row_tile);
    // Ranges of keys, none shorter than two tiles.  Few rows: one workgroup a compute unit, as it fills LDS then and keeps 64 KB
    // under way (8 sequences of 16384 keys: 105 us with one, 113 with four).
    const int64_t blocks = (int64_t)y.tiles * Hk * B;
    const bool f32 = g.q.type == ADHIP_F32;
    const int DP = attn::padded_size((int)D), step = f32 || DP > 128 ? 32 : 64;
    const double row_bytes = 4. * (double)B * (double)Lq * (double)H * (double)D, key_bytes = 4. * (double)B * (double)Lk * (double)Hk * (double)D;
    Ranges forward_ranges;
    if (!y.few_rows) forward_ranges = Ranges(g, {blocks, y.row_tile, step, f32 ? (DP <= 64 ? 2 : 1) : DP <= 64 ? 3 : DP <= 192 ? 2 : 1, (double)Lk, 1, row_bytes});
    else if (blocks > 0 && blocks < kUnits)
        forward_ranges.most = forward_ranges.now = (int)std::max<int64_t>(1, std::min({(kUnits + blocks - 1) / blocks, (Lk + 255) / 256, (int64_t)256}));
    y.splits = forward_ranges.now;
    size_t at = 0;
    // (whether documents are given or not: what a call needs goes by shapes alone)
    y.qrange = at;
    at += rounded((size_t)(B * ((Lq + attn::kRange - 1) / attn::kRange)) * sizeof(int2));
    y.krange = at;
    at += rounded((size_t)(B * ((Lk + attn::kRange - 1) / attn::kRange)) * sizeof(int2));
    y.parts = attn::in_parts(g.q.type, (int)D, backward ? false : y.few_rows);
    if (y.parts) {
        const size_t keys = rounded((size_t)(B * Lk * Hk * attn::parts_size((int)D)) * 6), rows = rounded((size_t)(B * Lq * H * attn::parts_size((int)D)) * 6);
        y.k3 = at;
        y.v3 = at + keys;
        at += 2 * keys;
        if (backward) {
            y.q3 = at;
            y.dout3 = at + rows;
            at += 2 * rows;
        }
    }
    size_t forward = at, back = at;
    // (what a call needs goes by shapes alone, how it is cut up by its masks too)
    const int64_t most = forward_ranges.most;
    if (most > 1) {
        y.part = forward;
        forward += rounded((size_t)(most * B * Hk * R * D) * 4);
        y.part_ml = forward;
        forward += rounded((size_t)(most * B * Hk * R * 2) * 4);
    }
    y.dq_splits = y.dk_splits = 1;
    if (backward) {
        y.stats = back;
        back += rounded((size_t)(B * Hk * R) * 2 * 4);
        // the walks of 128 rows over keys and of 128 keys over the rows of all their heads
        const Ranges of_rows(g, {(R + 127) / 128 * Hk * B, 128, step, DP <= (f32 ? 64 : 128) ? 2 : 1, (double)Lk, 1, row_bytes});
        const Ranges of_keys(g, {(Lk + 127) / 128 * Hk * B, 128, step, 1, (double)R, (int)(H / Hk), 2 * key_bytes});
        y.dq_splits = of_rows.now;
        y.dk_splits = of_keys.now;
        if (of_rows.most > 1) {
            y.part_dq = back;
            back += rounded((size_t)(of_rows.most * B * Hk * R * D) * 4);
        }
        if (of_keys.most > 1) {
            y.part_dk = back;
            back += rounded((size_t)(of_keys.most * B * Hk * Lk * D) * 4);
            y.part_dv = back;
            back += rounded((size_t)(of_keys.most * B * Hk * Lk * D) * 4);
        }
    }
    y.bytes = std::max(forward, back);
    return y;
}

// Shapes and types of q, k and v: what the workspace goes by
void check_sizes(const char* op, const adhip_attention_args& g) {
    ADHIP_CHECK(g.q.type == ADHIP_F32 || g.q.type == ADHIP_BF16, "%s: q is %s, f32 or bf16 is wanted", op, type_name(g.q.type));
    check_shape(op, "q", g.q, g.q.type, 4);
    check_shape(op, "k", g.k, g.q.type, 4);
    check_shape(op, "v", g.v, g.q.type, 4);
    const int64_t B = g.q.dims[0], Lq = g.q.dims[1], H = g.q.dims[2], D = g.q.dims[3], Lk = g.k.dims[1], Hk = g.k.dims[2];
    check_dims(op, "k", g.k, {B, Lk, Hk, D});
    check_dims(op, "v", g.v, {B, Lk, Hk, D});
    ADHIP_CHECK(D >= 1 && D <= 256, "%s: heads of %lld features, 1 to 256 are supported", op, (long long)D);
    ADHIP_CHECK(Hk >= 1 && H >= 1 && H % Hk == 0, "%s: %lld heads cannot share %lld key heads", op, (long long)H, (long long)Hk);
    // positions and rows in 32 bits, with room for a window on either side
    constexpr int64_t kMost = int64_t(1) << 28;
    ADHIP_CHECK(Lq <= kMost && Lk <= kMost && B <= kMost && H <= kMost && Lq * (H / Hk) <= kMost && B * H <= kMost, "%s: q %s and k %s are too large", op, array_str(g.q).c_str(),
                array_str(g.k).c_str());
    ADHIP_CHECK(B * Hk * ((Lq * (H / Hk) + 31) / 32 + (Lk + 31) / 32) <= kMost, "%s: q %s and k %s are too large", op, array_str(g.q).c_str(),
                array_str(g.k).c_str());
}

// Every kernel of a call fits a launch.
void check_launches(const char* op, const adhip_attention_args& g, const Layout& y, bool backward) {
    const int64_t B = g.q.dims[0], Lq = g.q.dims[1], H = g.q.dims[2], D = g.q.dims[3], Lk = g.k.dims[1], Hk = g.k.dims[2], R = Lq * (H / Hk);
    bool fit;
    if (!backward) fit = fits_launch(y.tiles * Hk * B * y.splits, y.row_tile == 256 ? 512 : 256);
    else fit = fits_launch((R + 127) / 128 * Hk * B * y.dq_splits, 256) && fits_launch((Lk + 127) / 128 * Hk * B * y.dk_splits, 512);
    if (y.parts) fit = fit && fits_launch(((backward ? std::max(Lq * H, Lk * Hk) : Lk * Hk) * B * (attn::parts_size((int)D) / 8) + 255) / 256, 256);
    fit = fit && fits_launch(((Lq + 31) / 32 + (Lk + 31) / 32 + 7) / 8 * B, 256);  // documents
    // (a tile of planes has 32 rows, whose offsets are to fit 31 bits, as those of the arrays' own tiles do)
    if (y.parts) fit = fit && (backward ? H : Hk) * attn::parts_size((int)D) <= (int64_t(1) << 25);
    ADHIP_CHECK(fit, "%s: q %s and k %s are too large for one call", op, array_str(g.q).c_str(), array_str(g.k).c_str());
}

Params checked(const char* op, const adhip_attention_args& g, const Layout& y, bool backward) {
    const int64_t B = g.q.dims[0], Lq = g.q.dims[1], H = g.q.dims[2], D = g.q.dims[3], Lk = g.k.dims[1], Hk = g.k.dims[2];
    auto tensor = [&](const char* name, const adhip_array& a, std::initializer_list<int64_t> dims, bool output) {
        check_array(op, name, a, g.q.type, 4);
        check_dims(op, name, a, dims);
        check_packed_rows(op, name, a);
        if (output) check_distinct(op, name, a);
        return tensor_of(a);
    };
    Params p = {};
    p.q = tensor("q", g.q, {B, Lq, H, D}, false);
    p.k = tensor("k", g.k, {B, Lk, Hk, D}, false);
    p.v = tensor("v", g.v, {B, Lk, Hk, D}, false);
    p.out = tensor("out", g.out, {B, Lq, H, D}, !backward);
    check_array(op, "lse", g.lse, ADHIP_F32, 3);
    check_dims(op, "lse", g.lse, {B, Lq, H});
    if (!backward) check_distinct(op, "lse", g.lse);
    p.lse = (float*)g.lse.data;
    p.lse_b = g.lse.strides[0], p.lse_l = g.lse.strides[1], p.lse_h = g.lse.strides[2];
    if (backward) {
        p.dout = tensor("out_grad", g.out_grad, {B, Lq, H, D}, false);
        p.dq = tensor("q_grad", g.q_grad, {B, Lq, H, D}, true);
        p.dk = tensor("k_grad", g.k_grad, {B, Lk, Hk, D}, true);
        p.dv = tensor("v_grad", g.v_grad, {B, Lk, Hk, D}, true);
    }
    if (g.slopes.data) {
        check_array(op, "slopes", g.slopes, ADHIP_F32, 1);
        check_dims(op, "slopes", g.slopes, {H});
        p.slopes = (const float*)g.slopes.data;
        p.slope_stride = g.slopes.strides[0];
    }
    if (g.lengths.data) {
        check_array(op, "lengths", g.lengths, ADHIP_I32, 1);
        check_dims(op, "lengths", g.lengths, {B});
        p.lengths = (const int*)g.lengths.data;
        p.lengths_s = g.lengths.strides[0];
    }
    if (g.prefix.data) {
        check_array(op, "prefix", g.prefix, ADHIP_I32, 1);
        check_dims(op, "prefix", g.prefix, {B});
        p.prefix = (const int*)g.prefix.data;
        p.prefix_s = g.prefix.strides[0];
    }
    const bool documents = g.query_documents.data || g.key_documents.data;
    if (documents) {
        check_array(op, "query_documents", g.query_documents, ADHIP_I32, 2);
        check_array(op, "key_documents", g.key_documents, ADHIP_I32, 2);
        check_dims(op, "query_documents", g.query_documents, {B, Lq});
        check_dims(op, "key_documents", g.key_documents, {B, Lk});
        for (const adhip_array* a : {&g.query_documents, &g.key_documents})  // a tile's offsets are to fit 31 bits
            ADHIP_CHECK(a->dims[1] <= 1 || a->strides[1] <= (1 << 20), "%s: documents lie %lld elements apart, at most %d are supported", op,
                        (long long)a->strides[1], 1 << 20);
        p.qdoc = (const int*)g.query_documents.data;
        p.kdoc = (const int*)g.key_documents.data;
        p.qdoc_b = g.query_documents.strides[0], p.qdoc_l = g.query_documents.strides[1];
        p.kdoc_b = g.key_documents.strides[0], p.kdoc_l = g.key_documents.strides[1];
    }
    ADHIP_CHECK(std::isfinite(g.scale), "%s: the scale is not finite", op);
    ADHIP_CHECK(std::isfinite(g.cap) && g.cap >= 0.f, "%s: the cap must be 0 (none) or positive, and finite", op);
    ADHIP_CHECK(g.window >= 0, "%s: the window must be 0 (none) or positive", op);
    ADHIP_CHECK(g.workspace_bytes >= y.bytes && (g.workspace || y.bytes == 0), "%s: a workspace of %zu bytes is given, %zu are needed", op,
                g.workspace ? (size_t)g.workspace_bytes : (size_t)0, y.bytes);
    ADHIP_CHECK((uintptr_t)g.workspace % 256 == 0, "%s: the workspace is not aligned to 256 bytes", op);
    char* const room = (char*)g.workspace;
    if (documents) {
        p.qrange = (const int2*)(room + y.qrange);
        p.krange = (const int2*)(room + y.krange);
        p.qranges = (int)((Lq + attn::kRange - 1) / attn::kRange);
        p.kranges = (int)((Lk + attn::kRange - 1) / attn::kRange);
    }
    p.B = (int)B, p.Lq = (int)Lq, p.Lk = (int)Lk, p.Hk = (int)Hk, p.G = (int)(H / Hk), p.D = (int)D, p.R = (int)(Lq * (H / Hk));
    p.scale = g.scale;
    p.cap = g.cap;
    p.causal = g.causal != 0;
    p.window = (int)std::min<int64_t>(g.window, int64_t(1) << 30);
    if (y.parts) {
        const int D3 = attn::parts_size((int)D);
        p.D3 = D3;
        p.k_plane = B * Lk * Hk * D3;
        p.q_plane = B * Lq * H * D3;
        p.k3 = {room + y.k3, Lk * Hk * D3, Hk * D3, D3, 1};
        p.v3 = {room + y.v3, Lk * Hk * D3, Hk * D3, D3, 1};
        p.q3 = {room + y.q3, Lq * H * D3, H * D3, D3, 1};
        p.dout3 = {room + y.dout3, Lq * H * D3, H * D3, D3, 1};
    }
    p.tiles = y.tiles;
    p.splits = y.splits;
    p.part = (float*)(room + y.part);
    p.part_ml = (float*)(room + y.part_ml);
    p.stats = (float*)(room + y.stats);
    p.dq_splits = y.dq_splits;
    p.dk_splits = y.dk_splits;
    p.part_dq = (float*)(room + y.part_dq);
    p.part_dk = (float*)(room + y.part_dk);
    p.part_dv = (float*)(room + y.part_dv);
    return p;
}

void document_ranges(const Params& p, hipStream_t stream) {
    const int entries = p.qranges + p.kranges;
    if (!p.qdoc || entries == 0 || p.B == 0) return;
    launch("adhip_attention", document_ranges_kernel, (unsigned)((entries + 7) / 8 * p.B), 256, stream, p.qdoc, p.qdoc_b, p.qdoc_l, p.Lq,
           (int2*)p.qrange, p.qranges, p.kdoc, p.kdoc_b, p.kdoc_l, p.Lk, (int2*)p.krange, p.kranges);
}

// Keys and values, with `rows` queries and out's gradient too, in parts
void split_into_parts(const Params& p, bool rows, hipStream_t stream) {
    PartsJobs jobs = {};
    const int64_t keys = (int64_t)p.B * p.Lk * p.Hk, queries = (int64_t)p.B * p.Lq * p.Hk * p.G;
    jobs.job[0] = {p.k, (bf16*)p.k3.data, keys, p.Lk, p.Hk};
    jobs.job[1] = {p.v, (bf16*)p.v3.data, keys, p.Lk, p.Hk};
    jobs.job[2] = {p.q, (bf16*)p.q3.data, queries, p.Lq, p.Hk * p.G};
    jobs.job[3] = {p.dout, (bf16*)p.dout3.data, queries, p.Lq, p.Hk * p.G};
    const int64_t most = (rows ? std::max(keys, queries) : keys) * (p.D3 / 8);
    if (most == 0) return;
    launch("adhip_attention", parts_kernel, dim3((unsigned)((most + 255) / 256), rows ? 4 : 2), 256, stream, jobs, p.D, p.D3);
}

}  // namespace
}  // namespace adhip

using namespace adhip;

extern "C" {

int adhip_attention_workspace(adhip_ctx* ctx, const adhip_attention_args* args, int backward, size_t* bytes) {
    return context_guarded(ctx, [&] {
        const char* op = "adhip_attention_workspace";
        ADHIP_CHECK(args && bytes, "%s: no arguments", op);
        check_sizes(op, *args);
        const Layout y = layout_of(*args, backward != 0);
        check_launches(op, *args, y, backward != 0);
        *bytes = y.bytes;
    });
}

int adhip_attention(adhip_ctx* ctx, const adhip_attention_args* args, void* stream) {
    return context_guarded(ctx, [&] {
        const char* op = "adhip_attention";
        ADHIP_CHECK(args, "%s: no arguments", op);
        check_sizes(op, *args);
        const Layout y = layout_of(*args, false);
        check_launches(op, *args, y, false);
        const Params p = checked(op, *args, y, false);
        if (p.R == 0 || p.B == 0) return;
        document_ranges(p, (hipStream_t)stream);
        if (y.parts) split_into_parts(p, false, (hipStream_t)stream);
        if (args->q.type == ADHIP_BF16) attn::forward_bf16(p, y.few_rows, (hipStream_t)stream);
        else attn::forward_f32(p, y.few_rows, (hipStream_t)stream);
    });
}

int adhip_attention_backward(adhip_ctx* ctx, const adhip_attention_args* args, void* stream) {
    return context_guarded(ctx, [&] {
        const char* op = "adhip_attention_backward";
        ADHIP_CHECK(args, "%s: no arguments", op);
        check_sizes(op, *args);
        const Layout y = layout_of(*args, true);
        check_launches(op, *args, y, true);
        const Params p = checked(op, *args, y, true);
        if (p.B == 0) return;
        document_ranges(p, (hipStream_t)stream);
        if (y.parts) split_into_parts(p, true, (hipStream_t)stream);
        if (args->q.type == ADHIP_BF16) attn::backward_bf16(p, (hipStream_t)stream);
        else attn::backward_f32(p, (hipStream_t)stream);
    });
}

}  // extern "C"

// C entry points of the head norms with rotation (heads.h), the gated projections (gated.h) and gradient clipping (clip.h).
#include <cstring>

#include "clip.h"
#include "gated.h"
#include "heads.h"
#include "nhip_internal.h"

using namespace nhipk;

namespace nhip {
namespace {

bool on(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// ---- heads ----------------------------------------------------------------------------------------------

// Heads of a launch, queries' and keys' together: 64 lanes of each are 2^31 threads, and a launch has to stay below 2^32.
constexpr int64_t kHeadsLaunchRows = int64_t(1) << 25;
// Workgroups of a backward launch at most: each leaves a row of partial sums that is read again. Two rounds of the three
// that fit a CU with chunks of 8 elements, 2048 otherwise ([4, 4096, 16 + 16, 128] in chunks of 4: 1536 101 us, 2048 88,
// 4096 87, whose sums take 2 us longer).
constexpr int64_t kHeadsBlocks8 = 1536, kHeadsBlocks = 2048;

FastDiv fast_div(uint32_t d) {
    FastDiv f{d, 0, 0};
    while (f.shift < 31 && (uint32_t(1) << f.shift) < d) ++f.shift;
    f.mul = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << f.shift) - d)) / d + 1);
    return f;
}

int heads_check(const nhip_heads_desc *d, const char *what) {
    const std::string at(what);
    if (d->batch < 0 || d->seq < 0 || d->heads < 0 || d->kv_heads < 0) return fail(at + ": negative sizes");
    if (d->head_dim < 1 || d->head_dim > kHeadsMost)
        return fail(at + ": a head dim of " + std::to_string(d->head_dim) + ": 1 to " + std::to_string(kHeadsMost));
    if (d->rot < 0 || d->rot > d->head_dim || d->rot % 2)
        return fail(at + ": " + std::to_string(d->rot) + " rotated elements: an even number up to the head dim");
    if (d->seq >= (int64_t(1) << 30) || d->heads >= (int64_t(1) << 20) || d->kv_heads >= (int64_t(1) << 20))
        return fail(at + ": sequences below 2^30 and heads below 2^20");
    if (d->table_rows < 1 && d->rot > 0 && d->batch * d->seq > 0) return fail(at + ": an empty table");
    if (d->dtype != NHIP_F32 && d->dtype != NHIP_BF16 && d->dtype != NHIP_F16) return fail(at + ": heads are float32, bf16 or f16");
    if (d->positions < NHIP_POS_NONE || d->positions > NHIP_POS_I64) return fail(at + ": positions are int32, int64 or none");
    return 0;
}

// Tokens of one launch.
int64_t heads_tokens(const nhip_heads_desc *d) {
    const int64_t heads = d->heads + d->kv_heads, most = kHeadsLaunchRows / (heads > 0 ? heads : 1);
    const int64_t tokens = d->batch * d->seq;
    return tokens < most ? tokens : most;
}

// Elements a chunk of the vector kernels, or 0: the general kernel. Both of a row's chunks start on a chunk's bytes.
struct HeadsPlan {
    int e, lanes;
    int64_t launches;
};

bool heads_strides(const nhip_heads_desc *d, int e, bool bwd) {
    const int64_t st[] = {d->q_b,  d->q_s,  d->q_n,  d->k_b,  d->k_s,  d->k_n,  d->oq_b, d->oq_s, d->oq_n,
                          d->ok_b, d->ok_s, d->ok_n, d->dq_b, d->dq_s, d->dq_n, d->dk_b, d->dk_s, d->dk_n};
    for (int i = 0; i < (bwd ? 18 : 12); ++i)
        if (st[i] % e) return false;
    return true;
}

HeadsPlan heads_plan(const nhip_heads_desc *d, bool bwd, std::initializer_list<const void *> heads, const float *cos,
                     const float *sin) {
    HeadsPlan p;
    const int64_t tokens = d->batch * d->seq, each = heads_tokens(d);
    p.launches = each ? (tokens + each - 1) / each : 0;
    p.e = 0;
    for (int e : {8, 4, 2}) {
        if (e == 8 && d->dtype == NHIP_F32) continue;  // 4 elements are 16 bytes
        const size_t bytes = size_t(e) * (d->dtype == NHIP_F32 ? 4 : 2);
        bool ok = d->head_dim % (2 * e) == 0 && d->rot % (2 * e) == 0 && d->head_dim / (2 * e) <= 64 && heads_strides(d, e, bwd);
        for (const void *h : heads) ok = ok && on(h, bytes);
        ok = ok && on(cos, e == 2 ? 8 : 16) && on(sin, e == 2 ? 8 : 16);
        if (ok) {
            p.e = e;
            break;
        }
    }
    const int64_t need = p.e ? d->head_dim / (2 * p.e) : d->rot / 2 + (d->head_dim - d->rot + 1) / 2;
    p.lanes = p.e ? 1 : 32;
    while (p.lanes < need && p.lanes < 64) p.lanes *= 2;
    return p;
}

struct HeadsBlocks {
    int64_t q, k;
};
// Workgroups of a backward launch for the queries and the keys, in proportion to their rows: four rows a group of lanes, but
// a workgroup a CU before that ([3, 331, 6 + 2, 80]: 497 workgroups of one row each leave as many rows to sum).
HeadsBlocks heads_blocks(const nhip_heads_desc *d, int lanes, int64_t cap) {
    const int64_t t = heads_tokens(d), q = t * d->heads, k = t * d->kv_heads, groups = 256 / lanes;
    auto share = [&](int64_t rows) -> int64_t {
        if (rows == 0) return 0;
        const int64_t need = (rows + groups - 1) / groups, part = 256 * rows / (q + k) + 1;
        const int64_t want = need / 4 > part ? need / 4 : (need < part ? need : part);
        const int64_t most = cap * rows / (q + k);  // both within the cap: one workgroup over it is another round
        return want < most ? want : most > 0 ? most : 1;
    };
    return {share(q), share(k)};
}

size_t heads_workspace(const nhip_heads_desc *d) {
    const int64_t tokens = d->batch * d->seq, each = heads_tokens(d);
    if (each == 0) return 0;
    return size_t((tokens + each - 1) / each) * size_t(kHeadsBlocks + 2) * size_t(d->head_dim) * 4;
}

template <typename T, int E>
int heads_launch_fwd(hipStream_t st, HeadsArgs &a) {
    const uint32_t groups = 256 / a.lanes;
    for (HeadsTensor &t : a.t) t.blocks = (t.rows + groups - 1) / groups;
    const uint32_t grid = a.t[0].blocks + a.t[1].blocks;
    if (!grid) return 0;
    hipLaunchKernelGGL((heads_fwd_kernel<T, E>), dim3(grid), dim3(256), 0, st, a);
    return check(hipGetLastError(), "heads_fwd_kernel launch");
}

template <typename T>
int heads_launch(hipStream_t st, HeadsArgs &a, int e, bool bwd) {
    if (!bwd) {
        if constexpr (!std::is_same<T, float>::value)
            if (e == 8) return heads_launch_fwd<T, 8>(st, a);
        if (e == 4) return heads_launch_fwd<T, 4>(st, a);
        if (e == 2) return heads_launch_fwd<T, 2>(st, a);
        for (HeadsTensor &t : a.t) {
            const int64_t blocks = (int64_t(t.rows) * a.lanes + 255) / 256;
            t.blocks = uint32_t(blocks < 16384 ? blocks : 16384);
        }
        const uint32_t grid = a.t[0].blocks + a.t[1].blocks;
        if (!grid) return 0;
        hipLaunchKernelGGL((heads_any_kernel<T, false>), dim3(grid), dim3(256), 0, st, a);
        return check(hipGetLastError(), "heads_any_kernel launch");
    }
    const uint32_t grid = a.t[0].blocks + a.t[1].blocks;
    if (!grid) return 0;
    if constexpr (!std::is_same<T, float>::value) {
        if (e == 8) {
            hipLaunchKernelGGL((heads_bwd_kernel<T, 8>), dim3(grid), dim3(256), 0, st, a);
            return check(hipGetLastError(), "heads_bwd_kernel launch");
        }
    }
    if (e == 4) hipLaunchKernelGGL((heads_bwd_kernel<T, 4>), dim3(grid), dim3(256), 0, st, a);
    else if (e == 2) hipLaunchKernelGGL((heads_bwd_kernel<T, 2>), dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((heads_any_kernel<T, true>), dim3(grid), dim3(256), 0, st, a);
    return check(hipGetLastError(), "heads_bwd_kernel launch");
}

HeadsArgs heads_args(const nhip_heads_desc *d, const HeadsPlan &p, const void *q, const void *k, const void *qw, const void *kw,
                     const float *cos, const float *sin, const void *pos) {
    HeadsArgs a;
    std::memset(&a, 0, sizeof(a));
    HeadsTensor &x = a.t[0], &y = a.t[1];
    x.x = q, y.x = k, x.w = qw, y.w = kw;
    x.x_b = d->q_b, x.x_s = d->q_s, x.x_n = d->q_n, y.x_b = d->k_b, y.x_s = d->k_s, y.x_n = d->k_n;
    x.y_b = d->oq_b, x.y_s = d->oq_s, x.y_n = d->oq_n, y.y_b = d->ok_b, y.y_s = d->ok_s, y.y_n = d->ok_n;
    x.dy_b = d->dq_b, x.dy_s = d->dq_s, x.dy_n = d->dq_n, y.dy_b = d->dk_b, y.dy_s = d->dk_s, y.dy_n = d->dk_n;
    x.heads = fast_div(uint32_t(d->heads > 0 ? d->heads : 1));
    y.heads = fast_div(uint32_t(d->kv_heads > 0 ? d->kv_heads : 1));
    a.cos = cos, a.sin = sin;
    a.positions = d->positions == NHIP_POS_NONE ? nullptr : pos;
    a.pos64 = d->positions == NHIP_POS_I64;
    a.table_rows = d->table_rows > 0 ? d->table_rows : 1;
    a.seq = d->seq;
    a.seq_div = fast_div(uint32_t(d->seq > 0 ? d->seq : 1));
    a.d = int(d->head_dim), a.rot = int(d->rot), a.interleaved = d->interleaved != 0;
    a.lanes = p.lanes;
    a.eps = d->eps;
    return a;
}

template <class F>
int by_type(int dtype, F &&f) {
    if (dtype == NHIP_F32) return f(float{});
    if (dtype == NHIP_BF16) return f(bf16_t{});
    return f(f16_t{});
}

}  // namespace

int heads_on(hipStream_t st, const nhip_heads_desc *d, const void *q, const void *k, const void *qw, const void *kw,
             const float *cos, const float *sin, const void *pos, void *oq, void *ok) {
    if (heads_check(d, "nhip_qk_norm_rope")) return 1;
    if (d->positions != NHIP_POS_NONE && !pos && d->batch * d->seq > 0) return fail("nhip_qk_norm_rope: no positions");
    const HeadsPlan p = heads_plan(d, false, {q, k, qw, kw, oq, ok}, cos, sin);
    HeadsArgs a = heads_args(d, p, q, k, qw, kw, cos, sin, pos);
    a.t[0].y = oq, a.t[1].y = ok;
    const int64_t tokens = d->batch * d->seq, each = heads_tokens(d);
    for (int64_t t0 = 0; t0 < tokens; t0 += each) {
        const int64_t n = tokens - t0 < each ? tokens - t0 : each;
        a.token0 = t0;
        a.t[0].rows = uint32_t(n * d->heads), a.t[1].rows = uint32_t(n * d->kv_heads);
        if (by_type(d->dtype, [&](auto t) { return heads_launch<decltype(t)>(st, a, p.e, false); })) return 1;
    }
    return 0;
}

int heads_bwd_on(hipStream_t st, const nhip_heads_desc *d, const void *q, const void *k, const void *qw, const void *kw,
                 const float *cos, const float *sin, const void *pos, const void *doq, const void *dok, void *dq, void *dk,
                 void *dqw, void *dkw, void *ws) {
    if (heads_check(d, "nhip_qk_norm_rope_bwd")) return 1;
    const int64_t tokens = d->batch * d->seq, each = heads_tokens(d);
    if (d->positions != NHIP_POS_NONE && !pos && tokens > 0) return fail("nhip_qk_norm_rope_bwd: no positions");
    if ((dqw || dkw) && !ws && heads_workspace(d) > 0) return fail("nhip_qk_norm_rope_bwd: no workspace");
    const HeadsPlan p = heads_plan(d, true, {q, k, qw, kw, doq, dok, dq, dk}, cos, sin);
    HeadsArgs a = heads_args(d, p, q, k, qw, kw, cos, sin, pos);
    a.t[0].dy = doq, a.t[1].dy = dok, a.t[0].y = dq, a.t[1].y = dk;
    const HeadsBlocks b = heads_blocks(d, p.lanes, p.e == 8 ? kHeadsBlocks8 : kHeadsBlocks);
    float *pq = static_cast<float *>(ws), *pk = pq ? pq + p.launches * b.q * d->head_dim : nullptr;
    for (int64_t i = 0; i < p.launches; ++i) {
        const int64_t t0 = i * each, n = tokens - t0 < each ? tokens - t0 : each;
        a.token0 = t0;
        a.t[0].rows = uint32_t(n * d->heads), a.t[1].rows = uint32_t(n * d->kv_heads);
        a.t[0].blocks = uint32_t(b.q), a.t[1].blocks = uint32_t(b.k);
        a.t[0].part = dqw ? pq + i * b.q * d->head_dim : nullptr;
        a.t[1].part = dkw ? pk + i * b.k * d->head_dim : nullptr;
        if (by_type(d->dtype, [&](auto t) { return heads_launch<decltype(t)>(st, a, p.e, true); })) return 1;
    }
    if (!dqw && !dkw) return 0;
    HeadsSum s;
    s.part[0] = pq, s.part[1] = pk, s.out[0] = dqw, s.out[1] = dkw;
    s.rows[0] = uint32_t(p.launches * b.q), s.rows[1] = uint32_t(p.launches * b.k);
    s.d = int(d->head_dim);
    return by_type(d->dtype, [&](auto t) {
        hipLaunchKernelGGL((heads_sum_kernel<decltype(t)>), dim3(unsigned((d->head_dim + 63) / 64), 2), dim3(1024), 0, st, s);
        return check(hipGetLastError(), "heads_sum_kernel launch");
    });
}

// ---- gated projections ----------------------------------------------------------------------------------

namespace {

enum { kSkinnyCfg = 0, kStream256, kStream128Cfg, kDeepCfg, kPartsCfg, kGatedConfigs };

int gated_check(const nhip_gated_desc *d, const char *what) {
    const std::string at(what);
    if (d->m < 0 || d->n < 0 || d->k < 0) return fail(at + ": negative sizes");
    if (d->dtype != NHIP_BF16 && d->dtype != NHIP_F16) return fail(at + ": bf16 or f16");
    if (d->activation < NHIP_ACT_SILU || d->activation > NHIP_ACT_SIGMOID) return fail(at + ": unknown activation");
    return 0;
}

int64_t tiles(int64_t m, int64_t bm, int64_t n, int64_t bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }

// Whether tiles of bm x bn, a workgroup of `threads` each, are a launch of fewer than 2^32 threads (their count within 64 bits).
bool tiles_ok(int64_t m, int64_t bm, int64_t n, int64_t bn, int threads) {
    const int64_t a = (m + bm - 1) / bm, b = (n + bn - 1) / bn;
    return a < (int64_t(1) << 32) && b < (int64_t(1) << 32) / (threads * (a > 0 ? a : 1));
}

// The stream kernels' k: some, and 256 rows of it within the 2^31 bytes of a buffer.
bool gated_stream_ok(const nhip_gated_desc *d) { return d->k > 0 && d->k < (int64_t(1) << 21); }
bool gated_skinny_ok(const nhip_gated_desc *d) { return d->m <= 64 && d->k < (int64_t(1) << 30); }

// Whether gated_stream can read rows of these lengths and distances in place (from 16-byte addresses).
bool gated_rows(const nhip_gated_desc *d) {
    return d->k % 8 == 0 && d->x_m % 8 == 0 && d->w_n % 8 == 0 &&
           stream_buffer_ok(d->m, d->n, d->k, false, false, d->x_m, 1, 1, d->w_n);
}

// Parts of k for kPartsCfg and the time that takes: the deep tiles' 5 us and 0.0065 a k, and the parts' writing and joining.
struct GatedSplit {
    int parts, k_part;
    double us;
};
GatedSplit gated_split(const nhip_gated_desc *d) {
    GatedSplit best{0, 0, 0.0};
    const int64_t total = (d->k + 63) / 64, t = tiles(d->m, 128, d->n, 64);
    for (int64_t s = 2; s <= 32; s *= 2) {
        const int64_t part = (total + s - 1) / s, parts = (total + part - 1) / part;
        if (best.parts && (part < 4 || t * parts > 256)) break;
        const double us = 5.0 + 0.0065 * 64.0 * double(part) + 4.2 + 16.0 * double(parts) * double(d->m) * double(d->n) / 6.13e6;
        if (!best.parts || us < best.us) best = GatedSplit{int(parts), int(part), us};
    }
    return best;
}

// Tile rows, columns and threads of a config's workgroups.
struct GatedTile {
    int rows, columns, threads;
};
GatedTile gated_tile(const nhip_gated_desc *d, int cfg) {
    if (cfg == kSkinnyCfg) return {64, 16, d->m <= 32 ? 512 : 256};
    return cfg == kStream256 ? GatedTile{256, 128, 512} : GatedTile{128, 64, 256};
}

int gated_default(const nhip_gated_desc *d) {
    const bool in_parts = d->k >= 1024 && gated_stream_ok(d) && tiles(d->m, 128, d->n, 64) <= 128;
    if (gated_skinny_ok(d)) {
        if (d->m <= 32 || d->k < 768 || !gated_stream_ok(d) || !gated_rows(d)) return kSkinnyCfg;
        // 33 to 64 rows of weights that leave gated_skinny more than a workgroup a CU, which then run one after the other:
        // tiles of 128 rows are faster though half of one is empty ([64, 2048] x [8192, 2048] 19.2 us, 24.1, [64, 4096] x
        // [11008, 4096] 33.9, 64.8; of 4096 features [64, 1024] 11.8, 8.2; of 32 rows [32, 2048] x [8192, 2048] 19.2, 18.3)
        if (d->n > 4096) return kDeepCfg;
        // one workgroup a CU at most: 3 us and 0.0039 (33 rows) to 0.0052 (64) a k ([64, 4096] x [1024, 4096] 23.9 us, in parts
        // 15.5; [33, 2048] 10.3, 11.1)
        return in_parts && gated_split(d).us < 3.0 + double(d->k) * (0.0026 + 0.00004 * double(d->m)) ? kPartsCfg : kSkinnyCfg;
    }
    if (tiles(d->m, 256, d->n, 128) >= 256) return kStream256;
    // one workgroup a CU: three stages ([1463, 3392] x [712, 3392] 28.9 us, in two 41.2), in parts where k is long and tiles
    // are few ([139, 3840] x [1464, 3840] 30.1 us, in parts 18.1; [500, 8192] x [2048, 8192] 60.4, 45.4; [256, 2048] x
    // [4096, 2048] 19.5, 21.0)
    if (tiles(d->m, 128, d->n, 64) > 256 || d->k < 768) return kStream128Cfg;
    return in_parts && gated_split(d).us < 5.0 + 0.0065 * double(d->k) ? kPartsCfg : kDeepCfg;
}

bool gated_launch_ok(const nhip_gated_desc *d, int cfg) {
    const GatedTile t = gated_tile(d, cfg);
    return tiles_ok(d->m, t.rows, d->n, t.columns, t.threads);
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

// Bytes of the operands' copies, which lie ahead of the parts.
size_t gated_pad_bytes(const nhip_gated_desc *d, int cfg) {
    if (cfg == kSkinnyCfg || gated_rows(d)) return 0;
    return up16(size_t(d->m + 2 * d->n) * size_t((d->k + 7) / 8 * 8) * 2);
}

size_t gated_workspace(const nhip_gated_desc *d) {
    const int cfg = d->config < 0 ? gated_default(d) : d->config;
    return gated_pad_bytes(d, cfg) + (cfg == kPartsCfg ? size_t(gated_split(d).parts) * 2 * size_t(d->m) * size_t(d->n) * 4 : 0);
}

// `more`: arguments past the output; parts: blockIdx.z.
template <class K, class Out, class... More>
int gated_go(hipStream_t st, K kern, GemmShape s, const GatedTile &t, int lds, const void *x, const void *gate, const void *up,
             const Out &out, int parts = 1, More... more) {
    s.tiles_m = int((s.m + t.rows - 1) / t.rows);
    s.tiles_n = int((s.n + t.columns - 1) / t.columns);
    if (lds > 64 * 1024 &&
        check(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
              "hipFuncSetAttribute"))
        return 1;
    hipLaunchKernelGGL(kern, dim3(unsigned(s.tiles_m * s.tiles_n), 1, unsigned(parts)), dim3(t.threads), lds, st, s,
                       static_cast<const uint16_t *>(x), static_cast<const uint16_t *>(gate), static_cast<const uint16_t *>(up),
                       out, more...);
    return check(hipGetLastError(), "gated kernel launch");
}

// Copies `count` matrices of rows of k elements to whole rows of 16-byte chunks at ws, one after the other.
int gated_pad(hipStream_t st, GatedPad &p, int count, const void *const *src, const int64_t *rows, const int64_t *to_rows,
              const int64_t *ld, int64_t k, void *ws) {
    std::memset(&p, 0, sizeof(p));
    p.k = k, p.kp = (k + 7) / 8 * 8;
    uint16_t *to = static_cast<uint16_t *>(ws);
    int64_t most = 1;
    for (int i = 0; i < count; ++i) {
        p.src[i] = static_cast<const uint16_t *>(src[i]);
        p.rows[i] = rows[i], p.to_rows[i] = to_rows[i], p.ld[i] = ld[i];
        p.dst[i] = to;
        to += to_rows[i] * p.kp;
        if (to_rows[i] > most) most = to_rows[i];
    }
    const int64_t blocks = (most * (p.kp / 8) + 255) / 256;
    hipLaunchKernelGGL(gated_pad_kernel, dim3(unsigned(blocks < 4096 ? (blocks ? blocks : 1) : 4096), unsigned(count)), dim3(256), 0, st, p);
    return check(hipGetLastError(), "gated_pad_kernel launch");
}

template <bool F16, bool ANY>
int gated_few(hipStream_t st, const GemmShape &s, const GatedTile &t, const void *x, const void *gate, const void *up, const GatedOut &o) {
    if (s.m <= 16) return gated_go(st, gated_skinny<F16, 1, 8, ANY>, s, t, 0, x, gate, up, o);
    if (s.m <= 32) return gated_go(st, gated_skinny<F16, 2, 8, ANY>, s, t, 0, x, gate, up, o);
    return gated_go(st, gated_skinny<F16, 4, 4, ANY>, s, t, 0, x, gate, up, o);
}

template <bool F16>
int gated_run(hipStream_t st, int cfg, const nhip_gated_desc *d, GemmShape s, const void *x, const void *gate, const void *up,
              const GatedOut &o, bool in_place, void *ws) {
    const GatedTile t = gated_tile(d, cfg);
    if (cfg == kSkinnyCfg) return in_place ? gated_few<F16, false>(st, s, t, x, gate, up, o) : gated_few<F16, true>(st, s, t, x, gate, up, o);
    if (!in_place) {
        GatedPad p;
        const int64_t rows[3] = {s.m, s.n, s.n}, ld[3] = {s.a_m, s.b_n, s.b_n};
        const void *src[3] = {x, gate, up};
        if (gated_pad(st, p, 3, src, rows, rows, ld, s.k, ws)) return 1;
        x = p.dst[0], gate = p.dst[1], up = p.dst[2];
        s.k = s.a_m = s.b_n = p.kp;
    }
    constexpr int deep = gemm_stream_lds_bytes<64, 2, 128, 3>();
    if (cfg == kStream256)
        return gated_go(st, gated_stream<F16, 256, 3>, s, t, gemm_stream_lds_bytes<64, 4>(), x, gate, up, o);
    if (cfg == kDeepCfg) return gated_go(st, gated_stream<F16, 128, 1, 3>, s, t, deep, x, gate, up, o);
    if (cfg == kStream128Cfg)
        return gated_go(st, gated_stream<F16, 128, 0>, s, t, gemm_stream_lds_bytes<64, 2, 128>(), x, gate, up, o);
    const GatedSplit p = gated_split(d);
    float *sums = reinterpret_cast<float *>(static_cast<char *>(ws) + gated_pad_bytes(d, cfg));
    GemmShape part = s;
    part.d_m = s.n;
    if (gated_go(st, gated_stream_part<F16>, part, t, deep, x, gate, up, GatedParts{sums}, p.parts, p.k_part)) return 1;
    const bool vec = s.n % 4 == 0;
    const int64_t blocks = (s.m * (vec ? s.n / 4 : s.n) + 255) / 256;
    const dim3 grid(unsigned(blocks < 4096 ? blocks : 4096));
    if (vec) hipLaunchKernelGGL((gated_join_kernel<4>), grid, dim3(256), 0, st, s, sums, p.parts, o);
    else hipLaunchKernelGGL((gated_join_kernel<1>), grid, dim3(256), 0, st, s, sums, p.parts, o);
    return check(hipGetLastError(), "gated_join_kernel launch");
}

}  // namespace

int gated_on(hipStream_t st, const nhip_gated_desc *d, const void *x, const void *gate, const void *up, void *h, float *g,
             float *u, void *ws) {
    if (gated_check(d, "nhip_gated_linear")) return 1;
    if (!g != !u) return fail("nhip_gated_linear: g and u go together");
    if (d->m == 0 || d->n == 0) return 0;
    int cfg = d->config < 0 ? gated_default(d) : d->config;
    if (cfg >= kGatedConfigs || !(cfg == kSkinnyCfg ? gated_skinny_ok(d) : gated_stream_ok(d)))
        return fail("nhip_gated_linear: config " + std::to_string(cfg) + " does not take these operands");
    if (!gated_launch_ok(d, cfg)) return fail("nhip_gated_linear: a launch of 2^32 threads");
    GemmShape s;
    std::memset(&s, 0, sizeof(s));
    s.m = d->m, s.n = d->n, s.k = d->k;
    s.a_m = d->x_m, s.a_k = 1, s.b_k = 1, s.b_n = d->w_n, s.d_m = d->h_m, s.d_n = 1;
    const bool rows = cfg == kSkinnyCfg ? d->k % 8 == 0 && d->x_m % 8 == 0 && d->w_n % 8 == 0 : gated_rows(d);
    const bool in_place = rows && on(x, 16) && on(gate, 16) && on(up, 16);
    if (!in_place && cfg != kSkinnyCfg) {
        if (rows) return fail("nhip_gated_linear: operands of such rows start on 16 bytes");
    }
    if (gated_workspace(d) && (!ws || !on(ws, 16))) return fail("nhip_gated_linear: no workspace, or one off 16 bytes");
    const GatedOut o{h, g, u, d->activation, d->dtype};
    return d->dtype == NHIP_F16 ? gated_run<true>(st, cfg, d, s, x, gate, up, o, in_place, ws)
                                : gated_run<false>(st, cfg, d, s, x, gate, up, o, in_place, ws);
}

int gated_grad_on(hipStream_t st, const nhip_gated_desc *d, const void *dh, const float *g, const float *u, void *dgu) {
    if (gated_check(d, "nhip_gated_linear_grad")) return 1;
    if (d->m == 0 || d->n == 0) return 0;
    const int64_t np = (d->n + 7) / 8 * 8;
    GatedGrad a{dh, g, u, dgu, d->m, d->n, np, d->h_m, d->activation};
    if (!on(dgu, 16)) return fail("nhip_gated_linear_grad: [dg | du] starts on 16 bytes");
    const bool whole_rows = d->n % 8 == 0 && d->h_m % 8 == 0 && on(dh, 16) && on(g, 16) && on(u, 16);
    const int64_t work = d->m * (np / 8), blocks = (work + 255) / 256;
    const dim3 grid(unsigned(blocks < 8192 ? blocks : 8192));
    if (d->dtype == NHIP_F16) {
        if (whole_rows) hipLaunchKernelGGL((gated_grad_kernel<f16_t, false>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((gated_grad_kernel<f16_t, true>), grid, dim3(256), 0, st, a);
    } else {
        if (whole_rows) hipLaunchKernelGGL((gated_grad_kernel<bf16_t, false>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((gated_grad_kernel<bf16_t, true>), grid, dim3(256), 0, st, a);
    }
    return check(hipGetLastError(), "gated_grad_kernel launch");
}

namespace {

// The tile and the parts of a product of z batches over `total` k tiles of 64: as many parts as make the tiles' rounds on the
// chip the shortest, each round as long as its k, the parts' writing and reading added. The rates are the split dots'
// (Plan._split_us), whose loops these are. longest: k tiles that a part may have at most.
struct PartPlan {
    int tm, parts, k_part;
    bool deep;  // at most a workgroup a CU of 128-row tiles: three stages
    double us;
};
// The parts' sums, written and added, of `elements` results.
double parts_us(int64_t elements, int64_t parts) { return parts > 1 ? 4.2 + 8.0 * double(parts) * double(elements) / 6.13e6 : 0.0; }

PartPlan part_plan(int64_t m, int64_t n, int64_t z, int64_t total, int64_t longest) {
    PartPlan best{0, 0, 0, false, 0.0};
    if (total < 1) total = 1;  // no tokens: nothing is launched, the workspace is asked for all the same
    for (int tm : {256, 128})
        for (int s = 1; s <= 64; s *= 2) {
            const int64_t part = (total + s - 1) / s, parts = (total + part - 1) / part;
            if (part > longest) continue;
            if (best.tm && parts > 1 && (part < 8 || parts * z * m * n * 4 > (int64_t(64) << 20))) continue;
            const int64_t t = tiles(m, tm, n, tm) * z * parts;
            // 256: a workgroup a CU; 128: two, one alone taking 0.79 of a round of both, 0.62 with three stages, whose LDS
            // leaves room for one ([2000, 1024] x [2048, 1024] weights' gradients 30.4 -> 23.8 us; launches of more than 256
            // are slower so: [1463, 3392] x [712, 3392] 26.7 -> 33.2)
            const bool deep = tm == 128 && t <= 256;
            double rounds = tm == 256 ? double((t + 255) / 256) : deep ? 0.62 : double(t / 512);
            const int64_t rest = t % 512;
            if (tm == 128 && !deep) rounds += rest == 0 ? 0.0 : rest <= 256 ? 0.79 : 1.0;
            const double us = 6.2 + 64.0 * double(part) * (tm == 256 ? 0.02355 : 0.0142) * rounds + parts_us(z * m * n, parts);
            if (!best.tm || us < best.us) best = PartPlan{tm, int(parts), int(part), deep, us};
        }
    return best;
}

int64_t whole(int64_t n) { return (n + 7) / 8 * 8; }  // rounded up to 16 bytes of elements

// The input's gradient, [m, k] of [dg | du] [m, 2 whole(n)] and the weights [n, k].
PartPlan input_grad_plan(const nhip_gated_desc *d) { return part_plan(d->m, d->k, 1, 2 * ((whole(d->n) + 63) / 64), int64_t(1) << 30); }

// The weights' gradients, [n, k] each: a part's rows of [dg | du] and of x lie within 2^31 bytes.
int64_t weight_grad_longest(const nhip_gated_desc *d) {
    const int64_t row = 2 * whole(d->n) > whole(d->x_m) ? 2 * whole(d->n) : whole(d->x_m);
    return ((int64_t(1) << 30) - 1024) / (64 * (row > 0 ? row : 1));
}
PartPlan weight_grad_plan(const nhip_gated_desc *d) {
    return part_plan(d->n, d->k, 2, (d->m + 63) / 64, weight_grad_longest(d));
}

bool weights_whole(const nhip_gated_desc *d) { return d->n % 8 == 0 && d->k % 8 == 0 && d->w_n % 8 == 0; }
bool input_whole(const nhip_gated_desc *d) { return d->k % 8 == 0 && d->x_m % 8 == 0; }

int backward_check(const nhip_gated_desc *d, const char *what) {
    if (gated_check(d, what)) return 1;
    if (d->n >= (int64_t(1) << 21) || whole(d->n) * (d->w_n > whole(d->k) ? d->w_n : whole(d->k)) >= (int64_t(1) << 30) - 1024 ||
        weight_grad_plan(d).tm == 0)
        return fail(std::string(what) + ": weights or rows of 2^31 bytes");
    // the input's gradient and the weights', in the smaller tiles
    if (!tiles_ok(d->m, 128, d->k, 128, 256) || !tiles_ok(d->n, 128, d->k, 128, 256))
        return fail(std::string(what) + ": a launch of 2^32 threads");
    return 0;
}

size_t input_grad_pad(const nhip_gated_desc *d) {
    return weights_whole(d) ? 0 : size_t(2 * whole(d->n)) * size_t(whole(d->k)) * 2;
}
size_t weight_grad_pad(const nhip_gated_desc *d) { return input_whole(d) ? 0 : size_t(d->m) * size_t(whole(d->k)) * 2; }
// Both products in one launch of at most a workgroup a CU, each in the parts that make the longer one the shortest, where that
// is faster than one after the other; tm 0: it is not.
struct GradPlans {
    PartPlan i, w;
};
GradPlans paired_plans(const nhip_gated_desc *d) {
    GradPlans best;
    std::memset(&best, 0, sizeof(best));
    if (d->m == 0 || d->n == 0 || d->k == 0) return best;
    const int64_t ki = 2 * ((whole(d->n) + 63) / 64), kw = (d->m + 63) / 64;
    const int64_t ti = tiles(d->m, 128, d->k, 128), tw = 2 * tiles(d->n, 128, d->k, 128);
    const PartPlan i = input_grad_plan(d), w = weight_grad_plan(d);
    if (!i.deep || !w.deep) return best;
    double least = i.us + w.us;
    for (int64_t a = 1; a <= 64; a *= 2)
        for (int64_t b = 1; b <= 64; b *= 2) {
            const int64_t pi = (ki + a - 1) / a, pw = (kw + b - 1) / b, ni = (ki + pi - 1) / pi, nw = (kw + pw - 1) / pw;
            if (ti * ni + tw * nw > 256 || pw > weight_grad_longest(d) || (ni > 1 && pi < 4) || (nw > 1 && pw < 4)) continue;
            const double us = 6.2 + 64.0 * double(pi > pw ? pi : pw) * 0.0142 * 0.62 + parts_us(d->m * d->k, ni) +
                              parts_us(2 * d->n * d->k, nw);
            if (us < least) least = us, best = GradPlans{{128, int(ni), int(pi), true, us}, {128, int(nw), int(pw), true, us}};
        }
    return best;
}

size_t input_grad_bytes(const nhip_gated_desc *d, const PartPlan &p) {
    return up16(input_grad_pad(d)) + up16(p.parts > 1 ? size_t(p.parts) * size_t(d->m) * size_t(d->k) * 4 : 0);
}

size_t weight_grad_bytes(const nhip_gated_desc *d, const PartPlan &p) {
    return up16(weight_grad_pad(d)) + up16(p.parts > 1 ? size_t(p.parts) * 2 * size_t(d->n) * size_t(d->k) * 4 : 0);
}

size_t backward_workspace(const nhip_gated_desc *d) {
    const GradPlans both = paired_plans(d);
    size_t most = both.i.tm ? input_grad_bytes(d, both.i) + weight_grad_bytes(d, both.w) : 0;
    for (size_t alone : {input_grad_bytes(d, input_grad_plan(d)), weight_grad_bytes(d, weight_grad_plan(d))})
        if (alone > most) most = alone;
    return most;
}

// One of the backward's products, ready to be launched: z batches of s, in parts to `sums` or whole to `to`.
struct GradProduct {
    GemmShape s;
    PartPlan p;
    int64_t z;
    const uint16_t *a, *b, *b2;
    AnyStore to;
    float *sums;

    // What the kernel stores: the result, or the parts' sums.
    GemmShape shape() const {
        GemmShape q = s;
        if (p.parts > 1) q.d_m = s.n, q.d_n = 1, q.d_batch[0] = s.m * s.n, q.d_split = z * s.m * s.n;
        return q;
    }
    AnyStore store() const { return p.parts > 1 ? AnyStore{sums, 0} : to; }
};

void product_ready(GradProduct &o) {
    o.s.tiles_m = int((o.s.m + o.p.tm - 1) / o.p.tm);
    o.s.tiles_n = int((o.s.n + o.p.tm - 1) / o.p.tm);
}

int input_product(hipStream_t st, const nhip_gated_desc *d, const void *dgu, const void *gate, const void *up, void *dx, void *ws,
                  const PartPlan &p, GradProduct &o) {
    o.p = p;
    if (!ws && input_grad_bytes(d, p)) return fail("nhip_gated_input_grad: no workspace");
    if (!on(dgu, 16) || !on(ws, 16)) return fail("nhip_gated_input_grad: [dg | du] and the workspace start on 16 bytes");
    if (!on(dx, 2)) return fail("nhip_gated_input_grad: the result starts on an element");
    GemmShape &s = o.s;
    std::memset(&s, 0, sizeof(s));
    const int64_t np = whole(d->n);
    s.m = d->m, s.n = d->k, s.k = 2 * np;
    s.a_m = 2 * np, s.a_k = 1, s.b_k = d->w_n, s.b_n = 1, s.d_m = d->k, s.d_n = 1;
    if (!weights_whole(d)) {
        GatedPad pad;
        const void *src[2] = {gate, up};
        const int64_t rows[2] = {d->n, d->n}, to_rows[2] = {np, np}, ld[2] = {d->w_n, d->w_n};
        if (gated_pad(st, pad, 2, src, rows, to_rows, ld, d->k, ws)) return 1;
        gate = pad.dst[0], up = pad.dst[1];
        s.b_k = pad.kp;
    } else if (!on(gate, 16) || !on(up, 16)) {
        return fail("nhip_gated_input_grad: weights of whole rows start on 16 bytes");
    }
    o.z = 1;
    o.a = static_cast<const uint16_t *>(dgu), o.b = static_cast<const uint16_t *>(gate), o.b2 = static_cast<const uint16_t *>(up);
    o.to = AnyStore{dx, d->dtype};
    o.sums = reinterpret_cast<float *>(static_cast<char *>(ws) + up16(input_grad_pad(d)));
    product_ready(o);
    return 0;
}

int weight_product(hipStream_t st, const nhip_gated_desc *d, const void *dgu, const void *x, void *dgate, void *dup, void *ws,
                   const PartPlan &p, GradProduct &o) {
    o.p = p;
    if (!ws && weight_grad_bytes(d, p)) return fail("nhip_gated_weight_grad: no workspace");
    if (!on(dgu, 16) || !on(ws, 16)) return fail("nhip_gated_weight_grad: [dg | du] and the workspace start on 16 bytes");
    if (!on(dgate, 2) || !on(dup, 2)) return fail("nhip_gated_weight_grad: results start on an element");
    GemmShape &s = o.s;
    std::memset(&s, 0, sizeof(s));
    const int64_t np = whole(d->n);
    s.m = d->n, s.n = d->k, s.k = d->m;
    s.a_m = 1, s.a_k = 2 * np, s.b_k = d->x_m, s.b_n = 1, s.d_m = d->k, s.d_n = 1;
    o.z = dup ? 2 : 1;
    s.nbatch = 1, s.batch[0] = o.z, s.a_batch[0] = np;
    // the second result as the first one's batch, wherever it lies
    if (dup) s.d_batch[0] = (static_cast<char *>(dup) - static_cast<char *>(dgate)) / 2;
    if (!input_whole(d)) {
        GatedPad pad;
        if (gated_pad(st, pad, 1, &x, &d->m, &d->m, &d->x_m, d->k, ws)) return 1;
        x = pad.dst[0];
        s.b_k = pad.kp;
    } else if (!on(x, 16)) {
        return fail("nhip_gated_weight_grad: whole rows of x start on 16 bytes");
    }
    o.a = static_cast<const uint16_t *>(dgu), o.b = static_cast<const uint16_t *>(x), o.b2 = nullptr;
    o.to = AnyStore{dgate, d->dtype};
    o.sums = reinterpret_cast<float *>(static_cast<char *>(ws) + up16(weight_grad_pad(d)));
    product_ready(o);
    return 0;
}

int lds_room(const void *kern, int lds) {
    return check(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute");
}

// The result of a product that ran in parts.
int parts_sum(hipStream_t st, const GradProduct &o) {
    if (o.p.parts == 1) return 0;
    uint16_t *out = static_cast<uint16_t *>(o.to.d);
    const GatedSum g{o.sums, {out, out + o.s.d_batch[0]}, o.s.m * o.s.n, o.p.parts};
    const bool vec = g.mn % 4 == 0 && on(g.out[0], 8) && on(g.out[1], 8);
    const int64_t blocks = ((vec ? g.mn / 4 : g.mn) + 255) / 256;
    const dim3 grid(unsigned(blocks < 4096 ? blocks : 4096), unsigned(o.z));
    if (o.to.dtype == NHIP_F16) {
        if (vec) hipLaunchKernelGGL((gated_sum_kernel<f16_t, 4>), grid, dim3(256), 0, st, g);
        else hipLaunchKernelGGL((gated_sum_kernel<f16_t, 1>), grid, dim3(256), 0, st, g);
    } else {
        if (vec) hipLaunchKernelGGL((gated_sum_kernel<bf16_t, 4>), grid, dim3(256), 0, st, g);
        else hipLaunchKernelGGL((gated_sum_kernel<bf16_t, 1>), grid, dim3(256), 0, st, g);
    }
    return check(hipGetLastError(), "gated_sum_kernel launch");
}

template <class K>
int product_go(hipStream_t st, K kern, const GradProduct &o, int lds) {
    if (lds_room(reinterpret_cast<const void *>(kern), lds)) return 1;
    hipLaunchKernelGGL(kern, dim3(unsigned(o.s.tiles_m * o.s.tiles_n), unsigned(o.z), unsigned(o.p.parts)), dim3(256), lds, st,
                       o.shape(), o.a, o.b, o.b2, o.store(), o.p.k_part);
    if (check(hipGetLastError(), "gated backward launch")) return 1;
    return parts_sum(st, o);
}

constexpr int kGradLds256 = gemm_stream_lds_bytes<64, 2>(), kGradLds128 = gemm_stream_lds_bytes<64, 2, 128>(),
              kGradLdsDeep = gemm_stream_lds_bytes<64, 2, 128, 3>();

template <bool F16>
int input_go(hipStream_t st, const GradProduct &o) {
    if (o.p.tm == 256) return product_go(st, gated_input_grad<F16, 256, 0>, o, kGradLds256);
    if (o.p.deep) return product_go(st, gated_input_grad<F16, 128, 3>, o, kGradLdsDeep);
    return product_go(st, gated_input_grad<F16, 128, 2>, o, kGradLds128);
}

template <bool F16>
int weight_go(hipStream_t st, const GradProduct &o) {
    if (o.p.tm == 256) return product_go(st, gated_weight_grad<F16, 256, 0>, o, kGradLds256);
    if (o.p.deep) return product_go(st, gated_weight_grad<F16, 128, 3>, o, kGradLdsDeep);
    return product_go(st, gated_weight_grad<F16, 128, 2>, o, kGradLds128);
}

template <bool F16>
int pair_go(hipStream_t st, const GradProduct &i, const GradProduct &w) {
    auto kern = gated_both_grads<F16>;
    if (lds_room(reinterpret_cast<const void *>(kern), kGradLdsDeep)) return 1;
    const int ti = i.s.tiles_m * i.s.tiles_n, tw = w.s.tiles_m * w.s.tiles_n;
    const dim3 grid(unsigned(ti > tw ? ti : tw), unsigned(w.z + 1), unsigned(i.p.parts > w.p.parts ? i.p.parts : w.p.parts));
    const GatedHalf gi{i.shape(), i.b, i.store(), i.p.k_part, i.p.parts}, gw{w.shape(), w.b, w.store(), w.p.k_part, w.p.parts};
    hipLaunchKernelGGL(kern, grid, dim3(256), kGradLdsDeep, st, gi, gw, i.a, i.b2);
    if (check(hipGetLastError(), "gated_both_grads launch")) return 1;
    return parts_sum(st, i) || parts_sum(st, w);
}

// A result of no terms.
int zero_grad(hipStream_t st, void *out, int64_t elements) { return fill_on(st, out, size_t(elements) * 2, 0); }

}  // namespace

int gated_input_grad_on(hipStream_t st, const nhip_gated_desc *d, const void *dgu, const void *gate, const void *up, void *dx,
                        void *ws) {
    if (backward_check(d, "nhip_gated_input_grad")) return 1;
    if (d->m == 0 || d->k == 0) return 0;
    if (d->n == 0) return zero_grad(st, dx, d->m * d->k);
    GradProduct o;
    if (input_product(st, d, dgu, gate, up, dx, ws, input_grad_plan(d), o)) return 1;
    return d->dtype == NHIP_F16 ? input_go<true>(st, o) : input_go<false>(st, o);
}

int gated_weight_grad_on(hipStream_t st, const nhip_gated_desc *d, const void *dgu, const void *x, void *dgate, void *dup, void *ws) {
    if (backward_check(d, "nhip_gated_weight_grad")) return 1;
    if (d->n == 0 || d->k == 0) return 0;
    if (d->m == 0) return zero_grad(st, dgate, d->n * d->k) || (dup && zero_grad(st, dup, d->n * d->k));
    GradProduct o;
    if (weight_product(st, d, dgu, x, dgate, dup, ws, weight_grad_plan(d), o)) return 1;
    return d->dtype == NHIP_F16 ? weight_go<true>(st, o) : weight_go<false>(st, o);
}

int gated_both_grads_on(hipStream_t st, const nhip_gated_desc *d, const void *dgu, const void *gate, const void *up, const void *x,
                        void *dx, void *dgate, void *dup, void *ws) {
    if (backward_check(d, "nhip_gated_backward")) return 1;
    const GradPlans both = paired_plans(d);
    if (!both.i.tm)
        return gated_weight_grad_on(st, d, dgu, x, dgate, dup, ws) || gated_input_grad_on(st, d, dgu, gate, up, dx, ws);
    GradProduct i, w;
    if (input_product(st, d, dgu, gate, up, dx, ws, both.i, i)) return 1;
    void *rest = ws ? static_cast<char *>(ws) + input_grad_bytes(d, both.i) : nullptr;
    if (weight_product(st, d, dgu, x, dgate, dup, rest, both.w, w)) return 1;
    return d->dtype == NHIP_F16 ? pair_go<true>(st, i, w) : pair_go<false>(st, i, w);
}

// ---- gradient clipping ----------------------------------------------------------------------------------

namespace {

// Launches of at least one table, and the most workgroups one leaves a sum for.
int64_t clip_launches(int64_t count) { return count <= 0 ? 1 : (count + kClipTensors - 1) / kClipTensors; }

}  // namespace

int clip_on(hipStream_t st, const nhip_clip_desc *d, const nhip_clip_tensor *t, const double *max_at, float *norm,
            float *scale, void *ws) {
    if (d->count < 0) return fail("nhip_clip_grad_norm: negative count");
    if (!ws) return fail("nhip_clip_grad_norm: no workspace");
    bool outs = false;
    for (int64_t i = 0; i < d->count; ++i) {
        if (t[i].numel < 0) return fail("nhip_clip_grad_norm: negative element count");
        if (t[i].dtype != NHIP_F32 && t[i].dtype != NHIP_BF16 && t[i].dtype != NHIP_F16)
            return fail("nhip_clip_grad_norm: tensors are float32, bf16 or f16");
        if (t[i].numel > 0 && !t[i].in) return fail("nhip_clip_grad_norm: a tensor without memory");
        outs = outs || (t[i].out && t[i].numel > 0);
    }
    const int64_t launches = clip_launches(d->count);
    double *part = static_cast<double *>(ws);
    int parts = 0;
    for (int pass = 0; pass < 2; ++pass) {
        // the norm alone takes one workgroup of the second pass
        for (int64_t l = 0; l < (pass == 1 && !outs ? 1 : launches); ++l) {
            ClipTable c;
            const int64_t first = l * kClipTensors;
            c.tensors = int(d->count - first < kClipTensors ? d->count - first : kClipTensors);
            int64_t chunks = 0;
            for (int i = 0; i < c.tensors; ++i) {
                const nhip_clip_tensor &x = t[first + i];
                c.in[i] = x.in, c.out[i] = x.out, c.numel[i] = x.numel, c.dtype[i] = uint8_t(x.dtype);
                c.first[i] = uint32_t(chunks);
                chunks += (x.numel + kClipChunk - 1) / kClipChunk;
                if (chunks > 0x7fffffff) return fail("nhip_clip_grad_norm: over 2^45 elements");
            }
            c.first[c.tensors] = uint32_t(chunks);
            if (pass == 0) {
                c.blocks = uint32_t(chunks < kClipBlocks ? (chunks ? chunks : 1) : kClipBlocks);
                hipLaunchKernelGGL(clip_squares_kernel, dim3(c.blocks), dim3(256), 0, st, c, part + parts);
                if (check(hipGetLastError(), "clip_squares_kernel launch")) return 1;
                parts += int(c.blocks);
            } else {
                c.blocks = uint32_t(!outs || chunks == 0 ? 1 : chunks < 2 * kClipBlocks ? chunks : 2 * kClipBlocks);
                if (!outs) c.first[c.tensors] = 0;
                hipLaunchKernelGGL(clip_scale_kernel, dim3(c.blocks), dim3(256), 0, st, c, part, parts, max_at, d->max_norm,
                                   d->eps, l == 0 ? norm : nullptr, l == 0 ? scale : nullptr);
                if (check(hipGetLastError(), "clip_scale_kernel launch")) return 1;
            }
        }
    }
    return 0;
}

}  // namespace nhip

using namespace nhip;

extern "C" {

#define NHIP_STREAM(st)                    \
    hipStream_t st = stream_of_current(); \
    if (!st) return fail("no HIP stream: call nhip_set_device first")

int nhip_qk_norm_rope(const nhip_heads_desc *desc, const void *q, const void *k, const void *q_weight, const void *k_weight,
                      const float *cos, const float *sin, const void *positions, void *q_out, void *k_out) {
    NHIP_STREAM(st);
    return heads_on(st, desc, q, k, q_weight, k_weight, cos, sin, positions, q_out, k_out);
}

int nhip_qk_norm_rope_bwd(const nhip_heads_desc *desc, const void *q, const void *k, const void *q_weight,
                          const void *k_weight, const float *cos, const float *sin, const void *positions,
                          const void *d_q_out, const void *d_k_out, void *dq, void *dk, void *d_q_weight, void *d_k_weight,
                          void *workspace) {
    NHIP_STREAM(st);
    return heads_bwd_on(st, desc, q, k, q_weight, k_weight, cos, sin, positions, d_q_out, d_k_out, dq, dk, d_q_weight,
                        d_k_weight, workspace);
}

int nhip_qk_norm_rope_workspace(const nhip_heads_desc *desc, size_t *bytes) {
    if (heads_check(desc, "nhip_qk_norm_rope_workspace")) return 1;
    *bytes = heads_workspace(desc);
    return 0;
}

int nhip_gated_linear(const nhip_gated_desc *desc, const void *x, const void *gate, const void *up, void *h, float *g, float *u,
                      void *workspace) {
    NHIP_STREAM(st);
    return gated_on(st, desc, x, gate, up, h, g, u, workspace);
}

int nhip_gated_linear_workspace(const nhip_gated_desc *desc, size_t *bytes) {
    if (gated_check(desc, "nhip_gated_linear_workspace")) return 1;
    if (!gated_skinny_ok(desc) && !gated_stream_ok(desc)) return fail("nhip_gated_linear_workspace: 1 to 2^21 - 1 elements a row");
    if (!gated_launch_ok(desc, desc->config < 0 ? gated_default(desc) : desc->config))
        return fail("nhip_gated_linear_workspace: a launch of 2^32 threads");
    *bytes = gated_workspace(desc);
    return 0;
}

int nhip_gated_input_grad(const nhip_gated_desc *desc, const void *dgu, const void *gate, const void *up, void *dx,
                          void *workspace) {
    NHIP_STREAM(st);
    return gated_input_grad_on(st, desc, dgu, gate, up, dx, workspace);
}

int nhip_gated_weight_grad(const nhip_gated_desc *desc, const void *dgu, const void *x, void *d_gate, void *d_up, void *workspace) {
    NHIP_STREAM(st);
    return gated_weight_grad_on(st, desc, dgu, x, d_gate, d_up, workspace);
}

int nhip_gated_backward(const nhip_gated_desc *desc, const void *dgu, const void *gate, const void *up, const void *x, void *dx,
                        void *d_gate, void *d_up, void *workspace) {
    NHIP_STREAM(st);
    return gated_both_grads_on(st, desc, dgu, gate, up, x, dx, d_gate, d_up, workspace);
}

int nhip_gated_backward_paired(const nhip_gated_desc *desc, int *paired) {
    if (backward_check(desc, "nhip_gated_backward_paired")) return 1;
    *paired = paired_plans(desc).i.tm != 0;
    return 0;
}

int nhip_gated_backward_workspace(const nhip_gated_desc *desc, size_t *bytes) {
    if (backward_check(desc, "nhip_gated_backward_workspace")) return 1;
    *bytes = backward_workspace(desc);
    return 0;
}

int nhip_gated_config_count(int *count) {
    *count = kGatedConfigs;
    return 0;
}

int nhip_gated_linear_grad(const nhip_gated_desc *desc, const void *dh, const float *g, const float *u, void *dgu) {
    NHIP_STREAM(st);
    return gated_grad_on(st, desc, dh, g, u, dgu);
}

int nhip_clip_grad_norm(const nhip_clip_desc *desc, const nhip_clip_tensor *tensors, const double *max_norm_at, float *norm,
                        float *scale, void *workspace) {
    NHIP_STREAM(st);
    return clip_on(st, desc, tensors, max_norm_at, norm, scale, workspace);
}

int nhip_clip_grad_norm_workspace(const nhip_clip_desc *desc, size_t *bytes) {
    if (desc->count < 0) return fail("nhip_clip_grad_norm_workspace: negative count");
    *bytes = size_t(clip_launches(desc->count)) * kClipBlocks * sizeof(double);
    return 0;
}

}  // extern "C"

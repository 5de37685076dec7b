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

constexpr int64_t kHeadsLaunchRows = int64_t(1) << 30;  // heads of a launch: row arithmetic is 32-bit
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
    int64_t most = d->heads > d->kv_heads ? d->heads : d->kv_heads;
    most = kHeadsLaunchRows / (most > 0 ? most : 1);
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
    for (int e : {8, 4}) {
        if (e == 8 && d->dtype == NHIP_F32) continue;  // 4 elements are 16 bytes
        const size_t bytes = size_t(e) * (d->dtype == NHIP_F32 ? 4 : 2);
        bool ok = d->head_dim % (2 * e) == 0 && d->rot % (2 * e) == 0 && d->head_dim / (2 * e) <= 64 && heads_strides(d, e, bwd);
        for (const void *h : heads) ok = ok && on(h, bytes);
        ok = ok && on(cos, 16) && on(sin, 16);
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
        const int64_t want = need / 4 > part ? need / 4 : (need < part ? need : part), most = cap * rows / (q + k) + 1;
        return want < most ? want : most;
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

enum { kSkinnyCfg = 0, kStream256, kStream128Cfg, kGatedConfigs };

int gated_check(const nhip_gated_desc *d, const char *what) {
    const std::string at(what);
    if (d->m < 0 || d->n < 0 || d->k < 0) return fail(at + ": negative sizes");
    if (d->dtype != NHIP_BF16 && d->dtype != NHIP_F16) return fail(at + ": bf16 or f16");
    if (d->activation < NHIP_ACT_SILU || d->activation > NHIP_ACT_SIGMOID) return fail(at + ": unknown activation");
    return 0;
}

int64_t tiles(int64_t m, int64_t bm, int64_t n, int64_t bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }

bool gated_skinny_ok(const nhip_gated_desc *d) { return d->m <= 64 && d->k < (int64_t(1) << 30); }

int gated_default(const nhip_gated_desc *d) {
    if (gated_skinny_ok(d)) return kSkinnyCfg;
    return tiles(d->m, 256, d->n, 128) >= 256 ? kStream256 : kStream128Cfg;
}

// Whether gated_stream can read rows of these lengths and distances in place (from 16-byte addresses).
bool gated_rows(const nhip_gated_desc *d) {
    return d->k % 8 == 0 && d->x_m % 8 == 0 && d->w_n % 8 == 0 &&
           stream_buffer_ok(d->m, d->n, d->k, false, false, d->x_m, 1, 1, d->w_n);
}

size_t gated_workspace(const nhip_gated_desc *d) {
    const int cfg = d->config < 0 ? gated_default(d) : d->config;
    if (cfg == kSkinnyCfg || gated_rows(d)) return 0;
    return size_t(d->m + 2 * d->n) * size_t((d->k + 7) / 8 * 8) * 2;
}

template <class K>
int gated_go(hipStream_t st, K kern, GemmShape s, int bm, int bn, int threads, int lds, const void *x, const void *gate,
             const void *up, const GatedOut &out) {
    s.tiles_m = int((s.m + bm - 1) / bm);
    s.tiles_n = int((s.n + bn - 1) / bn);
    if ((s.m + bm - 1) / bm * ((s.n + bn - 1) / bn) > 0x7fffffff) return fail("nhip_gated_linear: too many tiles");
    if (lds > 64 * 1024 &&
        check(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
              "hipFuncSetAttribute"))
        return 1;
    hipLaunchKernelGGL(kern, dim3(unsigned(s.tiles_m * s.tiles_n)), dim3(threads), lds, st, s, static_cast<const uint16_t *>(x),
                       static_cast<const uint16_t *>(gate), static_cast<const uint16_t *>(up), out);
    return check(hipGetLastError(), "gated kernel launch");
}

template <bool F16, bool ANY>
int gated_few(hipStream_t st, const GemmShape &s, const void *x, const void *gate, const void *up, const GatedOut &o) {
    if (s.m <= 16) return gated_go(st, gated_skinny<F16, 1, 8, ANY>, s, 64, 16, 512, 0, x, gate, up, o);
    if (s.m <= 32) return gated_go(st, gated_skinny<F16, 2, 8, ANY>, s, 64, 16, 512, 0, x, gate, up, o);
    return gated_go(st, gated_skinny<F16, 4, 4, ANY>, s, 64, 16, 256, 0, x, gate, up, o);
}

template <bool F16>
int gated_run(hipStream_t st, int cfg, GemmShape s, const void *x, const void *gate, const void *up, const GatedOut &o, bool in_place,
              void *ws) {
    if (cfg == kSkinnyCfg) return in_place ? gated_few<F16, false>(st, s, x, gate, up, o) : gated_few<F16, true>(st, s, x, gate, up, o);
    if (!in_place) {
        GatedPad p;
        p.k = s.k, p.kp = (s.k + 7) / 8 * 8;
        const void *src[3] = {x, gate, up};
        uint16_t *to = static_cast<uint16_t *>(ws);
        for (int i = 0; i < 3; ++i) {
            p.src[i] = static_cast<const uint16_t *>(src[i]);
            p.rows[i] = i ? s.n : s.m, p.ld[i] = i ? s.b_n : s.a_m;
            p.dst[i] = to;
            to += p.rows[i] * p.kp;
        }
        const int64_t blocks = ((s.m > s.n ? s.m : s.n) * (p.kp / 8) + 255) / 256;
        hipLaunchKernelGGL(gated_pad_kernel, dim3(unsigned(blocks < 4096 ? (blocks ? blocks : 1) : 4096)), dim3(256), 0, st, p);
        if (check(hipGetLastError(), "gated_pad_kernel launch")) return 1;
        x = p.dst[0], gate = p.dst[1], up = p.dst[2];
        s.k = s.a_m = s.b_n = p.kp;
    }
    if (cfg == kStream256)
        return gated_go(st, gated_stream<F16, 256>, s, 256, 128, 512, gemm_stream_lds_bytes<64, 4>(), x, gate, up, o);
    return gated_go(st, gated_stream<F16, 128>, s, 128, 64, 256, gemm_stream_lds_bytes<64, 2, 128>(), x, gate, up, o);
}

}  // namespace

int gated_on(hipStream_t st, const nhip_gated_desc *d, const void *x, const void *gate, const void *up, void *h, float *g,
             float *u, void *ws) {
    if (gated_check(d, "nhip_gated_linear")) return 1;
    if (!g != !u) return fail("nhip_gated_linear: g and u go together");
    if (d->m == 0 || d->n == 0) return 0;
    int cfg = d->config < 0 ? gated_default(d) : d->config;
    if (cfg >= kGatedConfigs || (cfg == kSkinnyCfg && !gated_skinny_ok(d)))
        return fail("nhip_gated_linear: config " + std::to_string(cfg) + " does not take these operands");
    GemmShape s;
    std::memset(&s, 0, sizeof(s));
    s.m = d->m, s.n = d->n, s.k = d->k;
    s.a_m = d->x_m, s.a_k = 1, s.b_k = 1, s.b_n = d->w_n, s.d_m = d->h_m, s.d_n = 1;
    const bool rows = cfg == kSkinnyCfg ? d->k % 8 == 0 && d->x_m % 8 == 0 && d->w_n % 8 == 0 : gated_rows(d);
    const bool in_place = rows && on(x, 16) && on(gate, 16) && on(up, 16);
    if (!in_place && cfg != kSkinnyCfg) {
        if (rows) return fail("nhip_gated_linear: operands of such rows start on 16 bytes");
        if (!ws || !on(ws, 16)) return fail("nhip_gated_linear: no workspace, or one off 16 bytes");
    }
    const GatedOut o{h, g, u, d->activation, d->dtype};
    return d->dtype == NHIP_F16 ? gated_run<true>(st, cfg, s, x, gate, up, o, in_place, ws)
                                : gated_run<false>(st, cfg, s, x, gate, up, o, in_place, ws);
}

int gated_grad_on(hipStream_t st, const nhip_gated_desc *d, const void *dh, const float *g, const float *u, void *dgu) {
    if (gated_check(d, "nhip_gated_linear_grad")) return 1;
    if (d->m == 0 || d->n == 0) return 0;
    GatedGrad a{dh, g, u, dgu, d->m, d->n, d->h_m, d->activation};
    const bool vec = d->n % 8 == 0 && d->h_m % 8 == 0 && on(dh, 16) && on(g, 16) && on(u, 16) && on(dgu, 16);
    const int64_t work = d->m * (vec ? d->n / 8 : d->n), blocks = (work + 255) / 256;
    const dim3 grid(unsigned(blocks < 8192 ? blocks : 8192));
    if (d->dtype == NHIP_F16) {
        if (vec) hipLaunchKernelGGL((gated_grad_kernel<f16_t, 8>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((gated_grad_kernel<f16_t, 1>), grid, dim3(256), 0, st, a);
    } else {
        if (vec) hipLaunchKernelGGL((gated_grad_kernel<bf16_t, 8>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((gated_grad_kernel<bf16_t, 1>), grid, dim3(256), 0, st, a);
    }
    return check(hipGetLastError(), "gated_grad_kernel launch");
}

namespace {

// The tile and the parts of a pair's k: as many parts as make the tiles' rounds on the chip the shortest, each round as
// long as its k, the parts' writing and reading added. The rates are the split dots' (Plan._split_us), whose loops these are.
struct PairPlan {
    int tm, splits, k_part;
};
PairPlan pair_plan(const nhip_gemm_desc *d) {
    const int half = int((d->k / 2 + 63) / 64), total = 2 * half;
    PairPlan best{128, 1, total};
    double least = 0;
    for (int tm : {256, 128})
        for (int s : {1, 2, 4, 8}) {
            if (s > 1 && (total / s < 8 || int64_t(s) * d->m * d->n * 4 > (int64_t(64) << 20))) continue;
            const int part = (total + s - 1) / s, parts = (total + part - 1) / part;
            const double t = double(tiles(d->m, tm, d->n, tm)) * parts;
            // 256: a workgroup a CU; 128: two, one alone taking 0.79 of a round of both
            double rounds = tm == 256 ? double((int64_t(t) + 255) / 256) : double(int64_t(t) / 512);
            const int64_t rest = int64_t(t) % 512;
            if (tm == 128) rounds += rest == 0 ? 0.0 : rest <= 256 ? 0.79 : 1.0;
            const double us = 6.2 + 64.0 * part * (tm == 256 ? 0.02355 : 0.0142) * rounds +
                              (parts > 1 ? 4.2 + 8.0 * parts * double(d->m) * double(d->n) / 6.13e6 : 0.0);
            if (least == 0 || us < least) least = us, best = PairPlan{tm, parts, part};
        }
    return best;
}

size_t pair_workspace(const nhip_gemm_desc *d) {
    const PairPlan p = pair_plan(d);
    return p.splits > 1 ? size_t(p.splits) * size_t(d->m) * size_t(d->n) * 4 : 0;
}

int pair_check(const nhip_gemm_desc *d) {
    if (d->m < 0 || d->n < 0 || d->k < 0) return fail("nhip_gemm_pair: negative sizes");
    if (d->a_dtype != d->b_dtype || (d->a_dtype != NHIP_BF16 && d->a_dtype != NHIP_F16)) return fail("nhip_gemm_pair: bf16 or f16");
    if (d->nbatch || d->a_k != 1 || d->b_n != 1 || d->k % 16 || d->n % 8 || d->a_m % 8 || d->b_k % 8 || d->a_m < d->k || d->b_k < d->n)
        return fail("nhip_gemm_pair: no batches, A along k and B along n in whole rows, both halves of k and n multiples of 8");
    const int64_t lim = int64_t(1) << 31;
    if ((255 * d->a_m + d->k) * 2 >= lim || (d->k / 2 * d->b_k + 256) * 2 >= lim || d->k >= lim)
        return fail("nhip_gemm_pair: an operand's tile spans 2^31 bytes");
    return 0;
}

template <bool F16, int TM>
int pair_go(hipStream_t st, GemmShape s, const PairPlan &p, const void *a, const void *b, const void *b2, const AnyStore &out) {
    s.tiles_m = int((s.m + TM - 1) / TM);
    s.tiles_n = int((s.n + TM - 1) / TM);
    if (tiles(s.m, TM, s.n, TM) > 0x7fffffff) return fail("nhip_gemm_pair: too many tiles");
    constexpr int lds = gemm_stream_lds_bytes<64, 2, TM>();
    auto kern = gemm_pair<F16, TM>;
    if (check(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
              "hipFuncSetAttribute"))
        return 1;
    hipLaunchKernelGGL(kern, dim3(unsigned(s.tiles_m * s.tiles_n), 1, unsigned(p.splits)), dim3(256), lds, st, s,
                       static_cast<const uint16_t *>(a), static_cast<const uint16_t *>(b), static_cast<const uint16_t *>(b2), out,
                       p.k_part);
    return check(hipGetLastError(), "gemm_pair launch");
}

}  // namespace

int pair_on(hipStream_t st, const nhip_gemm_desc *d, const void *a, const void *b, const void *b2, void *out, void *ws) {
    if (pair_check(d)) return 1;
    if (d->m == 0 || d->n == 0) return 0;
    if (!on(a, 16) || !on(b, 16) || !on(b2, 16)) return fail("nhip_gemm_pair: operands start on 16 bytes");
    GemmShape s;
    std::memset(&s, 0, sizeof(s));
    s.m = d->m, s.n = d->n, s.k = d->k;
    s.a_m = d->a_m, s.a_k = 1, s.b_k = d->b_k, s.b_n = 1;
    s.d_m = d->d_m, s.d_n = d->d_n;
    const AnyStore to{out, d->d_dtype};
    if (d->k == 0) {  // a sum of nothing
        hipLaunchKernelGGL(gemm_splitk_reduce, dim3(1024), dim3(256), 0, st, s, nullptr, 0, d->m * d->n, to);
        return check(hipGetLastError(), "gemm_splitk_reduce launch");
    }
    const PairPlan p = pair_plan(d);
    GemmShape parts = s;
    AnyStore first = to;
    if (p.splits > 1) {
        if (!ws) return fail("nhip_gemm_pair: no workspace");
        parts.d_m = d->n, parts.d_n = 1, parts.d_split = d->m * d->n;
        first = AnyStore{ws, 0};
    }
    const int rc = d->a_dtype == NHIP_F16
                       ? (p.tm == 256 ? pair_go<true, 256>(st, parts, p, a, b, b2, first) : pair_go<true, 128>(st, parts, p, a, b, b2, first))
                       : (p.tm == 256 ? pair_go<false, 256>(st, parts, p, a, b, b2, first) : pair_go<false, 128>(st, parts, p, a, b, b2, first));
    if (rc || p.splits == 1) return rc;
    const int64_t total = d->m * d->n, blocks = (total + 255) / 256;
    hipLaunchKernelGGL(gemm_splitk_reduce, dim3(unsigned(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, s,
                       static_cast<const float *>(ws), p.splits, total, to);
    return check(hipGetLastError(), "gemm_splitk_reduce launch");
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
    *bytes = gated_workspace(desc);
    return 0;
}

int nhip_gemm_pair(const nhip_gemm_desc *desc, const void *a, const void *b, const void *b2, void *d, void *workspace) {
    NHIP_STREAM(st);
    return pair_on(st, desc, a, b, b2, d, workspace);
}

int nhip_gemm_pair_workspace(const nhip_gemm_desc *desc, size_t *bytes) {
    if (pair_check(desc)) return 1;
    *bytes = pair_workspace(desc);
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

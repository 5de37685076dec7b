// C entry points of the cross entropy of a vocabulary head with its gradients (head.h).
#include <algorithm>
#include <cstring>
#include <string>
#include <type_traits>

#include "head.h"
#include "nhip_internal.h"
#include "parts.h"

using namespace nhip;
using namespace nhipk;

namespace nhip {
namespace {

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

int64_t blocks_of(const nhip_head_desc *d) { return (d->classes + 63) / 64; }
int64_t padded_k(const nhip_head_desc *d) { return up(d->k, 64); }

// Rows of a piece: what fits the bytes that the desc allows for its codes, a multiple of 256 (a tile's), and pieces of one size.
int64_t piece_rows(const nhip_head_desc *d) {
    const int64_t row = blocks_of(d) * 64 * 2;
    // the weight gradient reads a piece's codes, and its rows of h, through a buffer of 2^31 bytes each
    const int64_t buffer = (int64_t(1) << 31) - (int64_t(1) << 20);
    const int64_t fit = std::min(std::min(d->piece_bytes, buffer) / row, buffer / (padded_k(d) * 2));
    const int64_t most = std::max<int64_t>(fit / 256 * 256, 256);
    if (d->rows <= most) return d->rows;
    const int64_t pieces = (d->rows + most - 1) / most;
    return std::min(most, up((d->rows + pieces - 1) / pieces, 256));
}
// Rows of a piece of the losses alone: those whose blocks' maxima and sums fit the same bytes, a sixteenth of their codes.
int64_t loss_rows(const nhip_head_desc *d) {
    const int64_t fit = d->piece_bytes / (blocks_of(d) * int64_t(sizeof(float2)));
    return std::min(std::max<int64_t>(fit / 256 * 256, 256), d->rows);
}
int64_t pieces_of(const nhip_head_desc *d) { return d->rows > 0 ? (d->rows + piece_rows(d) - 1) / piece_rows(d) : 0; }

PartPlan input_plan(const nhip_head_desc *d) {
    return part_plan(piece_rows(d), d->k, 1, (d->classes + 63) / 64, int64_t(1) << 30);
}
PartPlan weight_plan(const nhip_head_desc *d) {
    const int64_t total = (piece_rows(d) + 63) / 64;
    PartPlan p = part_plan(d->classes, d->k, 1, total, int64_t(1) << 30);
    // few k tiles: the store is most of a tile, and two workgroups a CU hide one another's. Us with tiles of 256 rows and 128 (*
    // taken), of rows, k, classes: 128, 2048, 32000 114 76*; 271, 2560, 31856 170 126*; 512, 512, 32000 42 33*; 1024, 1024, 32000
    // 108 103*; 1536, 2048, 32000 262* 274; 2048, 512, 32000 82* 87; 4096, 512, 32000 135* 173
    if (p.tm == 256 && p.parts == 1 && total <= 16) p = PartPlan{128, 1, int(total), false, p.us};
    // the pieces' sums are added in the store, which parts do without
    if (pieces_of(d) > 1 && p.parts > 1) p = PartPlan{256, 1, int(total), false, 0.0};
    return p;
}

// Both products in one launch of at most two workgroups of 128-row tiles a CU, dh's in parts: parts 0 where one after the other is
// estimated shorter, by part_plan's rates for a launch of so many workgroups. Us with the parts' sums, one after the other and
// together (* taken), of rows, k, classes:
//   777, 520, 5003    40  31*      200, 1024, 5000  32  23*      128, 768, 8192   33  24*      900, 256, 8000   39  28*
//   1500, 300, 3000   40  34*      64, 256, 1000    23  17*      1024, 512, 2048  33  28*      2000, 72, 63     23* 31
struct BothPlan {
    int parts, k_part;
};
BothPlan both_plan(const nhip_head_desc *d) {
    if (pieces_of(d) != 1) return BothPlan{0, 0};
    const int64_t input = blocks_of(d), weight = (d->rows + 63) / 64;
    const int64_t ti = tiles(d->rows, 128, d->k, 128), tw = tiles(d->classes, 128, d->k, 128);
    BothPlan best{0, 0};
    double least = input_plan(d).us + weight_plan(d).us;
    for (int64_t s = 1; s <= 16; ++s) {
        const int64_t part = (input + s - 1) / s, parts = (input + part - 1) / part, t = ti * parts + tw;
        if (t > 512) break;
        const double us = 6.2 + 64.0 * double(std::max(part, weight)) * 0.0142 * (t <= 256 ? 0.79 : 1.0) + parts_us(d->rows * d->k, parts);
        if (us < least) least = us, best = BothPlan{int(parts), int(part)};
    }
    return best;
}

// Whether rows are copied first: no whole k tiles, or not on 16 bytes. The gradients always read a copy of h (head_copy).
bool copies(const nhip_head_desc *d, int64_t ld) { return d->k % 64 != 0 || ld % 8 != 0; }

struct HeadSpace {
    size_t h, w, part, picked, scale, codes, weight_sums, input_parts, weight_parts, bytes;
};
HeadSpace head_space(const nhip_head_desc *d, bool grad) {
    HeadSpace s{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t from = at;
        at += up256(bytes);
        return from;
    };
    const int64_t kp = padded_k(d), rows = grad ? piece_rows(d) : loss_rows(d);
    s.h = take(grad || copies(d, d->h_m) ? size_t(d->rows) * kp * 2 : 0);
    s.w = take(copies(d, d->w_n) ? size_t(d->classes) * kp * 2 : 0);
    s.part = take(size_t(rows) * blocks_of(d) * sizeof(float2));
    s.picked = take(size_t(rows) * 4);
    s.scale = take(8);
    if (grad) {
        const PartPlan pi = input_plan(d), pw = weight_plan(d);
        const BothPlan both = both_plan(d);
        auto parts_bytes = [](int64_t parts, int64_t elements) { return parts > 1 ? size_t(parts) * size_t(elements) * 4 : 0; };
        s.codes = take(size_t(rows) * blocks_of(d) * 64 * 2);
        s.weight_sums = take(pieces_of(d) > 1 ? size_t(d->classes) * d->k * 4 : 0);
        // the parts of one product at a time
        s.input_parts = s.weight_parts =
            take(std::max({parts_bytes(both.parts, rows * d->k), parts_bytes(pi.parts, rows * d->k), parts_bytes(pw.parts, d->classes * d->k)}));
    }
    s.bytes = at;
    return s;
}

int head_check(const nhip_head_desc *d, const char *what) {
    const std::string at(what);
    if (d->rows < 0 || d->classes < 1 || d->k < 1) return fail(at + ": needs rows >= 0, classes >= 1 and k >= 1");
    if (d->dtype != NHIP_BF16 && d->dtype != NHIP_F16) return fail(at + ": bf16 or f16 operands only");
    if (d->target_dtype != NHIP_LCE_I32 && d->target_dtype != NHIP_LCE_I64) return fail(at + ": targets must be int32 or int64");
    if (d->h_m < 0 || d->w_n < d->k) return fail(at + ": rows that lie backwards, or classes that overlap");
    const int64_t lim = (int64_t(1) << 30) - 1024, kp = padded_k(d);
    if (kp >= int64_t(1) << 20 || d->classes >= int64_t(1) << 22 || (d->classes + 256) * std::max(kp, d->w_n) >= lim)
        return fail(at + ": rows below 2^20 elements, 2^22 classes, and a weight within 2^31 bytes");
    if (d->h_m >= int64_t(1) << 40 || (!copies(d, d->h_m) && 256 * d->h_m + kp >= lim))
        return fail(at + ": a tile's rows of h within 2^31 bytes");
    if (d->rows >= int64_t(1) << 26 || tiles(d->rows, 128, d->classes, 128) >= int64_t(1) << 24 ||
        tiles(d->classes, 128, d->k, 128) >= int64_t(1) << 24 || tiles(d->rows, 128, d->k, 128) >= int64_t(1) << 24)
        return fail(at + ": a launch of 2^32 threads");
    if (d->piece_bytes < 0) return fail(at + ": negative sizes");
    if (256 * blocks_of(d) * 64 * 2 >= int64_t(1) << 31) return fail(at + ": a tile's rows of classes within 2^31 bytes");
    return 0;
}

template <int THREADS = 256, class... P>
int launch(hipStream_t st, void (*kern)(P...), dim3 grid, int lds, const char *what, std::common_type_t<P>... args) {
    if (check(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
              "hipFuncSetAttribute"))
        return 1;
    hipLaunchKernelGGL(kern, grid, dim3(THREADS), lds, st, args...);
    return check(hipGetLastError(), what);
}

constexpr int kLds256 = gemm_stream_lds_bytes<64, 2>(), kLds128 = gemm_stream_lds_bytes<64, 2, 128>(),
              kLdsDeep = gemm_stream_lds_bytes<64, 2, 128, 3>();

GemmShape shape(int64_t m, int64_t n, int64_t k, int tm) {
    GemmShape s;
    std::memset(&s, 0, sizeof(s));
    s.m = m, s.n = n, s.k = k, s.d_m = n, s.d_n = 1;
    s.tiles_m = int((m + tm - 1) / tm), s.tiles_n = int((n + tm - 1) / tm);
    return s;
}

template <bool F16, bool GRAD>
int logits(hipStream_t st, const nhip_head_desc *d, int64_t rows, const uint16_t *h, int64_t h_m, const uint16_t *w, int64_t w_n,
           const HeadOut<GRAD> &out) {
    // 256-row tiles where they fill the CUs
    const int tm = tiles(rows, 256, d->classes, 256) >= 256 ? 256 : 128;
    GemmShape s = shape(rows, d->classes, padded_k(d), tm);
    s.a_m = h_m, s.a_k = 1, s.b_k = 1, s.b_n = w_n;
    const dim3 grid(unsigned(s.tiles_m) * unsigned(s.tiles_n));
    if (tm == 256)
        return launch<512>(st, head_logits_kernel<F16, 256, GRAD>, grid, gemm_stream_lds_bytes<64, 4>(), "head_logits_kernel launch", s, h,
                           w, out);
    return launch(st, head_logits_kernel<F16, 128, GRAD>, grid, kLds128, "head_logits_kernel launch", s, h, w, out);
}

int parts_sum(hipStream_t st, const float *part, const PartPlan &p, int64_t mn, const HeadStore &to) {
    const int64_t blocks = (mn + 1023) / 1024;
    hipLaunchKernelGGL(head_sum_kernel, dim3(unsigned(std::min<int64_t>(blocks, 4096))), dim3(256), 0, st, part, p.parts, mn, to);
    return check(hipGetLastError(), "head_sum_kernel launch");
}

// One of the gradients' products, whole into `to` or in parts through `part`.
#define NHIP_HEAD_PRODUCT(KERN, WHAT)                                                                                        \
    const dim3 grid(unsigned(s.tiles_m) * unsigned(s.tiles_n), 1, unsigned(p.parts));                                         \
    if (p.parts == 1) {                                                                                                       \
        if (p.tm == 256) return launch(st, KERN<F16, 256, 0, HeadStore>, grid, kLds256, WHAT, s, a, b, to, p.k_part);           \
        if (p.deep) return launch(st, KERN<F16, 128, 3, HeadStore>, grid, kLdsDeep, WHAT, s, a, b, to, p.k_part);              \
        return launch(st, KERN<F16, 128, 2, HeadStore>, grid, kLds128, WHAT, s, a, b, to, p.k_part);                           \
    }                                                                                                                         \
    s.d_split = s.m * s.n;                                                                                                    \
    const AnyStore sums{part, 0};                                                                                             \
    if (p.tm == 256 ? launch(st, KERN<F16, 256, 0, AnyStore>, grid, kLds256, WHAT, s, a, b, sums, p.k_part)                    \
        : p.deep    ? launch(st, KERN<F16, 128, 3, AnyStore>, grid, kLdsDeep, WHAT, s, a, b, sums, p.k_part)                   \
                    : launch(st, KERN<F16, 128, 2, AnyStore>, grid, kLds128, WHAT, s, a, b, sums, p.k_part))                   \
        return 1;                                                                                                             \
    return parts_sum(st, part, p, s.m * s.n, to)

template <bool F16>
int input_grad(hipStream_t st, const nhip_head_desc *d, const PartPlan &p, int64_t rows, const uint16_t *a, const uint16_t *b, int64_t w_n,
               float *part, const HeadStore &to) {
    GemmShape s = shape(rows, d->k, d->classes, p.tm);
    s.a_m = blocks_of(d) * 64, s.a_k = 1, s.b_k = w_n, s.b_n = 1;
    NHIP_HEAD_PRODUCT(head_input_grad, "head_input_grad launch");
}

template <bool F16>
int weight_grad(hipStream_t st, const nhip_head_desc *d, const PartPlan &p, int64_t rows, const uint16_t *a, const uint16_t *b, int64_t h_m,
                float *part, const HeadStore &to) {
    GemmShape s = shape(d->classes, d->k, rows, p.tm);
    s.a_m = 1, s.a_k = blocks_of(d) * 64, s.b_k = h_m, s.b_n = 1;
    NHIP_HEAD_PRODUCT(head_weight_grad, "head_weight_grad launch");
}
#undef NHIP_HEAD_PRODUCT

template <bool F16, class InOut>
int both_go(hipStream_t st, const HeadBoth<InOut> &x, const uint16_t *d) {
    const int ti = x.input.tiles_m * x.input.tiles_n, tw = x.weight.tiles_m * x.weight.tiles_n;
    return launch(st, head_both_grads<F16, InOut>, dim3(unsigned(ti * x.parts + tw)), kLds128, "head_both_grads launch", x, d);
}

// input_grad and weight_grad of the only piece.
template <bool F16>
int both_grads(hipStream_t st, const nhip_head_desc *d, const BothPlan &p, const uint16_t *codes, const uint16_t *w, int64_t w_n,
               const uint16_t *h, int64_t h_m, float *part, const HeadStore &dh, const HeadStore &dw) {
    GemmShape i = shape(d->rows, d->k, d->classes, 128), s = shape(d->classes, d->k, d->rows, 128);
    i.a_m = blocks_of(d) * 64, i.a_k = 1, i.b_k = w_n, i.b_n = 1;
    s.a_m = 1, s.a_k = blocks_of(d) * 64, s.b_k = h_m, s.b_n = 1;
    const int all = int((d->rows + 63) / 64);
    if (p.parts == 1) return both_go<F16>(st, HeadBoth<HeadStore>{i, s, w, h, dh, dw, 1, p.k_part, all}, codes);
    i.d_split = i.m * i.n;
    if (both_go<F16>(st, HeadBoth<AnyStore>{i, s, w, h, AnyStore{part, 0}, dw, p.parts, p.k_part, all}, codes)) return 1;
    return parts_sum(st, part, PartPlan{128, p.parts, p.k_part, false, 0.0}, i.m * i.n, dh);
}

// The losses alone of h's rows where the products read them, as many rows at a time as the workspace holds maxima and sums of.
template <bool F16>
int losses_alone(hipStream_t st, const nhip_head_desc *d, int64_t most, const uint16_t *h, int64_t h_m, const uint16_t *w, int64_t w_n,
                 HeadTargets targets, float2 *part, float *picked, float *losses) {
    const int64_t blocks = blocks_of(d), tsize = targets.t64 ? 8 : 4;
    const char *target = static_cast<const char *>(targets.target);
    for (int64_t r0 = 0; r0 < d->rows; r0 += most) {
        const int64_t rows = std::min(most, d->rows - r0);
        targets.target = target + r0 * tsize;
        const HeadOut<false> out{part, picked, nullptr, targets, blocks};
        if (logits<F16, false>(st, d, rows, h + r0 * h_m, h_m, w, w_n, out)) return 1;
        hipLaunchKernelGGL(head_merge_kernel, dim3(unsigned(std::min<int64_t>(rows, 1 << 20))), dim3(256), 0, st, part, picked, targets, rows,
                           blocks, losses + r0);
        if (check(hipGetLastError(), "head_merge_kernel launch")) return 1;
    }
    return 0;
}

bool on(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A copy of `rows` rows at `dst`, by as many workgroups as it fills.
HeadCopy copy_of(const uint16_t *src, int64_t rows, int64_t ld, int64_t k, int64_t kp, char *dst, bool mask) {
    const int64_t groups = (rows * (kp / 8) + kPrepare - 1) / kPrepare;
    return HeadCopy{src, rows, ld, k, kp, reinterpret_cast<uint16_t *>(dst), mask, int32_t(std::min<int64_t>(groups, 2048))};
}

template <bool F16>
int head_run(hipStream_t st, const nhip_head_desc *d, const uint16_t *h, const uint16_t *w, const void *target, const float *g,
             float *losses, uint16_t *dh, uint16_t *dw, char *ws) {
    // the workspace is laid out by whether there are cotangents, as its size is asked for, also where neither gradient is wanted
    const HeadSpace at = head_space(d, g != nullptr);
    const bool grad = dh || dw;
    const int64_t most = g ? piece_rows(d) : loss_rows(d);
    if (!grad) g = nullptr;
    const int64_t kp = padded_k(d), blocks = blocks_of(d), tsize = d->target_dtype == NHIP_LCE_I64 ? 8 : 4;
    int64_t h_m = d->h_m, w_n = d->w_n;
    HeadTargets targets{target, d->ignore_index, d->classes, d->target_dtype == NHIP_LCE_I64};
    HeadCopy hc{}, wc{};
    if (grad || copies(d, h_m)) {
        hc = copy_of(h, d->rows, h_m, d->k, kp, ws + at.h, grad);
        h = hc.dst, h_m = kp;
    }
    if (copies(d, w_n)) {
        wc = copy_of(w, d->classes, w_n, d->k, kp, ws + at.w, false);
        w = wc.dst, w_n = kp;
    }
    float2 *part = reinterpret_cast<float2 *>(ws + at.part);
    float *picked = reinterpret_cast<float *>(ws + at.picked);
    float *scale = reinterpret_cast<float *>(ws + at.scale);
    uint16_t *codes = reinterpret_cast<uint16_t *>(ws + at.codes);
    if (!grad && !losses) return 0;
    if (const int groups = hc.groups + wc.groups + grad) {
        hipLaunchKernelGGL(head_prepare_kernel, dim3(unsigned(groups)), dim3(kPrepare), 0, st, hc, wc, g, targets, d->rows,
                           F16 ? 16384.0f : 1.0f, scale);
        if (check(hipGetLastError(), "head_prepare_kernel launch")) return 1;
    }
    if (!grad) return losses_alone<F16>(st, d, most, h, h_m, w, w_n, targets, part, picked, losses);
    const PartPlan pi = input_plan(d), pw = weight_plan(d);
    const int64_t pieces = pieces_of(d);
    float *sums = reinterpret_cast<float *>(ws + at.weight_sums), *parts = reinterpret_cast<float *>(ws + at.input_parts);
    const float *inverse = scale + 1;
    for (int64_t i = 0, r0 = 0; i < pieces; ++i, r0 += most) {
        const int64_t rows = std::min(most, d->rows - r0);
        const uint16_t *hp = h + r0 * h_m;
        targets.target = static_cast<const char *>(target) + r0 * tsize;
        if (logits<F16, true>(st, d, rows, hp, h_m, w, w_n, HeadOut<true>{part, picked, codes, targets, blocks})) return 1;
        const unsigned shares = unsigned(std::clamp<int64_t>(1024 / rows, 1, (blocks + 31) / 32));
        hipLaunchKernelGGL((head_grad_kernel<F16>), dim3(unsigned(rows), shares), dim3(256), 0, st, codes, part, picked, g + r0, scale,
                           targets, blocks, losses ? losses + r0 : nullptr);
        if (check(hipGetLastError(), "head_grad_kernel launch")) return 1;
        if (const BothPlan both = both_plan(d); both.parts && dh && dw) {
            if (both_grads<F16>(st, d, both, codes, w, w_n, hp, h_m, parts, HeadStore{nullptr, nullptr, dh, inverse, d->k, F16},
                                HeadStore{nullptr, nullptr, dw, inverse, d->k, F16}))
                return 1;
            break;
        }
        // a last piece of fewer rows keeps its plan: its sums are shorter, its tiles fewer
        if (dh && input_grad<F16>(st, d, pi, rows, codes, w, w_n, parts, HeadStore{nullptr, nullptr, dh + r0 * d->k, inverse, d->k, F16}))
            return 1;
        if (dw) {
            PartPlan p = pw;
            p.k_part = int(std::min<int64_t>(p.k_part, (rows + 63) / 64));
            if (weight_grad<F16>(st, d, p, rows, codes, hp, h_m, parts,
                                 HeadStore{i ? sums : nullptr, i + 1 < pieces ? sums : nullptr, dw, inverse, d->k, F16}))
                return 1;
        }
    }
    return 0;
}

}  // namespace

int head_on(hipStream_t st, const nhip_head_desc *d, const void *h, const void *w, const void *target, const float *g, float *losses,
            void *dh, void *dw, void *ws) {
    if (head_check(d, "nhip_head_loss")) return 1;
    if (!g && (dh || dw)) return fail("nhip_head_loss: gradients need the losses' cotangents");
    if (!on(ws, 256)) return fail("nhip_head_loss: the workspace starts on 256 bytes");
    if (!on(dh, 8) || !on(dw, 8)) return fail("nhip_head_loss: gradients start on 8 bytes");
    if ((!dh && !dw && !copies(d, d->h_m) && !on(h, 16)) || (!copies(d, d->w_n) && !on(w, 16)))
        return fail("nhip_head_loss: operands of whole rows start on 16 bytes");
    if (d->rows == 0) return dw ? fill_on(st, dw, size_t(d->classes) * d->k * 2, 0) : 0;
    if (!ws) return fail("nhip_head_loss: no workspace");
    if (!h || !w || !target) return fail("nhip_head_loss: an operand without memory");
    auto go = d->dtype == NHIP_F16 ? head_run<true> : head_run<false>;
    return go(st, d, static_cast<const uint16_t *>(h), static_cast<const uint16_t *>(w), target, g, losses, static_cast<uint16_t *>(dh),
              static_cast<uint16_t *>(dw), static_cast<char *>(ws));
}

}  // namespace nhip

extern "C" {

int nhip_head_loss(const nhip_head_desc *desc, const void *h, const void *w, const void *target, const float *g, float *losses, void *dh,
                   void *dw, void *workspace) {
    hipStream_t st = stream_of_current();
    if (!st) return fail("no HIP stream: call nhip_set_device first");
    return head_on(st, desc, h, w, target, g, losses, dh, dw, workspace);
}

int nhip_head_loss_workspace(const nhip_head_desc *desc, int gradients, size_t *bytes) {
    if (head_check(desc, "nhip_head_loss_workspace")) return 1;
    *bytes = head_space(desc, gradients != 0).bytes;
    return 0;
}

}  // extern "C"

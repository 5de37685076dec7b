// C entry points of packed self attention (packed.h).
#include <algorithm>
#include <cstring>
#include <string>

#include "packed.h"

using namespace nhip;
using namespace nhipk;

namespace nhip {
namespace {

constexpr int64_t kPackedTokens = int64_t(1) << 26, kPackedSequences = int64_t(1) << 20;

int64_t value_dim(const nhip_packed_desc *d) { return d->value_head_dim ? d->value_head_dim : d->head_dim; }
int64_t kernel_dim(const nhip_packed_desc *d) { return std::max(d->head_dim, value_dim(d)) <= 64 ? 64 : 128; }

// Queries a forward workgroup takes, and keys and queries the backward's.
constexpr int64_t kFwdBlock = 128, kKeyBlock = 128, kDqBlock = 256;

// Entries of a table: the most workgroups that any offsets give.
int64_t table_entries(const nhip_packed_desc *d, int64_t block) {
    return d->tokens / block + std::min(d->sequences, d->tokens) + 2;
}
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
bool few(const nhip_packed_desc *d) { return d->sequences < kPackedFew; }
// Whether the forward's workgroups find their tiles themselves: all run at once.
bool direct(const nhip_packed_desc *d) {
    constexpr int64_t CUS = 256;
    const int64_t at_once = CUS * (kernel_dim(d) == 64 ? FwdOccupancy<4, 64>::kBlocks : FwdOccupancy<4, 128>::kBlocks);
    return d->sequences <= kPackedDirect && table_entries(d, kFwdBlock) * d->heads <= at_once;
}
size_t table_bytes(const nhip_packed_desc *d, int64_t block) { return up256(table_entries(d, block) * sizeof(PackedTile)); }

// The most dS tiles of a head that any offsets give: ceil(l / 128) ceil(l / 64) over lengths l that add up to the tokens.
int64_t most_ds(const nhip_packed_desc *d) {
    return d->tokens * d->tokens / 8192 + 3 * d->tokens / 128 + 1 + std::min(d->sequences, d->tokens);
}
int64_t ds_room(const nhip_packed_desc *d) {
    if (d->ds_bytes <= 0 || d->heads <= 0) return 0;
    // below 2^24: what packed_tiles_few_kernel counts to
    return std::min<int64_t>(std::min(most_ds(d), d->ds_bytes / (d->heads * 128 * 64 * 2)), (1 << 24) - 1);
}

// Parts of a key block's query tiles where whole blocks leave half of the CUs or more idle: as many as give each CU a workgroup,
// but no more than three quarters of a block's tiles, since a part costs the K and V operands' loads and its sums' traffic. Blocks
// are estimated with half a one a sequence lost, tiles from the mean length. Us of the kernel and its sums by parts (* taken):
//   331 + 254 + 129 + 97 tokens, 6 heads of 2, dims 80, unmasked    1: 62   2: 39  4: 27  6: 22  7: 22*  8: 23  12: 30  16: 34
//   1500 + 500 + 48 tokens, 8 heads of 2, dims 128, causal          1: 259  2: 136  4: 76  6: 59  7: 55*  8: 55  12: 58  16: 60
//   200 + 300 + 12 tokens, 8 heads of 8, dims 64, causal            1: 19   2: 17  3: 15*  4: 16  6: 17  8: 19  12: 24
int64_t key_parts(const nhip_packed_desc *d) {
    const int64_t sequences = std::max<int64_t>(std::min(d->sequences, d->tokens), 1), kv_heads = std::max<int64_t>(d->kv_heads, 1);
    const int64_t blocks = (d->tokens / kKeyBlock + sequences / 2 + 1) * kv_heads;
    const int64_t tiles = (d->tokens + 64 * sequences - 1) / (64 * sequences) * (d->heads / kv_heads);
    return std::max<int64_t>(std::min<int64_t>({256 / blocks, (3 * tiles + 3) / 4, 16}), 1);
}

// The backward's workspace: delta and the base-2 LSE, the flag, both tables, dS.
struct BwdSpace {
    size_t stats, flag, keys, queries, sums, ds, bytes;
};
BwdSpace bwd_space(const nhip_packed_desc *d) {
    BwdSpace w{};
    w.stats = 0;
    w.flag = up256(2 * size_t(d->heads) * d->tokens * sizeof(float));
    w.keys = w.flag + 256;
    w.queries = w.keys + table_bytes(d, kKeyBlock);
    w.sums = w.queries + table_bytes(d, kDqBlock);
    const int64_t parts = key_parts(d);
    w.ds = w.sums + (parts > 1 ? size_t(parts) * table_entries(d, kKeyBlock) * d->kv_heads * 256 * kernel_dim(d) * sizeof(float) : 0);
    w.bytes = w.ds + size_t(ds_room(d)) * d->heads * (128 * 64 * 2);
    return w;
}

int packed_check(const nhip_packed_desc *d, const char *what) {
    const std::string at(what);
    if (d->tokens < 0 || d->sequences < 0 || d->heads < 0 || d->kv_heads < 0) return fail(at + ": negative sizes");
    for (int64_t hd : {d->head_dim, value_dim(d)})
        if (hd <= 0 || hd % 8 || hd > 128)
            return fail(at + ": head dim " + std::to_string(hd) + " (the hip kernels take multiples of 8 up to 128)");
    if (d->dtype != NHIP_BF16 && d->dtype != NHIP_F16) return fail(at + ": bf16 or f16 operands only");
    if (d->kv_heads ? d->heads % d->kv_heads : d->heads) return fail(at + ": heads must be a multiple of kv_heads");
    if (d->offsets_dtype != NHIP_POS_I32 && d->offsets_dtype != NHIP_POS_I64) return fail(at + ": offsets are int32 or int64");
    if (!(d->scale > 0.0f) || d->scale > 3.4e38f) return fail(at + ": the scale is positive");
    if (d->tokens > kPackedTokens || d->sequences > kPackedSequences)
        return fail(at + ": at most 2^26 tokens and 2^20 sequences");
    for (int64_t st : {d->q_s, d->q_n, d->k_s, d->k_n, d->v_s, d->v_n, d->o_s, d->o_n, d->do_s, d->do_n, d->dq_s, d->dq_n, d->dk_s,
                       d->dk_n, d->dv_s, d->dv_n})
        if (st % 8) return fail(at + ": every stride must be a multiple of 8 elements (16-byte rows)");
    const int64_t kd = kernel_dim(d), hv = value_dim(d);
    if ((d->head_dim != kd || hv != kd) &&
        !(attn_span_ok(d->tokens, d->q_s, d->head_dim) && attn_span_ok(d->tokens, d->k_s, d->head_dim) &&
          attn_span_ok(d->tokens, d->v_s, hv) && attn_span_ok(d->tokens, d->do_s, hv)))
        return fail(at + ": head dims " + std::to_string(d->head_dim) + " / " + std::to_string(hv) + " are padded to " +
                    std::to_string(kd) + ", which needs each head of an operand within 2 GiB");
    if (std::max(table_entries(d, 64), d->tokens / 8 + 1) * std::max<int64_t>({d->heads, d->kv_heads, 1}) >= int64_t(1) << 24)
        return fail(at + ": a launch of 2^32 threads");
    return 0;
}

int on16(const char *what, std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(std::string(what) + ": operands, results and the workspace start on 16 bytes");
    return 0;
}

int given(const char *what, std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (!p) return fail(std::string(what) + ": an operand or a result without memory");
    return 0;
}

AttnParams packed_params(const nhip_packed_desc *d) {
    AttnParams p{};
    p.sq = p.sk = d->tokens;
    p.heads = d->heads, p.kv_heads = d->kv_heads, p.batch = 1;
    p.hd = d->head_dim, p.hdv = value_dim(d);
    p.q_s = d->q_s, p.q_n = d->q_n, p.k_s = d->k_s, p.k_n = d->k_n, p.v_s = d->v_s, p.v_n = d->v_n;
    p.o_s = d->o_s, p.o_n = d->o_n, p.do_s = d->do_s, p.do_n = d->do_n;
    p.dq_s = d->dq_s, p.dq_n = d->dq_n, p.dk_s = d->dk_s, p.dk_n = d->dk_n, p.dv_s = d->dv_s, p.dv_n = d->dv_n;
    p.scale = d->scale;
    return p;
}

PackedTable table(const nhip_packed_desc *d, int64_t block, int order, void *tiles) {
    PackedTable t{static_cast<PackedTile *>(tiles), int32_t(table_entries(d, block)), int32_t(block), 0,
                  d->causal ? order : PACKED_FLAT};
    while (((d->tokens + block - 1) / block) >> t.shift >= kPackedBuckets) ++t.shift;
    return t;
}

PackedTables tables_of(const nhip_packed_desc *d, const void *offsets) {
    PackedTables a{};
    a.offsets = offsets, a.sequences = d->sequences, a.tokens = d->tokens, a.o64 = d->offsets_dtype == NHIP_POS_I64;
    return a;
}

int build_tables(hipStream_t st, const nhip_packed_desc *d, const PackedTables &a, int count) {
    if (few(d)) hipLaunchKernelGGL(packed_tiles_few_kernel, dim3(unsigned(count)), dim3(kPackedFew), 0, st, a);
    else hipLaunchKernelGGL(packed_tiles_kernel, dim3(unsigned(count)), dim3(kPackedBuckets), 0, st, a);
    return check(hipGetLastError(), "packed_tiles_kernel launch");
}

template <int D, bool F16, bool CAUSAL>
int fwd(hipStream_t st, const nhip_packed_desc *d, const AttnParams &p, uint16_t *rest, const PackedTables &a) {
    const dim3 grid(unsigned(a.t[0].most * d->heads));
    hipLaunchKernelGGL((packed_fwd_kernel<D, F16, CAUSAL, kFwdBlock / 32>), grid, dim3(256), 0, st, p, rest, a);
    return check(hipGetLastError(), "packed_fwd_kernel launch");
}

template <int D, bool F16, bool CAUSAL>
int dkdv(hipStream_t st, const nhip_packed_desc *d, const AttnParams &p, const PackedTables &a, const float *lse2, const int32_t *fits,
         float *sums, bool store) {
    const int64_t parts = key_parts(d);
    const dim3 grid(unsigned(a.t[0].most * d->kv_heads), unsigned(parts));
    auto kern = parts > 1 ? (store ? packed_dkdv_kernel<D, F16, CAUSAL, true, true> : packed_dkdv_kernel<D, F16, CAUSAL, false, true>)
                          : (store ? packed_dkdv_kernel<D, F16, CAUSAL, true, false> : packed_dkdv_kernel<D, F16, CAUSAL, false, false>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, p, lse2, a.t[0].tiles, d->tokens, fits, sums);
    return check(hipGetLastError(), "packed_dkdv_kernel launch");
}

template <int D, bool F16, bool CAUSAL>
int bwd(hipStream_t st, const nhip_packed_desc *d, const AttnParams &p, const uint16_t *rest, const PackedTables &a, bool store, bool again,
        float *sums) {
    float *lse2 = p.delta + size_t(d->heads) * d->tokens;
    constexpr int RPB = 256 / (D / 8);
    const int tables = few(d) ? 2 : 0;
    if (const int64_t blocks = (d->heads * d->tokens + RPB - 1) / RPB + tables) {
        hipLaunchKernelGGL((packed_prep_kernel<D, F16>), dim3(unsigned(blocks)), dim3(256), 0, st, p, rest, lse2, a, tables);
        if (check(hipGetLastError(), "packed delta launch")) return 1;
    }
    const dim3 gq(unsigned(a.t[1].most * d->heads));
    const int32_t *fits = store && again ? a.fits : nullptr;
    if (store) {
        if (dkdv<D, F16, CAUSAL>(st, d, p, a, lse2, fits, sums, true)) return 1;
        hipLaunchKernelGGL((packed_dq_ds_kernel<D, F16, CAUSAL>), gq, dim3(256), 0, st, p, a.t[1].tiles, fits);
        if (check(hipGetLastError(), "packed_dq_ds_kernel launch")) return 1;
    }
    if (again) {
        if (dkdv<D, F16, CAUSAL>(st, d, p, a, lse2, fits, sums, false)) return 1;
        if (!d->heads) return 0;  // no query: no tile to add to dK and dV, zeros
        hipLaunchKernelGGL((packed_dq_kernel<D, F16, CAUSAL>), gq, dim3(256), 0, st, p, lse2, a.t[1].tiles, d->tokens, fits);
        if (check(hipGetLastError(), "packed_dq_kernel launch")) return 1;
    }
    const int64_t parts = key_parts(d);
    if (parts == 1) return 0;
    hipLaunchKernelGGL((packed_dkdv_sum_kernel<D, F16>), dim3(unsigned(a.t[0].most * d->kv_heads), D / 16), dim3(256), 0, st, p,
                       a.t[0].tiles, sums, int(parts));
    return check(hipGetLastError(), "packed_dkdv_sum_kernel launch");
}

}  // namespace

int packed_fwd_on(hipStream_t st, const nhip_packed_desc *d, const void *q, const void *k, const void *v, const void *offsets, void *o,
                  void *rest, float *lse, void *ws) {
    if (packed_check(d, "nhip_packed_fwd") || on16("nhip_packed_fwd", {q, k, v, o, rest, ws})) return 1;
    if (d->tokens == 0 || d->heads == 0) return 0;
    if (!ws) return fail("nhip_packed_fwd: no workspace");
    if (given("nhip_packed_fwd", {q, k, v, offsets, o})) return 1;
    AttnParams p = packed_params(d);
    p.q = static_cast<const uint16_t *>(q), p.k = static_cast<const uint16_t *>(k), p.v = static_cast<const uint16_t *>(v);
    p.o = static_cast<uint16_t *>(o), p.lse = lse;
    uint16_t *left = static_cast<uint16_t *>(rest);
    PackedTables a = tables_of(d, offsets);
    a.t[0] = table(d, kFwdBlock, PACKED_RISING, direct(d) ? nullptr : ws);
    if (a.t[0].tiles && build_tables(st, d, a, 1)) return 1;
    const bool f16 = d->dtype == NHIP_F16;
#define NHIP_PACKED(DD)                                                                                      \
    return f16 ? (d->causal ? fwd<DD, true, true>(st, d, p, left, a) : fwd<DD, true, false>(st, d, p, left, a)) \
               : (d->causal ? fwd<DD, false, true>(st, d, p, left, a) : fwd<DD, false, false>(st, d, p, left, a))
    if (kernel_dim(d) == 64) NHIP_PACKED(64);
    NHIP_PACKED(128);
#undef NHIP_PACKED
}

int packed_bwd_on(hipStream_t st, const nhip_packed_desc *d, const void *q, const void *k, const void *v, const void *offsets,
                  const void *o, const void *rest, const void *d_o, const float *lse, void *dq, void *dk, void *dv, void *ws) {
    if (packed_check(d, "nhip_packed_bwd") || on16("nhip_packed_bwd", {q, k, v, o, rest, d_o, dq, dk, dv, ws})) return 1;
    if (d->tokens == 0 || d->kv_heads == 0) return 0;
    if (!ws) return fail("nhip_packed_bwd: no workspace");
    if (given("nhip_packed_bwd", {k, v, offsets, dk, dv}) || (d->heads && given("nhip_packed_bwd", {q, o, d_o, lse, dq}))) return 1;
    const BwdSpace w = bwd_space(d);
    char *at = static_cast<char *>(ws);
    AttnParams p = packed_params(d);
    p.q = static_cast<const uint16_t *>(q), p.k = static_cast<const uint16_t *>(k), p.v = static_cast<const uint16_t *>(v);
    p.o_in = static_cast<const uint16_t *>(o), p.d_o = static_cast<const uint16_t *>(d_o), p.lse_in = lse;
    p.dq = static_cast<uint16_t *>(dq), p.dk = static_cast<uint16_t *>(dk), p.dv = static_cast<uint16_t *>(dv);
    const uint16_t *left = static_cast<const uint16_t *>(rest);
    p.delta = reinterpret_cast<float *>(at + w.stats);
    p.ds = reinterpret_cast<uint16_t *>(at + w.ds);
    float *sums = reinterpret_cast<float *>(at + w.sums);
    const int64_t room = ds_room(d);
    const bool store = room > 0, again = room < most_ds(d);
    PackedTables a = tables_of(d, offsets);
    a.t[0] = table(d, kKeyBlock, PACKED_FALLING, at + w.keys);
    a.t[1] = table(d, kDqBlock, PACKED_RISING, at + w.queries);
    a.ds_tiles = room;
    a.fits = reinterpret_cast<int32_t *>(at + w.flag);
    if (!few(d) && build_tables(st, d, a, 2)) return 1;  // else the workgroups of bwd()'s first launch do
    const bool f16 = d->dtype == NHIP_F16;
#define NHIP_PACKED(DD)                                                                 \
    return f16 ? (d->causal ? bwd<DD, true, true>(st, d, p, left, a, store, again, sums)      \
                            : bwd<DD, true, false>(st, d, p, left, a, store, again, sums))    \
               : (d->causal ? bwd<DD, false, true>(st, d, p, left, a, store, again, sums)     \
                            : bwd<DD, false, false>(st, d, p, left, a, store, again, sums))
    if (kernel_dim(d) == 64) NHIP_PACKED(64);
    NHIP_PACKED(128);
#undef NHIP_PACKED
}

}  // namespace nhip

extern "C" {

int nhip_packed_fwd(const nhip_packed_desc *desc, const void *q, const void *k, const void *v, const void *offsets, void *o, void *rest,
                    float *lse, void *workspace) {
    hipStream_t st = stream_of_current();
    if (!st) return fail("no HIP stream: call nhip_set_device first");
    return packed_fwd_on(st, desc, q, k, v, offsets, o, rest, lse, workspace);
}

int nhip_packed_bwd(const nhip_packed_desc *desc, const void *q, const void *k, const void *v, const void *offsets, const void *o,
                    const void *rest, const void *d_o, const float *lse, void *dq, void *dk, void *dv, void *workspace) {
    hipStream_t st = stream_of_current();
    if (!st) return fail("no HIP stream: call nhip_set_device first");
    return packed_bwd_on(st, desc, q, k, v, offsets, o, rest, d_o, lse, dq, dk, dv, workspace);
}

int nhip_packed_workspace(const nhip_packed_desc *desc, int backward, size_t *bytes) {
    if (packed_check(desc, "nhip_packed_workspace")) return 1;
    *bytes = backward ? bwd_space(desc).bytes : table_bytes(desc, kFwdBlock);
    return 0;
}

}  // extern "C"

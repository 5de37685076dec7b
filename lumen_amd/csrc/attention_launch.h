// Launches of the flash attention kernels (attention.h), for attention.hip alone.
#pragma once

#include "attention.h"

namespace nhip {

template <int D, bool F16, bool CAUSAL, int NW>
int launch_fwd_nw(hipStream_t s, const nhipk::AttnParams &p, const nhip_attn_desc *d) {
    dim3 grid(unsigned((d->sq + 32 * NW - 1) / (32 * NW) * d->heads * d->batch));
    if constexpr (D == 64 && NW == 4) {
        // Waves a SIMD: two where a causal launch nearly fits them (FwdOccupancy); four where a launch without a mask
        // fits them and not three, which would run a second round for a few workgroups (us with three, four: 784
        // workgroups of 3494 keys 153.3, 148.3; 800 of 1212 58.8, 56.5; 832 of 141 17.6, 17.1; 988 of 6914 316, 308).
        constexpr int kWaves = CAUSAL ? 2 : 4;
        if (CAUSAL ? grid.x <= 640 : grid.x > 768 && grid.x <= 1024) {
            hipLaunchKernelGGL((nhipk::flash_fwd_kernel<D, F16, CAUSAL, NW, kWaves>), grid, dim3(64 * NW), 0, s, p);
            return check(hipGetLastError(), "flash_fwd launch");
        }
    }
    hipLaunchKernelGGL((nhipk::flash_fwd_kernel<D, F16, CAUSAL, NW>), grid, dim3(64 * NW), 0, s, p);
    return check(hipGetLastError(), "flash_fwd launch");
}

template <int D, bool F16, bool CAUSAL>
int launch_fwd(hipStream_t s, const nhipk::AttnParams &p, const nhip_attn_desc *d) {
    if constexpr (D > 128) {
        // head dim 256: 4 waves, one workgroup a CU (its K/V tiles fill 128 KiB of LDS), whatever the config
        return launch_fwd_nw<D, F16, CAUSAL, 4>(s, p, d);
    } else {
        // by default 128 queries a workgroup, or 64 at head dim 64 where there are no more and the workgroups are more
        // than the CUs hold, three each: waves without a query hold registers that others could use ([32, 1, 32 / 8, 64]
        // over 1 key 8.9 us, 6.6; over 65 11.6, 7.8; 64 queries over 256 keys 18.9, 16.9; but [32, 1, 16, 64] 5.8, 6.2)
        switch (d->config >= 0 ? d->config : D == 64 && d->sq <= 64 && d->heads * d->batch > 768 ? 2 : 0) {
            case 1: return launch_fwd_nw<D, F16, CAUSAL, 8>(s, p, d);
            case 2: return launch_fwd_nw<D, F16, CAUSAL, 2>(s, p, d);
            default: return launch_fwd_nw<D, F16, CAUSAL, 4>(s, p, d);
        }
    }
}

// Whether a forward divides the keys over waves (attention_split.h), and that launch: `ws` as
// flash_fwd_workspace_bytes says, or null for one workgroup a row tile.
bool split_keys(const nhip_attn_desc *d);
int launch_split(hipStream_t s, const nhipk::AttnParams &p, const nhip_attn_desc *d, void *ws);

int flash_fwd_on(hipStream_t s, const nhip_attn_desc *d, const void *q, const void *k, const void *v, void *o,
                 float *lse, void *ws) {
    if (check_attn(d, "flash attention", 256)) return 1;
    if (d->sq == 0 || d->batch == 0 || d->heads == 0) return 0;
    nhipk::AttnParams p = attn_params(d);
    p.q = static_cast<const uint16_t *>(q);
    p.k = static_cast<const uint16_t *>(k);
    p.v = static_cast<const uint16_t *>(v);
    p.o = static_cast<uint16_t *>(o);
    p.lse = lse;
    bool f16 = d->dtype == NHIP_F16;
    if (split_keys(d)) return launch_split(s, p, d, ws);
#define NHIP_FWD(DD, FF, CC) return launch_fwd<DD, FF, CC>(s, p, d)
    const int64_t kd = kernel_dim(d);
    if (kd == 256) {
        if (f16) { if (d->causal) NHIP_FWD(256, true, true); NHIP_FWD(256, true, false); }
        if (d->causal) NHIP_FWD(256, false, true);
        NHIP_FWD(256, false, false);
    }
    if (kd == 128) {
        if (f16) { if (d->causal) NHIP_FWD(128, true, true); NHIP_FWD(128, true, false); }
        if (d->causal) NHIP_FWD(128, false, true);
        NHIP_FWD(128, false, false);
    }
    if (f16) { if (d->causal) NHIP_FWD(64, true, true); NHIP_FWD(64, true, false); }
    if (d->causal) NHIP_FWD(64, false, true);
    NHIP_FWD(64, false, false);
#undef NHIP_FWD
}

template <int D, bool F16, bool CAUSAL>
int launch_bwd(hipStream_t s, const nhipk::AttnParams &p, const nhip_attn_desc *d) {
    const bool atomic = p.dqacc != nullptr;
    dim3 gd(unsigned((d->heads * d->sq + 3) / 4), unsigned(d->batch));
    // dK/dV: a workgroup per key block, or per pair of key blocks (i, nkb - 1 - i) (nhipk::DkdvPaired)
    const int64_t nkb = (d->sk + 127) / 128;
    dim3 gk(unsigned((nhipk::DkdvPaired<CAUSAL, false>::value ? (nkb + 1) / 2 : nkb) * d->kv_heads * d->batch));
    dim3 gka(unsigned((nhipk::DkdvPaired<CAUSAL, true>::value ? (nkb + 1) / 2 : nkb) * d->kv_heads * d->batch));
    dim3 gq(unsigned((d->sq + 127) / 128 * d->heads * d->batch));
    float *lse2 = p.delta + size_t(d->batch) * d->heads * d->sq;
    // 16-byte rows: D / 8 lanes each; else one wavefront a row
    const bool vec = d->head_dim == D && value_head_dim(d) == D && D % 8 == 0 && 64 % (D / 8 > 0 ? D / 8 : 1) == 0 && D / 8 <= 64 &&
                     ((reinterpret_cast<uintptr_t>(p.o_in) | reinterpret_cast<uintptr_t>(p.d_o)) & 15) == 0 &&
                     (p.o_b | p.o_n | p.o_s | p.do_b | p.do_n | p.do_s) % 8 == 0;
    if constexpr (D % 8 == 0 && D >= 8 && D <= 512 && 64 % (D / 8) == 0) {
        if (vec) {
            constexpr int RPB = 256 / (D / 8);
            dim3 gv(unsigned((d->heads * d->sq + RPB - 1) / RPB), unsigned(d->batch));
            hipLaunchKernelGGL((nhipk::flash_prep_vec_kernel<D, F16>), gv, dim3(256), 0, s, p, lse2);
        } else {
            hipLaunchKernelGGL((nhipk::flash_prep_kernel<D, F16>), gd, dim3(256), 0, s, p, lse2);
        }
    } else {
        hipLaunchKernelGGL((nhipk::flash_prep_kernel<D, F16>), gd, dim3(256), 0, s, p, lse2);
    }
    if (check(hipGetLastError(), "flash delta launch")) return 1;
    if (atomic) {
        hipLaunchKernelGGL((nhipk::flash_dkdv_kernel<D, F16, CAUSAL, true>), gka, dim3(256), 0, s, p, lse2);
        if (check(hipGetLastError(), "flash dkdv+dq launch")) return 1;
        const int64_t rows = d->batch * d->heads * d->sq;
        dim3 gc(unsigned((rows * (D / 8) + 255) / 256));
        hipLaunchKernelGGL((nhipk::flash_dq_round_kernel<D, F16>), gc, dim3(256), 0, s, p);
        return check(hipGetLastError(), "flash dq rounding launch");
    }
    if (p.ds) {
        hipLaunchKernelGGL((nhipk::flash_dkdv_kernel<D, F16, CAUSAL, false, true>), gk, dim3(256), 0, s, p, lse2);
        if (check(hipGetLastError(), "flash dkdv+dS launch")) return 1;
        dim3 gs(unsigned((d->sq + 255) / 256 * d->heads * d->batch));
        hipLaunchKernelGGL((nhipk::flash_dq_ds_kernel<D, F16, CAUSAL>), gs, dim3(256), 0, s, p);
        return check(hipGetLastError(), "flash dq from dS launch");
    }
    hipLaunchKernelGGL((nhipk::flash_dkdv_kernel<D, F16, CAUSAL>), gk, dim3(256), 0, s, p, lse2);
    if (check(hipGetLastError(), "flash dkdv launch")) return 1;
    hipLaunchKernelGGL((nhipk::flash_dq_kernel<D, F16, CAUSAL>), gq, dim3(256), 0, s, p, lse2);
    return check(hipGetLastError(), "flash dq launch");
}

int flash_bwd_on(hipStream_t s, const nhip_attn_desc *d, const void *q, const void *k, const void *v, const void *o,
                 const void *d_o, const float *lse, void *dq, void *dk, void *dv, void *ws) {
    if (check_attn(d, "flash attention backward")) return 1;
    if (d->batch == 0 || d->heads == 0) return 0;
    nhipk::AttnParams p = attn_params(d);
    p.q = static_cast<const uint16_t *>(q);
    p.k = static_cast<const uint16_t *>(k);
    p.v = static_cast<const uint16_t *>(v);
    p.o_in = static_cast<const uint16_t *>(o);
    p.d_o = static_cast<const uint16_t *>(d_o);
    p.lse_in = lse;
    p.dq = static_cast<uint16_t *>(dq);
    p.dk = static_cast<uint16_t *>(dk);
    p.dv = static_cast<uint16_t *>(dv);
    p.delta = static_cast<float *>(ws);
    p.dqacc = d->deterministic ? nullptr : reinterpret_cast<float *>(static_cast<char *>(ws) + flash_bwd_dq_offset(d));
    p.ds = d->deterministic == 1 ? reinterpret_cast<uint16_t *>(static_cast<char *>(ws) + flash_bwd_dq_offset(d)) : nullptr;
    bool f16 = d->dtype == NHIP_F16;
#define NHIP_BWD(DD, FF, CC) return launch_bwd<DD, FF, CC>(s, p, d)
    if (kernel_dim(d) == 128) {
        if (f16) { if (d->causal) NHIP_BWD(128, true, true); NHIP_BWD(128, true, false); }
        if (d->causal) NHIP_BWD(128, false, true);
        NHIP_BWD(128, false, false);
    }
    if (f16) { if (d->causal) NHIP_BWD(64, true, true); NHIP_BWD(64, true, false); }
    if (d->causal) NHIP_BWD(64, false, true);
    NHIP_BWD(64, false, false);
#undef NHIP_BWD
}

}  // namespace nhip

// C entry point of the AdamW step (adamw.h).
#include <cstring>

#include "adamw.h"
#include "nhip_internal.h"

using namespace nhipk;

namespace nhip {
namespace {

bool adam_rate(double x) { return x >= 0.0 && x < 1.0; }

// Whether every vector access of the tensor is aligned: four elements of each pointer's type.
bool adam_wide(const nhip_adamw_tensor &x) {
    const size_t e = x.dtype == NHIP_F32 ? 16 : 8;
    auto on = [](const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    return on(x.param_out, e) && on(x.grad, e) && on(x.m, 16) && on(x.v, 16) && on(x.m_out, 16) && on(x.v_out, 16) &&
           (x.master ? on(x.master, 16) && on(x.master_out, 16) : on(x.param, e));
}

static_assert(NHIP_F32 == 0 && NHIP_BF16 == 1 && NHIP_F16 == 2 && NHIP_POS_I32 == 1 && NHIP_POS_I64 == 2, "adamw.h's types");

int adam_check(const nhip_adamw_desc *d, const nhip_adamw_tensor *t, const void *step_at) {
    if (d->count < 0) return fail("nhip_adamw: negative count");
    if (!adam_rate(d->beta1) || !adam_rate(d->beta2)) return fail("nhip_adamw: betas are at least 0 and below 1");
    if (!(d->eps >= 0.0)) return fail("nhip_adamw: eps is at least 0");
    if (!step_at && !(d->step >= 1.0)) return fail("nhip_adamw: steps count from 1");
    if (d->step_type < NHIP_POS_NONE || d->step_type > NHIP_POS_I64) return fail("nhip_adamw: the step is float64, int32 or int64");
    for (int64_t i = 0; i < d->count; ++i) {
        const nhip_adamw_tensor &x = t[i];
        if (x.numel < 0) return fail("nhip_adamw: negative element count");
        if (x.dtype != NHIP_F32 && x.dtype != NHIP_BF16 && x.dtype != NHIP_F16)
            return fail("nhip_adamw: weights are float32, bf16 or f16");
        if (!x.master && x.master_out) return fail("nhip_adamw: a new master is an old one's");
        if (x.master && x.dtype == NHIP_F32) return fail("nhip_adamw: masters are of 16-bit weights");
        if (x.numel > 0 && (!(x.master ? static_cast<const void *>(x.master) : x.param) || !x.grad || !x.m || !x.v))
            return fail("nhip_adamw: a tensor without memory");
    }
    return 0;
}

}  // namespace

int adamw_on(hipStream_t st, const nhip_adamw_desc *d, const nhip_adamw_tensor *t, const double *lr_at, const void *step_at,
             const float *scale_at) {
    if (adam_check(d, t, step_at)) return 1;
    const AdamRates r{lr_at, step_at, scale_at, d->step_type, d->lr, d->step, d->beta1, d->beta2, d->eps, d->weight_decay};
    for (int64_t first = 0; first < d->count; first += kAdamTensors) {
        AdamTable a;
        std::memset(&a, 0, sizeof(a));
        a.tensors = int(d->count - first < kAdamTensors ? d->count - first : kAdamTensors);
        int64_t chunks = 0;
        for (int i = 0; i < a.tensors; ++i) {
            const nhip_adamw_tensor &x = t[first + i];
            a.t[i] = AdamTensor{x.master ? static_cast<const void *>(x.master) : x.param, x.grad, x.m, x.v, x.param_out,
                                x.master_out, x.m_out, x.v_out, x.numel};
            a.dtype[i] = uint8_t(x.dtype + (x.master ? 2 : 0)), a.wide[i] = adam_wide(x), a.first[i] = uint32_t(chunks);
            chunks += (x.numel + kAdamChunk - 1) / kAdamChunk;
            if (chunks > 0x7fffffff) return fail("nhip_adamw: over 2^43 elements");
        }
        a.first[a.tensors] = uint32_t(chunks);
        if (!chunks) continue;
        a.blocks = uint32_t(chunks < kAdamBlocks ? chunks : kAdamBlocks);
        hipLaunchKernelGGL(adamw_kernel, dim3(a.blocks), dim3(256), 0, st, a, r);
        if (check(hipGetLastError(), "adamw_kernel launch")) return 1;
    }
    return 0;
}

}  // namespace nhip

using namespace nhip;

extern "C" int nhip_adamw(const nhip_adamw_desc *desc, const nhip_adamw_tensor *tensors, const double *lr_at,
                          const void *step_at, const float *grad_scale_at) {
    hipStream_t st = stream_of_current();
    if (!st) return fail("no HIP stream: call nhip_set_device first");
    return adamw_on(st, desc, tensors, lr_at, step_at, grad_scale_at);
}

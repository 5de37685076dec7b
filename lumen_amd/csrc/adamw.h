// One AdamW step over many tensors:
//
//   m' = b1 m + (1 - b1) g,  v' = b2 v + (1 - b2) g^2
//   w' = w (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// w is the weight, or where a 16-bit weight has one its float32 master, of which the weight is then the rounded value. HBM
// bounds it: every operand is read once and every result written once (16-bit weights with masters 28 bytes an element,
// float32 ones the same). One launch for kAdamTensors tensors: workgroups walk chunks of kAdamChunk elements over all of
// them, which a table in the kernel's arguments maps to a tensor by binary search, so many small weights cost no more than
// one large one and the table needs no copy to the device.
//
// 39 million bf16 weights with masters (1.09 GB) 205 us, 5.3 TB/s; 203 million (5.7 GB) 1.05 to 1.06 ms, 5.4 TB/s, a copy being
// 5.1; 12 small float32 ones (8 MB) 7.7 us.
//
// The moments are float32 and so is everything of an element, each operation rounded on its own: the step's factors are
// worked out in float64 (b^t of a late step, 1 - b^t of an early one) and rounded once. A thread reads its elements
// before it writes them, so any result may lie over the operand that it replaces.
#pragma once

#include "device_common.h"

namespace nhipk {

constexpr int kAdamTensors = 44;      // a launch's table within the 4 KiB of kernel arguments
constexpr int kAdamBlocks = 2048;     // workgroups of a launch: eight a CU
constexpr int64_t kAdamChunk = 4096;  // elements: 16 a thread

struct AdamTensor {
    const void *w;  // the weight's values: float32 with a master, else of the weight's type
    const void *g;
    const float *m, *v;
    void *p_out;    // the weight; each result null where nothing reads it
    float *w_out;   // its master
    float *m_out, *v_out;
    int64_t numel;
};
struct AdamTable {
    AdamTensor t[kAdamTensors];
    uint32_t first[kAdamTensors + 1];  // each tensor's first chunk; the last entry their count
    uint8_t dtype[kAdamTensors];       // 0 float32, 1 bf16, 2 f16, 3 and 4 these with a master
    uint8_t wide[kAdamTensors];        // whether every pointer starts on four of its elements
    int32_t tensors;
    uint32_t blocks;
};
struct AdamRates {
    const double *lr_at;  // lr_at and step_at are read in place of lr and step where not null
    const void *step_at;
    const float *scale_at;          // a factor of the gradients, each rounded to its type again (null: 1)
    int32_t step_type;              // *step_at: 0 float64, 1 int32, 2 int64
    double lr, step, beta1, beta2, eps, decay;
};
static_assert(sizeof(AdamTable) + sizeof(AdamRates) <= 4096, "a launch's arguments");

struct AdamFactors {
    float b1, a1, b2, a2, keep, rate, root, eps, scale;
};

__device__ __forceinline__ double adam_step(const AdamRates &r) {
    if (!r.step_at) return r.step;
    if (r.step_type == 1) return *static_cast<const int32_t *>(r.step_at);
    if (r.step_type == 2) return double(*static_cast<const int64_t *>(r.step_at));
    return *static_cast<const double *>(r.step_at);
}

__device__ __forceinline__ AdamFactors adam_factors(const AdamRates &r) {
    const double lr = r.lr_at ? *r.lr_at : r.lr, t = adam_step(r);
    AdamFactors f;
    f.b1 = float(r.beta1), f.a1 = float(1.0 - r.beta1), f.b2 = float(r.beta2), f.a2 = float(1.0 - r.beta2);
    f.keep = float(1.0 - lr * r.decay);
    f.rate = float(lr / (1.0 - pow(r.beta1, t)));
    f.root = float(1.0 / sqrt(1.0 - pow(r.beta2, t)));
    f.eps = float(r.eps);
    f.scale = r.scale_at ? *r.scale_at : 1.0f;
    return f;
}

__device__ __forceinline__ void adam_element(const AdamFactors &f, float g, float &w, float &m, float &v) {
    m = m * f.b1 + g * f.a1;
    v = v * f.b2 + (g * g) * f.a2;
    w = w * f.keep - (m * f.rate) / (sqrtf(v) * f.root + f.eps);
}

// The tensor that chunk c lies in: the last whose first chunk is at most c (empty tensors have no chunk).
__device__ __forceinline__ int adam_tensor(const AdamTable &t, uint32_t c) {
    int lo = 0, hi = t.tensors;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ float adam_scaled(float g, float scale) {
    T r;
    store_f32_as(&r, g * scale);
    return load_as_f32(&r);
}

// Four elements' values from and to 16 or 8 aligned bytes.
__device__ __forceinline__ float4 adam_get(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ void adam_put(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
template <typename T>
__device__ __forceinline__ float4 adam_get(const T *p) {
    uint2 raw = *reinterpret_cast<const uint2 *>(p);
    T e[4];
    __builtin_memcpy(e, &raw, 8);
    return make_float4(load_as_f32(e), load_as_f32(e + 1), load_as_f32(e + 2), load_as_f32(e + 3));
}
template <typename T>
__device__ __forceinline__ void adam_put(T *p, float4 v) {
    T e[4];
    store_f32_as(e, v.x), store_f32_as(e + 1, v.y), store_f32_as(e + 2, v.z), store_f32_as(e + 3, v.w);
    uint2 raw;
    __builtin_memcpy(&raw, e, 8);
    *reinterpret_cast<uint2 *>(p) = raw;
}

template <typename T, typename W>
__device__ __forceinline__ void adam_chunk(const AdamTensor &t, const AdamFactors &f, bool scaled, bool wide, int64_t at, int n) {
    const W *w = static_cast<const W *>(t.w) + at;
    const T *g = static_cast<const T *>(t.g) + at;
    const float *m = t.m + at, *v = t.v + at;
    auto out = [&](auto *to) { return to ? to + at : nullptr; };
    T *p = out(static_cast<T *>(t.p_out));
    float *wo = out(t.w_out), *mo = out(t.m_out), *vo = out(t.v_out);
    const int whole = wide ? n / 4 : 0;
    constexpr int FLIGHT = 2;  // fours of a thread in flight
    auto four = [&](int i, float4 w4, float4 g4, float4 m4, float4 v4) __attribute__((always_inline)) {
        float we[4] = {w4.x, w4.y, w4.z, w4.w}, ge[4] = {g4.x, g4.y, g4.z, g4.w}, me[4] = {m4.x, m4.y, m4.z, m4.w},
              ve[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) adam_element(f, scaled ? adam_scaled<T>(ge[e], f.scale) : ge[e], we[e], me[e], ve[e]);
        const float4 wn = make_float4(we[0], we[1], we[2], we[3]);
        if (p) adam_put(p + 4 * i, wn);
        if (wo) adam_put(wo + 4 * i, wn);
        if (mo) adam_put(mo + 4 * i, make_float4(me[0], me[1], me[2], me[3]));
        if (vo) adam_put(vo + 4 * i, make_float4(ve[0], ve[1], ve[2], ve[3]));
    };
    int i = threadIdx.x;
    for (; i + (FLIGHT - 1) * 256 < whole; i += FLIGHT * 256) {
        float4 w4[FLIGHT], g4[FLIGHT], m4[FLIGHT], v4[FLIGHT];
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) {
            const int j = 4 * (i + 256 * k);
            w4[k] = adam_get(w + j), g4[k] = adam_get(g + j), m4[k] = adam_get(m + j), v4[k] = adam_get(v + j);
        }
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) four(i + 256 * k, w4[k], g4[k], m4[k], v4[k]);
    }
    for (; i < whole; i += 256) four(i, adam_get(w + 4 * i), adam_get(g + 4 * i), adam_get(m + 4 * i), adam_get(v + 4 * i));
    for (int j = 4 * whole + threadIdx.x; j < n; j += 256) {
        float we = load_as_f32(w + j), ge = load_as_f32(g + j), me = m[j], ve = v[j];
        adam_element(f, scaled ? adam_scaled<T>(ge, f.scale) : ge, we, me, ve);
        if (p) store_f32_as(p + j, we);
        if (wo) wo[j] = we;
        if (mo) mo[j] = me;
        if (vo) vo[j] = ve;
    }
}

__global__ __launch_bounds__(256) void adamw_kernel(AdamTable t, AdamRates r) {
    const AdamFactors f = adam_factors(r);
    const bool scaled = r.scale_at != nullptr;
    const uint32_t chunks = t.first[t.tensors];
    for (uint32_t c = blockIdx.x; c < chunks; c += t.blocks) {
        const int k = adam_tensor(t, c);
        const AdamTensor &x = t.t[k];
        const int64_t at = int64_t(c - t.first[k]) * kAdamChunk, left = x.numel - at;
        const int n = int(left < kAdamChunk ? left : kAdamChunk);
        const bool wide = t.wide[k];
        switch (t.dtype[k]) {
            case 0: adam_chunk<float, float>(x, f, scaled, wide, at, n); break;
            case 1: adam_chunk<bf16_t, bf16_t>(x, f, scaled, wide, at, n); break;
            case 2: adam_chunk<f16_t, f16_t>(x, f, scaled, wide, at, n); break;
            case 3: adam_chunk<bf16_t, float>(x, f, scaled, wide, at, n); break;
            default: adam_chunk<f16_t, float>(x, f, scaled, wide, at, n);
        }
    }
}

}  // namespace nhipk

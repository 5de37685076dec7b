// The cross entropy of a vocabulary head, and its gradients, without its logits: for rows h [t, k], classes w [v, k]
//
//   l = h w^T, lse = log(sum(exp(l))), loss = lse - l[target], p = exp(l - lse)
//   d = (p - onehot(target)) g, dh = d w, dw = d^T h        (g: a row's cotangent; an ignored row's loss and d are 0)
//
// Six t v k multiply-adds, half of what a backward that computes the logits again would add to the forward's two: the
// forward product's store leaves exp(l - m) as 16 bits for a piece of the rows, m being the maximum of its 64 classes, and
// one pass turns these into d in place once the row's lse is known. A piece's values are scratch that the next piece
// writes over; the logits exist in registers alone.
//
// exp(l - m), between 0 and 1, is kept as a float16 of 2^15 times it: off by 2^-11 relative to the value at most (an eighth of
// what a bf16 p would be) down to 2^-29, by 2^-40 below. d is then rounded once, to the operands'
// type, which the matrix instructions take, with the largest |g| taken to 1 (bf16: a mean's 1 / t would be rounded the
// same way in every row whose p is near 0, a gradient 2^-9 too long) or 2^14 (float16, whose range a mean's p would leave), and
// the products are multiplied by what it was (head_scale).
// Sums are float32; over classes of a row first float32 in blocks of 64, then float64.
//
// The products are MFMA's (gemm.h's streamed tiles) and the pass over the codes HBM's. Of 8192 rows and 32000 classes, us: the
// forward product with its store 382 at k = 512 (0.70 PFLOP/s: the store's exponentials and 0.5 GB are as long as the product) and
// 934 at k = 2048 (1.15), codes into d 201 (1.05 GB, 5.2 TB/s), dh 247 and 826 (1.09, 1.30), dw 242 and 927 (1.11, 1.16). Tiles
// of 128 rows, whose stores two workgroups a CU could hide, took the forward product from 391 to 451 and from 970 to 1249.
#pragma once

#include "device_common.h"
#include "gemm.h"

namespace nhipk {

// Where a class's target stands: clamped into the classes, and whether the row is ignored.
struct HeadTargets {
    const void *target;
    int64_t ignore, classes;
    int32_t t64;
    __device__ __forceinline__ int64_t at(int64_t r, bool &ignored) const {
        const int64_t t = t64 ? static_cast<const int64_t *>(target)[r] : static_cast<const int32_t *>(target)[r];
        ignored = t == ignore;
        return t < 0 ? 0 : t >= classes ? classes - 1 : t;
    }
};

constexpr float kHeadUnit = 1.0f / 32768;  // of the codes

// Two values, rounded to nearest.
__device__ __forceinline__ uint32_t head_codes(float a, float b) {
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    const half2 v = {_Float16(a), _Float16(b)};
    return __builtin_bit_cast(uint32_t, v);
}

// What the lanes of a row's two half-waves (lane, lane ^ 32) have, by a register swap.
typedef unsigned head_u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ head_u32x2 head_halves(float x) {
    return __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
}

// The store of the forward product, on a wave's sums in their registers: a lane and the one 32 further hold the 64 logits of a
// row's block, 32 each, in groups of four columns that alternate between them. The block's maximum and sum are 31 operations of
// a lane and one swap; the codes of two groups are swapped into 16 bytes of one row a lane. Columns past the classes
// count for nothing and are stored as zeros up to whole blocks. (Through LDS, four columns of 16 rows a lane at a time and rotations over
// 16 lanes for a row's block, the store took twice the product: [8192, 512] x [32000, 512] 1020 us.)
template <bool GRAD>
struct HeadOut {
    float2 *part;     // [rows, blocks]
    float *picked;    // [rows]
    uint16_t *codes;  // [rows, 64 blocks]
    HeadTargets targets;
    int64_t blocks;
    static constexpr int kPitch = 128 + 16, kStage = 32 * kPitch;  // a block of 32 rows

    template <int FM, int FN>
    __device__ __forceinline__ void store(const GemmShape &s, const f32x16_t (&acc)[FM][FN], char *stage, int64_t rbase, int64_t cbase,
                                          int lane) const {
        constexpr float kLog2e = 1.4426950408889634f;
        const int h = lane >> 5, l32 = lane & 31;
        int64_t cls[FM];
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int64_t r = rbase + 32 * i + l32;
            bool ignored;
            cls[i] = r < s.m ? targets.at(r, ignored) : -1;
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int64_t r = rbase + 32 * i + l32;
#pragma unroll
            for (int b = 0; b < FN / 2; ++b) {
                const int64_t c0 = cbase + 64 * b, block = c0 >> 6;
                if (block >= blocks) continue;  // the whole wave
                float x[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] = acc[i][2 * b + e / 16][e % 16];
                // element e is column c0 + 32 (e / 16) + 8 (e / 4 % 4) + 4 h + e % 4
                const int left = int(min(targets.classes - c0, int64_t(64))) - 4 * h;
                if (c0 + 64 > targets.classes) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * (e / 16) + 8 * (e / 4 % 4) + e % 4 >= left) x[e] = -INFINITY;
                }
                if (__any(cls[i] >= c0 && cls[i] < c0 + 64)) {
                    const int at = int(cls[i] - c0) - 4 * h;
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (at == 32 * (e / 16) + 8 * (e / 4 % 4) + e % 4) picked[r] = x[e];
                }
                float m = x[0];
#pragma unroll
                for (int e = 1; e < 32; ++e) m = fmaxf(m, x[e]);
                const head_u32x2 both = head_halves(m);
                m = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
                // the difference is exact near the maximum, where the terms matter, and no exponential is above 1
                const float ref = m == -INFINITY ? 0.0f : m;
                float sum = 0.0f;
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(x[e] - ref, kLog2e, 15.0f)),
                                q = __builtin_amdgcn_exp2f(fmaf(x[e + 1] - ref, kLog2e, 15.0f));
                    sum += p + q;
                    if constexpr (GRAD) w[e / 2] = head_codes(p, q);
                }
                const head_u32x2 sums = head_halves(sum);
                sum = (__uint_as_float(sums[0]) + __uint_as_float(sums[1])) * kHeadUnit;
                if (r < s.m && h == 0) part[r * blocks + block] = make_float2(m, sum);
                if constexpr (GRAD) {
#pragma unroll
                    for (int g = 0; g < 8; g += 2) {  // groups of eight columns g (the lower half's) and g + 1 (the upper's)
                        const head_u32x2 lo = __builtin_amdgcn_permlane32_swap(w[2 * g], w[2 * g + 2], false, false),
                                         hi = __builtin_amdgcn_permlane32_swap(w[2 * g + 1], w[2 * g + 3], false, false);
                        *reinterpret_cast<uint4 *>(stage + l32 * kPitch + 16 * (g + h)) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int row = 8 * k + lane / 8, chunk = lane % 8;
                        typedef unsigned head_u32x4 __attribute__((ext_vector_type(4)));
                        const head_u32x4 v = *reinterpret_cast<const head_u32x4 *>(stage + row * kPitch + 16 * chunk);
                        const int64_t to = rbase + 32 * i + row;
                        uint16_t *at = codes + to * blocks * 64 + c0 + 8 * chunk;
                        if (to < s.m) __builtin_nontemporal_store(v, reinterpret_cast<head_u32x4 *>(at));
                    }
                }
            }
        }
    }
};
template <bool GRAD>
struct TakesSums<HeadOut<GRAD>> : std::true_type {};

template <bool F16, int TM, bool GRAD>
__global__ __launch_bounds__(TM * 2) __attribute__((amdgpu_waves_per_eu(2, 2))) void head_logits_kernel(
    GemmShape s, const uint16_t *__restrict__ a, const uint16_t *__restrict__ b, HeadOut<GRAD> out) {
    extern __shared__ __align__(1024) char smem[];
    gemm_stream_tile<F16, 64, TM / 64, false, false, true, HeadOut<GRAD>, TM, TM == 256 ? 3 : 0>(s, a, b, out, smem);
}

// exp(x) of a block's or a wave's maximum less a larger one.
__device__ __forceinline__ float head_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// A row's log-sum-exp from its blocks' maxima and sums, by a workgroup: float64 from the blocks on. A block without a term (columns past
// the classes, logits of -inf) has a sum of 0 and is left out by it, not by its maximum: a NaN is in its block's sum and in no
// maximum, which of a block that holds nothing else is -inf.
__device__ __forceinline__ double head_lse(const float2 *__restrict__ p, int64_t blocks) {
    __shared__ float most[4];
    __shared__ double sums[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = -INFINITY;
    for (int64_t j = threadIdx.x; j < blocks; j += 256) m = fmaxf(m, p[j].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    double sum = 0.0;
    for (int64_t j = threadIdx.x; j < blocks; j += 256) {
        const float2 q = p[j];
        if (q.y != 0.0f) sum += double(q.y) * double(head_exp(q.x - m));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) most[wave] = m, sums[wave] = sum;
    __syncthreads();
    const float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (sums[i] != 0.0) sum += sums[i] * double(head_exp(most[i] - top));
    return double(top) + log(sum);
}

// The losses alone. A workgroup a row: 512 rows of 500 blocks 4.2 us (6.3 by a wavefront a row).
static __global__ __launch_bounds__(256) void head_merge_kernel(const float2 *__restrict__ part, const float *__restrict__ picked,
                                                                HeadTargets targets, int64_t rows, int64_t blocks,
                                                                float *__restrict__ losses) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const double lse = head_lse(part + row * blocks, blocks);
        if (threadIdx.x == 0) {
            bool ignored;
            targets.at(row, ignored);
            losses[row] = ignored ? 0.0f : float(lse - double(picked[row]));
        }
        __syncthreads();  // head_lse's LDS is read
    }
}

// Rows of any length, alignment or distance as the products read them: copied to rows of kp elements, zeros past k. `mask`: zeros
// in ignored rows too, whose d of 0 times a NaN or an infinity of theirs would be no 0 in dw.
constexpr int kPrepare = 1024;  // threads
struct HeadCopy {
    const uint16_t *src;
    int64_t rows, ld, k, kp;
    uint16_t *dst;
    int32_t mask, groups;  // workgroups: 0 if nothing is copied
};
__device__ __forceinline__ void head_copy(const HeadCopy &c, const HeadTargets &targets, int group) {
    const int64_t per = c.kp / 8, total = c.rows * per;
    for (int64_t i = int64_t(group) * kPrepare + threadIdx.x; i < total; i += int64_t(c.groups) * kPrepare) {
        const int64_t row = i / per, col = (i - row * per) * 8;
        bool ignored = false;
        if (c.mask) targets.at(row, ignored);
        *reinterpret_cast<uint4 *>(c.dst + row * c.kp + col) =
            col < c.k && !ignored ? load8_any(c.src + row * c.ld + col, c.k - col) : make_uint4(0, 0, 0, 0);
    }
}

// scale[0]: what takes the largest |g| of the rows that count to `top` (1 where it is zero or not finite); scale[1]: one over it.
__device__ __forceinline__ void head_scale(const float *__restrict__ g, const HeadTargets &targets, int64_t rows, float top,
                                           float *__restrict__ scale) {
    __shared__ float most[kPrepare / 64];
    float m = 0.0f;
    constexpr int FLIGHT = 8;
    for (int64_t i = threadIdx.x; i < rows; i += kPrepare * FLIGHT) {
        float v[FLIGHT];
        bool ignored[FLIGHT];
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) {
            const int64_t r = min(i + kPrepare * k, rows - 1);  // the last row again past the rows
            targets.at(r, ignored[k]);
            v[k] = fabsf(g[r]);
        }
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) m = fmaxf(m, ignored[k] ? 0.0f : v[k]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < kPrepare / 64; ++i) m = fmaxf(m, most[i]);
    // within what a float32 and its inverse can be
    m = m > 0.0f && m < INFINITY ? fminf(fmaxf(m, 0x1p-100f), 0x1p100f) : top;
    scale[0] = top / m, scale[1] = m / top;
}

// What comes ahead of the products, in one launch: unless g is null the scale, by the first workgroup, and the copies.
static __global__ __launch_bounds__(kPrepare) void head_prepare_kernel(HeadCopy h, HeadCopy w, const float *__restrict__ g,
                                                                       HeadTargets targets, int64_t rows, float top,
                                                                       float *__restrict__ scale) {
    const int group = int(blockIdx.x) - (g ? 1 : 0);
    if (group < 0) head_scale(g, targets, rows, top, scale);
    else if (group < h.groups) head_copy(h, targets, group);
    else head_copy(w, targets, group - h.groups);
}

// The codes of a piece's rows into d, in place: a workgroup a row (of few rows gridDim.y of them: 118 rows of 21312 classes 6.1 us,
// 10.9 by one each; 271 of 31856 11.2, 17.1), whose lse and loss it works out first, 8 classes a thread at a time. The target's d
// is g expm1(-loss), which p - 1 would cancel. HBM bounds it; codes are read and d written once and are more than the caches hold
// (nontemporal).
template <bool F16>
__global__ __launch_bounds__(256) void head_grad_kernel(uint16_t *__restrict__ codes, const float2 *__restrict__ part,
                                                        const float *__restrict__ picked, const float *__restrict__ g,
                                                        const float *__restrict__ scale, HeadTargets targets, int64_t blocks,
                                                        float *__restrict__ losses) {
    typedef uint32_t words4 __attribute__((ext_vector_type(4)));
    const int64_t row = blockIdx.x;
    const float2 *q = part + row * blocks;
    const double lse = head_lse(q, blocks);
    bool ignored;
    const int64_t cls = targets.at(row, ignored);
    const float l = float(lse), loss = float(lse - double(picked[row])), f = g[row] * scale[0];
    if (losses && threadIdx.x == 0 && blockIdx.y == 0) losses[row] = ignored ? 0.0f : loss;
    uint16_t *p = codes + row * blocks * 64;
    auto round = [](float v) { return uint32_t(F16 ? f32_to_f16(v) : f32_to_bf16(v)); };
    for (int64_t c = 8 * (threadIdx.x + 256 * blockIdx.y); c < blocks * 64; c += 2048 * gridDim.y) {
        words4 o = {0, 0, 0, 0};
        if (!ignored) {
            const words4 w = __builtin_nontemporal_load(reinterpret_cast<const words4 *>(p + c));
            const float k = f * kHeadUnit * head_exp(q[c >> 6].x - l);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i] = round(f16_to_f32(uint16_t(w[i] & 0xffff)) * k) | round(f16_to_f32(uint16_t(w[i] >> 16)) * k) << 16;
            if (cls >= c && cls < c + 8) {
                const uint32_t d = round(f * expm1f(-loss)), at = uint32_t(cls - c), shift = at % 2 * 16;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    if (at / 2 == i) o[i] = (o[i] & ~(0xffffu << shift)) | d << shift;
            }
        }
        __builtin_nontemporal_store(o, reinterpret_cast<words4 *>(p + c));
    }
}

// The store of a gradient's product: the float32 sums of the pieces before added, then kept as sums or rounded into the result.
struct HeadStore {
    const float *before;  // null: none
    float *sums;          // null: this is the last piece
    uint16_t *out;
    const float *inverse;  // what the products are multiplied by
    int64_t n;             // columns, a row's elements too
    int32_t f16;
    static constexpr int kPrefetch = 8;
    static constexpr bool kColSum = false;
    struct Pre {
        float4 v;
    };
    __device__ __forceinline__ Pre load(int64_t r, int64_t c) const {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (before) {
            const float *p = before + r * n + c;
            if (n % 4 == 0) v = *reinterpret_cast<const float4 *>(p);
            else v = make_float4(p[0], c + 1 < n ? p[1] : 0.0f, c + 2 < n ? p[2] : 0.0f, c + 3 < n ? p[3] : 0.0f);
        }
        return Pre{v};
    }
    __device__ __forceinline__ void operator()(int64_t r, int64_t c, float4 x, const Pre &pre) const {
        float e[4] = {x.x + pre.v.x, x.y + pre.v.y, x.z + pre.v.z, x.w + pre.v.w};
        if (sums) {
            float *p = sums + r * n + c;
            if (n % 4 == 0) *reinterpret_cast<float4 *>(p) = make_float4(e[0], e[1], e[2], e[3]);
            else
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < n) p[i] = e[i];
            return;
        }
        const float k = *inverse;
        uint16_t *p = out + r * n + c;
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = f16 ? f32_to_f16(e[i] * k) : f32_to_bf16(e[i] * k);
        if (n % 4 == 0) *reinterpret_cast<uint2 *>(p) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < n) p[i] = uint16_t(b[i]);
    }
};

// dh = d w over a piece's rows: d in whole blocks of classes, w's rows as they lie, those past v read as zeros.
template <bool F16, int TM, int ST, class Out>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(ST == 2 ? 2 : 1, ST == 2 ? 2 : 1))) void head_input_grad(
    GemmShape s, const uint16_t *__restrict__ d, const uint16_t *__restrict__ w, Out out, int k_part) {
    extern __shared__ __align__(1024) char smem[];
    gemm_stream_tile<F16, 64, 2, false, true, true, Out, TM, TM == 256 ? 3 : ST == 3 ? 1 : 0, 5, TM == 256 ? 0 : ST>(s, d, w, out, smem,
                                                                                                                  nullptr, k_part);
}

// dw = d^T h over a piece's rows.
template <bool F16, int TM, int ST, class Out>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(ST == 2 ? 2 : 1, ST == 2 ? 2 : 1))) void head_weight_grad(
    GemmShape s, const uint16_t *__restrict__ d, const uint16_t *__restrict__ h, Out out, int k_part) {
    extern __shared__ __align__(1024) char smem[];
    gemm_stream_tile<F16, 64, 2, true, true, true, Out, TM, TM == 256 ? 3 : ST == 3 ? 1 : 0, 3, TM == 256 ? 0 : ST>(s, d, h, out, smem,
                                                                                                                  nullptr, k_part);
}

// Both in one launch, for products whose workgroups fit the chip together, two a CU: dh's in parts first, then dw's whole. (As two
// rows of a grid as wide and deep as either needs, the empty workgroups, which hold LDS too, cost up to 10 us.)
template <class InOut>
struct HeadBoth {
    GemmShape input, weight;
    const uint16_t *w, *h;
    InOut input_out;
    HeadStore weight_out;
    int32_t parts, input_part, weight_part;  // k tiles of a part, and of all dw's
};
template <bool F16, class InOut>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void head_both_grads(HeadBoth<InOut> x,
                                                                                                  const uint16_t *__restrict__ d) {
    extern __shared__ __align__(1024) char smem[];
    const uint32_t tiles = uint32_t(x.input.tiles_m) * uint32_t(x.input.tiles_n), at = blockIdx.x, input = tiles * uint32_t(x.parts);
    if (at < input)
        gemm_stream_tile<F16, 64, 2, false, true, true, InOut, 128, 0, 5, 2>(x.input, d, x.w, x.input_out, smem, nullptr, x.input_part,
                                                                             at % tiles, at / tiles);
    else
        gemm_stream_tile<F16, 64, 2, true, true, true, HeadStore, 128, 0, 3, 2>(x.weight, d, x.h, x.weight_out, smem, nullptr,
                                                                                x.weight_part, at - input, 0);
}

// Float32 sums of a product's parts, P[part][mn], added in order and stored as HeadStore stores a tile (of one row).
static __global__ __launch_bounds__(256) void head_sum_kernel(const float *__restrict__ part, int parts, int64_t mn, HeadStore out) {
    out.n = mn;
    for (int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4; i < mn; i += int64_t(gridDim.x) * 1024) {
        float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < parts; ++k) {
            const float *p = part + k * mn + i;
            if (mn % 4 == 0) {
                const float4 v = *reinterpret_cast<const float4 *>(p);
                e[0] += v.x, e[1] += v.y, e[2] += v.z, e[3] += v.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < mn) e[j] += p[j];
            }
        }
        out(0, i, make_float4(e[0], e[1], e[2], e[3]), out.load(0, i));
    }
}

}  // namespace nhipk

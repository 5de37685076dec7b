// The gate and up projections of a gated MLP with the activation and the product in their store:
//
//   h[t, f] = act(g) u,  g = sum over k of x[t, k] gate[f, k],  u = sum over k of x[t, k] up[f, k]
//
// for bf16/f16 x [m, k] and weights [n, k], all contiguous along k. MFMA bounds it (4 m n k operations); the two products
// share x, and computing both of an element's sums in one lane means that neither g nor u need be written: 2 m n elements
// not stored and not read again. The sums stay float32 until h is rounded, once. In training the backward needs g and u,
// which are then stored too, in float32: rounded to 16 bits they would be the largest error of the gradients (three
// roundings on the way to dx instead of two). At [4096, 2048] x [8192, 2048] writing and reading them, 16 m n bytes, are 105
// us at a copy's rate, 16% of the six products' 660; in 16 bits they would be half of that, and to compute them again in the
// backward, two of the six products, twice.
//
// Kernels (gated_default chooses):
//  * gated_stream: gemm_stream_tile with PAIR 1, tiles of 256 rows x 128 columns or 128 x 64; rows that it cannot read in
//    place (no multiple of 8 elements, off 16 bytes) are copied first (gated_pad_kernel);
//  * gated_stream_part and gated_join_kernel: the 128 x 64 tiles over parts of k, where there are few of them;
//  * gated_skinny: at most 64 rows, 16 columns a workgroup, the waves divide k (as gemm_skinny).
// At [16384, 2048] x 2 [8192, 2048] 892 to 925 us by card and clock, 1.19 to 1.23 PFLOP/s, what a plain product of these sizes
// reaches; at [16, 2048], 67 MB of weights, 13.3 us (5.1 TB/s).
//
// The backward's elementwise half (gated_grad_kernel) turns dh, g and u into [dg | du], one row of 2 n a token, HBM-bound:
//   du = dh act(g), dg = dh u act'(g)
// so that [dg | du] is the operand of one product for both weight gradients and of one for dx. It is rounded to 16 bits, which
// the matrix instructions take: gradients in bf16 are 0.0023 off the 64-bit ones, with a float32 [dg | du] 0.0017 (f16 0.00029,
// 0.00021); in two terms of 16 bits it would cost every product of the backward twice.
#pragma once

#include "gemm.h"
#include "gemm_skinny.h"

namespace nhipk {

enum { kGatedSilu = 0, kGatedGelu = 1, kGatedRelu = 2, kGatedSigmoid = 3 };

constexpr float kLog2e = 1.44269504088896341f;

// 1 / (1 + exp(-x)): x = -inf gives 0, +inf 1, NaN NaN.
__device__ __forceinline__ float gated_sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * x));
}

// GELU's tanh form written as a sigmoid: (1 + tanh(v)) / 2 = 1 / (1 + exp(-2 v)).
constexpr float kGeluC = 0.7978845608f, kGeluA = 0.044715f;

__device__ __forceinline__ float gated_act(int act, float g) {
    if (act == kGatedSilu) return g * gated_sigmoid(g);
    if (act == kGatedGelu) return g * gated_sigmoid(2.0f * kGeluC * (g + kGeluA * g * g * g));
    if (act == kGatedRelu) return g <= 0.0f ? 0.0f : g;  // a NaN stays
    return gated_sigmoid(g);
}

// act(g) and its derivative.
__device__ __forceinline__ void gated_act_grad(int act, float g, float &a, float &da) {
    if (act == kGatedSilu) {
        const float s = gated_sigmoid(g);
        a = g * s;
        da = s * (1.0f + g * (1.0f - s));
    } else if (act == kGatedGelu) {
        const float s = gated_sigmoid(2.0f * kGeluC * (g + kGeluA * g * g * g));
        a = g * s;
        const float t = a * (1.0f - s) * (2.0f * kGeluC);  // 0 for large g, and g * g may be infinite
        da = s + t + 3.0f * kGeluA * (t * g) * g;
    } else if (act == kGatedRelu) {
        a = g <= 0.0f ? 0.0f : g;
        da = g > 0.0f ? 1.0f : 0.0f;
    } else {
        a = gated_sigmoid(g);
        da = a * gated_sigmoid(-g);  // 1 - a would cancel: at g = 10 it is off by 1e-3 of itself
    }
}

// Where a kernel's sums go: h (16-bit, rows h_m apart), and g and u (float32, [m, n]) unless null.
struct GatedOut {
    void *h;
    float *g, *u;
    int32_t act, dtype;  // dtype: 1 bf16, 2 f16

    // One element, for the kernels that store from registers.
    __device__ __forceinline__ void one(const GemmShape &s, int64_t row, int64_t col, float gv, float uv) const {
        const float v = gated_act(act, gv) * uv;
        uint16_t *p = static_cast<uint16_t *>(h) + row * s.d_m + col;
        *p = dtype == 1 ? f32_to_bf16(v) : f32_to_f16(v);
        if (g) {
            g[row * s.n + col] = gv;
            u[row * s.n + col] = uv;
        }
    }

    template <int FM, int FN, int WCOLS>
    __device__ __forceinline__ void store(const GemmShape &s, const f32x16_t (&acc)[FM][FN], char *stage, int64_t rbase,
                                          int64_t cbase, int lane) const;
};

// The sums of part blockIdx.z of k, for gated_join_kernel: sums [parts][g, u][m, n].
struct GatedParts {
    float *sums;
    template <int FM, int FN, int WCOLS>
    __device__ __forceinline__ void store(const GemmShape &s, const f32x16_t (&acc)[FM][FN], char *stage, int64_t rbase,
                                          int64_t cbase, int lane) const;
};

// The wave's LDS writes before its reads of them, and the other way round.
__device__ __forceinline__ void gated_wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Stores value(g, u) of 64 rows (half `half`) of one wave's sums: acc[i][j] and acc[i][j + FN / 2] hold g and u of the same
// elements, row 32 i + l32, column 32 j + 8 (e / 4) + 4 (lane / 32) + e % 4. Through the wave's own LDS rows, so that rows go
// out in 16-byte pieces; only this wave writes and reads them, which needs no barrier.
template <int FM, int FN, int WCOLS, class Value>
__device__ __forceinline__ void gated_store_half(const f32x16_t (&acc)[FM][FN], int half, Value &&value, const GemmShape &shape,
                                                 const AnyStore &to, char *stage, int64_t rbase, int64_t cbase, int lane) {
    constexpr int WC = WCOLS / 2, P = WC * 4 + 16;
    const int l32 = lane & 31, hl = lane >> 5;
#pragma unroll
    for (int ii = 0; ii < 2; ++ii)
#pragma unroll
        for (int j = 0; j < FN / 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const f32x16_t &g_ = acc[2 * half + ii][j], &u_ = acc[2 * half + ii][j + FN / 2];
                *reinterpret_cast<float4 *>(stage + (32 * ii + l32) * P + (32 * j + 2 * e + 4 * hl) * 4) =
                    make_float4(value(g_[e], u_[e]), value(g_[e + 1], u_[e + 1]), value(g_[e + 2], u_[e + 2]),
                                value(g_[e + 3], u_[e + 3]));
                __builtin_amdgcn_sched_barrier(0);
            }
    gated_wave_order();
    stream_store_dense<WC, P>(shape, to, 0, stage, rbase + 64 * half, cbase, lane);
    gated_wave_order();
}

template <int FM, int FN, int WCOLS>
__device__ __forceinline__ void GatedOut::store(const GemmShape &s, const f32x16_t (&acc)[FM][FN], char *stage, int64_t rbase,
                                                int64_t cbase, int lane) const {
    GemmShape full = s;  // of g and u
    full.d_m = s.n;
    auto out = [&](int half, auto value, const GemmShape &shape, const AnyStore &to) {
        gated_store_half<FM, FN, WCOLS>(acc, half, value, shape, to, stage, rbase, cbase, lane);
    };
#pragma unroll
    for (int half = 0; half < FM / 2; ++half) {
        if (g) {
            out(half, [](float a, float) { return a; }, full, AnyStore{g, 0});
            out(half, [](float, float b) { return b; }, full, AnyStore{u, 0});
        }
        // the activation is the same for every element: its branch is taken once
        if (act == kGatedSilu) out(half, [](float a, float b) { return gated_act(kGatedSilu, a) * b; }, s, AnyStore{h, dtype});
        else if (act == kGatedGelu) out(half, [](float a, float b) { return gated_act(kGatedGelu, a) * b; }, s, AnyStore{h, dtype});
        else if (act == kGatedRelu) out(half, [](float a, float b) { return gated_act(kGatedRelu, a) * b; }, s, AnyStore{h, dtype});
        else out(half, [](float a, float b) { return gated_act(kGatedSigmoid, a) * b; }, s, AnyStore{h, dtype});
    }
}

template <int FM, int FN, int WCOLS>
__device__ __forceinline__ void GatedParts::store(const GemmShape &s, const f32x16_t (&acc)[FM][FN], char *stage, int64_t rbase,
                                                  int64_t cbase, int lane) const {
    float *g = sums + int64_t(blockIdx.z) * 2 * s.m * s.n, *u = g + s.m * s.n;
#pragma unroll
    for (int half = 0; half < FM / 2; ++half) {
        gated_store_half<FM, FN, WCOLS>(acc, half, [](float a, float) { return a; }, s, AnyStore{g, 0}, stage, rbase, cbase, lane);
        gated_store_half<FM, FN, WCOLS>(acc, half, [](float, float b) { return b; }, s, AnyStore{u, 0}, stage, rbase, cbase, lane);
    }
}

// TM x TM / 2 tiles: 256 with 8 waves and the k loop placed by hand (with 4 waves the store's 512 registers spill: [16384, 2048] x
// [8192, 2048] 909 us, 1140), 128 with 4 waves, two workgroups a CU.
// KL, ST: the k loop and its stages: 3 (256), 0 with two stages (128), or 1 with three (128, one workgroup a CU): where the
// tiles leave one workgroup a CU anyway and k is long enough, its loads two tiles ahead hide their latency ([128, 2048] x [8192, 2048]
// 27.4 -> 19.6 us, [1463, 3392] x [712, 3392] 41.2 -> 28.9; [300, 512] x [2048, 512] 7.8 -> 8.4).
template <bool F16, int TM, int KL, int ST = 0>
__global__ __launch_bounds__(TM * 2) __attribute__((amdgpu_waves_per_eu(ST ? 1 : 2, ST ? 1 : 2))) void gated_stream(
    GemmShape s, const uint16_t *__restrict__ x, const uint16_t *__restrict__ gate, const uint16_t *__restrict__ up,
    GatedOut out) {
    extern __shared__ __align__(1024) char smem[];
    gemm_stream_tile<F16, 64, TM / 64, false, false, true, GatedOut, TM, KL, 1, ST>(s, x, gate, out, smem, up);
}

// The deep tiles over part blockIdx.z of k (k_part of its k tiles): few tiles of a long k leave CUs idle, and a tile's k loop
// is all latency ([139, 3840] x [1464, 3840], 46 tiles: 30.1 us whole, 18.1 in 4 parts and their join).
template <bool F16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void gated_stream_part(
    GemmShape s, const uint16_t *__restrict__ x, const uint16_t *__restrict__ gate, const uint16_t *__restrict__ up,
    GatedParts out, int k_part) {
    extern __shared__ __align__(1024) char smem[];
    gemm_stream_tile<F16, 64, 2, false, false, true, GatedParts, 128, 1, 4, 3>(s, x, gate, out, smem, up, k_part);
}

// g and u as the sums of their parts, in order, and h of them, V elements a thread.
template <int V>
__global__ __launch_bounds__(256) void gated_join_kernel(GemmShape s, const float *__restrict__ sums, int parts, GatedOut out) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const int64_t mn = s.m * s.n, per = s.n / V;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < s.m * per; i += int64_t(gridDim.x) * 256) {
        const float *p = sums + i * V;
        vec g = *reinterpret_cast<const vec *>(p), u = *reinterpret_cast<const vec *>(p + mn);
#pragma unroll 4
        for (int k = 1; k < parts; ++k) {
            g += *reinterpret_cast<const vec *>(p + 2 * k * mn);
            u += *reinterpret_cast<const vec *>(p + (2 * k + 1) * mn);
        }
        const int64_t row = i / per, col = (i - row * per) * V;
#pragma unroll
        for (int k = 0; k < V; ++k) out.one(s, row, col + k, g[k], u[k]);
    }
}

// 8 elements at p of any alignment as 4-byte words, which memory reads at full width where words at 2-byte addresses take
// several passes (one row of [1, 2047] x 2 [8192, 2047]: 31.7 us so, 20.6 with words; [64, 2047] 81, 40): the words that hold them, 5 of
// them where p is in a word's middle, and no others, so no read leaves the words that the row lies in.
__device__ __forceinline__ uint4 load8_words(const uint16_t *p) {
    typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(4)));
    const uint32_t odd = uint32_t(reinterpret_cast<uintptr_t>(p)) & 2;
    const uint32_t *q = reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(p) - odd);
    const words4 v = *reinterpret_cast<const words4 *>(q);
    const uint32_t last = q[odd ? 4 : 3], shift = odd * 8;
    return make_uint4(__builtin_amdgcn_alignbit(v[1], v[0], shift), __builtin_amdgcn_alignbit(v[2], v[1], shift),
                      __builtin_amdgcn_alignbit(v[3], v[2], shift), __builtin_amdgcn_alignbit(last, v[3], shift));
}

// Few rows: a workgroup takes 16 columns of both weights, its NW waves divide k 64 at a time, fragments straight from
// memory (v_mfma_f32_16x16x32: 16 rows of 64 contiguous bytes), the waves' sums added through LDS in wave order. Reading
// the weights once is all the work.
// ANY: rows of any length and alignment.
template <bool F16, int MT, int NW, bool ANY>
__global__ __launch_bounds__(64 * NW) void gated_skinny(GemmShape s, const uint16_t *__restrict__ x,
                                                         const uint16_t *__restrict__ gate, const uint16_t *__restrict__ up,
                                                         GatedOut out) {
    constexpr int U = MT == 1 ? 2 : 1;  // chunks of 64 k in flight
    __shared__ f32x4_t sums[NW][2][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    auto get = [](const uint16_t *p) {
        if constexpr (ANY) return load8_words(p);
        else return *reinterpret_cast<const uint4 *>(p);
    };
    const int64_t n0 = int64_t(blockIdx.x) * 16;
    // rows past the last one: the last one again, never stored
    const int64_t row = min(n0 + l16, s.n - 1) * s.b_n + 8 * g;
    const uint16_t *pb[2] = {gate + row, up + row};
    const uint16_t *pa[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) pa[i] = x + min(int64_t(16 * i + l16), s.m - 1) * s.a_m + 8 * g;

    f32x4_t acc[2][MT];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[w][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const int k = int(s.k), step = 64 * NW;
    int k0 = 64 * wave;
    for (; k0 + (U - 1) * step + 64 <= k; k0 += U * step) {
        uint4 fb[U][2][2], fa[U][2][MT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int w = 0; w < 2; ++w) fb[u][c][w] = get(pb[w] + k0 + u * step + 32 * c);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < MT; ++i) fa[u][c][i] = get(pa[i] + k0 + u * step + 32 * c);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int i = 0; i < MT; ++i) acc[w][i] = mfma16<F16>(fa[u][c][i], fb[u][c][w], acc[w][i]);
    }
    for (; k0 < k; k0 += step)  // the last chunks, a lane's 8 k past the end as zeros
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int left = k - (k0 + 32 * c + 8 * g);
            auto tail = [&](const uint16_t *p) {
                if constexpr (ANY)
                    return left >= 8 ? load8_words(p + k0 + 32 * c) : left > 0 ? load8_any(p + k0 + 32 * c, left) : make_uint4(0, 0, 0, 0);
                else return left > 0 ? get(p + k0 + 32 * c) : make_uint4(0, 0, 0, 0);
            };
            const uint4 f0 = tail(pb[0]), f1 = tail(pb[1]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const uint4 fa = tail(pa[i]);
                acc[0][i] = mfma16<F16>(fa, f0, acc[0][i]);
                acc[1][i] = mfma16<F16>(fa, f1, acc[1][i]);
            }
        }
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < MT; ++i) sums[wave][w][i][lane] = acc[w][i];
    __syncthreads();
    // C layout of a 16 x 16 block: lane holds column lane % 16, rows 4 (lane / 16) + e
    if (wave >= MT) return;
    f32x4_t gv = sums[0][0][wave][lane], uv = sums[0][1][wave][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) gv += sums[w][0][wave][lane], uv += sums[w][1][wave][lane];
    const int64_t col = n0 + l16, r0 = 16 * wave + 4 * g;
    if (col >= s.n) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (r0 + e < s.m) out.one(s, r0 + e, col, gv[e], uv[e]);
}

// Rows of any length, alignment or distance, as gated_stream reads them: each of x's m rows and the weights' 2 n copied to
// rows of kp = k rounded up to 8 elements, 16 bytes a thread, zeros past k, a matrix each blockIdx.y. A pass over the operands that a product of many
// rows hides and one of few rows does not need (gated_skinny reads any rows): [16384, 2047] x [8192, 2047] 60 of 970 us.
struct GatedPad {
    const uint16_t *src[3];
    uint16_t *dst[3];
    int64_t rows[3], to_rows[3], ld[3], k, kp;  // to_rows: rows written, those past `rows` zeros
};
static __global__ __launch_bounds__(256) void gated_pad_kernel(GatedPad a) {
    const int which = blockIdx.y;
    const int64_t per = a.kp / 8, total = a.to_rows[which] * per;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / per, c = (i - row * per) * 8;
        const uint16_t *src = a.src[which] + row * a.ld[which] + c;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < a.rows[which]) v = a.k - c >= 8 ? load8_words(src) : load8_any(src, a.k - c);
        *reinterpret_cast<uint4 *>(a.dst[which] + row * a.kp + c) = v;
    }
}

// The input's gradient: D = A[:, :k / 2] B + A[:, k / 2:] B2 with A = [dg | du] and the weights as they lie: one
// accumulator over both products, or (parts of k) float32 sums that gated_sum_kernel adds. Two products and their sum write
// and read 8 m n bytes more: [4096, 2048] of k 2 x 8192 243 us, 325.
// ST: 0 (tiles of 256, a workgroup a CU), 2 (128, two a CU) or 3 stages (128, one a CU, loads two tiles ahead).
template <bool F16, int TM, int ST>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(ST == 2 ? 2 : 1, ST == 2 ? 2 : 1))) void gated_input_grad(
    GemmShape s, const uint16_t *__restrict__ a, const uint16_t *__restrict__ b, const uint16_t *__restrict__ b2, AnyStore out,
    int k_part) {
    extern __shared__ __align__(1024) char smem[];
    gemm_stream_tile<F16, 64, 2, false, true, true, AnyStore, TM, TM == 256 ? 3 : ST == 3 ? 1 : 0, 2, TM == 256 ? 0 : ST>(s, a, b, out, smem, b2, k_part);
}

// The weights' gradients: D_i = A_i^T X for the two halves of A = [dg | du], one batch each, over tokens of any number.
template <bool F16, int TM, int ST>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(ST == 2 ? 2 : 1, ST == 2 ? 2 : 1))) void gated_weight_grad(
    GemmShape s, const uint16_t *__restrict__ a, const uint16_t *__restrict__ b, const uint16_t *, AnyStore out, int k_part) {
    extern __shared__ __align__(1024) char smem[];
    gemm_stream_tile<F16, 64, 2, true, true, true, AnyStore, TM, TM == 256 ? 3 : ST == 3 ? 1 : 0, 3, TM == 256 ? 0 : ST>(s, a, b, out, smem, nullptr, k_part);
}

// Both in one launch, for products that leave most of the chip idle: the input's as batch gridDim.y - 1, the weights' as the
// others, each over its own tiles and parts, a workgroup a CU at most in all ([777, 520] x 2 [1416, 520]: 14.8 and 13.7 us apart, 21.8
// together; the call in both directions 50.4 -> 43.9).
struct GatedHalf {
    GemmShape s;
    const uint16_t *b;
    AnyStore out;
    int32_t k_part, parts;
};
template <bool F16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void gated_both_grads(
    GatedHalf in, GatedHalf wt, const uint16_t *__restrict__ a, const uint16_t *__restrict__ up) {
    extern __shared__ __align__(1024) char smem[];
    const bool input = blockIdx.y == gridDim.y - 1;
    // values, not the chosen argument's address, which would put both in scratch memory
    const int tiles = input ? in.s.tiles_m * in.s.tiles_n : wt.s.tiles_m * wt.s.tiles_n, parts = input ? in.parts : wt.parts;
    if (int(blockIdx.x) >= tiles || int(blockIdx.z) >= parts) return;
    if (input) gemm_stream_tile<F16, 64, 2, false, true, true, AnyStore, 128, 1, 2, 3>(in.s, a, in.b, in.out, smem, up, in.k_part);
    else gemm_stream_tile<F16, 64, 2, true, true, true, AnyStore, 128, 1, 3, 3>(wt.s, a, wt.b, wt.out, smem, nullptr, wt.k_part);
}

// Float32 sums of the parts, P[part][z][mn], added in order and rounded once into result z (blockIdx.y). V elements a thread:
// four where the size and the results' alignment allow (2 parts of [4096, 2048] in 16.5 us, one a thread 24.8).
struct GatedSum {
    const float *part;
    void *out[2];
    int64_t mn;
    int32_t parts;
};
template <typename T, int V>
__global__ __launch_bounds__(256) void gated_sum_kernel(GatedSum a) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const int64_t step = int64_t(gridDim.y) * a.mn, first = int64_t(blockIdx.y) * a.mn;
    T *out = static_cast<T *>(a.out[blockIdx.y]);
    for (int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * V; i < a.mn; i += int64_t(gridDim.x) * 256 * V) {
        const float *p = a.part + first + i;
        vec v = *reinterpret_cast<const vec *>(p);
#pragma unroll 4
        for (int k = 1; k < a.parts; ++k) v += *reinterpret_cast<const vec *>(p + k * step);
        T r[V];
#pragma unroll
        for (int k = 0; k < V; ++k) store_f32_as(&r[k], v[k]);
        if constexpr (V == 4) {
            uint2 w;
            __builtin_memcpy(&w, r, 8);
            *reinterpret_cast<uint2 *>(out + i) = w;
        } else {
            out[i] = r[0];
        }
    }
}

// [dg | du] of 8 elements a thread. ANY: n, dh's rows or a pointer no multiple of 16 bytes (of [929, 5550] 13.8 us; one element
// a thread 14.7). Each half of a row of [dg | du] has np elements, n rounded up to 8, the last ones zeros: the
// products read whole chunks.
struct GatedGrad {
    const void *dh;
    const float *g, *u;
    void *out;  // [m, 2 np]
    int64_t m, n, np, dh_m;
    int32_t act;
};
template <typename T, bool ANY>
__global__ __launch_bounds__(256) void gated_grad_kernel(GatedGrad a) {
    typedef float vec16 __attribute__((ext_vector_type(4)));
    typedef float vec4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef std::conditional_t<ANY, vec4, vec16> vec;
    const int64_t per = a.np / 8, total = a.m * per;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / per, col = (i - row * per) * 8, left = a.n - col;
        const uint16_t *dh = static_cast<const uint16_t *>(a.dh) + row * a.dh_m + col;
        const float *g = a.g + row * a.n + col, *u = a.u + row * a.n + col;
        uint4 r;
        float gv[8], uv[8];
        if (!ANY || left >= 8) {
            if constexpr (ANY) r = load8_words(dh);
            else r = *reinterpret_cast<const uint4 *>(dh);
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                const vec p = *reinterpret_cast<const vec *>(g + k), q = *reinterpret_cast<const vec *>(u + k);
#pragma unroll
                for (int e = 0; e < 4; ++e) gv[k + e] = p[e], uv[k + e] = q[e];
            }
        } else {  // the row's last chunk: zeros past it
            r = load8_any(dh, left);
#pragma unroll
            for (int k = 0; k < 8; ++k) gv[k] = k < left ? g[k] : 0.0f, uv[k] = k < left ? u[k] : 0.0f;
        }
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        T dg[8], du[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const T bits{uint16_t(w[k / 2] >> (k % 2 * 16))};
            const float d = load_as_f32(&bits);
            float act, grad;
            gated_act_grad(a.act, gv[k], act, grad);
            store_f32_as(&dg[k], d * uv[k] * grad);
            store_f32_as(&du[k], d * act);
        }
        uint4 p, q;
        __builtin_memcpy(&p, dg, 16);
        __builtin_memcpy(&q, du, 16);
        T *out = static_cast<T *>(a.out) + row * 2 * a.np + col;
        *reinterpret_cast<uint4 *>(out) = p;
        *reinterpret_cast<uint4 *>(out + a.np) = q;
    }
}

}  // namespace nhipk

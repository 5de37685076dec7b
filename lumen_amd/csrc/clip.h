// The 2-norm over many gradients, and the gradients scaled by it:
//
//   norm = sqrt(sum over tensors and elements of g^2), scale = min(1, max_norm / (norm + eps)), out = g * scale
//
// HBM bounds both halves: every gradient is read for the norm and read again to be scaled, since the scale is known only
// after the last of them. Two launches whatever the number of tensors (to kClipTensors a launch): workgroups walk
// chunks of kClipChunk elements over all the tensors, which a table in the kernel's arguments maps to a tensor by
// binary search, so many small gradients cost no more than one large one and the table needs no copy to the device.
// The second launch walks the chunks backwards, the ones that the caches still hold first.
// 59 bf16 gradients of 950 MB: 183 us (5.2 TB/s) and 343 us (5.5 TB/s read and written); 26 of 83 MB, which the caches hold,
// 15.4 and 27.3; 15 of 1.3 MB 4.9 and 5.5.
//
// Squares are summed in float64: no gradient's square overflows or underflows, and the sum's order does not show in the
// float32 norm. Each workgroup of the first launch leaves one sum; every workgroup of the second adds all of them up
// itself, in the same order, instead of a third launch. No atomics: the same bits every run.
#pragma once

#include "device_common.h"

namespace nhipk {

constexpr int kClipTensors = 120;      // a launch's table within the 4 KiB of kernel arguments
constexpr int kClipBlocks = 1024;      // workgroups of a launch's sums: four a CU
constexpr int64_t kClipChunk = 16384;  // elements: 64 a thread

struct ClipTable {
    const void *in[kClipTensors];
    void *out[kClipTensors];
    int64_t numel[kClipTensors];
    uint32_t first[kClipTensors + 1];  // each tensor's first chunk; the last entry their count
    uint8_t dtype[kClipTensors];       // 0 float32, 1 bf16, 2 f16
    int32_t tensors;
    uint32_t blocks;
};
static_assert(sizeof(ClipTable) + 64 <= 4096, "a launch's arguments");

// The tensor that chunk c lies in: the last whose first chunk is at most c (empty tensors have no chunk).
__device__ __forceinline__ int clip_tensor(const ClipTable &t, uint32_t c) {
    int lo = 0, hi = t.tensors;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ float clip_up(bf16_t, uint32_t bits) { return bf16_to_f32(uint16_t(bits)); }
__device__ __forceinline__ float clip_up(f16_t, uint32_t bits) { return f16_to_f32(uint16_t(bits)); }
__device__ __forceinline__ uint32_t clip_down(bf16_t, float v) { return f32_to_bf16(v); }
__device__ __forceinline__ uint32_t clip_down(f16_t, float v) { return f32_to_f16(v); }

// Elements of 16 bytes.
template <typename T>
struct ClipVec;
template <>
struct ClipVec<float> {
    static constexpr int n = 4;
    __device__ __forceinline__ static void get(const uint4 &r, float (&v)[4]) {
        v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
    }
    __device__ __forceinline__ static uint4 put(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <typename T>
struct ClipVec16 {
    static constexpr int n = 8;
    __device__ __forceinline__ static void get(const uint4 &r, float (&v)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = clip_up(T{}, w[i] & 0xffff), v[2 * i + 1] = clip_up(T{}, w[i] >> 16);
    }
    __device__ __forceinline__ static uint4 put(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = clip_down(T{}, v[2 * i]) | clip_down(T{}, v[2 * i + 1]) << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct ClipVec<bf16_t> : ClipVec16<bf16_t> {};
template <>
struct ClipVec<f16_t> : ClipVec16<f16_t> {};

constexpr int kClipFlight = 4;  // 16-byte reads of a thread in flight

// Calls vec(offset of 16 aligned bytes, raw) and one(offset) for every element of [0, n) of p between them, n at most a
// chunk: 16 bytes at a time where p and the second pointer q are aligned to them, the rest element by element.
template <typename T, class Vec, class One>
__device__ __forceinline__ void clip_walk(const T *p, const void *q, int n, Vec &&vec, One &&one) {
    constexpr int E = ClipVec<T>::n;
    const int lanes = 256, t = threadIdx.x;
    int head = 0;
    if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15) == 0) {
        const uint4 *src = reinterpret_cast<const uint4 *>(p);
        const int chunks = n / E;
        int i = t;
        for (; i + (kClipFlight - 1) * lanes < chunks; i += kClipFlight * lanes) {
            uint4 r[kClipFlight];
#pragma unroll
            for (int k = 0; k < kClipFlight; ++k) r[k] = src[i + k * lanes];
#pragma unroll
            for (int k = 0; k < kClipFlight; ++k) vec(i + k * lanes, r[k]);
        }
        for (; i < chunks; i += lanes) vec(i, src[i]);
        head = chunks * E;
    }
    for (int i = head + t; i < n; i += lanes) one(i);
}

template <typename T>
__device__ __forceinline__ double clip_squares(const void *in, int64_t at, int n) {
    const T *p = static_cast<const T *>(in) + at;
    double sum = 0.0;
    clip_walk<T>(p, nullptr, n,
                 [&](int, const uint4 &r) {
                     float v[ClipVec<T>::n];
                     ClipVec<T>::get(r, v);
#pragma unroll
                     for (int i = 0; i < ClipVec<T>::n; ++i) sum = __builtin_fma(double(v[i]), double(v[i]), sum);
                 },
                 [&](int i) {
                     const double v = load_as_f32(p + i);
                     sum = __builtin_fma(v, v, sum);
                 });
    return sum;
}

// Sum over the workgroup's 256 threads, the same for every thread.
__device__ __forceinline__ double clip_block_sum(double v) {
    __shared__ double sums[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

__global__ __launch_bounds__(256) void clip_squares_kernel(ClipTable t, double *__restrict__ part) {
    double sum = 0.0;
    const uint32_t chunks = t.first[t.tensors];
    for (uint32_t c = blockIdx.x; c < chunks; c += t.blocks) {
        const int k = clip_tensor(t, c);
        const int64_t at = int64_t(c - t.first[k]) * kClipChunk, left = t.numel[k] - at;
        const int n = int(left < kClipChunk ? left : kClipChunk);
        if (t.dtype[k] == 0) sum += clip_squares<float>(t.in[k], at, n);
        else if (t.dtype[k] == 1) sum += clip_squares<bf16_t>(t.in[k], at, n);
        else sum += clip_squares<f16_t>(t.in[k], at, n);
    }
    sum = clip_block_sum(sum);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

template <typename T>
__device__ __forceinline__ void clip_scaled(const void *in, void *out, int64_t at, int n, float scale) {
    const T *p = static_cast<const T *>(in) + at;
    T *q = static_cast<T *>(out) + at;
    clip_walk<T>(p, q, n,
                 [&](int i, const uint4 &r) {
                     float v[ClipVec<T>::n];
                     ClipVec<T>::get(r, v);
#pragma unroll
                     for (int j = 0; j < ClipVec<T>::n; ++j) v[j] *= scale;
                     reinterpret_cast<uint4 *>(q)[i] = ClipVec<T>::put(v);
                 },
                 [&](int i) { store_f32_as(q + i, load_as_f32(p + i) * scale); });
}

// parts: the sums of every launch of clip_squares_kernel. max_at (or null: max_norm) is the bound on the device.
__global__ __launch_bounds__(256) void clip_scale_kernel(ClipTable t, const double *__restrict__ part, int parts,
                                                         const double *__restrict__ max_at, double max_norm, double eps,
                                                         float *__restrict__ norm_out, float *__restrict__ scale_out) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) sum += part[i];
    const double norm = sqrt(clip_block_sum(sum));
    double s = (max_at ? *max_at : max_norm) / (norm + eps);
    if (s > 1.0) s = 1.0;  // a NaN stays
    const float scale = float(s);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (norm_out) *norm_out = float(norm);
        if (scale_out) *scale_out = scale;
    }
    const uint32_t chunks = t.first[t.tensors];
    for (uint32_t i = blockIdx.x; i < chunks; i += t.blocks) {
        const uint32_t c = chunks - 1 - i;
        const int k = clip_tensor(t, c);
        const int64_t at = int64_t(c - t.first[k]) * kClipChunk, left = t.numel[k] - at;
        const int n = int(left < kClipChunk ? left : kClipChunk);
        if (!t.out[k]) continue;
        if (t.dtype[k] == 0) clip_scaled<float>(t.in[k], t.out[k], at, n, scale);
        else if (t.dtype[k] == 1) clip_scaled<bf16_t>(t.in[k], t.out[k], at, n, scale);
        else clip_scaled<f16_t>(t.in[k], t.out[k], at, n, scale);
    }
}

}  // namespace nhipk

// Norms and rotations of attention heads: queries and keys [B, S, heads, D], one pass over each.
//
//   inv = 1 / sqrt(mean(x^2) + eps), z = x inv w, y = R(p) z
//
// where R(p) turns the pairs of z's first `rot` elements by the angles of position p: (a, b) -> (a c - b s, b c + a s),
// pair i's c and s read from the tables' row p. Pairs are elements i and i + rot / 2, or 2 i and 2 i + 1 (interleaved).
// The backward takes the cotangent back through the turn, dz = R(p)^T dy, and needs two sums a row, both of values in
// registers: sum(x^2) and sum(dz w x); then with xhat = x inv, dx = inv (dz w - xhat inv sum(dz w x) / D) and dw = the
// sum over rows of dz xhat.
// Nothing but x is kept from the forward: inv costs the backward no read that it does not make anyway.
//
// HBM bounds both: a row is read once and written once (the backward reads x and dy), everything between in float32.
// A lane holds both elements of its pairs, 2 E of them in two chunks of 16 (8, 4) bytes, so the turn needs no
// exchange and the row sums are the only ones, over the D / (2 E) lanes of a row. A workgroup takes consecutive heads,
// so its reads are contiguous; the table's rows come from L1.
#pragma once

#include "device_common.h"

namespace nhipk {

// n / d for n < 2^31 as a multiply and a shift: q = (mulhi(n, mul) + n) >> shift with mul = ceil(2^(32 + shift) / d) - 2^32
// (the sum stays below 2^32, as mulhi(n, mul) <= n).
struct FastDiv {
    uint32_t d, mul, shift;
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct HeadsTensor {
    const void *x, *dy;  // dy: backward only
    void *y;             // the turned heads, or dx
    const void *w;       // [D] or null: ones
    float *part;         // backward: this tensor's partial weight gradients, one row of D floats a workgroup (null: none)
    int64_t x_b, x_s, x_n, dy_b, dy_s, dy_n, y_b, y_s, y_n;  // element strides
    uint32_t rows;       // tokens x heads of this launch
    uint32_t blocks;     // workgroups that take this tensor's rows
    FastDiv heads;
};

struct HeadsArgs {
    HeadsTensor t[2];  // queries, keys
    const float *cos, *sin;
    const void *positions;  // int32 or int64 [B, S], or null: 0 .. S - 1
    int64_t table_rows, seq, token0;  // token0: the first token of this launch
    FastDiv seq_div;
    int32_t d, rot, pos64, interleaved;
    int32_t lanes;  // of a row: a power of two, at least D / (2 E)
    float eps;
};

template <typename T, int E>
struct HeadsChunk;
template <>
struct HeadsChunk<float, 4> {
    typedef float4 raw;
    __device__ __forceinline__ static void get(const raw &r, float (&v)[4]) { v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w; }
    __device__ __forceinline__ static raw put(const float (&v)[4]) { return make_float4(v[0], v[1], v[2], v[3]); }
};
template <>
struct HeadsChunk<float, 2> {
    typedef float2 raw;
    __device__ __forceinline__ static void get(const raw &r, float (&v)[2]) { v[0] = r.x, v[1] = r.y; }
    __device__ __forceinline__ static raw put(const float (&v)[2]) { return make_float2(v[0], v[1]); }
};
__device__ __forceinline__ float heads_up(bf16_t, uint32_t bits) { return bf16_to_f32(uint16_t(bits)); }
__device__ __forceinline__ float heads_up(f16_t, uint32_t bits) { return f16_to_f32(uint16_t(bits)); }
__device__ __forceinline__ uint32_t heads_down(bf16_t, float v) { return f32_to_bf16(v); }
__device__ __forceinline__ uint32_t heads_down(f16_t, float v) { return f32_to_f16(v); }
template <typename T>
struct HeadsChunk<T, 8> {
    typedef uint4 raw;
    __device__ __forceinline__ static void get(const raw &r, float (&v)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = heads_up(T{}, w[i] & 0xffff), v[2 * i + 1] = heads_up(T{}, w[i] >> 16);
    }
    __device__ __forceinline__ static raw put(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = heads_down(T{}, v[2 * i]) | heads_down(T{}, v[2 * i + 1]) << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <typename T>
struct HeadsChunk<T, 4> {
    typedef uint2 raw;
    __device__ __forceinline__ static void get(const raw &r, float (&v)[4]) {
        v[0] = heads_up(T{}, r.x & 0xffff), v[1] = heads_up(T{}, r.x >> 16);
        v[2] = heads_up(T{}, r.y & 0xffff), v[3] = heads_up(T{}, r.y >> 16);
    }
    __device__ __forceinline__ static raw put(const float (&v)[4]) {
        return make_uint2(heads_down(T{}, v[0]) | heads_down(T{}, v[1]) << 16, heads_down(T{}, v[2]) | heads_down(T{}, v[3]) << 16);
    }
};

template <typename T>
struct HeadsChunk<T, 2> {
    typedef uint32_t raw;
    __device__ __forceinline__ static void get(const raw &r, float (&v)[2]) { v[0] = heads_up(T{}, r & 0xffff), v[1] = heads_up(T{}, r >> 16); }
    __device__ __forceinline__ static raw put(const float (&v)[2]) { return heads_down(T{}, v[0]) | heads_down(T{}, v[1]) << 16; }
};

// Where a lane's two chunks lie in a row, and its first pair: pairs[e] couples chunk 0's element e with chunk 1's, or
// (interleaved) elements 2 e and 2 e + 1 of the two chunks taken as one. turned: past `rot` nothing is.
struct HeadsLane {
    int c0, c1, pair;
    bool in, turned;
};
template <int E>
__device__ __forceinline__ HeadsLane heads_lane(const HeadsArgs &a, int l) {
    HeadsLane r;
    r.in = 2 * E * l < a.d;
    r.turned = 2 * E * l < a.rot;
    r.pair = E * l;
    const bool split = !a.interleaved && r.turned;
    r.c0 = split ? E * l : 2 * E * l;
    r.c1 = split ? a.rot / 2 + E * l : 2 * E * l + E;
    return r;
}

// (v0, v1) turned by the pairs' angles, or (BACK) by minus them.
template <bool BACK, int E>
__device__ __forceinline__ void heads_turn(float (&v0)[E], float (&v1)[E], const float (&c)[E], const float (&sn)[E],
                                           bool interleaved) {
    auto s = [&](int i) { return BACK ? -sn[i] : sn[i]; };
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            const float a = v0[2 * i], b = v0[2 * i + 1], p = v1[2 * i], q = v1[2 * i + 1];
            v0[2 * i] = a * c[i] - b * s(i);
            v0[2 * i + 1] = b * c[i] + a * s(i);
            v1[2 * i] = p * c[E / 2 + i] - q * s(E / 2 + i);
            v1[2 * i + 1] = q * c[E / 2 + i] + p * s(E / 2 + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float a = v0[i], b = v1[i];
            v0[i] = a * c[i] - b * s(i);
            v1[i] = b * c[i] + a * s(i);
        }
    }
}

// Sum over a row's lanes (a power of two of neighbours), in the same order for every lane.
__device__ __forceinline__ float heads_sum(float v, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ int64_t heads_position(const HeadsArgs &a, int64_t token, uint32_t s) {
    int64_t p = s;
    if (a.positions)
        p = a.pos64 ? static_cast<const int64_t *>(a.positions)[token] : int64_t(static_cast<const int32_t *>(a.positions)[token]);
    return p < 0 ? 0 : (p < a.table_rows ? p : a.table_rows - 1);  // as a gather's clamped index
}

// A row of tensor t: its token (of the whole batch), batch and sequence index, head and table row.
struct HeadsRow {
    int64_t token, b, p;
    uint32_t s, h;
};
__device__ __forceinline__ HeadsRow heads_row(const HeadsArgs &a, const HeadsTensor &t, uint32_t row) {
    HeadsRow r;
    const uint32_t k = t.heads.div(row);
    r.h = row - k * t.heads.d;
    r.token = a.token0 + k;
    // below 2^31: seq is below 2^30, a launch's tokens below 2^26
    const uint32_t first = uint32_t(a.token0 % a.seq);
    const uint32_t q = a.seq_div.div(first + k);
    r.b = a.token0 / a.seq + q;
    r.s = first + k - q * uint32_t(a.seq);
    r.p = heads_position(a, r.token, r.s);
    return r;
}

template <int E>
__device__ __forceinline__ void heads_table(const float *p, float (&v)[E]) {
    if constexpr (E == 2) {
        const float2 q = *reinterpret_cast<const float2 *>(p);
        v[0] = q.x, v[1] = q.y;
    } else {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 q = *reinterpret_cast<const float4 *>(p + i);
            v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
        }
    }
}

// One row a group of lanes. More rows a lane at a time only cost waves: at [4, 4096, 16 + 16, 128] in bf16 one row takes 48.4 us
// (5.5 TB/s), two 57.5, four 65.4.
template <typename T, int E>
__global__ __launch_bounds__(256) void heads_fwd_kernel(HeadsArgs a) {
    typedef HeadsChunk<T, E> C;
    const bool second = blockIdx.x >= a.t[0].blocks;
    const HeadsTensor &t = a.t[second];
    const uint32_t row = (blockIdx.x - (second ? a.t[0].blocks : 0)) * (256 / a.lanes) + threadIdx.x / a.lanes;
    const HeadsLane ln = heads_lane<E>(a, threadIdx.x & (a.lanes - 1));
    const bool in = row < t.rows && ln.in;
    const HeadsRow r = heads_row(a, t, row < t.rows ? row : 0);
    float v0[E], v1[E], w0[E], w1[E], c[E], s[E], sq = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) w0[i] = w1[i] = 1.0f;
    if (t.w && ln.in) {  // before the rows: their wait is then the only one
        const T *w = static_cast<const T *>(t.w);
        C::get(*reinterpret_cast<const typename C::raw *>(w + ln.c0), w0);
        C::get(*reinterpret_cast<const typename C::raw *>(w + ln.c1), w1);
    }
    typename C::raw x0, x1;
    if (in) {
        const T *x = static_cast<const T *>(t.x) + r.b * t.x_b + int64_t(r.s) * t.x_s + int64_t(r.h) * t.x_n;
        x0 = *reinterpret_cast<const typename C::raw *>(x + ln.c0);
        x1 = *reinterpret_cast<const typename C::raw *>(x + ln.c1);
        if (ln.turned) {
            heads_table<E>(a.cos + r.p * (a.rot / 2) + ln.pair, c);
            heads_table<E>(a.sin + r.p * (a.rot / 2) + ln.pair, s);
        }
    }
    if (in) {
        C::get(x0, v0);
        C::get(x1, v1);
#pragma unroll
        for (int i = 0; i < E; ++i) sq += v0[i] * v0[i] + v1[i] * v1[i];
    }
    sq = heads_sum(sq, a.lanes);
    if (!in) return;
    const float inv = rsqrtf(sq / float(a.d) + a.eps);
#pragma unroll
    for (int i = 0; i < E; ++i) v0[i] = v0[i] * inv * w0[i], v1[i] = v1[i] * inv * w1[i];
    if (ln.turned) heads_turn<false, E>(v0, v1, c, s, a.interleaved);
    T *y = static_cast<T *>(t.y) + r.b * t.y_b + int64_t(r.s) * t.y_s + int64_t(r.h) * t.y_n;
    *reinterpret_cast<typename C::raw *>(y + ln.c0) = C::put(v0);
    *reinterpret_cast<typename C::raw *>(y + ln.c1) = C::put(v1);
}

// The backward. Workgroups walk a tensor's rows, each group of lanes one at a time; a lane keeps the weight gradient of its
// own 2 E elements over all of them, and a workgroup writes one row of D partial sums. Its registers leave three workgroups
// a CU (E 8): launched as two rounds of them the case above takes 82 us (4.9 TB/s), as 1024 workgroups 100, with two rows at
// a time 90 at best, with the next row's reads ahead of this one's work 82, with the weights read again for each row (four
// workgroups a CU) 85.
template <typename T, int E>
__global__ __launch_bounds__(256) void heads_bwd_kernel(HeadsArgs a) {
    typedef HeadsChunk<T, E> C;
    __shared__ float sums[4][64][2 * E + 1];
    const bool second = blockIdx.x >= a.t[0].blocks;
    const HeadsTensor &t = a.t[second];
    const uint32_t block = blockIdx.x - (second ? a.t[0].blocks : 0);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t groups = 256 / a.lanes, group = threadIdx.x / a.lanes;
    const HeadsLane ln = heads_lane<E>(a, lane & (a.lanes - 1));
    float g0[E], g1[E], w0[E], w1[E];
#pragma unroll
    for (int i = 0; i < E; ++i) g0[i] = g1[i] = 0.0f, w0[i] = w1[i] = 1.0f;
    if (t.w && ln.in) {
        const T *w = static_cast<const T *>(t.w);
        C::get(*reinterpret_cast<const typename C::raw *>(w + ln.c0), w0);
        C::get(*reinterpret_cast<const typename C::raw *>(w + ln.c1), w1);
    }
    const float over_d = 1.0f / float(a.d);
    // 64-bit: the last step may pass 2^32
    for (uint64_t base = uint64_t(block) * groups; base < t.rows; base += uint64_t(t.blocks) * groups) {
        const bool in = base + group < t.rows && ln.in;
        const HeadsRow r = heads_row(a, t, base + group < t.rows ? uint32_t(base + group) : 0);
        typename C::raw x0, x1, y0, y1;
        float c[E], s[E];
        if (in) {
            const T *x = static_cast<const T *>(t.x) + r.b * t.x_b + int64_t(r.s) * t.x_s + int64_t(r.h) * t.x_n;
            const T *dy = static_cast<const T *>(t.dy) + r.b * t.dy_b + int64_t(r.s) * t.dy_s + int64_t(r.h) * t.dy_n;
            x0 = *reinterpret_cast<const typename C::raw *>(x + ln.c0);
            x1 = *reinterpret_cast<const typename C::raw *>(x + ln.c1);
            y0 = *reinterpret_cast<const typename C::raw *>(dy + ln.c0);
            y1 = *reinterpret_cast<const typename C::raw *>(dy + ln.c1);
            if (ln.turned) {
                heads_table<E>(a.cos + r.p * (a.rot / 2) + ln.pair, c);
                heads_table<E>(a.sin + r.p * (a.rot / 2) + ln.pair, s);
            }
        }
        float v0[E], v1[E], z0[E], z1[E], sq = 0.0f, dot = 0.0f;
        if (in) {
            C::get(x0, v0);
            C::get(x1, v1);
            C::get(y0, z0);
            C::get(y1, z1);
            if (ln.turned) heads_turn<true, E>(z0, z1, c, s, a.interleaved);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                sq += v0[i] * v0[i] + v1[i] * v1[i];
                dot += z0[i] * w0[i] * v0[i] + z1[i] * w1[i] * v1[i];
            }
        }
        sq = heads_sum(sq, a.lanes);
        dot = heads_sum(dot, a.lanes);
        if (!in) continue;
        const float inv = rsqrtf(sq * over_d + a.eps), mean = dot * over_d * inv;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float h0 = v0[i] * inv, h1 = v1[i] * inv;
            g0[i] += z0[i] * h0;
            g1[i] += z1[i] * h1;
            z0[i] = inv * (z0[i] * w0[i] - h0 * mean);
            z1[i] = inv * (z1[i] * w1[i] - h1 * mean);
        }
        if (!t.y) continue;  // the weight's gradient alone
        T *dx = static_cast<T *>(t.y) + r.b * t.y_b + int64_t(r.s) * t.y_s + int64_t(r.h) * t.y_n;
        *reinterpret_cast<typename C::raw *>(dx + ln.c0) = C::put(z0);
        *reinterpret_cast<typename C::raw *>(dx + ln.c1) = C::put(z1);
    }
    if (!t.part) return;
    // over the wave's groups by lane exchange, over the waves through LDS, both in a fixed order
#pragma unroll
    for (int i = 0; i < E; ++i) {
        float p = g0[i], q = g1[i];
        for (int o = a.lanes; o < 64; o <<= 1) p += __shfl_xor(p, o, 64), q += __shfl_xor(q, o, 64);
        sums[wave][lane][i] = p;
        sums[wave][lane][E + i] = q;
    }
    __syncthreads();
    if (wave == 0 && lane < a.lanes && ln.in) {
        float *out = t.part + int64_t(block) * a.d;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            out[ln.c0 + i] = (sums[0][lane][i] + sums[1][lane][i]) + (sums[2][lane][i] + sums[3][lane][i]);
            out[ln.c1 + i] = (sums[0][lane][E + i] + sums[1][lane][E + i]) + (sums[2][lane][E + i] + sums[3][lane][E + i]);
        }
    }
}

// Any head dim to kHeadsMost, alignment and rotated part: a lane takes a row's pairs l, l + lanes, ... one element at a
// time (the part past `rot` as pairs of neighbours, its last element alone where it is odd).
constexpr int kHeadsMost = 1024;

struct HeadsPair {
    int i0, i1;  // i1 < 0: none
    bool turned;
};
__device__ __forceinline__ HeadsPair heads_pair(const HeadsArgs &a, int k) {
    HeadsPair p;
    const int half = a.rot / 2;
    p.turned = k < half;
    if (p.turned) {
        p.i0 = a.interleaved ? 2 * k : k;
        p.i1 = a.interleaved ? 2 * k + 1 : half + k;
    } else {
        p.i0 = a.rot + 2 * (k - half);
        p.i1 = p.i0 + 1 < a.d ? p.i0 + 1 : -1;
    }
    return p;
}

template <typename T, bool BWD>
__global__ __launch_bounds__(256) void heads_any_kernel(HeadsArgs a) {
    __shared__ float sums[BWD ? 256 / 32 : 1][BWD ? kHeadsMost : 1];  // a row of weight gradients for each group of >= 32 lanes
    const bool second = blockIdx.x >= a.t[0].blocks;
    const HeadsTensor &t = a.t[second];
    const uint32_t block = blockIdx.x - (second ? a.t[0].blocks : 0);
    const uint32_t groups = 256 / a.lanes, group = threadIdx.x / a.lanes;
    const int l = threadIdx.x & (a.lanes - 1);
    const int pairs = a.rot / 2 + (a.d - a.rot + 1) / 2;
    const T *w = static_cast<const T *>(t.w);
    if constexpr (BWD)
        for (int i = threadIdx.x; i < int(groups) * a.d; i += 256) sums[i / a.d][i % a.d] = 0.0f;
    if constexpr (BWD) __syncthreads();
    const float over_d = 1.0f / float(a.d);
    for (uint64_t base = uint64_t(block) * groups; base < t.rows; base += uint64_t(t.blocks) * groups) {
        const bool in = base + group < t.rows;
        const HeadsRow r = heads_row(a, t, in ? uint32_t(base + group) : 0);
        const T *x = static_cast<const T *>(t.x) + r.b * t.x_b + int64_t(r.s) * t.x_s + int64_t(r.h) * t.x_n;
        const T *dy = static_cast<const T *>(t.dy) + r.b * t.dy_b + int64_t(r.s) * t.dy_s + int64_t(r.h) * t.dy_n;
        T *y = static_cast<T *>(t.y) + r.b * t.y_b + int64_t(r.s) * t.y_s + int64_t(r.h) * t.y_n;
        const float *cs = a.cos + r.p * (a.rot / 2), *sn = a.sin + r.p * (a.rot / 2);
        // a pair's x, weights and (backward) its cotangent turned back
        auto pair = [&](int k, float &v0, float &v1, float &q0, float &q1, float &z0, float &z1, HeadsPair &p) {
            p = heads_pair(a, k);
            v0 = load_as_f32(x + p.i0);
            v1 = p.i1 >= 0 ? load_as_f32(x + p.i1) : 0.0f;
            q0 = w ? load_as_f32(w + p.i0) : 1.0f;
            q1 = w && p.i1 >= 0 ? load_as_f32(w + p.i1) : 1.0f;
            if constexpr (BWD) {
                z0 = load_as_f32(dy + p.i0);
                z1 = p.i1 >= 0 ? load_as_f32(dy + p.i1) : 0.0f;
                if (p.turned) {
                    const float c = cs[k], s = sn[k], b = z0;
                    z0 = b * c + z1 * s;
                    z1 = z1 * c - b * s;
                }
            }
        };
        float v0, v1, q0, q1, z0, z1, sq = 0.0f, dot = 0.0f;
        HeadsPair p;
        if (in)
            for (int k = l; k < pairs; k += a.lanes) {
                pair(k, v0, v1, q0, q1, z0, z1, p);
                sq += v0 * v0 + v1 * v1;
                if constexpr (BWD) dot += z0 * q0 * v0 + z1 * q1 * v1;
            }
        sq = heads_sum(sq, a.lanes);
        if constexpr (BWD) dot = heads_sum(dot, a.lanes);
        if (!in) continue;
        const float inv = rsqrtf(sq * over_d + a.eps);
        for (int k = l; k < pairs; k += a.lanes) {
            pair(k, v0, v1, q0, q1, z0, z1, p);
            float o0, o1;
            if constexpr (BWD) {
                const float mean = dot * over_d * inv, h0 = v0 * inv, h1 = v1 * inv;
                o0 = inv * (z0 * q0 - h0 * mean);
                o1 = inv * (z1 * q1 - h1 * mean);
                sums[group][p.i0] += z0 * h0;  // this lane's own elements
                if (p.i1 >= 0) sums[group][p.i1] += z1 * h1;
            } else {
                o0 = v0 * inv * q0;
                o1 = v1 * inv * q1;
                if (p.turned) {
                    const float c = cs[k], s = sn[k], b = o0;
                    o0 = b * c - o1 * s;
                    o1 = o1 * c + b * s;
                }
            }
            if (!t.y) continue;  // the weight's gradient alone
            store_f32_as(y + p.i0, o0);
            if (p.i1 >= 0) store_f32_as(y + p.i1, o1);
        }
    }
    if constexpr (BWD) {
        __syncthreads();
        if (!t.part) return;
        for (int i = threadIdx.x; i < a.d; i += 256) {
            float v = sums[0][i];
            for (uint32_t g = 1; g < groups; ++g) v += sums[g][i];
            t.part[int64_t(block) * a.d + i] = v;
        }
    }
}

// dw[i] = the sum of `rows` partial rows' element i, in a fixed order: 64 columns x 16 row lanes a workgroup, the
// queries' and the keys' weights in one launch (blockIdx.y).
struct HeadsSum {
    const float *part[2];
    void *out[2];
    uint32_t rows[2];
    int32_t d;
};
template <typename T>
__global__ __launch_bounds__(1024) void heads_sum_kernel(HeadsSum a) {
    __shared__ float sums[16][64];
    const int column = blockIdx.x * 64 + (threadIdx.x & 63), lane = threadIdx.x >> 6, which = blockIdx.y;
    T *out = static_cast<T *>(a.out[which]);
    if (!out) return;  // the whole workgroup
    float v = 0.0f;
    if (column < a.d) {
#pragma unroll 8
        for (uint32_t r = lane; r < a.rows[which]; r += 16) v += a.part[which][int64_t(r) * a.d + column];
    }
    sums[lane][threadIdx.x & 63] = v;
    __syncthreads();
    if (lane == 0 && column < a.d) {
#pragma unroll
        for (int k = 1; k < 16; ++k) v += sums[k][threadIdx.x];
        store_f32_as(out + column, v);
    }
}

}  // namespace nhipk

// Self attention of sequences packed one after another: each within its own, forward and backward, by the tiles of
// attention.h over a table of workgroups made of the offsets on the device (packed_tiles_kernel, packed_tiles_few; packed_tile
// where a launch needs none).
//
// A workgroup's tile lies within one sequence and its loads end there, so that no row of another sequence (of padding, NaN
// or infinite) reaches it, not even with a probability of zero. The grid covers the most tiles that any offsets give
// (tokens / block, and one more a sequence); the table's unused entries end at once. Entries stand by falling work, whatever
// sequence they are of, so that the longest start first and the last ones fill the gaps. Tokens of no sequence (before the
// first offset and from the last one on) are entries too: their results are zeros.
//
// MFMA bounds long sequences, at the flash kernels' rates. 8 documents of 281 to 4096 tokens, 16 heads of 128, causal, us: forward
// 271 (719 TFLOP/s), rows' sums 38 (5.3 TB/s), dK and dV with dS stored 678 (575), dQ from it 187; an empty launch of either kernel
// of the other mode 5. Short ones are bound by launches and by the longest sequence's tiles one after another.
#pragma once

#include "attention.h"

namespace nhipk {

// A workgroup's tile: the sequence's first token and length, the block of it, and the first dS tile of the sequence (of one
// head). block < 0: zeros for `len` tokens from `start` on.
struct PackedTile {
    int32_t start, len, block, ds;
};

struct PackedTable {
    PackedTile *tiles;
    int32_t most;    // entries
    int32_t block;   // rows a workgroup
    int32_t shift;   // a tile's work in 2^shift blocks
    int32_t order;   // PACKED_*
};
enum { PACKED_FLAT = 0, PACKED_RISING = 1, PACKED_FALLING = 2 };  // how a sequence's blocks' work goes with their index

struct PackedTables {
    PackedTable t[2];
    const void *offsets;
    int64_t sequences, tokens;
    int32_t o64;
    int64_t ds_tiles;    // dS tiles of one head that there is room for
    int32_t *fits;       // whether all of them do (null: nobody asks)
};

constexpr int kPackedBuckets = 1024;  // also the builder's threads

__device__ __forceinline__ int packed_wave_max(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v = max(v, u);
    }
    return v;
}

template <typename T>
__device__ __forceinline__ T packed_wave_sum(T v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}

// Entry j behind the tiles: tokens of no sequence, then nothing.
__device__ __forceinline__ PackedTile packed_rest(int block, int j, int first, int last, int tokens) {
    const int lead = (first + block - 1) / block, tail = (tokens - last + block - 1) / block;
    int from = j * block, to = first;
    if (j >= lead) from = last + (j - lead) * block, to = j < lead + tail ? tokens : from;
    return PackedTile{from < tokens ? from : 0, min(max(to - from, 0), block), -1, 0};
}

__device__ __forceinline__ int packed_offset(const PackedTables &a, int64_t i) {
    const int64_t v = a.o64 ? static_cast<const int64_t *>(a.offsets)[i] : static_cast<const int32_t *>(a.offsets)[i];
    return int(v < 0 ? 0 : v > a.tokens ? a.tokens : v);
}

// One workgroup a table. Offsets are clamped into [the one before, tokens], so that whatever they hold every tile lies within
// the tokens and no token is of two sequences. Two passes over the sequences, 1024 at a time: the first counts the tiles of
// each amount of work (and dS tiles), the second places them; the order within an amount is whatever the atomics give and
// decides only which workgroup starts first.
static __global__ __launch_bounds__(kPackedBuckets) void packed_tiles_kernel(PackedTables a) {
    __shared__ int at[kPackedBuckets + 1];      // the chunk's clamped offsets
    __shared__ int ds_at[kPackedBuckets];
    __shared__ int waves[16];
    __shared__ long long wave_sums[16];
    __shared__ int bucket[kPackedBuckets];
    const PackedTable t = a.t[blockIdx.x];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int tokens = int(a.tokens);
    bucket[tid] = 0;
    const int first = packed_offset(a, 0);
    int last = first;
    for (int pass = 0; pass < 2; ++pass) {
        int carry = 0;
        long long ds_carry = 0;
        for (int64_t base = 0; base < a.sequences; base += kPackedBuckets) {
            const int here = int(min(a.sequences - base, int64_t(kPackedBuckets)));
            __syncthreads();  // the chunk before is done with `at` (and `bucket` is cleared)
            // offsets base .. base + here, each at least the one before
            int v = packed_wave_max(tid <= here ? packed_offset(a, base + tid) : 0, lane);
            if (lane == 63) waves[wave] = v;
            __syncthreads();
            int before = carry;
            for (int w = 0; w < wave; ++w) before = max(before, waves[w]);
            v = max(v, before);
            at[tid] = v;
            __syncthreads();
            if (tid == 0) at[kPackedBuckets] = here == kPackedBuckets ? max(at[kPackedBuckets - 1], packed_offset(a, base + here)) : 0;
            __syncthreads();
            carry = at[here];
            const int len = tid < here ? at[tid + 1] - at[tid] : 0;
            // the sequence's first dS tile
            const long long own = (long long)((len + 127) / 128) * ((len + 63) / 64);
            const long long sum = packed_wave_sum(own, lane);
            if (lane == 63) wave_sums[wave] = sum;
            __syncthreads();
            long long ds = ds_carry + sum - own;
            for (int w = 0; w < 16; ++w) {
                if (w < wave) ds += wave_sums[w];
                ds_carry += wave_sums[w];
            }
            ds_at[tid] = ds < a.ds_tiles ? int(ds) : 0;  // read only where all fit
            __syncthreads();
            auto tile = [&](int k, int blocks, int j) {
                const int work = t.order == PACKED_RISING ? j + 1 : t.order == PACKED_FALLING ? blocks - j : blocks;
                int *slot = bucket + (kPackedBuckets - 1 - min(work >> t.shift, kPackedBuckets - 1));
                const int n = atomicAdd(slot, 1);
                if (pass == 1) t.tiles[n] = PackedTile{at[k], at[k + 1] - at[k], j, ds_at[k]};
            };
            // short sequences a thread each, the others a wavefront
            constexpr int SHORT = 8;
            const int blocks = (len + t.block - 1) / t.block;
            if (blocks <= SHORT)
                for (int j = 0; j < blocks; ++j) tile(tid, blocks, j);
            for (int k = wave; k < here; k += 16) {
                const int n = (at[k + 1] - at[k] + t.block - 1) / t.block;
                if (n > SHORT)
                    for (int j = lane; j < n; j += 64) tile(k, n, j);
            }
        }
        last = max(first, carry);
        __syncthreads();
        if (pass == 1) break;
        if (a.fits && tid == 0 && blockIdx.x == 0) *a.fits = ds_carry <= a.ds_tiles;
        // counts to places
        const int count = bucket[tid], sum = packed_wave_sum(count, lane);
        if (lane == 63) waves[wave] = sum;
        __syncthreads();
        int place = sum - count;
        for (int w = 0; w < wave; ++w) place += waves[w];
        bucket[tid] = place;
    }
    const int placed = bucket[kPackedBuckets - 1];  // where the last amount's tiles end
    for (int i = placed + tid; i < t.most; i += kPackedBuckets) t.tiles[i] = packed_rest(t.block, i - placed, first, last, tokens);
}

// The same for fewer sequences than threads, without atomics: a tile's place is the tiles of more work, which are those of every
// sequence's blocks past its own work, and the sequences before its own that have as many blocks (3 sequences of 97 tokens: 3.2 us,
// 8.7 by amounts; 8 of 16384: 5.0, 11.5).
constexpr int kPackedFew = 256;
__device__ __forceinline__ void packed_tiles_few(const PackedTables &a, int table) {
    __shared__ int at[kPackedFew + 1], before[kPackedFew + 1], ds_at[kPackedFew];
    __shared__ __align__(16) int blocks[kPackedFew];
    __shared__ int waves[3][4];
    const PackedTable t = a.t[table];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, tokens = int(a.tokens), count = int(a.sequences);
    int v = packed_wave_max(tid <= count ? packed_offset(a, tid) : 0, lane);
    if (lane == 63) waves[0][wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v = max(v, waves[0][w]);
    at[tid] = v;
    __syncthreads();
    const int len = tid < count ? at[tid + 1] - v : 0, own = (len + t.block - 1) / t.block;
    // dS tiles of sequences that do not fit may be past 32 bits; their sum over a wavefront's is capped ahead of that
    const long long tiles = (long long)((len + 127) / 128) * ((len + 63) / 64);
    const int ds_own = int(min(tiles, (long long)(1 << 24)));
    const int sum = packed_wave_sum(own, lane), ds = packed_wave_sum(ds_own, lane);
    if (lane == 63) waves[1][wave] = sum, waves[2][wave] = ds;
    blocks[tid] = own;
    __syncthreads();
    int from = sum - own, ds_from = ds - ds_own, total = 0;
    long long ds_total = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < wave) from += waves[1][w], ds_from += waves[2][w];
        total += waves[1][w], ds_total += waves[2][w];
    }
    before[tid] = from;
    ds_at[tid] = ds_from;  // read only where all fit
    const int first = at[0], last = at[count];
    if (a.fits && tid == 0 && table == 0) *a.fits = ds_total <= a.ds_tiles;
    __syncthreads();
    for (int i = tid; i < total; i += kPackedFew) {
        int k = 0, hi = count;
        while (hi - k > 1) {
            const int mid = (k + hi) / 2;
            if (before[mid] <= i) k = mid;
            else hi = mid;
        }
        const int j = i - before[k], n = blocks[k];
        const int work = t.order == PACKED_RISING ? j + 1 : t.order == PACKED_FALLING ? n - j : n;
        int place = t.order == PACKED_FLAT ? j : 0;
        for (int s0 = 0; s0 < count; s0 += 4) {
            const int4 b4 = *reinterpret_cast<const int4 *>(blocks + s0);
            const int b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (t.order == PACKED_FLAT) place += b[e] > n || (b[e] == n && s0 + e < k) ? b[e] : 0;
                else place += max(b[e] - work, 0) + (b[e] >= work && s0 + e < k ? 1 : 0);
            }
        }
        t.tiles[place] = PackedTile{at[k], at[k + 1] - at[k], j, ds_at[k]};
    }
    for (int i = total + tid; i < t.most; i += kPackedFew) t.tiles[i] = packed_rest(t.block, i - total, first, last, tokens);
}
static __global__ __launch_bounds__(kPackedFew) void packed_tiles_few_kernel(PackedTables a) { packed_tiles_few(a, int(blockIdx.x)); }

// The tile of entry `idx` of a table of fewer sequences than lanes, in the sequences' order, without a table: where a launch's
// workgroups all run at once nothing is gained by the order (97 tokens, 16 heads: 8.2 us a call, 10.9 with a table).
constexpr int kPackedDirect = 63;
__device__ __forceinline__ PackedTile packed_tile(const PackedTables &a, int block, int idx) {
    const int lane = threadIdx.x & 63, count = int(a.sequences);
    const int v = packed_wave_max(lane <= count ? packed_offset(a, lane) : 0, lane);
    const int next = __shfl_down(v, 1, 64), len = lane < count ? next - v : 0, own = (len + block - 1) / block;
    const int before = packed_wave_sum(own, lane) - own;
    const int first = __builtin_amdgcn_readlane(v, 0), last = __builtin_amdgcn_readlane(v, count),
              total = __builtin_amdgcn_readlane(before, count);
    if (idx >= total) return packed_rest(block, idx - total, first, last, int(a.tokens));
    const int k = 63 - __builtin_clzll(__ballot(lane < count && before <= idx));
    return PackedTile{__builtin_amdgcn_readlane(v, k), __builtin_amdgcn_readlane(len, k), idx - __builtin_amdgcn_readlane(before, k), 0};
}

// The head and table entry of a workgroup: heads fastest, in runs that stay on one XCD (workgroups go round the eight) where
// they divide evenly, so that heads of one group read their keys through one L2.
__device__ __forceinline__ void packed_place(int64_t heads, int64_t &n, int64_t &idx) {
    const int64_t lin = blockIdx.x;
    idx = lin / heads, n = lin % heads;
    if (heads % 8 == 0) n = (n % 8) * (heads / 8) + n / 8;
}

__device__ __forceinline__ void packed_zeros(uint16_t *p, int64_t stride, int64_t cols, const PackedTile &t) {
    const int chunks = int(cols / 8);
    for (int i = threadIdx.x; i < t.len * chunks; i += blockDim.x)
        *reinterpret_cast<uint4 *>(p + (t.start + int64_t(i / chunks)) * stride + i % chunks * 8) = make_uint4(0, 0, 0, 0);
}

// The operands of a tile's sequence alone.
__device__ __forceinline__ void packed_sequence(AttnParams &p, const PackedTile &t) {
    p.q += t.start * p.q_s, p.k += t.start * p.k_s, p.v += t.start * p.v_s;
    p.sq = p.sk = t.len;
}

template <int D, bool F16, bool CAUSAL, int NW>
__global__ __launch_bounds__(64 * NW, (FwdOccupancy<NW, D>::kBlocks)) void packed_fwd_kernel(AttnParams p, uint16_t *rest,
                                                                                             PackedTables a) {
    int64_t n, idx;
    packed_place(p.heads, n, idx);
    const PackedTile t = a.t[0].tiles ? a.t[0].tiles[idx] : packed_tile(a, 32 * NW, int(idx));
    const int64_t tokens = a.tokens;
    const int64_t rest_s = p.heads * p.hdv;
    if (t.block < 0) {
        packed_zeros(p.o + n * p.o_n, p.o_s, p.hdv, t);
        if (rest) packed_zeros(rest + n * p.hdv, rest_s, p.hdv, t);
        return;
    }
    packed_sequence(p, t);
    p.o += t.start * p.o_s;
    if (rest) rest += t.start * rest_s + n * p.hdv;
    if (p.lse) p.lse += n * (tokens - t.len) + t.start;  // [heads, tokens], as flash_fwd_tile finds a row of sq
    flash_fwd_tile<D, F16, CAUSAL, NW, false, true>(p, 0, n, t.block, rest, rest_s);
}

// delta = rowsum(dO O) scale and lse log2 e of every token, those of no sequence too (nothing reads theirs): D / 8 lanes a row
// of 16 bytes each. O is taken with what its rounding left (rest, [tokens, heads, hdv], or null): without it the error of O is in
// every dS of a row alike, and of rows of few keys is as much as dS's own rounding: the gradients of sequences of 2 to 8 tokens
// were off by 3.1e-3 of their length (2.5e-3 with it, 1.7e-3 being their rounding), of 64 to 90 by 2.6e-3 (2.4e-3). The first
// `tables` workgroups build the tables meanwhile (packed_tiles_few): a launch less (5120 tokens, 8 heads, dims 64: 5.3 us for
// both, 9.6 apart).
template <int D, bool F16>
__global__ __launch_bounds__(256) void packed_prep_kernel(AttnParams p, const uint16_t *rest, float *lse2, PackedTables a, int tables) {
    if (int(blockIdx.x) < tables) {
        packed_tiles_few(a, int(blockIdx.x));
        return;
    }
    constexpr int LPR = D / 8;
    const int sub = threadIdx.x % LPR;
    const int64_t row = (int64_t(blockIdx.x) - tables) * (256 / LPR) + threadIdx.x / LPR;  // of [heads, tokens]
    const bool live = row < p.heads * p.sq;
    const int64_t n = live ? row / p.sq : 0, q = live ? row % p.sq : 0;
    float acc = 0.0f;
    if (live && 8 * sub < p.hdv) {
        const uint4 ov = *reinterpret_cast<const uint4 *>(p.o_in + n * p.o_n + q * p.o_s + 8 * sub);
        const uint4 gv = *reinterpret_cast<const uint4 *>(p.d_o + n * p.do_n + q * p.do_s + 8 * sub);
        const uint4 rv = rest ? *reinterpret_cast<const uint4 *>(rest + (q * p.heads + n) * p.hdv + 8 * sub) : make_uint4(0, 0, 0, 0);
        const uint32_t ow[4] = {ov.x, ov.y, ov.z, ov.w}, gw[4] = {gv.x, gv.y, gv.z, gv.w}, rw[4] = {rv.x, rv.y, rv.z, rv.w};
        auto low = [](uint32_t w) { return half_to_f32<F16>(uint16_t(w & 0xffffu)); };
        auto high = [](uint32_t w) { return half_to_f32<F16>(uint16_t(w >> 16)); };
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc += low(gw[e]) * (low(ow[e]) + low(rw[e]));
            acc += high(gw[e]) * (high(ow[e]) + high(rw[e]));
        }
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
    if (live && sub == 0) {
        p.delta[row] = acc * p.scale;
        lse2[row] = p.lse_in[row] * 1.4426950408889634f;
    }
}

// STORE: each tile's dS goes to the workspace for packed_dq_ds_kernel; else packed_dq_kernel computes it again. Where the
// room for dS may not do both are launched, and `fits` ends one of them. PARTS: a workgroup takes part blockIdx.y of a key
// block's query tiles, whose sums [parts][entries of all heads][256 D] packed_dkdv_sum_kernel adds.
template <int D, bool F16, bool CAUSAL, bool STORE, bool PARTS>
__global__ __launch_bounds__(256) void packed_dkdv_kernel(AttnParams p, const float *lse2, const PackedTile *tiles, int64_t tokens,
                                                          const int32_t *fits, float *sums) {
    if (fits && (*fits != 0) != STORE) return;
    int64_t n, idx;
    packed_place(p.kv_heads, n, idx);
    const PackedTile t = tiles[idx];
    if (t.block < 0) {
        if (PARTS && blockIdx.y) return;
        packed_zeros(p.dk + n * p.dk_n, p.dk_s, p.hd, t);
        packed_zeros(p.dv + n * p.dv_n, p.dv_s, p.hdv, t);
        return;
    }
    packed_sequence(p, t);
    p.d_o += t.start * p.do_s, p.dk += t.start * p.dk_s, p.dv += t.start * p.dv_s;
    p.delta += t.start;
    if (STORE) p.ds += t.ds * p.heads * (128 * 64);
    if (PARTS) sums += (int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * (256 * D);
    flash_dkdv_tile<D, F16, CAUSAL, false, STORE, false, PARTS>(p, lse2 + t.start, 0, n, t.block, (t.len + 127) / 128, tokens,
                                                                int(blockIdx.y), int(gridDim.y), sums);
}

// The parts' sums, added in order and rounded: blockIdx.y is a tile of 32 columns of dK, then of dV.
template <int D, bool F16>
__global__ __launch_bounds__(256) void packed_dkdv_sum_kernel(AttnParams p, const PackedTile *tiles, const float *__restrict__ sums,
                                                              int parts) {
    int64_t n, idx;
    packed_place(p.kv_heads, n, idx);
    const PackedTile t = tiles[idx];
    if (t.block < 0) return;
    const bool v = blockIdx.y >= D / 32;
    const int dt = int(blockIdx.y) % (D / 32), cols = int(v ? p.hdv : p.hd);
    const float4 *from = reinterpret_cast<const float4 *>(sums + int64_t(blockIdx.x) * (256 * D)) + int64_t(blockIdx.y) * 1024 +
                         threadIdx.x;
    float4 sum[4];
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) sum[e4] = from[256 * e4];
#pragma unroll 4
    for (int k = 1; k < parts; ++k)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
            const float4 x = from[int64_t(k) * gridDim.x * (64 * D) + 256 * e4];
            sum[e4].x += x.x, sum[e4].y += x.y, sum[e4].z += x.z, sum[e4].w += x.w;
        }
    // a key a lane, and every other four columns, as flash_dkdv_tile's
    const int lane = threadIdx.x & 63, key = t.block * 128 + int(threadIdx.x >> 6) * 32 + (lane & 31);
    if (key >= t.len) return;
    uint16_t *to = v ? p.dv + n * p.dv_n + (t.start + int64_t(key)) * p.dv_s : p.dk + n * p.dk_n + (t.start + int64_t(key)) * p.dk_s;
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4)
        if (32 * dt + 8 * e4 < cols)
            *reinterpret_cast<uint2 *>(to + 32 * dt + 8 * e4 + 4 * (lane >> 5)) =
                make_uint2(pack2<F16>(sum[e4].x, sum[e4].y), pack2<F16>(sum[e4].z, sum[e4].w));
}

template <int D, bool F16, bool CAUSAL>
__global__ __launch_bounds__(256, 2) void packed_dq_ds_kernel(AttnParams p, const PackedTile *tiles, const int32_t *fits) {
    if (fits && !*fits) return;
    int64_t n, idx;
    packed_place(p.heads, n, idx);
    const PackedTile t = tiles[idx];
    if (t.block < 0) {
        packed_zeros(p.dq + n * p.dq_n, p.dq_s, p.hd, t);
        return;
    }
    packed_sequence(p, t);
    p.dq += t.start * p.dq_s;
    p.ds += t.ds * p.heads * (128 * 64);
    flash_dq_ds_tile<D, F16, CAUSAL>(p, 0, n, t.block);
}

template <int D, bool F16, bool CAUSAL>
__global__ __launch_bounds__(256, 2) void packed_dq_kernel(AttnParams p, const float *lse2, const PackedTile *tiles, int64_t tokens,
                                                           const int32_t *fits) {
    if (fits && *fits) return;
    int64_t n, idx;
    packed_place(p.heads, n, idx);
    const PackedTile t = tiles[idx];
    // entries are of 256 rows, the kernel's tiles of 128: one half after the other
    if (t.block < 0) {
        packed_zeros(p.dq + n * p.dq_n, p.dq_s, p.hd, t);
        return;
    }
    packed_sequence(p, t);
    p.d_o += t.start * p.do_s, p.dq += t.start * p.dq_s;
    p.delta += t.start;
    for (int half = 0; half < 2; ++half) {
        const int64_t block = 2 * int64_t(t.block) + half;
        if (block * 128 >= t.len) break;
        if (half) __syncthreads();  // every wave is done with the first half's LDS tiles
        flash_dq_tile<D, F16, CAUSAL>(p, lse2 + t.start, 0, n, block, tokens);
    }
}

}  // namespace nhipk

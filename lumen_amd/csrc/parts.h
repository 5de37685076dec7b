// How a product of the streamed tiles (gemm.h) is divided: the tiles' size and the parts of k.
#pragma once

#include <cstdint>

namespace nhip {

inline int64_t tiles(int64_t m, int64_t bm, int64_t n, int64_t bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }

// Whether tiles of bm x bn, a workgroup of `threads` each, are a launch of fewer than 2^32 threads (their count within 64 bits).
inline bool tiles_ok(int64_t m, int64_t bm, int64_t n, int64_t bn, int threads) {
    const int64_t a = (m + bm - 1) / bm, b = (n + bn - 1) / bn;
    return a < (int64_t(1) << 32) && b < (int64_t(1) << 32) / (threads * (a > 0 ? a : 1));
}

// The tile and the parts of a product of z batches over `total` k tiles of 64: as many parts as make the tiles' rounds on the
// chip the shortest, each round as long as its k, the parts' writing and reading added. The rates are the split dots'
// (Plan._split_us), whose loops these are. longest: k tiles that a part may have at most.
struct PartPlan {
    int tm, parts, k_part;
    bool deep;  // at most a workgroup a CU of 128-row tiles: three stages
    double us;
};
// The parts' sums, written and added, of `elements` results.
inline double parts_us(int64_t elements, int64_t parts) { return parts > 1 ? 4.2 + 8.0 * double(parts) * double(elements) / 6.13e6 : 0.0; }

inline PartPlan part_plan(int64_t m, int64_t n, int64_t z, int64_t total, int64_t longest) {
    PartPlan best{0, 0, 0, false, 0.0};
    if (total < 1) total = 1;  // no tokens: nothing is launched, the workspace is asked for all the same
    for (int tm : {256, 128})
        for (int s = 1; s <= 64; s *= 2) {
            const int64_t part = (total + s - 1) / s, parts = (total + part - 1) / part;
            if (part > longest) continue;
            if (best.tm && parts > 1 && (part < 8 || parts * z * m * n * 4 > (int64_t(64) << 20))) continue;
            const int64_t t = tiles(m, tm, n, tm) * z * parts;
            // 256: a workgroup a CU; 128: two, one alone taking 0.79 of a round of both, 0.62 with three stages, whose LDS
            // leaves room for one ([2000, 1024] x [2048, 1024] weights' gradients 30.4 -> 23.8 us; launches of more than 256
            // are slower so: [1463, 3392] x [712, 3392] 26.7 -> 33.2)
            const bool deep = tm == 128 && t <= 256;
            double rounds = tm == 256 ? double((t + 255) / 256) : deep ? 0.62 : double(t / 512);
            const int64_t rest = t % 512;
            if (tm == 128 && !deep) rounds += rest == 0 ? 0.0 : rest <= 256 ? 0.79 : 1.0;
            const double us = 6.2 + 64.0 * double(part) * (tm == 256 ? 0.02355 : 0.0142) * rounds + parts_us(z * m * n, parts);
            if (!best.tm || us < best.us) best = PartPlan{tm, int(parts), int(part), deep, us};
        }
    return best;
}

}  // namespace nhip

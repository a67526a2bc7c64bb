// What the kernels that make work lists share: sums over a workgroup, and the
// limit on a piece's cost.
#pragma once
#include "attn_common.hpp"
#include "attn_paged_plan.hpp"

namespace pelica {

// A lane's value from another of the wave by a data-parallel move (DPP):
// row_shr 1, 2, 4, 8 within 16 lanes, then the last lane of a row, or of two,
// to the rows after it.  A few cycles each; a shuffle goes through LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int old, int x) {
    return __builtin_amdgcn_update_dpp(old, x, CTRL, ROWS, 0xF, false);
}
// inclusive sums over the wave's lanes
__device__ __forceinline__ int wave_scan(int x) {
    x += dpp<0x111, 0xF>(0, x);
    x += dpp<0x112, 0xF>(0, x);
    x += dpp<0x114, 0xF>(0, x);
    x += dpp<0x118, 0xF>(0, x);
    x += dpp<0x142, 0xA>(0, x);
    x += dpp<0x143, 0xC>(0, x);
    return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
template <typename F>
__device__ __forceinline__ float wave_fold(float x, F f) {
    auto at = [&](auto moved) { x = f(x, __uint_as_float(moved(__float_as_uint(x)))); };
    at([](int v) { return dpp<0x111, 0xF>(v, v); });
    at([](int v) { return dpp<0x112, 0xF>(v, v); });
    at([](int v) { return dpp<0x114, 0xF>(v, v); });
    at([](int v) { return dpp<0x118, 0xF>(v, v); });
    at([](int v) { return dpp<0x142, 0xA>(v, v); });
    at([](int v) { return dpp<0x143, 0xC>(v, v); });
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
__device__ __forceinline__ float wave_sum(float x) {
    // (a fold would add what a lane without a source keeps)
    auto at = [&](auto moved) { x += __uint_as_float(moved(__float_as_uint(x))); };
    at([](int v) { return dpp<0x111, 0xF>(0, v); });
    at([](int v) { return dpp<0x112, 0xF>(0, v); });
    at([](int v) { return dpp<0x114, 0xF>(0, v); });
    at([](int v) { return dpp<0x118, 0xF>(0, v); });
    at([](int v) { return dpp<0x142, 0xA>(0, v); });
    at([](int v) { return dpp<0x143, 0xC>(0, v); });
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}

// Exclusive sum of one value per thread over the workgroup (NT threads), and
// the whole sum; part: NT / 64 values of its own for each call.
template <int NT>
__device__ __forceinline__ int block_scan(int x, int* part, int& total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sum = wave_scan(x);
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    const int waves = wave_scan(lane < NT / 64 ? part[lane] : 0);
    total = __builtin_amdgcn_readlane(waves, NT / 64 - 1);
    return (wave > 0 ? __builtin_amdgcn_readlane(waves, wave > 0 ? wave - 1 : 0) : 0) + sum - x;
}

// Of three values at once, one barrier for all; part: 3 NT / 64 values.
template <int NT>
__device__ __forceinline__ void block_scan3(int (&x)[3], int* part, int (&total)[3]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int sum[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        sum[i] = wave_scan(x[i]);
        if (lane == 63) part[i * (NT / 64) + wave] = sum[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int waves = wave_scan(lane < NT / 64 ? part[i * (NT / 64) + lane] : 0);
        total[i] = __builtin_amdgcn_readlane(waves, NT / 64 - 1);
        x[i] = (wave > 0 ? __builtin_amdgcn_readlane(waves, wave > 0 ? wave - 1 : 0) : 0) + sum[i] - x[i];
    }
}

// largest s in [0, n) with a[s] <= x (a ascends, a[0] <= x)
template <typename T>
__device__ __forceinline__ int find_last(const T* a, int n, T x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (a[m] <= x) lo = m;
        else hi = m;
    }
    return lo;
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kPlanItems = 4096;  // items whose costs are weighed against each other

constexpr int kBuckets = 128;     // of pieces' costs, four to a doubling, narrow and wide

// The place in the launch of a piece of an item's k: of those that go `first`
// or of the others, longest first
__device__ __forceinline__ int plan_bucket(int cost, bool first, int k) {
    const int c = min(kBuckets / 2 - 1, max(0, (int)(__float_as_uint((float)cost / (float)k) >> 21) - (127 << 2)));
    return (first ? kBuckets / 2 - 1 : kBuckets - 1) - c;
}

struct PlanWeighLds {
    float est[kPlanWaves], limit[kPlanWaves];
    int hist[kPlanWaves][64];
};

// 1 / the limit on a piece's cost: each wave weighs one by the time that the
// step would take.  costs: of the items, in LDS (behind a barrier); a wide
// item's is negative, kWideCost a chunk, and a multiple.  SHARED: items that
// are one piece write partials, too.
template <bool SHARED>
__device__ __forceinline__ float plan_limit(const int* costs, int n_items, int fill, int max_slots, PlanWeighLds& x) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto& est = x.est;
    auto& limit = x.limit;
    auto& hist = x.hist;
    float total = 0.f;
    for (int i = lane; i < n_items; i += 64) total += (float)abs(costs[i]);
    const float share = fmaxf(wave_sum(total) / (float)fill, (float)kMinPiece);
    // wave w's limit: 0.72 .. 2.26 shares, the last wave's none (0.5 .. 3 and a
    // second round about the best: 3 us more, and steps as long)
    const float mine = wave == kPlanWaves - 1
                           ? 1e9f
                           : fmaxf(share * 0.72f * fast_exp2((float)wave * (1.65f / (kPlanWaves - 2))), (float)kMinPiece);
    const float inv = 1.f / mine;
    float time = 0.f, longest = 0.f;
    int pieces = 0, slots = 0;
    for (int i = lane; i < n_items; i += 64) {
        const int c = abs(costs[i]);
        const bool wide = costs[i] < 0;
        const int chunks = wide ? c / kWideCost : c;
        const int k = item_pieces(c, chunks, inv), m = k > 1 ? (int)ceilf((float)chunks / (float)k) : chunks;
        time += PlanCost::share(wide, m, SHARED || k > 1) * (float)k;
        longest = fmaxf(longest, PlanCost::piece(wide, m));
        pieces += k;
        slots += k > 1 ? k : 0;
    }
    time = wave_sum(time);
    longest = wave_fold(longest, [](float a, float b) { return fmaxf(a, b); });
    pieces = wave_sum(pieces);
    slots = wave_sum(slots);
    float last = longest;
    if (pieces > fill) {
        // Of more than g `fill` pieces, the g + 1 that share a slot are
        // at least as long as number g `fill` + 1 (longest first).  A
        // histogram of the lengths, in 64ths of the longest, finds it.
        hist[wave][lane] = 0;
        const float scale = 63.99f / longest;
        for (int i = lane; i < n_items; i += 64) {
            const int c = abs(costs[i]);
            const bool wide = costs[i] < 0;
            const int chunks = wide ? c / kWideCost : c;
            const int k = item_pieces(c, chunks, inv), m = k > 1 ? (int)ceilf((float)chunks / (float)k) : chunks;
            atomicAdd(&hist[wave][(int)(PlanCost::piece(wide, m) * scale)], k);
        }
        __builtin_amdgcn_wave_barrier();
        const int have = hist[wave][lane], longer = pieces - wave_scan(have) + have;  // as long as this bucket's
        for (int g = 1; g <= 3 && pieces > g * fill; ++g) {
            const int b = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(longer > g * fill) | 1);
            last = fmaxf(last, (float)(g + 1) * ((float)b + 0.5f) / scale);
        }
    }
    if (lane == 0) {
        est[wave] = slots <= max_slots ? PlanCost::step(time / (float)fill, last) : INFINITY;
        limit[wave] = mine;
    }
    __syncthreads();
    float best = INFINITY, l0 = 1e9f;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const float e = est[w];
        l0 = e < best ? limit[w] : l0;
        best = fminf(best, e);
    }
    return 1.f / l0;  // (the last wave's splits nothing, and is always one to take)
}

}  // namespace pelica

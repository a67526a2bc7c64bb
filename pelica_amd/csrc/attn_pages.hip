// One step's page bookkeeping and the attention's work list, on the GPU from
// the requests' lengths.
//
// All of it is integer sums over the requests (at most 4096) and then
// independent writes: new pages' table entries, per row a slot, a position
// and a request, per item its pieces.  Latency-bound: a launch, one round
// trip for the lengths, the scan, one for the list's entries, the stores.
// pages_append runs as many workgroups as its rows fill; each scans all
// requests by itself (8 bytes a request from L2), which costs less than a
// second launch or a wait between workgroups.
// Measured: 8 requests 3.6 us, 500 with prompts of up to 600 tokens 5.9, the
// release of 31 of them 4.1.
#include "attn_paged.hpp"
#include "attn_prof.hpp"

namespace pelica {

namespace {

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

// One where a wave's sum fits 32 bits and the workgroup's may not.
template <int NT>
__device__ __forceinline__ int64_t block_scan_long(int x, int* part, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sum = wave_scan(x);
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        before += w < wave ? part[w] : 0;
        all += part[w];
    }
    total = all;
    return before + sum - x;
}
// The same for any values.
template <int NT>
__device__ __forceinline__ int64_t block_scan_any(int64_t x, int64_t* part, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t sum = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t y = __shfl_up(sum, off, 64);
        if (lane >= off) sum += y;
    }
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        before += w < wave ? part[w] : 0;
        all += part[w];
    }
    total = all;
    return before + sum - x;
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

// place of a queue's entry number x in its ring
__device__ __forceinline__ int64_t queue_at(int64_t x, int n) {
    const int64_t r = x % n;
    return r < 0 ? r + n : r;
}

constexpr int kPagesThreads = 256;

__global__ __launch_bounds__(kPagesThreads) void pages_append_kernel(PagesParams p) {
    __shared__ int len[kPagedMaxSeq], add[kPagedMaxSeq];  // cached and new tokens of each request
    __shared__ int qs[kPagedMaxSeq + 1];     // its first row
    __shared__ int first[kPagedMaxSeq + 1];  // its first new page's number within the step
    __shared__ int part[2 * kPagesThreads / 64];
    __shared__ int served_end;
    const int tid = threadIdx.x;
    // (whatever the state holds, no entry outside the list is touched)
    const int64_t taken = p.free_in[0], given = p.free_in[1], avail = min<int64_t>(given - taken, p.n_pages);
    if (tid == 0) served_end = 0;
    for (int s = tid; s < p.n_seq; s += kPagesThreads) {
        len[s] = p.cached[s];
        add[s] = p.fresh[s];
    }
    __syncthreads();

    const int per = (p.n_seq + kPagesThreads - 1) / kPagesThreads;
    const int s0 = min(tid * per, p.n_seq), s1 = min(s0 + per, p.n_seq);
    struct Need {
        int c, n, have, pages, status;
    };
    // (n is cut off behind the last row, at 2^20 + 1 at most: such a request is
    // refused, and 1024 of them, a wave's, sum to less than 2^31)
    auto look = [&](int s) {
        Need x;
        const int c = len[s], n = add[s];
        const int64_t sum = (int64_t)c + n;
        x.status = c < 0 || n < 0 || sum > INT32_MAX ? 4 : 0;
        x.c = x.status ? 0 : c;
        x.n = min(max(n, 0), p.n_tokens + 1);
        const int64_t psz = 1LL << p.page_log2;
        x.have = (int)((x.c + psz - 1) >> p.page_log2);
        const int want = (int)((x.c + (int64_t)x.n + psz - 1) >> p.page_log2);
        if (!x.status && (sum + psz - 1) >> p.page_log2 > p.max_pages) x.status = 2;
        x.pages = x.status ? 0 : want - x.have;
        return x;
    };
    // rows and pages of the requests before.  Rows run out for a request and
    // every later one that has any, so that pages counted for it are no one
    // else's loss.
    int rows = 0, pages = 0;
    for (int s = s0; s < s1; ++s) {
        const Need x = look(s);
        rows += x.n;
        pages += x.pages;
    }
    int64_t all_rows, all_pages;
    int64_t row = block_scan_long<kPagesThreads>(rows, part, all_rows);
    int64_t page = block_scan_long<kPagesThreads>(pages, part + kPagesThreads / 64, all_pages);
    int served = 0;
    for (int s = s0; s < s1; ++s) {
        Need x = look(s);
        qs[s] = (int)min<int64_t>(row, p.n_tokens);
        first[s] = (int)page;
        row += x.n;
        page += x.pages;
        if (x.status == 0 && x.n > 0 && row > p.n_tokens) x.status = 3;
        if (x.status == 0 && x.pages > 0) {
            if (page > avail) x.status = 1;
            else served = (int)page;
        }
        if (blockIdx.x == 0) {
            p.q_start[s] = qs[s];
            p.kv_len[s] = x.status ? 0 : x.c + x.n;
            p.status[s] = x.status;
        }
    }
    // (the requests that get their pages are the first ones that need any)
    if (served > 0) atomicMax(&served_end, served);
    if (tid == 0) {
        qs[p.n_seq] = (int)min<int64_t>(all_rows, p.n_tokens);
        first[p.n_seq] = (int)all_pages;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        p.q_start[p.n_seq] = qs[p.n_seq];
        p.free_out[0] = taken + served_end;
        p.free_out[1] = given;
    }
    // page number i of the step, a queue entry
    const int64_t begin = queue_at(taken, p.n_pages);
    auto entry = [&](int i) {
        int64_t j = begin + i;
        if (j >= p.n_pages) j -= p.n_pages;  // (fewer pages than the queue has are taken)
        const int id = p.list[j];
        return (unsigned)id < (unsigned)p.n_pages ? id : -1;
    };
    const int nt = gridDim.x * kPagesThreads, g = blockIdx.x * kPagesThreads + tid;
    // new pages into the table
    for (int i = g; i < served_end; i += nt) {
        const int s = find_last(first, p.n_seq, i);
        const int have = (int)(((int64_t)len[s] + (1LL << p.page_log2) - 1) >> p.page_log2);
        p.table[(size_t)s * p.max_pages + have + (i - first[s])] = entry(i);
    }
    // rows
    for (int i = g; i < p.n_tokens; i += nt) {
        int64_t slot = -1;
        int pos = 0, seq = -1;
        if (i < qs[p.n_seq]) {
            const int s = find_last(qs, p.n_seq, i);
            const Need x = look(s);
            pos = x.c + (i - qs[s]);
            seq = s;
            if (x.status == 0 && qs[s] + x.n <= p.n_tokens && (x.pages == 0 || first[s] + x.pages <= avail)) {
                const int j = pos >> p.page_log2;
                int id;
                if (j < x.have) {
                    id = p.table[(size_t)s * p.max_pages + j];
                    if ((unsigned)id >= (unsigned)p.n_pages) id = -1;
                } else {
                    id = entry(first[s] + j - x.have);
                }
                if (id >= 0) slot = ((int64_t)id << p.page_log2) + (pos & ((1 << p.page_log2) - 1));
            }
        }
        p.slots[i] = slot;
        p.positions[i] = pos;
        p.token_seq[i] = seq;
    }
}

__global__ __launch_bounds__(kPagesThreads) void pages_release_kernel(PagesParams p) {
    __shared__ int count[kPagedMaxSeq];  // pages each request gives back
    __shared__ int64_t first[kPagedMaxSeq + 1];
    __shared__ int64_t part[kPagesThreads / 64];
    const int tid = threadIdx.x;
    const int64_t taken = p.free_in[0], given = p.free_in[1];
    for (int s = tid; s < p.n_seq; s += kPagesThreads) {
        const int64_t held = ((int64_t)p.cached[s] + (1LL << p.page_log2) - 1) >> p.page_log2;
        count[s] = p.ended[s] == 0 || p.cached[s] <= 0 ? 0 : (int)min<int64_t>(held, p.max_pages);
    }
    __syncthreads();
    const int per = (p.n_seq + kPagesThreads - 1) / kPagesThreads;
    const int s0 = min(tid * per, p.n_seq), s1 = min(s0 + per, p.n_seq);
    int64_t n = 0, total;
    for (int s = s0; s < s1; ++s) n += count[s];
    int64_t at = block_scan_any<kPagesThreads>(n, part, total);
    for (int s = s0; s < s1; ++s) {
        first[s] = at;
        at += count[s];
    }
    __syncthreads();
    if (given - taken + total > p.n_pages || total > p.n_pages) total = 0;
    if (blockIdx.x == 0 && tid == 0) {
        p.free_out[0] = taken;
        p.free_out[1] = given + total;
    }
    const int64_t begin = queue_at(given, p.n_pages);
    for (int64_t i = (int64_t)blockIdx.x * kPagesThreads + tid; i < total; i += (int64_t)gridDim.x * kPagesThreads) {
        const int s = find_last(first, p.n_seq, i);
        const int64_t j = begin + i;
        p.list[j >= p.n_pages ? j - p.n_pages : j] = p.table[(size_t)s * p.max_pages + (i - first[s])];
    }
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kPlanItems = 4096;  // items whose costs are weighed against each other

constexpr int kBuckets = 128;     // of pieces' costs, four to a doubling, narrow and wide

// The work list.  Items (requests' blocks of query rows) cost the chunks they
// walk; an item of k pieces is cut into equal ranges of them by a limit on a
// piece's cost.  Limits are weighed, a wave each, by the time that the step
// would take (PlanCost).  Latency-bound, one workgroup: the lengths' round
// trip, the scan, the limits, the pieces: 3.5 us for a step that is not split,
// 7.6 for one long request's token, 9 - 11 for 32 requests or a prompt's 250
// items; once a step, for all its layers.
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanParams p) {
    __shared__ int item0[kPagedMaxSeq + 1];  // first item of each request
    __shared__ int q0[kPagedMaxSeq + 1], kv[kPagedMaxSeq], pre[kPagedMaxSeq];  // q_start, kv_len, prefix
    __shared__ int costs[kPlanItems];
    __shared__ int part[kPlanWaves], part3[3 * kPlanWaves], decreasing;
    __shared__ float est[kPlanWaves], limit[kPlanWaves];
    __shared__ int at_bucket[kBuckets], hist[kPlanWaves][64];
    __shared__ int piece0[kPlanThreads + 1], place[kPlanThreads], slot0[kPlanThreads], seq_of[kPlanThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int W = wide_rows(p.hd);
    for (int s = tid; s <= p.n_seq; s += kPlanThreads) {
        q0[s] = p.q_start[s];
        if (s < p.n_seq) {
            kv[s] = p.kv_len[s];
            pre[s] = p.prefix ? p.prefix[s] : 0;
        }
    }
    if (tid < kBuckets) at_bucket[tid] = 0;
    if (tid == 0) decreasing = 0;
    __syncthreads();

    // tokens of a request; 0: no item (none, or lengths that do not fit together)
    auto tokens = [&](int s) {
        const int64_t a = q0[s], b = q0[s + 1], T = b - a;
        const bool ok = a >= 0 && b <= p.n_tokens && T > 0 && T <= p.max_q && kv[s] >= T && kv[s] <= p.max_keys;
        return ok ? (int)T : 0;
    };
    auto items_of = [&](int T) {
        const int R = T * p.hpk;
        return R <= kNarrowRows ? (R > 0 ? 1 : 0) : (R + W - 1) / W;
    };
    const int per = (p.n_seq + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(tid * per, p.n_seq), s1 = min(s0 + per, p.n_seq);
    int n = 0, n_items;
    for (int s = s0; s < s1; ++s) {
        n += items_of(tokens(s));
        // (rows of two requests: their items could be more than there is room for)
        if (q0[s + 1] < q0[s]) decreasing = 1;
    }
    int at = block_scan<kPlanThreads>(n, part, n_items);
    for (int s = s0; s < s1; ++s) {
        item0[s] = at;
        at += items_of(tokens(s));
    }
    if (tid == 0) item0[p.n_seq] = n_items;
    __syncthreads();
    if (decreasing) n_items = 0;

    // r / hpk (r < 2^30), as (r + 1/2) / hpk in f64: at least 1 / (2 hpk) from
    // a whole number, hpk <= 2^16
    const double inv_hpk = 1.0 / p.hpk;
    auto token = [&](int r) { return (int)(((double)r + 0.5) * inv_hpk); };
    struct Item {
        int s, T, r0, R, cost;
        ItemKeys k;
    };
    auto item_of = [&](int i, int s) {
        Item x;
        x.s = s;
        x.T = tokens(x.s);
        x.R = x.T * p.hpk;
        const bool narrow = x.R <= kNarrowRows;
        x.r0 = narrow ? 0 : (i - item0[x.s]) * W;
        const int rows = narrow ? x.R : imin(W, x.R - x.r0);
        const int pos0 = kv[x.s] - x.T;
        x.k = item_keys(pos0 + token(x.r0), pos0 + token(x.r0 + rows - 1), kv[x.s], p.window, pre[x.s]);
        x.cost = x.k.n_chunks * (narrow ? 1 : kWideCost);
        return x;
    };
    // (requests without items share their first item with the next one: the
    // last of them is the one that has it)
    auto item = [&](int i) { return item_of(i, find_last(item0, p.n_seq, i)); };
    // this thread's first item, the only one of most steps
    const Item own = tid < n_items ? item(tid) : Item{};
    auto item_at = [&](int i) { return i < kPlanThreads ? own : item(i); };

    auto piece = [&](const Item& y, int of, int nth, int slot) {
        PlanPiece z;
        z.seq = y.s;
        z.q0 = q0[y.s];
        z.R = y.R;
        z.r0 = y.r0;
        z.pos0 = kv[y.s] - y.T;
        z.len = kv[y.s];
        z.cb = (int)((int64_t)y.k.n_chunks * nth / of);
        z.ce = (int)((int64_t)y.k.n_chunks * (nth + 1) / of);
        z.slot = slot;
        z.n_pre = y.k.n_pre;
        z.lo_base = y.k.lo_base;
        z.lo = y.k.lo;
        z.kend = y.k.kend;
        z.pe = y.k.pe;
        z.pad[0] = z.pad[1] = 0;
        return z;
    };
    auto header = [&](int pieces, int joins) {
        PlanHeader h{};
        h.sig = p.sig;
        h.n_pieces = min(pieces, p.max_pieces);
        h.n_joins = min(joins, p.max_joins);
        return h;
    };
    // Narrow pieces start first, longest first: they wait for memory while
    // the wide ones beside them keep the matrix cores busy
    auto bucket_of = [&](const Item& x, int k) {
        const int c = min(kBuckets / 2 - 1, max(0, (int)(__float_as_uint((float)x.cost / (float)k) >> 21) - (127 << 2)));
        return (x.R <= kNarrowRows ? kBuckets / 2 - 1 : kBuckets - 1) - c;
    };
    // a step that is not split: an item a piece, in order
    if (!p.split) {
        for (int i = tid; i < n_items; i += kPlanThreads)
            if (i < p.max_pieces) p.pieces[i] = piece(item_at(i), 1, 0, -1);
        if (tid == 0) *p.head = header(n_items, 0);
        return;
    }

    float inv_limit = 0.f;  // (no limit)
    if (n_items > 0 && n_items <= kPlanItems) {
        // (a wide item's cost is negative: kWideCost a chunk, and a multiple)
        for (int i = tid; i < n_items; i += kPlanThreads) {
            const Item x = item_at(i);
            costs[i] = x.R <= kNarrowRows ? x.cost : -x.cost;
        }
        __syncthreads();
        float total = 0.f;
        for (int i = lane; i < n_items; i += 64) total += (float)abs(costs[i]);
        const float share = fmaxf(wave_sum(total) / (float)p.fill, (float)kMinPiece);
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
            time += PlanCost::share(wide, m, k > 1) * (float)k;
            longest = fmaxf(longest, PlanCost::piece(wide, m));
            pieces += k;
            slots += k > 1 ? k : 0;
        }
        time = wave_sum(time);
        longest = wave_fold(longest, [](float a, float b) { return fmaxf(a, b); });
        pieces = wave_sum(pieces);
        slots = wave_sum(slots);
        float last = longest;
        if (pieces > p.fill) {
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
            for (int g = 1; g <= 3 && pieces > g * p.fill; ++g) {
                const int b = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(longer > g * p.fill) | 1);
                last = fmaxf(last, (float)(g + 1) * ((float)b + 0.5f) / scale);
            }
        }
        if (lane == 0) {
            est[wave] = slots <= p.max_slots ? PlanCost::step(time / (float)p.fill, last) : INFINITY;
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
        inv_limit = 1.f / l0;  // (the last wave's splits nothing, and is always one to take)
    }

    // where each bucket's pieces begin
    for (int i = tid; i < n_items; i += kPlanThreads) {
        const Item x = item_at(i);
        const int k = item_pieces(x.cost, x.k.n_chunks, inv_limit);
        atomicAdd(&at_bucket[bucket_of(x, k)], k);
    }
    __syncthreads();
    if (wave == 0) {
        static_assert(kBuckets == 128, "two buckets a lane");
        const int a = at_bucket[2 * lane], b = at_bucket[2 * lane + 1], sum = wave_scan(a + b);
        at_bucket[2 * lane] = sum - a - b;
        at_bucket[2 * lane + 1] = sum - b;
    }
    __syncthreads();

    int n_pieces = 0, base_slot = 0, base_join = 0;
    for (int b = 0; b < n_items; b += kPlanThreads) {
        const int i = b + tid;
        Item x{};
        int k = 0;
        if (i < n_items) {
            x = item_at(i);
            k = item_pieces(x.cost, x.k.n_chunks, inv_limit);
        }
        // pieces of the items before, and split items' pieces and items
        int before[3] = {k, k > 1 ? k : 0, k > 1 ? 1 : 0}, all[3];
        block_scan3<kPlanThreads>(before, part3, all);
        const int sl = base_slot + before[1], jn = base_join + before[2];
        piece0[tid] = before[0];
        seq_of[tid] = x.s;
        place[tid] = k > 0 ? atomicAdd(&at_bucket[bucket_of(x, k)], k) : 0;
        slot0[tid] = k > 1 ? sl : -1;
        if (k > 1 && jn < p.max_joins) p.joins[jn] = PlanJoin{q0[x.s], x.R, x.r0, sl, k, {}};
        __syncthreads();
        const int n_here = min(kPlanThreads, n_items - b);
        for (int j = tid; j < all[0]; j += kPlanThreads) {
            const int t = find_last(piece0, n_here, j);
            const Item y = item_of(b + t, seq_of[t]);
            const int of = item_pieces(y.cost, y.k.n_chunks, inv_limit), nth = j - piece0[t];
            if (place[t] + nth < p.max_pieces)
                p.pieces[place[t] + nth] = piece(y, of, nth, slot0[t] < 0 ? -1 : slot0[t] + nth);
        }
        n_pieces += all[0];
        base_slot += all[1];
        base_join += all[2];
        __syncthreads();
    }
    if (tid == 0) *p.head = header(n_pieces, base_join);
}

}  // namespace

hipError_t launch_pages_append(const PagesParams& p, hipStream_t st) {
    const int grid = min((p.n_tokens + kPagesThreads - 1) / kPagesThreads, 256);
    ProfScope ps(kProfPages, st);
    hipLaunchKernelGGL(pages_append_kernel, dim3(grid), dim3(kPagesThreads), 0, st, p);
    return hipGetLastError();
}

hipError_t launch_pages_release(const PagesParams& p, hipStream_t st) {
    ProfScope ps(kProfPages, st);
    hipLaunchKernelGGL(pages_release_kernel, dim3(p.n_seq <= 64 ? 4 : 16), dim3(kPagesThreads), 0, st, p);
    return hipGetLastError();
}

hipError_t launch_paged_plan(const PlanParams& p, hipStream_t st) {
    ProfScope ps(kProfPagedPlan, st);
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    return hipGetLastError();
}

}  // namespace pelica

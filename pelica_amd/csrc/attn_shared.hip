// The work list of a step whose requests share their first keys: a prompt or
// a document that many requests begin with lies in the cache once, and its
// keys are walked once for all of them.
//
// A group is consecutive requests with the same first pages.  Their query rows
// lie side by side, so to the attention kernels the group is one more request:
// all its rows (token, head) over the shared keys [0, e), every one of which
// every row sees, in blocks of wide_rows.  Each request is an item over its own
// keys, from e on.  Both leave partials (m, l, O), and the join adds a row's:
//   M = max m_i,  O = sum 2^(m_i - M) O_i,  L = sum 2^(m_i - M) l_i,
// with the sink as for the pieces of one item.  e is a multiple of 32 keys: no
// chunk is walked twice, and no mask is needed ahead of e.
//
// One workgroup, latency-bound as the plain plan: groups first (their lengths'
// minimum by LDS atomics, whose order does not matter), then items, groups'
// ahead of requests', weighed and cut alike: 9.6 us for 8 requests, 12.5 for 60 in 3
// groups (the plain plan's 7 - 8 and what finding the groups takes).
// A layer of 64 readers of 16384 keys, 64 / 8 heads of 64, f32: 58 us + join 5.8
// (plain plan 154 + 4.6; the keys' bytes 26, the shared keys' products 25); 60 requests
// of three prompts, 32 / 4 of 128, f16: 45.5 + 5.0 (56.5 + 4.9; bytes 42).  Few readers gain
// nothing, 8 of 2000 keys 11.4 + 3.8 (11.4 + 4.0), and lose below: 8 of 250 keys 12 us a
// layer with the join (10).  Prompts' chunks lose: three of 700 tokens among 16 requests behind
// 13000 keys 833 + 19 (676 + 7).  Every group is walked as it is told.
#include "attn_paged.hpp"
#include "attn_plan_weigh.hpp"
#include "attn_prof.hpp"

namespace pelica {

namespace {

__global__ __launch_bounds__(kPlanThreads) void paged_shared_plan_kernel(SharedPlanParams sp) {
    const PlanParams& p = sp.plan;
    __shared__ int item0[kPagedMaxSeq + 1];   // first item of each request, behind the groups'
    __shared__ int q0[kPagedMaxSeq + 1], kv[kPagedMaxSeq];
    __shared__ int16_t group_of[kPagedMaxSeq];  // -1: none
    __shared__ int gstart[kSharedMaxGroups + 1], gitem0[kSharedMaxGroups + 1];
    __shared__ int ge[kSharedMaxGroups];      // shared keys that are walked once
    __shared__ int gcount[kSharedMaxGroups], gfirst[kSharedMaxGroups], glast[kSharedMaxGroups];  // requests with tokens
    __shared__ int gat[kSharedMaxGroups], gk[kSharedMaxGroups];    // partials: first row, pieces of a block
    __shared__ int gat2[kSharedMaxGroups], gk2[kSharedMaxGroups];  // of the last block
    __shared__ int costs[kPlanItems];
    __shared__ int part[kPlanWaves], part3[3 * kPlanWaves], bad;
    __shared__ PlanWeighLds weigh;
    __shared__ int at_bucket[kBuckets];
    __shared__ int piece0[kPlanThreads + 1], place[kPlanThreads], row0[kPlanThreads], owner[kPlanThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int W = wide_rows(p.hd);
    for (int s = tid; s <= p.n_seq; s += kPlanThreads) {
        q0[s] = p.q_start[s];
        if (s < p.n_seq) {
            kv[s] = p.kv_len[s];
            group_of[s] = -1;
        }
    }
    for (int g = tid; g <= sp.n_groups; g += kPlanThreads) {
        gstart[g] = sp.group_start[g];
        if (g < sp.n_groups) {
            ge[g] = sp.shared_len[g];
            gcount[g] = 0;
            gfirst[g] = kPagedMaxSeq;
            glast[g] = gat[g] = gk[g] = gat2[g] = gk2[g] = 0;
        }
    }
    if (tid < kBuckets) at_bucket[tid] = 0;
    if (tid == 0) bad = 0;
    __syncthreads();
    // tokens of a request; 0: no item (none, or lengths that do not fit together)
    auto tokens = [&](int s) {
        const int64_t a = q0[s], b = q0[s + 1], T = b - a;
        const bool ok = a >= 0 && b <= p.n_tokens && T > 0 && T <= p.max_q && kv[s] >= T && kv[s] <= p.max_keys;
        return ok ? (int)T : 0;
    };
    // (rows of two requests, requests of two groups: more items than there is room for)
    for (int s = tid; s < p.n_seq; s += kPlanThreads)
        if (q0[s + 1] < q0[s]) bad = 1;
    for (int g = tid; g <= sp.n_groups; g += kPlanThreads)
        if (gstart[g] < 0 || gstart[g] > p.n_seq || (g < sp.n_groups && gstart[g + 1] < gstart[g])) bad = 1;
    __syncthreads();
    if (bad) {
        if (tid == 0) {
            PlanHeader h{};
            h.sig = p.sig;
            *p.head = h;
        }
        return;
    }
    for (int s = tid; s < p.n_seq; s += kPlanThreads) {
        const int T = tokens(s);
        if (s < gstart[0] || s >= gstart[sp.n_groups]) continue;
        // (of empty groups that begin at one request the last holds it)
        const int g = find_last(gstart, sp.n_groups, s);
        group_of[s] = (int16_t)g;
        if (T == 0) continue;
        atomicAdd(&gcount[g], 1);
        atomicMin(&gfirst[g], s);
        atomicMax(&glast[g], s);
        atomicMin(&ge[g], kv[s] - T);  // (a token's own keys are not shared)
    }
    __syncthreads();
    auto blocks_of = [&](int R) { return R <= kNarrowRows ? (R > 0 ? 1 : 0) : (R + W - 1) / W; };
    auto group_rows_of = [&](int g) { return ge[g] > 0 ? (q0[glast[g] + 1] - q0[gfirst[g]]) * p.hpk : 0; };
    int n_group_items;
    {
        int n = 0;
        if (tid < sp.n_groups) {
            ge[tid] = gcount[tid] > 1 && ge[tid] > 0 ? ge[tid] & ~31 : 0;
            n = blocks_of(group_rows_of(tid));
        }
        static_assert(kSharedMaxGroups <= kPlanThreads, "a group a thread");
        const int at = block_scan<kPlanThreads>(n, part, n_group_items);
        if (tid < sp.n_groups) gitem0[tid] = at;
        if (tid == 0) gitem0[sp.n_groups] = n_group_items;
    }
    __syncthreads();
    const int per = (p.n_seq + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(tid * per, p.n_seq), s1 = min(s0 + per, p.n_seq);
    int n = 0, n_items;
    for (int s = s0; s < s1; ++s) n += blocks_of(tokens(s) * p.hpk);
    int at = block_scan<kPlanThreads>(n, part, n_items) + n_group_items;
    for (int s = s0; s < s1; ++s) {
        item0[s] = at;
        at += blocks_of(tokens(s) * p.hpk);
    }
    n_items += n_group_items;
    if (tid == 0) item0[p.n_seq] = n_items;
    __syncthreads();

    // r / hpk (r < 2^30), as (r + 1/2) / hpk in f64: at least 1 / (2 hpk) from
    // a whole number, hpk <= 2^16
    const double inv_hpk = 1.0 / p.hpk;
    auto token = [&](int r) { return (int)(((double)r + 0.5) * inv_hpk); };
    struct Item {
        int group, s;      // the group it is of (a request's: its own, or -1), its (first) request
        bool shared, narrow;  // of the group's shared keys; at most kNarrowRows rows
        int T, r0, R, rows, cost;
        int n_chunks, lo, kend;
    };
    auto item_of = [&](int i, int owner) {
        Item x;
        x.shared = i < n_group_items;
        int e, pos0;
        if (x.shared) {
            x.group = owner;
            x.s = gfirst[owner];
            x.R = group_rows_of(owner);
            x.T = 0;
            pos0 = ge[owner] - 1;  // (every row sees all of them)
            e = 0;
        } else {
            x.group = group_of[owner];
            x.s = owner;
            x.T = tokens(owner);
            x.R = x.T * p.hpk;
            pos0 = kv[owner] - x.T;
            e = x.group >= 0 ? ge[x.group] : 0;
        }
        x.narrow = x.R <= kNarrowRows;
        x.r0 = x.narrow ? 0 : (i - (x.shared ? gitem0[owner] : item0[owner])) * W;
        x.rows = x.narrow ? x.R : imin(W, x.R - x.r0);
        // (a group's last block may be as small as a request's item: 17 requests of
        // 8 heads a kv head, head dim 128: 128 rows and 8)
        if (x.shared && x.rows <= kNarrowRows) x.narrow = true;
        x.lo = e;
        x.kend = x.shared ? ge[owner] : pos0 + token(x.r0 + x.rows - 1) + 1;
        x.n_chunks = (x.kend - x.lo + 31) >> 5;
        x.cost = x.n_chunks * (x.narrow ? 1 : kWideCost);
        return x;
    };
    auto owner_of = [&](int i) { return i < n_group_items ? find_last(gitem0, sp.n_groups, i) : find_last(item0, p.n_seq, i); };
    auto item = [&](int i) { return item_of(i, owner_of(i)); };
    // this thread's first item, the only one of most steps
    const Item own = tid < n_items ? item(tid) : Item{};
    auto item_at = [&](int i) { return i < kPlanThreads ? own : item(i); };
    // partials: of a group's keys, of requests that have such, of split items
    auto partial = [&](const Item& x, int k) { return x.shared || k > 1 || x.lo > 0; };

    float inv_limit = 0.f;  // (no limit)
    if (n_items > 0 && n_items <= kPlanItems) {
        for (int i = tid; i < n_items; i += kPlanThreads) {
            const Item x = item_at(i);
            costs[i] = x.narrow ? x.cost : -x.cost;
        }
        __syncthreads();
        inv_limit = plan_limit<true>(costs, n_items, p.fill, p.max_slots, weigh);
    }

    // Wide pieces first, longest first, unlike the plain plan's: a group's are few
    // and long, about one a CU, and the requests' narrow ones, which come next, wait for
    // memory beside them.  Narrow ones first fill both slots of every CU, and the wide ones
    // follow alone (64 readers of 16384 keys 77 -> 57 us, drafts 66 -> 59, 60 requests of
    // three prompts 47 -> 46; f32, three prompts 51 -> 46).  Wide chunks weighed at 4, 5, 7
    // instead of 3: 70, 65, 68 us of the 57.
    auto bucket_of = [&](const Item& x, int k) { return plan_bucket(x.cost, !x.narrow, k); };
    for (int i = tid; i < n_items; i += kPlanThreads) {
        const Item x = item_at(i);
        const int k = item_pieces(x.cost, x.n_chunks, inv_limit);
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

    int n_pieces = 0, base_row = 0, base_join = 0;
    for (int b = 0; b < n_items; b += kPlanThreads) {
        const int i = b + tid;
        Item x{};
        int k = 0;
        if (i < n_items) {
            x = item_at(i);
            k = item_pieces(x.cost, x.n_chunks, inv_limit);
        }
        const bool parts = k > 0 && partial(x, k), joined = parts && !x.shared;
        // of the items before: pieces, partial rows, joins
        int before[3] = {k, parts ? k * x.rows : 0, joined ? 1 : 0}, all[3];
        block_scan3<kPlanThreads>(before, part3, all);
        const int row = base_row + before[1], jn = base_join + before[2];
        piece0[tid] = before[0];
        owner[tid] = x.shared ? x.group : x.s;
        place[tid] = k > 0 ? atomicAdd(&at_bucket[bucket_of(x, k)], k) : 0;
        row0[tid] = parts ? row : -1;
        // (all but a group's last block are whole, and cut alike)
        if (k > 0 && x.shared) {
            if (x.r0 == 0) gat[x.group] = row, gk[x.group] = k;
            if (x.r0 + x.rows == x.R) gat2[x.group] = row, gk2[x.group] = k;
        }
        __syncthreads();
        if (joined && jn < p.max_joins) {
            const int g = x.group;
            const bool with = g >= 0 && ge[g] > 0;
            SharedJoin j{};
            j.q0 = q0[x.s];
            j.r0 = x.r0;
            j.rows = x.rows;
            j.at = row;
            j.k = k;
            if (with) {
                j.g_at = gat[g];
                j.g_k = gk[g];
                j.g_row = (q0[x.s] - q0[gfirst[g]]) * p.hpk + x.r0;
                j.g_R = group_rows_of(g);
                j.g_at2 = gat2[g];
                j.g_k2 = gk2[g];
            }
            sp.joins[jn] = j;
        }
        const int n_here = min(kPlanThreads, n_items - b);
        for (int j = tid; j < all[0]; j += kPlanThreads) {
            const int t = find_last(piece0, n_here, j);
            const Item y = item_of(b + t, owner[t]);
            const int of = item_pieces(y.cost, y.n_chunks, inv_limit), nth = j - piece0[t];
            if (place[t] + nth >= p.max_pieces) continue;
            PlanPiece z;
            z.seq = y.s;
            z.q0 = q0[y.s];
            z.R = y.R;
            z.r0 = y.r0;
            z.pos0 = y.shared ? y.kend - 1 : kv[y.s] - y.T;
            z.len = y.shared ? y.kend : kv[y.s];
            z.cb = (int)((int64_t)y.n_chunks * nth / of);
            z.ce = (int)((int64_t)y.n_chunks * (nth + 1) / of);
            z.slot = row0[t] < 0 ? -1 : row0[t] + nth * y.rows;
            z.n_pre = 0;
            z.lo_base = z.lo = y.lo;
            z.kend = y.kend;
            z.pe = 0;
            z.rows = y.rows;
            z.narrow = y.shared && y.narrow;
            p.pieces[place[t] + nth] = z;
        }
        n_pieces += all[0];
        base_row += all[1];
        base_join += all[2];
        __syncthreads();
    }
    if (tid == 0) {
        PlanHeader h{};
        h.sig = p.sig;
        h.n_pieces = min(n_pieces, p.max_pieces);
        h.n_joins = min(base_join, p.max_joins);
        *p.head = h;
    }
}

}  // namespace

hipError_t launch_paged_shared_plan(const SharedPlanParams& p, hipStream_t st) {
    ProfScope ps(kProfPagedPlan, st);
    hipLaunchKernelGGL(paged_shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    return hipGetLastError();
}

}  // namespace pelica

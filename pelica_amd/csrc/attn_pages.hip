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
#include "attn_paged.hpp"
#include "attn_prof.hpp"

namespace pelica {

namespace {

// Exclusive sum of one value per thread over the workgroup (NT threads),
// and the whole sum.
template <int NT, typename T>
__device__ __forceinline__ T block_scan(T x, T* part, T& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T sum = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const T y = __shfl_up(sum, off, 64);
        if (lane >= off) sum += y;
    }
    __syncthreads();  // (part of the scan before is read)
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const T v = part[w];
        if (w < wave) before += v;
        all += v;
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

constexpr int kPagesThreads = 256;

__global__ __launch_bounds__(kPagesThreads) void pages_append_kernel(PagesParams p) {
    __shared__ int qs[kPagedMaxSeq + 1];       // first row of each request
    __shared__ int64_t first[kPagedMaxSeq + 1];  // its first new page's number within the step
    __shared__ int64_t part[kPagesThreads / 64];
    __shared__ int64_t served_end;
    const int tid = threadIdx.x;
    const int per = (p.n_seq + kPagesThreads - 1) / kPagesThreads;
    const int s0 = min(tid * per, p.n_seq), s1 = min(s0 + per, p.n_seq);
    const int64_t taken = p.free_in[0], avail = p.free_in[1] - taken;
    const int64_t psz = 1LL << p.page_log2;
    if (tid == 0) served_end = 0;

    // rows and pages of this thread's requests
    struct Need {
        int64_t c, n, have, pages;
        int status;
    };
    auto look = [&](int s) {
        Need x;
        const int c = p.cached[s], n = p.fresh[s];
        x.status = c < 0 || n < 0 || (int64_t)c + n > INT32_MAX ? 4 : 0;
        x.c = x.status ? 0 : c;
        x.n = n < 0 ? 0 : n;
        x.have = (x.c + psz - 1) >> p.page_log2;
        const int64_t want = (x.c + x.n + psz - 1) >> p.page_log2;
        if (!x.status && want > p.max_pages) x.status = 2;
        x.pages = x.status ? 0 : want - x.have;
        return x;
    };
    int64_t rows = 0;
    for (int s = s0; s < s1; ++s) rows += look(s).n;
    int64_t all_rows, all_pages;
    int64_t row = block_scan<kPagesThreads>(rows, part, all_rows);
    int64_t pages = 0;
    {
        int64_t r = row;
        for (int s = s0; s < s1; ++s) {
            const Need x = look(s);
            r += x.n;
            pages += r > p.n_tokens ? 0 : x.pages;  // (a request whose rows do not fit takes none)
        }
    }
    int64_t page = block_scan<kPagesThreads>(pages, part, all_pages);
    for (int s = s0; s < s1; ++s) {
        Need x = look(s);
        qs[s] = (int)min<int64_t>(row, p.n_tokens);
        row += x.n;
        if (row > p.n_tokens && x.n > 0 && x.status == 0) x.status = 3;
        if (x.status == 3) x.pages = 0;
        first[s] = page;
        page += x.pages;
        if (x.status == 0 && x.pages > 0 && page > avail) x.status = 1;
        if (x.status == 0 && x.pages > 0) atomicMax((unsigned long long*)&served_end, (unsigned long long)page);
        // (the requests that go unserved for want of pages are those behind avail)
        if (blockIdx.x == 0) {
            p.q_start[s] = qs[s];
            p.kv_len[s] = x.status ? 0 : (int)(x.c + x.n);
            p.status[s] = x.status;
        }
    }
    if (tid == 0) {
        qs[p.n_seq] = (int)min<int64_t>(all_rows, p.n_tokens);
        first[p.n_seq] = all_pages;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        p.q_start[p.n_seq] = qs[p.n_seq];
        p.free_out[0] = taken + served_end;
        p.free_out[1] = taken + avail;
    }
    // page number i of the step, a queue entry
    auto entry = [&](int64_t i) {
        const int id = p.list[(taken + i) % p.n_pages];
        return (unsigned)id < (unsigned)p.n_pages ? id : -1;
    };
    // new pages into the table
    const int64_t nt = (int64_t)gridDim.x * kPagesThreads, g = (int64_t)blockIdx.x * kPagesThreads + tid;
    for (int64_t i = g; i < served_end; i += nt) {
        const int s = find_last(first, p.n_seq, i);
        const Need x = look(s);
        p.table[(size_t)s * p.max_pages + x.have + (i - first[s])] = entry(i);
    }
    // rows
    for (int64_t i = g; i < p.n_tokens; i += nt) {
        int64_t slot = -1;
        int pos = 0, seq = -1;
        if (i < qs[p.n_seq]) {
            const int s = find_last(qs, p.n_seq, (int)i);
            const Need x = look(s);
            const int64_t at = x.c + (i - qs[s]);
            pos = (int)at;
            seq = s;
            const bool fits = x.status == 0 && qs[s] + x.n <= p.n_tokens;
            if (fits && (x.pages == 0 || first[s] + x.pages <= avail)) {
                const int64_t j = at >> p.page_log2;
                int id;
                if (j < x.have) {
                    id = p.table[(size_t)s * p.max_pages + j];
                    if ((unsigned)id >= (unsigned)p.n_pages) id = -1;
                } else {
                    id = entry(first[s] + j - x.have);
                }
                if (id >= 0) slot = ((int64_t)id << p.page_log2) + (at & (psz - 1));
            }
        }
        p.slots[i] = slot;
        p.positions[i] = pos;
        p.token_seq[i] = seq;
    }
}

__global__ __launch_bounds__(kPagesThreads) void pages_release_kernel(PagesParams p) {
    __shared__ int64_t first[kPagedMaxSeq + 1];
    __shared__ int64_t part[kPagesThreads / 64];
    const int tid = threadIdx.x;
    const int per = (p.n_seq + kPagesThreads - 1) / kPagesThreads;
    const int s0 = min(tid * per, p.n_seq), s1 = min(s0 + per, p.n_seq);
    const int64_t taken = p.free_in[0], given = p.free_in[1];
    auto held = [&](int s) -> int64_t {
        if (p.ended[s] == 0 || p.cached[s] <= 0) return 0;
        return min<int64_t>(((int64_t)p.cached[s] + (1LL << p.page_log2) - 1) >> p.page_log2, p.max_pages);
    };
    int64_t n = 0, total;
    for (int s = s0; s < s1; ++s) n += held(s);
    int64_t at = block_scan<kPagesThreads>(n, part, total);
    for (int s = s0; s < s1; ++s) {
        first[s] = at;
        at += held(s);
    }
    __syncthreads();
    if (given - taken + total > p.n_pages) total = 0;
    if (blockIdx.x == 0 && tid == 0) {
        p.free_out[0] = taken;
        p.free_out[1] = given + total;
    }
    for (int64_t i = (int64_t)blockIdx.x * kPagesThreads + tid; i < total; i += (int64_t)gridDim.x * kPagesThreads) {
        const int s = find_last(first, p.n_seq, i);
        p.list[(given + i) % p.n_pages] = p.table[(size_t)s * p.max_pages + (i - first[s])];
    }
}

constexpr int kPlanThreads = 1024;

// The work list.  Items (requests' blocks of query rows) cost the chunks they
// walk; where the items are fewer than fill the chip, the smallest piece
// limit is taken whose pieces are no more than fill it, so that all
// workgroups end together; else only items of over twice the mean share are
// cut.  An item's pieces are equal in chunks.
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanParams p) {
    __shared__ int item0[kPagedMaxSeq + 1];     // first item of each request
    __shared__ int64_t part[kPlanThreads / 64];
    __shared__ int piece0[kPlanThreads + 1], slot0[kPlanThreads];
    const int tid = threadIdx.x;
    const int per = (p.n_seq + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(tid * per, p.n_seq), s1 = min(s0 + per, p.n_seq);
    const int W = wide_rows(p.hd);

    struct Seq {
        int q0, T, len, prefix;
    };
    // T = 0: no item (no tokens, or lengths that do not fit together)
    auto seq = [&](int s) {
        Seq x;
        x.q0 = p.q_start[s];
        const int64_t q1 = p.q_start[s + 1];
        x.len = p.kv_len[s];
        x.prefix = p.prefix ? p.prefix[s] : 0;
        const int64_t T = q1 - x.q0;
        const bool ok = x.q0 >= 0 && q1 <= p.n_tokens && T > 0 && T <= p.max_q && x.len >= T && x.len <= p.max_keys;
        x.T = ok ? (int)T : 0;
        return x;
    };
    auto items_of = [&](const Seq& x) {
        const int R = x.T * p.hpk;
        return R <= kNarrowRows ? (R > 0 ? 1 : 0) : (R + W - 1) / W;
    };
    int64_t n = 0, total;
    for (int s = s0; s < s1; ++s) n += items_of(seq(s));
    int64_t at = block_scan<kPlanThreads>(n, part, total);
    const int n_items = (int)total;
    for (int s = s0; s < s1; ++s) {
        item0[s] = (int)at;
        at += items_of(seq(s));
    }
    if (tid == 0) item0[p.n_seq] = n_items;
    __syncthreads();

    struct Item {
        Seq q;
        int s, r0, R, cost;
        ItemKeys k;
    };
    auto item = [&](int i) {
        Item x;
        // (requests without items share their first item with the next one:
        // the last of them is the one that has it)
        x.s = find_last(item0, p.n_seq, i);
        x.q = seq(x.s);
        x.R = x.q.T * p.hpk;
        const bool narrow = x.R <= kNarrowRows;
        // a prompt's last block, the longest, first
        x.r0 = narrow ? 0 : (item0[x.s + 1] - 1 - i) * W;
        const int rows = narrow ? x.R : imin(W, x.R - x.r0);
        const int pos0 = x.q.len - x.q.T;
        x.k = item_keys(pos0 + x.r0 / p.hpk, pos0 + (x.r0 + rows - 1) / p.hpk, x.q.len, p.window, x.q.prefix);
        x.cost = x.k.n_chunks * (narrow ? 1 : kWideCost);
        return x;
    };

    int64_t cost = 0;
    Item mine{};
    for (int i = tid; i < n_items; i += kPlanThreads) {
        mine = item(i);
        cost += mine.cost;
    }
    block_scan<kPlanThreads>(cost, part, total);
    int64_t L = kMinPiece;
    if (!p.split) {
        L = INT32_MAX;
    } else if (n_items > p.fill) {
        L = max<int64_t>(kMinPiece, 2 * ((total + p.fill - 1) / p.fill));
    } else if (n_items > 0) {
        // (fill <= kPlanThreads: one item a thread)
        // (at total / (fill - items) the pieces, at most total / L + items, fit)
        int64_t lo = max<int64_t>(kMinPiece, (total + p.fill - 1) / p.fill);
        int64_t hi = max(lo, p.fill > n_items ? (total + p.fill - n_items - 1) / (p.fill - n_items) : total);
        lo = min<int64_t>(lo, INT32_MAX);
        hi = min<int64_t>(hi, INT32_MAX);
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            int64_t pieces;
            block_scan<kPlanThreads>((int64_t)(tid < n_items ? item_pieces(mine.cost, mine.k.n_chunks, (int)mid) : 0), part, pieces);
            if (pieces <= p.fill) hi = mid;
            else lo = mid + 1;
        }
        L = lo;
    }
    L = min<int64_t>(L, INT32_MAX);

    int base_piece = 0, base_slot = 0, base_join = 0;
    for (int b = 0; b < n_items; b += kPlanThreads) {
        const int i = b + tid;
        Item x{};
        int k = 0;
        if (i < n_items) {
            x = item(i);
            k = item_pieces(x.cost, x.k.n_chunks, (int)L);
        }
        // pieces, split pieces and split items of the items before, packed
        int64_t all;
        const int64_t mine3 = k | (k > 1 ? (int64_t)k << 24 | (int64_t)1 << 48 : 0);
        const int64_t sum = block_scan<kPlanThreads>(mine3, part, all);
        const int pc = base_piece + (int)(sum & 0xFFFFFF), sl = base_slot + (int)((sum >> 24) & 0xFFFFFF),
                  jn = base_join + (int)(sum >> 48);
        piece0[tid] = pc;
        slot0[tid] = k > 1 ? sl : -1;
        if (tid == 0) piece0[kPlanThreads] = base_piece + (int)(all & 0xFFFFFF);
        if (k > 1 && jn < p.max_joins) p.joins[jn] = PlanJoin{x.q.q0, x.R, x.r0, sl, k, {}};
        __syncthreads();
        const int n_here = min(kPlanThreads, n_items - b), end = piece0[kPlanThreads];
        for (int j = base_piece + tid; j < end && j < p.max_pieces; j += kPlanThreads) {
            const int t = find_last(piece0, n_here, j);
            const Item y = item(b + t);
            const int of = item_pieces(y.cost, y.k.n_chunks, (int)L), at_ = j - piece0[t];
            PlanPiece z;
            z.seq = y.s;
            z.q0 = y.q.q0;
            z.R = y.R;
            z.r0 = y.r0;
            z.pos0 = y.q.len - y.q.T;
            z.len = y.q.len;
            z.cb = (int)((int64_t)y.k.n_chunks * at_ / of);
            z.ce = (int)((int64_t)y.k.n_chunks * (at_ + 1) / of);
            z.slot = slot0[t] < 0 ? -1 : slot0[t] + at_;
            z.n_pre = y.k.n_pre;
            z.lo_base = y.k.lo_base;
            z.lo = y.k.lo;
            z.kend = y.k.kend;
            z.pe = y.k.pe;
            z.pad[0] = z.pad[1] = 0;
            p.pieces[j] = z;
        }
        base_piece = end;
        base_slot += (int)((all >> 24) & 0xFFFFFF);
        base_join += (int)(all >> 48);
        __syncthreads();
    }
    if (tid == 0) {
        PlanHeader h{};
        h.sig = p.sig;
        h.n_pieces = min(base_piece, p.max_pieces);
        h.n_joins = min(base_join, p.max_joins);
        *p.head = h;
    }
}

}  // namespace

hipError_t launch_pages_append(const PagesParams& p, hipStream_t st) {
    // a workgroup for each 1024 rows (its scan is paid once for them)
    const int grid = p.n_tokens <= 1024 ? 1 : min((p.n_tokens + 1023) / 1024, 256);
    ProfScope ps(kProfPages, st);
    hipLaunchKernelGGL(pages_append_kernel, dim3(grid), dim3(kPagesThreads), 0, st, p);
    return hipGetLastError();
}

hipError_t launch_pages_release(const PagesParams& p, hipStream_t st) {
    ProfScope ps(kProfPages, st);
    hipLaunchKernelGGL(pages_release_kernel, dim3(p.n_seq <= 64 ? 1 : 8), dim3(kPagesThreads), 0, st, p);
    return hipGetLastError();
}

hipError_t launch_paged_plan(const PlanParams& p, hipStream_t st) {
    ProfScope ps(kProfPagedPlan, st);
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    return hipGetLastError();
}

}  // namespace pelica

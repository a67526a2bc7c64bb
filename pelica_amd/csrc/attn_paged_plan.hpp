// Plain arithmetic of the paged kernels, the same lines in the library, in its
// kernels and in a host test: which keys a block of query rows walks, which rows
// of a cache page a load may touch, how the work list is cut.
#pragma once
#include <math.h>

#include <cstddef>
#include <cstdint>

#ifdef __HIPCC__
#define PELICA_HD __host__ __device__ __forceinline__
#else
#define PELICA_HD inline
#endif

namespace pelica {

// Query rows of a request are (token, head of the kv head's group) pairs,
// row = token * hpk + head.  A request of at most kNarrowRows rows is one item
// whose four waves share the keys (narrow); others are cut into items of
// wide_rows rows whose waves share the rows (wide).
constexpr int kNarrowRows = 32;
PELICA_HD constexpr int wide_rows(int hd) { return hd == 64 ? 256 : 128; }

// Costs of the work list, in the time a narrow workgroup's wave takes for a
// chunk of 32 keys (~0.45 us): a wide workgroup's chunk (1.0 - 1.4 us at both
// head dims, two workgroups a CU), the least cost of a piece, a piece's start
// and end, and the partials that a split item's piece writes and the join
// reads.  (Pieces cut at the limit with the rest behind, instead of equal ones,
// fill the slots better by this model, and on the chip 3% better to 2% worse:
// two workgroups of a CU share what one of them leaves.)
constexpr int kWideCost = 3;
constexpr int kMinPiece = 4;
struct PlanCost {
    // a piece's own time, and what it takes of the whole chip's
    static PELICA_HD float piece(bool wide, int chunks) {
        return (float)(wide ? kWideCost * chunks + 10 : ((chunks + 3) & ~3) + 10);  // (four waves share a narrow one's)
    }
    static PELICA_HD float share(bool wide, int chunks, bool split) {
        return piece(wide, chunks) + (split ? wide ? 20.f : 1.f : 0.f);
    }
    // the step: the chip's mean, or a slot with `last` to do (its one piece, or
    // the pieces that have to share a slot), which runs faster once its
    // neighbours are done
    static PELICA_HD float step(float mean, float last) { return last > mean ? mean + 0.6f * (last - mean) : mean; }
};

// 32-key chunks of the keys that any row of an item sees: its window's and
// the causal ones [lo, kend), and the prefix's [0, pe).  Chunks count from
// key 0 over the prefix, then (where a gap of whole chunks lies between) from
// chunk n_pre at key lo_base.
struct ItemKeys {
    int n_pre, lo_base, n_chunks;
    int lo, kend, pe;
};

PELICA_HD int imin(int a, int b) { return a < b ? a : b; }
PELICA_HD int imax(int a, int b) { return a > b ? a : b; }

// positions [pos_first, pos_last] of a request of len keys
PELICA_HD ItemKeys item_keys(int pos_first, int pos_last, int len, int window, int prefix) {
    ItemKeys k;
    k.pe = imax(0, imin(prefix, len));
    k.kend = pos_last + 1;
    k.lo = window > 0 && pos_first >= window ? pos_first - window + 1 : 0;
    const int lo32 = k.lo & ~31;
    const int pre = (int)(((unsigned)k.pe + 31u) >> 5);
    if (k.pe > 0 && pre < (lo32 >> 5)) {
        k.n_pre = pre;
        k.lo_base = lo32;
        k.n_chunks = pre + (int)(((unsigned)(k.kend - lo32) + 31u) >> 5);
    } else {
        k.n_pre = 0;
        k.lo_base = k.pe > 0 ? 0 : lo32;
        k.n_chunks = (int)(((unsigned)(imax(k.kend, k.pe) - k.lo_base) + 31u) >> 5);
    }
    return k;
}

// first key of chunk c
PELICA_HD int chunk_key(int c, int n_pre, int lo_base) { return c < n_pre ? 32 * c : lo_base + 32 * (c - n_pre); }

// x between 0 and n, on the scalar unit: as a minimum of a maximum the compiler
// makes it a vector instruction, and every address that follows with it
PELICA_HD int clamp_to(int x, int n) {
#ifdef __HIP_DEVICE_COMPILE__
    int y;
    __asm__("s_max_i32 %0, %1, 0" : "=s"(y) : "s"(x) : "scc");
    return imin(y, n);
#else
    return imin(imax(x, 0), n);
#endif
}
// Of n consecutive keys from kg (all in one page), the rows [first, first +
// count) that a load touches: those that some row of the item sees, and, where
// the prefix ends and the window begins within them, what lies between
// (gap_in_run).  No others: they may lie in a page that was given away.
PELICA_HD void group_rows(int kg, int n, int lo, int kend, int pe, int& first, int& count) {
    const int a = clamp_to(pe - kg, n);  // of the prefix: [0, a)
    const int b0 = clamp_to(lo - kg, n), b1 = clamp_to(kend - kg, n);
    first = a > 0 ? 0 : b0;
    const int end = b1 > b0 ? imax(a, b1) : a;
    count = imax(end - first, 0);
}
// Whether a run of 8 rows holds keys [pe, lo) between a prefix and a window,
// which no row of the item sees, beside keys of both
PELICA_HD bool gap_in_run(int lo, int pe) { return pe > 0 && pe < lo && (pe - 1) >> 3 == lo >> 3; }

// Pieces of an item of `cost` where a piece's may be 1 / inv_limit
PELICA_HD int item_pieces(int cost, int n_chunks, float inv_limit) {
    const float k = ceilf((float)cost * inv_limit);
    return k >= (float)n_chunks ? n_chunks : imax(1, (int)k);
}

// most items of a step: one for each request with tokens, and one for each
// whole block of wide_rows rows
inline int64_t plan_items(int64_t n_seq, int64_t n_tokens, int hpk, int hd) {
    return (n_seq < n_tokens ? n_seq : n_tokens) + n_tokens * hpk / wide_rows(hd);
}
// pieces (per kv head) that fill the chip once: two workgroups a CU
inline int plan_fill(int n_kv, int cus) {
    const int n = (2 * cus + n_kv - 1) / n_kv;
    return n > 1 ? n : 1;
}
// most pieces that split items have together (each a slot of partials), and
// most pieces of a step
inline int plan_slots(int fill) { return 2 * fill; }
inline int64_t plan_pieces(int64_t items, int fill) { return items + plan_slots(fill); }

// the plan buffer: header, joins, pieces
struct PlanHeader {
    uint32_t sig;
    int n_pieces, n_joins, pad[13];
};
struct PlanPiece {
    int seq, q0, R, r0;        // request, its first row of q, its query rows, the item's first
    int pos0, len, cb, ce;     // position of its first token, its keys; chunks [cb, ce)
    int slot, n_pre, lo_base;  // partial slot, or -1: the item's only piece
    int lo, kend, pe, pad[2];
};
struct PlanJoin {
    int q0, R, r0, slot0, n_slots, pad[3];
};
static_assert(sizeof(PlanHeader) == 64 && sizeof(PlanPiece) == 64 && sizeof(PlanJoin) == 32, "plan layout");

}  // namespace pelica

// The C entry points over a paged cache (include/pelica_attn.h): checks of
// descriptors and arguments, sizes, launches.
#include <algorithm>
#include <cmath>

#include "../../include/pelica_attn.h"
#include "attn_error.hpp"
#include "attn_paged.hpp"

namespace {

using pelica::fail;

bool misaligned(const void* p, int a = 16) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

int log2_of(int32_t page) {
    if (page < 8 || page > 65536 || (page & (page - 1))) return -1;
    return __builtin_ctz((unsigned)page);
}

// compute units of the current device (queried once per process)
int device_cus() {
    static const int n = [] {
        int dev = 0, cus = 0;
        if (hipGetDevice(&dev) != hipSuccess ||
            hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
            cus = 256;  // MI355X
        return cus;
    }();
    return n;
}

constexpr int kMaxTokens = 1 << 20;

int check_pages(const PelicaPageDesc* d) {
    if (!d) return fail(PELICA_ATTN_EINVAL, "desc is NULL");
    if (d->n_seq <= 0 || d->n_seq > PELICA_ATTN_PAGED_MAX_SEQ)
        return fail(PELICA_ATTN_EINVAL, "n_seq %d (1 .. %d)", d->n_seq, PELICA_ATTN_PAGED_MAX_SEQ);
    if (log2_of(d->page_size) < 0) return fail(PELICA_ATTN_EUNSUPPORTED, "page_size %d (a power of two, 8 .. 65536)", d->page_size);
    if (d->n_pages <= 0 || d->max_pages <= 0)
        return fail(PELICA_ATTN_EINVAL, "n_pages %d and max_pages %d must be positive", d->n_pages, d->max_pages);
    return PELICA_ATTN_OK;
}

// The arrays of a call over pages.  Every workgroup reads all of the inputs
// while others write, so an output shares no byte with another array.
struct Array {
    const char* name;
    const void* at;
    int64_t n;
    int size;
    bool out;
};
template <int N>
int check_arrays(const char* call, const Array (&a)[N]) {
    for (const Array& x : a)
        if (!x.at) return fail(PELICA_ATTN_EINVAL, "every array of %s must be non-NULL", call);
    for (const Array& x : a)
        if (misaligned(x.at, x.size)) return fail(PELICA_ATTN_EINVAL, "arrays of %s must be aligned to their values", call);
    for (const Array& x : a)
        for (const Array& y : a) {
            const uintptr_t p = reinterpret_cast<uintptr_t>(x.at), q = reinterpret_cast<uintptr_t>(y.at);
            if (x.out && &x != &y && p < q + (uint64_t)y.n * y.size && q < p + (uint64_t)x.n * x.size)
                return fail(PELICA_ATTN_EINVAL, "%s: %s overlaps %s", call, x.name, y.name);
        }
    return PELICA_ATTN_OK;
}

int64_t row_stride(const PelicaPagedDesc* d) { return d->row_stride ? d->row_stride : (int64_t)d->n_kv * d->hd; }
int64_t head_stride(const PelicaPagedDesc* d) { return d->head_stride ? d->head_stride : d->hd; }
int64_t page_stride(const PelicaPagedDesc* d) { return d->page_stride ? d->page_stride : (int64_t)d->page_size * row_stride(d); }

// The pool's shape; attention reads 16-byte pieces (8 values), the qkv step writes 8-byte ones (4);
// 8-bit rows are read in pieces of up to 16 values
int check_pool(const PelicaPagedDesc* d, int piece) {
    if (!d) return fail(PELICA_ATTN_EINVAL, "desc is NULL");
    if (d->n_head <= 0 || d->n_kv <= 0 || d->n_head % d->n_kv || d->n_head > 65536)
        return fail(PELICA_ATTN_EINVAL, "n_head %d must be a positive multiple of n_kv %d, <= 65536", d->n_head, d->n_kv);
    if (d->n_tokens <= 0 || d->n_tokens > kMaxTokens)
        return fail(PELICA_ATTN_EINVAL, "n_tokens %d (1 .. %d)", d->n_tokens, kMaxTokens);
    if (log2_of(d->page_size) < 0) return fail(PELICA_ATTN_EUNSUPPORTED, "page_size %d (a power of two, 8 .. 65536)", d->page_size);
    if (d->n_pages <= 0) return fail(PELICA_ATTN_EINVAL, "n_pages %d must be positive", d->n_pages);
    const int64_t rs = row_stride(d), hs = head_stride(d), ps = page_stride(d);
    if (rs < d->hd || hs < d->hd || ps < d->hd || rs % piece || hs % piece || ps % piece)
        return fail(PELICA_ATTN_EINVAL, "page, row and head strides (%lld, %lld, %lld): at least hd, multiples of %d",
                    (long long)ps, (long long)rs, (long long)hs, piece);
    // (a page's rows are addressed with 32-bit byte offsets, a page with 64)
    if (rs >= 1 << 24 || rs * d->page_size >= 1LL << 31 || hs >= 1LL << 40 || ps >= 1LL << 40)
        return fail(PELICA_ATTN_EUNSUPPORTED, "page, row and head strides (%lld, %lld, %lld) too large", (long long)ps,
                    (long long)rs, (long long)hs);
    return PELICA_ATTN_OK;
}

// `n` pieces of `bytes` each, the first at `at`, `step` bytes between their beginnings
struct Pieces {
    const char* name;
    const void* at;
    int64_t n, step, bytes;
};
// Whether rows of an output may share a byte with another array: not where the one's
// ends lie ahead of the other or behind it, where both have one step and their pieces
// take turns (K's and V's rows in one buffer), or where all rows lie between two pieces.
bool may_overlap(const Pieces& rows, const Pieces& y) {
    typedef __int128 wide;
    const wide p = reinterpret_cast<uintptr_t>(rows.at), q = reinterpret_cast<uintptr_t>(y.at);
    const wide p_end = p + (wide)(rows.n - 1) * rows.step + rows.bytes, q_end = q + (wide)(y.n - 1) * y.step + y.bytes;
    if (p >= q_end || q >= p_end) return false;
    if (rows.step == y.step) {
        const wide d = ((p - q) % y.step + y.step) % y.step;  // from a piece to the row after it
        return d < y.bytes || y.step - d < rows.bytes;
    }
    const wide d = (p - q) % y.step;
    return p < q || d < y.bytes || d + (p_end - p) > y.step;
}

int64_t scale_row(const PelicaPagedDesc* d, const PelicaPagedQ8* x) {
    return x->row_stride ? x->row_stride : (int64_t)d->n_kv * (d->hd / pelica::kQ8Group);
}
pelica::Q8Strides scale_strides(const PelicaPagedDesc* d, const PelicaPagedQ8* x) {
    const int64_t row = scale_row(d, x);
    return {x->page_stride ? x->page_stride : d->page_size * row, row, x->head_stride ? x->head_stride : d->hd / pelica::kQ8Group};
}

// Scales beside 8-bit pages (whose strides are whole 16-byte pieces)
int check_q8(const PelicaPagedDesc* d, const PelicaPagedQ8* x) {
    const int rc = check_pool(d, 16);
    if (rc) return rc;
    if (!x) return fail(PELICA_ATTN_EINVAL, "q8 is NULL");
    if (!x->k_scales || !x->v_scales || misaligned(x->k_scales, 2) || misaligned(x->v_scales, 2))
        return fail(PELICA_ATTN_EINVAL, "k_scales and v_scales must be non-NULL and aligned to their values");
    const pelica::Q8Strides st = scale_strides(d, x);
    const int64_t g = d->hd / pelica::kQ8Group;
    if (st.row < g || st.head < g || st.page < g)
        return fail(PELICA_ATTN_EINVAL, "page, row and head strides of scales (%lld, %lld, %lld): at least hd / 32",
                    (long long)st.page, (long long)st.row, (long long)st.head);
    if (st.row >= 1 << 24 || st.row * d->page_size >= 1LL << 30 || st.head >= 1LL << 40 || st.page >= 1LL << 40)
        return fail(PELICA_ATTN_EUNSUPPORTED, "page, row and head strides of scales (%lld, %lld, %lld) too large",
                    (long long)st.page, (long long)st.row, (long long)st.head);
    return PELICA_ATTN_OK;
}

int check_paged(const PelicaPagedDesc* d) {
    int rc = check_pool(d, 8);
    if (rc) return rc;
    if (d->hd != 64 && d->hd != 128) return fail(PELICA_ATTN_EUNSUPPORTED, "hd %d unsupported (64 or 128)", d->hd);
    if (d->n_seq <= 0 || d->n_seq > PELICA_ATTN_PAGED_MAX_SEQ)
        return fail(PELICA_ATTN_EINVAL, "n_seq %d (1 .. %d)", d->n_seq, PELICA_ATTN_PAGED_MAX_SEQ);
    if (d->max_q <= 0 || d->max_q > d->n_tokens) return fail(PELICA_ATTN_EINVAL, "max_q %d (1 .. n_tokens %d)", d->max_q, d->n_tokens);
    if (d->max_pages <= 0 || (int64_t)d->max_pages * d->page_size > (1 << 30))
        return fail(PELICA_ATTN_EINVAL, "max_pages %d: at least 1, and at most 2^30 keys", d->max_pages);
    if (d->window < 0) return fail(PELICA_ATTN_EINVAL, "window %d must be >= 0", d->window);
    if (!(d->scale >= 0.f) || std::isinf(d->scale)) return fail(PELICA_ATTN_EINVAL, "scale must be finite, >= 0");
    if (!(d->softcap >= 0.f) || std::isinf(d->softcap)) return fail(PELICA_ATTN_EINVAL, "softcap must be finite, >= 0");
    if (d->softcap > 0.f && (d->softcap < 1e-30f || d->softcap > 1e30f))
        return fail(PELICA_ATTN_EUNSUPPORTED, "softcap %g (0, or 1e-30 .. 1e30)", (double)d->softcap);
    if ((int64_t)d->n_tokens * d->n_head > (1 << 30))
        return fail(PELICA_ATTN_EUNSUPPORTED, "n_tokens x n_head above 2^30");
    if (!d->q_start || !d->seq_kv_len || !d->page_table)
        return fail(PELICA_ATTN_EINVAL, "q_start, seq_kv_len and page_table must be non-NULL");
    if (misaligned(d->q_start, 4) || misaligned(d->seq_kv_len, 4) || misaligned(d->page_table, 4) ||
        misaligned(d->prefix_len, 4) || misaligned(d->alibi, 4))
        return fail(PELICA_ATTN_EINVAL, "arrays of the descriptor must be aligned to their values");
    return PELICA_ATTN_OK;
}

// Keys that requests share: what such a plan takes of the descriptor, and its groups
int check_shared(const PelicaPagedDesc* d, const PelicaPagedShared* x) {
    const int rc = check_paged(d);
    if (rc) return rc;
    if (!x) return fail(PELICA_ATTN_EINVAL, "shared is NULL");
    if (x->n_groups <= 0 || x->n_groups > PELICA_ATTN_PAGED_MAX_GROUPS || x->n_groups > d->n_seq)
        return fail(PELICA_ATTN_EINVAL, "n_groups %d (1 .. %d, and at most n_seq %d)", x->n_groups, PELICA_ATTN_PAGED_MAX_GROUPS, d->n_seq);
    if (!x->group_start || !x->shared_len || misaligned(x->group_start, 4) || misaligned(x->shared_len, 4))
        return fail(PELICA_ATTN_EINVAL, "group_start and shared_len must be non-NULL and aligned to their values");
    if (d->window) return fail(PELICA_ATTN_EUNSUPPORTED, "shared keys and a window (such layers take a plain plan)");
    if (d->prefix_len) return fail(PELICA_ATTN_EUNSUPPORTED, "shared keys and prefix_len");
    if (d->alibi) return fail(PELICA_ATTN_EUNSUPPORTED, "shared keys and alibi: rows of one position each have their own bias");
    if ((int64_t)d->n_tokens * d->n_head > 1 << 28) return fail(PELICA_ATTN_EUNSUPPORTED, "shared keys and n_tokens x n_head above 2^28");
    return PELICA_ATTN_OK;
}

struct PagedPlan {
    int hpk, fill, rows, max_joins, max_rows;
    int64_t max_pieces;
    bool wide, split;
    size_t join_at, piece_at, bytes, ml_bytes, ws_bytes;
    uint32_t sig;
};

PagedPlan plan_of(const PelicaPagedDesc* d, const PelicaPagedShared* shared = nullptr) {
    PagedPlan x;
    x.hpk = d->n_head / d->n_kv;
    // (the rows of a group are one item's)
    x.wide = (int64_t)(shared ? d->n_tokens : d->max_q) * x.hpk > pelica::kNarrowRows;
    x.fill = pelica::plan_fill(d->n_kv, device_cus());
    int64_t items = x.wide ? pelica::plan_items(d->n_seq, d->n_tokens, x.hpk, d->hd)
                           : std::min(d->n_seq, d->n_tokens);
    x.max_joins = shared ? (int)items : 0;  // (of requests; groups have none)
    if (shared) items += x.wide ? pelica::plan_items(shared->n_groups, d->n_tokens, x.hpk, d->hd) : shared->n_groups;
    x.rows = x.wide ? pelica::wide_rows(d->hd)
                    : std::min(pelica::kNarrowRows, (shared ? d->n_tokens : d->max_q) * x.hpk);
    x.max_rows = std::min((int64_t)d->max_q * x.hpk, (int64_t)x.rows);
    // a step whose items are at most two chunks a wave (window layers) is not
    // split, and has no second kernel
    const int64_t keys = (int64_t)d->max_pages * d->page_size;
    const int64_t span = d->window > 0 && !d->prefix_len ? std::min(keys, (int64_t)d->window + d->max_q - 1) : keys;
    x.split = shared || x.wide || span / 32 + 2 > 8;
    x.max_pieces = x.split ? pelica::plan_pieces(items, x.fill) : items;
    if (!shared) x.max_joins = x.split ? (int)std::min<int64_t>(items, pelica::plan_slots(x.fill) / 2) : 0;
    auto al = [](size_t b) { return (b + 255) & ~(size_t)255; };
    x.join_at = 64;
    x.piece_at = 64 + (((size_t)x.max_joins * (shared ? sizeof(pelica::SharedJoin) : sizeof(pelica::PlanJoin)) + 63) & ~(size_t)63);
    x.bytes = x.piece_at + (size_t)x.max_pieces * sizeof(pelica::PlanPiece);
    // (rows of partials; with shared keys each row has one of its request's and one of its group's at least)
    const size_t slots = x.split ? ((size_t)pelica::plan_slots(x.fill) * x.rows + (shared ? 2 * (size_t)d->n_tokens * x.hpk : 0)) * d->n_kv : 0;
    x.ml_bytes = al(slots * 8);
    x.ws_bytes = x.split ? x.ml_bytes + al(slots * d->hd * 4) : 0;
    // what a plan depends on (FNV-1a)
    const int32_t parts[] = {d->n_head, d->n_kv, d->hd, d->n_seq, d->n_tokens, d->max_q, d->page_size, d->n_pages,
                             d->max_pages, d->window, d->prefix_len ? 1 : 0, x.fill};
    x.sig = 2166136261u ^ (shared ? (uint32_t)shared->n_groups : 0u);
    for (int32_t v : parts)
        for (int b = 0; b < 4; ++b) x.sig = (x.sig ^ ((uint32_t)v >> (8 * b) & 255)) * 16777619u;
    return x;
}

// The work list's parameters; 0 where the buffer will do
int plan_params(const PelicaPagedDesc* d, const PagedPlan& x, void* plan, size_t plan_bytes, pelica::PlanParams& p) {
    if (!plan || misaligned(plan)) return fail(PELICA_ATTN_EINVAL, "plan must be non-NULL and 16-byte aligned");
    if (plan_bytes < x.bytes) return fail(PELICA_ATTN_EWORKSPACE, "plan of %zu bytes needed, %zu given", x.bytes, plan_bytes);
    char* pl = static_cast<char*>(plan);
    p.q_start = d->q_start;
    p.kv_len = d->seq_kv_len;
    p.prefix = d->prefix_len;
    p.head = reinterpret_cast<pelica::PlanHeader*>(pl);
    p.joins = reinterpret_cast<pelica::PlanJoin*>(pl + x.join_at);
    p.pieces = reinterpret_cast<pelica::PlanPiece*>(pl + x.piece_at);
    p.n_seq = d->n_seq;
    p.n_tokens = d->n_tokens;
    p.max_q = d->max_q;
    p.hpk = x.hpk;
    p.hd = d->hd;
    p.window = d->window;
    p.fill = x.fill;
    p.max_keys = (int64_t)d->max_pages * d->page_size;
    p.max_joins = x.max_joins;
    p.max_pieces = (int)x.max_pieces;
    p.sig = x.sig;
    p.split = x.split;
    p.max_slots = pelica::plan_slots(x.fill);
    p.rows = x.rows;
    return PELICA_ATTN_OK;
}

// (q8: NULL for f16 pages)
int run_paged(const PelicaPagedDesc* d, const PelicaPagedShared* shared, const PelicaPagedQ8* q8, const void* plan, size_t plan_bytes, const void* q, const void* k,
              const void* v, const float* sinks, void* out, void* workspace, size_t workspace_bytes, bool f32, void* stream) {
    if (!plan || !q || !k || !v || !out) return fail(PELICA_ATTN_EINVAL, "plan, q, k_pages, v_pages and out must be non-NULL");
    if (misaligned(plan) || misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || misaligned(workspace))
        return fail(PELICA_ATTN_EINVAL, "plan, q, k_pages, v_pages, out and workspace must be 16-byte aligned");
    const int es = f32 ? 4 : 2;
    const int64_t row = (int64_t)d->n_head * d->hd;
    for (const int64_t st : {d->q_token_stride, d->out_token_stride})
        if (st != 0 && (st < row || (st * es) % 16 || st >= 1LL << 31))
            return fail(PELICA_ATTN_EINVAL, "token stride %lld: 0, or >= n_head*hd (%lld), < 2^31 and a whole number of "
                        "16-byte pieces", (long long)st, (long long)row);
    if (misaligned(sinks, 4)) return fail(PELICA_ATTN_EINVAL, "sinks must be aligned to its values");
    const PagedPlan x = plan_of(d, shared);
    // (kernels read pieces beside the header that says whether they are theirs)
    if (plan_bytes < x.bytes) return fail(PELICA_ATTN_EWORKSPACE, "plan of %zu bytes needed, %zu given", x.bytes, plan_bytes);
    if (x.ws_bytes && (!workspace || workspace_bytes < x.ws_bytes))
        return fail(PELICA_ATTN_EWORKSPACE, "workspace of %zu bytes needed, %zu given", x.ws_bytes,
                    workspace ? workspace_bytes : (size_t)0);
    if (x.max_pieces * d->n_kv >= 1 << 24) return fail(PELICA_ATTN_EUNSUPPORTED, "more than 2^24 workgroups");
    pelica::PagedParams p{};
    p.q = q;
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    const char* pl = static_cast<const char*>(plan);
    p.head = reinterpret_cast<const pelica::PlanHeader*>(pl);
    p.joins = reinterpret_cast<const pelica::PlanJoin*>(pl + x.join_at);
    p.shared_joins = shared ? reinterpret_cast<const pelica::SharedJoin*>(pl + x.join_at) : nullptr;
    p.pieces = reinterpret_cast<const pelica::PlanPiece*>(pl + x.piece_at);
    p.table = d->page_table;
    p.sinks = sinks;
    p.alibi = d->alibi;
    p.sinks_or_q = sinks ? sinks : static_cast<const float*>(q);
    p.alibi_or_q = d->alibi ? d->alibi : static_cast<const float*>(q);
    p.inv_hpk = 1.0 / x.hpk;
    p.out = out;
    p.ws_ml = x.ws_bytes ? static_cast<float*>(workspace) : nullptr;
    p.ws_o = x.ws_bytes ? reinterpret_cast<float*>(static_cast<char*>(workspace) + x.ml_bytes) : nullptr;
    const int size = q8 ? 1 : 2;
    p.page_b = page_stride(d) * size;
    p.head_b = head_stride(d) * size;
    p.row_b = (uint32_t)(row_stride(d) * size);
    if (q8) {
        const pelica::Q8Strides s = scale_strides(d, q8);
        p.ks = q8->k_scales;
        p.vs = q8->v_scales;
        p.spage_b = s.page * 2;
        p.shead_b = s.head * 2;
        p.srow_b = (uint32_t)(s.row * 2);
    }
    p.q_tok = d->q_token_stride ? d->q_token_stride : row;
    p.o_tok = d->out_token_stride ? d->out_token_stride : row;
    p.sig = x.sig;
    p.n_kv = d->n_kv;
    p.hpk = x.hpk;
    p.n_pages = d->n_pages;
    p.max_pages = d->max_pages;
    p.page_log2 = log2_of(d->page_size);
    p.window = d->window;
    p.rows = x.rows;
    p.qscale = (d->scale > 0.f ? d->scale : 1.f / std::sqrt((float)d->hd)) * pelica::kLog2e;
    p.cap = d->softcap;
    pelica::capped_poly(p);
    p.hd = d->hd;
    p.max_pieces = (int)x.max_pieces;
    p.max_joins = x.max_joins;
    p.max_rows = x.max_rows;
    p.all_rows = d->n_tokens * d->n_head;
    p.f32 = f32;
    p.wide = x.wide;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e = q8 ? pelica::launch_paged_q8(p, st) : pelica::launch_paged(p, st);
    if (e == hipSuccess && x.split) e = pelica::launch_paged_join(p, st);
    if (e != hipSuccess) return fail(PELICA_ATTN_EHIP, "paged attention launch: %s", hipGetErrorString(e));
    return PELICA_ATTN_OK;
}

// (q8: NULL for f16 pages)
int run_qkv(const PelicaPagedDesc* d, const PelicaPagedRope* rope, const PelicaPagedQ8* q8, const float* q, const float* k,
            const float* v, int64_t token_stride, const float* q_norm, const float* k_norm, float eps,
            const int64_t* slots, void* q_out, int32_t q_half, int64_t q_out_stride, void* k_pages, void* v_pages,
            void* stream) {
    if (d->hd != 64 && d->hd != 128 && d->hd != 256) return fail(PELICA_ATTN_EUNSUPPORTED, "hd %d (64, 128 or 256)", d->hd);
    if (!q || !k || !v || !slots || !q_out || !k_pages || !v_pages)
        return fail(PELICA_ATTN_EINVAL, "q, k, v, slots, q_out and the pages must be non-NULL");
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(q_out, q_half ? 8 : 16) || misaligned(q_norm) ||
        misaligned(k_norm) || misaligned(k_pages, q8 ? 16 : 8) || misaligned(v_pages, q8 ? 16 : 8) || misaligned(slots, 8))
        return fail(PELICA_ATTN_EINVAL, "q, k, v, f32 q_out, norms and 8-bit pages must be 16-byte aligned, f16 q_out, slots and f16 pages 8");
    const int64_t wq = (int64_t)d->n_head * d->hd, wkv = (int64_t)d->n_kv * d->hd;
    if (token_stride && (token_stride < wq || token_stride < wkv || token_stride % 4))
        return fail(PELICA_ATTN_EINVAL, "token_stride %lld: 0, or at least a token's heads and a multiple of 4", (long long)token_stride);
    if (q_out_stride && (q_out_stride < wq || q_out_stride % 4))
        return fail(PELICA_ATTN_EINVAL, "q_out_stride %lld: 0, or >= n_head*hd and a multiple of 4", (long long)q_out_stride);
    if (q_out == (const void*)q && (q_half || (q_out_stride ? q_out_stride : wq) != (token_stride ? token_stride : wq)))
        return fail(PELICA_ATTN_EINVAL, "q_out may be q in f32 only, and at its stride");
    if (!(eps >= 0.f)) return fail(PELICA_ATTN_EINVAL, "eps must be >= 0");
    pelica::PagedQkvParams p{};
    if (rope && rope->rot) {
        if (rope->rot < 0 || rope->rot % 2 || rope->rot > d->hd) return fail(PELICA_ATTN_EINVAL, "rot %d", rope->rot);
        if (!rope->table || misaligned(rope->table, 8) || rope->table_split < 0 || rope->table_rows <= 0)
            return fail(PELICA_ATTN_EINVAL, "rope table missing, or not 8-byte aligned");
        if (rope->table_split && rope->table_rows < (int64_t)rope->table_split + 256)
            return fail(PELICA_ATTN_EINVAL, "a two-level rope table needs %lld rows", (long long)rope->table_split + 256);
        if (rope->n_axes < 1 || rope->n_axes > 4) return fail(PELICA_ATTN_EINVAL, "n_axes %d (1 .. 4)", rope->n_axes);
        if (!rope->positions || misaligned(rope->positions, 4)) return fail(PELICA_ATTN_EINVAL, "positions missing");
        if (rope->axis_stride != 0 && rope->axis_stride < d->n_tokens)
            return fail(PELICA_ATTN_EINVAL, "axis_stride %lld: 0, or >= n_tokens", (long long)rope->axis_stride);
        if (rope->pair_axis)
            for (int j = 0; j < rope->rot / 2; ++j) {
                if (rope->pair_axis[j] >= rope->n_axes)
                    return fail(PELICA_ATTN_EINVAL, "pair %d turns by axis %d of %d", j, rope->pair_axis[j], rope->n_axes);
                p.axis[j / 16] |= (uint32_t)rope->pair_axis[j] << (2 * (j % 16));
            }
        p.table = rope->table;
        p.positions = rope->positions;
        p.axis_stride = rope->axis_stride;
        p.rot = rope->rot;
        p.neox = rope->neox ? 1 : 0;
        p.table_split = rope->table_split;
        p.covered = (int)std::min<int64_t>(rope->table_split ? 256LL * rope->table_split : rope->table_rows, INT32_MAX);
        p.n_axes = rope->n_axes;
    }
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.slots = slots;
    p.q_out = q_out;
    p.k_pages = static_cast<uint16_t*>(k_pages);
    p.v_pages = static_cast<uint16_t*>(v_pages);
    if (q8) {
        p.q8 = true;
        p.k_scales = q8->k_scales;
        p.v_scales = q8->v_scales;
        p.sc = scale_strides(d, q8);
    }
    p.tok_q = token_stride ? token_stride : wq;
    p.tok_kv = token_stride ? token_stride : wkv;
    p.tok_o = q_out_stride ? q_out_stride : wq;
    p.page_stride = page_stride(d);
    p.row_stride = row_stride(d);
    p.head_stride = head_stride(d);
    p.page_log2 = log2_of(d->page_size);
    p.n_slots = (int64_t)d->n_pages << p.page_log2;
    p.n_head = d->n_head;
    p.n_kv = d->n_kv;
    p.n_tokens = d->n_tokens;
    p.eps = eps;
    p.hd = d->hd;
    p.half = q_half != 0;
    if ((int64_t)d->n_tokens * ((d->n_head + 2 * d->n_kv) * (d->hd / 4) / 256 + 1) >= 1 << 24)
        return fail(PELICA_ATTN_EUNSUPPORTED, "more than 2^24 workgroups");
    const hipError_t e = pelica::launch_paged_qkv(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(PELICA_ATTN_EHIP, "paged_qkv launch: %s", hipGetErrorString(e));
    return PELICA_ATTN_OK;
}

}  // namespace

extern "C" {

int pelica_attn_pages_append(const PelicaPageDesc* d, const int32_t* cached_len, const int32_t* new_len,
                             int32_t* page_table, const int32_t* free_list, const int64_t* free_in, int64_t* free_out,
                             int32_t* q_start, int32_t* seq_kv_len, int64_t* slots, int32_t* positions,
                             int32_t* token_seq, int32_t* status, void* stream) {
    pelica::clear_error();
    int rc = check_pages(d);
    if (rc) return rc;
    if (d->n_tokens <= 0 || d->n_tokens > kMaxTokens) return fail(PELICA_ATTN_EINVAL, "n_tokens %d (1 .. %d)", d->n_tokens, kMaxTokens);
    const int64_t cells = (int64_t)d->n_seq * d->max_pages;
    const Array arrays[] = {
        {"cached_len", cached_len, d->n_seq, 4, false}, {"new_len", new_len, d->n_seq, 4, false},
        {"page_table", page_table, cells, 4, true},     {"free_list", free_list, d->n_pages, 4, false},
        {"free_in", free_in, 2, 8, false},              {"free_out", free_out, 2, 8, true},
        {"q_start", q_start, d->n_seq + 1, 4, true},    {"seq_kv_len", seq_kv_len, d->n_seq, 4, true},
        {"slots", slots, d->n_tokens, 8, true},         {"positions", positions, d->n_tokens, 4, true},
        {"token_seq", token_seq, d->n_tokens, 4, true}, {"status", status, d->n_seq, 4, true}};
    rc = check_arrays("pages_append", arrays);
    if (rc) return rc;
    pelica::PagesParams p{};
    p.cached = cached_len;
    p.fresh = new_len;
    p.free_in = free_in;
    p.free_out = free_out;
    p.table = page_table;
    p.list = const_cast<int32_t*>(free_list);
    p.q_start = q_start;
    p.kv_len = seq_kv_len;
    p.positions = positions;
    p.token_seq = token_seq;
    p.status = status;
    p.slots = slots;
    p.n_seq = d->n_seq;
    p.n_tokens = d->n_tokens;
    p.page_log2 = log2_of(d->page_size);
    p.n_pages = d->n_pages;
    p.max_pages = d->max_pages;
    const hipError_t e = pelica::launch_pages_append(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(PELICA_ATTN_EHIP, "pages_append launch: %s", hipGetErrorString(e));
    return PELICA_ATTN_OK;
}

int pelica_attn_pages_release(const PelicaPageDesc* d, const int32_t* ended, const int32_t* cached_len,
                              const int32_t* page_table, int32_t* free_list, const int64_t* free_in, int64_t* free_out,
                              void* stream) {
    pelica::clear_error();
    int rc = check_pages(d);
    if (rc) return rc;
    const int64_t cells = (int64_t)d->n_seq * d->max_pages;
    const Array arrays[] = {{"ended", ended, d->n_seq, 4, false},   {"cached_len", cached_len, d->n_seq, 4, false},
                            {"page_table", page_table, cells, 4, false}, {"free_list", free_list, d->n_pages, 4, true},
                            {"free_in", free_in, 2, 8, false},      {"free_out", free_out, 2, 8, true}};
    rc = check_arrays("pages_release", arrays);
    if (rc) return rc;
    pelica::PagesParams p{};
    p.ended = ended;
    p.cached = cached_len;
    p.free_in = free_in;
    p.free_out = free_out;
    p.table = const_cast<int32_t*>(page_table);
    p.list = free_list;
    p.n_seq = d->n_seq;
    p.page_log2 = log2_of(d->page_size);
    p.n_pages = d->n_pages;
    p.max_pages = d->max_pages;
    const hipError_t e = pelica::launch_pages_release(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(PELICA_ATTN_EHIP, "pages_release launch: %s", hipGetErrorString(e));
    return PELICA_ATTN_OK;
}

size_t pelica_attn_paged_plan_bytes(const PelicaPagedDesc* d) {
    pelica::clear_error();
    if (check_paged(d)) return 0;
    return plan_of(d).bytes;
}

int pelica_attn_paged_plan(const PelicaPagedDesc* d, void* plan, size_t plan_bytes, void* stream) {
    pelica::clear_error();
    int rc = check_paged(d);
    if (rc) return rc;
    pelica::PlanParams p{};
    rc = plan_params(d, plan_of(d), plan, plan_bytes, p);
    if (rc) return rc;
    const hipError_t e = pelica::launch_paged_plan(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(PELICA_ATTN_EHIP, "paged_plan launch: %s", hipGetErrorString(e));
    return PELICA_ATTN_OK;
}

size_t pelica_attn_paged_workspace_bytes(const PelicaPagedDesc* d) {
    pelica::clear_error();
    if (check_paged(d)) return 0;
    return plan_of(d).ws_bytes;
}

int pelica_attn_paged(const PelicaPagedDesc* d, const void* plan, size_t plan_bytes, const uint16_t* q,
                      const uint16_t* k_pages, const uint16_t* v_pages, const float* sinks, uint16_t* out,
                      void* workspace, size_t workspace_bytes, void* stream) {
    pelica::clear_error();
    const int rc = check_paged(d);
    if (rc) return rc;
    return run_paged(d, nullptr, nullptr, plan, plan_bytes, q, k_pages, v_pages, sinks, out, workspace, workspace_bytes, false, stream);
}

int pelica_attn_paged_f32(const PelicaPagedDesc* d, const void* plan, size_t plan_bytes, const float* q,
                          const uint16_t* k_pages, const uint16_t* v_pages, const float* sinks, float* out,
                          void* workspace, size_t workspace_bytes, void* stream) {
    pelica::clear_error();
    const int rc = check_paged(d);
    if (rc) return rc;
    return run_paged(d, nullptr, nullptr, plan, plan_bytes, q, k_pages, v_pages, sinks, out, workspace, workspace_bytes, true, stream);
}

int pelica_attn_paged_qkv(const PelicaPagedDesc* d, const PelicaPagedRope* rope, const float* q, const float* k,
                          const float* v, int64_t token_stride, const float* q_norm, const float* k_norm, float eps,
                          const int64_t* slots, void* q_out, int32_t q_half, int64_t q_out_stride, uint16_t* k_pages,
                          uint16_t* v_pages, void* stream) {
    pelica::clear_error();
    const int rc = check_pool(d, 4);
    if (rc) return rc;
    return run_qkv(d, rope, nullptr, q, k, v, token_stride, q_norm, k_norm, eps, slots, q_out, q_half, q_out_stride, k_pages,
                   v_pages, stream);
}

int pelica_attn_paged_qkv_q8(const PelicaPagedDesc* d, const PelicaPagedRope* rope, const PelicaPagedQ8* q8, const float* q,
                             const float* k, const float* v, int64_t token_stride, const float* q_norm,
                             const float* k_norm, float eps, const int64_t* slots, void* q_out, int32_t q_half,
                             int64_t q_out_stride, int8_t* k_pages, int8_t* v_pages, void* stream) {
    pelica::clear_error();
    const int rc = check_q8(d, q8);
    if (rc) return rc;
    return run_qkv(d, rope, q8, q, k, v, token_stride, q_norm, k_norm, eps, slots, q_out, q_half, q_out_stride, k_pages,
                   v_pages, stream);
}

int pelica_attn_paged_q8(const PelicaPagedDesc* d, const PelicaPagedQ8* q8, const void* plan, size_t plan_bytes, const void* q,
                         int32_t half, const int8_t* k_pages, const int8_t* v_pages, const float* sinks, void* out,
                         void* workspace, size_t workspace_bytes, void* stream) {
    pelica::clear_error();
    int rc = check_paged(d);
    if (!rc) rc = check_q8(d, q8);
    if (rc) return rc;
    return run_paged(d, nullptr, q8, plan, plan_bytes, q, k_pages, v_pages, sinks, out, workspace, workspace_bytes, half == 0, stream);
}

size_t pelica_attn_paged_shared_plan_bytes(const PelicaPagedDesc* d, const PelicaPagedShared* shared) {
    pelica::clear_error();
    if (check_shared(d, shared)) return 0;
    return plan_of(d, shared).bytes;
}

int pelica_attn_paged_shared_plan(const PelicaPagedDesc* d, const PelicaPagedShared* shared, void* plan, size_t plan_bytes,
                                  void* stream) {
    pelica::clear_error();
    int rc = check_shared(d, shared);
    if (rc) return rc;
    const PagedPlan x = plan_of(d, shared);
    pelica::SharedPlanParams p{};
    rc = plan_params(d, x, plan, plan_bytes, p.plan);
    if (rc) return rc;
    p.group_start = shared->group_start;
    p.shared_len = shared->shared_len;
    p.joins = reinterpret_cast<pelica::SharedJoin*>(static_cast<char*>(plan) + x.join_at);
    p.n_groups = shared->n_groups;
    const hipError_t e = pelica::launch_paged_shared_plan(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(PELICA_ATTN_EHIP, "paged_shared_plan launch: %s", hipGetErrorString(e));
    return PELICA_ATTN_OK;
}

size_t pelica_attn_paged_shared_workspace_bytes(const PelicaPagedDesc* d, const PelicaPagedShared* shared) {
    pelica::clear_error();
    if (check_shared(d, shared)) return 0;
    return plan_of(d, shared).ws_bytes;
}

int pelica_attn_paged_shared(const PelicaPagedDesc* d, const PelicaPagedShared* shared, const PelicaPagedQ8* q8, const void* plan,
                             size_t plan_bytes, const void* q, int32_t half, const void* k_pages, const void* v_pages,
                             const float* sinks, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    pelica::clear_error();
    int rc = check_shared(d, shared);
    if (!rc && q8) rc = check_q8(d, q8);
    if (rc) return rc;
    return run_paged(d, shared, q8, plan, plan_bytes, q, k_pages, v_pages, sinks, out, workspace, workspace_bytes, half == 0, stream);
}

int pelica_attn_pages_read(const PelicaPagedDesc* d, const PelicaPagedQ8* q8, const int64_t* slots, const void* k_pages,
                           const void* v_pages, uint16_t* k_out, uint16_t* v_out, int64_t out_stride, void* stream) {
    pelica::clear_error();
    const int rc = q8 ? check_q8(d, q8) : check_pool(d, 8);
    if (rc) return rc;
    if (d->hd != 64 && d->hd != 128 && d->hd != 256) return fail(PELICA_ATTN_EUNSUPPORTED, "hd %d (64, 128 or 256)", d->hd);
    if (!slots || !k_pages || !v_pages || !k_out || !v_out)
        return fail(PELICA_ATTN_EINVAL, "slots, the pages, k_out and v_out must be non-NULL");
    if (misaligned(k_pages) || misaligned(v_pages) || misaligned(k_out) || misaligned(v_out) || misaligned(slots, 8))
        return fail(PELICA_ATTN_EINVAL, "pages, k_out and v_out must be 16-byte aligned, slots 8");
    if (k_out == v_out || k_out == k_pages || v_out == v_pages || k_out == v_pages || v_out == k_pages)
        return fail(PELICA_ATTN_EINVAL, "k_out, v_out and the pages must be different arrays");
    const int64_t row = (int64_t)d->n_kv * d->hd;
    if (out_stride && (out_stride < row || out_stride % 8 || out_stride >= 1LL << 31))
        return fail(PELICA_ATTN_EINVAL, "out_stride %lld: 0, or >= n_kv*hd (%lld), < 2^31 and a multiple of 8", (long long)out_stride,
                    (long long)row);
    if (d->n_tokens * row > 1LL << 33) return fail(PELICA_ATTN_EUNSUPPORTED, "more than 2^33 values");
    // (other workgroups read while one writes)
    const int size = q8 ? 1 : 2;
    const int64_t step = 2 * (out_stride ? out_stride : row);
    const int64_t page_bytes = size * ((d->page_size - 1) * row_stride(d) + (d->n_kv - 1) * head_stride(d) + d->hd);
    const Pieces k_rows{"k_out", k_out, d->n_tokens, step, 2 * row}, v_rows{"v_out", v_out, d->n_tokens, step, 2 * row};
    Pieces others[6] = {v_rows, {"slots", slots, 1, 8LL * d->n_tokens, 8LL * d->n_tokens},
                        {"k_pages", k_pages, d->n_pages, page_stride(d) * size, page_bytes},
                        {"v_pages", v_pages, d->n_pages, page_stride(d) * size, page_bytes}};
    int n_others = 4;
    if (q8) {
        const pelica::Q8Strides sc = scale_strides(d, q8);
        const int64_t bytes = 2 * ((d->page_size - 1) * sc.row + (d->n_kv - 1) * sc.head + d->hd / pelica::kQ8Group);
        others[n_others++] = {"k_scales", q8->k_scales, d->n_pages, 2 * sc.page, bytes};
        others[n_others++] = {"v_scales", q8->v_scales, d->n_pages, 2 * sc.page, bytes};
    }
    for (int i = 0; i < n_others; ++i) {
        if (may_overlap(k_rows, others[i])) return fail(PELICA_ATTN_EINVAL, "pages_read: k_out overlaps %s", others[i].name);
        if (i > 0 && may_overlap(v_rows, others[i])) return fail(PELICA_ATTN_EINVAL, "pages_read: v_out overlaps %s", others[i].name);
    }
    pelica::PagesReadParams p{};
    p.slots = slots;
    p.k = static_cast<const char*>(k_pages);
    p.v = static_cast<const char*>(v_pages);
    if (q8) {
        p.k_scales = q8->k_scales;
        p.v_scales = q8->v_scales;
        p.sc = scale_strides(d, q8);
    }
    p.k_out = k_out;
    p.v_out = v_out;
    p.page_b = page_stride(d) * size;
    p.row_b = row_stride(d) * size;
    p.head_b = head_stride(d) * size;
    p.out_stride = out_stride ? out_stride : row;
    p.page_log2 = log2_of(d->page_size);
    p.n_slots = (int64_t)d->n_pages << p.page_log2;
    p.n_tokens = d->n_tokens;
    p.n_kv = d->n_kv;
    p.hd = d->hd;
    const hipError_t e = pelica::launch_pages_read(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(PELICA_ATTN_EHIP, "pages_read launch: %s", hipGetErrorString(e));
    return PELICA_ATTN_OK;
}

}  // extern "C"

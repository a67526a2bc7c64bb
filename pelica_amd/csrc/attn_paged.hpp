// Launch parameters of the paged kernels (attn_pages.hip, attn_paged.hip,
// attn_paged_qkv.hip).
#pragma once
#include <cmath>

#include "attn_common.hpp"
#include "attn_paged_plan.hpp"

namespace pelica {

constexpr int kPagedMaxSeq = 4096;

struct PagesParams {
    const int32_t *cached, *fresh, *ended;
    const int64_t* free_in;
    int64_t* free_out;
    int32_t *table, *list, *q_start, *kv_len, *positions, *token_seq, *status;
    int64_t* slots;
    int n_seq, n_tokens, page_log2, n_pages, max_pages;
};
hipError_t launch_pages_append(const PagesParams& p, hipStream_t st);
hipError_t launch_pages_release(const PagesParams& p, hipStream_t st);

struct PlanParams {
    const int32_t *q_start, *kv_len, *prefix;
    PlanHeader* head;
    PlanJoin* joins;
    PlanPiece* pieces;
    int n_seq, n_tokens, max_q, hpk, hd, window, fill;
    int64_t max_keys;
    int max_joins, max_pieces;
    int max_slots;  // most pieces of split items
    int rows;       // partial rows of a kv head and piece
    bool split;     // no: every item is one piece
    uint32_t sig;
};
hipError_t launch_paged_plan(const PlanParams& p, hipStream_t st);

constexpr int kSharedMaxGroups = 1024;
struct SharedPlanParams {
    PlanParams plan;
    const int32_t *group_start, *shared_len;
    SharedJoin* joins;
    int n_groups;
};
hipError_t launch_paged_shared_plan(const SharedPlanParams& p, hipStream_t st);

struct PagedParams {
    const void* q;
    const uint16_t *k, *v;
    const PlanHeader* head;
    const PlanPiece* pieces;
    const int32_t* table;
    const float *sinks, *alibi;
    const float *sinks_or_q, *alibi_or_q;  // (never NULL: a load that needs no branch)
    double inv_hpk;             // 1 / hpk
    void* out;
    float* ws_ml;               // of a piece [n_kv][its rows] x (max, sum), base-2 max
    float* ws_o;                // [n_kv][its rows][hd]
    const PlanJoin* joins;
    int64_t page_b, head_b;     // bytes between pages, between kv heads of a row
    int64_t q_tok, o_tok;       // values between tokens
    uint32_t row_b, sig;        // bytes between rows of a page
    int n_kv, hpk, n_pages, max_pages, page_log2, window, rows;
    float qscale, cap;          // scale * log2 e; softcap (0: none)
    // of raw products up to tanh_to[i]: the capped score (log2 domain) as s times
    // a polynomial in s^2, of f32 and of f16 queries
    float tanh_c[5], tanh_h[3], tanh_to[2];
    // host side only
    int hd, max_pieces, max_joins, max_rows;  // (of a request's item)
    int all_rows;                             // n_tokens n_head
    bool f32, wide;
    // (behind what all calls read: a line of the arguments more is a round trip more)
    const SharedJoin* shared_joins;  // (not NULL: a plan of shared keys)
    // 8-bit pages: scales, bytes between pages, heads, rows of theirs
    const uint16_t *ks, *vs;
    int64_t spage_b, shead_b;
    uint32_t srow_b;
};
// cap tanh(y), y = s scale / cap, of small y: tanh(y) / y as the polynomial in
// y^2 that interpolates it at the Chebyshev nodes of [0, y_max^2].  Up to 0.55:
// 2^-22.7 relative with every rounding counted.  (1 - 2 / (1 + e^2y) is off by
// 2^-23 of the cap, however small the score is.)  Of f16 queries
// three terms, up to 0.3: 1.2e-6 relative, less than the roundings of a large
// score's own products; at cap 50 a weight is off by 1.7e-5 (2^-15.8) at most,
// where f16 rounds it by 2^-11.  (2000 tokens of head dim 64: five terms 97 us, three 83.)
inline void capped_poly(PagedParams& p) {
    if (!(p.cap > 0.f)) return;
    const double f = (double)p.qscale / kLog2e / p.cap;  // y = f s
    auto scaled = [&](const double* c, int n, double most, float* to, float& limit) {
        double g = (double)p.cap * kLog2e * f;
        limit = (float)(most / f);
        for (int i = 0; i < n; ++i, g *= f * f) {
            to[i] = (float)(c[i] * g);
            // (a tiny cap: all scores take the other form)
            if (!(std::fabs(c[i] * g) < 1e30)) limit = -1.f;
        }
    };
    constexpr double c[5] = {0.999999967298071, -0.333327914802321, 0.133188187804409, -0.05258626003574007, 0.01631040386184039};
    constexpr double h[3] = {0.9999988351337193, -0.33309988804316676, 0.1263358239158045};
    scaled(c, 5, 0.55, p.tanh_c, p.tanh_to[0]);
    scaled(h, 3, 0.3, p.tanh_h, p.tanh_to[1]);
}

constexpr int kQ8Group = 32;  // values that share a scale
struct Q8Strides {
    int64_t page, row, head;  // f16 values
};

hipError_t launch_paged(const PagedParams& p, hipStream_t st);
hipError_t launch_paged_q8(const PagedParams& p, hipStream_t st);
hipError_t launch_paged_join(const PagedParams& p, hipStream_t st);

struct PagedQkvParams {
    const float *q, *k, *v, *q_norm, *k_norm, *table;
    const int64_t* slots;
    const int32_t* positions;
    void* q_out;
    uint16_t *k_pages, *v_pages;      // (f16 values, or 8-bit ones with scales)
    uint16_t *k_scales, *v_scales;
    Q8Strides sc;
    int64_t tok_q, tok_kv, tok_o, axis_stride;
    int64_t page_stride, row_stride, head_stride, n_slots;
    int n_head, n_kv, n_tokens, rot, neox, table_split, covered, page_log2, n_axes;
    float eps;
    uint32_t axis[8];  // 2 bits a pair
    int hd;            // host side only
    bool half, q8;
};
hipError_t launch_paged_qkv(const PagedQkvParams& p, hipStream_t st);

struct PagesReadParams {
    const int64_t* slots;
    const char *k, *v;
    const uint16_t *k_scales, *v_scales;  // NULL: f16 pages
    uint16_t *k_out, *v_out;
    int64_t page_b, row_b, head_b;        // bytes
    Q8Strides sc;
    int64_t out_stride, n_slots;
    int n_tokens, n_kv, page_log2, hd;
};
hipError_t launch_pages_read(const PagesReadParams& p, hipStream_t st);

}  // namespace pelica

// attn_paged_plan.hpp for ctypes: which keys an item walks, which rows a load touches.
#include "../pelica_amd/csrc/attn_paged_plan.hpp"

using namespace pelica;

extern "C" void item_keys_of(int pos_first, int pos_last, int len, int window, int prefix, int* out) {
    const ItemKeys k = item_keys(pos_first, pos_last, len, window, prefix);
    const int v[] = {k.n_pre, k.lo_base, k.n_chunks, k.lo, k.kend, k.pe};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
}
extern "C" int chunk_key_of(int c, int n_pre, int lo_base) { return chunk_key(c, n_pre, lo_base); }
extern "C" void group_rows_of(int kg, int n, int lo, int kend, int pe, int* out) {
    group_rows(kg, n, lo, kend, pe, out[0], out[1]);
}
extern "C" int gap_in_run_of(int lo, int pe) { return gap_in_run(lo, pe); }
extern "C" int item_pieces_of(int cost, int n_chunks, float limit) { return item_pieces(cost, n_chunks, 1.f / limit); }
extern "C" int64_t plan_items_of(int64_t n_seq, int64_t n_tokens, int hpk, int hd) {
    return plan_items(n_seq, n_tokens, hpk, hd);
}

// Rows of a paged cache as dense f16 rows, by slot: n s of 8-bit pages (a f16
// multiplication, rounded to nearest), or f16 pages as they are.
//
// A lane takes 8 values of a head, of K and of V: 8 bytes and a scale in, 16
// bytes out, each a whole line with its neighbours.  HBM-bound: 30000 rows of 4
// heads of 128 from twelve pools in turn (94 MB a call, 1.1 GB in all: more than
// the caches hold) 22.7 us, 4.2 TB/s with start and end (a copy as large, as cold: 4.8);
// 300000 rows 179 us, 5.3 TB/s (a 1 GiB copy's 5.04); one pool again and again, which
// the 256 MB cache keeps, 16.5 us.  f16 pages 26.9, 236, 19.6 us.  333 rows of 8 heads of 64
// 2.8 us, a launch and two round trips (slot, row).
#include "attn_paged.hpp"
#include "attn_prof.hpp"
#include "attn_q8.hpp"

namespace pelica {

namespace {

template <bool Q8>
__global__ __launch_bounds__(256) void pages_read_kernel(PagesReadParams p, int log2_ppr, int pieces) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;  // (row, head, piece)
    const uint32_t head_at = i >> log2_ppr, piece = i & ((1u << log2_ppr) - 1u);
    const uint32_t t = head_at / (uint32_t)p.n_kv, h = head_at - t * (uint32_t)p.n_kv;
    if (i >= (uint32_t)pieces) return;
    const int64_t row = p.slots[t];
    if (row < 0 || row >= p.n_slots) return;
    const int64_t page = row >> p.page_log2, in = row & ((1LL << p.page_log2) - 1);
    const int64_t at = page * p.page_b + in * p.row_b + (int64_t)h * p.head_b;
    const int64_t to = (int64_t)t * p.out_stride + (int64_t)h * p.hd + 8 * piece;
    half8 k, v;
    if constexpr (Q8) {
        const int64_t sc = page * p.sc.page + in * p.sc.row + (int64_t)h * p.sc.head + piece / 4;
        const u32x2 a = *reinterpret_cast<const u32x2*>(p.k + at + 8 * piece);
        const u32x2 b = *reinterpret_cast<const u32x2*>(p.v + at + 8 * piece);
        k = q8_values(a, p.k_scales[sc]);
        v = q8_values(b, p.v_scales[sc]);
    } else {
        k = load16(p.k + at + 16 * piece);
        v = load16(p.v + at + 16 * piece);
    }
    *reinterpret_cast<half8*>(p.k_out + to) = k;
    *reinterpret_cast<half8*>(p.v_out + to) = v;
}

}  // namespace

hipError_t launch_pages_read(const PagesReadParams& p, hipStream_t st) {
    const int ppr = p.hd / 8, pieces = p.n_tokens * p.n_kv * ppr;
    ProfScope ps(kProfPagesRead, st);
    auto kernel = p.k_scales ? pages_read_kernel<true> : pages_read_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((pieces + 255) / 256), dim3(256), 0, st, p, __builtin_ctz(ppr), pieces);
    return hipGetLastError();
}

}  // namespace pelica

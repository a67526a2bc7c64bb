// The paged attention kernels over f16 pages, and the join of split items.
#include "attn_paged_body.hpp"

namespace pelica {

namespace {

// The pieces of a split item, joined with the sink: per row (M, L, O) of each
// slot, weights 2^(M_i - M).  HD / 4 lanes hold a row's dims, 4 each; a wave's
// lane groups (and WPR waves) take one row's slots in turn and meet through
// lane exchanges and LDS in a fixed order, or, where the slots are few, a
// row each.  Bound by the partials' bytes (a mixed step's 48 MB: 12.7 us, 3.8
// TB/s), and for single tokens by its two round trips (plan, partials) behind
// the attention kernel: 3.9 - 4.8 us.
template <int HD, bool F32, int WPR, bool SHARED>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p) {
    constexpr int LPR = HD / 4, GPW = 64 / LPR, U = 4;
    __shared__ float st[WPR > 1 ? WPR : 1][64][6];
    const int j = blockIdx.x / p.n_kv, kvh = blockIdx.x % p.n_kv;
    const std::conditional_t<SHARED, SharedJoin, PlanJoin> z = [&] {
        if constexpr (SHARED) return p.shared_joins[j];
        else return p.joins[j];
    }();
    const uint32_t sig = p.head->sig;
    const int n_joins = p.head->n_joins;
    __asm__ volatile("" ::"s"(z.q0), "s"(z.r0), "s"(sig), "s"(n_joins));
    if (sig != p.sig || j >= n_joins) return;
    int rows, n_slots;
    if constexpr (SHARED) rows = z.rows, n_slots = z.k + max(z.g_k, z.g_k2);
    else rows = min(z.R - z.r0, p.rows), n_slots = z.n_slots;
    // row r of partial sl
    auto partial = [&](int sl, int r) -> size_t {
        if constexpr (SHARED) {
            if (sl < z.k) return (size_t)(z.at + sl * z.rows) * p.n_kv + (size_t)kvh * z.rows + r;
            constexpr int W = wide_rows(HD);
            const int gr = z.g_row + r, b = gr / W, of = min(W, z.g_R - b * W);
            const bool last = (b + 1) * W >= z.g_R;
            if (sl - z.k >= (last ? z.g_k2 : z.g_k)) return ~(size_t)0;  // (the other block's)
            const int at = last ? z.g_at2 : z.g_at + b * W * z.g_k;
            return (size_t)(at + (sl - z.k) * of) * p.n_kv + (size_t)kvh * of + (gr - b * W);
        } else {
            return ((size_t)(z.slot0 + sl) * p.n_kv + kvh) * p.rows + r;
        }
    };
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = 4 * (lane % LPR), grp = lane / LPR;
    const bool spread = WPR > 1 || n_slots > 8;  // a row's slots over the lane groups
    const int ph = WPR > 1 ? wave * GPW + grp : spread ? grp : 0, n_ph = WPR > 1 ? GPW * WPR : spread ? GPW : 1;
    const int per_wave = spread ? 1 : GPW;  // rows
    const int step = WPR > 1 ? (int)gridDim.y : (int)gridDim.y * 4 * per_wave;
    for (int r0 = WPR > 1 ? (int)blockIdx.y : ((int)blockIdx.y * 4 + wave) * per_wave; r0 < rows; r0 += step) {
        const int r = min(r0 + (spread ? 0 : grp), rows - 1);
        float m = -INFINITY, l = 0.f;
        float4v o = {};
        for (int s0 = 0; s0 < n_slots; s0 += n_ph * U) {
            float2 ml[U];
            float4v v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int sl = s0 + ph + n_ph * u;
                ml[u] = make_float2(-INFINITY, 0.f);
                v[u] = float4v{};
                bool there = sl < n_slots;
                size_t at = 0;
                if constexpr (SHARED) {
                    at = there ? partial(sl, r) : 0;
                    there &= at != ~(size_t)0;
                }
                if (there) {
                    if constexpr (!SHARED) at = partial(sl, r);
                    ml[u] = reinterpret_cast<const float2*>(p.ws_ml)[at];
                    v[u] = *reinterpret_cast<const float4v*>(p.ws_o + at * HD + d);
                }
            }
            float mb = m;
#pragma unroll
            for (int u = 0; u < U; ++u) mb = fmaxf(mb, ml[u].x);
            const float ms = mb == -INFINITY ? 0.f : mb, f = fast_exp2(m - ms);
            l *= f;
            o *= f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float w = fast_exp2(ml[u].x - ms);
                l += ml[u].y * w;
                o += v[u] * w;
            }
            m = mb;
        }
        if (spread) {
#pragma unroll
            for (int off = LPR; off < 64; off <<= 1) {
                const float m2 = __shfl_xor(m, off, 64), l2 = __shfl_xor(l, off, 64);
                const float M = fmaxf(m, m2), ms = M == -INFINITY ? 0.f : M;
                const float a = fast_exp2(m - ms), b = fast_exp2(m2 - ms);
                l = l * a + l2 * b;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = o[i] * a + __shfl_xor(o[i], off, 64) * b;
                m = M;
            }
        }
        if (WPR > 1) {
            __syncthreads();
            float* x = st[wave][lane];
            x[0] = m, x[1] = l, x[2] = o[0], x[3] = o[1], x[4] = o[2], x[5] = o[3];
            __syncthreads();
            if (wave > 0) continue;
            float M = m;
#pragma unroll
            for (int w = 1; w < WPR; ++w) M = fmaxf(M, st[w][lane][0]);
            const float ms = M == -INFINITY ? 0.f : M, f = fast_exp2(m - ms);
            l *= f;
            o *= f;
#pragma unroll
            for (int w = 1; w < WPR; ++w) {
                const float* y = st[w][lane];
                const float g = fast_exp2(y[0] - ms);
                l += y[1] * g;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] += y[2 + i] * g;
            }
            m = M;
        }
        if (spread ? lane >= LPR : r0 + grp >= rows) continue;
        const int rr = z.r0 + r, t = token_of(p, rr), h = kvh * p.hpk + rr - t * p.hpk;
        o *= row_weight(sink_of(p, h), m, l);
        const size_t at = (size_t)(z.q0 + t) * p.o_tok + (size_t)h * HD + d;
        if constexpr (F32) {
            *reinterpret_cast<float4v*>(static_cast<float*>(p.out) + at) = o;
        } else {
            *reinterpret_cast<half4*>(static_cast<uint16_t*>(p.out) + at) =
                half4{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
        }
    }
}

}  // namespace

hipError_t launch_paged(const PagedParams& p, hipStream_t st) { return launch_paged_as<false>(p, st); }

hipError_t launch_paged_join(const PagedParams& p, hipStream_t st) {
    ProfScope ps(kProfPagedJoin, st);
    return with_shape(p, [&](auto hd, auto f32) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool F32 = decltype(f32)::value;
        const unsigned x = (unsigned)p.max_joins * p.n_kv;
        if (p.shared_joins) {
            // a row a wave, or, of rows that leave most of the chip idle, a workgroup
            // (8 chats of 32 heads: 5.9 -> 3.9 us)
            if (p.all_rows <= 2048) {
                hipLaunchKernelGGL((paged_join_kernel<HD, F32, 4, true>), dim3(x, std::min(p.max_rows, 32)), dim3(256), 0, st, p);
            } else {
                const unsigned y = (unsigned)std::min((p.max_rows + 3) / 4, 16);
                hipLaunchKernelGGL((paged_join_kernel<HD, F32, 1, true>), dim3(x, y), dim3(256), 0, st, p);
            }
        } else if (p.wide) {
            hipLaunchKernelGGL((paged_join_kernel<HD, F32, 1, false>), dim3(x, 16), dim3(256), 0, st, p);
        } else {
            hipLaunchKernelGGL((paged_join_kernel<HD, F32, 4, false>), dim3(x, std::min(p.rows, 32)), dim3(256), 0, st, p);
        }
        return hipGetLastError();
    });
}

}  // namespace pelica

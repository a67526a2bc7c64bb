// The step before attention over pages: per-head RMS norm of the q and k heads
// (x w / sqrt(mean x^2 + eps)), rotary embedding with a position per axis
// (pair j turns by the angle of row positions[axis(j)] of the table), q to its
// own rows (f32 or f16), k and v rounded to f16 into the row of the token's
// slot.
//
// Head slots [0, n_head) are q heads, then n_kv k heads, then n_kv v heads; a
// lane holds 4 consecutive elements (16-byte accesses), a wave IT groups of
// 64 / (HD / 4) heads of one token, whose (cos, sin) it loads once.
// HBM-bound: every byte is touched once; small steps are one dependent chain
// of loads (slot and positions, table rows beside the heads) and stores.
#include <type_traits>

#include "attn_paged.hpp"
#include "attn_prof.hpp"

namespace pelica {

namespace {

// EX: rotation partners lie whole lanes away (or in the lane); else they are
// exchanged through LDS (NeoX pairs, rot not a multiple of 8).
template <int HD, int IT, bool HALF, bool EX>
__global__ __launch_bounds__(256) void paged_qkv_kernel(PagedQkvParams p, int wg_heads) {
    constexpr int LPH = HD / 4, HPW = 64 / LPH;
    __shared__ float xch[EX ? 1 : 4][EX ? 1 : HPW][EX ? 1 : HD];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, sub = lane / LPH, e0 = 4 * (lane % LPH);
    const int t = blockIdx.x / wg_heads, n_slot = p.n_head + 2 * p.n_kv;
    const int slot0 = ((blockIdx.x % wg_heads) * 4 + wave) * (HPW * IT) + sub;
    if (slot0 - sub >= n_slot) return;
    const int64_t row = p.slots[t];
    float4v x[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const int h = min(slot0 + HPW * it, n_slot - 1), hk = h - p.n_head, hv = hk - p.n_kv;
        const float* src = hk < 0 ? p.q + (size_t)t * p.tok_q + (size_t)h * HD
                                  : (hv < 0 ? p.k + (size_t)hk * HD : p.v + (size_t)hv * HD) + (size_t)t * p.tok_kv;
        x[it] = *reinterpret_cast<const float4v*>(src + e0);
    }
    const float4v one = {1.f, 1.f, 1.f, 1.f};
    const float4v wq = p.q_norm ? *reinterpret_cast<const float4v*>(p.q_norm + e0) : one;
    const float4v wk = p.k_norm ? *reinterpret_cast<const float4v*>(p.k_norm + e0) : one;
    // cos, sin of this lane's elements
    const int half = p.rot / 2;
    const bool rot = e0 < p.rot;
    float c[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
    if (rot) {
        int pos[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) pos[a] = a < p.n_axes ? p.positions[(size_t)a * p.axis_stride + t] : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = e0 + i;
            if (e >= p.rot) continue;
            const int j = p.neox ? (e < half ? e : e - half) : e >> 1;
            int at = pos[0];
            if (p.n_axes > 1) {
                uint32_t word = p.axis[0];
#pragma unroll
                for (int w = 1; w < 8; ++w) word = (j >> 4) == w ? p.axis[w] : word;
                const int a = (word >> (2 * (j & 15))) & 3;
                at = a == 0 ? pos[0] : a == 1 ? pos[1] : a == 2 ? pos[2] : pos[3];
            }
            if ((unsigned)at >= (unsigned)p.covered) {
                c[i] = sn[i] = NAN;
            } else if (p.table_split <= 0) {
                const float2 v = *reinterpret_cast<const float2*>(p.table + ((size_t)at * half + j) * 2);
                c[i] = v.x, sn[i] = v.y;
            } else {
                // angle addition of the rows for pos / 256 and pos % 256
                const float2 u = *reinterpret_cast<const float2*>(p.table + ((size_t)(at >> 8) * half + j) * 2);
                const float2 v = *reinterpret_cast<const float2*>(
                    p.table + ((size_t)(p.table_split + (at & 255)) * half + j) * 2);
                c[i] = u.x * v.x - u.y * v.y;
                sn[i] = u.y * v.x + u.x * v.y;
            }
        }
    }
    if (row < 0 || row >= p.n_slots) return;  // (uniform: a padding row)
    const int64_t base = (row >> p.page_log2) * p.page_stride + (row & ((1LL << p.page_log2) - 1)) * p.row_stride;
    const bool hi = p.neox && e0 >= half;
    const int partner = !rot || !p.neox ? lane : hi ? lane - half / 4 : lane + half / 4;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const int h = slot0 + HPW * it, hk = h - p.n_head, hv = hk - p.n_kv;
        float4v y = x[it];
        if (p.q_norm || p.k_norm) {
            float ss = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll
            for (int off = LPH / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
            if (hk < 0 ? p.q_norm != nullptr : hv < 0 && p.k_norm) {
                const float inv = 1.f / __builtin_sqrtf(ss / (float)HD + p.eps);
                const float4v w = hk < 0 ? wq : wk;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = y[i] * inv * w[i];
            }
        }
        if (p.rot) {
            float4v z;
            if constexpr (EX) {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = p.neox ? __shfl(y[i], partner, 64) : y[i ^ 1];
            } else {
                // (a wave's LDS accesses complete in order)
                *reinterpret_cast<float4v*>(&xch[wave][sub][e0]) = y;
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = e0 + i;
                    z[i] = xch[wave][sub][e >= p.rot ? e : p.neox ? (e < half ? e + half : e - half) : e ^ 1];
                }
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            }
            if (rot && hv < 0) {
                float4v r;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool second = p.neox ? e0 + i >= half : (i & 1) != 0;
                    r[i] = e0 + i >= p.rot ? y[i] : second ? z[i] * sn[i] + y[i] * c[i] : y[i] * c[i] - z[i] * sn[i];
                }
                y = r;
            }
        }
        if (h >= n_slot) break;
        const half4 f = {(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
        if (hk < 0) {
            const size_t at = (size_t)t * p.tok_o + (size_t)h * HD + e0;
            if constexpr (HALF) *reinterpret_cast<half4*>(static_cast<uint16_t*>(p.q_out) + at) = f;
            else *reinterpret_cast<float4v*>(static_cast<float*>(p.q_out) + at) = y;
        } else {
            uint16_t* dst = hv < 0 ? p.k_pages + (int64_t)hk * p.head_stride : p.v_pages + (int64_t)hv * p.head_stride;
            *reinterpret_cast<half4*>(dst + base + e0) = f;
        }
    }
}

}  // namespace

hipError_t launch_paged_qkv(const PagedQkvParams& p, hipStream_t st) {
    const int hpw = 64 / (p.hd / 4), n_slot = p.n_head + 2 * p.n_kv;
    const int groups = (n_slot + hpw - 1) / hpw;
    // one group a wave while a step waits for its one round trip, two once its
    // bytes bound it
    const int it = (long long)groups * p.n_tokens <= 10240 ? 1 : 2;
    const int wg_heads = ((groups + it - 1) / it + 3) / 4;
    const bool ex = !p.neox || p.rot % 8 == 0;
    ProfScope ps(kProfPagedQkv, st);
    const dim3 grid((unsigned)p.n_tokens * wg_heads);
    auto go = [&](auto hd, auto i, auto half, auto e) {
        hipLaunchKernelGGL((paged_qkv_kernel<decltype(hd)::value, decltype(i)::value, decltype(half)::value, decltype(e)::value>),
                           grid, dim3(256), 0, st, p, wg_heads);
        return hipGetLastError();
    };
    auto c = [&](auto hd, auto i, auto half) {
        return ex ? go(hd, i, half, std::true_type{}) : go(hd, i, half, std::false_type{});
    };
    auto b = [&](auto hd, auto i) { return p.half ? c(hd, i, std::true_type{}) : c(hd, i, std::false_type{}); };
    auto a = [&](auto hd) {
        return it == 1 ? b(hd, std::integral_constant<int, 1>{}) : b(hd, std::integral_constant<int, 2>{});
    };
    switch (p.hd) {
        case 64: return a(std::integral_constant<int, 64>{});
        case 128: return a(std::integral_constant<int, 128>{});
        case 256: return a(std::integral_constant<int, 256>{});
        default: return hipErrorNotSupported;
    }
}

}  // namespace pelica

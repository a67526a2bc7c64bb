// The step before attention over pages: per-head RMS norm of the q and k heads
// (x w / sqrt(mean x^2 + eps)), rotary embedding with a position per axis
// (pair j turns by the angle of row positions[axis(j)] of the table), q to its
// own rows (f32 or f16), k and v rounded to f16 into the row of the token's
// slot; or to 8-bit integers and a scale for each 32 values (Q8): s the smallest
// f16 number with 127 s >= the group's largest magnitude, n = x / s to nearest
// (4000 tokens as below 29.3 us, 32 tokens 4.6: k's 64-bit work and its registers).
//
// Head slots [0, n_head) are q heads, then n_kv k heads, then n_kv v heads.  A
// lane holds 8 elements of a head, 4 from each half of the rotated part (and
// of the rest): NeoX pairs (j, j + rot / 2) and neighbouring pairs both lie in
// one lane, so a rotation moves nothing between lanes.  A wave takes IT groups
// of 64 / (HD / 8) heads of one token.  The token's (cos, sin) come once a
// wave, a pair a lane whatever axis it turns by, and through LDS to the lanes
// that need them.
// HBM-bound in large steps (4000 tokens of 32 + 4 heads of 128, three axes: 24.3
// us, 5.1 TB/s, a copy's rate), where the instructions a value costs come next
// (4 elements a lane, partners over lane exchanges: 36 us; four scattered table
// loads a lane as well: 42.9); small steps are one dependent chain of loads (slot
// and positions, table rows beside the heads) and stores: 32 tokens 3.7 us.
#include <type_traits>

#include "attn_paged.hpp"
#include "attn_prof.hpp"

namespace pelica {

namespace {

template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false));
}

// Sum over the N (8, 16, 32) lanes of a head, in every one of them.
template <int N>
__device__ __forceinline__ float head_sum(float x) {
    x = add_dpp<0xB1>(x);   // lane ^ 1
    x = add_dpp<0x4E>(x);   // lane ^ 2
    x = add_dpp<0x141>(x);  // the other four of eight
    if constexpr (N >= 16) x = add_dpp<0x140>(x);  // the other eight of sixteen
    if constexpr (N >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// 1 / sqrt(x) to the last bit or two: the instruction's result (1 unit) after
// values below its range are scaled into it.
__device__ __forceinline__ float rsqrt_full(float x) {
    const bool small = x < 0x1p-100f;
    return __builtin_amdgcn_rsqf(small ? x * 0x1p100f : x) * (small ? 0x1p50f : 1.f);
}

__device__ __forceinline__ half4 to_half(float4v x) {
    return {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}

// max over lanes l, l ^ 1, l ^ 2, l ^ 3
__device__ __forceinline__ double quad_max(double x) {
    auto with = [&](auto moved) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint64_t v = (uint64_t)(uint32_t)moved((int)(u >> 32)) << 32 | (uint32_t)moved((int)u);
        x = fmax(x, __builtin_bit_cast(double, v));
    };
    with([](int v) { return __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false); });
    with([](int v) { return __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false); });
    return x;
}

// the last bytes of eight words
__device__ __forceinline__ u32x2 last_bytes(const uint32_t (&n)[8]) {
    auto pack = [&](int i) {
        const uint32_t lo = __builtin_amdgcn_perm(n[i + 1], n[i], 0x0C0C0400u), hi = __builtin_amdgcn_perm(n[i + 3], n[i + 2], 0x04000C0Cu);
        return lo | hi;
    };
    return u32x2{pack(0), pack(4)};
}

// Eight consecutive values of a lane, a group in four lanes, as 8-bit integers
// and their scale's bits.  Of v, whose values are given: the quotient's integer,
// put right by its remainder.
__device__ __forceinline__ u32x2 quantise8(const float4v& a, const float4v& b, uint16_t& scale) {
    // (as integers an infinity or a NaN is larger than all numbers)
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        top = max(top, max(__float_as_uint(a[i]) & 0x7FFFFFFFu, __float_as_uint(b[i]) & 0x7FFFFFFFu));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp((int)top, (int)top, 0xB1, 0xF, 0xF, false));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp((int)top, (int)top, 0x4E, 0xF, 0xF, false));
    const float most = __uint_as_float(top);
    uint16_t bits = __builtin_bit_cast(uint16_t, (_Float16)(most * (1.f / 127.f)));
    // (that is one of the two f16 numbers around the quotient; 127 s is exact in f32)
    if ((float)__builtin_bit_cast(_Float16, bits) * 127.f < most) ++bits;
    if (!(most < INFINITY)) bits = 0x7E00;
    const float f = (float)__builtin_bit_cast(_Float16, bits);
    const float inv = f > 0.f ? __builtin_amdgcn_rcpf(f) : 0.f, half = 0.5f * f;
    scale = bits;
    // the sum's last byte is n: 2^23 takes the places behind the point.  The
    // remainder is exact by the fma; of two integers as near the even one is taken.
    uint32_t n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = i < 4 ? a[i & 3] : b[i & 3];
        float t = __builtin_fmaf(x, inv, 12582912.f);
        const float r = __builtin_fmaf(12582912.f - t, f, x);
        const float most_r = __uint_as_float(__float_as_uint(half) - (__float_as_uint(t) & 1u));
        t += r > most_r ? 1.f : r < -most_r ? -1.f : 0.f;
        n[i] = __float_as_uint(t);
    }
    return last_bytes(n);
}

// Of k, in 64 bits as its norm and turn are: an integer next to a border is
// decided by a value's last bits (in f32 1 of 30000 was the other one; 4000 tokens
// of 32 + 4 heads of 128 took 26.6 us, and take 29.8).
__device__ __forceinline__ u32x2 quantise8(const double (&x)[8], uint16_t& scale) {
    double top = 0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        top = fmax(top, fabs(x[i]));
        bad |= !(fabs(x[i]) < INFINITY);
    }
    top = quad_max(bad ? INFINITY : top);
    uint16_t bits = __builtin_bit_cast(uint16_t, (_Float16)((float)top * (1.f / 127.f)));
    // (that is one of the two f16 numbers around the quotient)
    if ((double)__builtin_bit_cast(_Float16, bits) * 127 < top) ++bits;
    if (!(top < INFINITY)) bits = 0x7E00;
    const double s = (double)__builtin_bit_cast(_Float16, bits);
    const double inv = s > 0 ? 1 / s : 0;
    scale = bits;
    uint32_t n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // the quotient, rounded once, and 2^52: the sum's last byte is n
        const double y = x[i] * inv, q = fma(fma(-y, s, x[i]), inv, y);
        n[i] = (uint32_t)__builtin_bit_cast(uint64_t, q + 6755399441055744.0);
    }
    return last_bytes(n);
}

// EX: a lane holds both values of its pairs; else (rot not a multiple of 8)
// partners are exchanged through LDS.
template <int HD, int IT, bool HALF, bool EX, bool Q8>
__global__ __launch_bounds__(256) void paged_qkv_kernel(PagedQkvParams p, int tok_waves) {
    constexpr int LPH = HD / 8, HPW = 64 / LPH;
    __shared__ __attribute__((aligned(16))) float turn[4][HD];  // (cos, sin) of the token's pairs
    __shared__ __attribute__((aligned(16))) float xch[EX ? 1 : 4][EX ? 1 : HPW][EX ? 4 : HD];
    __shared__ __attribute__((aligned(16))) double rows8[Q8 ? 4 : 1][Q8 ? HPW : 1][Q8 ? HD : 2];  // k and v heads, normed
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, sub = lane / LPH, l = lane % LPH;
    const uint32_t gw = blockIdx.x * 4u + wave;  // waves follow the tokens, workgroups do not
    const int t = (int)(gw / (uint32_t)tok_waves), n_slot = p.n_head + 2 * p.n_kv;
    const int slot0 = (int)(gw - (uint32_t)t * tok_waves) * (HPW * IT) + sub;
    if (t >= p.n_tokens) return;
    const int half = p.rot / 2;
    const bool rot = EX && l < p.rot / 8;
    // this lane's elements: ea .. ea + 3 and eb .. eb + 3
    const int ea = !EX ? 4 * l : rot ? 4 * l : half + 4 * l;
    const int eb = !EX ? HD / 2 + 4 * l : rot ? half + 4 * l : HD / 2 + 4 * l;
    const int64_t row = p.slots[t];
    float4v x[IT][2];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const int h = min(slot0 + HPW * it, n_slot - 1), hk = h - p.n_head, hv = hk - p.n_kv;
        const float* src = hk < 0 ? p.q + (size_t)t * p.tok_q + (size_t)h * HD
                                  : (hv < 0 ? p.k + (size_t)hk * HD : p.v + (size_t)hv * HD) + (size_t)t * p.tok_kv;
        x[it][0] = *reinterpret_cast<const float4v*>(src + ea);
        x[it][1] = *reinterpret_cast<const float4v*>(src + eb);
    }
    const float4v one = {1.f, 1.f, 1.f, 1.f};
    float4v wq[2] = {one, one}, wk[2] = {one, one};
    if (p.q_norm) {
        wq[0] = *reinterpret_cast<const float4v*>(p.q_norm + ea);
        wq[1] = *reinterpret_cast<const float4v*>(p.q_norm + eb);
    }
    if (p.k_norm) {
        wk[0] = *reinterpret_cast<const float4v*>(p.k_norm + ea);
        wk[1] = *reinterpret_cast<const float4v*>(p.k_norm + eb);
    }
    float4v cs[2] = {one, one};  // (cos, sin) of the lane's pairs: two, two
    if (p.rot) {
        int pos[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) pos[a] = a < p.n_axes ? p.positions[(size_t)a * p.axis_stride + t] : 0;
#pragma unroll
        for (int jj = 0; jj < (HD + 127) / 128; ++jj) {
            const int j = lane + 64 * jj;
            if (j >= half) break;
            int at = pos[0];
            if (p.n_axes > 1) {
                uint32_t word = p.axis[0];
#pragma unroll
                for (int w = 1; w < HD / 32; ++w) word = (j >> 4) == w ? p.axis[w] : word;
                const int a = (word >> (2 * (j & 15))) & 3;
                at = a == 0 ? pos[0] : a == 1 ? pos[1] : a == 2 ? pos[2] : pos[3];
            }
            const bool there = (unsigned)at < (unsigned)p.covered;
            const int at_ = there ? at : 0;
            float2 v = *reinterpret_cast<const float2*>(
                p.table + ((size_t)(p.table_split > 0 ? at_ >> 8 : at_) * half + j) * 2);
            if (p.table_split > 0) {
                // angle addition of the rows for pos / 256 and pos % 256
                const float2 u = *reinterpret_cast<const float2*>(
                    p.table + ((size_t)(p.table_split + (at_ & 255)) * half + j) * 2);
                v = make_float2(v.x * u.x - v.y * u.y, v.y * u.x + v.x * u.y);
            }
            *reinterpret_cast<float2*>(&turn[wave][2 * j]) = there ? v : make_float2(NAN, NAN);
        }
        // (a wave's LDS accesses complete in order)
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        if (rot) {
            // NeoX: pairs ea .. ea + 3; else ea / 2, ea / 2 + 1 and eb / 2, eb / 2 + 1
            cs[0] = *reinterpret_cast<const float4v*>(&turn[wave][p.neox ? 2 * ea : ea]);
            cs[1] = *reinterpret_cast<const float4v*>(&turn[wave][p.neox ? 2 * ea + 4 : eb]);
        }
    }
    if (row < 0 || row >= p.n_slots) return;  // (uniform: a padding row)
    const int64_t base = (row >> p.page_log2) * p.page_stride + (row & ((1LL << p.page_log2) - 1)) * p.row_stride;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const int h = slot0 + HPW * it, hk = h - p.n_head, hv = hk - p.n_kv;
        float4v a = x[it][0], b = x[it][1];
        if constexpr (Q8) {
            // k and v heads through LDS: a group's 32 values to four lanes, eight each
            double* const row8 = rows8[wave][sub];
            float* const row4 = reinterpret_cast<float*>(row8);
            if (hk >= 0 && hv < 0) {
                double inv = 1;
                if (p.k_norm) {
                    double ss = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) ss = fma((double)a[i], (double)a[i], fma((double)b[i], (double)b[i], ss));
#pragma unroll
                    for (int off = 1; off < LPH; off <<= 1) ss += __shfl_xor(ss, off, 64);
                    inv = 1 / sqrt(ss / HD + (double)p.eps);
                }
                double u[4], w[4];  // (wk: ones without a norm)
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = (double)a[i] * inv * (double)wk[0][i], w[i] = (double)b[i] * inv * (double)wk[1][i];
                if (EX && rot) {
                    auto turn2 = [](double& x, double& y, float c, float sn) {
                        const double t = fma(-y, (double)sn, x * (double)c);
                        y = fma(x, (double)sn, y * (double)c);
                        x = t;
                    };
                    if (p.neox) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) turn2(u[i], w[i], cs[i >> 1][2 * (i & 1)], cs[i >> 1][2 * (i & 1) + 1]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            turn2(u[i], u[i + 1], cs[0][i], cs[0][i + 1]);
                            turn2(w[i], w[i + 1], cs[1][i], cs[1][i + 1]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) row8[ea + i] = u[i], row8[eb + i] = w[i];
            } else if (hk >= 0) {
                *reinterpret_cast<float4v*>(row4 + ea) = a;
                *reinterpret_cast<float4v*>(row4 + eb) = b;
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            if (hk >= 0 && h < n_slot) {
                uint16_t s;
                u32x2 n;
                if (hv < 0) {
                    double y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = row8[8 * l + i];
                    if constexpr (!EX) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int e = 8 * l + i;
                            const bool second = p.neox ? e >= half : (e & 1) != 0;
                            const int j = e >= p.rot ? 0 : !p.neox ? e >> 1 : second ? e - half : e;
                            const double z = row8[!p.neox ? e ^ 1 : second ? j : j + half];
                            const double c = (double)turn[wave][2 * j], sn = (double)turn[wave][2 * j + 1];
                            const double r = fma(second ? z : -z, sn, y[i] * c);
                            y[i] = e < p.rot ? r : y[i];
                        }
                    }
                    n = quantise8(y, s);
                } else {
                    n = quantise8(*reinterpret_cast<const float4v*>(row4 + 8 * l), *reinterpret_cast<const float4v*>(row4 + 8 * l + 4), s);
                }
                const bool is_k = hv < 0;
                const int hc = is_k ? hk : hv;
                int8_t* const pages = reinterpret_cast<int8_t*>(is_k ? p.k_pages : p.v_pages);
                *reinterpret_cast<u32x2*>(pages + base + (int64_t)hc * p.head_stride + 8 * l) = n;
                const int64_t at = (row >> p.page_log2) * p.sc.page + (row & ((1LL << p.page_log2) - 1)) * p.sc.row + (int64_t)hc * p.sc.head;
                if (l % 4 == 0) (is_k ? p.k_scales : p.v_scales)[at + l / 4] = s;
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        }
        if (p.q_norm || p.k_norm) {
            const float ss = head_sum<LPH>(((a[0] * a[0] + a[1] * a[1]) + (a[2] * a[2] + a[3] * a[3])) +
                                           ((b[0] * b[0] + b[1] * b[1]) + (b[2] * b[2] + b[3] * b[3])));
            if (hk < 0 ? p.q_norm != nullptr : hv < 0 && p.k_norm) {
                const float inv = rsqrt_full(ss * (1.f / HD) + p.eps);
                const float4v wa = hk < 0 ? wq[0] : wk[0], wb = hk < 0 ? wq[1] : wk[1];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = a[i] * inv * wa[i], b[i] = b[i] * inv * wb[i];
            }
        }
        if constexpr (EX) {
            if (rot && hv < 0) {
                if (p.neox) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float c = cs[i >> 1][2 * (i & 1)], sn = cs[i >> 1][2 * (i & 1) + 1], u = a[i], w = b[i];
                        a[i] = u * c - w * sn;
                        b[i] = u * sn + w * c;
                    }
                } else {
                    auto turn2 = [](float4v& y, const float4v r) {
                        const float4v u = y;
                        y[0] = u[0] * r[0] - u[1] * r[1], y[1] = u[0] * r[1] + u[1] * r[0];
                        y[2] = u[2] * r[2] - u[3] * r[3], y[3] = u[2] * r[3] + u[3] * r[2];
                    };
                    turn2(a, cs[0]);
                    turn2(b, cs[1]);
                }
            }
        } else {
            *reinterpret_cast<float4v*>(&xch[wave][sub][ea]) = a;
            *reinterpret_cast<float4v*>(&xch[wave][sub][eb]) = b;
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = (i < 4 ? ea : eb) + (i & 3);
                const bool second = p.neox ? e >= half : (e & 1) != 0;
                const int j = e >= p.rot ? 0 : !p.neox ? e >> 1 : second ? e - half : e;
                const float own = i < 4 ? a[i & 3] : b[i & 3];
                const float z = xch[wave][sub][!p.neox ? e ^ 1 : second ? j : j + half], c = turn[wave][2 * j], sn = turn[wave][2 * j + 1];
                const float r = second ? z * sn + own * c : own * c - z * sn;
                const float y = e < p.rot && hv < 0 ? r : own;
                if (i < 4) a[i & 3] = y;
                else b[i & 3] = y;
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        }
        if (Q8 && hk >= 0) continue;
        if (h >= n_slot) break;
        if (!HALF && hk < 0) {
            float* dst = static_cast<float*>(p.q_out) + (size_t)t * p.tok_o + (size_t)h * HD;
            *reinterpret_cast<float4v*>(dst + ea) = a;
            *reinterpret_cast<float4v*>(dst + eb) = b;
        } else {
            uint16_t* dst = hk < 0   ? static_cast<uint16_t*>(p.q_out) + (size_t)t * p.tok_o + (size_t)h * HD
                            : hv < 0 ? p.k_pages + base + (int64_t)hk * p.head_stride
                                     : p.v_pages + base + (int64_t)hv * p.head_stride;
            *reinterpret_cast<half4*>(dst + ea) = to_half(a);
            *reinterpret_cast<half4*>(dst + eb) = to_half(b);
        }
    }
}

// Head groups a wave of a large step (4000 tokens of 32 + 4 heads of 128: one
// group 30.1 us, two 27.0, three 28.1, five 29.0; 1000 tokens 11.2, 9.6, 9.5,
// 9.8; the step's bytes at a copy's rate: 24.1).
constexpr int kQkvGroups = 2;

}  // namespace

hipError_t launch_paged_qkv(const PagedQkvParams& p, hipStream_t st) {
    const int hpw = 64 / (p.hd / 8), n_slot = p.n_head + 2 * p.n_kv;
    const int groups = (n_slot + hpw - 1) / hpw;
    // one group a wave while a step waits for its one round trip (500 tokens:
    // one and two alike, 6.7 us), two once its bytes bound it
    const int it = (long long)groups * p.n_tokens <= 5120 ? 1 : kQkvGroups;
    const int tok_waves = (groups + it - 1) / it;
    const bool ex = p.rot % 8 == 0;
    ProfScope ps(kProfPagedQkv, st);
    const dim3 grid((unsigned)(((int64_t)p.n_tokens * tok_waves + 3) / 4));
    auto go = [&](auto hd, auto i, auto half, auto e) {
        auto kernel = p.q8 ? paged_qkv_kernel<decltype(hd)::value, decltype(i)::value, decltype(half)::value, decltype(e)::value, true>
                           : paged_qkv_kernel<decltype(hd)::value, decltype(i)::value, decltype(half)::value, decltype(e)::value, false>;
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p, tok_waves);
        return hipGetLastError();
    };
    auto c = [&](auto hd, auto i, auto half) {
        return ex ? go(hd, i, half, std::true_type{}) : go(hd, i, half, std::false_type{});
    };
    auto b = [&](auto hd, auto i) { return p.half ? c(hd, i, std::true_type{}) : c(hd, i, std::false_type{}); };
    auto a = [&](auto hd) {
        return it == 1 ? b(hd, std::integral_constant<int, 1>{}) : b(hd, std::integral_constant<int, kQkvGroups>{});
    };
    switch (p.hd) {
        case 64: return a(std::integral_constant<int, 64>{});
        case 128: return a(std::integral_constant<int, 128>{});
        case 256: return a(std::integral_constant<int, 256>{});
        default: return hipErrorNotSupported;
    }
}

}  // namespace pelica

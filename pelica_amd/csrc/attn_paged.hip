// Attention of every request's new tokens over a paged f16 cache, gfx950:
// single tokens, drafts and prompt chunks in one launch, from the work list of
// attn_pages.hip.
//
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x_j = log2(e) s_j,
//   s_j = scale q.k_j, or cap tanh(scale q.k_j / cap), minus slope |pos - j|
//
// over the keys j a token sees, one pass with running max m and sum; a sink
// starts them at (sink, 1).  Query rows are (token, head) pairs of one kv
// head's group, so a key row in LDS serves the whole group.
//
// A workgroup (four waves) takes one piece of the work list for one kv head:
// narrow (an item of at most 32 rows): the waves take 32-key chunks in turn,
// each with K and V buffers of its own, no barrier until their states are
// merged through LDS; wide: the waves hold RT tiles of 32 rows each and walk
// 64-key tiles together, double-buffered, one barrier a tile.
//
// v_mfma_f32_32x32x16_f16, S^T = K Q^T (K from LDS as A, the queries in
// registers as B: a lane holds 16 scores of one row), O^T += V^T P^T (V by
// transposing LDS reads, P straight from the score registers).  f32 queries:
// q and p as f16 hi + lo parts, two products each, so that the output keeps
// f32's precision (the cache's f16 rows are exact).
//
// Cache rows go HBM -> LDS by buffer loads, one resource per group of 8 (head
// dim 64) or 4 rows: they lie in one page, whose base is scalar arithmetic on
// its table entry, in 64 bits.  The resource ends with the rows the item may
// see: what lies behind is not touched and reads as zeros.
#include <algorithm>
#include <type_traits>

#include "attn_paged.hpp"
#include "attn_prof.hpp"

namespace pelica {

namespace {

typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kNW = 4;  // waves of a workgroup
constexpr int kBufFlags = 0x00020000;  // 32-bit raw buffer

__device__ __forceinline__ float16v mfma32(const half8& a, const half8& b, const float16v& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float half_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// LDS byte of 16-byte piece p of key row k of a K tile (XOR-swizzled: 32 rows'
// same piece spreads over the banks), and of a V tile (the transposing reads of
// 4 rows' 16 dims do).
template <int HD>
__device__ __forceinline__ int k_slot(int k, int p) {
    return k * (HD * 2) + ((p ^ (k & 7)) << 4);
}
template <int HD>
__device__ __forceinline__ int v_slot(int k, int p) {
    return k * (HD * 2) + ((p ^ ((k & 3) << 1)) << 4);
}

// s_waitcnt vmcnt(N), other counters untouched
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "vmcnt is 6 bits");
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
    __asm__ volatile("" ::: "memory");
}
// this wave's LDS reads are done, and no access moves across
__device__ __forceinline__ void lds_done() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __asm__ volatile("" ::: "memory");
}

// a table entry as a scalar load
__device__ __forceinline__ int table_entry(const int32_t* t, size_t i) {
    typedef const __attribute__((address_space(4))) int32_t* cptr;
    return *(cptr)(reinterpret_cast<uintptr_t>(t + i));
}

template <int HD, int RT, int KG>
struct PagedShape {
    static constexpr int KS = HD / 16, DT = HD / 32, PPR = HD / 8;
    static constexpr int NWG = kNW / KG;                 // waves of a key group
    static constexpr int TK = KG == 1 ? 64 : 32;         // keys a tile
    static constexpr int CPT = TK / 32;
    static constexpr int NB = KG == 1 ? 2 : HD == 64 ? 2 : 1;  // buffers of K (and of V) a group
    static constexpr int TILE = TK * HD * 2;
    static constexpr int RPI = 64 / PPR;                 // rows of a load instruction
    static constexpr int WI = TK / RPI / NWG;            // its instructions a wave and tile
    static constexpr int STREAM = KG * 2 * NB * TILE;
    static constexpr int MERGE = KG > 1 ? kNW * DT * RT * 64 * 64 + kNW * RT * 64 * 8 : 0;
    static constexpr int LDS = STREAM > MERGE ? STREAM : MERGE;
};

template <int HD, int RT, int KG, bool F32, bool SC>
__device__ __forceinline__ void paged_body(const PagedParams& p, const PlanPiece& z, int kvh, char* lds) {
    using S = PagedShape<HD, RT, KG>;
    constexpr int KS = S::KS, DT = S::DT, PPR = S::PPR, NWG = S::NWG, CPT = S::CPT, NB = S::NB;
    constexpr int TILE = S::TILE, RPI = S::RPI, WI = S::WI;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int h2 = lane >> 5, c32 = lane & 31;
    const int kg = wave / NWG, wr = wave % NWG;

    // rows: the queries as the B operand (column c32 of each 32-row tile)
    half8 qh[RT][KS], ql[F32 ? RT : 1][F32 ? KS : 1];
    int posr[RT], lor[RT];
    bool valid[RT];
    float slope[RT];
    constexpr int QES = F32 ? 4 : 2;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = z.r0 + (wr * RT + rt) * 32 + c32;
        valid[rt] = r < z.R && r - z.r0 < (KG > 1 ? kNarrowRows : kNW * RT * 32);
        const int rc = min(r, z.R - 1), t = rc / p.hpk, h = kvh * p.hpk + rc % p.hpk;
        const char* src = static_cast<const char*>(p.q) + ((size_t)(z.q0 + t) * p.q_tok + (size_t)h * HD + 8 * h2) * QES;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if constexpr (F32) {
                const float4v a = *reinterpret_cast<const float4v*>(src + 64 * ks);
                const float4v b = *reinterpret_cast<const float4v*>(src + 64 * ks + 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    _Float16 hi, lo;
                    split_f16(a[i], hi, lo);
                    qh[rt][ks][i] = hi, ql[rt][ks][i] = lo;
                    split_f16(b[i], hi, lo);
                    qh[rt][ks][4 + i] = hi, ql[rt][ks][4 + i] = lo;
                }
            } else {
                qh[rt][ks] = load16(src + 32 * ks);
            }
        }
        const int pos = z.pos0 + t;
        posr[rt] = valid[rt] ? pos : -1;
        lor[rt] = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
        slope[rt] = SC && p.alibi ? p.alibi[h] * kLog2e : 0.f;
    }
    // every row sees the keys [lo_all, hi_all] and those below z.pe
    const int r_last = min(z.R, z.r0 + (KG > 1 ? kNarrowRows : kNW * RT * 32)) - 1;
    const int hi_all = z.pos0 + z.r0 / p.hpk, pos_last = z.pos0 + r_last / p.hpk;
    const int lo_all = p.window > 0 && pos_last >= p.window ? pos_last - p.window + 1 : 0;

    float m[RT], l[RT];
    float16v o[DT][RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.f;
        if (p.sinks && z.slot < 0 && kg == 0) {  // (a split item's sink joins with its pieces)
            const int rc = min(z.r0 + (wr * RT + rt) * 32 + c32, z.R - 1);
            m[rt] = p.sinks[kvh * p.hpk + rc % p.hpk] * kLog2e;
            l[rt] = h2 == 0 ? 1.f : 0.f;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt][rt] = float16v{};
    }

    // Cache rows: instruction i of this wave fills rows RPI (NWG i + wr) .. of a
    // tile.  lane constants: the row within the group and the piece that the
    // swizzled layout puts in the lane's slot (RPI divides 8, so the slot's
    // key & 7 is the row's within 8)
    char* const kbuf = lds + kg * 2 * NB * TILE;
    char* const vbuf = kbuf + NB * TILE;
    const int lrow = lane / PPR, phys = lane % PPR;
    const char* const kbase = reinterpret_cast<const char*>(p.k) + (size_t)kvh * p.head_b;
    const char* const vbase = reinterpret_cast<const char*>(p.v) + (size_t)kvh * p.head_b;
    const size_t trow = (size_t)z.seq * p.max_pages;
    bool bad = false;
    // one group: K or V rows of tile keys kt .. of chunk-relative row r0g
    struct Group {
        int64_t off;     // bytes from the head's base to the first row wanted
        uint32_t skip;   // bytes ahead of it within the group
        uint32_t nrec;   // bytes of rows wanted
    };
    auto group = [&](int c, int row) {  // chunk c, first row within the chunk
        Group g;
        const int key = chunk_key(c, z.n_pre, z.lo_base) + row;
        int first, count;
        group_rows(key, RPI, z.lo, z.kend, z.pe, first, count);
        if (c >= z.ce) count = 0;
        g.skip = (uint32_t)first * p.row_b;
        g.nrec = (uint32_t)count * p.row_b;
        g.off = 0;
        if (count > 0) {
            const int id = table_entry(p.table, trow + (key >> p.page_log2));
            bad |= (unsigned)id >= (unsigned)p.n_pages;
            const int page = min(max(id, 0), p.n_pages - 1);
            g.off = (int64_t)page * p.page_b + (int64_t)((key & ((1 << p.page_log2) - 1)) + first) * p.row_b;
        }
        return g;
    };
    auto load = [&](const char* base, const Group& g, char* dst, int i, bool is_v) {
        const int row = RPI * (NWG * i + wr) + lrow;  // within the tile
        const int piece = is_v ? phys ^ ((row & 3) << 1) : phys ^ (row & 7);
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc((void*)(base + g.off), (short)0, (int)g.nrec, kBufFlags);
        lds_dma16_untracked(rs, (uint32_t)lrow * p.row_b + 16u * piece - g.skip, dst + 1024 * (NWG * i + wr));
    };
    // tile t of this key group: its first chunk
    auto tile_chunk = [&](int t) { return KG > 1 ? z.cb + kg + KG * t : z.cb + CPT * t; };
    auto load_tile = [&](int t, bool is_v) {
        char* const dst = (is_v ? vbuf : kbuf) + (t % NB) * TILE;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int row = RPI * (NWG * i + wr);
            load(is_v ? vbase : kbase, group(tile_chunk(t) + row / 32, row % 32), dst, i, is_v);
        }
    };
    const int n = z.ce - z.cb;
    const int n_tiles = KG > 1 ? (n - kg + KG - 1) / KG : (n + CPT - 1) / CPT;  // (kg <= n + KG - 1: >= 0)

    // chunk c's scores: S^T, then in the log2 domain, masked
    auto scores = [&](const char* kt, int sub, int c, float16v (&s)[RT]) {
        const int krow = 32 * sub + c32;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt] = float16v{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const half8 ka = *reinterpret_cast<const half8*>(kt + k_slot<HD>(krow, 2 * ks + h2));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                s[rt] = mfma32(ka, qh[rt][ks], s[rt]);
                if constexpr (F32) s[rt] = mfma32(ka, ql[rt][ks], s[rt]);
            }
        }
    };
    auto transform = [&](int c, float16v (&s)[RT]) {
        const int kb = chunk_key(c, z.n_pre, z.lo_base);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (SC && p.cap > 0.f) {
                // tanh(y) = 1 - 2 / (1 + e^(2 y)), saturating at both ends
                const float c2 = p.cap * kLog2e, f = 2.f * p.qscale / p.cap;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[rt][i] = c2 - 2.f * c2 * __builtin_amdgcn_rcpf(1.f + fast_exp2(s[rt][i] * f));
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[rt][i] *= p.qscale;
            }
            if (SC && p.alibi) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = kb + 8 * (i / 4) + 4 * h2 + i % 4;
                    s[rt][i] -= slope[rt] * fabsf((float)(posr[rt] - key));
                }
            }
        }
        const bool all = kb + 31 < z.pe || (kb >= lo_all && kb + 31 <= hi_all);
        if (!all) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = kb + 8 * (i / 4) + 4 * h2 + i % 4;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if (!(key < z.pe || (key >= lor[rt] && key <= posr[rt]))) s[rt][i] = -INFINITY;
            }
        }
    };
    // running softmax over one chunk; P as the B operand of the PV product
    auto softmax = [&](float16v (&s)[RT], half8 (&ph)[2][RT], half8 (&pl)[2][RT]) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float x = s[rt][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) x = fmaxf(x, s[rt][i]);
            const float mn = fmaxf(m[rt], half_max(x));
            if (__builtin_amdgcn_ballot_w64(mn > m[rt])) {
                const float cf = mn > m[rt] ? fast_exp2(m[rt] - mn) : 1.f;  // (0 while m was -inf)
                l[rt] *= cf;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt][rt] *= cf;
                m[rt] = mn;
            }
            const float ms = m[rt] == -INFINITY ? 0.f : m[rt];
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = fast_exp2(s[rt][i] - ms);
                if constexpr (F32) {
                    _Float16 hi, lo;
                    split_f16(e, hi, lo);
                    ph[i / 8][rt][i % 8] = hi;
                    pl[i / 8][rt][i % 8] = lo;
                    sum += e;
                } else {
                    ph[i / 8][rt][i % 8] = (_Float16)e;
                    sum += (float)ph[i / 8][rt][i % 8];
                }
            }
            l[rt] += sum;
        }
    };
    auto pv = [&](const char* vt, int sub, const half8 (&ph)[2][RT], const half8 (&pl)[2][RT]) {
        const int G = lane >> 4, r4 = (lane & 15) >> 2, q4 = lane & 3;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                // lanes of 16-lane group G: keys 16 w + 4 h2 + r4 (+ 8), dims 32 dt + 16 (G & 1) + 4 q4
                const int key = 32 * sub + 16 * w + 4 * h2 + r4, dim = 32 * dt + 16 * (G & 1) + 4 * q4;
                const _Float16* a0 = reinterpret_cast<const _Float16*>(vt + v_slot<HD>(key, dim >> 3) + ((dim & 7) << 1));
                const _Float16* a1 = reinterpret_cast<const _Float16*>(vt + v_slot<HD>(key + 8, dim >> 3) + ((dim & 7) << 1));
                const half8 va = cat8(lds_read_tr(a0), lds_read_tr(a1));
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    o[dt][rt] = mfma32(va, ph[w][rt], o[dt][rt]);
                    if constexpr (F32) o[dt][rt] = mfma32(va, pl[w][rt], o[dt][rt]);
                }
            }
        }
    };

    // A chunk that some rows see in part may hold infinities or NaN in rows of
    // V that they do not see, and 0 times those is NaN.  Where it does, they
    // are taken out of the tile here and added after the last chunk to the rows
    // that see them.
    auto partly_seen = [&](int c) {
        const int kb = chunk_key(c, z.n_pre, z.lo_base);
        return pos_last > hi_all && !(kb + 31 < z.pe || (kb >= lo_all && kb + 31 <= hi_all));
    };
    auto finite = [](_Float16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7C00) != 0x7C00; };
    bool special = false;
    auto clean = [&](char* vt, int sub) {
        typedef _Float16 half2 __attribute__((ext_vector_type(2)));
        char* const at = vt + 64 * HD * sub + 16 * lane;
        float a = 0.f;  // (any infinity or NaN times 0)
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            const half8 x = *reinterpret_cast<const half8*>(at + 1024 * i);
#pragma unroll
            for (int k = 0; k < 8; k += 2) a = __builtin_amdgcn_fdot2(half2{x[k], x[k + 1]}, half2{0, 0}, a, false);
        }
        if (__builtin_amdgcn_ballot_w64(a != 0.f) == 0) return;
        special = true;
        // (the waves of a wide workgroup may do so at once: each writes zeros
        // over what it finds before it reads the tile)
#pragma unroll 1
        for (int i = 0; i < HD / 16; ++i) {
            half8 x = *reinterpret_cast<const half8*>(at + 1024 * i);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = finite(x[k]) ? x[k] : (_Float16)0;
            *reinterpret_cast<half8*>(at + 1024 * i) = x;
        }
        lds_done();
    };
    auto add_special = [&](int c) {
        const int kb = chunk_key(c, z.n_pre, z.lo_base);
#pragma unroll 1
        for (int key = kb; key < kb + 32; ++key) {
            int first, count;
            group_rows(key, 1, z.lo, z.kend, z.pe, first, count);
            if (count == 0) continue;
            const int id = min(max(table_entry(p.table, trow + (key >> p.page_log2)), 0), p.n_pages - 1);
            const char* const src = vbase + (int64_t)id * p.page_b + (int64_t)(key & ((1 << p.page_log2) - 1)) * p.row_b;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    const half4 x = *reinterpret_cast<const half4*>(src + 2 * (32 * dt + 8 * i4 + 4 * h2));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const bool sees = key < z.pe || (key >= lor[rt] && key <= posr[rt]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (sees && !finite(x[i])) o[dt][rt][4 * i4 + i] += (float)x[i];
                    }
                }
        }
    };

    half8 ph[2][RT], pl[2][RT];
    float16v s[RT];
    if constexpr (KG > 1) {
        // requests in order K0 V0 (K1 V1): ahead of a tile's wait stand the
        // 2 NB - 1 tiles after it (past the last one: empty requests)
        constexpr int AHEAD = WI * (2 * NB - 1);
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            load_tile(t, false);
            load_tile(t, true);
        }
        for (int t = 0; t < n_tiles; ++t) {
            const int c = tile_chunk(t);
            wait_loads<AHEAD>();
            scores(kbuf + (t % NB) * TILE, 0, c, s);
            lds_done();
            load_tile(t + NB, false);
            transform(c, s);
            softmax(s, ph, pl);
            wait_loads<AHEAD>();
            if (partly_seen(c)) clean(vbuf + (t % NB) * TILE, 0);
            pv(vbuf + (t % NB) * TILE, 0, ph, pl);
            lds_done();
            load_tile(t + NB, true);
        }
        wait_loads<0>();
    } else {
        load_tile(0, false);
        load_tile(0, true);
        for (int t = 0; t < n_tiles; ++t) {
            wait_loads<0>();
            __syncthreads();  // tile t is there, and no wave reads tile t - 1
            if (t + 1 < n_tiles) {
                load_tile(t + 1, false);
                load_tile(t + 1, true);
            }
#pragma unroll
            for (int sub = 0; sub < CPT; ++sub) {
                const int c = tile_chunk(t) + sub;
                if (c >= z.ce) break;
                scores(kbuf + (t % NB) * TILE, sub, c, s);
                transform(c, s);
                softmax(s, ph, pl);
                if (partly_seen(c)) clean(vbuf + (t % NB) * TILE, sub);
                pv(vbuf + (t % NB) * TILE, sub, ph, pl);
            }
        }
    }
    const bool any_bad = __syncthreads_or(bad);  // (and every wave is done with the tiles)
    if (KG == 1) special = __syncthreads_or(special);
    if (special)
#pragma unroll 1
        for (int t = 0; t < n_tiles; ++t)
#pragma unroll 1
            for (int c = tile_chunk(t); c < min(tile_chunk(t) + CPT, z.ce); ++c)
                if (partly_seen(c)) add_special(c);

    // a row's final state: (M, L), and 4 consecutive dims at 32 dt + 8 i4 + 4 h2
    const size_t part = (size_t)(z.slot * p.n_kv + kvh) * p.rows;
    auto store_ml = [&](int rl, float M, float L) {
        reinterpret_cast<float2*>(p.ws_ml)[part + rl] = make_float2(M, any_bad ? NAN : L);
    };
    auto store4 = [&](int rl, int dt, int i4, float4v x, float inv) {
        const int d = 32 * dt + 8 * i4 + 4 * h2;
        if (z.slot >= 0) {
            *reinterpret_cast<float4v*>(p.ws_o + (part + rl) * HD + d) = x;
            return;
        }
        if (any_bad) inv = NAN;
        x *= inv;
        const int r = z.r0 + rl;
        const size_t at = (size_t)(z.q0 + r / p.hpk) * p.o_tok + (size_t)(kvh * p.hpk + r % p.hpk) * HD + d;
        if constexpr (F32) {
            *reinterpret_cast<float4v*>(static_cast<float*>(p.out) + at) = x;
        } else {
            *reinterpret_cast<half4*>(static_cast<uint16_t*>(p.out) + at) =
                half4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
        }
    };
    if constexpr (KG > 1) {
        // the waves' states through LDS, merged in wave order: wave g takes
        // the output tiles g, g + KG, ...
        static_assert(RT == 1, "narrow items are one row tile");
        float4v* const so = reinterpret_cast<float4v*>(lds);
        float2* const sml = reinterpret_cast<float2*>(lds + kNW * DT * 64 * 64);
        sml[wave * 64 + lane] = make_float2(m[0], half_sum(l[0]));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4)
                so[((wave * DT + dt) * 4 + i4) * 64 + lane] =
                    float4v{o[dt][0][4 * i4], o[dt][0][4 * i4 + 1], o[dt][0][4 * i4 + 2], o[dt][0][4 * i4 + 3]};
        __syncthreads();
        if (!valid[0]) return;
        float2 ml[KG];
        float M = -INFINITY;
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            ml[g] = sml[g * 64 + lane];
            M = fmaxf(M, ml[g].x);
        }
        const float ms = M == -INFINITY ? 0.f : M;
        float L = 0.f, w[KG];
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            w[g] = fast_exp2(ml[g].x - ms);  // 0 where the wave saw no key
            L += ml[g].y * w[g];
        }
        const float inv = 1.f / L;
        if (z.slot >= 0 && wave == 0 && h2 == 0) store_ml(c32, M, L);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            if (dt % KG != kg) continue;
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                float4v x = so[(dt * 4 + i4) * 64 + lane] * w[0];
#pragma unroll
                for (int g = 1; g < KG; ++g) x += so[((g * DT + dt) * 4 + i4) * 64 + lane] * w[g];
                store4(c32, dt, i4, x, inv);
            }
        }
    } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float L = half_sum(l[rt]);
            if (!valid[rt]) continue;
            const int rl = (wr * RT + rt) * 32 + c32;
            if (z.slot >= 0 && h2 == 0) store_ml(rl, m[rt], L);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4)
                    store4(rl, dt, i4,
                           float4v{o[dt][rt][4 * i4], o[dt][rt][4 * i4 + 1], o[dt][rt][4 * i4 + 2], o[dt][rt][4 * i4 + 3]},
                           1.f / L);
        }
    }
}

template <int HD, bool F32, bool SC, bool WIDE>
__global__ __launch_bounds__(64 * kNW) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_kernel(PagedParams p) {
    constexpr int RT = HD == 64 ? 2 : 1;
    constexpr int LN = PagedShape<HD, 1, kNW>::LDS, LW = WIDE ? PagedShape<HD, RT, 1>::LDS : 0;
    __shared__ __attribute__((aligned(16))) char lds[LN > LW ? LN : LW];
    const int id = blockIdx.x / p.n_kv, kvh = blockIdx.x % p.n_kv;
    if (p.head->sig != p.sig || id >= p.head->n_pieces) return;
    const PlanPiece z = p.pieces[id];
    if (WIDE && z.R > kNarrowRows) paged_body<HD, RT, 1, F32, SC>(p, z, kvh, lds);
    else paged_body<HD, 1, kNW, F32, SC>(p, z, kvh, lds);
}

// The pieces of a split item, joined in key order with the sink: per row
// (M, L, O) of each slot, weights 2^(M_i - M).  WPR waves a row: HD / 4 lanes
// hold 4 dims each, the other lane groups and waves take slots in turn and
// meet through lane exchanges and LDS in a fixed order.
template <int HD, bool F32, int WPR>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p) {
    constexpr int LPR = HD / 4, GPW = 64 / LPR, PH = GPW * WPR, U = 8;
    __shared__ float st[WPR > 1 ? WPR : 1][64][6];
    const int j = blockIdx.x / p.n_kv, kvh = blockIdx.x % p.n_kv;
    if (p.head->sig != p.sig || j >= p.head->n_joins) return;
    const PlanJoin z = p.joins[j];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = 4 * (lane % LPR);
    const int ph = (WPR > 1 ? wave * GPW : 0) + lane / LPR;
    const int rows = min(z.R - z.r0, p.rows);
    for (int r = WPR > 1 ? (int)blockIdx.y : (int)blockIdx.y * (4 / WPR) + wave; r < rows;
         r += (WPR > 1 ? 1 : 4) * (int)gridDim.y) {
        float m = -INFINITY, l = 0.f;
        float4v o = {};
        for (int s0 = ph; s0 < z.n_slots; s0 += PH * U) {
            float2 ml[U];
            float4v v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int sl = s0 + PH * u;
                const size_t at = ((size_t)(z.slot0 + min(sl, z.n_slots - 1)) * p.n_kv + kvh) * p.rows + r;
                ml[u] = reinterpret_cast<const float2*>(p.ws_ml)[at];
                v[u] = *reinterpret_cast<const float4v*>(p.ws_o + at * HD + d);
                if (sl >= z.n_slots) ml[u] = make_float2(-INFINITY, 0.f);
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
        // the lane groups of a wave, then the waves
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
        const int rr = z.r0 + r, h = kvh * p.hpk + rr % p.hpk;
        if (p.sinks) {
            const float sk = p.sinks[h] * kLog2e, M = fmaxf(m, sk), f = fast_exp2(m - M);
            l = l * f + fast_exp2(sk - M);
            o *= f;
        }
        if (lane >= LPR) continue;
        o *= 1.f / l;
        const size_t at = (size_t)(z.q0 + rr / p.hpk) * p.o_tok + (size_t)h * HD + d;
        if constexpr (F32) {
            *reinterpret_cast<float4v*>(static_cast<float*>(p.out) + at) = o;
        } else {
            *reinterpret_cast<half4*>(static_cast<uint16_t*>(p.out) + at) =
                half4{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
        }
    }
}

template <typename F>
hipError_t with_shape(const PagedParams& p, F f) {
    auto hd = [&](auto h) {
        return p.f32 ? f(h, std::true_type{}) : f(h, std::false_type{});
    };
    return p.hd == 64 ? hd(std::integral_constant<int, 64>{}) : hd(std::integral_constant<int, 128>{});
}

}  // namespace

hipError_t launch_paged(const PagedParams& p, hipStream_t st) {
    ProfScope ps(kProfPaged, st);
    return with_shape(p, [&](auto hd, auto f32) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool F32 = decltype(f32)::value;
        const dim3 grid((unsigned)p.max_pieces * p.n_kv);
        const bool sc = p.cap > 0.f || p.alibi;
        if (p.wide) {
            if (sc) hipLaunchKernelGGL((paged_kernel<HD, F32, true, true>), grid, dim3(64 * kNW), 0, st, p);
            else hipLaunchKernelGGL((paged_kernel<HD, F32, false, true>), grid, dim3(64 * kNW), 0, st, p);
        } else {
            if (sc) hipLaunchKernelGGL((paged_kernel<HD, F32, true, false>), grid, dim3(64 * kNW), 0, st, p);
            else hipLaunchKernelGGL((paged_kernel<HD, F32, false, false>), grid, dim3(64 * kNW), 0, st, p);
        }
        return hipGetLastError();
    });
}

hipError_t launch_paged_join(const PagedParams& p, hipStream_t st) {
    ProfScope ps(kProfPagedJoin, st);
    return with_shape(p, [&](auto hd, auto f32) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool F32 = decltype(f32)::value;
        const unsigned x = (unsigned)p.max_joins * p.n_kv;
        if (p.wide) hipLaunchKernelGGL((paged_join_kernel<HD, F32, 1>), dim3(x, 8), dim3(256), 0, st, p);
        else hipLaunchKernelGGL((paged_join_kernel<HD, F32, 4>), dim3(x, std::min(p.rows, 32)), dim3(256), 0, st, p);
        return hipGetLastError();
    });
}

}  // namespace pelica

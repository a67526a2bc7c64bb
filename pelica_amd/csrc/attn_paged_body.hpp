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
// A workgroup (four waves, two a CU) takes one piece of the work list for one kv
// head: narrow (an item of at most 32 rows: tokens, drafts), whose waves take
// 32-key chunks in turn and are merged at the end, or wide (a chunk's 256 rows
// of head dim 64, 128 of 128), whose waves share the keys.  Neighbouring
// workgroups are the kv heads of one piece: with 8 kv heads an XCD's L2 holds
// one head's keys for all the pieces that read them.
//
// S^T = K Q^T (K from LDS as A, the queries in registers as B: a lane's scores
// are all of one row), O^T += V^T P^T (V by transposing LDS reads, P straight
// from the score registers).  f32 queries: q and p as f16 hi + lo parts, two
// products each, so that the output keeps f32's precision (2^-22; the cache's
// f16 rows are exact).  f16 queries: p is rounded to f16 (2^-11) in the sum as in
// the product; the output's rounding is as large.
//
// Cache rows go HBM -> LDS by buffer loads, one resource per run of 8 rows: they
// lie in one page, whose base is scalar arithmetic on its table entry, in 64
// bits.  The resource ends with the rows the item may see: what lies behind is
// not touched and reads as zeros.
//
// Measured, medians of warm traced launches (floors: bytes at a copy's 5.13 TB/s,
// or operations at a large f16 product's 1.17 PFLOP/s):
//   32 tokens over 512 - 16384 keys, 32 / 4 heads of 128   115 us (118)
//   16 tokens with a bias over 300 - 6000, 16 / 16 of 128   95 us (99)
//   one token over 32768, 64 / 8 of 64                      16 - 19 us by card + join 3.9 (13)
//   64 tokens on windows of 128, 64 / 8 of 64              8.6 - 8.9 us (3.7: latency)
//   512 tokens over 30512, 64 / 8 of 64                    266 - 300 us by card + join 7.9 (217)
//   4001 tokens, 32 / 4 of 128                             156 us + join 4.6 (112)
//   3 chunks of 700 and 28 drafts, 64 / 8 of 64            205 us + join 12.6 (111)
//   2000 tokens, capped, 600 of prefix, 32 / 4 of 128       69 us + join 6.8 (30.5)
#pragma once
#include <algorithm>
#include <type_traits>
#include <utility>

#include "attn_paged.hpp"
#include "attn_prof.hpp"
#include "attn_q8.hpp"

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

// LDS byte of 16-byte piece p of key row k of a K tile: pieces XOR-swizzled so
// that 16 consecutive rows' same piece, which 16 lanes read at once, lie in 64
// banks (a row of 128 bytes is half of them).
template <int HD>
__device__ __forceinline__ constexpr int k_swizzle(int k) {
    return HD == 64 ? (k >> 1) & 7 : k & 15;
}
template <int HD>
__device__ __forceinline__ int k_slot(int k, int p) {
    return k * (HD * 2) + ((p ^ k_swizzle<HD>(k)) << 4);
}
// ... and of a V tile, whose transposing reads take 4 rows' 16 dims a 16-lane
// group, 32 lanes at once: two groups rows 4 apart (narrow) or dims 16 apart
// (wide).
template <int HD>
__device__ __forceinline__ constexpr int v_swizzle(int k) {
    return HD == 64 ? ((k & 3) ^ ((k >> 2) & 1)) << 1 : ((k & 3) << 2) | ((k >> 1) & 2);
}
template <int HD>
__device__ __forceinline__ int v_slot(int k, int p) {
    return k * (HD * 2) + ((p ^ v_swizzle<HD>(k)) << 4);
}

// split_f16 of two values: two packed conversions and, between them, a mixed
// multiply-add each (x - hi is exact in f32)
__device__ __forceinline__ void split_pair(float x, float y, half2& hi, half2& lo) {
    float minus = -1.f;
    __asm__("" : "+s"(minus));  // (known, it would be a conversion and a subtraction)
    hi = half2{(_Float16)x, (_Float16)y};
    lo = half2{(_Float16)__builtin_fmaf((float)hi[0], minus, x), (_Float16)__builtin_fmaf((float)hi[1], minus, y)};
}

// f(0) .. f(N - 1), the indexes as types
template <typename F, int... I>
__device__ __forceinline__ void unrolled_(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
    unrolled_(f, std::make_integer_sequence<int, N>{});
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

__device__ __forceinline__ uint32_t lds_byte(const char* p) {
    return (uint32_t)(size_t)(__attribute__((address_space(3))) const char*)p;
}

// a table entry as a scalar load
__device__ __forceinline__ int table_entry(const int32_t* t, size_t i) {
    typedef const __attribute__((address_space(4))) int32_t* cptr;
    return *(cptr)(reinterpret_cast<uintptr_t>(t + i));
}

// V^T of 16 keys from row `key` of a tile, dims 32 dt .. + 31, as the A operand
// of the PV product: lanes of 16-lane group G read keys 4 h2 + r4 (+ 8) at dims
// 16 (G & 1) + 4 q4, and the read transposes
template <int HD>
__device__ __forceinline__ half8 v_operand(const char* vt, int key, int dt, int lane) {
    const int G = lane >> 4, r4 = (lane & 15) >> 2, q4 = lane & 3;
    const int k = key + 4 * (lane >> 5) + r4, dim = 32 * dt + 16 * (G & 1) + 4 * q4;
    const _Float16* a0 = reinterpret_cast<const _Float16*>(vt + v_slot<HD>(k, dim >> 3) + ((dim & 7) << 1));
    const _Float16* a1 = reinterpret_cast<const _Float16*>(vt + v_slot<HD>(k + 8, dim >> 3) + ((dim & 7) << 1));
    return cat8(lds_read_tr(a0), lds_read_tr(a1));
}

// A chunk that some rows see in part may hold infinities or NaN in rows of V
// that they do not see, and 0 times those is NaN.  Where it does, they are
// taken out of the tile (clean_chunk: whether any were there) and added after
// the last chunk to the rows that see them (add_special).  The waves of a wide
// workgroup may clean a chunk at once: each has written zeros over what it
// found before it reads the chunk.  Such rows are the keys of the item's later
// tokens, and keys between a prefix and a window that share a run with both.
template <int RUN = 8>
__device__ __forceinline__ bool may_hide(const PlanPiece& z, int hi_all, int pos_last) {
    return pos_last > hi_all || gap_in_run<RUN>(z.lo, z.pe);
}
__device__ __forceinline__ bool is_finite(_Float16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7C00) != 0x7C00; }

// Whether a row sees a key: its own span of keys from lo on, or the prefix
__device__ __forceinline__ bool sees(int key, int pe, int lo, unsigned span) {
    return (key < pe) | ((unsigned)(key - lo) <= span);
}

template <int HD>
__device__ __forceinline__ bool clean_chunk(char* vt, int lane) {
    char* const at = vt + 16 * lane;
    float a = 0.f;  // (any infinity or NaN times 0)
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
        const half8 x = *reinterpret_cast<const half8*>(at + 1024 * i);
#pragma unroll
        for (int k = 0; k < 8; k += 2) a = __builtin_amdgcn_fdot2(half2{x[k], x[k + 1]}, half2{0, 0}, a, false);
    }
    if (__builtin_amdgcn_ballot_w64(a != 0.f) == 0) return false;
#pragma unroll 1
    for (int i = 0; i < HD / 16; ++i) {
        half8 x = *reinterpret_cast<const half8*>(at + 1024 * i);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = is_finite(x[k]) ? x[k] : (_Float16)0;
        *reinterpret_cast<half8*>(at + 1024 * i) = x;
    }
    lds_done();
    return true;
}

// The cache rows of one kv head: a wave fills runs of 8 consecutive rows of a
// tile, which lie in one page (pages are at least 8 rows).  A run's address is
// scalar: its table entry, in 64 bits; a lane adds its row and piece, a
// constant.
template <int HD>
struct CacheRows {
    static constexpr int PPR = HD / 8, RPI = 64 / PPR, IPR = 8 / RPI;  // pieces a row; rows, instructions of a run
    const PagedParams& p;
    const PlanPiece& z;
    uint64_t k, v;            // the head's rows of page 0
    const int32_t* table;     // the request's row
    int last, bad = 0;        // last key that a row sees; a page of a wanted key is none of the pool's
    uint32_t klane[2][IPR], vlane[IPR];  // (K's by the run's parity)

    struct Run {
        uint64_t off;         // bytes to the first row wanted
        uint32_t nrec, skip;  // bytes of the rows wanted, bytes of the run ahead of them
    };

    __device__ __forceinline__ CacheRows(const PagedParams& p_, const PlanPiece& z_, int kvh, int lane) : p(p_), z(z_) {
        k = reinterpret_cast<uintptr_t>(p.k) + (uint64_t)kvh * p.head_b;
        v = reinterpret_cast<uintptr_t>(p.v) + (uint64_t)kvh * p.head_b;
        table = p.table + (size_t)z.seq * p.max_pages;
        last = imax(z.kend, z.pe) - 1;
        const int lrow = lane / PPR, phys = lane % PPR;
#pragma unroll
        for (int j = 0; j < IPR; ++j) {
            const int row = RPI * j + lrow;
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                klane[odd][j] = (uint32_t)row * p.row_b + 16u * (phys ^ k_swizzle<HD>(8 * odd + row));
                __asm__("" : "+v"(klane[odd][j]));  // (else taken apart again at each use)
            }
            vlane[j] = (uint32_t)row * p.row_b + 16u * (phys ^ v_swizzle<HD>(row));
            __asm__("" : "+v"(vlane[j]));
        }
    }
    __device__ __forceinline__ int entry(int key) const { return table_entry(table, imin(key, last) >> p.page_log2); }
    struct VRow {
        const char* at;
        __device__ __forceinline__ half4 dims(int d) const { return *reinterpret_cast<const half4*>(at + 2 * d); }
    };
    __device__ __forceinline__ VRow v_row(int key) const {
        const unsigned page = min((unsigned)entry(key), (unsigned)p.n_pages - 1u);
        return {reinterpret_cast<const char*>(v + (uint64_t)page * (uint64_t)p.page_b +
                                              (uint32_t)((key & ((1 << p.page_log2) - 1)) * p.row_b))};
    }
    // keys key .. key + 7; none are wanted unless `any`
    __device__ __forceinline__ Run run(int key, bool any, int id) {
        int first, count;
        group_rows(key, 8, z.lo, z.kend, z.pe, first, count);
        count = any ? count : 0;
        bad |= count > 0 ? (unsigned)id >= (unsigned)p.n_pages : 0;
        const unsigned page = min((unsigned)id, (unsigned)p.n_pages - 1u);
        Run r;
        r.skip = (uint32_t)first * p.row_b;
        r.nrec = (uint32_t)count * p.row_b;
        r.off = (uint64_t)page * (uint64_t)p.page_b + (uint32_t)((key & ((1 << p.page_log2) - 1)) * p.row_b) + r.skip;
        return r;
    }
    // instruction j of a run (an odd or even one of its tile) into 1 KB of LDS
    // at byte `to`
    template <bool V>
    __device__ __forceinline__ void load(const Run& r, int odd, int j, uint32_t to) const {
        const uint64_t base = (V ? v : k) + r.off;
        // (uniform, though not where the compiler has put them in every case)
        const u32x4 rs = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base),
                          (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32)),
                          (uint32_t)__builtin_amdgcn_readfirstlane(r.nrec), (uint32_t)kBufFlags};
        uint32_t saved;
        __asm__ volatile(
            "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
            "buffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
            : "=&s"(saved)
            : "s"(to), "v"((V ? vlane[j] : klane[odd][j]) - r.skip), "s"(rs));
    }
};

// 8-bit rows of one kv head, the same runs.  They pass through registers: a
// lane holds HD / 8 values of a row and the scale of their group, takes them
// from memory a chunk or more ahead of their use and writes them into the
// tile as f16, in CacheRows' order.  (Eight lanes a row, one load a run: whole
// lines where a head's rows lie side by side.)
// Bound by HBM over long keys, by issue where keys come from L2 (7 instructions
// take 4 values apart).  Medians of traced launches (floors: bytes at a copy's 5.04
// TB/s, or operations at a large f16 product's 1.18 PFLOP/s):
//   32 tokens over 512 - 16384 keys, 32 / 4 heads of 128   67.4 us (64)
//   64 tokens on windows of 128, 64 / 8 of 64               9.1 us (2.2: latency)
//   one token over 32768, 64 / 8 of 64                     15.2 us (7.1)
//   512 tokens over 30512, 64 / 8 of 64                     301 - 340 us by card (215)
// The wide items of f16 queries spill 34 - 60 vector registers at head dim 64: the
// same chunk capped takes 442 us (374 over f16 pages), with a distance bias 671 (512).
template <int HD>
struct Q8Rows {
    static constexpr int VB = HD / 8, WORDS = VB / 4;  // bytes, words of a lane
    static constexpr int PARTS = WORDS / 2;            // 16-byte pieces of f16 a lane makes
    const PagedParams& p;
    const PlanPiece& z;
    uint64_t k, v, ks, vs;    // the head's rows and scales of page 0
    const int32_t* table;
    int last, bad = 0;
    uint32_t dlane, slane;    // bytes from a run's first row and scale
    uint32_t kto, vto;        // bytes from a run's place in an even run's tile

    struct Run {             // 8 rows, or 16 of a page that holds them
        uint64_t off, soff;  // bytes to the run's first row and scales
        int first, count;    // the rows wanted
    };
    struct Regs {
        uint32_t w[WORDS];
        uint16_t s;
    };

    __device__ __forceinline__ Q8Rows(const PagedParams& p_, const PlanPiece& z_, int kvh, int lane) : p(p_), z(z_) {
        k = reinterpret_cast<uintptr_t>(p.k) + (uint64_t)kvh * p.head_b;
        v = reinterpret_cast<uintptr_t>(p.v) + (uint64_t)kvh * p.head_b;
        ks = reinterpret_cast<uintptr_t>(p.ks) + (uint64_t)kvh * p.shead_b;
        vs = reinterpret_cast<uintptr_t>(p.vs) + (uint64_t)kvh * p.shead_b;
        table = p.table + (size_t)z.seq * p.max_pages;
        last = imax(z.kend, z.pe) - 1;
        const int row = lane >> 3, part = lane & 7;
        dlane = (uint32_t)row * p.row_b + (uint32_t)(VB * part);
        slane = (uint32_t)row * p.srow_b + 2u * (uint32_t)(VB * part / kQ8Group);
        kto = (uint32_t)k_slot<HD>(row, PARTS * part);
        vto = (uint32_t)v_slot<HD>(row, PARTS * part);
    }
    __device__ __forceinline__ int entry(int key) const { return table_entry(table, imin(key, last) >> p.page_log2); }
    // N keys from key on; none are wanted unless `any`
    template <int N = 8>
    __device__ __forceinline__ Run run(int key, bool any, int id) {
        int first, count;
        group_rows(key, N, z.lo, z.kend, z.pe, first, count);
        count = any ? count : 0;
        bad |= count > 0 ? (unsigned)id >= (unsigned)p.n_pages : 0;
        const unsigned page = min((unsigned)id, (unsigned)p.n_pages - 1u);
        const uint32_t in = (uint32_t)(key & ((1 << p.page_log2) - 1));
        Run r;
        r.first = first;
        r.count = count;
        r.off = (uint64_t)page * (uint64_t)p.page_b + in * p.row_b;
        r.soff = (uint64_t)page * (uint64_t)p.spage_b + in * p.srow_b;
        return r;
    }
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(uint64_t base, uint32_t bytes) {
        // (uniform, though not where the compiler has put them in every case)
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32));
        return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), 0,
                                                 __builtin_amdgcn_readfirstlane(bytes), kBufFlags);
    }
    // from the first row wanted on: a lane ahead of it is past the end, too
    template <bool V>
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t data(const Run& r) const {
        return resource((V ? v : k) + r.off + (uint32_t)r.first * p.row_b, (uint32_t)r.count * p.row_b);
    }
    template <bool V>
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t scales(const Run& r) const {
        return resource((V ? vs : ks) + r.soff + (uint32_t)r.first * p.srow_b, (uint32_t)r.count * p.srow_b);
    }
    // the run's rows 8 half .. + 7
    __device__ __forceinline__ Regs load(__amdgpu_buffer_rsrc_t d, __amdgpu_buffer_rsrc_t s, const Run& r, int half) const {
        const uint32_t at = dlane + (uint32_t)(8 * half - r.first) * p.row_b, sat = slane + (uint32_t)(8 * half - r.first) * p.srow_b;
        Regs x;
        if constexpr (WORDS == 4) {
            const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(d, at, 0, 0));
            x.w[0] = w[0], x.w[1] = w[1], x.w[2] = w[2], x.w[3] = w[3];
        } else {
            const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(d, at, 0, 0));
            x.w[0] = w[0], x.w[1] = w[1];
        }
        x.s = __builtin_amdgcn_raw_buffer_load_b16(s, sat, 0, 0);
        return x;
    }
    template <bool V>
    __device__ __forceinline__ Regs fetch(const Run& r) const {
        return load(data<V>(r), scales<V>(r), r, 0);
    }
    template <bool V>
    __device__ __forceinline__ void fetch16(const Run& r, Regs (&x)[2]) const {
        const __amdgpu_buffer_rsrc_t d = data<V>(r), s = scales<V>(r);
        x[0] = load(d, s, r, 0);
        x[1] = load(d, s, r, 1);
    }
    // part i of a lane's values, run `run` of the tile
    template <bool V>
    __device__ __forceinline__ void put(const Regs& x, char* tile, int run, int i) const {
        uint32_t to = V ? vto : kto;
        if (!V && (run & 1)) to ^= HD;  // (rows 8 on: k_swizzle's bit 2 of 64 dims, 3 of 128)
        to ^= (uint32_t)i << 4;         // (a lane's parts: the slots of pieces 2 n and 2 n + 1)
        uint32_t a = x.w[2 * i], b = x.w[2 * i + 1];
        uint16_t c = x.s;
        // (else their first instructions go to the loads, to wait for them there)
        __asm__ volatile("" : "+v"(a), "+v"(b), "+v"(c));
        *reinterpret_cast<half8*>(tile + 8 * HD * 2 * run + to) = q8_values(u32x2{a, b}, c);
    }
    template <bool V>
    __device__ __forceinline__ void put(const Regs& x, char* tile, int run) const {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) put<V>(x, tile, run, i);
    }

    struct VRow {
        const char* at;
        const uint16_t* scales;
        __device__ __forceinline__ half4 dims(int d) const {
            return q8_word(*reinterpret_cast<const uint32_t*>(at + d), q8_scale(scales[d / kQ8Group]));
        }
    };
    __device__ __forceinline__ VRow v_row(int key) const {
        const unsigned page = min((unsigned)entry(key), (unsigned)p.n_pages - 1u);
        const uint32_t in = (uint32_t)(key & ((1 << p.page_log2) - 1));
        return {reinterpret_cast<const char*>(v + (uint64_t)page * (uint64_t)p.page_b + in * p.row_b),
                reinterpret_cast<const uint16_t*>(vs + (uint64_t)page * (uint64_t)p.spage_b + in * p.srow_b)};
    }
};
template <int HD, bool Q8>
using RowsOf = std::conditional_t<Q8, Q8Rows<HD>, CacheRows<HD>>;

// (see clean_chunk) of the chunk at key kb, to the rows of 32-row tiles
template <int HD, int RT, typename Rows>
__device__ __forceinline__ void add_special(const PlanPiece& z, const Rows& rows, int kb, int h2,
                                            const int (&lor)[RT], const unsigned (&span)[RT], float16v (&o)[HD / 32][RT]) {
#pragma unroll 1
    for (int key = kb; key < kb + 32; ++key) {
        int first, count;
        group_rows(key, 1, z.lo, z.kend, z.pe, first, count);
        if (count == 0) continue;
        const auto src = rows.v_row(key);
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const half4 x = src.dims(32 * dt + 8 * i4 + 4 * h2);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const bool seen = sees(key, z.pe, lor[rt], span[rt]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[dt][rt][4 * i4 + i] += (seen & !is_finite(x[i])) ? (float)x[i] : 0.f;
                }
            }
    }
}

// A wide item's tiles: 64 keys, two buffers each of K and V, of whose rows a
// wave fills 16.
template <int HD>
struct WideShape {
    static constexpr int RT = HD == 64 ? 2 : 1;  // row tiles of 32 a wave
    static constexpr int KS = HD / 16, DT = HD / 32;
    static constexpr int TILE = 64 * HD * 2;
    static constexpr int NR = 2, WI = NR * CacheRows<HD>::IPR;  // runs of 8 rows, load instructions
    static constexpr int LDS = 4 * TILE;
};
// A narrow item's: 32 keys, each wave's own; at head dim 64 two buffers.
// (8-bit rows wait in registers instead of a second one)
template <int HD, int NT, bool Q8>
struct NarrowShape {
    static constexpr int KS = HD / 32, DT = HD / 16;
    static constexpr int NB = HD == 64 && !Q8 ? 2 : 1;
    static constexpr int TILE = 32 * HD * 2;
    static constexpr int NR = 4, WI = NR * CacheRows<HD>::IPR;
    // a wave's tiles, later its state: O, then (m, l)
    static constexpr int MERGE_O = DT * NT * 64 * 16, MERGE = MERGE_O + NT * 64 * 8;
    static constexpr int WAVE = 2 * NB * TILE > MERGE ? 2 * NB * TILE : MERGE;
    static constexpr int LDS = kNW * WAVE;
};

// r / hpk (r < 2^30), as (r + 1/2) / hpk: at least 1 / (2 hpk) from a whole
// number, hpk <= 2^16, far more than f64 is off by.  (An integer division is
// ~25 dependent instructions ahead of the queries' and the output's addresses.)
__device__ __forceinline__ int token_of(const PagedParams& p, int r) { return (int)(((double)r + 0.5) * p.inv_hpk); }

// What a row's state (max M, sum L, both of the keys only) is multiplied by for
// the output: the sink joins here, last, so that probabilities are relative
// to the keys' max and keep their bits however large the sink is.
// sink: in the log2 domain, -inf for none.
__device__ __forceinline__ float row_weight(float sink, float M, float L) {
    const float top = fmaxf(M, sink), f = fast_exp2(M - top);
    return f / (L * f + fast_exp2(sink - top));
}
__device__ __forceinline__ float sink_of(const PagedParams& p, int h) { return p.sinks ? p.sinks[h] * kLog2e : -INFINITY; }

// Row rl of a piece's partials
__device__ __forceinline__ size_t partial_row(const PagedParams& p, const PlanPiece& z, int kvh, int rl) {
    return (uint32_t)z.slot * (uint32_t)p.n_kv + (uint32_t)(kvh * z.rows + rl);  // (below 2^31)
}

// Where row rl of the piece's item goes: its output, or the partial sums of a
// split item's piece
template <int HD, bool F32>
struct RowOut {
    char* at;
    bool part;
    __device__ __forceinline__ RowOut(const PagedParams& p, const PlanPiece& z, int kvh, int rl) {
        part = z.slot >= 0;
        const int r = z.r0 + rl, t = token_of(p, r), h = kvh * p.hpk + r - t * p.hpk;
        at = part ? reinterpret_cast<char*>(p.ws_o + partial_row(p, z, kvh, rl) * HD)
                  : static_cast<char*>(p.out) + ((size_t)(z.q0 + t) * p.o_tok + (size_t)h * HD) * (F32 ? 4 : 2);
    }
    // 4 dims from d on
    __device__ __forceinline__ void store(int d, const float4v& x, float w) const {
        if (F32 || part) *reinterpret_cast<float4v*>(at + 4 * d) = part ? x : x * w;
        else *reinterpret_cast<half4*>(at + 2 * d) =
            half4{(_Float16)(x[0] * w), (_Float16)(x[1] * w), (_Float16)(x[2] * w), (_Float16)(x[3] * w)};
    }
};
__device__ __forceinline__ void store_sum(const PagedParams& p, const PlanPiece& z, int kvh, int rl, float M, float L) {
    reinterpret_cast<float2*>(p.ws_ml)[partial_row(p, z, kvh, rl)] = make_float2(M, L);
}

// The polynomial; times s, the capped score of a raw product up to tanh_to
template <bool F16>
__device__ __forceinline__ float capped_small(const PagedParams& p, float s) {
    const float u = s * s;
    if constexpr (F16) return __builtin_fmaf(__builtin_fmaf(p.tanh_h[2], u, p.tanh_h[1]), u, p.tanh_h[0]);
    float y = __builtin_fmaf(p.tanh_c[4], u, p.tanh_c[3]);
    y = __builtin_fmaf(y, u, p.tanh_c[2]);
    y = __builtin_fmaf(y, u, p.tanh_c[1]);
    return __builtin_fmaf(y, u, p.tanh_c[0]);
}

// Raw products to capped scores in the log2 domain, minus m: the polynomial, and
// cap tanh(y) = cap - 2 cap / (1 + e^(2 y)), saturating at both ends, past it
template <int N, bool F16, typename V>
__device__ __forceinline__ void cap_scores(const PagedParams& p, V& s, float m = 0.f) {
    float most = 0.f;  // (NaN keeps to the polynomial, and is NaN there)
    const float to = p.tanh_to[F16];
#pragma unroll
    for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(s[i]));
    if (__builtin_amdgcn_ballot_w64(most > to)) {
        const float c2 = p.cap * kLog2e, f = 2.f * p.qscale / p.cap;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float far = c2 - m - 2.f * c2 * __builtin_amdgcn_rcpf(1.f + fast_exp2(s[i] * f));
            s[i] = fabsf(s[i]) <= to ? __builtin_fmaf(s[i], capped_small<F16>(p, s[i]), -m) : far;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = __builtin_fmaf(s[i], capped_small<F16>(p, s[i]), -m);
    }
}

// Scores of a chunk (raw products, 16-bit or f32 queries) in the log2 domain:
// scaled, capped, with the distance bias; v of a lane's scores at once.
template <bool SC, typename V, int N, typename KEY>
__device__ __forceinline__ void finish_scores(const PagedParams& p, V& s, std::integral_constant<int, N>, float slope, int pos,
                                              KEY key) {
    if (SC && p.cap > 0.f) {
        cap_scores<N, false>(p, s);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] *= p.qscale;
    }
    if (SC && p.alibi) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] -= slope * fabsf((float)(pos - key(i)));
    }
}

// The running max is kept 14 below the largest score: p up to 2^14 in f16, or as
// hi + lo parts, whose last step is 2^-24 of 2^14 then.  (With p up to 1, of
// 20000 keys 2^-20 of one other each can be 2^-25 off, and their sum 2^-11.)
constexpr float kAbove = 14.f;
// ... and 8 below a wide item's of f16 queries, whose max moves only when a
// chunk's weights sum to more than 2^14
constexpr float kAboveWide = 8.f;

__device__ __forceinline__ float ror8(float x) {  // lane l's from lane l ^ 8
    const int v = __float_as_uint(x);
    return __uint_as_float(__builtin_amdgcn_update_dpp(v, v, 0x128, 0xF, 0xF, false));
}

// A narrow item: NT tiles of 16 rows.  v_mfma_f32_16x16x32_f16: S^T = K Q^T (a
// lane holds 4 keys of one row from each 16), O^T += V^T P^T (the 8 scores of
// a lane are its part of P; V's rows are read in that order).  Each wave takes
// every fourth chunk of the piece, waits for its own loads only, and the
// four states are merged through LDS.
// f32 queries: PACK (at most 8 rows): hi parts in columns 0-7, lo parts in 8-15
// of one operand, the scores added by a lane exchange, the outputs at the end;
// otherwise two products each.
// HBM-bound over long keys (32 ragged requests at the copy's rate: 116 us);
// short ones are a chain of latencies: 64 windows of 128 keys are 8.6 us, of
// which 1.5 until the piece and its table entries are there, 1 to request the
// tiles, 2 until they land, 1.3 for the chunks, 2.4 for merge and store.  With
// 32-row tiles, every tile requested and two merge barriers they were 11.4;
// with a pack of 8 rows in a tile of 16, a 32768-key token went from 17.5 to 16.
// SHARED: the item may be a group's last block, which begins at a row of its own.
template <int HD, int NT, bool F32, bool SC, bool PACK, bool Q8, bool SHARED>
__device__ __forceinline__ void narrow_body(const PagedParams& p, const PlanPiece& z, int kvh, char* lds) {
    static_assert(!PACK || (F32 && NT == 1), "packed hi and lo parts: f32, one tile");
    using S_ = NarrowShape<HD, NT, Q8>;
    using Rows = RowsOf<HD, Q8>;
    constexpr int KS = S_::KS, DT = S_::DT, NB = S_::NB, TILE = S_::TILE, NR = S_::NR, WI = S_::WI;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, c16 = lane & 15;
    const int r0 = SHARED ? z.r0 : 0;
    char* const kbuf = lds + wave * S_::WAVE;
    char* const vbuf = kbuf + NB * TILE;
    Rows rows(p, z, kvh, lane);
    const uint32_t to = lds_byte(lds) + wave * S_::WAVE;
    auto tile_chunk = [&](int t) { return z.cb + wave + kNW * t; };
    // (a chunk in one page needs one entry)
    const bool paged_by_32 = p.page_log2 >= 5;
    auto fetch = [&](int t, int (&id)[NR]) {
        const int kb = chunk_key(tile_chunk(t), z.n_pre, z.lo_base);
        id[0] = rows.entry(kb);
        if (!paged_by_32) {
#pragma unroll
            for (int r = 1; r < NR; ++r) id[r] = rows.entry(kb + 8 * r);
        }
    };
    auto place = [&](int t, const int (&id)[NR], typename Rows::Run (&run)[NR]) {
        if constexpr (Q8) return;
        else {
            const int kb = chunk_key(tile_chunk(t), z.n_pre, z.lo_base);
            const bool whole = paged_by_32 & (kb >= z.lo) & (kb + 32 <= z.kend);
            const uint32_t run_b = 8u * p.row_b;
            run[0] = rows.run(kb, true, id[0]);
            if (!whole) {
                unrolled<NR - 1>([&](auto i) {
                    constexpr int r = decltype(i)::value + 1;
                    run[r] = rows.run(kb + 8 * r, true, paged_by_32 ? id[0] : id[r]);
                });
            } else {
                unrolled<NR - 1>([&](auto i) {
                    constexpr int r = decltype(i)::value + 1;
                    run[r].off = run[0].off + (uint32_t)r * run_b;
                    run[r].nrec = run_b;
                    run[r].skip = 0;
                });
            }
        }
    };
    auto load_tile = [&](int t, const typename Rows::Run (&run)[NR], auto is_v) {
        constexpr bool V = decltype(is_v)::value;
        if constexpr (Q8) return;
        else
#pragma unroll
        for (int x = 0; x < WI; ++x)
            rows.template load<V>(run[x / Rows::IPR], (x / Rows::IPR) & 1, x % Rows::IPR,
                                  to + ((V ? NB : 0) + t % NB) * TILE + 1024 * x);
    };
    using K_ = std::false_type;
    using V_ = std::true_type;
    const int n_tiles = (z.ce - z.cb - wave + kNW - 1) / kNW;
    // 8-bit rows: the next chunk's in registers, K's and V's, in runs as long as a page
    // allows; lane r's table entry is run r's, of the chunk after
    typename Q8Rows<HD>::Regs regs[Q8 ? 2 : 1][NR];
    typename Q8Rows<HD>::Run run32;
    auto entries_of = [&](int t) {
        const int key = chunk_key(tile_chunk(t), z.n_pre, z.lo_base) + 8 * (lane & 3);
        return rows.table[imin(key, rows.last) >> p.page_log2];
    };
    auto request = [&](auto is_v, int t, bool any, int entries) {
        constexpr bool V = decltype(is_v)::value;
        if constexpr (Q8) {
            int kb = chunk_key(tile_chunk(t), z.n_pre, z.lo_base);
            auto of_runs = [&](auto len) {
                constexpr int N = decltype(len)::value;
#pragma unroll
                for (int x = 0; x < 32 / N; ++x) {
                    typename Rows::Run r;
                    if (V && N == 32) {
                        r = run32;  // (K's; several are made again, for want of scalar registers)
                    } else {
                        __asm__ volatile("" : "+s"(kb));
                        r = rows.template run<N>(kb + N * x, any, __builtin_amdgcn_readlane(entries, x * (N / 8)));
                    }
                    if (N == 32) run32 = r;
                    const auto d = rows.template data<V>(r), sc = rows.template scales<V>(r);
#pragma unroll
                    for (int y = 0; y < N / 8; ++y) regs[V][x * (N / 8) + y] = rows.load(d, sc, r, y);
                }
            };
            if (p.page_log2 >= 5) of_runs(std::integral_constant<int, 32>{});
            else if (p.page_log2 == 4) of_runs(std::integral_constant<int, 16>{});
            else of_runs(std::integral_constant<int, 8>{});
        }
    };
    auto put_tile = [&](char* tile, auto is_v) {
        constexpr bool V = decltype(is_v)::value;
        if constexpr (Q8) {
#pragma unroll
            for (int r = 0; r < NR; ++r) rows.template put<V>(regs[V][r], tile, r);
        }
    };
    // the first tiles are requested ahead of the queries, whose use waits for
    // all that was requested before it
    int id[NB + 1][NR];
    typename Rows::Run run[NR];
    int entries = 0, next_entries = 0;  // of the chunk requested last, of the one after
    if constexpr (Q8) {
        entries = entries_of(0);
        next_entries = entries_of(1);
        __asm__ volatile("" : "+v"(entries), "+v"(next_entries)::"memory");  // (ahead of the tiles: not waited for with them)
        if (n_tiles > 0) {
            request(K_{}, 0, true, entries);
            request(V_{}, 0, true, entries);
        }
    } else {
#pragma unroll
        for (int t = 0; t <= NB; ++t) fetch(t, id[t]);
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            if (t < n_tiles) {
                place(t, id[t], run);
                load_tile(t, run, K_{});
                load_tile(t, run, V_{});
            }
        }
    }
    // queries: column c16 of each tile, dims 8 g .. of every 32
    half8 qh[NT][KS], ql[F32 && !PACK ? NT : 1][F32 && !PACK ? KS : 1];
    int posr[NT], lor[NT];
    unsigned span[NT];
    bool valid[NT];
    float slope[NT], sink[NT];  // (raw: nothing here waits for a load)
    const bool low = PACK && c16 >= 8;  // this column holds lo parts
    constexpr int QES = F32 ? 4 : 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int rl = 16 * nt + (PACK ? c16 & 7 : c16), r = min(r0 + rl, z.R - 1);
        valid[nt] = r0 + rl < z.R;
        const int t = token_of(p, r), h = kvh * p.hpk + r - t * p.hpk;
        const char* src = static_cast<const char*>(p.q) + ((size_t)(z.q0 + t) * p.q_tok + (size_t)h * HD + 8 * g) * QES;
        sink[nt] = p.sinks_or_q[p.sinks ? h : 0];
        slope[nt] = SC ? p.alibi_or_q[p.alibi ? h : 0] : 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if constexpr (F32) {
                const float4v a = *reinterpret_cast<const float4v*>(src + 128 * ks);
                const float4v b = *reinterpret_cast<const float4v*>(src + 128 * ks + 16);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    _Float16 hi, lo;
                    split_f16(i < 4 ? a[i % 4] : b[i % 4], hi, lo);
                    qh[nt][ks][i] = low ? lo : hi;
                    if constexpr (!PACK) ql[nt][ks][i] = lo;
                }
            } else {
                qh[nt][ks] = load16(src + 64 * ks);
            }
        }
        const int pos = z.pos0 + t;
        posr[nt] = pos;
        lor[nt] = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
        span[nt] = (unsigned)(pos - lor[nt]);
        if (!valid[nt]) lor[nt] = INT32_MAX, span[nt] = 0;  // (sees none)
    }
    // every row sees the keys [lo_all, hi_all] and those below z.pe
    const int hi_all = z.pos0, pos_last = z.len - 1;
    const int lo_all = p.window > 0 && pos_last >= p.window ? pos_last - p.window + 1 : 0;
    const bool hide = may_hide<Q8 ? 32 : 8>(z, hi_all, pos_last);

    float m[NT], l[NT];
    float4v o[DT][NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt][nt] = float4v{};
    }
    bool special = false;

#pragma unroll
    for (int nt = 0; nt < NT; ++nt) slope[nt] = SC && p.alibi ? slope[nt] * kLog2e : 0.f;

    // requests in order K0 V0 (K1 V1), the next ones as their buffers become
    // free: behind a tile's stand the 2 NB - 1 tiles after it, fewer at the end;
    // table entries come a tile earlier
    constexpr int AHEAD = WI * (2 * NB - 1);
    for (int t = 0; t < n_tiles; ++t) {
        const int c = tile_chunk(t), kb = chunk_key(c, z.n_pre, z.lo_base);
        const char* const kt_ = kbuf + (t % NB) * TILE;
        char* const vt = vbuf + (t % NB) * TILE;
        const int left = n_tiles - 1 - t;
        if constexpr (Q8) {
            // (behind the last chunk's the loads fetch nothing; skipped, the
            // compiler would wait for V's with K's)
            put_tile(kbuf, K_{});
            entries = next_entries;
            request(K_{}, t + 1, left >= 1, entries);
            next_entries = entries_of(t + 2);
        } else if (left >= NB - 1) {
            wait_loads<AHEAD>();
        } else {
            wait_loads<WI>();
        }
        typedef float float8v __attribute__((ext_vector_type(8)));
        float8v s[NT];
        {
            float4v sh[NT][2], sl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) sh[nt][kt] = sl[nt][kt] = float4v{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const half8 ka = *reinterpret_cast<const half8*>(kt_ + k_slot<HD>(16 * kt + c16, 4 * ks + g));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        sh[nt][kt] = mfma16(ka, qh[nt][ks], sh[nt][kt]);
                        if constexpr (F32 && !PACK) sl[nt][kt] = mfma16(ka, ql[nt][ks], sl[nt][kt]);
                    }
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float x = sh[nt][i / 4][i % 4];
                    if constexpr (PACK) x += ror8(x);
                    else if constexpr (F32) x += sl[nt][i / 4][i % 4];
                    s[nt][i] = x;
                }
        }
        if constexpr (!Q8)
            if (left >= NB) {
                lds_done();
                place(t + NB, id[NB], run);
                fetch(t + NB + 1, id[NB]);
                load_tile(t + NB, run, K_{});
            }

        auto key = [&](int i) { return kb + 16 * (i / 4) + 4 * g + i % 4; };
        const bool all = kb + 31 < z.pe || (kb >= lo_all && kb + 31 <= hi_all);
        half8 ph[NT], pl[F32 && !PACK ? NT : 1];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            finish_scores<SC>(p, s[nt], std::integral_constant<int, 8>{}, slope[nt], posr[nt], key);
            if (!all) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[nt][i] = sees(key(i), z.pe, lor[nt], span[nt]) ? s[nt][i] : -INFINITY;
            }
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaxf(s[nt][i], s[nt][4 + i]);
            const float mn = fmaxf(m[nt], group4_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))) - kAbove);
            if (__builtin_amdgcn_ballot_w64(mn > m[nt])) {
                const float cf = mn > m[nt] ? fast_exp2(m[nt] - mn) : 1.f;  // (0 while m was -inf)
                l[nt] *= cf;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt][nt] *= cf;
                m[nt] = mn;
            }
            const float ms = m[nt] == -INFINITY ? 0.f : m[nt];
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                e[i] = fast_exp2(s[nt][i] - ms);
                e[i + 1] = fast_exp2(s[nt][i + 1] - ms);
                if constexpr (F32) {
                    half2 hi, lo;
                    split_pair(e[i], e[i + 1], hi, lo);
                    const half2 own = low ? lo : hi;
                    ph[nt][i] = own[0], ph[nt][i + 1] = own[1];
                    if constexpr (!PACK) pl[nt][i] = lo[0], pl[nt][i + 1] = lo[1];
                } else {
                    ph[nt][i] = (_Float16)e[i], ph[nt][i + 1] = (_Float16)e[i + 1];
                    e[i] = (float)ph[nt][i], e[i + 1] = (float)ph[nt][i + 1];
                }
            }
            l[nt] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        }
        if constexpr (Q8) {
            put_tile(vbuf, V_{});
            request(V_{}, t + 1, left >= 1, entries);
        } else if (left >= NB) {
            wait_loads<AHEAD>();
        } else if (left == NB - 1) {
            wait_loads<2 * WI * (NB - 1)>();
        } else {
            wait_loads<0>();
        }
        if (!all && hide) special |= clean_chunk<HD>(vt, lane);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            // 4 rows' 16 dims a 16-lane group, transposed: keys 4 g .. and 16 + 4 g ..
            const int k = 4 * g + (c16 >> 2), dim = 16 * dt + 4 * (c16 & 3);
            const _Float16* a0 = reinterpret_cast<const _Float16*>(vt + v_slot<HD>(k, dim >> 3) + ((dim & 7) << 1));
            const _Float16* a1 = reinterpret_cast<const _Float16*>(vt + v_slot<HD>(k + 16, dim >> 3) + ((dim & 7) << 1));
            const half8 va = cat8(lds_read_tr(a0), lds_read_tr(a1));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[dt][nt] = mfma16(va, ph[nt], o[dt][nt]);
                if constexpr (F32 && !PACK) o[dt][nt] = mfma16(va, pl[nt], o[dt][nt]);
            }
        }
        if constexpr (!Q8)
            if (left >= NB) {
                lds_done();
                load_tile(t + NB, run, V_{});
            }
    }
    if (__builtin_expect(special, 0))
#pragma unroll 1
        for (int t = 0; t < n_tiles; ++t) {
            const int kb = chunk_key(tile_chunk(t), z.n_pre, z.lo_base);
            if (kb + 31 < z.pe || (kb >= lo_all && kb + 31 <= hi_all)) continue;
#pragma unroll 1
            for (int key = kb; key < kb + 32; ++key) {
                int first, count;
                group_rows(key, 1, z.lo, z.kend, z.pe, first, count);
                if (count == 0) continue;
                const auto src = rows.v_row(key);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const half4 x = src.dims(16 * dt + 4 * g);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const bool seen = !low & sees(key, z.pe, lor[nt], span[nt]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[dt][nt][i] += (seen & !is_finite(x[i])) ? (float)x[i] : 0.f;
                    }
                }
            }
        }

    // The waves' states through LDS, each in the room of its own tiles (which
    // it has read), merged in wave order: wave w takes the output tiles w, w +
    // 4, ...  A page outside the pool makes its wave's sums NaN.
    auto so = [&](int w) { return reinterpret_cast<float4v*>(lds + w * S_::WAVE); };
    auto sml = [&](int w) { return reinterpret_cast<float2*>(lds + w * S_::WAVE + S_::MERGE_O); };
    lds_done();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        sml(wave)[nt * 64 + lane] = make_float2(m[nt], rows.bad ? NAN : group4_sum(l[nt]));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) so(wave)[(dt * NT + nt) * 64 + lane] = o[dt][nt];
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float2 ml[kNW];
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kNW; ++w) {
            ml[w] = sml(w)[nt * 64 + lane];
            M = fmaxf(M, ml[w].x);
        }
        M += kAbove;  // (p up to 1 from here on)
        const float ms = M == -INFINITY ? 0.f : M;
        float L = 0.f, wt[kNW];
#pragma unroll
        for (int w = 0; w < kNW; ++w) {
            wt[w] = fast_exp2(ml[w].x - ms);  // 0 where the wave saw no key
            L += ml[w].y * wt[w];
        }
        const int rl = 16 * nt + (PACK ? c16 & 7 : c16);
        const bool stores = valid[nt] && !low;
        const float weight = row_weight(p.sinks ? sink[nt] * kLog2e : -INFINITY, M, L);
        const RowOut<HD, F32> out(p, z, kvh, min(rl, z.R - 1 - r0));
        if (stores && z.slot >= 0 && wave == 0 && g == 0) store_sum(p, z, kvh, rl, M, L);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            if ((dt * NT + nt) % kNW != wave) continue;
            float4v x = so(0)[(dt * NT + nt) * 64 + lane] * wt[0];
#pragma unroll
            for (int w = 1; w < kNW; ++w) x += so(w)[(dt * NT + nt) * 64 + lane] * wt[w];
            if constexpr (PACK) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] += ror8(x[i]);
            }
            if (stores) out.store(16 * dt + 4 * g, x, weight);
        }
    }
}

// A wide item's output.  A lane holds 4 dims of every 8 of its row: a wave's 32
// rows go through its part of the tiles' LDS (16-byte slots, their number
// xor the row's last bits: no bank twice), so that each store covers whole rows.
template <int HD, bool F32, int RT>
__device__ __forceinline__ void store_wide(const PagedParams& p, const PlanPiece& z, int kvh, int wave, int lane, bool bad,
                                           const float (&m)[RT], const float (&l)[RT], const float16v (&o)[HD / 32][RT],
                                           char* lds) {
    const int h2 = lane >> 5, c32 = lane & 31;
    float4v* const mine = reinterpret_cast<float4v*>(lds) + wave * (32 * HD / 4);
    const bool part = z.slot >= 0;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float L = bad ? NAN : half_sum(l[rt]);
        const int rl = (wave * RT + rt) * 32 + c32, r = min(z.r0 + rl, z.R - 1);
        if (part && h2 == 0 && z.r0 + rl < z.R) store_sum(p, z, kvh, rl, m[rt], L);
        const float w = part ? 1.f : row_weight(sink_of(p, kvh * p.hpk + r - token_of(p, r) * p.hpk), m[rt], L);
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4)
                mine[c32 * (HD / 4) + ((8 * dt + 2 * i4 + h2) ^ (c32 & 7))] =
                    float4v{o[dt][rt][4 * i4], o[dt][rt][4 * i4 + 1], o[dt][rt][4 * i4 + 2], o[dt][rt][4 * i4 + 3]} * w;
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        auto rows = [&](auto dims) {  // of a lane
            constexpr int D = decltype(dims)::value, LPR = HD / D, RPI = 64 / LPR;
#pragma unroll
            for (int j = 0; j < 32 / RPI; ++j) {
                const int rr = j * RPI + lane / LPR, d4 = (lane % LPR) * (D / 4), at = (wave * RT + rt) * 32 + rr;
                const float4v x = mine[rr * (HD / 4) + (d4 ^ (rr & 7))];
                float4v y = x;
                if constexpr (D == 8) y = mine[rr * (HD / 4) + ((d4 + 1) ^ (rr & 7))];
                if (z.r0 + at < z.R) {
                    const RowOut<HD, F32> to(p, z, kvh, at);
                    if constexpr (D == 8)
                        *reinterpret_cast<half8*>(to.at + 8 * d4) =
                            half8{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3],
                                  (_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
                    else *reinterpret_cast<float4v*>(to.at + 16 * d4) = x;
                }
            }
        };
        if (F32 || part) rows(std::integral_constant<int, 4>{});
        else rows(std::integral_constant<int, 8>{});
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    }
}

// The wide item with f32 queries: hi and lo products, a chunk at a time: loads run
// ahead, but scores, softmax and PV follow one another, where the f16 item's
// overlap (a prompt's queries may be had in f16 from the step before).  2000
// tokens of 32 / 4 heads of 128: a whole call 110 us, f16 69; the products, twice
// f16's, at a large product's rate 56.  (A pipeline over chunks has no registers left
// at head dim 64: 512 tokens over 30512 keys 657 us instead of 634; at 128 it is alike:
// the two waves of a SIMD overlap by themselves.)
template <int HD, bool SC, bool Q8>
__device__ __forceinline__ void wide_f32_body(const PagedParams& p, const PlanPiece& z, int kvh, char* lds) {
    using S = WideShape<HD>;
    constexpr int RT = S::RT, KS = S::KS, DT = S::DT, TILE = S::TILE, NR = S::NR;
    using Rows = RowsOf<HD, Q8>;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int h2 = lane >> 5, c32 = lane & 31;

    char* const kbuf = lds;
    char* const vbuf = lds + 2 * TILE;
    Rows rows(p, z, kvh, lane);
    const uint32_t to = lds_byte(lds) + 16 * HD * 2 * wave;
    // this wave fills rows 16 wave .. + 15 of a tile: two runs of one chunk
    auto run_key = [&](int t, int r) {
        return chunk_key(z.cb + 2 * t + (wave >> 1), z.n_pre, z.lo_base) + 16 * (wave & 1) + 8 * r;
    };
    auto fetch = [&](int t, int (&id)[NR]) {
#pragma unroll
        for (int r = 0; r < NR; ++r) id[r] = rows.entry(run_key(t, r));
    };
    typename Q8Rows<HD>::Regs regs[2][NR];  // of the tile after
    auto load_tile = [&](int t, const int (&id)[NR]) {
        typename Rows::Run run[NR];
        const bool any = z.cb + 2 * t + (wave >> 1) < z.ce;
        if constexpr (Q8) {
            if (p.page_log2 >= 4) {
                run[0] = rows.template run<16>(run_key(t, 0), any, id[0]);
                rows.template fetch16<false>(run[0], regs[0]);
                rows.template fetch16<true>(run[0], regs[1]);
            } else {
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    run[r] = rows.run(run_key(t, r), any, id[r]);
                    regs[0][r] = rows.template fetch<false>(run[r]);
                    regs[1][r] = rows.template fetch<true>(run[r]);
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < NR; ++r) run[r] = rows.run(run_key(t, r), any, id[r]);
            const uint32_t at = to + (t & 1) * TILE;
#pragma unroll
            for (int x = 0; x < S::WI; ++x) {
                rows.template load<false>(run[x / Rows::IPR], (x / Rows::IPR) & 1, x % Rows::IPR, at + 1024 * x);
                rows.template load<true>(run[x / Rows::IPR], (x / Rows::IPR) & 1, x % Rows::IPR, at + 2 * TILE + 1024 * x);
            }
        }
    };
    auto put_tile = [&](int t) {
        if constexpr (Q8) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                rows.template put<false>(regs[0][r], kbuf + (t & 1) * TILE + 16 * HD * 2 * wave, r);
                rows.template put<true>(regs[1][r], vbuf + (t & 1) * TILE + 16 * HD * 2 * wave, r);
            }
        }
    };
    const int n_tiles = (z.ce - z.cb + 1) / 2;
    // (ahead of the queries, whose use waits for all that was requested before)
    int id[NR];  // table entries of the next tile to request
    fetch(0, id);
    load_tile(0, id);
    fetch(1, id);

    // rows: the queries as the B operand (column c32 of each 32-row tile)
    half8 qh[RT][KS], ql[RT][KS];
    int posr[RT], lor[RT];  // position, first key of the window
    unsigned span[RT];      // keys behind that one that the row sees
    bool valid[RT];
    float slope[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = z.r0 + (wave * RT + rt) * 32 + c32;
        valid[rt] = r < z.R;
        const int rc = min(r, z.R - 1), t = token_of(p, rc), h = kvh * p.hpk + rc - t * p.hpk;
        const char* src = static_cast<const char*>(p.q) + ((size_t)(z.q0 + t) * p.q_tok + (size_t)h * HD + 8 * h2) * 4;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const float4v a = *reinterpret_cast<const float4v*>(src + 64 * ks);
            const float4v b = *reinterpret_cast<const float4v*>(src + 64 * ks + 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                _Float16 hi, lo;
                split_f16(i < 4 ? a[i % 4] : b[i % 4], hi, lo);
                qh[rt][ks][i] = hi, ql[rt][ks][i] = lo;
            }
        }
        const int pos = z.pos0 + t;
        posr[rt] = pos;
        lor[rt] = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
        span[rt] = (unsigned)(pos - lor[rt]);
        if (!valid[rt]) lor[rt] = INT32_MAX, span[rt] = 0;  // (sees none)
        slope[rt] = SC && p.alibi ? p.alibi[h] * kLog2e : 0.f;
    }
    // every row sees the keys [lo_all, hi_all] and those below z.pe
    const int r_last = min(z.R, z.r0 + kNW * RT * 32) - 1;
    const int hi_all = z.pos0 + token_of(p, z.r0), pos_last = z.pos0 + token_of(p, r_last);
    const int lo_all = p.window > 0 && pos_last >= p.window ? pos_last - p.window + 1 : 0;
    const bool hide = may_hide<Q8 ? 16 : 8>(z, hi_all, pos_last);

    float m[RT], l[RT];
    float16v o[DT][RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt][rt] = float16v{};
    }


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
                s[rt] = mfma32(ka, ql[rt][ks], s[rt]);
            }
        }
    };
    auto transform = [&](int c, float16v (&s)[RT]) {
        const int kb = chunk_key(c, z.n_pre, z.lo_base);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            finish_scores<SC>(p, s[rt], std::integral_constant<int, 16>{}, slope[rt], posr[rt],
                              [&](int i) { return kb + 8 * (i / 4) + 4 * h2 + i % 4; });
        const bool all = kb + 31 < z.pe || (kb >= lo_all && kb + 31 <= hi_all);
        if (!all) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = kb + 8 * (i / 4) + 4 * h2 + i % 4;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    s[rt][i] = sees(key, z.pe, lor[rt], span[rt]) ? s[rt][i] : -INFINITY;
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
            const float mn = fmaxf(m[rt], half_max(x) - kAbove);
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
            for (int i = 0; i < 16; i += 2) {
                const float e = fast_exp2(s[rt][i] - ms), f = fast_exp2(s[rt][i + 1] - ms);
                half2 hi, lo;
                split_pair(e, f, hi, lo);
                ph[i / 8][rt][i % 8] = hi[0], ph[i / 8][rt][i % 8 + 1] = hi[1];
                pl[i / 8][rt][i % 8] = lo[0], pl[i / 8][rt][i % 8 + 1] = lo[1];
                sum = (sum + e) + f;
            }
            l[rt] += sum;
        }
    };
    auto pv = [&](const char* vt, int sub, const half8 (&ph)[2][RT], const half8 (&pl)[2][RT]) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const half8 va = v_operand<HD>(vt, 32 * sub + 16 * w, dt, lane);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    o[dt][rt] = mfma32(va, ph[w][rt], o[dt][rt]);
                    o[dt][rt] = mfma32(va, pl[w][rt], o[dt][rt]);
                }
            }
        }
    };
    auto partly_seen = [&](int c) {
        const int kb = chunk_key(c, z.n_pre, z.lo_base);
        return hide && !(kb + 31 < z.pe || (kb >= lo_all && kb + 31 <= hi_all));
    };
    bool special = false;

    half8 ph[2][RT], pl[2][RT];
    float16v s[RT];
    if (Q8) put_tile(0);
    for (int t = 0; t < n_tiles; ++t) {
        if (!Q8) wait_loads<0>();
        __syncthreads();  // tile t is there, and no wave reads tile t - 1
        if (t + 1 < n_tiles) {
            load_tile(t + 1, id);
            fetch(t + 2, id);
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int c = z.cb + 2 * t + sub;
            if (c >= z.ce) break;
            scores(kbuf + (t & 1) * TILE, sub, c, s);
            transform(c, s);
            softmax(s, ph, pl);
            if (partly_seen(c)) special |= clean_chunk<HD>(vbuf + (t & 1) * TILE + 64 * HD * sub, lane);
            pv(vbuf + (t & 1) * TILE, sub, ph, pl);
        }
        if (Q8 && t + 1 < n_tiles) put_tile(t + 1);
    }
    const bool any_bad = __syncthreads_or(rows.bad);  // (and every wave is done with the tiles)
    if (__syncthreads_or(special))
#pragma unroll 1
        for (int c = z.cb; c < z.ce; ++c)
            if (partly_seen(c)) add_special<HD, RT>(z, rows, chunk_key(c, z.n_pre, z.lo_base), h2, lor, span, o);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float down = fast_exp2(-kAbove);  // (p up to 1 from here on)
        m[rt] += kAbove;
        l[rt] *= down;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt][rt] *= down;
    }
    store_wide<HD, true>(p, z, kvh, wave, lane, any_bad, m, l, o, lds);
}

// MFMAs between a wide step's LDS reads and their use (4, 6: alike, and more registers)
constexpr int kAhead = 2;

// Scores: scaled; capped; with a distance bias, capped or not.  (A cap between
// the MFMAs as well: 76 us instead of 77 at head dim 128, 122 instead of 107 at
// 64, for its registers.)
enum ScoreMode { kPlain, kCapped, kBiased };

// The wide item with f16 queries, as a software pipeline over 32-key chunks:
// while the softmax of chunk c runs on the vector ALUs, the matrix cores take
// QK^T of chunk c + 1 and PV of chunk c - 1, one MFMA at a time between the
// softmax's instructions.  P = 2^(x - m) with a max m that moves only when a
// chunk's row sum passes 2^14 (below it nothing overflowed f16, and keys far
// enough below m to lose bits are negligible beside the one m was taken from,
// 2^8 in weight), or is not set yet:
// then the wave takes the chunk's max, rescales O and the sum, and
// recomputes P.
//
// K and V tiles of 64 keys, double-buffered; K runs a tile ahead of V.  In
// step c = 2 t + 1 the loads of K tile t + 2 and V tile t + 1 go out between
// the MFMAs (in a burst ahead of them a wave stalls at each); the barrier after
// step 2 t orders them behind the last reads of their buffers and ahead of
// their first.  A tile's table entries are loaded a step before its loads.
//
// Bound by issue and clock: of a step's ~1900 cycles (two waves a SIMD, 1.7 -
// 1.9 GHz under load) the matrix cores are busy 1024; at head dim 64 the exp2s
// and their VALU work take as long, at 128 the LDS operands (16 rows' tile a
// wave, each read once).  4001 tokens of 32 / 4 heads of 128: 0.80 PFLOP/s; 512
// over 30512 keys of 64 / 8 of 64: 0.87.  A simple loop over tiles took 239
// and 467 us for these calls, plan and join included, which now take 167 and 293.
template <int HD, int MODE, bool Q8>
__device__ __forceinline__ void wide_body(const PagedParams& p, const PlanPiece& z, int kvh, char* lds) {
    using S_ = WideShape<HD>;
    constexpr int RT = S_::RT, KS = S_::KS, DT = S_::DT, TILE = S_::TILE, NR = S_::NR, WI = S_::WI;
    using Rows = RowsOf<HD, Q8>;
    constexpr int IPR = CacheRows<HD>::IPR;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int h2 = lane >> 5, c32 = lane & 31;
    char* const kbuf = lds;
    char* const vbuf = lds + 2 * TILE;
    const int n = z.ce - z.cb;

    Rows rows(p, z, kvh, lane);
    // this wave fills rows 16 wave .. + 15 of a tile: two runs of one chunk
    const uint32_t to_k = lds_byte(lds) + 16 * HD * 2 * wave, to_v = to_k + 2 * TILE;
    auto run_key = [&](int t, int r) {
        return chunk_key(z.cb + 2 * t + (wave >> 1), z.n_pre, z.lo_base) + 16 * (wave & 1) + 8 * r;
    };
    auto wanted = [&](int t) { return 2 * t + (wave >> 1) < n; };
    // the first tiles, then the queries beside them
    int id[NR], vid[NR];                   // table entries of the next K tile to request (8-bit rows: and V tile)
    typename Rows::Run rk[NR], rv[NR];     // runs of the K tile and the V tile to request
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        vid[r] = rows.entry(run_key(1, r));
        if constexpr (!Q8) {
            rk[r] = rows.run(run_key(0, r), wanted(0), rows.entry(run_key(0, r)));
            rv[r] = rows.run(run_key(1, r), wanted(1), vid[r]);
        }
    }
    // 8-bit rows wait in registers: V tile 0 and K tile 1, written in step 0.
    // rk[0]: the 16 rows of the last K tile requested, which are the next V
    // tile's; pages of 8 rows take two runs, made again.
    typename Q8Rows<HD>::Regs kr[NR], vr[NR];
    const bool pages16 = p.page_log2 >= 4;
    auto load_k8 = [&](int t, const int (&ids)[NR]) {
        if constexpr (Q8) {
            int key = run_key(t, 0);
            // (a run is made here and now: made ahead, it would take the scalar registers of all else)
            __asm__ volatile("" : "+s"(key));
            if (pages16) {
                rk[0] = rows.template run<16>(key, wanted(t), ids[0]);
                rows.template fetch16<false>(rk[0], kr);
            } else {
#pragma unroll
                for (int r = 0; r < NR; ++r) kr[r] = rows.template fetch<false>(rows.run(key + 8 * r, wanted(t), ids[r]));
            }
        }
    };
    auto load_v8 = [&](int t, const int (&ids)[NR]) {
        if constexpr (Q8) {
            int key = run_key(t, 0);
            __asm__ volatile("" : "+s"(key));
            if (pages16) {
                rows.template fetch16<true>(rk[0], vr);
            } else {
#pragma unroll
                for (int r = 0; r < NR; ++r) vr[r] = rows.template fetch<true>(rows.run(key + 8 * r, wanted(t), ids[r]));
            }
        }
    };
    if constexpr (Q8) {
        int first[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) first[r] = rows.entry(run_key(0, r));
        load_k8(0, first);
        load_v8(0, first);
#pragma unroll
        for (int r = 0; r < NR; ++r) rows.template put<false>(kr[r], kbuf + 16 * HD * 2 * wave, r);
        load_k8(1, vid);
    } else {
#pragma unroll
        for (int x = 0; x < WI; ++x) rows.template load<false>(rk[x / IPR], (x / IPR) & 1, x % IPR, to_k + 1024 * x);
#pragma unroll
        for (int x = 0; x < WI; ++x) rows.template load<true>(rk[x / IPR], (x / IPR) & 1, x % IPR, to_v + 1024 * x);
#pragma unroll
        for (int x = 0; x < WI; ++x) rows.template load<false>(rv[x / IPR], (x / IPR) & 1, x % IPR, to_k + TILE + 1024 * x);
    }
    // (the first step's empty PV product reads V tile 1's buffer)
#pragma unroll
    for (int i = 0; i < TILE / (16 * 64 * kNW); ++i)
        *reinterpret_cast<u32x4*>(vbuf + TILE + 16 * (64 * wave + lane + 64 * kNW * i)) = u32x4{0, 0, 0, 0};

    half8 qb[RT][KS];
    int posr[RT], lor[RT];  // position, first key of the window
    unsigned span[RT];      // keys behind that one that the row sees
    bool valid[RT];
    float slope[RT], m[RT], l[RT];
    float16v o[DT][RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = z.r0 + (wave * RT + rt) * 32 + c32;
        valid[rt] = r < z.R;
        const int rc = min(r, z.R - 1), t = token_of(p, rc), h = kvh * p.hpk + rc - t * p.hpk;
        const char* src = static_cast<const char*>(p.q) + ((size_t)(z.q0 + t) * p.q_tok + (size_t)h * HD + 8 * h2) * 2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qb[rt][ks] = load16(src + 32 * ks);
        const int pos = z.pos0 + t;
        posr[rt] = pos;
        lor[rt] = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
        span[rt] = (unsigned)(pos - lor[rt]);
        if (!valid[rt]) lor[rt] = INT32_MAX, span[rt] = 0;  // (sees none)
        slope[rt] = MODE == kBiased ? p.alibi[h] * kLog2e : 0.f;
        m[rt] = valid[rt] ? -INFINITY : 0.f;
        l[rt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt][rt] = float16v{};
    }
    const int r_last = min(z.R, z.r0 + kNW * RT * 32) - 1;
    const int hi_all = z.pos0 + token_of(p, z.r0), pos_last = z.pos0 + token_of(p, r_last);
    const int lo_all = p.window > 0 && pos_last >= p.window ? pos_last - p.window + 1 : 0;
    const bool hide = may_hide<Q8 ? 16 : 8>(z, hi_all, pos_last);

    // a chunk that not every row sees whole; its V rows may hold infinities or
    // NaN that some rows do not see (see clean_chunk)
    auto key_of = [&](int c) { return chunk_key(z.cb + c, z.n_pre, z.lo_base); };
    auto partly = [&](int kb) { return !(kb + 31 < z.pe || (kb >= lo_all && kb + 31 <= hi_all)); };
    bool special = false;
    // Chunks [w0, w0 + w_n] that every row sees whole (of a prefix's only those
    // that run into them), one compare a step; the others are looked at closer.
    const int w_end = z.n_pre + ((hi_all + 1 - z.lo_base) >> 5) - z.cb;
    int w0 = z.n_pre + ((imax(lo_all - z.lo_base, 0) + 31) >> 5) - z.cb;
    if (z.n_pre == 0 && z.lo_base == 0 && (z.pe >> 5) >= w0 + z.cb) w0 = -z.cb;
    const unsigned w_n = (unsigned)imax(w_end - w0 - 1, 0);

    // S^T of the first chunk
    auto v_chunk = [&](int c) { return vbuf + ((c >> 1) & 1) * TILE + 64 * HD * (c & 1); };

    float16v s_a[RT], s_b[RT];
    half8 p_a[2][RT], p_b[2][RT];
    const float qs = MODE == kBiased && p.cap > 0.f ? 1.f : p.qscale;

    auto step = [&](auto par, int c, float16v (&s_cur)[RT], float16v (&s_nxt)[RT], const half8 (&p_prv)[2][RT],
                    half8 (&p_cur)[2][RT]) {
        constexpr int PAR = decltype(par)::value;
        const int t = c >> 1;
        const int kb = key_of(c);
        if constexpr ((PAR & 1) == 0) {
#pragma unroll
            for (int r = 0; r < NR; ++r) id[r] = rows.entry(run_key(t + 2, r));
        } else {
#pragma unroll
            for (int r = 0; r < NR; ++r)
                if constexpr (!Q8) rk[r] = rows.run(run_key(t + 2, r), wanted(t + 2), id[r]);
        }
        auto load_nth = [&](auto x_) {
            constexpr int x = decltype(x_)::value;
            if constexpr (Q8) {
                if constexpr (x == 0) load_v8(t + 1, vid);  // (ahead of K's, whose run it takes)
                else load_k8(t + 2, id);
            } else if constexpr (x < WI)  // K tile t + 2
                rows.template load<false>(rk[x / IPR], (x / IPR) & 1, x % IPR, to_k + ((PAR >> 1) & 1) * TILE + 1024 * x);
            else  // V tile t + 1
                rows.template load<true>(rv[x / IPR - NR], (x / IPR) & 1, x % IPR, to_v + (((PAR >> 1) + 1) & 1) * TILE + 1024 * (x - WI));
        };
        // (an even step) a part of K tile t + 1 or V tile t, 8-bit rows as f16
        constexpr int PARTS = Q8Rows<HD>::PARTS, NPUT = Q8 && (PAR & 1) == 0 ? 2 * NR * PARTS : 0;
        auto put_nth = [&](auto x_) {
            constexpr int x = decltype(x_)::value % (NR * PARTS);
            if constexpr (!Q8) return;
            else if constexpr (decltype(x_)::value < NR * PARTS)
                rows.template put<true>(vr[x / PARTS], vbuf + (PAR >> 1) * TILE + 16 * HD * 2 * wave, x / PARTS, x % PARTS);
            else
                rows.template put<false>(kr[x / PARTS], kbuf + ((PAR >> 1) ^ 1) * TILE + 16 * HD * 2 * wave, x / PARTS, x % PARTS);
        };
        float ms[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            ms[rt] = m[rt] == -INFINITY ? 0.f : m[rt];
            if (MODE == kCapped) cap_scores<16, true>(p, s_cur[rt], ms[rt]);
            if (MODE == kBiased && p.cap > 0.f) cap_scores<16, true>(p, s_cur[rt]);
        }
        if ((unsigned)(c - 1 - w0) >= w_n) {  // this chunk or the one before
            if (c > 0 && hide && partly(key_of(c - 1))) special |= clean_chunk<HD>(v_chunk(c - 1), lane);
            if (partly(kb)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = kb + 8 * (i / 4) + 4 * h2 + i % 4;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        s_cur[rt][i] = sees(key, z.pe, lor[rt], span[rt]) ? s_cur[rt][i] : -INFINITY;
                }
            }
        }
        // operands: KS pieces of K (chunk c + 1), then 2 DT of V^T (chunk
        // c - 1), each read kAhead MFMAs ahead of its first
        constexpr int NOPD = KS + 2 * DT, NM = KS * RT + 2 * DT * RT;
        half8 opd[NOPD];
        const char* const kt = kbuf + (((PAR + 1) >> 1) & 1) * TILE;
        const char* const vt = vbuf + (((PAR + 3) >> 1) & 1) * TILE;
        const int krow = 32 * ((PAR + 1) & 1) + c32;
        auto read_opd = [&](auto r_) {
            constexpr int r = decltype(r_)::value;
            if constexpr (r < KS) {
                opd[r] = *reinterpret_cast<const half8*>(kt + k_slot<HD>(krow, 2 * r + h2));
            } else {
                constexpr int w = (r - KS) / DT, dt = (r - KS) % DT;
                opd[r] = v_operand<HD>(vt, 32 * ((PAR + 3) & 1) + 16 * w, dt, lane);
            }
        };
        constexpr int AHEAD = kAhead / RT;
        unrolled<AHEAD>([&](auto i) { read_opd(i); });
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s_nxt[rt] = float16v{};
        // The softmax's stages (x - m, exp2, f16 pairs, row sum) are skewed by a
        // slot (an MFMA) each, NS / NM scores a slot.
        constexpr int NS = 16 * RT, NP = NS / 2, S = NS / NM;
        static_assert(NS % NM == 0, "whole scores a slot");
        constexpr int NLD = (PAR & 1) ? 2 * (Q8 ? 1 : WI) : 0;
        constexpr int LSL = HD == 128 ? NM : NM / 2;  // slots the loads go out in
        float acc[RT][2], e[NS], ahead[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            acc[rt][0] = acc[rt][1] = 0.f;
            if (MODE == kBiased) ahead[rt] = (float)(posr[rt] - kb - 4 * h2);
        }
        auto op_fma = [&](int i) {
            if (MODE == kCapped || i >= NS) return;
            const int rt = i / 16;
            float x = __builtin_fmaf(s_cur[rt][i % 16], qs, -ms[rt]);
            if constexpr (MODE == kBiased)
                x = __builtin_fmaf(-slope[rt], fabsf(ahead[rt] - (float)(8 * (i % 16 / 4) + i % 4)), x);
            s_cur[rt][i % 16] = x;
        };
        auto op_exp = [&](int i) {
            if (i < NS) e[i] = fast_exp2(s_cur[i / 16][i % 16]);
        };
        auto op_pack = [&](int k) {
            const int rt = k / 8, i = 2 * (k % 8);
            p_cur[i / 8][rt][i % 8] = (_Float16)e[2 * k];
            p_cur[i / 8][rt][i % 8 + 1] = (_Float16)e[2 * k + 1];
        };
        auto op_sum = [&](int k) {
            const int rt = k / 8, i = 2 * (k % 8);
            acc[rt][k & 1] = __builtin_amdgcn_fdot2(half2{p_cur[i / 8][rt][i % 8], p_cur[i / 8][rt][i % 8 + 1]},
                                                    half2{1, 1}, acc[rt][k & 1], false);
        };
        // pairs whose exp2s are done after slot u
        auto ready = [](int u) { return u < 0 ? 0 : (S * (u + 1)) / 2; };
#pragma unroll
        for (int j = 0; j < S; ++j) op_fma(j);
        unrolled<NM>([&](auto u_) {
            constexpr int u = decltype(u_)::value;
            constexpr bool of_k = u < KS * RT;
            constexpr int r = u / RT, rt = u % RT;
            if constexpr (rt == 0 && r + AHEAD < NOPD) read_opd(std::integral_constant<int, r + AHEAD>{});
            unrolled<NLD>([&](auto i) {
                if constexpr (decltype(i)::value * LSL / NLD == u) load_nth(i);
            });
            unrolled<NPUT>([&](auto i) {
                if constexpr (decltype(i)::value * NM / NPUT + NM / NPUT - 1 == u) put_nth(i);
            });
            if constexpr (of_k) {
                s_nxt[rt] = mfma32(opd[r], qb[rt][r], s_nxt[rt]);
            } else {
                constexpr int w = (r - KS) / DT, dt = (r - KS) % DT;
                o[dt][rt] = mfma32(opd[r], p_prv[w][rt], o[dt][rt]);
            }
#pragma unroll
            for (int k = ready(u - 3); k < ready(u - 2); ++k) op_sum(k);
#pragma unroll
            for (int k = ready(u - 2); k < ready(u - 1); ++k) op_pack(k);
#pragma unroll
            for (int j = 0; j < S; ++j) op_exp(S * u + j);
#pragma unroll
            for (int j = 0; j < S; ++j) op_fma(S * (u + 1) + j);
            __builtin_amdgcn_sched_barrier(0);
        });
#pragma unroll
        for (int k = ready(NM - 2); k < NP; ++k) op_pack(k);
#pragma unroll
        for (int k = ready(NM - 3); k < NP; ++k) op_sum(k);
        float ls[RT];
        bool redo = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            ls[rt] = acc[rt][0] + acc[rt][1];
            redo |= !(ls[rt] <= 16384.f) || m[rt] == -INFINITY;
        }
        if (__builtin_amdgcn_ballot_w64(redo)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float x = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) x = fmaxf(x, s_cur[rt][i]);
                const float mn = fmaxf(m[rt], half_max(x) + ms[rt] - kAboveWide);
                if (mn > m[rt]) {
                    const float cf = fast_exp2(m[rt] - mn);  // 0 while m was -inf
                    l[rt] *= cf;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[dt][rt] *= cf;
                    m[rt] = mn;
                }
                const float shift = ms[rt] - (m[rt] == -INFINITY ? 0.f : m[rt]);
                float a = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p_cur[i / 8][rt][i % 8] = (_Float16)fast_exp2(s_cur[rt][i] + shift);
                    a += (float)p_cur[i / 8][rt][i % 8];
                }
                ls[rt] = a;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) l[rt] += ls[rt];
        if constexpr (PAR & 1) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                if constexpr (Q8) vid[r] = id[r];
                else rv[r] = rk[r];
            }
        } else {
            if (!Q8) wait_loads<0>();
            __syncthreads();
        }
    };

    if (!Q8) wait_loads<0>();
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s_a[rt] = float16v{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const half8 ka = *reinterpret_cast<const half8*>(kbuf + k_slot<HD>(c32, 2 * ks + h2));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s_a[rt] = mfma32(ka, qb[rt][ks], s_a[rt]);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) p_b[w][rt] = half8{0, 0, 0, 0, 0, 0, 0, 0};
    using P0 = std::integral_constant<int, 0>;
    using P1 = std::integral_constant<int, 1>;
    using P2 = std::integral_constant<int, 2>;
    using P3 = std::integral_constant<int, 3>;
    // Of the waves of two workgroups on a SIMD the older one's instructions go
    // first: it would end well ahead of the other, which then has the SIMD
    // alone.  Of long pieces the wave with more to do goes first instead (512
    // tokens over 30000 keys: 322 -> 308 us; short ones leave their slots to
    // the next pieces: 2000 tokens took 81 us instead of 77).
    auto priority = [&](int left) {
        if (n <= 64) return;
        if (left > 64) __builtin_amdgcn_s_setprio(3);
        else if (left > 24) __builtin_amdgcn_s_setprio(2);
        else if (left > 8) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
    };
    int c = 0;
    for (; c + 4 <= n; c += 4) {
        priority(n - c);
        step(P0{}, c, s_a, s_b, p_b, p_a);
        step(P1{}, c + 1, s_b, s_a, p_a, p_b);
        step(P2{}, c + 2, s_a, s_b, p_b, p_a);
        step(P3{}, c + 3, s_b, s_a, p_a, p_b);
    }
    const int rem = n - c;
    if (rem >= 1) step(P0{}, c, s_a, s_b, p_b, p_a);
    if (rem >= 2) step(P1{}, c + 1, s_b, s_a, p_a, p_b);
    if (rem >= 3) step(P2{}, c + 2, s_a, s_b, p_b, p_a);
    if (!Q8) wait_loads<0>();  // (what was requested past the last tile)
    if (hide && partly(key_of(n - 1))) special |= clean_chunk<HD>(v_chunk(n - 1), lane);
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const half8 va = v_operand<HD>(v_chunk(n - 1), 16 * w, dt, lane);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[dt][rt] = mfma32(va, (n & 1) ? p_a[w][rt] : p_b[w][rt], o[dt][rt]);
        }
    const bool any_bad = __syncthreads_or(rows.bad);
    if (__syncthreads_or(special))
#pragma unroll 1
        for (int i = 0; i < n; ++i)
            if (partly(key_of(i))) add_special<HD, RT>(z, rows, key_of(i), h2, lor, span, o);
    store_wide<HD, false>(p, z, kvh, wave, lane, any_bad, m, l, o, lds);
}

// Rows of the step's largest item: at most 8, 16 or 32 (narrow), or more; or more
// and, of a plan of shared keys, a group's last block among them.
enum RowLimit { kRows8, kRows16, kRows32, kRowsWide, kRowsShared };
// Whether plain plans' wide steps have a kernel of their own.  Narrow items that
// begin at a row of their own, a group's last blocks, cost the wide items beside them
// registers where those are fewest: f16 pages, head dim 64, capped, 512 tokens over 30512
// keys 412 us in one kernel for both plans (53 scalar spills more), 371 apart, a prompt of
// 4001 252 and 219, uncapped alike.  Apart, the others gain nothing or lose by
// the order that their instructions happen to fall into: a capped prompt of head dim 128 181
// and 188, a capped f32 chunk over 8-bit pages of 64 768 and 793.
template <int HD, bool Q8>
constexpr bool kPlainWide = HD == 64 && !Q8;

template <int HD, bool F32, int MODE, int ROWS, bool Q8>
__global__ __launch_bounds__(64 * kNW) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_kernel(PagedParams p) {
    constexpr bool SHARED = ROWS == kRowsShared, WIDE = ROWS == kRowsWide || SHARED, SC = MODE != kPlain;
    constexpr int LN = NarrowShape<HD, ROWS >= kRows32 ? 2 : 1, Q8>::LDS, LW = WIDE ? WideShape<HD>::LDS : 0;
    __shared__ __attribute__((aligned(16))) char lds[LN > LW ? LN : LW];
    const int id = blockIdx.x / p.n_kv, kvh = blockIdx.x % p.n_kv;
    // (the piece beside the header, not after it: one round trip)
    const PlanPiece z = p.pieces[id];
    const uint32_t sig = p.head->sig;
    const int n_pieces = p.head->n_pieces;
    // (and what the end reads of the arguments: a line's first touch is a round trip)
    __asm__ volatile("" ::"s"(z.seq), "s"(z.cb), "s"(z.slot), "s"(z.kend), "s"(sig), "s"(n_pieces), "s"(p.out), "s"(p.o_tok),
                     "s"(p.qscale), "s"(z.rows));
    if (sig != p.sig || id >= n_pieces) return;
    if constexpr (WIDE) {
        if (z.R > kNarrowRows && !(SHARED && z.narrow)) {
            if constexpr (F32) wide_f32_body<HD, SC, Q8>(p, z, kvh, lds);
            else wide_body<HD, MODE, Q8>(p, z, kvh, lds);
        } else if (z.R - (SHARED ? z.r0 : 0) > 16) {
            narrow_body<HD, 2, F32, SC, false, Q8, SHARED>(p, z, kvh, lds);
        } else {
            narrow_body<HD, 1, F32, SC, false, Q8, SHARED>(p, z, kvh, lds);
        }
    } else {
        narrow_body<HD, ROWS == kRows32 ? 2 : 1, F32, SC, F32 && ROWS == kRows8, Q8, false>(p, z, kvh, lds);
    }
}

template <typename F>
hipError_t with_shape(const PagedParams& p, F f) {
    auto hd = [&](auto h) {
        return p.f32 ? f(h, std::true_type{}) : f(h, std::false_type{});
    };
    return p.hd == 64 ? hd(std::integral_constant<int, 64>{}) : hd(std::integral_constant<int, 128>{});
}

template <bool Q8>
hipError_t launch_paged_as(const PagedParams& p, hipStream_t st) {
    ProfScope ps(kProfPaged, st);
    return with_shape(p, [&](auto hd, auto f32) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool F32 = decltype(f32)::value;
        const dim3 grid((unsigned)p.max_pieces * p.n_kv);
        auto go = [&](auto s, auto rows) {
            hipLaunchKernelGGL((paged_kernel<HD, F32, decltype(s)::value, decltype(rows)::value, Q8>), grid, dim3(64 * kNW), 0, st, p);
        };
        auto wide = [&](auto s) {
            // (no distance bias over shared keys; capped f32 scores take its path)
            constexpr bool both = decltype(s)::value != kBiased || F32;
            if constexpr (!kPlainWide<HD, Q8>) go(s, std::integral_constant<int, kRowsShared>{});
            else if (both && p.shared_joins) go(s, std::integral_constant<int, both ? kRowsShared : kRowsWide>{});
            else go(s, std::integral_constant<int, kRowsWide>{});
        };
        auto by_rows = [&](auto s) {
            // (f16 queries have no parts to pack)
            if (p.wide) wide(s);
            else if (p.rows > 16) go(s, std::integral_constant<int, kRows32>{});
            else if (p.rows > 8 || !F32) go(s, std::integral_constant<int, kRows16>{});
            else go(s, std::integral_constant<int, F32 ? kRows8 : kRows16>{});
        };
        // (all but the wide items of f16 queries take either score by one path)
        if (p.cap > 0.f && !p.alibi && p.wide) wide(std::integral_constant<int, F32 ? kBiased : kCapped>{});
        else if (p.cap > 0.f || p.alibi) by_rows(std::integral_constant<int, kBiased>{});
        else by_rows(std::integral_constant<int, kPlain>{});
        return hipGetLastError();
    });
}

}  // namespace

}  // namespace pelica

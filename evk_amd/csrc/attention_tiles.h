// Pieces of the MFMA attention kernels (window.hip, prefix.hip): tiles of rows in
// LDS, their fragments, the running softmax, and what keeps hidden rows apart.
//
// v_mfma_f32_16x16x32_f16 throughout: S^T = K Q^T gives a lane one query
// (column l16 = lane % 16) and rows 4 g + j (g = lane / 16) of each 16-row
// block, which is the B operand of O^T += V^T P^T as it stands (slot s: row
// 4 g + s of the first, 4 g + s - 4 of the second block); V^T comes from the
// row-major tile by ds_read_b64_tr_b16.
#pragma once

#include "kernels.h"

#include <math.h>

namespace evkhip {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

DEV void wave_sync() {  // the wave's LDS accesses before this are done
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int BK = 64;               // list entries per tile
constexpr float RESCALE_LOG2 = 8.0f;  // O and l are rescaled when a score passes the reference by 2^8

template <int DH>
struct Geo {
    static constexpr int KS = DH / 32, DT = DH / 16;
    static constexpr int W = DH <= 32 ? 32 : DH <= 64 ? 64 : DH <= 128 ? 128 : 256;  // halves of an LDS row
    static constexpr int CPR = W / 8;                                               // 16-byte chunks of it
};
// Chunk c of row r lies at slot c ^ swz(r).  LDS serves a transposed read in
// halves of the wave (rows 0 .. 7, 8 .. 15 at one pair of chunks) and a 16-byte
// read in four sets of lanes, each with all 16 rows, rows 4 .. 11 at the chunk
// of the neighbouring g: both meet every bank once (measured: no conflicts).
template <int W>
DEV int swz(int r) {
    return 2 * (W >= 128 ? r & 7 : W == 64 ? (r >> 1) & 3 : (r >> 2) & 1);
}
// A lane's places in a tile: offsets are sums of a row's and exclusive ors of
// a chunk's part.
template <int DH>
struct Frag {
    static constexpr int W = Geo<DH>::W;
    int row_at, col_at;
    DEV explicit Frag(int lane) {
        const int l16 = lane & 15, g = lane >> 4, r = 4 * g + (l16 >> 2), c = l16 & 3;
        row_at = l16 * W + ((g ^ swz<W>(l16)) << 3);
        col_at = r * W + (((c >> 1) ^ swz<W>(r)) << 3) + (c & 1) * 4;
    }
    // row r0 + l16 (r0 a multiple of 16), chunk 4 ks + g
    DEV half8 row(const f16* t, int r0, int ks) const {
        return *reinterpret_cast<const half8*>(t + r0 * W + (row_at ^ (ks << 5)));
    }
    // column 16 d + l16 of rows r0 + 4 g .. + 3 and 16 further (r0 a multiple of 32): two transposed reads
    DEV half8 col(const f16* t, int r0, int d) const {
        const f16* p = t + r0 * W + (col_at ^ (d << 4));
        return cat4(lds_read_tr(p), lds_read_tr(p + 16 * W));
    }
};

// buf_rsrc of values that are the same in the whole wave, wherever they were computed
DEV __amdgpu_buffer_rsrc_t wave_rsrc(const void* base, uint32_t bytes) {
    const uint64_t p = (uint64_t)base;
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)p), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32));
    return buf_rsrc((const void*)(hi << 32 | lo), (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes));
}

// ROWS rows of 16-byte chunks into LDS by NWV waves: the lane's share of one
// tile is chunk `chunk(i)` of row `row(i)`, i < PER, each 16 bytes to
// lds + 1 KB (wave PER + i) + 16 lane.
template <int DH, int ROWS, int NWV>
struct TileDma {
    using G = Geo<DH>;
    static constexpr int RPI = 64 / G::CPR, PER = ROWS / RPI / NWV;
    static_assert(PER >= 1 && ROWS % (RPI * NWV) == 0, "tile shape");
    int wave, lane;
    DEV int row(int i) const { return (wave * PER + i) * RPI + lane / G::CPR; }
    DEV int chunk(int i) const { return (lane % G::CPR) ^ swz<G::W>(row(i)); }
    DEV void go(__amdgpu_buffer_rsrc_t res, const uint32_t (&off)[PER], f16* lds) const {
        const uint32_t at = lds_addr(lds) + wave * PER * 1024;
#pragma unroll
        for (int i = 0; i < PER; ++i) dma16(res, off[i], at + i * 1024);
    }
};

// This wave's loads have arrived, and no access moves ahead of that.  The builtin
// tells the compiler as much, which otherwise waits in the loop for registers
// that were loaded before it, and so for the loads into LDS.
DEV void wait_loads() {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    asm volatile("" ::: "memory");
}

// N steps, each of M MFMAs on fragments that R LDS reads brought: the reads of
// step i + AHEAD go out before the MFMAs of step i (read(i, slot) into slot
// i % (AHEAD + 1) of a ring, use(i, slot)).  start() requests the first ones,
// ahead of work that hides them; `pin` holds the scheduler to this order.
template <int N, int AHEAD>
struct Ring {
    static constexpr int SLOTS = AHEAD + 1;
    template <int R, class F>
    static DEV void start(F&& read) {
        static_for<AHEAD>([&](auto i) { read(i, i); });
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * R, 0);
    }
    template <int M, int R, class F, class U>
    static DEV void run(F&& read, U&& use) {
        static_for<N>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            if constexpr (i + AHEAD < N) {
                read(std::integral_constant<int, i + AHEAD>{}, std::integral_constant<int, (i + AHEAD) % SLOTS>{});
                __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
            }
            use(ic, std::integral_constant<int, i % SLOTS>{});
            __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
        });
    }
};

DEV float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// over the four lanes of a query (16 and 32 apart)
DEV float query_max(float m) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
DEV float query_sum(float m) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// Hidden rows.  The MFMA's product of a weight of 0 and a NaN or an infinity is
// NaN, and the rows of a tile that some of its columns (queries; keys in the
// kernel of dK and dV) do not see may hold either: stale cache rows, padding, a
// gradient that overflowed.  In tiles that are not seen whole, the wave that
// loads a row looks at it and leaves zeros in LDS where it finds such a value;
// the columns that do see the row add it at the end, from memory and in 32 bits,
// unless their sums are NaN by then.  So it reaches those alone, and what it
// costs goes by the rows at the ends of a list, not by pairs: 4096 queries of 8
// heads over 2 of 128 values, window 512, both directions 111 us, with one
// infinite row of dO 129, an infinity in every hundredth value of dO 497, a third
// of all rows NaN 382.

// NaN or infinity among the values: a product with 0 is 0 for every other one
DEV half2_t wild2(const half8& x, half2_t w) {
    const half2_t z = {(f16)0.0f, (f16)0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) w = __builtin_elementwise_fma(half2_t{x[2 * i], x[2 * i + 1]}, z, w);
    return w;
}

DEV bool is_wild(half2_t w) { return !((float)w[0] == 0.0f && (float)w[1] == 0.0f); }
DEV bool wild_row(const f16* p, int n) {  // n a multiple of 8
    half2_t w = {(f16)0.0f, (f16)0.0f};
    for (int i = 0; i < n; i += 8) w = wild2(*reinterpret_cast<const half8*>(p + i), w);
    return is_wild(w);
}
// This wave's part of a tile in LDS, with zeros for the rows that hold a NaN or
// an infinity; their bits, the part's first row lowest.
template <class Dma>
DEV uint32_t clean_rows(const Dma& dma, f16* tile) {
    constexpr int CPR = Dma::G::CPR, RPI = Dma::RPI;
    int lane = dma.lane;
    asm volatile("" : "+v"(lane));  // addresses formed here, not kept through the kernel
    uint32_t rows = 0;
#pragma unroll
    for (int i = 0; i < Dma::PER; ++i) {
        u32x4* const p = reinterpret_cast<u32x4*>(tile + ((dma.wave * Dma::PER + i) * 64 + lane) * 8);
        const uint64_t hit = __ballot(is_wild(wild2(as_half8(*p), half2_t{(f16)0.0f, (f16)0.0f})));
        if (!hit) continue;
        constexpr uint64_t ROW = (1ull << CPR) - 1;
        if (hit >> (lane / CPR * CPR) & ROW) *p = u32x4{0u, 0u, 0u, 0u};
        for (int k = 0; k < RPI; ++k) rows |= (hit >> (k * CPR) & ROW ? 1u : 0u) << (i * RPI + k);
    }
    return rows;
}
// What follows runs for such rows only, a few loads at a time and from places
// formed on the spot: kept from the kernel's start, they would cost every call
// the registers.
//
// products of the columns' operands (values 32 ks + 8 g and on) and a row, in each column's four lanes
template <int KS, int QB>
DEV void row_dot(float (&v)[QB], const half8 (&x)[QB][KS], const f16* row, int dh, int g) {
    asm volatile("" : "+v"(g));
#pragma unroll
    for (int q = 0; q < QB; ++q) v[q] = 0.0f;
#pragma unroll
    for (int k0 = 0; k0 < KS; k0 += 4) {
        u32x4 y[4];
#pragma unroll
        for (int k = 0; k < 4 && k0 + k < KS; ++k) y[k] = *reinterpret_cast<const u32x4*>(row + min(32 * (k0 + k) + 8 * g, dh - 8));
#pragma unroll
        for (int k = 0; k < 4 && k0 + k < KS; ++k) {
            const half8 r = as_half8(32 * (k0 + k) + 8 * g < dh ? y[k] : u32x4{0u, 0u, 0u, 0u});
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                u32x4 u = as_u32x4(x[q][k0 + k]);
                asm volatile("" : "+v"(u));  // else converted once, for the lengths at the start, and kept
                const half8 c = as_half8(u);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[q] = __builtin_fmaf((float)c[i], (float)r[i], v[q]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int q = 0; q < QB; ++q) v[q] = query_sum(v[q]);
}
// The same of the queries of an MFMA's columns and a row of K, as the MFMA had it: with any other order of the sum,
// exponents of large scores would differ from those that the sums l hold.
template <int KS, int QB>
DEV void row_scores(float (&v)[QB], const half8 (&x)[QB][KS], const f16* row, int dh, int g) {
    asm volatile("" : "+v"(g));
    floatx4 s[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q) s[q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k0 = 0; k0 < KS; k0 += 4) {
        u32x4 y[4];
#pragma unroll
        for (int k = 0; k < 4 && k0 + k < KS; ++k) y[k] = *reinterpret_cast<const u32x4*>(row + min(32 * (k0 + k) + 8 * g, dh - 8));
#pragma unroll
        for (int k = 0; k < 4 && k0 + k < KS; ++k) {
            const half8 r = as_half8(32 * (k0 + k) + 8 * g < dh ? y[k] : u32x4{0u, 0u, 0u, 0u});  // each of 16 rows
#pragma unroll
            for (int q = 0; q < QB; ++q) s[q] = mfma16(r, x[q][k0 + k], s[q]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int q = 0; q < QB; ++q) v[q] = s[q][0];
}
// acc[d][q] += w[q] row, for the columns that see it (and what nobody stores: values past dh)
template <int DT, int QB>
DEV void add_row(floatx4 (&acc)[DT][QB], const float (&w)[QB], const bool (&sees)[QB], const f16* row, int dh, int g) {
    asm volatile("" : "+v"(g));
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += 8) {
        half4 v[8];
#pragma unroll
        for (int d = 0; d < 8 && d0 + d < DT; ++d) v[d] = *reinterpret_cast<const half4*>(row + min(16 * (d0 + d) + 4 * g, dh - 4));
#pragma unroll
        for (int d = 0; d < 8 && d0 + d < DT; ++d)
#pragma unroll
            for (int q = 0; q < QB; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float o = acc[d0 + d][q][j];
                    acc[d0 + d][q][j] = sees[q] ? __builtin_fmaf(w[q], (float)v[d][j], o) : o;
                }
        __builtin_amdgcn_sched_barrier(0);
    }
}
// Columns whose sums in this lane are all NaN, which nothing that is added changes
template <int DT, int QB>
DEV void spoilt(bool (&nan)[QB], const floatx4 (&acc)[DT][QB]) {
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        nan[q] = true;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) nan[q] &= acc[d][q][j] != acc[d][q][j];
    }
}
template <int QB>
DEV bool any_open(const bool (&sees)[QB], const bool (&nan)[QB]) {
    bool open = false;
#pragma unroll
    for (int q = 0; q < QB; ++q) open |= sees[q] & !nan[q];
    return __any(open);
}

// Exponents, in powers of two: (s - m) c2 + LIFT with m a score (raw, as s is), in one product and sum from the rounded
// LIFT - m c2.  While |m| c2 stays below 2^12, that rounding moves a weight by 2^-13 at most.  From there on (FAR) the
// difference is formed first, which 32 bits hold: a rounding of m c2 would shift all weights of a row, by powers of two
// from 2^24 on (at 2^29 past fp16's largest value), and those of every part of its list by another one.  Such rows are
// done again from the list's start (8 x 500 tokens, 16 heads over 4 of 128, behind 4096 rows: 156 us, with scores of tens
// of thousands 302): both ways in one loop, by a branch, cost every prompt 3 to 5% (the products no longer run under the
// exponentials) or a third more registers.
constexpr float FAR_LOG2 = 4096.0f;

// P, l and O carry 2^LIFT: P then is 2^15 at most, and fp16 holds all its bits down to 2^-21 of the reference (2^-14
// without).  A first row that draws most of the weight and holds little of the values, as models have it (what sinks are
// kept for), leaves the output to many small weights.
constexpr int LIFT = 7;

// The running softmax state of QB blocks of 16 queries (a lane: query l16 of
// each) and the products of a tile of 16 KB rows into it.
template <int DH, int QB>
struct Softmax {
    static constexpr int DT = Geo<DH>::DT, W = Geo<DH>::W;
    floatx4 o[DT][QB];  // O^T: dh 16 d + 4 g + j, query l16
    float m[QB], l[QB];  // the score that exponents refer to (-inf: none yet), this lane's part of the sum
    bool far;            // |m| c2 has passed FAR_LOG2 for some query of the wave
    DEV Softmax() { reset(); }
    DEV void reset() {
        far = false;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            m[q] = -INFINITY;
            l[q] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // What a score's difference to m starts from, and what is taken off first
    template <bool FAR>
    DEV void refer(int q, float c2, float& base, float& off) const {
        const bool none = m[q] == -INFINITY;
        base = FAR ? (float)LIFT : none ? 0.0f : __builtin_fmaf(-m[q], c2, (float)LIFT);
        off = FAR && !none ? m[q] : 0.0f;
    }
    // Scores s (raw) of KB blocks of rows to probabilities, as B operands: P is
    // rounded to fp16 for the product (V is fp16 as well), the sum l is not.
    template <bool FAR, int KB>
    DEV void probs(const floatx4 (&s)[KB][QB], float c2, half8 (&p)[KB / 2][QB]) {
        float mx[QB];
        bool grow = false;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            mx[q] = fmaxf(max3(s[0][q][0], s[0][q][1], s[0][q][2]), s[0][q][3]);
#pragma unroll
            for (int kb = 1; kb < KB; ++kb)
                mx[q] = max3(max3(s[kb][q][0], s[kb][q][1], mx[q]), s[kb][q][2], s[kb][q][3]);
            grow |= (mx[q] - m[q]) * c2 > RESCALE_LOG2;
        }
        if (__any(grow)) {
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                const float mn = fmaxf(m[q], query_max(mx[q]));
                const float keep = m[q] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[q] - mn) * c2);
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d][q] *= keep;
                l[q] *= keep;
                m[q] = mn;
                if (!FAR) far |= __any((fabsf(mn) * c2 >= FAR_LOG2) & (fabsf(mn) < INFINITY));
            }
        }
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            float base, off;
            refer<FAR>(q, c2, base, off);
#pragma unroll
            for (int k2 = 0; k2 < KB / 2; ++k2) {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = s[2 * k2 + i / 4][q][i % 4];
                    e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(FAR ? x - off : x, c2, base));
                }
                l[q] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
                p[k2][q] = as_half8(u32x4{pack_h2(e[0], e[1]), pack_h2(e[2], e[3]), pack_h2(e[4], e[5]), pack_h2(e[6], e[7])});
            }
        }
    }
    // V's row of an entry that the queries of `sees` see, whose probability the sums l already hold (`again`: by FAR's way)
    DEV void add_row(const bool (&sees)[QB], const f16* k, const f16* v, const half8 (&qf)[QB][Geo<DH>::KS], int dh, float c2, int g, bool again) {
        float w[QB];
        bool nan[QB];
        spoilt(nan, o);
        if (!any_open(sees, nan)) return;
        row_scores(w, qf, k, dh, g);
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            float base, off, far_base, far_off;
            refer<false>(q, c2, base, off);
            refer<true>(q, c2, far_base, far_off);
            w[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[q] - (again ? far_off : off), c2, again ? far_base : base));
        }
        ::evkhip::add_row(o, w, sees, v, dh, g);
    }
    // log-sum-exp, l the whole sum
    static DEV float lse(float m, float l, float scale) { return __builtin_fmaf(m, scale, (log2f(l) - (float)LIFT) * kLn2); }
};
// The factor of a state whose exponents refer to m in one that refer to `most`
DEV float state_weight(float m, float most, float c2) { return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - most) * c2); }

// f(entry) for the entries of the tiles of `len`, from tile t0 in steps of dt, that
// are not seen whole (plain) and whose rows (null: none) hold a NaN or an infinity
template <class Plain, class Row, class F>
DEV void each_wild(Plain&& plain, Row&& row, int dh, int len, int t0, int t1, int dt, int lane, F&& f) {
#pragma unroll 1
    for (int t = t0; t < t1; t += dt) {
        if (plain(t)) continue;
        const f16* const x = lane < len ? row(t * len + lane) : nullptr;
        uint64_t m = __ballot(x && wild_row(x, dh));
#pragma unroll 1
        for (; m; m &= m - 1) f(t * len + (int)__builtin_ctzll(m));
    }
}

// The tiles [t0, t1) of a list into the states of a wave's queries: 4 waves share
// each tile of K and V, in one of two LDS stages (smem: 4 tiles), filled by
// LDS-direct loads (load(t, K, V), the first one on its way already) while the
// tile before is used; one barrier a tile.  plain(t): every query of the
// workgroup sees the whole tile; seen(q)(entry): whether the lane's query of block
// q does.  Non-zero: rows were left out (clean_rows).
template <bool FAR, int DH, int QB, class Dma, class Load, class Plain, class Seen>
DEV uint32_t walk_tiles(Softmax<DH, QB>& sm, const half8 (&qf)[QB][Geo<DH>::KS], float c2, f16* smem, const Dma& dma, int t0, int t1, Load&& load,
                          Plain&& plain, Seen&& seen) {
    constexpr int KS = Geo<DH>::KS, DT = Geo<DH>::DT, TILE = BK * Geo<DH>::W;
    const int g = dma.lane >> 4;
    const Frag<DH> fr(dma.lane);
    uint32_t wild = 0;
    for (int t = t0; t < t1; ++t) {
        f16* const sk = smem + ((t - t0) & 1) * 2 * TILE;
        f16* const sv = sk + TILE;
        const bool whole = plain(t);  // workgroup-uniform
        wait_loads();  // this wave's part of tile t is in LDS
        if (!whole) wild |= clean_rows(dma, sv);
        __syncthreads();  // everyone's; the other stage is free
        if (t + 1 < t1) {
            f16* const nx = smem + ((t + 1 - t0) & 1) * 2 * TILE;
            load(t + 1, nx, nx + TILE);
        }
        using Rows = Ring<4 * KS, 3>;
        using Cols = Ring<2 * DT, 2>;
        floatx4 s[4][QB];
        half8 kf[Rows::SLOTS], vf[Cols::SLOTS];
        auto row = [&](auto i, auto slot) { kf[slot] = fr.row(sk, 16 * (i / KS), i % KS); };
        auto col = [&](auto i, auto slot) { vf[slot] = fr.col(sv, 32 * (i / DT), i % DT); };
        Rows::template start<1>(row);
        Rows::template run<QB, 1>(row, [&](auto i, auto slot) {
#pragma unroll
            for (int q = 0; q < QB; ++q)
                s[i / KS][q] = mfma16(kf[slot], qf[q][i % KS], i % KS ? s[i / KS][q] : floatx4{0.0f, 0.0f, 0.0f, 0.0f});
        });
        if (!whole) {
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                const auto see = seen(q);
#pragma unroll
                for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[kb][q][j] = see(t * BK + 16 * kb + 4 * g + j) ? s[kb][q][j] : -INFINITY;
            }
        }
        half8 p[2][QB];
        sm.template probs<FAR, 4>(s, c2, p);
        Cols::template start<2>(col);
        Cols::template run<QB, 2>(col, [&](auto i, auto slot) {
#pragma unroll
            for (int q = 0; q < QB; ++q) sm.o[i % DT][q] = mfma16(vf[slot], p[i / DT][q], sm.o[i % DT][q]);
        });
    }
    return wild;
}
// The same, and again where scores are FAR: then sm.far is true for the whole
// workgroup.  f(): rows that were left out, to be added.
template <int DH, int QB, class Dma, class Load, class Plain, class Seen, class F>
DEV void attend_tiles(Softmax<DH, QB>& sm, const half8 (&qf)[QB][Geo<DH>::KS], float c2, f16* smem, const Dma& dma, int t0, int t1, Load&& load,
                      Plain&& plain, Seen&& seen, F&& f) {
    const uint32_t wild = walk_tiles<false>(sm, qf, c2, smem, dma, t0, t1, load, plain, seen);
    if (!__syncthreads_or(wild | (sm.far ? 1u : 0u))) return;
    if (__syncthreads_or(sm.far)) {
        sm.reset();
        load(t0, smem, smem + BK * Geo<DH>::W);
        walk_tiles<true>(sm, qf, c2, smem, dma, t0, t1, load, plain, seen);
        sm.far = true;
    }
    if (__syncthreads_or(wild)) f();
}

// Every NW-th step of 32 entries into the states of 16 queries, by one wave: K
// goes from memory straight into A operands, V through the wave's own LDS slot
// (32 rows), no barrier; the next step's loads are in flight meanwhile.
template <int DH, int NW>
struct Steps {
    using G = Geo<DH>;
    static constexpr int KS = G::KS, DT = G::DT, W = G::W, VPER = 32 * G::CPR / 64;
    f16* const slot;
    const int lane;
    const Frag<DH> fr;
    u32x4 kr[2][KS], vr[VPER];
    DEV Steps(f16* s, int l) : slot(s), lane(l), fr(l) {}
    template <class Row>
    DEV void load_k(int step, Row&& k_row, int dh) {
        const int l16 = lane & 15, g = lane >> 4;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const f16* src = k_row(32 * step + 16 * kb + l16);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                kr[kb][ks] = u32x4{0u, 0u, 0u, 0u};
                if (32 * ks + 8 * g < dh) kr[kb][ks] = *reinterpret_cast<const u32x4*>(src + 32 * ks + 8 * g);
            }
        }
    }
    template <class Row>
    DEV void load_v(int step, Row&& v_row, int dh) {
#pragma unroll
        for (int i = 0; i < VPER; ++i) {
            const int row = (lane + 64 * i) / G::CPR, chunk = (lane + 64 * i) % G::CPR ^ swz<W>(row);
            vr[i] = u32x4{0u, 0u, 0u, 0u};
            if (chunk * 8 < dh) vr[i] = *reinterpret_cast<const u32x4*>(v_row(32 * step + row) + chunk * 8);
        }
    }
    template <class KRow, class VRow>
    DEV void load(int step, KRow&& k_row, VRow&& v_row, int dh) {
        load_k(step, k_row, dh);
        load_v(step, v_row, dh);
    }
    // from `step`, which is loaded, on; k_row, v_row: an entry's row, past the list's end any row that is there.  Again
    // where scores are FAR.
    template <class KRow, class VRow, class Plain, class Seen>
    DEV uint64_t run(Softmax<DH, 1>& sm, const half8 (&qf)[1][KS], float c2, int step, int end, KRow&& k_row, VRow&& v_row, int dh, Plain&& plain,
                     Seen&& seen) {
        const uint64_t wild = walk<false>(sm, qf, c2, step, end, k_row, v_row, dh, plain, seen);
        if (__builtin_expect(sm.far, 0)) {  // code behind the kernel's (between the loop and what follows: 16 tokens of a head of 256 10.8 us, 11.2)
            sm.reset();
            load(step, k_row, v_row, dh);
            walk<true>(sm, qf, c2, step, end, k_row, v_row, dh, plain, seen);
            sm.far = true;
        }
        return wild;
    }
    template <bool FAR, class KRow, class VRow, class Plain, class Seen>
    DEV uint64_t walk(Softmax<DH, 1>& sm, const half8 (&qf)[1][KS], float c2, int step, int end, KRow&& k_row, VRow&& v_row, int dh, Plain&& plain,
                      Seen&& seen) {
        const int g = lane >> 4;
        uint64_t wild = 0;
        for (; step < end; step += NW) {
            const bool whole = plain(step);
            if (!whole) {
#pragma unroll
                for (int i = 0; i < VPER; ++i) {
                    const uint64_t hit = __ballot(is_wild(wild2(as_half8(vr[i]), half2_t{(f16)0.0f, (f16)0.0f})));
                    if (hit >> (lane / G::CPR * G::CPR) & ((1ull << G::CPR) - 1)) vr[i] = u32x4{0u, 0u, 0u, 0u};
                    wild |= hit;
                }
            }
#pragma unroll
            for (int i = 0; i < VPER; ++i) *reinterpret_cast<u32x4*>(slot + (lane + 64 * i) * 8) = vr[i];
            if (step + NW < end) load_v(step + NW, v_row, dh);
            half8 vf[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) vf[d] = fr.col(slot, 0, d);
            floatx4 s[2][1];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                s[kb][0] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s[kb][0] = mfma16(as_half8(kr[kb][ks]), qf[0][ks], s[kb][0]);
            }
            if (step + NW < end) load_k(step + NW, k_row, dh);
            if (!whole) {
                const auto see = seen(0);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[kb][0][j] = see(32 * step + 16 * kb + 4 * g + j) ? s[kb][0][j] : -INFINITY;
            }
            half8 p[1][1];
            sm.template probs<FAR, 2>(s, c2, p);
#pragma unroll
            for (int d = 0; d < DT; ++d) sm.o[d][0] = mfma16(vf[d], p[0][0], sm.o[d][0]);
        }
        return wild;
    }
};

// Bytes of LDS that NW waves of Steps and merge_waves take
template <int DH, int NW>
constexpr int steps_bytes() {
    constexpr int SLOT = 32 * Geo<DH>::W * 2, STATE = 16 * (DH + 4) * 4;  // of a wave's V, then of its state
    return NW * (SLOT > STATE ? SLOT : STATE);
}
// The waves' states of 16 queries as one: store(query, value, m, l, four values of
// O^T) for all of them
template <int DH, int NW, class Store>
DEV void merge_waves(const Softmax<DH, 1>& sm, float c2, char* smem, float (*sm_m)[16], float (*sm_l)[16], int lane, int wave, Store&& store) {
    constexpr int DT = Geo<DH>::DT, OW = DH + 4;
    const int l16 = lane & 15, g = lane >> 4;
    __syncthreads();  // the slots have been read
    float* const st = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<floatx4*>(st + (wave * 16 + l16) * OW + 16 * d + 4 * g) = sm.o[d][0];
    const float l = query_sum(sm.l[0]);
    if (g == 0) {
        sm_m[wave][l16] = sm.m[0];
        sm_l[wave][l16] = l;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * (DH / 4); e += 64 * NW) {
        const int q = e / (DH / 4), d = e % (DH / 4) * 4;
        float m = -INFINITY, ls = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, sm_m[w][q]);
        floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = state_weight(sm_m[w][q], m, c2);
            ls += f * sm_l[w][q];
            o += f * *reinterpret_cast<const floatx4*>(st + (w * 16 + q) * OW + d);
        }
        store(q, d, m, ls, o);
    }
}

// The DH that serves a head size, from `least` on
uint64_t head_width(int dh, int least) {
    return dh <= 32 && least <= 32 ? 32 : dh <= 64 ? 64 : dh <= 96 ? 96 : dh <= 128 ? 128 : 256;
}
template <class F>
hipError_t by_head64(int dh, F&& f) {
    switch (head_width(dh, 64)) {
        case 64: f(std::integral_constant<int, 64>{}); break;
        case 96: f(std::integral_constant<int, 96>{}); break;
        case 128: f(std::integral_constant<int, 128>{}); break;
        default: f(std::integral_constant<int, 256>{}); break;
    }
    return hipGetLastError();
}
template <class F>
hipError_t by_head(int dh, F&& f) {
    if (head_width(dh, 32) > 32) return by_head64(dh, f);
    f(std::integral_constant<int, 32>{});
    return hipGetLastError();
}

}  // namespace
}  // namespace evkhip

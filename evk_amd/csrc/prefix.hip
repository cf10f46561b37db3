// Grouped-query attention of a batch whose sequences share a prefix: its keys
// and values lie in memory once, behind them each sequence has rows of its own
// (no counterpart in the reference, which recomputes every sequence whole).
//
// Query t of sequence b stands at own row p = p0 + t; it sees all P rows of the
// prefix and the own rows j <= p.
//   S = Q [Kp; K]^T / sqrt(Dh), O = softmax(S) [Vp; V]
// One that sees nothing (P = 0, p < 0) has O = 0, LSE = -inf; one whose scores
// are all -inf has no softmax: O = NaN, LSE = -inf.  Own rows that a query does
// not see stay out of its sums, whatever they hold.
#include "attention_tiles.h"

#include <algorithm>

namespace evkhip {

namespace {

// Own rows that query t of sequence b sees
DEV int own_rows(const PrefixArgs& a, int b, int t) {
    const int64_t p = (int64_t)(a.offsets ? a.offsets[b] : a.p0) + t;
    return (int)(p < 0 ? 0 : p < a.R ? p + 1 : a.R);
}

// ---------------------------------------------------------------------------
// One wave per query row, any head size and alignment: 64 rows of K at a time, a
// lane each, then V's columns over the lanes.  For what the MFMA kernels do not
// take; bounded by the latency of its loads (16 sequences, 8 heads over 2 of 100
// values, 1000 rows and up to 300: 120 us).
// ---------------------------------------------------------------------------
constexpr int SMAX = 256;  // largest head size

struct RowLds {
    float x[SMAX], p[64];
    const f16* v[64];
};
__global__ __launch_bounds__(64) void prefix_rows(PrefixArgs a) {
    __shared__ RowLds s;
    const int lane = threadIdx.x, dh = a.dh;
    const int64_t row = blockIdx.x;
    const int h = (int)(row % a.H), t = (int)(row / a.H % a.N), b = (int)(row / a.H / a.N), c = h / (a.H / a.KV);
    const int64_t ld = (int64_t)a.KV * dh, own = (int64_t)b * a.R * ld + (int64_t)c * dh;
    const int64_t total = (int64_t)a.P + own_rows(a, b, t);
    auto at = [&](const f16* shared, const f16* mine, int64_t j) {
        return j < a.P ? shared + j * ld + (int64_t)c * dh : mine + own + (j - a.P) * ld;
    };
    for (int d = lane; d < dh; d += 64) s.x[d] = (float)a.q[row * dh + d];
    wave_sync();
    const float c2 = a.scale * kLog2e;
    float m = -INFINITY, l = 0.0f, o[SMAX / 64] = {};  // m a score, not scaled
    for (int64_t i0 = 0; i0 < total; i0 += 64) {
        const int n = (int)min((int64_t)64, total - i0);
        const int64_t j = min(i0 + lane, total - 1);
        float sc = -INFINITY;
        if (lane < n) {
            const f16* const k = at(a.pk, a.k, j);
            sc = 0.0f;
            int d = 0;
            for (; d + 8 <= dh; d += 8) {
                const half8 x = ld_h8(k + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) sc += (float)x[e] * s.x[d + e];
            }
            for (; d < dh; ++d) sc += (float)k[d] * s.x[d];
        }
        const float m_new = fmaxf(m, wave_max(sc));
        const float keep = m == -INFINITY ? 0.0f : exp2f((m - m_new) * c2);
        const float e = lane < n ? exp2f((sc - (m_new == -INFINITY ? 0.0f : m_new)) * c2) : 0.0f;
        l = l * keep + wave_sum(e);
        m = m_new;
        s.p[lane] = e;
        s.v[lane] = at(a.pv, a.v, j);
        wave_sync();
#pragma unroll
        for (int u = 0; u < SMAX / 64; ++u) {
            const int d = lane + 64 * u;
            if (d >= dh) break;
            float v = o[u] * keep;
#pragma unroll 16
            for (int i = 0; i < n; ++i) v += s.p[i] * (float)s.v[i][d];
            o[u] = v;
        }
        wave_sync();
    }
#pragma unroll
    for (int u = 0; u < SMAX / 64; ++u)
        if (lane + 64 * u < dh) a.out[row * dh + lane + 64 * u] = (f16)(total ? o[u] / l : 0.0f);
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.H + h) * a.N + t] = total ? __builtin_fmaf(m, a.scale, log2f(l) * kLn2) : -INFINITY;
}

// ---------------------------------------------------------------------------
// MFMA kernels: head sizes that are multiples of 8 (zero-filled to DH = 32, 64,
// 96, 128 or 256), 16-byte aligned pointers.
//
// The query side of a key head is a matrix of B N G rows (G = H / KV), row r
// being query r / G (sequence r / G / N) of the group's head r % G.  Rows of all
// sequences see the same prefix, so that a tile of them reads it once.
// ---------------------------------------------------------------------------

// Where a row of the matrix lies, and what it sees
struct Rows {
    int group;
    int64_t q0;  // of head c
    DEV Rows(const PrefixArgs& a, int c) : group(a.H / a.KV), q0((int64_t)c * group) {}
    DEV int64_t row(const PrefixArgs& a, int r) const { return (int64_t)(r / group) * a.H + q0 + r % group; }  // of q
    DEV int own(const PrefixArgs& a, int r) const { return own_rows(a, r / group / a.N, r / group % a.N); }
    DEV int64_t lse(const PrefixArgs& a, int r) const {
        return ((int64_t)(r / group / a.N) * a.H + q0 + r % group) * a.N + r / group % a.N;
    }
};

// States of parts of a row's list: m, l, 2 unused, O
template <int DH>
DEV float* state_at(float* ws, int64_t row, int slots, int slot) {
    return ws + (row * slots + slot) * (DH + 4);
}

// Tiles of 64 QB rows over the prefix and, where they are one sequence's, its own
// rows behind it.  The prefix is padded to whole tiles of the list, so that a tile
// lies behind one descriptor.
//
// Bounded by the softmax's instructions beside the MFMA: 8 x 500 tokens, 16 heads
// over 4 of 128, behind 4096 rows, 142 GFLOP in 150-159 us = 890-950 TFLOP/s (a product of
// the library at 8192^3 runs at 1156).
struct TileWork {
    int per, tiles;    // rows of one sequence (B N G: all of them together, over the prefix alone), tiles of them
    int own;           // their own rows are part of the list
    int splits, slots; // parts of the list; states of a row (0: none, the output is written)
};
struct Sees {  // the entries [0, P) and [sl, last), without && (as branches they cost more)
    int P, sl, last;
    DEV bool operator()(int e) const { return (e < P) | ((e >= sl) & (e < last)); }
};
template <int DH, int QB>
DEV void tile_rows(const PrefixArgs& a, const TileWork& w, int item, float* ws, f16* smem) {
    using G = Geo<DH>;
    constexpr int KS = G::KS, DT = G::DT, TILE = BK * G::W, ROWS = 64 * QB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int split = item % w.splits, tile = w.tiles - 1 - item / w.splits % w.tiles, bc = item / w.splits / w.tiles, c = bc % a.KV, b = bc / a.KV;
    const Rows rows(a, c);
    const int R0 = b * w.per + tile * ROWS, end = (b + 1) * w.per, wr0 = R0 + wave * 16 * QB;
    const int sl = w.own ? (a.P + BK - 1) / BK * BK : a.P;  // entries before the own rows
    const int least = w.own ? __builtin_amdgcn_readfirstlane(rows.own(a, R0)) : 0;
    const int most = w.own ? __builtin_amdgcn_readfirstlane(rows.own(a, min(R0 + ROWS, end) - 1)) : 0;
    const int n = sl + most, nt = (n + BK - 1) / BK;
    const int t0 = (int)((int64_t)nt * split / w.splits), t1 = (int)((int64_t)nt * (split + 1) / w.splits);
    const uint32_t ld = (uint32_t)a.KV * a.dh * 2;
    const int64_t own0 = (int64_t)b * a.R * a.KV * a.dh + (int64_t)c * a.dh;

    TileDma<DH, BK, 4> dma{wave, lane};
    uint32_t off[TileDma<DH, BK, 4>::PER];
#pragma unroll
    for (int i = 0; i < TileDma<DH, BK, 4>::PER; ++i) off[i] = oob_or(dma.chunk(i) * 8 < a.dh, dma.row(i) * ld + dma.chunk(i) * 16);
    const auto k_row = [&](int e) { return (e < sl ? a.pk + (int64_t)c * a.dh + (int64_t)e * (ld / 2) : a.k + own0 + (int64_t)(e - sl) * (ld / 2)); };
    const auto v_row = [&](int e) { return (e < sl ? a.pv + (int64_t)c * a.dh + (int64_t)e * (ld / 2) : a.v + own0 + (int64_t)(e - sl) * (ld / 2)); };
    const auto load = [&](int t, f16* sk, f16* sv) {
        const int i0 = t * BK;
        const uint32_t span = (uint32_t)min((i0 < sl ? a.P : n) - i0, BK) * ld;  // what lies past it reads as zeros
        dma.go(wave_rsrc(k_row(i0), span), off, sk);
        dma.go(wave_rsrc(v_row(i0), span), off, sv);
    };
    if (t0 < t1) load(t0, smem, smem + TILE);

    half8 qf[QB][KS];
    int own[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int r = min(wr0 + 16 * q + l16, end - 1);
        own[q] = w.own ? rows.own(a, r) : 0;
        const f16* src = a.q + rows.row(a, r) * a.dh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qf[q][ks] = half8{};
            if (32 * ks + 8 * g < a.dh) qf[q][ks] = *reinterpret_cast<const half8*>(src + 32 * ks + 8 * g);
        }
    }
    const float c2 = a.scale * kLog2e;
    Softmax<DH, QB> sm;
    const auto plain = [&](int t) {
        const int i1 = (t + 1) * BK;
        return (i1 <= a.P) | ((i1 > sl) & (i1 <= sl + least));
    };
    const auto seen = [&](int q) { return Sees{a.P, sl, sl + own[q]}; };
    attend_tiles(sm, qf, c2, smem, dma, t0, t1, load, plain, seen, [&] {
        each_wild(plain, [&](int e) { return (((e < a.P) | (e >= sl)) & (e < n)) ? v_row(e) : nullptr; }, a.dh, BK, t0, t1, 1, lane, [&](int e) {
            bool sees[QB];
#pragma unroll
            for (int q = 0; q < QB; ++q) sees[q] = Sees{a.P, sl, sl + own[q]}(e);
            sm.add_row(sees, k_row(e), v_row(e), qf, a.dh, c2, g, sm.far);
        });
    });
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int r = wr0 + 16 * q + l16;
        const float l = query_sum(sm.l[q]);
        if (r >= end) continue;
        if (w.slots) {
            float* dst = state_at<DH>(ws, rows.row(a, r), w.slots, split);
#pragma unroll
            for (int d = 0; d < DT; ++d) *reinterpret_cast<floatx4*>(dst + 4 + 16 * d + 4 * g) = sm.o[d][q];
            if (g == 0) dst[0] = sm.m[q], dst[1] = l;
            continue;
        }
        const bool none = a.P + own[q] == 0;
        const float inv = none ? 0.0f : 1.0f / l;
        f16* dst = a.out + rows.row(a, r) * a.dh;
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (16 * d + 4 * g < a.dh)
                *reinterpret_cast<uint2*>(dst + 16 * d + 4 * g) =
                    uint2{pack_h2(sm.o[d][q][0] * inv, sm.o[d][q][1] * inv), pack_h2(sm.o[d][q][2] * inv, sm.o[d][q][3] * inv)};
        if (a.lse && g == 0) a.lse[rows.lse(a, r)] = none ? -INFINITY : sm.lse(sm.m[q], l, a.scale);
    }
}
template <int DH, int QB>
__global__ __launch_bounds__(256, DH > 128 ? 1 : 2) void prefix_tiles(PrefixArgs a, TileWork w, float* ws) {
    __shared__ __attribute__((aligned(1024))) f16 smem[4 * BK * Geo<DH>::W];
    // an XCD takes items that follow each other, which share rows of K and V
    tile_rows<DH, QB>(a, w, xcd_tile(blockIdx.x, gridDim.x), ws, smem);
}

// 16 rows of one sequence, the waves' steps over its own rows and, where nobody
// else sees to it, the prefix before them: a few queries use few of a product's
// columns, and nothing waits but for memory.  One token, 32 heads over 8 of 128
// behind 16000 rows: 17.9 us with the join = 3.7 TB/s; 64 sequences of 12 over 4 of
// 64, 300 rows and up to 300: 8.0.
struct StepWork {
    int tiles;
    int prefix;               // rows of the prefix in the list: P or 0
    int splits, slots, slot;  // parts of the list; states of a row (0: none) and this list's first
    int groups;               // parts of all lists
};
template <int DH, int NW>
DEV void step_rows(const PrefixArgs& a, const StepWork& w, int item, float* ws, char* smem, float (*sm_m)[16], float (*sm_l)[16]) {
    using G = Geo<DH>;
    constexpr int KS = G::KS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    // Parts go round the XCDs, so that each gets as many long ones, a part's tiles on one of them (sequences in turn on an XCD:
    // 64 tokens, 32 heads over 8 of 128 behind 4096 rows, up to 1024 of their own, longest first: 52, now 43).
    const int part = item / 8 / w.tiles * 8 + item % 8, tile = item / 8 % w.tiles;
    const int split = part % w.splits, bc = part / w.splits, c = bc % a.KV, b = bc / a.KV;
    if (part >= w.groups) return;
    const Rows rows(a, c);
    const int per = a.N * rows.group, R0 = b * per + tile * 16, end = (b + 1) * per, pre = w.prefix;
    const int least = __builtin_amdgcn_readfirstlane(rows.own(a, R0)), most = __builtin_amdgcn_readfirstlane(rows.own(a, min(R0 + 16, end) - 1));
    const int n = pre + most, steps = (n + 31) / 32;
    const int c0 = (int)((int64_t)steps * split / w.splits), c1 = (int)((int64_t)steps * (split + 1) / w.splits), first = c0 + wave;
    const int64_t ld = (int64_t)a.KV * a.dh, own0 = (int64_t)b * a.R * ld + (int64_t)c * a.dh;
    const auto k_row = [&](int e) {
        e = min(e, n - 1);
        return e < pre ? a.pk + (int64_t)c * a.dh + e * ld : a.k + own0 + (e - pre) * ld;
    };
    const auto v_row = [&](int e) {
        e = min(e, n - 1);
        return e < pre ? a.pv + (int64_t)c * a.dh + e * ld : a.v + own0 + (e - pre) * ld;
    };
    Steps<DH, NW> walk(reinterpret_cast<f16*>(smem) + wave * 32 * G::W, lane);
    if (first < c1) walk.load(first, k_row, v_row, a.dh);
    const int r = min(R0 + l16, end - 1), last = pre + rows.own(a, r);
    half8 qf[1][KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qf[0][ks] = half8{};
        if (32 * ks + 8 * g < a.dh) qf[0][ks] = *reinterpret_cast<const half8*>(a.q + rows.row(a, r) * a.dh + 32 * ks + 8 * g);
    }
    const float c2 = a.scale * kLog2e;
    Softmax<DH, 1> sm;
    const auto plain = [&](int step) { return 32 * step + 32 <= pre + least; };
    const auto seen = [&](int) { return Sees{last, 0, 0}; };
    const uint64_t wild = walk.run(sm, qf, c2, first, c1, k_row, v_row, a.dh, plain, seen);
    if (wild)
        each_wild(plain, [&](int e) { return e < n ? v_row(e) : nullptr; }, a.dh, 32, first, c1, NW, lane, [&](int e) {
            const bool sees[1] = {e < last};
            sm.add_row(sees, k_row(e), v_row(e), qf, a.dh, c2, g, sm.far);
        });
    merge_waves<DH, NW>(sm, c2, smem, sm_m, sm_l, lane, wave, [&](int q, int d, float m, float l, const floatx4& o) {
        const int row = R0 + q;
        if (row >= end) return;
        if (w.slots) {
            float* dst = state_at<DH>(ws, rows.row(a, row), w.slots, w.slot + split);
            *reinterpret_cast<floatx4*>(dst + 4 + d) = o;
            if (d == 0) dst[0] = m, dst[1] = l;
            return;
        }
        const bool none = pre + rows.own(a, row) == 0;
        const float inv = none ? 0.0f : 1.0f / l;
        if (d < a.dh)
            *reinterpret_cast<uint2*>(a.out + rows.row(a, row) * a.dh + d) = uint2{pack_h2(o[0] * inv, o[1] * inv), pack_h2(o[2] * inv, o[3] * inv)};
        if (a.lse && d == 0) a.lse[rows.lse(a, row)] = none ? -INFINITY : sm.lse(m, l, a.scale);
    });
}
template <int DH>
struct StepGeo {
    static constexpr int NW = DH <= 128 ? 8 : 4;  // waves; 256 values take the registers of two
};
template <int DH>
__global__ __launch_bounds__(64 * StepGeo<DH>::NW, StepGeo<DH>::NW / 4) void prefix_steps(PrefixArgs a, StepWork w, float* ws) {
    constexpr int NW = StepGeo<DH>::NW;
    __shared__ __attribute__((aligned(16))) char smem[steps_bytes<DH, NW>()];
    __shared__ float sm_m[NW][16], sm_l[NW][16];
    step_rows<DH, NW>(a, w, blockIdx.x, ws, smem, sm_m, sm_l);
}

// The prefix by tiles and the own rows by steps in one launch: the former wait for
// their products, the latter for memory.  Each XCD starts its part of the tiles
// first, which take the same time all, and fills up with own rows, which end when
// they end.  64 tokens, 32 heads over 8 of 128 behind 8192 rows, up to 1024 of their
// own: 45-48 us for 34 MB of prefix, whose products are 8.6 GFLOP, and 134 MB of own
// rows, which alone take 31-38.  4 tokens each behind 4096 rows, with the join: 42, in
// launches of their own 52.
template <int DH, int QB>
__global__ __launch_bounds__(256, DH > 128 ? 1 : 2) void prefix_mixed(PrefixArgs a, TileWork tw, int wide, StepWork sw, float* ws) {
    constexpr int TILES = 4 * BK * Geo<DH>::W * 2, STEPS = steps_bytes<DH, 4>();
    __shared__ __attribute__((aligned(1024))) char smem[TILES > STEPS ? TILES : STEPS];
    __shared__ float sm_m[4][16], sm_l[4][16];
    const int tiles = (wide + 7) / 8 * 8, tile = xcd_tile(blockIdx.x, tiles);
    if ((int)blockIdx.x >= tiles) step_rows<DH, 4>(a, sw, blockIdx.x - tiles, ws, smem, sm_m, sm_l);
    else if (tile < wide) tile_rows<DH, QB>(a, tw, tile, ws, reinterpret_cast<f16*>(smem));
}

// The states of a row, added in order by one wave: groups of DH / 4 lanes take
// every HPW-th of them, 16 bytes a lane, all requested before the weights are
// known.  2048 rows of 14 states: 5.0 us, a launch and two latencies.
constexpr int JOIN_MOST = 64;  // a lane weighs one
template <int DH>
__global__ __launch_bounds__(256) void prefix_join(PrefixArgs a, int slots, int64_t rows, const float* ws) {
    constexpr int LPS = DH <= 32 ? 8 : DH <= 64 ? 16 : DH <= 128 ? 32 : 64, HPW = 64 / LPS, AHEAD = 8;
    const int lane = threadIdx.x & 63, d = lane % LPS * 4, part = lane / LPS;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const float* src = ws + row * slots * (DH + 4);
    const bool is = lane < slots;
    const float mine = is ? src[lane * (DH + 4)] : -INFINITY, mine_l = is ? src[lane * (DH + 4) + 1] : 0.0f;
    auto load = [&](int s) {
        return *reinterpret_cast<const floatx4*>(src + min(s, slots - 1) * (DH + 4) + 4 + min(d, DH - 4));
    };
    floatx4 ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) ahead[i] = load(part + HPW * i);
    const float m = wave_top(mine), f = state_weight(mine, m, a.scale * kLog2e);
    const float l = wave_add(is ? f * mine_l : 0.0f);
    floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < slots; s0 += HPW * AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int s = s0 + part + HPW * i;
            const float fs = __shfl(f, min(s, 63), 64);
            if (s < slots) o += fs * ahead[i];
            ahead[i] = load(s + HPW * AHEAD);
        }
    }
#pragma unroll
    for (int k = LPS; k < 64; k *= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], k, 64);
    const int h = (int)(row % a.H), t = (int)(row / a.H % a.N), b = (int)(row / a.H / a.N);
    const bool none = a.P + own_rows(a, b, t) == 0;
    const float inv = none ? 0.0f : 1.0f / l;
    if (part == 0 && d < a.dh)
        *reinterpret_cast<uint2*>(a.out + row * a.dh + d) = uint2{pack_h2(o[0] * inv, o[1] * inv), pack_h2(o[2] * inv, o[3] * inv)};
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.H + h) * a.N + t] = none ? -INFINITY : Softmax<DH, 1>::lse(m, l, a.scale);
}

bool mfma_ok(const PrefixArgs& a) {
    for (const void* p : {(const void*)a.q, (const void*)a.pk, (const void*)a.pv, (const void*)a.k, (const void*)a.v, (const void*)a.out})
        if (!aligned16(p)) return false;
    // a tile's rows behind one descriptor
    return a.dh % 8 == 0 && (int64_t)a.KV * a.dh * 2 * (BK + 1) < INT32_MAX;
}

// How a shape runs.  us in the comments: one side of a rule and the other.
struct Plan {
    enum { TILES, STEPS, SHARED } kind;
    int qb;          // query blocks of a wave in tiles
    TileWork tiles;  // TILES: all; SHARED: the prefix
    StepWork steps;  // STEPS: all; SHARED: the own rows
    int slots;
    int64_t wide, few;  // workgroups of tiles and of steps
};
Plan plan_for(int64_t B, int64_t N, int64_t P, int64_t R, int64_t H, int64_t KV, int dh) {
    Plan p{};
    const int64_t per = N * (H / KV), heads = B * KV, all = B * per;
    auto ceil = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    auto some = [](int64_t most, int64_t a, int64_t b) { return std::max<int64_t>(1, std::min({most, a, b})); };
    // Prompts: tiles of one sequence's rows over the prefix and its own.  From 256 rows of a key head on (8 sequences of 120
    // tokens, 16 heads over 4 of 128, behind 4096 rows: 62, the other way 89), from 128 on where that gives every CU a
    // tile (32 of 50 tokens behind 1000 rows 32 and 58; 8 of 40, 8 over 2 of 64, behind 200 rows, 48 tiles: 11.2 and 6.0;
    // 64 rows each, 64 sequences behind 8192 rows: 269 and 184).
    if (per >= 256 || (per >= 128 && heads * ceil(per, 64) >= 256)) {
        p.kind = Plan::TILES;
        p.qb = dh <= 128 && heads * ceil(per, 128) > 256 ? 2 : 1;  // as in window_attention
        const int64_t tiles = ceil(per, 64 * p.qb), groups = heads * tiles;
        // parts of the list where CUs are idle: of 4 tiles and more, of 16 where a quarter is busy (10 tiles over 4200 rows:
        // 15.7, with 16 tiles a part 21; 104 over 600 rows, parts of 8 15.1, none 10.3; 256 over 300: 21.6 and 8.5)
        const int64_t splits = groups >= 256 ? 1 : some(JOIN_MOST, 512 / groups, ceil(P + R, (groups >= 64 ? 16 : 4) * BK));
        p.slots = splits > 1 ? (int)splits : 0;
        p.tiles = {(int)per, (int)tiles, 1, (int)splits, p.slots};
        p.wide = groups * splits;
        return p;
    }
    const int64_t tiles = ceil(per, 16), groups = heads * tiles;
    // A few rows: each sequence's steps over both, in one workgroup while its waves take no more than four each, else in
    // parts with a second launch to join them; while reading the prefix again for each costs less than sharing it: 64 MB
    // against a second launch (64 sequences, 12 heads over 4 of 64, 300 rows, 19 MB: 7.4 and 10.4; 32 over 8 of 128, 500 rows,
    // 129 MB: 28.8 and 23.4), 4 MB where there is one anyway (16 sequences of 8 over 1 of 64, 4096 rows, 16 MB: 9.6 and 9.3;
    // 4 of 32 over 8 of 128, 16000 rows, 197 MB: 45 and 22).
    const int64_t steps = ceil(P + R, 32), waves = dh <= 128 ? 8 : 4;
    const bool alone = steps <= 4 * waves;
    if (B == 1 || (double)(B - 1) * P * KV * dh * 4 < (alone ? 64 << 20 : 4 << 20)) {
        p.kind = Plan::STEPS;
        const int64_t splits = alone ? 1 : some(JOIN_MOST, 256 / groups, ceil(steps, waves));
        p.slots = splits > 1 ? (int)splits : 0;
        p.steps = {(int)tiles, (int)P, (int)splits, p.slots, 0, (int)(heads * splits)};
        p.few = ceil(heads * splits, 8) * 8 * tiles;
        return p;
    }
    // The prefix for all sequences at once, by tiles of 64 rows, of 128 where those are enough to keep the products busy
    // (256 rows of 8 heads over 8192 rows 52 and 60; 64 rows over 2048 13.4 and 11.6); of the latter 192 workgroups beside the
    // own rows, up to two a CU where each would have more than 18 tiles of the prefix (64 x 8
    // tokens, 32 heads over 8 of 128, 8192 rows: 167 and 129; 16 x 40, 16 over 4, 4096 rows: 53 and 44; 18 or 10 tiles at 64
    // tokens, 32 over 8, 16000 rows: 58 and 65).  The own rows in parts of up to 16 steps of 128 values, which end at about the
    // same time (one part 55, two 50; 256 values, 500 rows: 22 and 16).  Few rows leave the join's other states to the prefix
    // (5 tokens, 2 heads over one of 256 behind 16000 rows: 32 parts 21.1, 61 18.9).
    p.kind = Plan::SHARED;
    p.qb = dh <= 128 && KV * ceil(all, 128) * ceil(P, 512) >= 256 ? 2 : 1;
    const int64_t wide = KV * ceil(all, 64 * p.qb);
    const int64_t s2 = some(JOIN_MOST / 2, JOIN_MOST / 2, ceil(R, dh <= 128 ? 512 : 256));
    const int64_t fill = p.qb == 2 ? std::max<int64_t>(192, std::min<int64_t>(512, wide * ceil(P, BK) / 18)) : 512;
    const int64_t s1 = some(JOIN_MOST - s2, fill / wide, ceil(P, 4 * BK));
    p.slots = (int)(s1 + s2);
    p.wide = wide * s1;
    p.few = ceil(heads * s2, 8) * 8 * tiles;
    p.tiles = {(int)all, (int)(wide / KV), 0, (int)s1, p.slots};
    p.steps = {(int)tiles, 0, (int)s2, p.slots, (int)s1, (int)(heads * s2)};
    return p;
}

}  // namespace

uint64_t prefix_workspace(int B, int N, int P, int R, int H, int KV, int dh) {
    if (dh % 8) return 0;
    return (uint64_t)plan_for(B, N, P, R, H, KV, dh).slots * B * N * H * (head_width(dh, 32) + 4) * sizeof(float);
}

int prefix_forward(const PrefixArgs& a, void* ws, hipStream_t st) {
    const char* op = "prefix_attention";
    const int64_t rows = (int64_t)a.B * a.N * a.H;
    hipError_t e;
    if (!mfma_ok(a)) {
        const int rc = check_grid(op, rows, 64);
        if (rc != EVKHIP_OK) return rc;
        hipLaunchKernelGGL(prefix_rows, dim3((unsigned)rows), dim3(64), 0, st, a);
        e = hipGetLastError();
        return e == hipSuccess ? EVKHIP_OK : check_hip(e, "prefix_attention launch");
    }
    const Plan p = plan_for(a.B, a.N, a.P, a.R, a.H, a.KV, a.dh);
    const int64_t groups = p.kind == Plan::SHARED ? (p.wide + 7) / 8 * 8 + p.few : p.wide + p.few;
    const dim3 grid((unsigned)groups);
    int rc = check_grid(op, groups, p.kind == Plan::STEPS ? 512 : 256);
    if (rc == EVKHIP_OK && p.slots) rc = check_grid(op, (rows + 3) / 4, 256);
    if (rc != EVKHIP_OK) return rc;
    float* const part = (float*)ws;
    e = by_head(a.dh, [&](auto dhc) {
        constexpr int DH = decltype(dhc)::value;
        auto with = [&](auto qb) {
            constexpr int QB = decltype(qb)::value;
            if (p.kind == Plan::SHARED)
                hipLaunchKernelGGL((prefix_mixed<DH, QB>), grid, dim3(256), 0, st, a, p.tiles, (int)p.wide, p.steps, part);
            else
                hipLaunchKernelGGL((prefix_tiles<DH, QB>), grid, dim3(256), 0, st, a, p.tiles, part);
        };
        if (p.kind == Plan::STEPS) {
            hipLaunchKernelGGL(prefix_steps<DH>, grid, dim3(64 * StepGeo<DH>::NW), 0, st, a, p.steps, part);
        } else if constexpr (DH > 128) {
            with(std::integral_constant<int, 1>{});
        } else {
            if (p.qb == 2) with(std::integral_constant<int, 2>{});
            else with(std::integral_constant<int, 1>{});
        }
        if (p.slots) hipLaunchKernelGGL(prefix_join<DH>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, p.slots, rows, (const float*)part);
    });
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "prefix_attention launch");
}

}  // namespace evkhip

// Grouped-query attention over a sliding window and the first tokens (sinks),
// forward, backward and for single tokens (no counterpart in the reference,
// whose attention sees every earlier position).
//
// Query t of sequence b stands at position p = p0 + t and sees the rows
//   [0, s) and [lo, hi)   with hi = min(p + 1, rows), lo = max(0, p - W + 1),
//                              s = min(sinks, lo)
// of its K and V; a query that sees nothing (p < 0) has O = 0, LSE = -inf.  One
// whose scores are all -inf has no softmax: O = NaN, LSE = -inf.
//   S = Q K^T / sqrt(Dh), P = exp(S - LSE), O = P V
//   backward: D = rowsum(dO * O), dS = P (dO V^T - D),
//             dQ = dS K / sqrt(Dh), dK = dS^T Q / sqrt(Dh), dV = P^T dO,
//             dK and dV summed over the heads that share the row.
//
// Rows that a query does not see are never read for it, so that whatever they
// hold (stale cache rows, infinities, NaN) stays out of its sums.
#include "attention_tiles.h"

#include <algorithm>

namespace evkhip {

namespace {

// The rows that a query at position p sees.
struct Span {
    int lo, hi, s;
    DEV int count() const { return s + hi - lo; }
    DEV int row(int i) const { return i < s ? i : lo + (i - s); }
};
DEV Span span_of(int p, const WindowArgs& a) {
    Span v;
    v.hi = p < 0 ? 0 : min(p, a.R - 1) + 1;
    v.lo = min(max(0, p - a.window + 1), v.hi);
    v.s = min(a.sinks, v.lo);
    return v;
}
// Position of query t of sequence b, -1 for any that sees nothing.  Windows
// longer than any cache (R <= 2^30 = WINDOW_MOST) run as ones of 2^30 rows, with
// positions moved down by the difference (`far`) where the window starts past
// row 0, so that neither a position nor the end of its window passes 32 bits;
// other positions past 2^31 - 1 see what that one sees, the sinks.
DEV int position_of(const WindowArgs& a, int b, int t) {
    int64_t p = (int64_t)(a.offsets ? a.offsets[b] : a.p0) + t;
    if (a.far) p = max(min(p, (int64_t)a.R - 1), p - a.far);
    return (int)(p < 0 ? -1 : p < INT32_MAX ? p : INT32_MAX);
}

// ---------------------------------------------------------------------------
// One wave per query row (or per K, V row), any head size and alignment.
// Latency-bound chains of scalar loads: the path of head sizes and pointers
// that the MFMA kernels do not take (1000 queries of 8 heads over 2 of 100
// values, window 512: 187 us, backward 3.7 ms).
// ---------------------------------------------------------------------------
constexpr int SMAX = 256;  // largest head size

DEV float dot_row(const f16* x, const float* y, int n) {
    float v = 0.0f;
    for (int i = 0; i < n; ++i) v += (float)x[i] * y[i];
    return v;
}

// LDS of a wave that works row by row
struct RowLds {
    float x[SMAX], y[SMAX], p[64], q[64];
    int64_t j[64];
};
// O and LSE of query row `row` = ((b N) + t) H + h
DEV void fwd_row(const WindowArgs& a, int64_t row, RowLds& s, int lane) {
    const int dh = a.dh, h = (int)(row % a.H), t = (int)(row / a.H % a.N), b = (int)(row / a.H / a.N);
    const int64_t kv_ld = (int64_t)a.KV * dh;
    const int64_t kv0 = (int64_t)b * a.R * kv_ld + (int64_t)(h / (a.H / a.KV)) * dh;
    const Span sp = span_of(position_of(a, b, t), a);
    wave_sync();
    for (int d = lane; d < dh; d += 64) s.x[d] = (float)a.q[row * dh + d];
    wave_sync();
    const float c2 = a.scale * kLog2e;
    float m = -INFINITY, l = 0.0f, o[SMAX / 64] = {};  // m a score, not scaled
    for (int i0 = 0; i0 < sp.count(); i0 += 64) {
        const int n = min(64, sp.count() - i0);
        const int64_t j = sp.row(min(i0 + lane, sp.count() - 1)) * kv_ld;
        const float sc = lane < n ? dot_row(a.k + kv0 + j, s.x, dh) : -INFINITY;
        const float m_new = fmaxf(m, wave_max(sc));
        const float keep = m == -INFINITY ? 0.0f : exp2f((m - m_new) * c2);
        const float e = lane < n ? exp2f((sc - (m_new == -INFINITY ? 0.0f : m_new)) * c2) : 0.0f;
        l = l * keep + wave_sum(e);
        m = m_new;
        s.p[lane] = e;
        s.j[lane] = j;
        wave_sync();
#pragma unroll
        for (int u = 0; u < SMAX / 64; ++u) {
            const int d = lane + 64 * u;
            if (d >= dh) break;
            float v = o[u] * keep;
            for (int i = 0; i < n; ++i) v += s.p[i] * (float)a.v[kv0 + s.j[i] + d];
            o[u] = v;
        }
        wave_sync();
    }
#pragma unroll
    for (int u = 0; u < SMAX / 64; ++u)
        if (lane + 64 * u < dh) a.out[row * dh + lane + 64 * u] = (f16)(sp.count() ? o[u] / l : 0.0f);
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.H + h) * a.N + t] = sp.count() ? __builtin_fmaf(m, a.scale, log2f(l) * kLn2) : -INFINITY;
}

// dQ of one query row
DEV void dq_row(const WindowArgs& a, int64_t row, RowLds& s, int lane) {
    const int dh = a.dh, h = (int)(row % a.H), t = (int)(row / a.H % a.N), b = (int)(row / a.H / a.N);
    const int64_t kv_ld = (int64_t)a.KV * dh;
    const int64_t kv0 = (int64_t)b * a.R * kv_ld + (int64_t)(h / (a.H / a.KV)) * dh;
    const Span sp = span_of(position_of(a, b, t), a);
    float dsum = 0.0f;
    wave_sync();
    for (int d = lane; d < dh; d += 64) {
        s.x[d] = (float)a.q[row * dh + d];
        s.y[d] = (float)a.dO[row * dh + d];
        dsum += s.y[d] * (float)a.o[row * dh + d];
    }
    dsum = wave_sum(dsum);
    wave_sync();
    const float lse2 = a.lse[((int64_t)b * a.H + h) * a.N + t] * kLog2e;
    float o[SMAX / 64] = {};
    for (int i0 = 0; i0 < sp.count(); i0 += 64) {
        const int n = min(64, sp.count() - i0);
        const int64_t j = sp.row(min(i0 + lane, sp.count() - 1)) * kv_ld;
        float ds = 0.0f;
        if (lane < n) {
            const float sc = dot_row(a.k + kv0 + j, s.x, dh);
            ds = exp2f(sc * a.scale * kLog2e - lse2) * (dot_row(a.v + kv0 + j, s.y, dh) - dsum);
        }
        s.p[lane] = ds;
        s.j[lane] = j;
        wave_sync();
#pragma unroll
        for (int u = 0; u < SMAX / 64; ++u) {
            const int d = lane + 64 * u;
            if (d >= dh) break;
            for (int i = 0; i < n; ++i) o[u] += s.p[i] * (float)a.k[kv0 + s.j[i] + d];
        }
        wave_sync();
    }
#pragma unroll
    for (int u = 0; u < SMAX / 64; ++u)
        if (lane + 64 * u < dh) a.out[row * dh + lane + 64 * u] = (f16)(o[u] * a.scale);
}

// dK and dV of row `at` = ((b R) + j) KV + c: over the queries that see it, 64
// (position, head) pairs at a time
DEV void dkdv_row(const WindowArgs& a, int64_t at, RowLds& s, int lane) {
    const int dh = a.dh, G = a.H / a.KV;
    const int c = (int)(at % a.KV), j = (int)(at / a.KV % a.R), b = (int)(at / a.KV / a.R);
    wave_sync();
    for (int d = lane; d < dh; d += 64) {
        s.x[d] = (float)a.k[at * dh + d];
        s.y[d] = (float)a.v[at * dh + d];
    }
    wave_sync();
    // backward: positions from 0 and as many rows as queries
    const int t_end = j < a.sinks || a.window > a.N - j ? a.N : j + a.window;
    const int64_t pairs = (int64_t)(t_end - j) * G;
    float gk[SMAX / 64] = {}, gv[SMAX / 64] = {};
    for (int64_t i0 = 0; i0 < pairs; i0 += 64) {
        const int n = (int)min((int64_t)64, pairs - i0);
        const int64_t i = min(i0 + lane, pairs - 1);
        const int t = j + (int)(i / G), h = c * G + (int)(i % G);
        const int64_t row = ((int64_t)b * a.N + t) * a.H + h;
        float p = 0.0f, ds = 0.0f;
        if (lane < n) {
            const float sc = dot_row(a.q + row * dh, s.x, dh);
            float dsum = 0.0f;
            for (int d = 0; d < dh; ++d) dsum += (float)a.dO[row * dh + d] * (float)a.o[row * dh + d];
            p = exp2f((sc * a.scale - a.lse[((int64_t)b * a.H + h) * a.N + t]) * kLog2e);
            ds = p * (dot_row(a.dO + row * dh, s.y, dh) - dsum);
        }
        s.p[lane] = p;
        s.q[lane] = ds;
        s.j[lane] = row * dh;
        wave_sync();
#pragma unroll
        for (int u = 0; u < SMAX / 64; ++u) {
            const int d = lane + 64 * u;
            if (d >= dh) break;
            for (int q = 0; q < n; ++q) {
                gk[u] += s.q[q] * (float)a.q[s.j[q] + d];
                gv[u] += s.p[q] * (float)a.dO[s.j[q] + d];
            }
        }
        wave_sync();
    }
#pragma unroll
    for (int u = 0; u < SMAX / 64; ++u) {
        const int d = lane + 64 * u;
        if (d >= dh) break;
        a.dK[at * dh + d] = (f16)(gk[u] * a.scale);
        a.dV[at * dh + d] = (f16)gv[u];
    }
}

__global__ __launch_bounds__(64) void window_fwd_rows(WindowArgs a) {
    __shared__ RowLds s;
    fwd_row(a, blockIdx.x, s, threadIdx.x);
}
__global__ __launch_bounds__(64) void window_dq_rows(WindowArgs a) {
    __shared__ RowLds s;
    dq_row(a, blockIdx.x, s, threadIdx.x);
}
__global__ __launch_bounds__(64) void window_dkdv_rows(WindowArgs a) {
    __shared__ RowLds s;
    dkdv_row(a, blockIdx.x, s, threadIdx.x);
}

// ---------------------------------------------------------------------------
// MFMA kernels: head sizes that are multiples of 8 (zero-filled to DH = 32, 64,
// 96, 128 or 256), 16-byte aligned pointers.
//
// The query side of a key head is a matrix of N G rows (G = H / KV), row r
// being query r / G of the group's head r % G: a tile's rows share the rows of
// K and V that it reads.  The rows that some query of a tile sees are numbered
// along a list: the sinks that lie before the window, then the window; a tile
// of the list is a tile of K and of V, so that a few sinks cost a few rows, no
// tile of their own.  Only the tiles at the list's start and end hold rows that
// some query does not see; the others run without a compare per score.
// ---------------------------------------------------------------------------
// The list of the rows that the queries t0 .. t1 of sequence b see.
struct List {
    int pmin, pmax;  // positions of the first and last query (-1: sees nothing)
    int lo, hi, s;   // window [lo, hi); sinks [0, s) before it, none where they meet it (then lo is 0)
    int sl, n;       // entries before the window (s, or padded to whole tiles), entries
    int first;       // entries below this one are sinks
    DEV List(const WindowArgs& a, int b, int t0, int t1, bool pad) {
        pmin = __builtin_amdgcn_readfirstlane(position_of(a, b, t0));
        pmax = __builtin_amdgcn_readfirstlane(position_of(a, b, t1));
        hi = pmax < 0 ? 0 : min(pmax, a.R - 1) + 1;
        lo = min(max(0, pmin - a.window + 1), hi);
        s = a.sinks;
        if (s >= lo) lo = s = 0;
        sl = pad ? (s + BK - 1) / BK * BK : s;
        n = sl + hi - lo;
        first = lo ? s : a.sinks;
    }
    DEV bool has(int i) const { return (i < n) & ((i < s) | (i >= sl)); }
    DEV int row(int i) const { return i < sl ? i : lo + (i - sl); }
    // every query of the tile sees the entries [i0, i0 + len)
    DEV bool plain(const WindowArgs& a, int i0, int len) const {
        const bool ends = (pmin >= 0) & (i0 + len <= n) & (i0 + len <= sl + min(pmin, a.R - 1) - lo + 1);
        return ends & ((i0 + len <= first) | (i0 >= sl + max(0, pmax - a.window + 1 - lo)));
    }
};
// The entries that one query sees: [0, first) and [lo, hi].  Written without
// && and ||: as branches they cost more than the compares, and this compiler
// dropped a masked store among them.
struct Seen {
    int lo, hi, first;
    DEV Seen(const WindowArgs& a, const List& l, int p)
        : lo(l.sl + max(0, p - a.window + 1 - l.lo)), hi(p < 0 ? -1 : l.sl + min(p, a.R - 1) - l.lo), first(l.first) {}
    DEV bool operator()(int i) const { return (i <= hi) & ((i < first) | (i >= lo)); }
};

// K and V of one sequence and key head behind buffer descriptors that start at
// a tile's first row and end with the list (what lies past them reads as
// zeros): a lane's offsets are the same in every tile.  Only a tile that holds
// both sinks and window forms its own; while a sequence's rows stay below 2 GiB
// their distance fits the offset, past that (WindowArgs::big) the sinks are
// padded to whole tiles.
template <int DH, int NWV>
struct KvTiles {
    using Dma = TileDma<DH, BK, NWV>;
    const f16 *k, *v;
    uint32_t ld;  // bytes of a row
    Dma dma;
    uint32_t off[Dma::PER];
    DEV KvTiles(const WindowArgs& a, int b, int c, int wave, int lane) : dma{wave, lane} {
        ld = (uint32_t)a.KV * a.dh * 2;
        const int64_t at = (int64_t)b * a.R * a.KV * a.dh + (int64_t)c * a.dh;
        k = a.k + at;
        v = a.v + at;
#pragma unroll
        for (int i = 0; i < Dma::PER; ++i) off[i] = oob_or(dma.chunk(i) * 8 < a.dh, dma.row(i) * ld + dma.chunk(i) * 16);
    }
    DEV void load(const List& l, int i0, f16* sk, f16* sv) const {
        const int64_t skip = (int64_t)l.row(i0) * (ld / 2);
        if (i0 < l.sl && i0 + BK > l.s) {  // sinks, then the window (or padding)
            const int gap = l.sl == l.s ? l.lo - l.sl : l.hi;
            const uint32_t rows = l.sl == l.s ? min(i0 + BK, l.n) - i0 + gap : l.s - i0;
            uint32_t o[Dma::PER];
#pragma unroll
            for (int i = 0; i < Dma::PER; ++i) {
                const bool far = i0 + dma.row(i) >= l.s;
                o[i] = oob_or((off[i] < 0x80000000u) & !(far & (l.sl != l.s)), off[i] + (far ? (uint32_t)gap * ld : 0u));
            }
            dma.go(wave_rsrc(k + skip, rows * ld), o, sk);
            dma.go(wave_rsrc(v + skip, rows * ld), o, sv);
            return;
        }
        const uint32_t span = (uint32_t)min(l.n - i0, BK) * ld;
        dma.go(wave_rsrc(k + skip, span), off, sk);
        dma.go(wave_rsrc(v + skip, span), off, sv);
    }
};

// n / d for 0 <= n < d + 2^16, d < 2^21: the quotient of n + 1/2 is at least
// 1 / (2 d) from a whole number, its error at most 2^-22.
struct SmallDiv {
    float inv;
    DEV explicit SmallDiv(int d) : inv(1.0f / (float)d) {}
    DEV int operator()(int n) const { return (int)(((float)n + 0.5f) * inv); }
};

// Forward.  Workgroup: 4 waves of 16 QB rows of one key head; K and V tiles in
// two LDS stages, filled by LDS-direct loads while the tile before is used; one
// barrier a tile.  Bound by the MFMA and the softmax's instructions beside it:
// 8192 queries of 16 heads over 4 of 128 values, window 1024 and 4 sinks, 82-84
// us call after call = 770-790 TFLOP/s of the visible pairs (whole tiles are 6%
// more; 86-90 us under a profiler, at its clocks); 97 us before the tiles' rows
// were placed without bank conflicts and read ahead of the MFMAs.
// Workgroups of eight waves, reads further ahead and a priority for waves in
// their products changed nothing.
template <int DH, int QB>
__global__ __launch_bounds__(256, DH > 128 ? 1 : 2) void window_fwd(WindowArgs a, int tiles) {
    using G = Geo<DH>;
    constexpr int KS = G::KS, DT = G::DT, TILE = BK * G::W, ROWS = 64 * QB;
    __shared__ __attribute__((aligned(1024))) f16 smem[4 * TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    // an XCD takes tiles that follow each other, which share most of their rows
    const int at = xcd_tile(blockIdx.x, gridDim.x);
    const int tile = tiles - 1 - at % tiles, bc = at / tiles, c = bc % a.KV, b = bc / a.KV;
    const int group = a.H / a.KV, NR = a.N * group, R0 = tile * ROWS, wr0 = R0 + wave * 16 * QB;
    const List list(a, b, R0 / group, (min(R0 + ROWS, NR) - 1) / group, a.big);
    const KvTiles<DH, 4> kv(a, b, c, wave, lane);
    const int nt = (list.n + BK - 1) / BK;
    if (nt > 0) kv.load(list, 0, smem, smem + TILE);

    half8 qf[QB][KS];
    int qp[QB];
    const int64_t q0 = ((int64_t)b * a.N * a.H + c * group) * a.dh;
    auto row_at = [&](int r) { return q0 + ((int64_t)(r / group) * a.H + r % group) * a.dh; };
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int r = min(wr0 + 16 * q + l16, NR - 1);
        qp[q] = position_of(a, b, r / group);
        const f16* src = a.q + row_at(r);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qf[q][ks] = half8{};
            if (32 * ks + 8 * g < a.dh) qf[q][ks] = *reinterpret_cast<const half8*>(src + 32 * ks + 8 * g);
        }
    }
    const float c2 = a.scale * kLog2e;
    Softmax<DH, QB> sm;
    const auto plain = [&](int t) { return list.plain(a, t * BK, BK); };
    attend_tiles(sm, qf, c2, smem, kv.dma, 0, nt, [&](int t, f16* sk, f16* sv) { kv.load(list, t * BK, sk, sv); }, plain,
                 [&](int q) { return Seen(a, list, qp[q]); }, [&] {
        const int64_t ld = (int64_t)a.KV * a.dh;
        each_wild(plain, [&](int e) { return list.has(e) ? kv.v + list.row(e) * ld : nullptr; }, a.dh, BK, 0, nt, 1, lane, [&](int e) {
            bool sees[QB];
#pragma unroll
            for (int q = 0; q < QB; ++q) sees[q] = Seen(a, list, qp[q])(e);
            sm.add_row(sees, kv.k + list.row(e) * ld, kv.v + list.row(e) * ld, qf, a.dh, c2, g, sm.far);
        });
    });
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int r = wr0 + 16 * q + l16;
        const float l = query_sum(sm.l[q]);
        const bool none = span_of(qp[q], a).count() == 0;
        const float inv = none ? 0.0f : 1.0f / l;
        if (r >= NR) continue;
        f16* dst = a.out + row_at(r);
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (16 * d + 4 * g < a.dh)
                *reinterpret_cast<uint2*>(dst + 16 * d + 4 * g) =
                    uint2{pack_h2(sm.o[d][q][0] * inv, sm.o[d][q][1] * inv), pack_h2(sm.o[d][q][2] * inv, sm.o[d][q][3] * inv)};
        if (a.lse && g == 0)
            a.lse[((int64_t)b * a.H + c * group + r % group) * a.N + r / group] = none ? -INFINITY : sm.lse(sm.m[q], l, a.scale);
    }
}

// Forward for few query rows (single tokens, short prompts): a workgroup takes
// 16 rows of one key head, its NW waves every NW-th step of 32 entries, each
// with a softmax of its own; the waves' states meet in LDS.  K goes from memory
// straight into A operands, V through the wave's own LDS slot, no barrier
// before the end: what counts is that every wave has its loads in flight.  A
// long list is split over workgroups as well, whose states window_join adds.
// Bound by memory: 64 sequences' tokens of 32 heads over 8 of 128 values, window
// 1024, 53 us for 254 MB = 4.8 TB/s; 32 over 8, 131072 rows 108 us = 5.0 TB/s; a
// lone token of 12 heads over 4 of 64, window 512, 6.8, a launch and two loads'
// latencies.
template <int DH>
struct SplitGeo {
    static constexpr int NW = DH <= 128 ? 8 : 4;  // waves; 256 values take the registers of two
};

template <int DH>
__global__ __launch_bounds__(64 * SplitGeo<DH>::NW, SplitGeo<DH>::NW / 4) void window_split(WindowArgs a, int tiles, int splits, float* ws) {
    using G = Geo<DH>;
    constexpr int KS = G::KS, NW = SplitGeo<DH>::NW;
    __shared__ __attribute__((aligned(16))) char smem[steps_bytes<DH, NW>()];
    __shared__ float sm_m[NW][16], sm_l[NW][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int at = xcd_tile(blockIdx.x, gridDim.x);
    const int split = at % splits, tile = at / splits % tiles, bc = at / splits / tiles, c = bc % a.KV, b = bc / a.KV;
    const int group = a.H / a.KV, NR = a.N * group, R0 = tile * 16;
    const List list(a, b, R0 / group, (min(R0 + 16, NR) - 1) / group, false);
    const int steps = (list.n + 31) / 32;
    const int c0 = (int)((int64_t)steps * split / splits), c1 = (int)((int64_t)steps * (split + 1) / splits);
    const int64_t ld = (int64_t)a.KV * a.dh, kv0 = (int64_t)b * a.R * ld + (int64_t)c * a.dh;
    const auto at_entry = [&](int e) { return kv0 + list.row(min(e, list.n - 1)) * ld; };
    Steps<DH, NW> walk(reinterpret_cast<f16*>(smem) + wave * 32 * G::W, lane);
    const auto k_row = [&](int e) { return a.k + at_entry(e); };
    const auto v_row = [&](int e) { return a.v + at_entry(e); };
    const int first = c0 + wave;
    if (first < c1) walk.load(first, k_row, v_row, a.dh);
    const int r = min(R0 + l16, NR - 1), qp[1] = {position_of(a, b, r / group)};
    const int64_t q_at = ((int64_t)b * a.N + r / group) * a.H + c * group + r % group;  // row of q
    half8 qf[1][KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qf[0][ks] = half8{};
        if (32 * ks + 8 * g < a.dh) qf[0][ks] = *reinterpret_cast<const half8*>(a.q + q_at * a.dh + 32 * ks + 8 * g);
    }
    const float c2 = a.scale * kLog2e;
    Softmax<DH, 1> sm;
    const auto plain = [&](int step) { return list.plain(a, 32 * step, 32); };
    const uint64_t wild = walk.run(sm, qf, c2, first, c1, k_row, v_row, a.dh, plain, [&](int q) { return Seen(a, list, qp[q]); });
    if (wild)
        each_wild(plain, [&](int e) { return list.has(e) ? v_row(e) : nullptr; }, a.dh, 32, first, c1, NW, lane, [&](int e) {
            const bool sees[1] = {Seen(a, list, qp[0])(e)};
            sm.add_row(sees, k_row(e), v_row(e), qf, a.dh, c2, g, sm.far);
        });
    merge_waves<DH, NW>(sm, c2, smem, sm_m, sm_l, lane, wave, [&](int q, int d, float m, float ls, const floatx4& o) {
        const int row = R0 + q;
        if (row >= NR) return;
        if (splits > 1) {
            float* dst = ws + (((int64_t)bc * NR + row) * splits + split) * (DH + 4);
            *reinterpret_cast<floatx4*>(dst + 4 + d) = o;
            if (d == 0) dst[0] = m, dst[1] = ls;
            return;
        }
        const int64_t at_row = ((int64_t)b * a.N + row / group) * a.H + c * group + row % group;
        const bool none = span_of(position_of(a, b, row / group), a).count() == 0;
        const float inv = none ? 0.0f : 1.0f / ls;
        if (d < a.dh)
            *reinterpret_cast<uint2*>(a.out + at_row * a.dh + d) = uint2{pack_h2(o[0] * inv, o[1] * inv), pack_h2(o[2] * inv, o[3] * inv)};
        if (a.lse && d == 0)
            a.lse[((int64_t)b * a.H + c * group + row % group) * a.N + row / group] = none ? -INFINITY : sm.lse(m, ls, a.scale);
    });
}

// The states of one query row's splits (at most JOIN_MOST): each thread weighs
// one, then each of NW waves adds every NW-th one's sums, and theirs are
// added in order.
constexpr int JOIN_MOST = 256;  // CUs
template <int DH>
__global__ __launch_bounds__(JOIN_MOST) void window_join(WindowArgs a, int splits, const float* ws) {
    constexpr int NW = 4, PER = DH < 64 ? 1 : DH / 64 + (DH % 64 ? 1 : 0);
    __shared__ float part[NW][64 * PER], weight[JOIN_MOST], red[2][NW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = a.H / a.KV, NR = a.N * group;
    const int row = blockIdx.x % NR, bc = blockIdx.x / NR, c = bc % a.KV, b = bc / a.KV;
    const float* src = ws + (int64_t)blockIdx.x * splits * (DH + 4);
    const float mine = tid < splits ? src[tid * (DH + 4)] : -INFINITY;
    float l = tid < splits ? src[tid * (DH + 4) + 1] : 0.0f, m = wave_max(mine);
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, red[0][w]);
    const float f = state_weight(mine, m, a.scale * kLog2e);
    weight[tid] = f;
    l = wave_sum(f * l);
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    float o[PER] = {};
#pragma unroll 8
    for (int s = wave; s < splits; s += NW)
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 64 * i < DH) o[i] += weight[s] * src[s * (DH + 4) + 4 + lane + 64 * i];
#pragma unroll
    for (int i = 0; i < PER; ++i) part[wave][lane + 64 * i] = o[i];
    __syncthreads();
    const int64_t at = ((int64_t)b * a.N + row / group) * a.H + c * group + row % group;
    const bool none = span_of(position_of(a, b, row / group), a).count() == 0;
    const float inv = none ? 0.0f : 1.0f / l;
    for (int d = tid; d < a.dh; d += 256)
        a.out[at * a.dh + d] = (f16)(((part[0][d] + part[1][d]) + (part[2][d] + part[3][d])) * inv);
    if (a.lse && tid == 0)
        a.lse[((int64_t)b * a.H + c * group + row % group) * a.N + row / group] = none ? -INFINITY : Softmax<DH, 1>::lse(m, l, a.scale);
}

// P and dS are rounded to fp16 for their products, which has 30 powers of two
// above its subnormals: P of a flat row of n is 1 / n, dS follows the lengths of
// the output's gradient.  Both therefore carry powers of two that leave the sums
// at the end.
//   dV: P is at most 1, but for the error of its exponent (scores of millions),
//       and carries 2^P_LIFT: full precision down to 2^-27.
//   dK: |dS| <= P |dO| (|V| + |O|), Cauchy-Schwarz.  Each wave bounds that by its
//       own keys' V and by the largest |dO| and |dO| |O| among its queries, which
//       window_dq leaves, and takes that bound to 2^DS_TOP: nothing overflows.
//   dQ: |dS| <= |dO| max |V_i - V_j| / 4, and V is not known before it is read: a
//       query's dO is made shorter than 1 and dS lifted by 2^DQ_LIFT.  A query
//       whose sums overflow (V longer than some hundreds, along dO) is done again
//       with DQ_STEP less, and once more: at 2^-4 no V of fp16 overflows.
// One power for both products of dK and dV, set by |dO| alone, and none for dS
// in dQ, lost bits from 16k rows on (131072 rows of one head of 64, no window: the
// later half of dQ off by 4.8 H of its norm and that of dV by 14, H half a step of
// fp16; now 0.6 both, at any length).
constexpr int P_LIFT = 13, DS_TOP = 14, DQ_LIFT = 10, DQ_STEP = 7;
constexpr int K_LEAST = -24;  // of rows that are zero, or not finite (those spoil what they are part of at any power)
typedef short short2_t __attribute__((ext_vector_type(2)));  // a pair of exponents
DEV short2_t max_xor(short2_t v, int o) {
    return __builtin_elementwise_max(v, __builtin_bit_cast(short2_t, __shfl_xor(__builtin_bit_cast(int, v), o, 64)));
}
DEV int length_exponent(float squares) {  // |x| < 2^k
    return (squares > 0.0f) & (squares < INFINITY) ? (__builtin_amdgcn_frexp_expf(squares) + 1) >> 1 : K_LEAST;
}

// Backward, dQ and the rows' statistics.  Workgroup as in the forward:
//   S^T = K Q^T, dP^T = V dO^T, P = 2^(S c - lse), dS = P (dP - D),
//   dQ^T += K^T dS^T (K^T by transposed reads of the same tile),
// Stores -lse / scale and -D of every row, flat by key head (`rows` of each),
// and the largest length exponents of dO and of dO times O among each wave's rows
// for the kernel of dK and dV.
// Bound as the forward is, with three products for two: 2 x 1999 queries of 8
// heads over 2 of 128 values, window 512, 26.5 us (504 workgroups, two for a CU).
template <int DH, int QB>
__global__ __launch_bounds__(256, DH > 128 ? 1 : 2) void window_dq(WindowArgs a, int tiles, float* stats, int64_t rows, short2_t* tops) {
    using G = Geo<DH>;
    constexpr int KS = G::KS, DT = G::DT, W = G::W, TILE = BK * W, ROWS = 64 * QB;
    __shared__ __attribute__((aligned(1024))) f16 smem[4 * TILE];
    __shared__ uint32_t zeroed[2][4];  // rows of a tile that clean_rows has made zeros, 16 of each wave
    static_assert(BK == 64, "16 rows a wave");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const Frag<DH> fr(lane);
    const int at = xcd_tile(blockIdx.x, gridDim.x);
    const int tile = tiles - 1 - at % tiles, bc = at / tiles, c = bc % a.KV, b = bc / a.KV;
    const int group = a.H / a.KV, NR = a.N * group, R0 = tile * ROWS, wr0 = R0 + wave * 16 * QB;
    const List list(a, b, R0 / group, (min(R0 + ROWS, NR) - 1) / group, a.big);
    const KvTiles<DH, 4> kv(a, b, c, wave, lane);
    const int nt = (list.n + BK - 1) / BK;
    kv.load(list, 0, smem, smem + TILE);

    half8 qf[QB][KS], gf[QB][KS];
    int qp[QB];
    float lse2[QB], dsum[QB];
    int lift[QB];
    short2_t top = {K_LEAST, 2 * K_LEAST};
    const int64_t q0 = ((int64_t)b * a.N * a.H + c * group) * a.dh;
    auto row_at = [&](int r) { return q0 + ((int64_t)(r / group) * a.H + r % group) * a.dh; };
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int r = min(wr0 + 16 * q + l16, NR - 1);
        qp[q] = r / group;
        const float lse = a.lse[((int64_t)b * a.H + c * group + r % group) * a.N + r / group];
        half8 of[KS];
        const int64_t src = row_at(r) + 8 * g;
        const f16 *q_at = a.q + src, *g_at = a.dO + src, *o_at = a.o + src;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qf[q][ks] = gf[q][ks] = of[ks] = half8{};
            if (32 * ks + 8 * g < a.dh) {
                qf[q][ks] = *reinterpret_cast<const half8*>(q_at + 32 * ks);
                gf[q][ks] = *reinterpret_cast<const half8*>(g_at + 32 * ks);
                of[ks] = *reinterpret_cast<const half8*>(o_at + 32 * ks);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // every load out before the first sum waits
        float sum = 0.0f, squares = 0.0f, o_squares = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum += (float)gf[q][ks][i] * (float)of[ks][i];
                squares += (float)gf[q][ks][i] * (float)gf[q][ks][i];
                o_squares += (float)of[ks][i] * (float)of[ks][i];
            }
        dsum[q] = query_sum(sum);
        if (g == 0 && wr0 + 16 * q + l16 < NR) {
            stats[(int64_t)bc * NR + r] = -lse / a.scale;
            stats[rows + (int64_t)bc * NR + r] = -dsum[q];
        }
        const int kg = length_exponent(query_sum(squares)), ko = length_exponent(query_sum(o_squares));
        lift[q] = kg - DQ_LIFT;
        lse2[q] = lse * kLog2e + (float)lift[q];  // into P
        top = __builtin_elementwise_max(top, short2_t{(short)kg, (short)(kg + ko)});
    }
    for (int o = 32; o > 0; o >>= 1) top = max_xor(top, o);
    if (lane == 0) tops[((int64_t)bc * tiles + tile) * 4 + wave] = top;
    const float c2 = a.scale * kLog2e;
    floatx4 acc[DT][QB];
    uint32_t wild = 0;
    auto store = [&] {
        int at_lane = lane;
        asm volatile("" : "+v"(at_lane));  // places formed here, not kept from before the loop
        const int l16 = at_lane & 15, g = at_lane >> 4;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            const int r = wr0 + 16 * q + l16;
            if (r >= NR) continue;
            f16* dst = a.out + row_at(r);
            const float back = __builtin_ldexpf(a.scale, lift[q]);
#pragma unroll
            for (int d = 0; d < DT; ++d)
                if (16 * d + 4 * g < a.dh)
                    *reinterpret_cast<uint2*>(dst + 16 * d + 4 * g) =
                        uint2{pack_h2(acc[d][q][0] * back, acc[d][q][1] * back), pack_h2(acc[d][q][2] * back, acc[d][q][3] * back)};
        }
    };
    for (int left = DQ_LIFT;; left -= DQ_STEP) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int q = 0; q < QB; ++q) acc[d][q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int t = 0; t < nt; ++t) {
            f16* const sk = smem + (t & 1) * 2 * TILE;
            f16* const sv = sk + TILE;
            wait_loads();  // this wave's part of tile t is in LDS
            const bool whole = list.plain(a, t * BK, BK);
            if (!whole) {
                const uint32_t hit = clean_rows(kv.dma, sk);
                if (lane == 0) zeroed[t & 1][wave] = hit;
                wild |= hit;
            }
            __syncthreads();  // everyone's; the other stage is free
            if (t + 1 < nt) {
                f16* const nx = smem + ((t + 1) & 1) * 2 * TILE;
                kv.load(list, (t + 1) * BK, nx, nx + TILE);
            }
            using Rows = Ring<2 * KS, 2>;
            using Cols = Ring<DT, 2>;
            half8 kf[Rows::SLOTS], vf[Rows::SLOTS], kt[Cols::SLOTS];
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                auto row = [&](auto i, auto slot) {
                    kf[slot] = fr.row(sk, 32 * k2 + 16 * (i / KS), i % KS);
                    vf[slot] = fr.row(sv, 32 * k2 + 16 * (i / KS), i % KS);
                };
                auto col = [&](auto i, auto slot) { kt[slot] = fr.col(sk, 32 * k2, i); };
                floatx4 s[2][QB], dp[2][QB];
                Rows::template start<2>(row);
                Rows::template run<2 * QB, 2>(row, [&](auto i, auto slot) {
#pragma unroll
                    for (int q = 0; q < QB; ++q) {
                        const floatx4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                        s[i / KS][q] = mfma16(kf[slot], qf[q][i % KS], i % KS ? s[i / KS][q] : zero);
                        dp[i / KS][q] = mfma16(vf[slot], gf[q][i % KS], i % KS ? dp[i / KS][q] : zero);
                    }
                });
                // workgroup-uniform: every query sees these rows, and all of them are here
                const bool plain = list.plain(a, t * BK + 32 * k2, 32) && (whole || __builtin_amdgcn_readfirstlane(zeroed[t & 1][2 * k2] | zeroed[t & 1][2 * k2 + 1]) == 0);
                half8 ds[QB];
#pragma unroll
                for (int q = 0; q < QB; ++q) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][q][i % 4], c2, -lse2[q]));
                        e[i] = p * (dp[i / 4][q][i % 4] - dsum[q]);
                    }
                    if (!plain) {
                        const Seen see(a, list, qp[q]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const bool zero = zeroed[t & 1][2 * k2 + i / 4] >> (4 * g + i % 4) & 1;
                            e[i] = see(t * BK + 32 * k2 + 16 * (i / 4) + 4 * g + i % 4) & !zero ? e[i] : 0.0f;
                        }
                    }
                    ds[q] = as_half8(u32x4{pack_h2(e[0], e[1]), pack_h2(e[2], e[3]), pack_h2(e[4], e[5]), pack_h2(e[6], e[7])});
                }
                Cols::template start<2>(col);
                Cols::template run<QB, 2>(col, [&](auto i, auto slot) {
#pragma unroll
                    for (int q = 0; q < QB; ++q) acc[i][q] = mfma16(kt[slot], ds[q], acc[i][q]);
                });
            }
        }
        store();
        // sums past fp16 of queries whose own terms are finite
        bool over = false;
        if (left >= 0) {
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                bool mine = false;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mine |= !(fabsf(acc[d][q][j]) < INFINITY);
                mine = query_max(mine ? 1.0f : 0.0f) > 0.0f && fabsf(dsum[q]) < INFINITY && fabsf(lse2[q]) < INFINITY;
                lift[q] += mine ? DQ_STEP : 0;
                lse2[q] += mine ? (float)DQ_STEP : 0.0f;
                over |= mine;
            }
        }
        if (!__syncthreads_or(over | (wild != 0))) return;
        if (!__syncthreads_or(over)) break;
        kv.load(list, 0, smem, smem + TILE);
    }
    const int64_t ld = (int64_t)a.KV * a.dh;
    each_wild([&](int t) { return list.plain(a, t * BK, BK); }, [&](int e) { return list.has(e) ? kv.k + list.row(e) * ld : nullptr; }, a.dh, BK, 0, nt, 1, lane, [&](int i) {
        const int64_t row = list.row(i);
        float ds[QB], dp[QB];
        bool sees[QB], nan[QB];
#pragma unroll
        for (int q = 0; q < QB; ++q) sees[q] = Seen(a, list, qp[q])(i);
        spoilt(nan, acc);
        if (!any_open(sees, nan)) return;
        row_dot(ds, qf, kv.k + row * ld, a.dh, g);
        row_dot(dp, gf, kv.v + row * ld, a.dh, g);
#pragma unroll
        for (int q = 0; q < QB; ++q) ds[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(ds[q], c2, -lse2[q])) * (dp[q] - dsum[q]);
        add_row(acc, ds, sees, kv.k + row * ld, a.dh, g);
    });
    store();
}

// Backward, dK and dV.  Workgroup: NWV waves of 16 KB rows (keys) of one key head
// and one part of the queries that see any of them; Q and dO come in tiles of
// QT flat rows through two LDS stages.
//   S = Q K^T - lse / scale and dP = dO V^T - D (a lane: one key, rows 4 g + j
//   of a 16-row block; the rows' terms are what the sums start from),
//   P = 2^(S c), dS = P dP, which are then the B operands of dV^T += dO^T P and
//   dK^T += Q^T dS, whose A operands are transposed reads of the same tiles.
// The sum over the heads of a group is part of the sum over rows.  Four products
// for the forward's two, over the same pairs as window_dq: 47 us at its size,
// 313 TFLOP/s; 168 registers hold three workgroups a CU.  32 keys a wave, tiles of
// 64 rows and eight waves were no faster.
//
// Parts: the queries from the first key's position to the last one that sees
// the block are cut every `unit` positions (KEYS times Parts::q).  A block with
// one part writes dK and dV; the others (the sinks' blocks, which every later
// query sees, and all where the grid would not fill the chip otherwise) leave
// 32-bit sums that window_dkdv_join adds in the order of the parts (11.8 us for
// 45 MB there).
struct Parts {
    int q;       // key blocks' lengths of queries per part
    int blocks;  // key blocks of a sequence
    int full;    // the first of them, seen by every later query: block i has ceil((blocks - i) / q) parts
    int rest;    // parts of each other block
    int items;   // parts of one key head
    int slots;   // of them with sums in the workspace, the first ones
    __host__ __device__ __forceinline__ int parts_of(int i) const { return i < full ? (blocks - i + q - 1) / q : rest; }
    __host__ __device__ __forceinline__ int64_t sum(int64_t n) const {  // of ceil(m / q) for m = 1 .. n
        const int64_t k = n / q;
        return q * k * (k + 1) / 2 + (n - q * k) * (k + 1);
    }
    __host__ __device__ __forceinline__ int64_t before(int i) const {  // parts before block i
        const int f = i < full ? i : full;
        return sum(blocks) - sum(blocks - f) + (int64_t)(i - f) * rest;
    }
    // the block and the part that item `it` is: the first blocks in groups of q of equally many parts
    DEV void find(int it, int* blk, int* part) const {
        int k = (blocks + q - 1) / q, first = 0, n = min(full, blocks - (k - 1) * q);
        while (first < full && it >= n * k) {
            it -= n * k--;
            first += n;
            n = min(q, full - first);
        }
        if (first >= full) k = rest;
        *blk = first + it / k;
        *part = it % k;
    }
};

template <int DH>
struct KvGrad {
    static constexpr int KB = 1, NWV = 4;  // 16-key blocks of a wave, waves
    static constexpr int KEYS = 16 * KB * NWV, QT = Geo<DH>::W >= 128 ? 32 : 64;
};
template <int DH>
__global__ __launch_bounds__(64 * KvGrad<DH>::NWV, DH <= 128 ? 3 : 1) void window_dkdv(WindowArgs a, Parts pt, const float* stats, int64_t rows, const short2_t* tops, int tops_n, int tops_lg, float* ws) {
    using G = Geo<DH>;
    constexpr int KS = G::KS, DT = G::DT, W = G::W, KB = KvGrad<DH>::KB, NWV = KvGrad<DH>::NWV, KEYS = KvGrad<DH>::KEYS;
    constexpr int QT = KvGrad<DH>::QT, TILE = QT * W;
    __shared__ __attribute__((aligned(1024))) f16 smem[4 * TILE];
    __shared__ __attribute__((aligned(1024))) float sst[2][2][256];  // -lse / scale and -D of a tile's rows; a wave's load fills 1 KB
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const Frag<DH> fr(lane);
    const int at = xcd_tile(blockIdx.x, gridDim.x);
    auto uni = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // quotients come in vector registers
    const int bc = uni(at / pt.items), c = uni(bc % a.KV), b = uni(bc / a.KV), item = uni(at % pt.items);
    int blk, part;
    pt.find(item, &blk, &part);
    blk = uni(blk);
    part = uni(part);
    const int nparts = uni(pt.parts_of(blk));
    const int group = uni(a.H / a.KV), NR = a.N * group;
    const int k0 = blk * KEYS, klast = min(k0 + KEYS, a.N) - 1;
    // queries of this part: flat rows [ra, rb_end)
    const int64_t unit = (int64_t)pt.q * KEYS;
    const int64_t t_end = k0 < a.sinks ? a.N : min((int64_t)a.N, (int64_t)klast + a.window);
    const int ta = (int)min(t_end, k0 + part * unit), tb = (int)min(t_end, k0 + (part + 1) * unit);
    const int ra = ta * group, rb_end = tb * group;
    const int nt = (rb_end - ra + QT - 1) / QT;

    const int64_t qb0 = (int64_t)b * a.N * a.H + c * group;  // row of (position 0, head 0 of the group)
    const SmallDiv by_group(group);
    // a tile's rows begin with row m0 of a position's `group`; where tiles hold whole positions m0 is 0 throughout
    using Dma = TileDma<DH, QT, NWV>;
    const Dma dma{wave, lane};
    auto offset = [&](int i, int m0) {
        Dma dma{wave, lane};
        // formed for every tile: kept, they were spilled (DH 128 holds 168 registers) and a reload waits for the loads before it
        if constexpr (DH == 128) asm volatile("" : "+v"(dma.lane));
        const int m = m0 + dma.row(i), t = by_group(m);
        return oob_or(dma.chunk(i) * 8 < a.dh, (uint32_t)((t * a.H + (m - t * group)) * a.dh + dma.chunk(i) * 8) * 2);
    };
    // tile at flat row r0, row m0 of position t0
    const uint32_t whole = (uint32_t)uni((by_group(QT - 1) * a.H + (QT - 1 - by_group(QT - 1) * group) + 1) * a.dh * 2);
    auto load = [&](int r0, int t0, int m0, f16* sq, f16* sg) {
        const int64_t base = (qb0 + (int64_t)t0 * a.H) * a.dh;
        if (m0 == 0 && r0 + QT <= rb_end) {
            uint32_t off[Dma::PER];
#pragma unroll
            for (int i = 0; i < Dma::PER; ++i) off[i] = offset(i, 0);
            dma.go(wave_rsrc(a.q + base, whole), off, sq);
            dma.go(wave_rsrc(a.dO + base, whole), off, sg);
            return;
        }
        const int rows = min(QT, rb_end - r0), tl = by_group(m0 + rows - 1);  // up to the end of the last row
        const uint32_t span = (uint32_t)(tl * a.H + (m0 + rows - 1 - tl * group) + 1) * a.dh * 2;
        uint32_t o[Dma::PER];
        // rows past the last one may lie before its end in memory (other heads' rows of the same position)
#pragma unroll
        for (int i = 0; i < Dma::PER; ++i) o[i] = oob_or(dma.row(i) < rows, offset(i, m0));
        dma.go(wave_rsrc(a.q + base, span), o, sq);
        dma.go(wave_rsrc(a.dO + base, span), o, sg);
    };
    auto load_stats = [&](int r0, int stage) {
        // whole lanes: up to three values past the rows are the other array's or the exponents', and masked
        if (wave < 2)
            dma16(wave_rsrc(stats + (wave ? rows : 0) + (int64_t)bc * NR + r0, (uint32_t)(min(QT, rb_end - r0) + 3) / 4 * 16),
                  (uint32_t)lane * 16, lds_addr(reinterpret_cast<const f16*>(sst)) + (2 * stage + wave) * 1024);
    };
    short2_t top = {K_LEAST, 2 * K_LEAST}, v_top = {K_LEAST, 0};
    if (nt > 0) {
        load(ra, ta, 0, smem, smem + TILE);
        load_stats(ra, 0);
        // an entry for every 2^tops_lg rows, tops_n a key head
        for (int i = (ra >> tops_lg) + lane; i <= (rb_end - 1) >> tops_lg; i += 64)
            top = __builtin_elementwise_max(top, (tops + (int64_t)bc * tops_n)[i]);
    }
    half8 kf[KB][KS], vf[KB][KS];
    const int64_t kv_ld = (int64_t)a.KV * a.dh, kv0 = (int64_t)b * a.R * kv_ld + (int64_t)c * a.dh;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int64_t src = kv0 + min(k0 + (wave * KB + kb) * 16 + l16, a.N - 1) * kv_ld;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            kf[kb][ks] = vf[kb][ks] = half8{};
            if (32 * ks + 8 * g < a.dh) {
                kf[kb][ks] = *reinterpret_cast<const half8*>(a.k + src + 32 * ks + 8 * g);
                vf[kb][ks] = *reinterpret_cast<const half8*>(a.v + src + 32 * ks + 8 * g);
            }
        }
        float squares = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i) squares += (float)vf[kb][ks][i] * (float)vf[kb][ks][i];
        v_top.x = max((int)v_top.x, length_exponent(query_sum(squares)));
    }
    floatx4 gk[DT][KB], gv[DT][KB];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) gk[d][kb] = gv[d][kb] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const float c2 = a.scale * kLog2e;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        top = max_xor(top, o);
        if (o < 16) v_top = max_xor(v_top, o);  // the lanes of a key hold the same
    }
    // |dS| < P 2^(DS_TOP - lift)
    const int lift = __builtin_amdgcn_readfirstlane(DS_TOP - 1 - max(top.x + v_top.x, (int)top.y));  // -27 .. 61
    const float lift_ds = exp2i(lift - P_LIFT);
    uint32_t wild = 0;
    // 32 rows of a tile
    auto step_of = [&](int t, int r0, int tf, int m0, int h, const f16* sq, const f16* sg, bool plain) {
        using Rows = Ring<2 * KS, 3>;
        using Cols = Ring<DT, 3>;
        half8 qf[Rows::SLOTS], gf[Rows::SLOTS], qt[Cols::SLOTS], gt[Cols::SLOTS], p[KB], ds[KB];
        floatx4 s[2][KB], dp[2][KB];
        auto row = [&](auto i, auto slot) {
            qf[slot] = fr.row(sq, 32 * h + 16 * (i / KS), i % KS);
            gf[slot] = fr.row(sg, 32 * h + 16 * (i / KS), i % KS);
        };
        auto col = [&](auto i, auto slot) {
            gt[slot] = fr.col(sg, 32 * h, i);
            qt[slot] = fr.col(sq, 32 * h, i);
        };
        floatx4 x0[2], y0[2];
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            x0[rb] = *reinterpret_cast<const floatx4*>(&sst[t & 1][0][32 * h + 16 * rb + 4 * g]);
            y0[rb] = *reinterpret_cast<const floatx4*>(&sst[t & 1][1][32 * h + 16 * rb + 4 * g]);
        }
        Rows::template start<2>(row);
        Rows::template run<2 * KB, 2>(row, [&](auto i, auto slot) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                s[i / KS][kb] = mfma16(qf[slot], kf[kb][i % KS], i % KS ? s[i / KS][kb] : x0[i / KS]);
                dp[i / KS][kb] = mfma16(gf[slot], vf[kb][i % KS], i % KS ? dp[i / KS][kb] : y0[i / KS]);
            }
        });
        if (!plain) {  // workgroup-uniform: hidden scores to -inf, hidden dP to 0
#pragma unroll
            for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 32 * h + 16 * rb + 4 * g + j, pos = tf + by_group(m0 + r);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
                        const int key = k0 + (wave * KB + kb) * 16 + l16;
                        const bool see = (r0 + r < rb_end) & (key <= pos) & ((key > pos - a.window) | (key < a.sinks));
                        s[rb][kb][j] = see ? s[rb][kb][j] : -INFINITY;
                        dp[rb][kb][j] = see ? dp[rb][kb][j] : 0.0f;
                    }
                }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            u32x4 pu, du;
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
                float e[4], f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][kb][j], c2, (float)P_LIFT));
                    f[j] = e[j] * lift_ds * dp[rb][kb][j];
                }
                pu[2 * rb] = pack_h2(e[0], e[1]);
                pu[2 * rb + 1] = pack_h2(e[2], e[3]);
                du[2 * rb] = pack_h2(f[0], f[1]);
                du[2 * rb + 1] = pack_h2(f[2], f[3]);
            }
            p[kb] = as_half8(pu);
            ds[kb] = as_half8(du);
        }
        Cols::template start<4>(col);
        Cols::template run<2 * KB, 4>(col, [&](auto i, auto slot) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                gv[i][kb] = mfma16(gt[slot], p[kb], gv[i][kb]);
                gk[i][kb] = mfma16(qt[slot], ds[kb], gk[i][kb]);
            }
        });
    };
    int t0 = ta, m0 = 0;
    // every query of the tile at flat row r0 (position tf; the next tile is at row mn of position tn) sees every key of the
    // block: the first query the last key, the last query (before the next tile) the first key outside the sinks
    auto plain_at = [&](int r0, int tf, int tn, int mn) {
        const int tl = mn ? tn : tn - 1;
        return (r0 + QT <= rb_end) & (klast <= tf) & ((klast < a.sinks) | (max(k0, a.sinks) > tl - a.window));
    };
    for (int t = 0; t < nt; ++t) {
        f16* const sq = smem + (t & 1) * 2 * TILE;
        f16* const sg = sq + TILE;
        const int r0 = ra + t * QT;
        const int gone = __builtin_amdgcn_readfirstlane(by_group(m0 + QT)), tf = t0, mf = m0;  // positions up to the next tile
        t0 += gone;
        m0 += QT - gone * group;
        const bool plain = plain_at(r0, tf, t0, m0);
        wait_loads();  // this wave's part of tile t is in LDS
        if (!plain) wild |= clean_rows(dma, sq) | clean_rows(dma, sg);
        __syncthreads();  // everyone's; the other stage is free
        if (t + 1 < nt) {
            f16* const nx = smem + ((t + 1) & 1) * 2 * TILE;
            load(r0 + QT, t0, m0, nx, nx + TILE);
            load_stats(r0 + QT, (t + 1) & 1);
        }
#pragma unroll
        for (int h = 0; h < QT / 32; ++h) {
            step_of(t, r0, tf, mf, h, sq, sg, plain);
        }
    }
    if (__syncthreads_or(wild)) {
#pragma unroll 1
        for (int t = 0; t < nt; ++t) {
            const int r0 = ra + t * QT;
            if (plain_at(r0, r0 / group, (r0 + QT) / group, (r0 + QT) % group)) continue;
            const int rl = r0 + lane;
            auto at_row = [&](int r) { return (qb0 + (int64_t)(r / group) * a.H + r % group) * a.dh; };
            const bool is_row = (lane < QT) & (rl < rb_end);
            const uint64_t mq = __ballot(is_row && wild_row(a.q + at_row(is_row ? rl : r0), a.dh));
            const uint64_t mg = __ballot(is_row && wild_row(a.dO + at_row(is_row ? rl : r0), a.dh));
#pragma unroll 1
            for (uint64_t m = mq | mg; m; m &= m - 1) {
                const int i = __builtin_ctzll(m), r = r0 + i, pos = r / group;
                const f16 *qr = a.q + at_row(r), *gr = a.dO + at_row(r);
                float p[KB], ds[KB];
                bool sees[KB], nan_k[KB], nan_v[KB];
                spoilt(nan_k, gk);
                spoilt(nan_v, gv);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const int key = k0 + (wave * KB + kb) * 16 + l16;
                    sees[kb] = (key <= pos) & ((key > pos - a.window) | (key < a.sinks));
                    nan_k[kb] &= nan_v[kb];
                }
                if (!any_open(sees, nan_k)) continue;
                const float x0 = stats[(int64_t)bc * NR + r], y0 = stats[rows + (int64_t)bc * NR + r];
                row_dot(p, kf, qr, a.dh, g);
                row_dot(ds, vf, gr, a.dh, g);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    p[kb] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[kb] + x0, c2, (float)P_LIFT));
                    ds[kb] = p[kb] * lift_ds * (ds[kb] + y0);
                }
                if (mq >> i & 1) add_row(gk, ds, sees, qr, a.dh, g);
                if (mg >> i & 1) {
                    add_row(gv, p, sees, gr, a.dh, g);
                } else {  // q is not finite, and dO is in the sums, with a weight from zeros in q's place
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                        for (int d = 0; d < DT; ++d) gv[d][kb] += sees[kb] ? p[kb] * 0.0f : 0.0f;
                }
            }
        }
    }
    const float back_v = exp2i(-P_LIFT), back_k = a.scale * exp2i(-lift);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        if (nparts > 1) {
            // [key][dK, dV]; the parts of blocks that have one come after these
            float* dst = ws + ((int64_t)bc * pt.slots + item) * (2 * KEYS * DH) + ((wave * KB + kb) * 16 + l16) * (2 * DH);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                *reinterpret_cast<floatx4*>(dst + 16 * d + 4 * g) = gk[d][kb] * back_k;
                *reinterpret_cast<floatx4*>(dst + DH + 16 * d + 4 * g) = gv[d][kb] * back_v;
            }
            continue;
        }
        const int key = k0 + (wave * KB + kb) * 16 + l16;
        if (key >= a.N) continue;
        const int64_t dst = kv0 + key * kv_ld;
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (16 * d + 4 * g < a.dh) {
                const floatx4 k = gk[d][kb] * back_k, v = gv[d][kb] * back_v;
                *reinterpret_cast<uint2*>(a.dK + dst + 16 * d + 4 * g) = uint2{pack_h2(k[0], k[1]), pack_h2(k[2], k[3])};
                *reinterpret_cast<uint2*>(a.dV + dst + 16 * d + 4 * g) = uint2{pack_h2(v[0], v[1]), pack_h2(v[2], v[3])};
            }
    }
}

// The sums of the parts of one key, a wave each.
template <int DH, int KEYS>
__global__ __launch_bounds__(64) void window_dkdv_join(WindowArgs a, Parts pt, int blocks, const float* ws) {
    constexpr int PER = 2 * DH / 64;
    const int lane = threadIdx.x, j = blockIdx.x % (blocks * KEYS), bc = blockIdx.x / (blocks * KEYS);
    const int blk = j / KEYS, nparts = pt.parts_of(blk), c = bc % a.KV, b = bc / a.KV;
    if (nparts < 2 || j >= a.N) return;
    const float* src = ws + ((int64_t)bc * pt.slots + pt.before(blk)) * (2 * KEYS * DH) + (j % KEYS) * (2 * DH) + lane * PER;
    float v[PER] = {};
    for (int p = 0; p < nparts; ++p)
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] += src[(int64_t)p * (2 * KEYS * DH) + i];
    const int64_t row = ((int64_t)b * a.R + j) * a.KV + c;
    const bool is_k = lane < 32;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int d = lane % 32 * PER + i;
        if (d < a.dh) (is_k ? a.dK : a.dV)[row * a.dh + d] = (f16)v[i];
    }
}

// The MFMA kernels' shapes
bool mfma_ok(const WindowArgs& a) {
    if (a.dh % 8 || !aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out)) return false;
    if (a.dO && (!aligned16(a.dO) || !aligned16(a.o) || !aligned16(a.dK) || !aligned16(a.dV))) return false;
    // a tile's rows behind one descriptor
    return (int64_t)a.KV * a.dh * 2 * (BK + 1) < INT32_MAX && (int64_t)a.H * a.dh * 2 * 260 < INT32_MAX;
}
}  // namespace

namespace {
// Blocks of 16 queries of a wave in window_fwd and window_dq: two, each LDS read
// serving both, where that gives every CU more than one workgroup (forward of 8
// heads over 2 of 128 values, window 512, us with one and two: 252 workgroups of
// two 18.7 and 20.0, 378 30.0 and 27.7, 1008 56.4 and 50.5); 256 values leave no
// registers for two.
int query_blocks(int64_t rows, int64_t heads, int dh) { return dh <= 128 && heads * ((rows + 127) / 128) > 256 ? 2 : 1; }

// How the forward of a shape runs: 16-row tiles with the list split `splits`
// ways (window_split), or (splits 0) tiles of 64 rows and more (window_fwd).
// The latter from 65 such tiles on (us, window_fwd and window_split: 4 x 300
// queries of 4 heads over 1 of 256 values, 76 tiles, 13.5 and 23.1; 1 x 256 of
// 16 over 4 of 128, 64 tiles, 18.9 and 24.4 with a window of 1024, 104.2 and
// 84.4 over 8192 rows; 32 tiles 18.7 and 14.4, 104.3 and 51.5).
int fwd_splits(int B, int N, int R, int H, int KV, int dh, int window, int sinks) {
    const int64_t rows = (int64_t)N * (H / KV), heads = (int64_t)B * KV;
    const int64_t tiles = heads * ((rows + 15) / 16);
    if (rows > 64 && heads * ((rows + 63) / 64) > 64) return 0;
    const int64_t waves = dh <= 128 ? 8 : 4;
    const int64_t list = std::min<int64_t>(R, (int64_t)window + sinks + 16), steps = (list + 31) / 32;
    // One workgroup of `waves` steps at a time up to four of them; longer lists split down to one, as far as every
    // workgroup has a CU of its own (single tokens, us with one and four steps a wave: 8 heads over 1 of 128 values,
    // 65536 rows 15.1 and 18.4; 32 over 8, 8192 rows 12.0 and 18.7; 17 steps of 12 over 4 of 64 values 6.4, split 8.7;
    // 512 workgroups for 256: 64 sequences of 8 over 1, 4096 rows 30.3, 27.4).
    if (steps <= 4 * waves) return 1;
    return (int)std::max<int64_t>(1, std::min((steps + waves - 1) / waves, JOIN_MOST / tiles));
}
}  // namespace

uint64_t window_fwd_workspace(int B, int N, int R, int H, int KV, int dh, int window, int sinks) {
    if (dh % 8) return 0;
    const int splits = fwd_splits(B, N, R, H, KV, dh, window, sinks);
    return splits > 1 ? (uint64_t)B * N * H * splits * (head_width(dh, 32) + 4) * sizeof(float) : 0;
}

int window_forward(const WindowArgs& args, void* ws, hipStream_t st) {
    WindowArgs a = args;
    a.big = (int64_t)a.R * a.KV * a.dh * 2 >= INT32_MAX;
    const int64_t rows = (int64_t)a.B * a.N * a.H;
    const int64_t nr = (int64_t)a.N * (a.H / a.KV), heads = (int64_t)a.B * a.KV;
    const int splits = fwd_splits(a.B, a.N, a.R, a.H, a.KV, a.dh, a.window, a.sinks);
    hipError_t e;
    const int fwd_rows = 64 * query_blocks(nr, heads, a.dh);
    int rc = !mfma_ok(a) ? check_grid("window_attention", rows, 64)
             : splits    ? check_grid("window_attention", (nr + 15) / 16 * heads * splits, 512)
                         : check_grid("window_attention", (nr + fwd_rows - 1) / fwd_rows * heads, 256);
    if (rc == EVKHIP_OK && mfma_ok(a) && splits > 1) rc = check_grid("window_attention", nr * heads, 256);
    if (rc != EVKHIP_OK) return rc;
    if (!mfma_ok(a)) {
        hipLaunchKernelGGL(window_fwd_rows, dim3((unsigned)rows), dim3(64), 0, st, a);
        e = hipGetLastError();
    } else if (splits == 0) {
        e = by_head(a.dh, [&](auto dhc) {
            constexpr int DH = decltype(dhc)::value;
            auto go = [&](auto qb) {
                constexpr int QB = decltype(qb)::value;
                const int tiles = (int)((nr + 64 * QB - 1) / (64 * QB));
                hipLaunchKernelGGL((window_fwd<DH, QB>), dim3((unsigned)(tiles * heads)), dim3(256), 0, st, a, tiles);
            };
            if constexpr (DH <= 128) {
                if (query_blocks(nr, heads, a.dh) == 2) return go(std::integral_constant<int, 2>{});
            }
            go(std::integral_constant<int, 1>{});
        });
    } else {
        e = by_head(a.dh, [&](auto dhc) {
            constexpr int DH = decltype(dhc)::value;
            const int tiles = (int)((nr + 15) / 16);
            hipLaunchKernelGGL(window_split<DH>, dim3((unsigned)(tiles * splits * heads)), dim3(64 * SplitGeo<DH>::NW), 0, st, a, tiles, splits,
                               (float*)ws);
            if (splits > 1)
                hipLaunchKernelGGL(window_join<DH>, dim3((unsigned)(nr * heads)), dim3(256), 0, st, a, splits, (const float*)ws);
        });
    }
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "window_attention launch");
}

namespace {
Parts parts_for(int B, int N, int H, int KV, int dh, int window, int sinks) {
    const int64_t keys = dh <= 128 ? KvGrad<128>::KEYS : KvGrad<256>::KEYS, heads = (int64_t)B * KV;
    const int64_t blocks = (N + keys - 1) / keys;
    const int64_t full = window >= N ? blocks : std::min<int64_t>(blocks, ((int64_t)sinks + keys - 1) / keys);
    // queries that see a block, in key blocks' lengths: the window, or every later one
    const int64_t span = full == blocks ? blocks : std::min(blocks, ((int64_t)window + keys - 2) / keys + 1);
    auto items = [&](int64_t q) {
        const Parts p{(int)q, (int)blocks, (int)full, (int)((span + q - 1) / q), 0, 0};
        return p.before((int)blocks);
    };
    // long parts, as few as make 500 workgroups, two for a CU (2 x 1999 queries of 8 heads over 2 of 128 values, window
    // 512, the whole backward: 250 97 us, 500 84, 1000 97; one sequence of 4000, no window: 245, 203, 208), none of
    // under 128 rows (one sequence of 4000, 2 heads over 1 of 64 values, window 512: 50.1 us, with this limit 40.0;
    // 2000, one head of 128, no window: 67.5, 58.9), and fewer than 2^24
    int64_t q = full == blocks ? std::max<int64_t>(1, span / 4) : span;
    while (q > 1 && items(q) * heads < 500 && q * keys * (H / KV) > 256) q /= 2;
    while (items(q) * heads >= (1 << 24) && q < blocks) q *= 2;
    Parts p{};
    p.q = (int)q;
    p.blocks = (int)blocks;
    p.full = (int)full;
    p.rest = (int)((span + q - 1) / q);
    p.items = (int)items(q);
    p.slots = p.rest > 1 ? p.items : p.items - (int)(blocks - full);
    return p;
}
}  // namespace

// The backward workspace: the rows' statistics, the length exponents of waves' rows, the parts' sums, each a multiple of
// 16 bytes.
namespace {
uint64_t window_stats_rows(int B, int N, int H) { return ((uint64_t)B * N * H + 3) / 4 * 4; }  // of each of two
uint64_t window_tops_bytes(int B, int N, int H, int KV, int dh) {
    const int64_t nr = (int64_t)N * (H / KV), per = 64 * query_blocks(nr, (int64_t)B * KV, dh);
    return (uint64_t)B * KV * ((nr + per - 1) / per) * 4 * sizeof(short2_t);
}
}  // namespace

uint64_t window_bwd_workspace(int B, int N, int H, int KV, int dh, int window, int sinks) {
    if (dh % 8) return 0;
    const Parts p = parts_for(B, N, H, KV, dh, window, sinks);
    static_assert(KvGrad<64>::KEYS == KvGrad<256>::KEYS, "one length of key blocks");
    const uint64_t part = KvGrad<64>::KEYS * 2 * head_width(dh, 64) * sizeof(float);
    return 2 * window_stats_rows(B, N, H) * sizeof(float) + window_tops_bytes(B, N, H, KV, dh) + (uint64_t)B * KV * p.slots * part;
}

int window_backward(const WindowArgs& args, void* ws, hipStream_t st) {
    WindowArgs a = args;
    a.big = (int64_t)a.R * a.KV * a.dh * 2 >= INT32_MAX;
    const int64_t rows = (int64_t)a.B * a.N * a.H, kv_rows = (int64_t)a.B * a.R * a.KV;
    hipError_t e;
    // the widest launches of either path: a wave for each key (rounded up to blocks of 64) or query row, four for a tile
    const int64_t group = a.H / a.KV, heads = (int64_t)a.B * a.KV, dq_rows = 64 * query_blocks(a.N * group, heads, a.dh);
    int rc = check_grid("window_attention_bwd", mfma_ok(a) ? heads * ((a.N + 63) / 64 * 64) : std::max(rows, kv_rows), 64);
    if (rc == EVKHIP_OK && mfma_ok(a)) rc = check_grid("window_attention_bwd", (a.N * group + dq_rows - 1) / dq_rows * heads, 256);
    if (rc != EVKHIP_OK) return rc;
    if (mfma_ok(a)) {
        const int64_t nr = (int64_t)a.N * (a.H / a.KV);
        const int qb = query_blocks(nr, (int64_t)a.B * a.KV, a.dh), tiles = (int)((nr + 64 * qb - 1) / (64 * qb));
        const int64_t srows = (int64_t)window_stats_rows(a.B, a.N, a.H);
        float* const stats = (float*)ws;
        short2_t* const tops = (short2_t*)(stats + 2 * srows);
        float* const sums = (float*)((char*)tops + window_tops_bytes(a.B, a.N, a.H, a.KV, a.dh));
        e = by_head(a.dh, [&](auto dhc) {
            constexpr int DH = decltype(dhc)::value;
            const dim3 grid((unsigned)((int64_t)tiles * a.B * a.KV));
            if constexpr (DH <= 128) {
                if (qb == 2) {
                    hipLaunchKernelGGL((window_dq<DH, 2>), grid, dim3(256), 0, st, a, tiles, stats, srows, tops);
                    return;
                }
            }
            hipLaunchKernelGGL((window_dq<DH, 1>), grid, dim3(256), 0, st, a, tiles, stats, srows, tops);
        });
        const Parts p = parts_for(a.B, a.N, a.H, a.KV, a.dh, a.window, a.sinks);
        if (e == hipSuccess)
            e = by_head64(a.dh, [&](auto dhc) {
                constexpr int DH = decltype(dhc)::value, KEYS = KvGrad<DH>::KEYS;
                hipLaunchKernelGGL(window_dkdv<DH>, dim3((unsigned)(p.items * a.B * a.KV)), dim3(64 * KvGrad<DH>::NWV), 0, st, a, p, stats, srows, tops,
                                   tiles * 4, qb == 2 ? 5 : 4, sums);
                const int joined = p.rest > 1 ? p.blocks : p.full;
                if (p.slots > 0 && joined > 0)
                    hipLaunchKernelGGL((window_dkdv_join<DH, KEYS>), dim3((unsigned)((int64_t)joined * KEYS * a.B * a.KV)), dim3(64), 0, st, a,
                                       p, joined, sums);
            });
    } else {
        hipLaunchKernelGGL(window_dkdv_rows, dim3((unsigned)kv_rows), dim3(64), 0, st, a);
        hipLaunchKernelGGL(window_dq_rows, dim3((unsigned)rows), dim3(64), 0, st, a);
        e = hipGetLastError();
    }
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "window_attention_bwd launch");
}

}  // namespace evkhip

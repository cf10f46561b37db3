// Grouped-query attention over a sliding window and the first tokens (sinks),
// forward, backward and for single tokens (no counterpart in the reference,
// whose attention sees every earlier position).
//
// Query t of sequence b stands at position p = p0 + t and sees the rows
//   [0, s) and [lo, hi)   with hi = min(p + 1, rows), lo = max(0, p - W + 1),
//                              s = min(sinks, lo)
// of its K and V; a query that sees nothing (p < 0) has O = 0, LSE = -inf.
//   S = Q K^T / sqrt(Dh), P = exp(S - LSE), O = P V
//   backward: D = rowsum(dO * O), dS = P (dO V^T - D),
//             dQ = dS K / sqrt(Dh), dK = dS^T Q / sqrt(Dh), dV = P^T dO,
//             dK and dV summed over the heads that share the row.
//
// Rows that a query does not see are never read for it, so that whatever they
// hold (stale cache rows, infinities, NaN) stays out of its sums.
#include "kernels.h"

#include <algorithm>

#include <math.h>

namespace evkhip {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
// Position of query t of sequence b, -1 for any that sees nothing.
DEV int position_of(const WindowArgs& a, int b, int t) {
    const int64_t p = (int64_t)(a.offsets ? a.offsets[b] : a.p0) + t;
    return (int)(p < 0 ? -1 : p < INT32_MAX ? p : INT32_MAX);
}

// ---------------------------------------------------------------------------
// One wave per query row (or per K, V row), any head size and alignment.
// Latency-bound chains of scalar loads: the path of head sizes and pointers
// that the MFMA kernels do not take.
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
DEV void wave_sync() {  // the wave's LDS accesses before this are done
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// O and LSE of query row `row` = ((b N) + t) H + h
DEV void fwd_row(const WindowArgs& a, int64_t row, RowLds& s, int lane) {
    const int dh = a.dh, h = (int)(row % a.H), t = (int)(row / a.H % a.N), b = (int)(row / a.H / a.N);
    const int64_t kv_ld = (int64_t)a.KV * dh;
    const int64_t kv0 = (int64_t)b * a.R * kv_ld + (int64_t)(h / (a.H / a.KV)) * dh;
    const Span sp = span_of(position_of(a, b, t), a);
    wave_sync();
    for (int d = lane; d < dh; d += 64) s.x[d] = (float)a.q[row * dh + d];
    wave_sync();
    float m = -INFINITY, l = 0.0f, o[SMAX / 64] = {};
    for (int i0 = 0; i0 < sp.count(); i0 += 64) {
        const int n = min(64, sp.count() - i0);
        const int64_t j = sp.row(min(i0 + lane, sp.count() - 1)) * kv_ld;
        const float sc = lane < n ? dot_row(a.k + kv0 + j, s.x, dh) * a.scale * kLog2e : -INFINITY;
        const float m_new = fmaxf(m, wave_max(sc));
        const float keep = m == -INFINITY ? 0.0f : exp2f(m - m_new);
        const float e = lane < n ? exp2f(sc - m_new) : 0.0f;
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
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.H + h) * a.N + t] = sp.count() ? (m + log2f(l)) * kLn2 : -INFINITY;
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
//
// v_mfma_f32_16x16x32_f16 throughout: S^T = K Q^T gives a lane one query
// (column l16 = lane % 16) and rows 4 g + j (g = lane / 16) of each 16-row
// block, which is the B operand of O^T += V^T P^T as it stands (slot s: row
// 4 g + s of the first, 4 g + s - 4 of the second block); V^T comes from the
// row-major tile by ds_read_b64_tr_b16.
// ---------------------------------------------------------------------------
constexpr int BK = 64;               // list entries per tile
constexpr float RESCALE_LOG2 = 8.0f;  // O and l are rescaled when a score passes the reference by 2^8

template <int DH>
struct Geo {
    static constexpr int KS = DH / 32, DT = DH / 16;
    static constexpr int W = DH <= 32 ? 32 : DH <= 64 ? 64 : DH <= 128 ? 128 : 256;  // halves of an LDS row
    static constexpr int CPR = W / 8;                                               // 16-byte chunks of it
};
// Chunk c of row r lies at slot c ^ swz(r): the reads of eight rows at one
// chunk and of four rows at one pair of chunks both hit distinct banks.
template <int W>
DEV int swz(int r) {
    return W == 32 ? 2 * ((r >> 1) & 1) | ((r >> 2) & 1) : 2 * (r & 3) | ((r >> 2) & 1);
}
template <int W>
DEV half8 row_frag(const f16* t, int r, int chunk) {
    return *reinterpret_cast<const half8*>(t + r * W + ((chunk ^ swz<W>(r)) << 3));
}
// rows r .. r + 3 and r + 16 .. r + 19 (r = 4 g + trow of a 32-row step) of the 16 columns of block d
template <int W>
DEV half8 col_frag(const f16* t, int r, int d, int tcol) {
    auto at = [&](int q) { return t + q * W + (((2 * d + (tcol >> 3)) ^ swz<W>(q)) << 3 | (tcol & 7)); };
    return cat4(lds_read_tr(at(r)), lds_read_tr(at(r + 16)));
}

// ROWS rows of 16-byte chunks into LDS; off(row): byte offset of row `row` from the descriptor's base, or < 0 for
// none.  Rows and chunks that are not there read as zeros.
template <int DH, int ROWS, int NWV, class F>
DEV void rows_to_lds(__amdgpu_buffer_rsrc_t res, int dh, f16* lds, int wave, int lane, F&& off) {
    using G = Geo<DH>;
    constexpr int RPI = 64 / G::CPR, PER = ROWS / RPI / NWV;
    static_assert(PER >= 1 && ROWS % (RPI * NWV) == 0, "tile shape");
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int q = wave * PER + i, row = q * RPI + lane / G::CPR;
        const int chunk = (lane % G::CPR) ^ swz<G::W>(row);
        const int64_t o = off(row);
        dma16(res, oob_or(o >= 0 && chunk * 8 < dh, (uint32_t)(o + chunk * 16)), lds_addr(lds + q * 512));
    }
}

// The list of the rows that the queries t0 .. t1 of sequence b see.
struct List {
    int pmin, pmax;  // positions of the first and last query (-1: sees nothing)
    int lo, hi, s;   // window [lo, hi); sinks [0, s) before it, none where they meet it (then lo is 0)
    int sl, n;       // entries before the window (s, or padded to whole tiles), entries
    int first;       // entries below this one are sinks
    DEV List(const WindowArgs& a, int b, int t0, int t1, bool pad) {
        pmin = position_of(a, b, t0);
        pmax = position_of(a, b, t1);
        hi = pmax < 0 ? 0 : min(pmax, a.R - 1) + 1;
        lo = min(max(0, pmin - a.window + 1), hi);
        s = a.sinks;
        if (s >= lo) lo = s = 0;
        sl = pad ? (s + BK - 1) / BK * BK : s;
        n = sl + hi - lo;
        first = lo ? s : a.sinks;
    }
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

// K and V of one sequence and key head behind buffer descriptors.  While a
// sequence's rows stay below 2 GiB one descriptor serves any row; past that
// (WindowArgs::big) the sinks are padded to whole tiles and every tile has a
// descriptor from its own first row on.
struct KvTiles {
    const f16 *k, *v;
    int64_t bytes;  // of the sequence's rows from k on
    uint32_t ld;    // bytes of a row
    DEV KvTiles(const WindowArgs& a, int b, int c) {
        ld = (uint32_t)a.KV * a.dh * 2;
        const int64_t at = (int64_t)b * a.R * a.KV * a.dh + (int64_t)c * a.dh;
        k = a.k + at;
        v = a.v + at;
        bytes = (int64_t)a.R * ld - (int64_t)c * a.dh * 2;
    }
    template <int DH, int NWV>
    DEV void load(const WindowArgs& a, const List& l, int i0, f16* sk, f16* sv, int wave, int lane) const {
        const int first = a.big ? l.row(i0) : 0;
        const int64_t skip = (int64_t)first * ld;
        const uint32_t span = (uint32_t)min(bytes - skip, (int64_t)INT32_MAX);
        auto off = [&](int r) -> int64_t {
            const int i = i0 + r;
            return (i < l.n) & ((i < l.s) | (i >= l.sl)) ? (int64_t)(l.row(i) - first) * ld : -1;
        };
        rows_to_lds<DH, BK, NWV>(buf_rsrc(k + skip / 2, span), a.dh, sk, wave, lane, off);
        rows_to_lds<DH, BK, NWV>(buf_rsrc(v + skip / 2, span), a.dh, sv, wave, lane, off);
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

// NaN or infinity among the values: a product with 0 is 0 for every other one
DEV half2_t wild2(const half8& x, half2_t w) {
    const half2_t z = {(f16)0.0f, (f16)0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) w = __builtin_elementwise_fma(half2_t{x[2 * i], x[2 * i + 1]}, z, w);
    return w;
}

// The running softmax state of QB blocks of 16 queries (a lane: query l16 of
// each) and the products of a tile of 16 KB rows into it.
template <int DH, int QB>
struct Softmax {
    static constexpr int DT = Geo<DH>::DT, W = Geo<DH>::W;
    floatx4 o[DT][QB];  // O^T: dh 16 d + 4 g + j, query l16
    float m[QB], l[QB];  // reference of the exponents (base 2; -inf: none yet), this lane's part of the sum
    DEV Softmax() {
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            m[q] = -INFINITY;
            l[q] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // Scores s (raw) of KB blocks of rows to probabilities, as B operands: P is
    // rounded to fp16 for the product (V is fp16 as well), the sum l is not.
    template <int KB>
    DEV void probs(floatx4 (&s)[KB][QB], float c2, half8 (&p)[KB / 2][QB]) {
        float mx[QB];
        bool grow = false;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            mx[q] = fmaxf(max3(s[0][q][0], s[0][q][1], s[0][q][2]), s[0][q][3]);
#pragma unroll
            for (int kb = 1; kb < KB; ++kb)
                mx[q] = max3(max3(s[kb][q][0], s[kb][q][1], mx[q]), s[kb][q][2], s[kb][q][3]);
            mx[q] *= c2;
            grow |= mx[q] > m[q] + RESCALE_LOG2;
        }
        if (__any(grow)) {
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                const float mn = fmaxf(m[q], query_max(mx[q]));
                const float keep = m[q] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[q] - mn);
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d][q] *= keep;
                l[q] *= keep;
                m[q] = mn;
            }
        }
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            const float base = m[q] == -INFINITY ? 0.0f : -m[q];
#pragma unroll
            for (int k2 = 0; k2 < KB / 2; ++k2) {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * k2 + i / 4][q][i % 4], c2, base));
                l[q] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
                p[k2][q] = as_half8(u32x4{pack_h2(e[0], e[1]), pack_h2(e[2], e[3]), pack_h2(e[4], e[5]), pack_h2(e[6], e[7])});
            }
        }
    }
};

// Forward.  Workgroup: 4 waves of 16 QB rows of one key head; K and V tiles in
// two LDS stages, filled by LDS-direct loads while the tile before is used; one
// barrier a tile.
//
// The product of a probability of 0 and a NaN or an infinity is NaN, so a tile
// that some query does not wholly see is looked at for such values in V; a wave
// that meets one computes its rows again at the end, row by row.
template <int DH, int QB>
__global__ __launch_bounds__(256, 2) void window_fwd(WindowArgs a, int tiles) {
    using G = Geo<DH>;
    constexpr int KS = G::KS, DT = G::DT, W = G::W, TILE = BK * W, ROWS = 64 * QB;
    __shared__ __attribute__((aligned(1024))) f16 smem[4 * TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4, trow = l16 >> 2, tcol = (l16 & 3) * 4;
    // an XCD takes tiles that follow each other, which share most of their rows
    const int at = xcd_tile(blockIdx.x, gridDim.x);
    const int tile = tiles - 1 - at % tiles, bc = at / tiles, c = bc % a.KV, b = bc / a.KV;
    const int group = a.H / a.KV, NR = a.N * group, R0 = tile * ROWS, wr0 = R0 + wave * 16 * QB;
    const List list(a, b, R0 / group, (min(R0 + ROWS, NR) - 1) / group, a.big);
    const KvTiles kv(a, b, c);
    const int nt = (list.n + BK - 1) / BK;
    if (nt > 0) kv.load<DH, 4>(a, list, 0, smem, smem + TILE, wave, lane);

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
    half2_t wild = {(f16)0.0f, (f16)0.0f};
    for (int t = 0; t < nt; ++t) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of tile t is in LDS
        __syncthreads();                     // everyone's; the other stage is free
        f16* const sk = smem + (t & 1) * 2 * TILE;
        f16* const sv = sk + TILE;
        if (t + 1 < nt) {
            f16* const nx = smem + ((t + 1) & 1) * 2 * TILE;
            kv.load<DH, 4>(a, list, (t + 1) * BK, nx, nx + TILE, wave, lane);
        }
        floatx4 s[4][QB];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
            for (int q = 0; q < QB; ++q) s[kb][q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const half8 kf = row_frag<W>(sk, 16 * kb + l16, 4 * ks + g);
#pragma unroll
                for (int q = 0; q < QB; ++q) s[kb][q] = mfma16(kf, qf[q][ks], s[kb][q]);
            }
        }
        const bool plain = list.plain(a, t * BK, BK);  // workgroup-uniform
        if (!plain) {
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                const Seen see(a, list, qp[q]);
#pragma unroll
                for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[kb][q][j] = see(t * BK + 16 * kb + 4 * g + j) ? s[kb][q][j] : -INFINITY;
            }
        }
        half8 p[2][QB];
        sm.template probs<4>(s, c2, p);
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
            half8 vf[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) vf[d] = col_frag<W>(sv, 32 * k2 + 4 * g + trow, d, tcol);
            if (!plain) {
#pragma unroll
                for (int d = 0; d < DT; ++d) wild = wild2(vf[d], wild);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int q = 0; q < QB; ++q) sm.o[d][q] = mfma16(vf[d], p[k2][q], sm.o[d][q]);
        }
    }
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int r = wr0 + 16 * q + l16;
        const float l = query_sum(sm.l[q]), inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (r >= NR) continue;
        f16* dst = a.out + row_at(r);
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (16 * d + 4 * g < a.dh)
                *reinterpret_cast<uint2*>(dst + 16 * d + 4 * g) =
                    uint2{pack_h2(sm.o[d][q][0] * inv, sm.o[d][q][1] * inv), pack_h2(sm.o[d][q][2] * inv, sm.o[d][q][3] * inv)};
        if (a.lse && g == 0)
            a.lse[((int64_t)b * a.H + c * group + r % group) * a.N + r / group] = l == 0.0f ? -INFINITY : (sm.m[q] + log2f(l)) * kLn2;
    }
    static_assert(4 * sizeof(RowLds) <= sizeof(smem), "a wave's rows");
    const bool again = __any(!((float)wild[0] == 0.0f && (float)wild[1] == 0.0f));
    if (!__syncthreads_or(again) || !again) return;
#pragma unroll 1
    for (int r = wr0; r < min(wr0 + 16 * QB, NR); ++r)
        fwd_row(a, ((int64_t)b * a.N + r / group) * a.H + c * group + r % group, reinterpret_cast<RowLds*>(smem)[wave], lane);
}

// Backward, dQ and the rows' statistics.  Workgroup as in the forward:
//   S^T = K Q^T, dP^T = V dO^T, P = 2^(S c - lse), dS = P (dP - D),
//   dQ^T += K^T dS^T (K^T by transposed reads of the same tile),
// dS rounded to fp16 for the product.  Stores (lse log2 e, D) of every row,
// flat by key head, for the kernel of dK and dV.
template <int DH, int QB>
__global__ __launch_bounds__(256, 2) void window_dq(WindowArgs a, int tiles, float2* stats) {
    using G = Geo<DH>;
    constexpr int KS = G::KS, DT = G::DT, W = G::W, TILE = BK * W, ROWS = 64 * QB;
    __shared__ __attribute__((aligned(1024))) f16 smem[4 * TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4, trow = l16 >> 2, tcol = (l16 & 3) * 4;
    const int at = xcd_tile(blockIdx.x, gridDim.x);
    const int tile = tiles - 1 - at % tiles, bc = at / tiles, c = bc % a.KV, b = bc / a.KV;
    const int group = a.H / a.KV, NR = a.N * group, R0 = tile * ROWS, wr0 = R0 + wave * 16 * QB;
    const List list(a, b, R0 / group, (min(R0 + ROWS, NR) - 1) / group, a.big);
    const KvTiles kv(a, b, c);
    const int nt = (list.n + BK - 1) / BK;
    kv.load<DH, 4>(a, list, 0, smem, smem + TILE, wave, lane);

    half8 qf[QB][KS], gf[QB][KS];
    int qp[QB];
    float lse2[QB], dsum[QB];
    const int64_t q0 = ((int64_t)b * a.N * a.H + c * group) * a.dh;
    auto row_at = [&](int r) { return q0 + ((int64_t)(r / group) * a.H + r % group) * a.dh; };
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int r = min(wr0 + 16 * q + l16, NR - 1);
        qp[q] = r / group;
        lse2[q] = a.lse[((int64_t)b * a.H + c * group + r % group) * a.N + r / group] * kLog2e;
        float sum = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            half8 of = {};
            qf[q][ks] = gf[q][ks] = half8{};
            if (32 * ks + 8 * g < a.dh) {
                const int64_t src = row_at(r) + 32 * ks + 8 * g;
                qf[q][ks] = *reinterpret_cast<const half8*>(a.q + src);
                gf[q][ks] = *reinterpret_cast<const half8*>(a.dO + src);
                of = *reinterpret_cast<const half8*>(a.o + src);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += (float)gf[q][ks][i] * (float)of[i];
        }
        dsum[q] = query_sum(sum);
        if (g == 0 && wr0 + 16 * q + l16 < NR) stats[(int64_t)bc * NR + r] = float2{lse2[q], dsum[q]};
    }
    const float c2 = a.scale * kLog2e;
    floatx4 acc[DT][QB];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int q = 0; q < QB; ++q) acc[d][q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    half2_t wild = {(f16)0.0f, (f16)0.0f};
    for (int t = 0; t < nt; ++t) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of tile t is in LDS
        __syncthreads();                     // everyone's; the other stage is free
        f16* const sk = smem + (t & 1) * 2 * TILE;
        f16* const sv = sk + TILE;
        if (t + 1 < nt) {
            f16* const nx = smem + ((t + 1) & 1) * 2 * TILE;
            kv.load<DH, 4>(a, list, (t + 1) * BK, nx, nx + TILE, wave, lane);
        }
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {  // 32 entries at a time
            floatx4 s[2][QB], dp[2][QB];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int q = 0; q < QB; ++q) s[kb][q] = dp[kb][q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const half8 kf = row_frag<W>(sk, 32 * k2 + 16 * kb + l16, 4 * ks + g);
                    const half8 vf = row_frag<W>(sv, 32 * k2 + 16 * kb + l16, 4 * ks + g);
#pragma unroll
                    for (int q = 0; q < QB; ++q) {
                        s[kb][q] = mfma16(kf, qf[q][ks], s[kb][q]);
                        dp[kb][q] = mfma16(vf, gf[q][ks], dp[kb][q]);
                    }
                }
            const bool plain = list.plain(a, t * BK + 32 * k2, 32);  // workgroup-uniform
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
                    for (int i = 0; i < 8; ++i) e[i] = see(t * BK + 32 * k2 + 16 * (i / 4) + 4 * g + i % 4) ? e[i] : 0.0f;
                }
                ds[q] = as_half8(u32x4{pack_h2(e[0], e[1]), pack_h2(e[2], e[3]), pack_h2(e[4], e[5]), pack_h2(e[6], e[7])});
            }
            half8 kt[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) kt[d] = col_frag<W>(sk, 32 * k2 + 4 * g + trow, d, tcol);
            if (!plain) {
#pragma unroll
                for (int d = 0; d < DT; ++d) wild = wild2(kt[d], wild);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int q = 0; q < QB; ++q) acc[d][q] = mfma16(kt[d], ds[q], acc[d][q]);
        }
    }
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        const int r = wr0 + 16 * q + l16;
        if (r >= NR) continue;
        f16* dst = a.out + row_at(r);
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (16 * d + 4 * g < a.dh)
                *reinterpret_cast<uint2*>(dst + 16 * d + 4 * g) = uint2{pack_h2(acc[d][q][0] * a.scale, acc[d][q][1] * a.scale),
                                                                        pack_h2(acc[d][q][2] * a.scale, acc[d][q][3] * a.scale)};
    }
    static_assert(4 * sizeof(RowLds) <= sizeof(smem), "a wave's rows");
    const bool again = __any(!((float)wild[0] == 0.0f && (float)wild[1] == 0.0f));
    if (!__syncthreads_or(again) || !again) return;
#pragma unroll 1
    for (int r = wr0; r < min(wr0 + 16 * QB, NR); ++r)
        dq_row(a, ((int64_t)b * a.N + r / group) * a.H + c * group + r % group, reinterpret_cast<RowLds*>(smem)[wave], lane);
}

// Backward, dK and dV.  Workgroup: 4 waves of 16 KB rows (keys) of one key head
// and one part of the queries that see any of them; Q and dO come in tiles of
// QT flat rows through two LDS stages.
//   S = Q K^T and dP = dO V^T (a lane: one key, rows 4 g + j of a 16-row
//   block), P and dS are then the B operands of dV^T += dO^T P and
//   dK^T += Q^T dS, whose A operands are transposed reads of the same tiles.
// The sum over the heads of a group is part of the sum over rows.
//
// Parts: the queries from the first key's position to the last one that sees
// the block are cut every `unit` positions (KEYS times Parts::q).  A block with
// one part writes dK and dV; the others (the sinks' blocks, which every later
// query sees, and all where the grid would not fill the chip otherwise) leave
// 32-bit sums that window_dkdv_join adds in the order of the parts.
struct Parts {
    int q;         // key blocks' lengths of queries per part
    int blocks;    // key blocks of a sequence
    int full;      // the first of them, seen by every later query
    int rest;      // parts of each other block
    int64_t items;  // parts of one key head, slots of one key head
    int64_t slots;
    __host__ __device__ __forceinline__ int64_t sum(int64_t n) const {  // of ceil(m / q) for m = 1 .. n
        const int64_t k = n / q;
        return q * k * (k + 1) / 2 + (n - q * k) * (k + 1);
    }
    // parts before block i
    __host__ __device__ __forceinline__ int64_t before(int i) const {
        const int f = i < full ? i : full;
        return sum(blocks) - sum(blocks - f) + (int64_t)(i - f) * rest;
    }
    __host__ __device__ __forceinline__ int parts_of(int i) const { return i < full ? (blocks - i + q - 1) / q : rest; }
    DEV int block_of(int64_t item) const {  // the block that holds part `item`
        int lo = 0, hi = blocks - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before(mid) <= item) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
};

template <int DH, int KB>
__global__ __launch_bounds__(256, KB == 1 && DH > 128 ? 1 : 2) void window_dkdv(WindowArgs a, Parts pt, const float2* stats, float* ws) {
    using G = Geo<DH>;
    constexpr int KS = G::KS, DT = G::DT, W = G::W, KEYS = 64 * KB, QT = 32, TILE = QT * W;
    __shared__ __attribute__((aligned(1024))) f16 smem[4 * TILE];
    __shared__ float2 sst[2][QT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4, trow = l16 >> 2, tcol = (l16 & 3) * 4;
    const int64_t at = (int64_t)xcd_tile(blockIdx.x, gridDim.x);
    const int bc = (int)(at / pt.items), c = bc % a.KV, b = bc / a.KV;
    const int64_t item = at % pt.items;
    const int blk = pt.block_of(item), part = (int)(item - pt.before(blk)), nparts = pt.parts_of(blk);
    const int group = a.H / a.KV, NR = a.N * group;
    const int k0 = blk * KEYS, klast = min(k0 + KEYS, a.N) - 1;
    // queries of this part: flat rows [ra, rb)
    const int64_t unit = (int64_t)pt.q * KEYS;
    const int64_t t_end = k0 < a.sinks ? a.N : min((int64_t)a.N, (int64_t)klast + a.window);
    const int ta = (int)min(t_end, k0 + part * unit), tb = (int)min(t_end, k0 + (part + 1) * unit);
    const int ra = ta * group, rb = tb * group;
    const int nt = (rb - ra + QT - 1) / QT;

    const int64_t qb0 = (int64_t)b * a.N * a.H + c * group;  // row of (position 0, head 0 of the group)
    auto load = [&](int r0, f16* sq, f16* sg) {
        const int t0 = r0 / group;
        const int64_t base = (qb0 + (int64_t)t0 * a.H) * a.dh;
        const uint32_t span = (uint32_t)min(((int64_t)a.B * a.N * a.H * a.dh - base) * 2, (int64_t)INT32_MAX);
        auto off = [&](int r) -> int64_t {
            const int row = r0 + r;
            return row < rb ? ((int64_t)(row / group - t0) * a.H + row % group) * a.dh * 2 : -1;
        };
        rows_to_lds<DH, QT, 4>(buf_rsrc(a.q + base, span), a.dh, sq, wave, lane, off);
        rows_to_lds<DH, QT, 4>(buf_rsrc(a.dO + base, span), a.dh, sg, wave, lane, off);
    };
    float2 st = {0.0f, 0.0f};
    auto load_stats = [&](int r0) {
        if (threadIdx.x < QT) st = r0 + (int)threadIdx.x < rb ? stats[(int64_t)bc * NR + r0 + threadIdx.x] : float2{0.0f, 0.0f};
    };
    if (nt > 0) {
        load(ra, smem, smem + TILE);
        load_stats(ra);
    }
    half8 kf[KB][KS], vf[KB][KS];
    int key[KB];
    const int64_t kv_ld = (int64_t)a.KV * a.dh, kv0 = (int64_t)b * a.R * kv_ld + (int64_t)c * a.dh;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        key[kb] = k0 + (wave * KB + kb) * 16 + l16;
        const int64_t src = kv0 + min(key[kb], a.N - 1) * kv_ld;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            kf[kb][ks] = vf[kb][ks] = half8{};
            if (32 * ks + 8 * g < a.dh) {
                kf[kb][ks] = *reinterpret_cast<const half8*>(a.k + src + 32 * ks + 8 * g);
                vf[kb][ks] = *reinterpret_cast<const half8*>(a.v + src + 32 * ks + 8 * g);
            }
        }
    }
    floatx4 gk[DT][KB], gv[DT][KB];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) gk[d][kb] = gv[d][kb] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const float c2 = a.scale * kLog2e;
    half2_t wild = {(f16)0.0f, (f16)0.0f};
    for (int t = 0; t < nt; ++t) {
        if (threadIdx.x < QT) sst[t & 1][threadIdx.x] = st;
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of tile t is in LDS
        __syncthreads();                     // everyone's; the other stage is free
        f16* const sq = smem + (t & 1) * 2 * TILE;
        f16* const sg = sq + TILE;
        const int r0 = ra + t * QT;
        if (t + 1 < nt) {
            f16* const nx = smem + ((t + 1) & 1) * 2 * TILE;
            load(r0 + QT, nx, nx + TILE);
            load_stats(r0 + QT);
        }
        floatx4 s[2][KB], dp[2][KB];
#pragma unroll
        for (int rb2 = 0; rb2 < 2; ++rb2) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) s[rb2][kb] = dp[rb2][kb] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const half8 qf = row_frag<W>(sq, 16 * rb2 + l16, 4 * ks + g);
                const half8 gf = row_frag<W>(sg, 16 * rb2 + l16, 4 * ks + g);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    s[rb2][kb] = mfma16(qf, kf[kb][ks], s[rb2][kb]);
                    dp[rb2][kb] = mfma16(gf, vf[kb][ks], dp[rb2][kb]);
                }
            }
        }
        // every query of the tile sees every key of the block: the first query the last key, the last query the first
        // key outside the sinks
        const int tf = r0 / group, tl = min(r0 + QT, rb) - 1;
        const bool plain = (r0 + QT <= rb) & (klast <= tf) &
                           ((klast < a.sinks) | (max(k0, a.sinks) > tl / group - a.window));
        half8 p[KB], ds[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            float e[8], f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 q = sst[t & 1][16 * (i / 4) + 4 * g + i % 4];
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][kb][i % 4], c2, -q.x));
                f[i] = e[i] * (dp[i / 4][kb][i % 4] - q.y);
            }
            if (!plain) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = r0 + 16 * (i / 4) + 4 * g + i % 4, pos = r / group;
                    const bool see = (r < rb) & (key[kb] <= pos) & ((key[kb] > pos - a.window) | (key[kb] < a.sinks));
                    e[i] = see ? e[i] : 0.0f;
                    f[i] = see ? f[i] : 0.0f;
                }
            }
            p[kb] = as_half8(u32x4{pack_h2(e[0], e[1]), pack_h2(e[2], e[3]), pack_h2(e[4], e[5]), pack_h2(e[6], e[7])});
            ds[kb] = as_half8(u32x4{pack_h2(f[0], f[1]), pack_h2(f[2], f[3]), pack_h2(f[4], f[5]), pack_h2(f[6], f[7])});
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const half8 gt = col_frag<W>(sg, 4 * g + trow, d, tcol), qt = col_frag<W>(sq, 4 * g + trow, d, tcol);
            if (!plain) wild = wild2(qt, wild2(gt, wild));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                gv[d][kb] = mfma16(gt, p[kb], gv[d][kb]);
                gk[d][kb] = mfma16(qt, ds[kb], gk[d][kb]);
            }
        }
    }
    bool again = __any(!((float)wild[0] == 0.0f && (float)wild[1] == 0.0f));
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        if (nparts > 1) {
            // [key][dK, dV]; the parts of blocks that have one come after these
            float* dst = ws + ((int64_t)bc * pt.slots + item) * (2 * KEYS * DH) + ((wave * KB + kb) * 16 + l16) * (2 * DH);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                *reinterpret_cast<floatx4*>(dst + 16 * d + 4 * g) = gk[d][kb];
                *reinterpret_cast<floatx4*>(dst + DH + 16 * d + 4 * g) = gv[d][kb];
            }
            continue;
        }
        if (key[kb] >= a.N) continue;
        const int64_t dst = kv0 + key[kb] * kv_ld;
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (16 * d + 4 * g < a.dh) {
                *reinterpret_cast<uint2*>(a.dK + dst + 16 * d + 4 * g) =
                    uint2{pack_h2(gk[d][kb][0] * a.scale, gk[d][kb][1] * a.scale), pack_h2(gk[d][kb][2] * a.scale, gk[d][kb][3] * a.scale)};
                *reinterpret_cast<uint2*>(a.dV + dst + 16 * d + 4 * g) =
                    uint2{pack_h2(gv[d][kb][0], gv[d][kb][1]), pack_h2(gv[d][kb][2], gv[d][kb][3])};
            }
    }
    if (nparts > 1) again = false;  // window_dkdv_join looks at the sums
    static_assert(4 * sizeof(RowLds) <= sizeof(smem), "a wave's rows");
    if (!__syncthreads_or(again) || !again) return;
#pragma unroll 1
    for (int j = k0 + wave * 16 * KB; j < min(k0 + (wave + 1) * 16 * KB, a.N); ++j)
        dkdv_row(a, ((int64_t)b * a.R + j) * a.KV + c, reinterpret_cast<RowLds*>(smem)[wave], lane);
}

// The sums of the parts of one key, a wave each.  A sum that is not finite may
// be a hidden NaN's work: that key is computed again, row by row.
template <int DH, int KEYS>
__global__ __launch_bounds__(64) void window_dkdv_join(WindowArgs a, Parts pt, int blocks, const float* ws) {
    constexpr int PER = 2 * DH / 64;
    __shared__ RowLds lds;
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
    bool bad = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        bad |= !(fabsf(v[i]) < INFINITY);
        const int d = lane % 32 * PER + i;
        if (d < a.dh) (is_k ? a.dK : a.dV)[row * a.dh + d] = (f16)(is_k ? v[i] * a.scale : v[i]);
    }
    if (__any(bad)) dkdv_row(a, row, lds, lane);
}

// The MFMA kernels' shapes
bool mfma_ok(const WindowArgs& a) {
    if (a.dh % 8 || !aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out)) return false;
    if (a.dO && (!aligned16(a.dO) || !aligned16(a.o) || !aligned16(a.dK) || !aligned16(a.dV))) return false;
    // a tile's rows behind one descriptor
    return (int64_t)a.KV * a.dh * 2 * (BK + 1) < INT32_MAX && (int64_t)a.H * a.dh * 2 * 260 < INT32_MAX;
}
template <class F>
hipError_t by_head64(int dh, F&& f) {
    if (dh <= 64) f(std::integral_constant<int, 64>{});
    else if (dh <= 96) f(std::integral_constant<int, 96>{});
    else if (dh <= 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 256>{});
    return hipGetLastError();
}
template <class F>
hipError_t by_head(int dh, F&& f) {
    if (dh <= 32) f(std::integral_constant<int, 32>{});
    else if (dh <= 64) f(std::integral_constant<int, 64>{});
    else if (dh <= 96) f(std::integral_constant<int, 96>{});
    else if (dh <= 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 256>{});
    return hipGetLastError();
}

}  // namespace

int window_forward(const WindowArgs& args, hipStream_t st) {
    WindowArgs a = args;
    a.big = (int64_t)a.R * a.KV * a.dh * 2 >= INT32_MAX;
    const int64_t rows = (int64_t)a.B * a.N * a.H;
    hipError_t e;
    if (mfma_ok(a)) {
        e = by_head(a.dh, [&](auto dhc) {
            constexpr int DH = decltype(dhc)::value, QB = DH <= 128 ? 2 : 1;
            const int64_t nr = (int64_t)a.N * (a.H / a.KV);
            const int tiles = (int)((nr + 64 * QB - 1) / (64 * QB));
            hipLaunchKernelGGL((window_fwd<DH, QB>), dim3((unsigned)((int64_t)tiles * a.B * a.KV)), dim3(256), 0, st, a, tiles);
        });
    } else {
        hipLaunchKernelGGL(window_fwd_rows, dim3((unsigned)rows), dim3(64), 0, st, a);
        e = hipGetLastError();
    }
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "window_attention launch");
}

namespace {
// dK, dV workgroups: keys of one (64 KB), by head size
constexpr int kv_blocks(int dh) { return dh <= 128 ? 2 : 1; }

Parts parts_for(int B, int N, int KV, int dh, int window, int sinks) {
    const int64_t keys = 64 * kv_blocks(dh);
    Parts p{};
    p.blocks = (int)((N + keys - 1) / keys);
    p.full = window >= N ? p.blocks : (int)std::min<int64_t>(p.blocks, (sinks + keys - 1) / keys);
    // queries that see a block, in key blocks' lengths: the window, or every later one
    const int64_t span = p.full == p.blocks ? p.blocks : ((int64_t)window + keys - 2) / keys + 1;
    auto set = [&](int64_t q) {
        p.q = (int)q;
        p.rest = (int)((span + q - 1) / q);
        p.items = p.before(p.blocks);
        p.slots = p.rest > 1 ? p.items : p.before(p.full);
    };
    // long parts, as few as fill the chip
    int64_t q = p.full == p.blocks ? std::max<int64_t>(1, span / 4) : span;
    set(q);
    while (q > 1 && p.items * B * KV < 768) set(q = q / 2);
    return p;
}
}  // namespace

uint64_t window_bwd_workspace(int B, int N, int H, int KV, int dh, int window, int sinks) {
    if (dh % 8) return 0;
    const Parts p = parts_for(B, N, KV, dh, window, sinks);
    uint64_t row = 0;
    (void)by_head64(dh, [&](auto dhc) { row = 2 * decltype(dhc)::value * sizeof(float); });
    return ((uint64_t)B * N * H + 1) / 2 * 2 * sizeof(float2) + (uint64_t)B * KV * p.slots * 64 * kv_blocks(dh) * row;
}

int window_backward(const WindowArgs& args, void* ws, hipStream_t st) {
    WindowArgs a = args;
    a.big = (int64_t)a.R * a.KV * a.dh * 2 >= INT32_MAX;
    const int64_t rows = (int64_t)a.B * a.N * a.H, kv_rows = (int64_t)a.B * a.R * a.KV;
    hipError_t e;
    if (mfma_ok(a)) {
        // stats first: 8 bytes a row, rounded up so that the sums behind them are aligned
        float2* const stats = (float2*)ws;
        float* const sums = (float*)(stats + (rows + 1) / 2 * 2);
        e = by_head(a.dh, [&](auto dhc) {
            constexpr int DH = decltype(dhc)::value, QB = DH <= 128 ? 2 : 1;
            const int64_t nr = (int64_t)a.N * (a.H / a.KV);
            const int tiles = (int)((nr + 64 * QB - 1) / (64 * QB));
            hipLaunchKernelGGL((window_dq<DH, QB>), dim3((unsigned)((int64_t)tiles * a.B * a.KV)), dim3(256), 0, st, a, tiles, stats);
        });
        const Parts p = parts_for(a.B, a.N, a.KV, a.dh, a.window, a.sinks);
        if (e == hipSuccess)
            e = by_head64(a.dh, [&](auto dhc) {
                constexpr int DH = decltype(dhc)::value, KB = kv_blocks(DH), KEYS = 64 * KB;
                hipLaunchKernelGGL((window_dkdv<DH, KB>), dim3((unsigned)(p.items * a.B * a.KV)), dim3(256), 0, st, a, p, stats, sums);
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

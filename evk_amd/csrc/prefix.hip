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
#include "kernels.h"

#include <algorithm>

#include <math.h>

namespace evkhip {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Own rows that query t of sequence b sees
DEV int own_rows(const PrefixArgs& a, int b, int t) {
    const int64_t p = (int64_t)(a.offsets ? a.offsets[b] : a.p0) + t;
    return (int)(p < 0 ? 0 : p < a.R ? p + 1 : a.R);
}

// ---------------------------------------------------------------------------
// One wave per query row, any head size and alignment.
// ---------------------------------------------------------------------------
constexpr int SMAX = 256;  // largest head size

struct RowLds {
    float x[SMAX], p[64];
    const f16* v[64];
};
DEV void wave_sync() {  // the wave's LDS accesses before this are done
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

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
    float m = -INFINITY, l = 0.0f, o[SMAX / 64] = {};
    for (int64_t i0 = 0; i0 < total; i0 += 64) {
        const int n = (int)min((int64_t)64, total - i0);
        const int64_t j = min(i0 + lane, total - 1);
        float sc = -INFINITY;
        if (lane < n) {
            const f16* const k = at(a.pk, a.k, j);
            sc = 0.0f;
            for (int d = 0; d < dh; ++d) sc += (float)k[d] * s.x[d];
            sc *= a.scale * kLog2e;
        }
        const float m_new = fmaxf(m, wave_max(sc));
        const float keep = m == -INFINITY ? 0.0f : exp2f(m - m_new);
        const float e = lane < n ? exp2f(sc - (m_new == -INFINITY ? 0.0f : m_new)) : 0.0f;
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
            for (int i = 0; i < n; ++i) v += s.p[i] * (float)s.v[i][d];
            o[u] = v;
        }
        wave_sync();
    }
#pragma unroll
    for (int u = 0; u < SMAX / 64; ++u)
        if (lane + 64 * u < dh) a.out[row * dh + lane + 64 * u] = (f16)(total ? o[u] / l : 0.0f);
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.H + h) * a.N + t] = total ? (m + log2f(l)) * kLn2 : -INFINITY;
}

}  // namespace

uint64_t prefix_workspace(int B, int N, int P, int R, int H, int KV, int dh) {
    (void)B, (void)N, (void)P, (void)R, (void)H, (void)KV, (void)dh;
    return 0;
}

int prefix_forward(const PrefixArgs& a, void* ws, hipStream_t st) {
    (void)ws;
    const int64_t rows = (int64_t)a.B * a.N * a.H;
    const int rc = check_grid("prefix_attention", rows, 64);
    if (rc != EVKHIP_OK) return rc;
    hipLaunchKernelGGL(prefix_rows, dim3((unsigned)rows), dim3(64), 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "prefix_attention launch");
}

}  // namespace evkhip

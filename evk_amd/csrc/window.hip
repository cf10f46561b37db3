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
// Position of query t of sequence b.
DEV int position_of(const WindowArgs& a, int b, int t) {
    const int64_t p = (int64_t)(a.offsets ? a.offsets[b] : a.p0) + t;
    return (int)(p < INT32_MAX ? p : INT32_MAX);
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

__global__ __launch_bounds__(64) void window_fwd_simple(WindowArgs a) {
    __shared__ float qs[SMAX], ps[64];
    __shared__ int js[64];
    const int lane = threadIdx.x, dh = a.dh;
    const int64_t row = blockIdx.x;  // ((b N) + t) H + h
    const int h = (int)(row % a.H), t = (int)(row / a.H % a.N), b = (int)(row / a.H / a.N);
    const int64_t kv_ld = (int64_t)a.KV * dh;
    const int64_t kv0 = (int64_t)b * a.R * kv_ld + (int64_t)(h / (a.H / a.KV)) * dh;
    const Span sp = span_of(position_of(a, b, t), a);
    for (int d = lane; d < dh; d += 64) qs[d] = (float)a.q[row * dh + d];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[SMAX / 64] = {};
    for (int i0 = 0; i0 < sp.count(); i0 += 64) {
        const int n = min(64, sp.count() - i0);
        const int j = sp.row(min(i0 + lane, sp.count() - 1));
        const float s = lane < n ? dot_row(a.k + kv0 + j * kv_ld, qs, dh) * a.scale * kLog2e : -INFINITY;
        const float m_new = fmaxf(m, wave_max(s));
        const float keep = m == -INFINITY ? 0.0f : exp2f(m - m_new);
        const float e = lane < n ? exp2f(s - m_new) : 0.0f;
        l = l * keep + wave_sum(e);
        m = m_new;
        ps[lane] = e;
        js[lane] = j;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < SMAX / 64; ++u) {
            const int d = lane + 64 * u;
            if (d >= dh) break;
            float v = o[u] * keep;
            for (int i = 0; i < n; ++i) v += ps[i] * (float)a.v[kv0 + js[i] * kv_ld + d];
            o[u] = v;
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < SMAX / 64; ++u)
        if (lane + 64 * u < dh) a.out[row * dh + lane + 64 * u] = (f16)(l > 0.0f ? o[u] / l : sp.count() ? o[u] : 0.0f);
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.H + h) * a.N + t] = sp.count() ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// dQ of one query row.
__global__ __launch_bounds__(64) void window_dq_simple(WindowArgs a) {
    __shared__ float qs[SMAX], gs[SMAX], ps[64];
    __shared__ int js[64];
    const int lane = threadIdx.x, dh = a.dh;
    const int64_t row = blockIdx.x;
    const int h = (int)(row % a.H), t = (int)(row / a.H % a.N), b = (int)(row / a.H / a.N);
    const int64_t kv_ld = (int64_t)a.KV * dh;
    const int64_t kv0 = (int64_t)b * a.R * kv_ld + (int64_t)(h / (a.H / a.KV)) * dh;
    const Span sp = span_of(position_of(a, b, t), a);
    float dsum = 0.0f;
    for (int d = lane; d < dh; d += 64) {
        qs[d] = (float)a.q[row * dh + d];
        gs[d] = (float)a.dO[row * dh + d];
        dsum += gs[d] * (float)a.o[row * dh + d];
    }
    dsum = wave_sum(dsum);
    __syncthreads();
    const float lse2 = a.lse[((int64_t)b * a.H + h) * a.N + t] * kLog2e;
    float o[SMAX / 64] = {};
    for (int i0 = 0; i0 < sp.count(); i0 += 64) {
        const int n = min(64, sp.count() - i0);
        const int j = sp.row(min(i0 + lane, sp.count() - 1));
        float ds = 0.0f;
        if (lane < n) {
            const float s = dot_row(a.k + kv0 + j * kv_ld, qs, dh);
            ds = exp2f(s * a.scale * kLog2e - lse2) * (dot_row(a.v + kv0 + j * kv_ld, gs, dh) - dsum);
        }
        ps[lane] = ds;
        js[lane] = j;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < SMAX / 64; ++u) {
            const int d = lane + 64 * u;
            if (d >= dh) break;
            for (int i = 0; i < n; ++i) o[u] += ps[i] * (float)a.k[kv0 + js[i] * kv_ld + d];
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < SMAX / 64; ++u)
        if (lane + 64 * u < dh) a.out[row * dh + lane + 64 * u] = (f16)(o[u] * a.scale);
}

// dK and dV of one row: over the queries that see it, 64 (position, head)
// pairs at a time.
__global__ __launch_bounds__(64) void window_dkdv_simple(WindowArgs a) {
    __shared__ float ks[SMAX], vs[SMAX], ps[64], ds_[64];
    __shared__ int64_t rs[64];
    const int lane = threadIdx.x, dh = a.dh, G = a.H / a.KV;
    const int64_t at = blockIdx.x;  // ((b R) + j) KV + c
    const int c = (int)(at % a.KV), j = (int)(at / a.KV % a.R), b = (int)(at / a.KV / a.R);
    for (int d = lane; d < dh; d += 64) {
        ks[d] = (float)a.k[at * dh + d];
        vs[d] = (float)a.v[at * dh + d];
    }
    __syncthreads();
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
            const float s = dot_row(a.q + row * dh, ks, dh);
            float dsum = 0.0f;
            for (int d = 0; d < dh; ++d) dsum += (float)a.dO[row * dh + d] * (float)a.o[row * dh + d];
            p = exp2f((s * a.scale - a.lse[((int64_t)b * a.H + h) * a.N + t]) * kLog2e);
            ds = p * (dot_row(a.dO + row * dh, vs, dh) - dsum);
        }
        ps[lane] = p;
        ds_[lane] = ds;
        rs[lane] = row * dh;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < SMAX / 64; ++u) {
            const int d = lane + 64 * u;
            if (d >= dh) break;
            for (int q = 0; q < n; ++q) {
                gk[u] += ds_[q] * (float)a.q[rs[q] + d];
                gv[u] += ps[q] * (float)a.dO[rs[q] + d];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < SMAX / 64; ++u) {
        const int d = lane + 64 * u;
        if (d >= dh) break;
        a.dK[at * dh + d] = (f16)(gk[u] * a.scale);
        a.dV[at * dh + d] = (f16)gv[u];
    }
}

}  // namespace

int window_forward(const WindowArgs& a, hipStream_t st) {
    const int64_t rows = (int64_t)a.B * a.N * a.H;
    hipLaunchKernelGGL(window_fwd_simple, dim3((unsigned)rows), dim3(64), 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "window_attention launch");
}

int window_backward(const WindowArgs& a, hipStream_t st) {
    const int64_t rows = (int64_t)a.B * a.N * a.H, kv_rows = (int64_t)a.B * a.R * a.KV;
    hipLaunchKernelGGL(window_dkdv_simple, dim3((unsigned)kv_rows), dim3(64), 0, st, a);
    hipLaunchKernelGGL(window_dq_simple, dim3((unsigned)rows), dim3(64), 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "window_attention_bwd launch");
}

}  // namespace evkhip

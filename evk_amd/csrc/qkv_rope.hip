// Norms of queries and keys for each head with the position rotation, the
// values and the cache rows in the same pass, and its gradient (no counterpart
// in the reference, whose rms_norm and rope are passes of their own over whole
// rows).
//
//   y = x r w, r = 1 / sqrt(mean(x^2) + eps) over a head, w the norm's weights;
//   pairs (2 i, 2 i + 1) of y turned by the angle p base^(-2 i / Dh).
// Gradient, with g the output's gradient turned back:
//   dw = sum over rows of g x r,  dx = r (g w - x r^2 mean(g w x)).
//
// Memory-bound: every value read once and written once.  A head lies in LPH
// lanes of eight consecutive values (16-byte accesses at any alignment; the
// last lane of a head size that is no multiple of 8 takes what is left), a
// wave holds 64 / LPH heads of one token at a time and walks the token's heads
// by `per` such groups, so that the angles of its eight values, which are the
// same in every head, are formed once.  Far positions lose the angle in 32
// bits: turns are counted in 64 (p times the frequency that the host computed)
// and only their fraction goes on in 32.
//
// Forward of 8192 tokens of 32 + 8 + 8 heads of 128 values: 42.7 us, 4.7 TB/s
// (a copy of 1 GiB runs at 5.2); of 7996 tokens of 12 + 4 + 4 heads of 64 11.4
// us, 3.6 TB/s, a wave's groups of heads one after another with no load ahead; 16
// single tokens 4.0, a launch.  Gradient of the 7996 tokens 15.9 us, 3.9 TB/s, and
// 3.8 for the weights' sums.
#include "kernels.h"

#include <algorithm>

#include <math.h>

namespace evkhip {

namespace {

// Turns per position of pair i: base^(-2 i / dh) / (2 pi).  A lane multiplies
// its first pair's from the powers of two in i, so that any head size is a few
// arguments.
struct Turns {
    double unit;  // pair 0
    double r[7];  // ratio of pairs 2^k apart
};

Turns turns_of(float base, int dh) {
    static thread_local Turns tab;
    static thread_local float tab_base = 0.0f;
    static thread_local int tab_dh = 0;
    if (tab_base != base || tab_dh != dh) {
        tab.unit = 1.0 / (2.0 * M_PI);
        for (int k = 0; k < 7; ++k) tab.r[k] = pow((double)base, -2.0 * (1 << k) / dh);
        tab_base = base;
        tab_dh = dh;
    }
    return tab;
}

DEV void load_n(const f16* p, int n, float* x) {
    half8 h = {};
    if (n == 8) {
        h = ld_h8(p);
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < n) h[e] = p[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
}
DEV void store_n(f16* p, int n, const float* x) {
    half8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (f16)x[e];
    if (n == 8) {
        st_h8(p, h);
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < n) p[e] = h[e];
    }
}

// What a lane knows of its token: the turned pairs' cosines and sines.  The
// hardware's take turns; over a turn they are within 1.25e-7 of the exact ones
// (measured), half a step of fp16 being 4.9e-4.  By the library's functions the
// 7996 tokens above took 17 us.
struct Angles {
    float cs[4], sn[4];
    DEV void set(const Turns& tn, int i0, int64_t p) {
        double f = tn.unit;
#pragma unroll
        for (int k = 2; k < 7; ++k) f *= (i0 >> (k + 1)) & 1 ? tn.r[k] : 1.0;
        const double p0 = f * (double)p, p1 = p0 * tn.r[0];
        const double t[4] = {p0, p1, p0 * tn.r[1], p1 * tn.r[1]};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float x = (float)(t[u] - floor(t[u]));
            sn[u] = __builtin_amdgcn_sinf(x);
            cs[u] = __builtin_amdgcn_cosf(x);
        }
    }
    DEV void turn(float* y, float sign) const {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float a = y[2 * u], b = y[2 * u + 1], s = sign * sn[u];
            y[2 * u] = a * cs[u] - b * s;
            y[2 * u + 1] = a * s + b * cs[u];
        }
    }
};

template <int LPH>
__global__ __launch_bounds__(256) void qkv_rope_k(QkvRopeArgs a, Turns tn, int per, int splits, int64_t waves) {
    constexpr int HPW = 64 / LPH;
    const int lane = threadIdx.x & 63, HT = a.H + 2 * a.KV, dh = a.dh;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= waves) return;
    const int64_t token = w / splits;
    const int b = (int)(token / a.N), t = (int)(token % a.N);
    const int g0 = (int)(w % splits) * per, g1 = min(g0 + per, (HT + HPW - 1) / HPW);
    const int i0 = (lane % LPH) * 8, n = min(8, dh - i0);
    const int64_t p = (int64_t)(a.offsets ? a.offsets[b] : a.p0) + t;  // past 2^31 for the last offsets
    Angles ang;
    ang.set(tn, i0, a.first + p);
    float wq[8], wk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) wq[e] = wk[e] = 1.0f;
    if (n > 0 && a.wq) load_n(a.wq + i0, n, wq);
    if (n > 0 && a.wk) load_n(a.wk + i0, n, wk);
    for (int g = g0; g < g1; ++g) {
        const int head = g * HPW + lane / LPH;
        const bool ok = head < HT && n > 0;
        float x[8] = {};
        if (ok) load_n(a.qkv + (token * HT + head) * dh + i0, n, x);
        if (head < a.H + a.KV) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
            ss = lanes_sum<LPH>(ss);
            const float r = rsqrtf(ss / (float)dh + a.eps);
            const bool is_q = head < a.H;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= r * (is_q ? wq[e] : wk[e]);
            ang.turn(x, 1.0f);
        }
        if (!ok) continue;
        if (head < a.H) {
            store_n(a.q + (token * a.H + head) * dh + i0, n, x);
        } else if (p >= 0 && p < a.R) {
            const bool is_k = head < a.H + a.KV;
            const int c = head - a.H - (is_k ? 0 : a.KV);
            store_n((is_k ? a.k : a.v) + (((int64_t)b * a.R + p) * a.KV + c) * dh + i0, n, x);
        }
    }
}

// The gradient: a wave takes tokens w, w + waves, ...; the lanes' sums of the
// weights' gradients meet in LDS and go to the workspace, one row of 2 dh sums
// for each workgroup, which qkv_rope_dw_k adds in a fixed order.
template <int LPH>
__global__ __launch_bounds__(256) void qkv_rope_bwd_k(QkvRopeArgs a, Turns tn, float* part) {
    constexpr int HPW = 64 / LPH;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, HT = a.H + 2 * a.KV, dh = a.dh;
    const int64_t tokens = (int64_t)a.B * a.N, waves = (int64_t)gridDim.x * 4;
    const int groups = (HT + HPW - 1) / HPW;
    const int i0 = (lane % LPH) * 8, n = min(8, dh - i0);
    float wq[8], wk[8], sq[8] = {}, sk[8] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) wq[e] = wk[e] = 1.0f;
    if (n > 0 && a.wq) load_n(a.wq + i0, n, wq);
    if (n > 0 && a.wk) load_n(a.wk + i0, n, wk);
    for (int64_t token = (int64_t)blockIdx.x * 4 + wave; token < tokens; token += waves) {
        Angles ang;
        ang.set(tn, i0, a.p0 + (int)(token % a.N));
        for (int g = 0; g < groups; ++g) {
            const int head = g * HPW + lane / LPH;
            const bool ok = head < HT && n > 0, is_q = head < a.H, normed = head < a.H + a.KV;
            const int c = is_q ? head : head - a.H - (normed ? 0 : a.KV);
            const f16* src = is_q ? a.dq : normed ? a.dk : a.dv;
            float gr[8] = {}, x[8] = {};
            if (ok) load_n(src + (token * (is_q ? a.H : a.KV) + c) * dh + i0, n, gr);
            if (normed) {
                if (ok) load_n(a.qkv + (token * HT + head) * dh + i0, n, x);
                ang.turn(gr, -1.0f);
                float ss = 0.0f, gx = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    ss += x[e] * x[e];
                    gx += gr[e] * (is_q ? wq[e] : wk[e]) * x[e];
                }
                ss = lanes_sum<LPH>(ss);
                gx = lanes_sum<LPH>(gx);
                const float r = rsqrtf(ss / (float)dh + a.eps), back = gx / (float)dh * r * r;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float dw = gr[e] * x[e] * r;
                    sq[e] += is_q ? dw : 0.0f;
                    sk[e] += is_q ? 0.0f : dw;
                    gr[e] = r * (gr[e] * (is_q ? wq[e] : wk[e]) - x[e] * back);
                }
            }
            if (ok) store_n(a.dqkv + (token * HT + head) * dh + i0, n, gr);
        }
    }
    if (!part) return;  // launch-uniform: no weight has a gradient
    __shared__ float red[4][HPW][2 * LPH * 8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        red[wave][lane / LPH][i0 + e] = sq[e];
        red[wave][lane / LPH][LPH * 8 + i0 + e] = sk[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * dh; c += 256) {
        const int at = c < dh ? c : LPH * 8 + c - dh;
        float v = 0.0f;
        for (int u = 0; u < 4 * HPW; ++u) v += red[u / HPW][u % HPW][at];
        part[(int64_t)blockIdx.x * 2 * dh + c] = v;
    }
}

// Column c of the partial sums: 64 threads take every 64th row, in order, and
// their sums are added in order.
__global__ __launch_bounds__(1024) void qkv_rope_dw_k(QkvRopeArgs a, const float* part, int rows) {
    __shared__ float red[64][17];
    const int x = threadIdx.x % 16, u = threadIdx.x / 16, c = blockIdx.x * 16 + x;
    float v = 0.0f;
    if (c < 2 * a.dh)
#pragma unroll 4
        for (int r = u; r < rows; r += 64) v += part[(int64_t)r * 2 * a.dh + c];
    red[u][x] = v;
    __syncthreads();
    if (u || c >= 2 * a.dh) return;
    v = 0.0f;
    for (int r = 0; r < 64; ++r) v += red[r][x];
    f16* dst = c < a.dh ? a.dwq : a.dwk;
    if (!dst) return;
    dst += c < a.dh ? c : c - a.dh;
    *dst = (f16)(a.accumulate ? v + (float)*dst : v);
}

// lanes of a head: a power of two of at least dh / 8
int lanes_per_head(int dh) {
    int l = 1;
    while (l * 8 < dh) l *= 2;
    return l;
}

template <class F>
hipError_t by_lanes(int dh, F&& f) {
    switch (lanes_per_head(dh)) {
        case 1: f(std::integral_constant<int, 1>{}); break;
        case 2: f(std::integral_constant<int, 2>{}); break;
        case 4: f(std::integral_constant<int, 4>{}); break;
        case 8: f(std::integral_constant<int, 8>{}); break;
        case 16: f(std::integral_constant<int, 16>{}); break;
        default: f(std::integral_constant<int, 32>{}); break;
    }
    return hipGetLastError();
}

// 7996 tokens, us of the pass and of the weights' sums: 512 workgroups 18.8 and
// 4.1, 1024 15.8 and 3.9, 2048 15.8 and 7.7
int bwd_groups(uint64_t tokens) { return (int)std::min<uint64_t>((tokens + 3) / 4, 1024); }

}  // namespace

uint64_t qkv_rope_bwd_workspace(uint64_t tokens, int dh) { return (uint64_t)bwd_groups(tokens) * 2 * dh * sizeof(float); }

int qkv_rope_forward(const QkvRopeArgs& a, hipStream_t st) {
    const int64_t tokens = (int64_t)a.B * a.N;
    const int rc = check_grid("qkv_norm_rope", (std::max<int64_t>(tokens, 8192) + 3) / 4, 256);
    if (rc != EVKHIP_OK) return rc;
    const Turns tn = turns_of(a.base, a.dh);
    const hipError_t e = by_lanes(a.dh, [&](auto lph) {
        constexpr int LPH = decltype(lph)::value;
        const int groups = (a.H + 2 * a.KV + 64 / LPH - 1) / (64 / LPH);
        // A wave for a part of a token's heads up to 4096 waves, past that one for the token, which forms its angles
        // once (us, split and not: 1 token of 32 + 8 + 8 heads of 128 values 2.7 and 7.2, 64 tokens 2.9 and 8.4, 200
        // tokens 3.6 and 8.5; 1500 tokens of 12 + 4 + 4 heads of 64 4.9 and 4.5).
        int splits = 1;
        while (splits < groups && tokens * splits < 4096) splits = std::min(groups, splits * 2);
        const int per = (groups + splits - 1) / splits;
        splits = (groups + per - 1) / per;
        const int64_t waves = tokens * splits;
        hipLaunchKernelGGL(qkv_rope_k<LPH>, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a, tn, per, splits, waves);
    });
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "qkv_norm_rope launch");
}

int qkv_rope_backward(const QkvRopeArgs& a, float* part, hipStream_t st) {
    const int rows = bwd_groups((uint64_t)a.B * a.N);
    const Turns tn = turns_of(a.base, a.dh);
    hipError_t e = by_lanes(a.dh, [&](auto lph) {
        hipLaunchKernelGGL(qkv_rope_bwd_k<decltype(lph)::value>, dim3(rows), dim3(256), 0, st, a, tn, part);
    });
    if (e == hipSuccess && part) {
        hipLaunchKernelGGL(qkv_rope_dw_k, dim3((2 * a.dh + 15) / 16), dim3(1024), 0, st, a, part, rows);
        e = hipGetLastError();
    }
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "qkv_norm_rope_backward launch");
}

}  // namespace evkhip

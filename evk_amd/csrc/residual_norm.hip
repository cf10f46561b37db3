// Norms after and before a block, with the block's gate and the residual scale,
// in one pass, and its gradient (no counterpart in the reference, whose block
// adds its products to the stream and norms them without weights, a pass each).
//
//   n = y q, q = 1 / sqrt(mean(y^2) + eps)      (post_norm; else n = y)
//   s = a x + g (n wo)                          the stream behind the block
//   u = s r, r = 1 / sqrt(mean(s^2) + eps),  h = u wi   what the next block reads
// With c = dh wi and S = ds + r (c - u mean(c u)), the gradient of s:
//   dx = a S,  dwi = sum dh u,  e = g wo S,  dy = q (e - n mean(e n))
//   P = sum of S n over the rows of a gate:  dg = wo P,  dwo = sum over gates of g P
// so that both gradients come from one sum.  Without y: s = x, which is not
// written.
//
// Memory-bound: every value read once and written once.  A row lies in TPR
// threads' registers, NV vectors of eight values each, at any alignment (the
// last vector takes what is left; narrow rows share a wave: 40000 rows of 256 14 us
// and 30 with gradient, a wave each 21 and 50); weights and gates stay in registers from row
// to row.  The sums of a row are in 32 bits, as is everything between the loads
// and the stores.  8192 rows of 4096: 50 us = 5.3 TB/s (a copy of 1 GiB runs at
// 5.1), the norm alone (no y) 26 = 5.2; 7996 of 768, where the launch counts, 13.8 =
// 3.6; 16 rows 3.8.  Rows that are no multiple of 8, whose last values come one by
// one: 8000 of 1001 15.0 = 4.3 TB/s, of 5001 114 = 2.8 (of 5000 77 = 4.2).
#include "kernels.h"

#include <algorithm>

namespace evkhip {

namespace {

DEV half8 ld_part(const f16* p, int n) {  // n values, the rest zeros
    half8 h = {};
    if (n >= 8) {
        h = ld_h8(p);
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < n) h[e] = p[e];
    }
    return h;
}
DEV void st_part(f16* p, int n, const float (&x)[8]) {
    half8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (f16)x[e];
    if (n >= 8) {
        st_h8(p, h);
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < n) p[e] = h[e];
    }
}
DEV half8 ones() {
    half8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (f16)1.0f;
    return h;
}

constexpr int threads_of(int tpr) { return tpr < 256 ? 256 : tpr; }
constexpr int waves_of(int tpr) { return tpr < 64 ? 1 : tpr / 64; }  // of a row

// Sums over the TPR threads of a row.  Wider rows than a wave meet in LDS, in two
// places in turn: who writes one again has passed the barrier of the other,
// which everyone reaches after reading the first.
template <int TPR>
struct RowSum {
    static constexpr int NW = waves_of(TPR);
    int turn = 0;
    template <int M>
    DEV void operator()(float (&v)[M], float (*lds)[2][NW]) {
#pragma unroll
        for (int i = 0; i < M; ++i) v[i] = TPR < 64 ? lanes_sum<TPR < 64 ? TPR : 1>(v[i]) : wave_add(v[i]);
        if constexpr (NW > 1) {
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < M; ++i) lds[turn][i][wave] = v[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < M; ++i) {
                v[i] = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) v[i] += lds[turn][i][w];
            }
            turn ^= 1;
        }
    }
};

// The stream behind the block, from a row's vectors: s, and n = y q
template <bool Y, int NV>
DEV void stream(const ResidualNormArgs& a, const half8 (&x)[NV], const half8 (&y)[NV], const half8 (&g)[NV], const half8 (&wo)[NV], float q,
                float (&s)[NV][8]) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            s[v][e] = Y ? __builtin_fmaf(a.scale, (float)x[v][e], (float)y[v][e] * q * (float)wo[v][e] * (float)g[v][e]) : (float)x[v][e];
}

template <int TPR, int NV, bool Y>
__global__ __launch_bounds__(threads_of(TPR)) void residual_norm_k(ResidualNormArgs a) {
    constexpr int RPW = threads_of(TPR) / TPR;
    __shared__ float red[2][2][waves_of(TPR)];
    const int t = threadIdx.x % TPR, D = a.D;
    RowSum<TPR> sum;
    int at[NV], n[NV];
    half8 wi[NV], wo[NV], g[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        at[v] = 8 * (t + TPR * v);
        n[v] = D - at[v];
        wi[v] = a.wi ? ld_part(a.wi + at[v], n[v]) : ones();
        wo[v] = a.wo ? ld_part(a.wo + at[v], n[v]) : ones();
        g[v] = a.gate && !a.gate_rows ? ld_part(a.gate + at[v], n[v]) : ones();
    }
    for (int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / TPR; row < a.rows; row += (int64_t)gridDim.x * RPW) {
        const int64_t base = row * D;
        half8 x[NV], y[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            x[v] = ld_part(a.x + base + at[v], n[v]);
            if (Y) y[v] = ld_part(a.y + base + at[v], n[v]);
        }
        if (Y && a.gate_rows)
#pragma unroll
            for (int v = 0; v < NV; ++v) g[v] = ld_part(a.gate + row / a.gate_rows * D + at[v], n[v]);
        float q = 1.0f, ss[1] = {0.0f};
        if (Y && a.post) {
            float yy[1] = {0.0f};
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) yy[0] += (float)y[v][e] * (float)y[v][e];
            sum(yy, red);
            q = rsqrtf(yy[0] / (float)D + a.eps);
        }
        float s[NV][8];
        stream<Y>(a, x, y, g, wo, q, s);
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss[0] += s[v][e] * s[v][e];
        sum(ss, red);
        const float r = rsqrtf(ss[0] / (float)D + a.eps);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (Y) st_part(a.s + base + at[v], n[v], s[v]);
            float h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = s[v][e] * r * (float)wi[v][e];
            st_part(a.h + base + at[v], n[v], h);
        }
    }
}

// The gradient.  A workgroup takes a run of rows of one gate (`parts` runs a
// gate), keeps the columns' sums dh u and S n in registers and leaves them in the
// workspace, one row of 2 D sums, which residual_norm_sums_k adds in a fixed
// order.  A row's sums wait for each other three times; the next row is on its way
// meanwhile.  4096 rows of 4096: 41 us = 4.9 TB/s; 7996 of 768: 20 = 3.8; 8000
// of 5001, with the sums, 205 = 2.3 (of 5000 114 = 4.2).
template <int TPR, int NV, bool Y>
__global__ __launch_bounds__(threads_of(TPR)) void residual_norm_bwd_k(ResidualNormArgs a, int64_t rows_gate, int parts, float* part) {
    constexpr int RPW = threads_of(TPR) / TPR;
    // Room for the weights, the next row and the sums beside a row in the registers of its threads: else the former are read
    // when they are needed and the sums lie in LDS (1000 rows of 16384, both directions: 108 us; all in registers, which then
    // do not suffice, 230).
    constexpr bool ROOM = TPR < 1024;
    __shared__ floatx4 kept[ROOM ? 1 : 4 * NV][ROOM ? 1 : TPR];  // dwi and dsn of a thread's vectors, in halves
    __shared__ float red[2][2][waves_of(TPR)];
    __shared__ float cols[RPW > 1 ? RPW : 1][RPW > 1 ? 2 * TPR * NV * 8 : 1];
    const int t = threadIdx.x % TPR, D = a.D;
    const int64_t gate = blockIdx.x / parts, r0 = blockIdx.x % parts;
    const int64_t first = gate * rows_gate + rows_gate * r0 / parts, end = gate * rows_gate + rows_gate * (r0 + 1) / parts;
    RowSum<TPR> sum;
    int at[NV], n[NV];
    half8 wi[NV], wo[NV], g[NV];
    float dwi[NV][8] = {}, dsn[NV][8] = {};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        at[v] = 8 * (t + TPR * v);
        n[v] = D - at[v];
    }
    auto weights = [&] {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            wi[v] = a.wi ? ld_part(a.wi + at[v], n[v]) : ones();
            wo[v] = a.wo ? ld_part(a.wo + at[v], n[v]) : ones();
            g[v] = a.gate ? ld_part(a.gate + (a.gate_rows ? gate * D : 0) + at[v], n[v]) : ones();
        }
    };
    if (!ROOM)
#pragma unroll
        for (int k = 0; k < 4 * NV; ++k) kept[k][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    auto anew = [](auto&... values) {  // formed anew behind a barrier, not kept as 32 bits across it
        if (!ROOM) (forget(values), ...);
    };
    half8 nx[NV], ny[NV], nds[NV] = {}, ndh[NV];
    auto load = [&](int64_t row) {
        const int64_t base = row * D;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            nx[v] = ld_part(a.x + base + at[v], n[v]);
            if (Y) ny[v] = ld_part(a.y + base + at[v], n[v]);
            ndh[v] = ld_part(a.dh + base + at[v], n[v]);
            if (a.ds) nds[v] = ld_part(a.ds + base + at[v], n[v]);
        }
    };
    const int64_t row0 = first + threadIdx.x / TPR;
    if (ROOM) {
        if (row0 < end) load(row0);
        weights();
    }
    for (int64_t row = row0; row < end; row += RPW) {
        const int64_t base = row * D;
        half8 x[NV], y[NV], ds[NV], dh[NV];
        if (!ROOM) {
            weights();
            load(row);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) x[v] = nx[v], y[v] = ny[v], ds[v] = nds[v], dh[v] = ndh[v];
        if (ROOM && row + RPW < end) load(row + RPW);  // on their way during this row's sums
        float q = 1.0f;
        if (Y && a.post) {
            float yy[1] = {0.0f};
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) yy[0] += (float)y[v][e] * (float)y[v][e];
            sum(yy, red);
            q = rsqrtf(yy[0] / (float)D + a.eps);
        }
        anew(x, y, g, wo);
        float s[NV][8], sc[2] = {0.0f, 0.0f};
        stream<Y>(a, x, y, g, wo, q, s);
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sc[0] += s[v][e] * s[v][e];
                sc[1] += s[v][e] * ((float)dh[v][e] * (float)wi[v][e]);
            }
        sum(sc, red);
        anew(y, ds, dh, wi, g, wo);
        const float r = rsqrtf(sc[0] / (float)D + a.eps), back = sc[1] * r / (float)D;  // mean(c u)
        float en[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float dx[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float u = s[v][e] * r, d = (float)dh[v][e];
                if (ROOM) dwi[v][e] += d * u;
                else dwi[v][e] = d * u;
                const float S = (float)ds[v][e] + r * (d * (float)wi[v][e] - u * back);
                s[v][e] = S;
                dx[e] = (Y ? a.scale : 1.0f) * S;
                if (Y) {
                    const float m = (float)y[v][e] * q;
                    if (ROOM) dsn[v][e] += S * m;
                    else dsn[v][e] = S * m;
                    en[0] += S * (float)g[v][e] * (float)wo[v][e] * m;
                }
            }
            st_part(a.dx + base + at[v], n[v], dx);
            if (!ROOM)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        kept[4 * v + k][t][e] += dwi[v][4 * k + e];
                        if (Y) kept[4 * v + 2 + k][t][e] += dsn[v][4 * k + e];
                    }
        }
        if (!Y) continue;
        if (a.post) sum(en, red);
        anew(y, g, wo);
        const float mean = a.post ? en[0] / (float)D : 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float dy[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) dy[e] = q * (s[v][e] * (float)g[v][e] * (float)wo[v][e] - (float)y[v][e] * q * mean);
            st_part(a.dy + base + at[v], n[v], dy);
        }
    }
    if (!ROOM)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dwi[v][e] = kept[4 * v + e / 4][t][e % 4];
                dsn[v][e] = kept[4 * v + 2 + e / 4][t][e % 4];
            }
    if (!part) return;  // launch-uniform: neither weights nor gates have gradients
    float* const dst = part + (int64_t)blockIdx.x * 2 * D;
    if constexpr (RPW == 1) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (n[v] >= 8) {
                __builtin_memcpy(dst + at[v], dwi[v], 32);
                if (Y) __builtin_memcpy(dst + D + at[v], dsn[v], 32);
            } else {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (e < n[v]) {
                        dst[at[v] + e] = dwi[v][e];
                        if (Y) dst[D + at[v] + e] = dsn[v][e];
                    }
            }
    } else {
        constexpr int W = TPR * NV * 8;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                cols[threadIdx.x / TPR][at[v] + e] = dwi[v][e];
                cols[threadIdx.x / TPR][W + at[v] + e] = dsn[v][e];
            }
        __syncthreads();
        for (int c = threadIdx.x; c < (Y ? 2 : 1) * D; c += threads_of(TPR)) {
            const int from = c < D ? c : W + c - D;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < RPW; ++w) v += cols[w][from];
            dst[c] = v;
        }
    }
}

// Sums over the runs: block (job, 64 columns), job 0 dwi, 1 dwo (and the gradient
// of the one gate that there is), from 2 on the gradients of 64 / lanes gates.  64
// groups of 16 threads, four columns a thread: `lanes` of them (a power of two, no
// more than the runs of a gate need) take a gate's runs in turn, all 64 those of
// dwi and dwo, eight at once, and their sums are added in order.  512 runs of 768, 4
// gates: 5.0 us, 256 of 4096: 5.0, a launch and the latency of what other XCDs wrote.
constexpr int SUM_COLS = 64;
__global__ __launch_bounds__(1024) void residual_norm_sums_k(ResidualNormArgs a, const float* part, int parts, int gates, int blocks, int gate_lanes) {
    __shared__ float red[64][SUM_COLS + 4];
    const int x = threadIdx.x % 16 * 4, u = threadIdx.x / 16, job = blockIdx.x / blocks, c0 = blockIdx.x % blocks * SUM_COLS, D = a.D;
    const int lanes = job < 2 ? 64 : gate_lanes, gate0 = job < 2 ? 0 : (job - 2) * (64 / lanes), gate = gate0 + u / lanes;
    const int64_t r0 = (int64_t)gate * parts + u % lanes, r1 = job < 2 ? (int64_t)gates * parts : gate < gates ? (int64_t)(gate + 1) * parts : 0;
    const int cx = min(c0 + x, max(D - 4, 0));  // the row's last columns are read with those before them
    const float* const src = part + (job ? D : 0) + cx;
    const bool weigh = job == 1 && a.gate_rows;
    float v[4] = {};
    if (D >= 4) {
        constexpr int AHEAD = 8;
        for (int64_t r = r0; r < r1; r += AHEAD * lanes) {
            float p[AHEAD][4];
            half4 g[AHEAD];
            auto at = [&](int k) { return min(r + k * lanes, r1 - 1); };
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) __builtin_memcpy(p[k], src + at(k) * 2 * D, 16);
            if (weigh)
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) __builtin_memcpy(&g[k], a.gate + (int64_t)((int)at(k) / parts) * D + cx, 8);
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (r + k * lanes < r1) v[i] += weigh ? p[k][i] * (float)g[k][i] : p[k][i];
        }
    } else {
        for (int64_t r = r0; r < r1; r += lanes)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (cx + i < D) v[i] += src[r * 2 * D + i] * (weigh ? (float)a.gate[(int64_t)((int)r / parts) * D + cx + i] : 1.0f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (cx + i >= c0) red[u][cx + i - c0] = v[i];
    __syncthreads();
    const int col = threadIdx.x % SUM_COLS, group = threadIdx.x / SUM_COLS, c = c0 + col;
    auto put = [&](f16* out, float sum) {
        if (out) out[c] = (f16)(a.accumulate ? sum + (float)out[c] : sum);
    };
    const float wo = a.wo && c < D ? (float)a.wo[c] : 1.0f;
    if (lanes == 64) {  // four groups each, then the sixteen
        float sum = ((red[4 * group][col] + red[4 * group + 1][col]) + red[4 * group + 2][col]) + red[4 * group + 3][col];
        __syncthreads();
        red[group][col] = sum;
        __syncthreads();
        if (group || c >= D) return;
        sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += red[r][col];
        if (job == 0) return put(a.dwi, sum);
        if (job > 1) return put(a.dgate + (int64_t)gate0 * D, sum * wo);
        put(a.dwo, a.gate && !a.gate_rows ? sum * (float)a.gate[c] : sum);
        if (!a.gate_rows) put(a.dgate, sum * wo);
        return;
    }
    if (c >= D) return;
    for (int g = group; g < 64 / lanes && gate0 + g < gates; g += 16) {
        float sum = 0.0f;
        for (int r = 0; r < lanes; ++r) sum += red[g * lanes + r][col];
        put(a.dgate + (int64_t)(gate0 + g) * D, sum * wo);
    }
}

template <class F>
void by_width(int D, F&& f) {
    if (D <= 64) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    if (D <= 128) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    if (D <= 256) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
    if (D <= 512) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    if (D <= 1024) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    if (D <= 2048) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
    if (D <= 4096) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    if (D <= 8192) return f(std::integral_constant<int, 512>{}, std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
}
static_assert(RESIDUAL_NORM_MOST == 1024 * 2 * 8, "the widest row");

// Runs of rows of one gate: long ones, whose sums cost less to write and add, as
// far as every CU keeps rows in flight (us of the gradient with 256, 512 and 1024
// runs: 7996 rows of 768 30, 27, 34; 4096 rows of 4096 54, 57, 66; 3000 of 8192
// 81, 92, 101), each with a row for all of a workgroup's threads and two at least
// (1, 2 and 4: 64 rows of 4096 12.7, 13.4, 16.8; 256 rows 19.4, 17.0, 19.2)
int64_t runs(int64_t rows, int64_t gates, int D) {
    const int64_t rows_gate = rows / gates, all = D <= 1024 ? 512 : 256;
    int64_t least = 0;
    by_width(D, [&](auto tpr, auto) { least = std::max(2, threads_of(decltype(tpr)::value) / decltype(tpr)::value); });
    return std::max<int64_t>(1, std::min((rows_gate + least - 1) / least, (all + gates - 1) / gates));
}

}  // namespace

uint64_t residual_norm_bwd_workspace(uint64_t rows, uint64_t gates, int D) {
    return gates * runs((int64_t)rows, (int64_t)gates, D) * 2 * D * sizeof(float);
}

int residual_norm_forward(const ResidualNormArgs& a, hipStream_t st) {
    by_width(a.D, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, NT = threads_of(TPR), RPW = NT / TPR;
        const int64_t groups = std::min<int64_t>((a.rows + RPW - 1) / RPW, 1 << 20);
        if (a.y) hipLaunchKernelGGL((residual_norm_k<TPR, NV, true>), dim3((unsigned)groups), dim3(NT), 0, st, a);
        else hipLaunchKernelGGL((residual_norm_k<TPR, NV, false>), dim3((unsigned)groups), dim3(NT), 0, st, a);
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "residual_norm launch");
}

int residual_norm_backward(const ResidualNormArgs& a, float* part, hipStream_t st) {
    const int64_t gates = a.gate_rows ? a.rows / a.gate_rows : 1, parts = runs(a.rows, gates, a.D);
    const int blocks = (a.D + SUM_COLS - 1) / SUM_COLS;
    int lanes = 1;
    while (lanes < 64 && lanes < parts) lanes *= 2;
    const int64_t jobs = 2 + (a.dgate && a.gate_rows ? (gates + 64 / lanes - 1) / (64 / lanes) : 0);
    int rc = EVKHIP_OK;
    by_width(a.D, [&](auto tpr, auto) { rc = check_grid("residual_norm_backward", gates * parts, threads_of(decltype(tpr)::value)); });
    if (rc == EVKHIP_OK && part) rc = check_grid("residual_norm_backward", jobs * blocks, 1024);
    if (rc != EVKHIP_OK) return rc;
    by_width(a.D, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, NT = threads_of(TPR);
        const dim3 grid((unsigned)(gates * parts));
        if (a.y) hipLaunchKernelGGL((residual_norm_bwd_k<TPR, NV, true>), grid, dim3(NT), 0, st, a, a.rows / gates, (int)parts, part);
        else hipLaunchKernelGGL((residual_norm_bwd_k<TPR, NV, false>), grid, dim3(NT), 0, st, a, a.rows / gates, (int)parts, part);
    });
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && part) {
        hipLaunchKernelGGL(residual_norm_sums_k, dim3((unsigned)(jobs * blocks)), dim3(1024), 0, st, a, part, (int)parts, (int)gates, blocks, lanes);
        e = hipGetLastError();
    }
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "residual_norm_backward launch");
}

}  // namespace evkhip

// Log-probabilities of given tokens with the entropy of their distributions and
// the most likely alternatives, and the gradient (no counterpart in the
// reference, whose loss is one mean over all rows).
//
//   m = max l, L = log sum exp(c (l_j - m)),  log p_j = c (l_j - m) - L
//   H = L - sum p_j c (l_j - m)
//   dl_j = c (w ([j = t] - p_j) - e p_j (log p_j + H)), w and e the gradients of
//          log p_t and H
// Differences to the largest logit are formed before they are scaled, so that
// their error is relative to them and not to the logits; m and L are kept apart
// for the gradient, for the same reason.
//
// Memory-bound: every logit read once, a row in the registers of one workgroup
// (ids have 16 bits, so a row is at most 65536 logits).
#include "kernels.h"

#include <math.h>

namespace evkhip {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int CAND = 1024;  // alternatives to choose from

// Order of the alternatives: larger values first, then lower ids, as one number.
// Zeros of both signs are one value, NaN is above all.
DEV uint32_t value_key(f16 h) {
    const uint32_t b = __builtin_bit_cast(uint16_t, h);
    if ((b & 0x7FFFu) > 0x7C00u) return 0xFFFFu;
    if (b == 0x8000u) return 0x8000u;
    return b & 0x8000u ? 0xFFFFu - b : 0x8000u + b;
}
DEV uint32_t order_key(f16 h, int id) { return value_key(h) << 16 | (uint32_t)(0xFFFF - id); }

template <int NW>
DEV float block_sum(float v, float* lds) {
    v = wave_sum(v);
    if (NW == 1) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += lds[w];
    return v;
}
template <int NW>
DEV uint32_t block_max(uint32_t v, uint32_t* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    if (NW == 1) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) v = max(v, lds[w]);
    return v;
}

// The k-th largest of the lanes' 16-bit numbers, k <= 64
DEV uint32_t wave_kth(uint32_t v, int k) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 15; bit >= 0; --bit) {
        const uint32_t up = t | 1u << bit;
        if (__popcll(__ballot(v >= up)) >= k) t = up;
    }
    return t;
}

template <int NT, int NV>
__global__ __launch_bounds__(NT) void token_logprobs_k(TokenLogprobsArgs a) {
    constexpr int NW = NT / 64;
    __shared__ float red[3][NW];
    __shared__ uint32_t redk[2][NW], cand[CAND], count;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, V = a.V;
    const f16* const l = a.logits + row * V;
    const int token = a.tokens[row];
    const float l_t = (float)l[min(token, V - 1)];
    half8 x[NV];
    int n[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int at = 8 * (tid + NT * v);
        n[v] = V - at;
        if (n[v] >= 8) {
            x[v] = ld_h8(l + at);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[v][e] = e < n[v] ? l[at + e] : (f16)-INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, (float)x[v][e]);
    const float mine = m;
    m = wave_max(m);
    if (a.top) {  // this wave's bound from below of the K-th largest logit
        const uint32_t t = wave_kth(value_key((f16)mine), a.top);
        if ((tid & 63) == 0) redk[0][tid >> 6] = t;
    }
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    if (tid == 0) count = 0;
    __syncthreads();
    uint32_t bound = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        m = fmaxf(m, red[0][w]);
        if (a.top) bound = max(bound, redk[0][w]);
    }
    const float c2 = a.scale * kLog2e;
    float sum = 0.0f, dot = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = ((float)x[v][e] - m) * c2, p = __builtin_amdgcn_exp2f(t);
            sum += p;
            dot += p * fmaxf(t, -1000.0f);  // p is 0 from there on, a NaN in t is one in p
        }
    sum = block_sum<NW>(sum, red[1]);
    dot = block_sum<NW>(dot, red[2]);
    const float L = logf(sum);
    if (tid == 0) {
        a.logprobs[row] = token < V ? a.scale * (l_t - m) - L : 0.0f;
        if (a.entropy) a.entropy[row] = L - kLn2 * dot / sum;
        if (a.stats) {
            a.stats[2 * row] = m;
            a.stats[2 * row + 1] = L;
        }
    }
    if (!a.top) return;
    auto put = [&](uint32_t key, int rank) {
        const int id = 0xFFFF - (int)(key & 0xFFFFu);
        a.top_ids[row * a.top + rank] = (uint16_t)id;
        a.top_logprobs[row * a.top + rank] = a.scale * ((float)l[id] - m) - L;
    };
    // Every logit at the bound or above: K at least, seldom more than a few times that.
    if (sum == sum)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n[v] && value_key(x[v][e]) >= bound) {
                    const uint32_t i = atomicAdd(&count, 1u);
                    if (i < CAND) cand[i] = order_key(x[v][e], 8 * (tid + NT * v) + e);
                }
    __syncthreads();
    const uint32_t found = count;
    if (sum == sum && found <= CAND) {  // each one's rank among them
        for (uint32_t i = tid; i < found; i += NT) {
            const uint32_t key = cand[i];
            int rank = 0;
            for (uint32_t j = 0; j < found; ++j) rank += cand[j] > key;
            if (rank < a.top) put(key, rank);
        }
        return;
    }
    // Rows with very many equal logits, or NaN: the largest below the last one, K times.
    uint32_t last = 0;
    for (int rank = 0; rank < a.top; ++rank) {
        uint32_t best = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n[v]) {
                    const uint32_t key = order_key(x[v][e], 8 * (tid + NT * v) + e);
                    if (rank == 0 || key < last) best = max(best, key);
                }
        last = block_max<NW>(best, redk[rank & 1]);
        if (tid == 0) put(last, rank);
    }
}

template <int NT>
__global__ __launch_bounds__(NT) void token_logprobs_bwd_k(TokenLogprobsArgs a, int segments) {
    const int64_t row = blockIdx.x / segments;
    const int seg = blockIdx.x % segments, V = a.V, token = a.tokens[row];
    const float w = a.dlogprobs && token < V ? a.dlogprobs[row] : 0.0f, h = a.dentropy ? a.dentropy[row] : 0.0f;
    const float m = a.stats[2 * row], L = a.stats[2 * row + 1], H = a.dentropy ? a.entropy[row] : 0.0f, c2 = a.scale * kLog2e;
    const f16* const l = a.logits + row * V;
    f16* const d = a.dlogits + row * V;
    const int at = 8 * (threadIdx.x + NT * seg), n = V - at;
    if (n <= 0) return;
    half8 x = {};
    const bool idle = w == 0.0f && h == 0.0f;  // nothing asked of this row: zeros, whatever it holds
    if (!idle) {
        if (n >= 8) {
            x = ld_h8(l + at);
        } else {
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < n) x[e] = l[at + e];
        }
    }
    half8 g;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float t = ((float)x[e] - m) * c2 - L * kLog2e, p = __builtin_amdgcn_exp2f(t);
        const float v = (at + e == token ? w : 0.0f) - p * (w + h * (kLn2 * fmaxf(t, -1000.0f) + H));
        g[e] = (f16)(idle ? 0.0f : a.scale * v);
    }
    if (n >= 8) {
        st_h8(d + at, g);
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < n) d[at + e] = g[e];
    }
}

}  // namespace

int token_logprobs_forward(const TokenLogprobsArgs& a, hipStream_t st) {
    auto go = [&](auto nt, auto nv) {
        hipLaunchKernelGGL((token_logprobs_k<decltype(nt)::value, decltype(nv)::value>), dim3((unsigned)a.rows), dim3(decltype(nt)::value), 0, st, a);
    };
    const int nt = a.V <= 1024 ? 64 : a.V <= 8192 ? 256 : 1024;
    const int rc = check_grid("token_logprobs", a.rows, nt);
    if (rc != EVKHIP_OK) return rc;
    if (a.V <= 1024) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (a.V <= 8192) go(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else if (a.V <= 32768) go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 8>{});
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "token_logprobs launch");
}

int token_logprobs_backward(const TokenLogprobsArgs& a, hipStream_t st) {
    constexpr int NT = 256;
    const int segments = (a.V + 8 * NT - 1) / (8 * NT);
    const int rc = check_grid("token_logprobs_backward", a.rows * segments, NT);
    if (rc != EVKHIP_OK) return rc;
    hipLaunchKernelGGL(token_logprobs_bwd_k<NT>, dim3((unsigned)(a.rows * segments)), dim3(NT), 0, st, a, segments);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "token_logprobs_backward launch");
}

}  // namespace evkhip

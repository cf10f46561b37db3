// Log-probabilities of given tokens with the entropy of their distributions and
// the most likely alternatives, and the gradient (no counterpart in the
// reference, whose loss is one mean over all rows).
//
//   t_j = c2 (l_j - m), m = max l, c2 = c log2(e);  S = sum 2^t_j
//   log p_j = ln 2 (t_j - log2 S),  H = ln 2 (log2 S - sum 2^t_j t_j / S)
//   dl_j = c (w ([j = t] - p_j) - e p_j (log p_j + H)), w and e the gradients of
//          log p_t and H
// Differences to the largest logit are formed before they are scaled: the error
// is relative to them, not to the logits, and the largest has t = 0.  m and log2 S
// are kept apart for the gradient, for the same reason.
//
// Memory-bound: every logit read once, a row in the registers of one workgroup
// (ids have 16 bits, so a row is at most 65536 logits).  2560 rows of 32000: 31 us =
// 5.3 TB/s (a copy of 1 GiB runs at 5.1), with 5 alternatives 37: a reading back of
// the few logits that may be among them, two barriers more.  The gradient 64 us =
// 5.1 TB/s.  Logits whose gradient follows (stats are asked for) are read through
// the caches, others past them: both calls 84 us for 89, the first alone 34 for 33.
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
    if ((b & 0x7FFFu) > 0x7C00u) return 0xFFFEu;
    if (b == 0x8000u) return 0x8000u;
    return b & 0x8000u ? 0xFFFFu - b : 0x8000u + b;
}
DEV uint32_t order_key(f16 h, int id) { return value_key(h) << 16 | (uint32_t)(0xFFFF - id); }

DEV f16 key_value(uint32_t k) { return __builtin_bit_cast(f16, (uint16_t)(k & 0x8000u ? k - 0x8000u : 0xFFFFu - k)); }

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

// The logits i .. i + 7 of a row (i + 8 <= V, or i = 0 of a shorter row)
DEV half8 row_part(const f16* l, int i, int V) {
    if (V >= 8) return ld_h8(l + i);
    half8 h = {};
    for (int e = 0; e < V; ++e) h[e] = l[e];
    return h;
}

// The larger of two pairs of halves, as the instruction has it: the compiler's
// own puts one before it for each side, for NaN that signal.  (One NaN is passed
// over, in a row with NaN the sum is NaN.)
DEV uint32_t pk_max(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(d) : "v"(a), "v"(b));
    return d;
}

template <int NT, int NV>
__global__ __launch_bounds__(NT, NV == 16 ? 4 : 1) void token_logprobs_k(TokenLogprobsArgs a) {
    constexpr int NW = NT / 64, PAIRS = (NV + 1) / 2;
    __shared__ float red[3][NW];
    __shared__ uint32_t redk[2][NW], cand[CAND], count, pairs;
    __shared__ uint16_t list[CAND / 4];
    static_assert(PAIRS * NT <= 65536, "a pair's number");
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, wave = tid >> 6, V = a.V;
    const f16* const l = a.logits + row * V;
    const int token = a.tokens[row];
    // Vector v of this thread holds the logits from(v) .. + 7; the row's last ones are read with those before them, which
    // belong to another thread and are no logits here, like all of a vector past the end.
    auto at = [&](int v) { return 8 * (tid + NT * v); };
    auto from = [&](int v) { return min(at(v), max(V - 8, 0)); };
    auto is = [&](int v, int e) { return (from(v) + e >= at(v)) & (from(v) + e < V); };
    half8 x[NV];
    if (NV == 1 && V < 8) {
        x[0] = row_part(l, 0, V);
    } else if (a.stats) {  // a gradient follows and reads them again
#pragma unroll
        for (int v = 0; v < NV; ++v) x[v] = ld_h8(l + from(v));
    } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) x[v] = ld_once(l + from(v));
    }
    const f16 l_t = l[min(token, V - 1)];
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if ((NV == 1 || v >= NV / 2) && 8 * NT * (v + 1) > V)  // by_vocab: more than half of the places hold logits
#pragma unroll
            for (int e = 0; e < 8; ++e) x[v][e] = is(v, e) ? x[v][e] : (f16)-INFINITY;
    uint32_t most[PAIRS];  // of each two vectors, in halves
    uint32_t top = 0xFC00FC00u;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const u32x4 u = as_u32x4(x[v]);
        const uint32_t w = pk_max(pk_max(u[0], u[1]), pk_max(u[2], u[3]));
        most[v / 2] = v % 2 ? pk_max(most[v / 2], w) : w;
        if (v % 2 || v + 1 == NV) top = pk_max(top, most[v / 2]);
    }
    auto low = [](uint32_t u) { return __builtin_bit_cast(half2_t, u)[0]; };
    auto high = [](uint32_t u) { return __builtin_bit_cast(half2_t, u)[1]; };
    const float mine = fmaxf((float)low(top), (float)high(top));
    float m = wave_top(mine);
    uint32_t bound = 0;
    if (a.top) bound = wave_kth(value_key((f16)mine), a.top);  // this wave's bound from below of the K-th largest logit
    if constexpr (NW > 1) {
        if ((tid & 63) == 0) {
            red[0][wave] = m;
            redk[0][wave] = bound;
        }
        if (tid == 0) count = pairs = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            m = fmaxf(m, red[0][w]);
            bound = max(bound, redk[0][w]);
        }
    } else {
        count = pairs = 0;
    }
    const float c2 = a.scale * kLog2e;
    float sum = 0.0f, dot = 0.0f;
    forget(x);  // else each value is kept as the maximum's pass had it, in as many registers as the reads then wait for
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = ((float)x[v][e] - m) * c2, p = __builtin_amdgcn_exp2f(t);
            sum += p;
            dot = __builtin_fmaf(p, fmaxf(t, -1000.0f), dot);  // p is 0 from there on; 0 times -inf would be NaN
        }
        asm volatile("" : "+v"(sum), "+v"(dot));  // a vector's exponentials end here
    }
    auto block = [&](float v, float* lds) {
        v = wave_add(v);
        if constexpr (NW > 1) {
            if ((tid & 63) == 0) lds[wave] = v;
        }
        return v;
    };
    auto all = [&](float v, const float* lds) {
        if constexpr (NW > 1) {
            v = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += lds[w];
        }
        return v;
    };
    sum = block(sum, red[1]);
    dot = block(dot, red[2]);
    if constexpr (NW > 1) __syncthreads();
    sum = all(sum, red[1]);
    dot = all(dot, red[2]);
    const float L = log2f(sum);
    auto log_p = [&](f16 h) { return kLn2 * (((float)h - m) * c2 - L); };
    if (tid == 0) {
        a.logprobs[row] = token < V ? log_p(l_t) : 0.0f;
        if (a.entropy) a.entropy[row] = kLn2 * (L - dot / sum);
        if (a.stats) {
            a.stats[2 * row] = m;
            a.stats[2 * row + 1] = L;
        }
    }
    if (!a.top) return;
    auto put = [&](uint32_t key, int rank) {
        a.top_ids[row * a.top + rank] = (uint16_t)(0xFFFFu - (key & 0xFFFFu));
        a.top_logprobs[row * a.top + rank] = log_p(key_value(key >> 16));
    };
    // Every logit at the bound or above: K at least, seldom more than a few times that.  A bound of -inf says that a wave
    // holds fewer than K others; then those, and the first ids of the rest.  The few pairs of vectors that hold any are
    // read again, a thread a logit: looking for them in the registers, unrolled, took longer than that (2560 rows of
    // 32000: 47 us, without alternatives 30).
    const f16 least = key_value(bound);
    const bool open = least == (f16)-INFINITY;
    auto takes = [&](f16 v) { return open ? v > least : v >= least; };
    if (sum == sum && __any(takes((f16)mine)))
#pragma unroll
        for (int p = 0; p < PAIRS; ++p)
            if (takes(low(most[p])) | takes(high(most[p]))) {
                const uint32_t i = atomicAdd(&pairs, 1u);
                if (i < CAND / 4) list[i] = (uint16_t)(p * NT + tid);
            }
    __syncthreads();
    const int n_pairs = (int)pairs;
    if (n_pairs <= CAND / 4)
        for (int i = tid; i < 16 * n_pairs; i += NT) {
            const int pair = list[i / 16], id = 8 * (pair % NT + NT * (2 * (pair / NT) + i / 8 % 2)) + i % 8;
            const f16 h = id < V ? l[id] : (f16)-INFINITY;
            if (id < V && takes(h)) {
                const uint32_t k = atomicAdd(&count, 1u);
                if (k < CAND) cand[k] = order_key(h, id);
            }
        }
    __syncthreads();
    const int found = (int)count;
    if (sum == sum && n_pairs <= CAND / 4 && found <= CAND) {  // each one's rank among them
        if (found <= 64) {
            if (wave) return;
            const uint32_t key = tid < found ? cand[tid] : 0u;
            int rank = 0;
            for (int j = 0; j < found; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)key, j) > key;
            if (tid < found && rank < a.top) put(key, rank);
        } else {
            for (int i = tid; i < found; i += NT) {
                const uint32_t key = cand[i];
                int rank = 0;
                for (int j = 0; j < found; ++j) rank += cand[j] > key;
                if (rank < a.top) put(key, rank);
            }
        }
        if (found < a.top && wave == 0) {  // fewer than 32 others: 64 ids hold what is missing
            const f16 h = tid < V ? l[tid] : (f16)0.0f;
            const uint64_t rest = __ballot(h == (f16)-INFINITY);
            const int rank = found + __popcll(rest & ((1ull << tid) - 1));
            if ((rest >> tid & 1) && rank < a.top) put(order_key(h, tid), rank);
        }
        return;
    }
    // Rows with very many equal logits, infinities or NaN: the largest below the last one, K times.
    uint32_t last = 0xFFFFFFFFu;
    for (int rank = 0; rank < a.top; ++rank) {
        uint32_t best = 0;
        for (int i = 8 * tid; i < V; i += 8 * NT) {
            const int i0 = min(i, max(V - 8, 0));
            const half8 h = row_part(l, i0, V);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t key = order_key(h[e], i0 + e);
                best = ((i0 + e < V) & (key < last)) ? max(best, key) : best;
            }
        }
        last = block_max<NW>(best, redk[rank & 1]);
        if (tid == 0) put(last, rank);
    }
}

// The gradient of NV vectors of each thread, all requested before the first is
// used: TPR threads on a segment of a row, short rows several a workgroup.
template <int NT, int TPR, int NV>
__global__ __launch_bounds__(NT) void token_logprobs_bwd_k(TokenLogprobsArgs a, int segments) {
    const int64_t row = TPR < NT ? (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR : blockIdx.x / segments;
    if (TPR < NT && row >= a.rows) return;
    const int seg = TPR < NT ? 0 : blockIdx.x % segments, V = a.V, token = a.tokens[row];
    const float w = a.dlogprobs && token < V ? a.dlogprobs[row] : 0.0f, h = a.dentropy ? a.dentropy[row] : 0.0f;
    const float m = a.stats[2 * row], L = a.stats[2 * row + 1], H = a.dentropy ? a.entropy[row] : 0.0f, c2 = a.scale * kLog2e;
    const f16* const l = a.logits + row * V;
    f16* const d = a.dlogits + row * V;
    auto at = [&](int v) { return 8 * (int)(threadIdx.x % TPR) + 8 * TPR * (NV * seg + v); };
    half8 x[NV];
    const bool idle = w == 0.0f && h == 0.0f;  // nothing asked of this row: zeros, whatever it holds
    if (!idle) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (at(v) + 8 <= V) x[v] = ld_once(l + at(v));
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int n = V - at(v);
        if (n <= 0) break;
        if (n < 8 && !idle) {
#pragma unroll
            for (int e = 0; e < 7; ++e) x[v][e] = e < n ? l[at(v) + e] : (f16)0.0f;
        }
        half8 g;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = ((float)x[v][e] - m) * c2 - L, p = __builtin_amdgcn_exp2f(t);
            const float y = (at(v) + e == token ? w : 0.0f) - p * (w + h * (kLn2 * fmaxf(t, -1000.0f) + H));
            g[e] = (f16)(idle ? 0.0f : a.scale * y);
        }
        if (n >= 8) {
            st_once(d + at(v), g);
        } else {
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < n) d[at(v) + e] = g[e];
        }
    }
}

// Threads and vectors of a row: as few waves as its registers fit.  Their barriers
// cost less than more loads at once save, for few rows too (with 5 alternatives,
// us of 256 threads and of 1024: 64 rows of 32000 8.1 and 9.0, 1024 rows 19.5 and
// 25.1; of 512 threads 4001 rows 64.3, of 256 61.3).  A row pays for all vectors of
// its shape: TB/s of thousands of rows at a shape's end and past it, 4.2 (4000) and
// 2.7 (4200), 4.9 (8000) and 3.1 (9000), 5.0 (16000) and 3.0 (17000), 4.9 (32000) and
// 2.9 (33000); 4.4 at 24000, 3.9 at 50257.
template <class F>
void by_vocab(int V, F&& f) {
#define EVK_SHAPE(NT, NV) f(std::integral_constant<int, NT>{}, std::integral_constant<int, NV>{})
    if (V <= 512) EVK_SHAPE(64, 1);
    else if (V <= 1024) EVK_SHAPE(64, 2);
    else if (V <= 2048) EVK_SHAPE(64, 4);
    else if (V <= 4096) EVK_SHAPE(64, 8);
    else if (V <= 8192) EVK_SHAPE(256, 4);
    else if (V <= 16384) EVK_SHAPE(256, 8);
    else if (V <= 32768) EVK_SHAPE(256, 16);
    else EVK_SHAPE(512, 16);
#undef EVK_SHAPE
}

}  // namespace

int token_logprobs_forward(const TokenLogprobsArgs& a, hipStream_t st) {
    int rc = EVKHIP_OK;
    by_vocab(a.V, [&](auto nt, auto) { rc = check_grid("token_logprobs", a.rows, decltype(nt)::value); });
    if (rc != EVKHIP_OK) return rc;
    by_vocab(a.V, [&](auto nt, auto nv) {
        hipLaunchKernelGGL((token_logprobs_k<decltype(nt)::value, decltype(nv)::value>), dim3((unsigned)a.rows), dim3(decltype(nt)::value), 0, st, a);
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "token_logprobs launch");
}

int token_logprobs_backward(const TokenLogprobsArgs& a, hipStream_t st) {
    constexpr int NT = 256, NV = 2;  // 2560 rows of 32000, us: one vector 80, two 64, four 66, eight 67
    int rc = EVKHIP_OK;
    auto launch = [&](auto tprc) {
        constexpr int TPR = decltype(tprc)::value;
        const int segments = TPR < NT ? 1 : (a.V + 8 * NT * NV - 1) / (8 * NT * NV);
        const int64_t groups = TPR < NT ? (a.rows + NT / TPR - 1) / (NT / TPR) : a.rows * segments;
        rc = check_grid("token_logprobs_backward", groups, NT);
        if (rc == EVKHIP_OK) hipLaunchKernelGGL((token_logprobs_bwd_k<NT, TPR, NV>), dim3((unsigned)groups), dim3(NT), 0, st, a, segments);
    };
    // As few threads as a row fills (us, and with a workgroup a row: 2560 rows of 144 3.3 and 3.9, 65536 12.6 and 47.5, 30000 of
    // 500 15.8 and 29.8, 20000 of 1001 18.5 and 27.4).
    if (a.V <= 256) launch(std::integral_constant<int, 16>{});
    else if (a.V <= 512) launch(std::integral_constant<int, 32>{});
    else if (a.V <= 1024) launch(std::integral_constant<int, 64>{});
    else if (a.V <= 2048) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, NT>{});
    if (rc != EVKHIP_OK) return rc;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EVKHIP_OK : check_hip(e, "token_logprobs_backward launch");
}

}  // namespace evkhip

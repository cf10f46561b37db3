// Tests of evk::ai's grouped-query block operators and their Graph nodes
// (include/evk_ai.h) on the gfx950 kernels, against plain loops in double and
// against the ops of the reference's block where those compute the same.
#include <evk_ai.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#define TEST(expr)                                                            \
    do {                                                                      \
        if (expr) {                                                           \
            std::printf(" TEST(" #expr ") [PASS]\n");                        \
        } else {                                                              \
            std::printf(" TEST(" #expr ") [FAIL] [%s:%d]\n", __FILE__, __LINE__); \
            std::fflush(stdout);                                              \
            std::exit(1);                                                     \
        }                                                                     \
    } while (0)

static void upload(Tensor& t, const std::vector<float>& v) {
    float16_t* h = t.cpu();
    for (size_t i = 0; i < v.size(); ++i) h[i] = float16_t(v[i]);
    t.cpu_upload();
}
static std::vector<float> download(Tensor& t) {
    t.cpu_download();
    const float16_t* h = t.cpu();
    return std::vector<float>(h, h + t.shape.count());
}
static std::vector<float> random_vec(size_t n, uint64_t seed) {
    uint64_t s = seed * 2862933555777941757ull + 3037000493ull;
    std::vector<float> v(n);
    for (float& x : v) {
        s = s * 6364136223846793005ull + 1442695040888963407ull;
        x = float(float16_t(float(int64_t(s >> 40) - (1ll << 23)) / float(1 << 23)));
    }
    return v;
}
static double worst(const std::vector<float>& a, const std::vector<float>& b) {
    double w = a.size() == b.size() ? 0.0 : 1e30;
    for (size_t i = 0; i < a.size() && i < b.size(); ++i) w = std::fmax(w, std::isfinite(a[i]) ? std::fabs(double(a[i]) - b[i]) : 1e30);
    return w;
}
constexpr double kHalf = 1.0 / 2048;  // half a step of fp16, relative

// One head over every earlier position is Graph::causal_attention: outputs and
// gradients of values in [-1, 1].  Each side rounds P (or dS) and its result:
// two roundings of sums of at most sum(P |v|) <= 1 a side; gradients of the
// order of 1 are sums of up to N such terms that were rounded, P summing to at
// most N over the queries of one key.
static void test_window_against_causal_attention(uint32_t B, uint32_t N, uint32_t D) {
    std::printf("test_window_against_causal_attention(%u, %u, %u)\n", B, N, D);
    Graph a, b;
    Tensor *in[2][3], *out[2];
    for (int g = 0; g < 2; ++g) {
        Graph& graph = g ? b : a;
        for (int i = 0; i < 3; ++i) {
            in[g][i] = &graph.tensor({B, N, D}, true);
            upload(*in[g][i], random_vec(B * N * D, 10 + i));
        }
        out[g] = g ? &b.window_attention(*in[g][0], *in[g][1], *in[g][2], D) : &a.causal_attention(*in[g][0], *in[g][1], *in[g][2]);
        // a loss whose gradient reaches every output
        Tensor& target = graph.tensor({B, N, D});
        upload(target, random_vec(B * N * D, 20));
        graph.mse_loss(*out[g], target);
        graph.eval(true);
    }
    TEST(worst(download(*out[0]), download(*out[1])) <= 4 * kHalf);
    for (int i = 0; i < 3; ++i) {
        const std::vector<float> x = download(in[0][i]->grad()), y = download(in[1][i]->grad());
        double size = 0.0, off = 0.0;
        for (size_t j = 0; j < x.size(); ++j) size += double(x[j]) * x[j], off += (double(x[j]) - y[j]) * (double(x[j]) - y[j]);
        // the loss's gradients are near fp16's subnormals (2 / count): steps of 2^-24 besides the relative ones
        TEST(std::sqrt(off) <= 8 * kHalf * std::sqrt(size) + std::sqrt(double(x.size())) * 4 * std::ldexp(1.0, -24));
    }
}

// Sliding window, sinks, groups of heads and offsets in 32-bit storage.
static void test_window_rows() {
    std::printf("test_window_rows()\n");
    const uint32_t B = 2, R = 40, H = 4, KV = 2, dh = 16, W = 7, S = 2;
    Tensor q({B, 1, H * dh}), k({B, R, KV * dh}), v({B, R, KV * dh}), o({B, 1, H * dh}), lse({B, H, 1, 2}), off({B, 2});
    const std::vector<float> qv = random_vec(B * H * dh, 1), kv = random_vec(B * R * KV * dh, 2), vv = random_vec(B * R * KV * dh, 3);
    upload(q, qv), upload(k, kv), upload(v, vv);
    const int32_t pos[2] = {33, 5};
    std::memcpy(off.cpu(), pos, sizeof pos);
    off.cpu_upload();
    evk::ai::window_attention(q, k, v, o, dh, W, S, 0, &off, &lse);
    const std::vector<float> got = download(o);
    lse.cpu_download();
    const float* l = reinterpret_cast<const float*>(lse.cpu());
    double off_o = 0.0, off_l = 0.0;
    for (uint32_t b = 0; b < B; ++b)
        for (uint32_t h = 0; h < H; ++h) {
            std::vector<double> e(R, 0.0), acc(dh, 0.0);
            double sum = 0.0;
            for (int j = 0; j <= pos[b]; ++j) {
                if (!(j > pos[b] - int(W) || j < int(S))) continue;
                double s = 0.0;
                for (uint32_t d = 0; d < dh; ++d) s += double(qv[(b * H + h) * dh + d]) * kv[((b * R + j) * KV + h / (H / KV)) * dh + d];
                e[j] = std::exp(s / std::sqrt(double(dh)));
                sum += e[j];
                for (uint32_t d = 0; d < dh; ++d) acc[d] += e[j] * vv[((b * R + j) * KV + h / (H / KV)) * dh + d];
            }
            for (uint32_t d = 0; d < dh; ++d) off_o = std::fmax(off_o, std::fabs(got[(b * H + h) * dh + d] - acc[d] / sum));
            off_l = std::fmax(off_l, std::fabs(l[b * H + h] - std::log(sum)));
        }
    TEST(off_o <= 2 * kHalf + 1e-5);
    TEST(off_l <= 1e-5);
}

// One head without weights: rms_norm and rope of the reference's block, which
// round once more in between.
static void test_qkv_norm_rope() {
    std::printf("test_qkv_norm_rope()\n");
    const uint32_t B = 2, N = 9, D = 64;
    Graph g;
    Tensor& qkv = g.tensor({B, N, 3 * D}, true);
    const std::vector<float> x = random_vec(B * N * 3 * D, 5);
    upload(qkv, x);
    Graph::Heads heads = g.qkv_norm_rope(qkv, 1, 1, D);
    g.eval();
    Tensor part({B * N, D}), normed({B * N, D}), turned({B, N, D});
    Tensor* outs[3] = {&heads.q, &heads.k, &heads.v};
    for (int i = 0; i < 3; ++i) {
        std::vector<float> p(B * N * D);
        for (uint32_t r = 0; r < B * N; ++r)
            for (uint32_t d = 0; d < D; ++d) p[r * D + d] = x[(r * 3 + i) * D + d];
        if (i < 2) {
            upload(part, p);
            evk::ai::rms_norm(part, normed);
            evk::ai::rope(normed, turned, B, N, D);
            // normalised values of at most sqrt(3): two and one roundings, and rope's angle in 32 bits
            TEST(worst(download(turned), download(*outs[i])) <= 3 * kHalf * 2.5 + 1e-4);
        } else {
            TEST(worst(p, download(*outs[i])) == 0.0);
        }
    }
}

static void test_gated_linear(evk::ai::Activation act) {
    std::printf("test_gated_linear(%d)\n", int(act));
    const uint32_t T = 5, D = 24, F = 40;
    Graph g;
    Tensor& x = g.tensor({T, D}, true);
    Tensor& w = g.tensor({2, D, F}, true);
    const std::vector<float> xv = random_vec(T * D, 7), wv = random_vec(2 * D * F, 8);
    upload(x, xv), upload(w, wv);
    Tensor& h = g.gated_linear(x, w, act);
    Tensor& target = g.tensor({T, F});
    upload(target, random_vec(T * F, 9));
    g.mse_loss(h, target);
    g.eval(true);
    const std::vector<float> got = download(h), dh = download(h.grad()), gx = download(x.grad()), gw = download(w.grad());
    auto f = [&](double a) {
        if (act == evk::ai::Activation::Relu) return a > 0 ? a : 0.0;
        if (act == evk::ai::Activation::Silu) return a / (1 + std::exp(-a));
        return 0.5 * a * (1 + std::tanh(0.7978845608028654 * (a + 0.044715 * a * a * a)));
    };
    std::vector<double> wx(T * D, 0.0), ww(2 * D * F, 0.0);
    double off = 0.0;
    for (uint32_t t = 0; t < T; ++t)
        for (uint32_t c = 0; c < F; ++c) {
            double a = 0.0, u = 0.0;
            for (uint32_t d = 0; d < D; ++d) a += double(xv[t * D + d]) * wv[d * F + c], u += double(xv[t * D + d]) * wv[(D + d) * F + c];
            off = std::fmax(off, std::fabs(got[t * F + c] - f(a) * u) / (1.0 + std::fabs(f(a) * u)));
            const double e = 1e-6, slope = act == evk::ai::Activation::Relu ? double(a > 0) : (f(a + e) - f(a - e)) / (2 * e);
            const double da = dh[t * F + c] * u * slope, du = dh[t * F + c] * f(a);
            for (uint32_t d = 0; d < D; ++d) {
                wx[t * D + d] += da * wv[d * F + c] + du * wv[(D + d) * F + c];
                ww[d * F + c] += xv[t * D + d] * da;
                ww[(D + d) * F + c] += xv[t * D + d] * du;
            }
        }
    TEST(off <= kHalf + 1e-5);
    // three roundings (gate and up, their gradients, the result) of the norm, and subnormal steps
    auto close = [](const std::vector<float>& a, const std::vector<double>& b) {
        double size = 0.0, diff = 0.0;
        for (size_t i = 0; i < a.size(); ++i) size += b[i] * b[i], diff += (a[i] - b[i]) * (a[i] - b[i]);
        return std::sqrt(diff) <= 4 * kHalf * std::sqrt(size) + std::sqrt(double(a.size())) * 4 * std::ldexp(1.0, -24);
    };
    TEST(close(gx, wx));
    TEST(close(gw, ww));
}

// Runs and has gradients everywhere.
static void test_graph_block() {
    std::printf("test_graph_block()\n");
    const uint32_t B = 2, N = 20, D = 32, H = 4, KV = 2, dh = 8, F = 48;
    Graph g;
    Tensor& x = g.tensor({B, N, D}, true);
    Tensor& wqkv = g.tensor({D, (H + 2 * KV) * dh}, true);
    Tensor& nq = g.tensor({dh}, true);
    Tensor& nk = g.tensor({dh}, true);
    Tensor& wo = g.tensor({H * dh, D}, true);
    Tensor& wg = g.tensor({2, D, F}, true);
    Tensor& wd = g.tensor({F, D}, true);
    Tensor* params[] = {&x, &wqkv, &nq, &nk, &wo, &wg, &wd};
    uint64_t seed = 40;
    for (Tensor* p : params) upload(*p, random_vec(p->shape.count(), seed++));
    Graph::Heads heads = g.qkv_norm_rope(g.matmul(g.rms_norm(x), wqkv), H, KV, dh, &nq, &nk);
    Tensor& x1 = g.residual(x, g.matmul(g.window_attention(heads.q, heads.k, heads.v, dh, 6, 1), wo));
    Tensor& y = g.residual(x1, g.matmul(g.gated_linear(g.rms_norm(x1), wg), wd));
    Tensor& target = g.tensor({B, N, D});
    upload(target, random_vec(B * N * D, 60));
    g.mse_loss(y, target);
    g.eval(true);
    for (Tensor* p : params) {
        double sum = 0.0;
        for (float v : download(p->grad())) sum += std::fabs(v);
        TEST(std::isfinite(sum) && sum > 0.0);
    }
    g.step(0.01f);
    g.eval(true);
}

int main() {
    std::setvbuf(stdout, nullptr, _IONBF, 0);
    if (!evk::InitializeEVK(evk::EvkDesc{.applicationName = "evk block tests"})) {
        std::printf("no gfx950 device\n");
        return 2;
    }
    evk::ai::initialize();
    test_window_against_causal_attention(2, 48, 64);
    test_window_against_causal_attention(3, 160, 256);
    test_window_rows();
    test_qkv_norm_rope();
    for (int a = 0; a < 3; ++a) test_gated_linear(evk::ai::Activation(a));
    test_graph_block();
    evk::ai::shutdown();
    std::printf("ALL PASSED\n");
    return 0;
}

// Tests of evk::ai's operators of a group of continuations and their Graph nodes
// (include/evk_ai.h) on the gfx950 kernels, against plain loops in double.
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
static std::vector<float> download32(Tensor& t) {  // 32-bit values in fp16 storage
    t.cpu_download();
    std::vector<float> v(t.shape.count() / 2);
    std::memcpy(v.data(), t.cpu(), v.size() * 4);
    return v;
}
template <class T>
static void upload_raw(Tensor& t, const std::vector<T>& v) {
    std::memcpy(t.cpu(), v.data(), v.size() * sizeof(T));
    t.cpu_upload();
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
constexpr double kHalf = 1.0 / 2048;  // half a step of fp16, relative
// off by two roundings of the norm at most (the result's, and room for the 32-bit sums), and subnormal steps
static bool close(const std::vector<float>& a, const std::vector<double>& b) {
    double size = 0.0, diff = 0.0;
    for (size_t i = 0; i < a.size(); ++i) size += b[i] * b[i], diff += (a[i] - b[i]) * (a[i] - b[i]);
    return a.size() == b.size() && std::sqrt(diff) <= 2 * kHalf * std::sqrt(size) + std::sqrt(double(a.size())) * std::ldexp(1.0, -25);
}

// Both norms with a gate for each sequence, through the Graph, gradients included.
static void test_residual_norm() {
    std::printf("test_residual_norm()\n");
    const uint32_t B = 2, N = 5, D = 40;
    const float scale = 0.5f, eps = 1e-4f;
    Graph g;
    Tensor &x = g.tensor({B, N, D}, true), &y = g.tensor({B, N, D}, true), &wo = g.tensor({D}, true), &gate = g.tensor({B, D}, true),
           &wi = g.tensor({D}, true);
    Tensor* all[] = {&x, &y, &wo, &gate, &wi};
    std::vector<float> v[5];
    for (int i = 0; i < 5; ++i) upload(*all[i], v[i] = random_vec(all[i]->shape.count(), 30 + i));
    Graph::Joined j = g.residual_norm(x, y, &wo, &gate, &wi, scale, true, eps);
    // s reaches a later block, h the next one
    Tensor &t1 = g.tensor({B, N, D}), &t2 = g.tensor({B, N, D});
    upload(t1, random_vec(B * N * D, 50)), upload(t2, random_vec(B * N * D, 51));
    g.mse_loss(j.s, t1), g.mse_loss(j.h, t2);
    g.eval(true);
    const std::vector<float> ds = download(j.s.grad()), dh = download(j.h.grad());
    std::vector<double> ws(B * N * D), wh(B * N * D), dx(B * N * D), dy(B * N * D), dwo(D, 0.0), dg(B * D, 0.0), dwi(D, 0.0);
    for (uint32_t r = 0; r < B * N; ++r) {
        const uint32_t b = r / N, o = r * D;
        double yy = 0, ss = 0, cu = 0, en = 0;
        for (uint32_t d = 0; d < D; ++d) yy += double(v[1][o + d]) * v[1][o + d];
        const double q = 1 / std::sqrt(yy / D + eps);
        for (uint32_t d = 0; d < D; ++d) {
            ws[o + d] = scale * v[0][o + d] + double(v[3][b * D + d]) * v[1][o + d] * q * v[2][d];
            ss += ws[o + d] * ws[o + d];
        }
        const double k = 1 / std::sqrt(ss / D + eps);
        for (uint32_t d = 0; d < D; ++d) {
            wh[o + d] = ws[o + d] * k * v[4][d];
            cu += double(dh[o + d]) * v[4][d] * ws[o + d] * k / D;
        }
        std::vector<double> S(D), e(D);
        for (uint32_t d = 0; d < D; ++d) {
            const double u = ws[o + d] * k, n = v[1][o + d] * q;
            S[d] = ds[o + d] + k * (double(dh[o + d]) * v[4][d] - u * cu);
            e[d] = S[d] * v[3][b * D + d] * v[2][d];
            en += e[d] * n / D;
            dx[o + d] = scale * S[d];
            dwi[d] += double(dh[o + d]) * u;
            dg[b * D + d] += S[d] * n * v[2][d];
            dwo[d] += S[d] * n * v[3][b * D + d];
        }
        for (uint32_t d = 0; d < D; ++d) dy[o + d] = q * (e[d] - v[1][o + d] * q * en);
    }
    TEST(close(download(j.s), ws));
    TEST(close(download(j.h), wh));
    TEST(close(download(x.grad()), dx));
    TEST(close(download(y.grad()), dy));
    TEST(close(download(wo.grad()), dwo));
    TEST(close(download(gate.grad()), dg));
    TEST(close(download(wi.grad()), dwi));
}

// Two sequences behind one prefix, rows of their own up to offsets in 32-bit storage.
static void test_prefix_attention() {
    std::printf("test_prefix_attention()\n");
    const uint32_t B = 2, R = 9, P = 21, H = 4, KV = 2, dh = 16;
    Tensor q({B, 1, H * dh}), pk({P, KV * dh}), pv({P, KV * dh}), k({B, R, KV * dh}), v({B, R, KV * dh}), o({B, 1, H * dh}), lse({B, H, 1, 2}), off({B, 2});
    Tensor* all[] = {&q, &pk, &pv, &k, &v};
    std::vector<float> x[5];
    for (int i = 0; i < 5; ++i) upload(*all[i], x[i] = random_vec(all[i]->shape.count(), 70 + i));
    const std::vector<int32_t> at = {6, -1};  // the second has no rows of its own yet
    upload_raw(off, at);
    evk::ai::prefix_attention(q, pk, pv, k, v, o, dh, 0, &off, &lse);
    const std::vector<float> got = download(o), l = download32(lse);
    double off_o = 0.0, off_l = 0.0;
    for (uint32_t b = 0; b < B; ++b)
        for (uint32_t h = 0; h < H; ++h) {
            const uint32_t c = h / (H / KV);
            std::vector<double> acc(dh, 0.0);
            double sum = 0.0;
            for (int j = 0; j < int(P) + at[b] + 1; ++j) {
                const bool own = j >= int(P);
                const float* kr = own ? &x[3][((b * R + j - P) * KV + c) * dh] : &x[1][(j * KV + c) * dh];
                const float* vr = own ? &x[4][((b * R + j - P) * KV + c) * dh] : &x[2][(j * KV + c) * dh];
                double s = 0.0;
                for (uint32_t d = 0; d < dh; ++d) s += double(x[0][(b * H + h) * dh + d]) * kr[d];
                const double e = std::exp(s / std::sqrt(double(dh)));
                sum += e;
                for (uint32_t d = 0; d < dh; ++d) acc[d] += e * vr[d];
            }
            for (uint32_t d = 0; d < dh; ++d) off_o = std::fmax(off_o, std::fabs(got[(b * H + h) * dh + d] - acc[d] / sum));
            off_l = std::fmax(off_l, std::fabs(l[b * H + h] - std::log(sum)));
        }
    TEST(off_o <= 2 * kHalf + 1e-5);
    TEST(off_l <= 1e-5);
}

// Scores with alternatives, and a policy gradient through the Graph.
static void test_token_logprobs() {
    std::printf("test_token_logprobs()\n");
    const uint32_t B = 2, N = 3, V = 50, K = 4, T = B * N;
    Graph g;
    Tensor &logits = g.tensor({B, N, V}, true), &tokens = g.tensor({B, N}), &dlp = g.tensor({T, 2}), &dent = g.tensor({T, 2});
    std::vector<float> x = random_vec(T * V, 90);
    for (float& f : x) f = float(float16_t(4 * f));
    upload(logits, x);
    const std::vector<uint16_t> ids = {3, 49, 0, 17, 0xFFFF, 8};  // one place without a token
    upload_raw(tokens, ids);
    const std::vector<float> w = {1.0f, -2.0f, 0.5f, 3.0f, 7.0f, -1.0f}, e = {0.1f, 0.0f, -0.2f, 0.3f, 0.1f, 0.0f};
    Graph::Scores sc = g.token_logprobs(logits, tokens, dlp, &dent);
    upload_raw(dlp, w), upload_raw(dent, e);
    g.eval(true);
    Tensor top({T, K}), alt({T, K, 2}), lp({T, 2});
    evk::ai::token_logprobs(logits, tokens, lp, nullptr, &top, &alt);
    const std::vector<float> got = download32(sc.logprobs), ent = download32(sc.entropy), again = download32(lp), a = download32(alt);
    top.cpu_download();
    std::vector<uint16_t> best(T * K);
    std::memcpy(best.data(), top.cpu(), best.size() * 2);
    std::vector<double> want(T * V);
    double off = 0.0;
    bool order = true;
    for (uint32_t r = 0; r < T; ++r) {
        double sum = 0.0, h = 0.0;
        for (uint32_t j = 0; j < V; ++j) sum += std::exp(double(x[r * V + j]));
        auto logp = [&](uint32_t j) { return x[r * V + j] - std::log(sum); };
        for (uint32_t j = 0; j < V; ++j) h -= std::exp(logp(j)) * logp(j);
        const bool there = ids[r] < V;
        off = std::fmax(off, std::fabs(got[r] - (there ? logp(ids[r]) : 0.0)));
        off = std::fmax(off, std::fabs(ent[r] - h));
        off = std::fmax(off, std::fabs(again[r] - got[r]));
        for (uint32_t j = 0; j < V; ++j) {
            const double p = std::exp(logp(j)), wt = there ? w[r] : 0.0;
            want[r * V + j] = wt * ((j == ids[r]) - p) - e[r] * p * (logp(j) + h);
        }
        std::vector<bool> used(V, false);
        for (uint32_t i = 0; i < K; ++i) {
            uint32_t m = V;
            for (uint32_t j = 0; j < V; ++j)
                if (!used[j] && (m == V || x[r * V + j] > x[r * V + m])) m = j;
            used[m] = true;
            order &= best[r * K + i] == m;
            off = std::fmax(off, std::fabs(a[r * K + i] - logp(m)));
        }
    }
    TEST(off <= 2e-5);  // 100 roundings of 32 bits of values up to 10
    TEST(order);
    TEST(close(download(logits.grad()), want));
}

// A run of them as a model's ends: a first norm, a block joined, scored and trained.
static void test_graph_group() {
    std::printf("test_graph_group()\n");
    const uint32_t B = 2, N = 12, D = 32, H = 4, KV = 2, dh = 8, F = 48, V = 60;
    Graph g;
    Tensor &x = g.tensor({B, N, D}, true), &w0 = g.tensor({D}, true), &wqkv = g.tensor({D, (H + 2 * KV) * dh}, true), &po = g.tensor({D}, true),
           &pr = g.tensor({D}, true), &wa = g.tensor({H * dh, D}, true), &wg = g.tensor({2, D, F}, true), &wd = g.tensor({F, D}, true),
           &gate = g.tensor({D}, true), &pr2 = g.tensor({D}, true), &out = g.tensor({D, V}, true), &tokens = g.tensor({B, N}), &dlp = g.tensor({B * N, 2});
    Tensor* params[] = {&x, &w0, &wqkv, &po, &pr, &wa, &wg, &wd, &gate, &pr2, &out};
    uint64_t seed = 40;
    for (Tensor* p : params) upload(*p, random_vec(p->shape.count(), seed++));
    std::vector<uint16_t> ids(B * N);
    for (size_t i = 0; i < ids.size(); ++i) ids[i] = uint16_t(i * 7 % V);
    upload_raw(tokens, ids);
    Graph::Heads heads = g.qkv_norm_rope(g.matmul(g.weighted_norm(x, w0), wqkv), H, KV, dh);
    Graph::Joined a = g.residual_norm(x, g.matmul(g.window_attention(heads.q, heads.k, heads.v, dh), wa), &po, nullptr, &pr);
    Graph::Joined b = g.residual_norm(a.s, g.matmul(g.gated_linear(a.h, wg), wd), nullptr, &gate, &pr2, 1.0f, false);
    Graph::Scores sc = g.token_logprobs(g.matmul(b.h, out), tokens, dlp);
    upload_raw(dlp, std::vector<float>(B * N, -1.0f));
    g.eval(true);
    for (Tensor* p : params) {
        double sum = 0.0;
        for (float v : download(p->grad())) sum += std::fabs(v);
        TEST(std::isfinite(sum) && sum > 0.0);
    }
    for (float v : download32(sc.logprobs)) TEST(v < 0.0f);
    g.step(0.01f);
    g.eval(true);
}

int main() {
    std::setvbuf(stdout, nullptr, _IONBF, 0);
    if (!evk::InitializeEVK(evk::EvkDesc{.applicationName = "evk group tests"})) {
        std::printf("no gfx950 device\n");
        return 2;
    }
    evk::ai::initialize();
    test_residual_norm();
    test_prefix_attention();
    test_token_logprobs();
    test_graph_group();
    evk::ai::shutdown();
    std::printf("ALL PASSED\n");
    return 0;
}

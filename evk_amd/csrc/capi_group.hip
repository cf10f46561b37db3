// C ABI entry points of the operators of a group of continuations of one prompt
// (include/evkhip.h): every check happens on the host before any HIP call.
#include "capi_checks.h"

using namespace evkhip;

namespace {

// Rows of the last dimension; sizes whose product leaves 64 bits are refused.
int rows_of(const char* op, const evkhip_tensor* t, uint64_t* rows) {
    uint64_t all = 1;
    bool none = false, past = false;
    for (uint32_t i = 0; i < t->rank; ++i) {
        none |= t->dims[i] == 0;
        past |= __builtin_mul_overflow(all, (uint64_t)t->dims[i], &all);
    }
    EVK_RETURN_IF(past && !none, EVKHIP_ERR_UNSUPPORTED, "%s: more values than 64 bits count", op);
    *rows = dim_at(t, -1) == 0 ? 0 : none ? 0 : batch_of(t, 1);
    EVK_RETURN_IF(*rows > kMaxRows, EVKHIP_ERR_UNSUPPORTED, "%s: more than 2^30 rows", op);
    return EVKHIP_OK;
}

int check_floats(const char* op, const char* name, const float* p) {
    EVK_RETURN_IF((uintptr_t)p & 3, EVKHIP_ERR_INVALID_ARG, "%s: %s is not 4-byte aligned", op, name);
    return EVKHIP_OK;
}

struct Norm {
    uint64_t rows, gates;
    uint32_t D;
};
int norm_shapes(const char* op, const evkhip_tensor* x, const evkhip_tensor* y, const evkhip_tensor* wo, const evkhip_tensor* gate,
                const evkhip_tensor* wi, float scale, int post, float eps, Norm* s) {
    CHECK(check_tensor(x, op, 1, EVKHIP_MAX_DIMS));
    CHECK(rows_of(op, x, &s->rows));
    s->D = dim_at(x, -1);
    s->gates = 1;
    EVK_RETURN_IF(s->D > (uint32_t)RESIDUAL_NORM_MOST, EVKHIP_ERR_UNSUPPORTED, "%s: rows of %u values, at most %d", op, s->D, RESIDUAL_NORM_MOST);
    if (y) {
        CHECK(check_tensor(y, op, 1, EVKHIP_MAX_DIMS));
        EVK_RETURN_IF(!same_dims(x, y), EVKHIP_ERR_SHAPE, "%s: y must match x", op);
    }
    EVK_RETURN_IF(!y && (wo || gate), EVKHIP_ERR_INVALID_ARG, "%s: a weight or gate of a y that is not there", op);
    EVK_RETURN_IF(!y && scale != 1.0f, EVKHIP_ERR_INVALID_ARG, "%s: residual_scale %g without y", op, scale);
    EVK_RETURN_IF(wo && !post, EVKHIP_ERR_INVALID_ARG, "%s: the weight of a norm that is not there", op);
    CHECK(check_weight(op, "post_weight", wo, s->D));
    CHECK(check_weight(op, "pre_weight", wi, s->D));
    if (gate) {
        CHECK(check_tensor(gate, op, 1, 2));
        EVK_RETURN_IF(dim_at(gate, -1) != s->D, EVKHIP_ERR_SHAPE, "%s: gates of %u values for rows of %u", op, dim_at(gate, -1), s->D);
        if (gate->rank == 2) {
            EVK_RETURN_IF(x->rank < 2 || gate->dims[0] != x->dims[0], EVKHIP_ERR_SHAPE, "%s: %u gates for the %u sequences of x", op, gate->dims[0],
                          x->rank < 2 ? 1 : x->dims[0]);
            s->gates = gate->dims[0];
        }
    }
    EVK_RETURN_IF(!(eps >= 0.0f) || isinf(eps), EVKHIP_ERR_INVALID_ARG, "%s: eps %g", op, eps);
    // as fp16 holds them: s and its square stay inside 32 bits
    const float size = fabsf(scale);
    EVK_RETURN_IF(!(size == 0.0f || (size >= 0x1p-24f && size <= 65504.0f)), EVKHIP_ERR_INVALID_ARG, "%s: residual_scale %g", op, scale);
    return EVKHIP_OK;
}
const f16* data_of(const evkhip_tensor* t) { return t ? (const f16*)t->data : nullptr; }
f16* out_of(const evkhip_tensor* t) { return t ? (f16*)t->data : nullptr; }

ResidualNormArgs norm_args(const Norm& s, const evkhip_tensor* x, const evkhip_tensor* y, const evkhip_tensor* wo, const evkhip_tensor* gate,
                           const evkhip_tensor* wi, float scale, int post, float eps) {
    ResidualNormArgs a{};
    a.x = data_of(x);
    a.y = data_of(y);
    a.wo = data_of(wo);
    a.gate = data_of(gate);
    a.wi = data_of(wi);
    a.rows = (int64_t)s.rows;
    a.gate_rows = gate && gate->rank == 2 ? (int64_t)(s.rows / s.gates) : 0;
    a.D = (int)s.D;
    a.post = post ? 1 : 0;
    a.scale = scale;
    a.eps = eps;
    return a;
}

int logits_shapes(const char* op, const evkhip_tensor* logits, const evkhip_tensor* tokens, float scale, uint64_t* rows) {
    CHECK(check_tensor(logits, op, 1, EVKHIP_MAX_DIMS));
    CHECK(check_tensor(tokens, op, 1, EVKHIP_MAX_DIMS));
    CHECK(rows_of(op, logits, rows));
    const uint32_t V = dim_at(logits, -1);
    EVK_RETURN_IF(V == 0, EVKHIP_ERR_SHAPE, "%s: rows of no logits", op);
    EVK_RETURN_IF(V > LOGPROBS_VOCAB, EVKHIP_ERR_UNSUPPORTED, "%s: %u logits, ids have 16 bits", op, V);
    uint64_t n, all = 1;
    bool past = false;
    for (uint32_t i = 0; i < tokens->rank; ++i) past |= __builtin_mul_overflow(all, (uint64_t)tokens->dims[i], &all);
    n = past ? UINT64_MAX : all;
    EVK_RETURN_IF(n != *rows, EVKHIP_ERR_SHAPE, "%s: %llu tokens for %llu rows", op, (unsigned long long)n, (unsigned long long)*rows);
    EVK_RETURN_IF(!(scale > 0.0f && scale <= 65504.0f && scale >= 0x1p-24f), EVKHIP_ERR_INVALID_ARG, "%s: input_scale %g", op, scale);
    return EVKHIP_OK;
}

// Whether the call takes these sizes; those that it refuses need no workspace.
bool prefix_sizes(uint32_t B, uint32_t N, uint32_t P, uint32_t R, uint32_t H, uint32_t KV, uint32_t dh) {
    return B && N && H && KV && H % KV == 0 && dh && dh <= 256 && N <= kMaxRows && R <= kMaxRows && P <= kMaxRows / KV && (uint64_t)P + R <= kMaxRows &&
           (uint64_t)B * N <= kMaxRows / H && (uint64_t)B * R <= kMaxRows / KV && (uint64_t)H + 2 * KV <= kMaxRows;
}

}  // namespace

extern "C" {

int evkhip_residual_norm(const evkhip_tensor* x, const evkhip_tensor* y, const evkhip_tensor* post_weight, const evkhip_tensor* gate,
                         const evkhip_tensor* pre_weight, const evkhip_tensor* s, const evkhip_tensor* h, float residual_scale, int post_norm,
                         float eps, void* stream) {
    const char* op = "residual_norm";
    Norm n;
    CHECK(norm_shapes(op, x, y, post_weight, gate, pre_weight, residual_scale, post_norm, eps, &n));
    CHECK(check_tensor(h, op, 1, EVKHIP_MAX_DIMS));
    EVK_RETURN_IF(!same_dims(x, h), EVKHIP_ERR_SHAPE, "%s: h must match x", op);
    EVK_RETURN_IF(!s != !y, EVKHIP_ERR_INVALID_ARG, "%s: %s", op, s ? "s without y" : "null s");
    if (s) {
        CHECK(check_tensor(s, op, 1, EVKHIP_MAX_DIMS));
        EVK_RETURN_IF(!same_dims(x, s), EVKHIP_ERR_SHAPE, "%s: s must match x", op);
    }
    CHECK(check_apart(op, {bytes_of("s", s), bytes_of("h", h)},
                      {bytes_of("x", x), bytes_of("y", y), bytes_of("post_weight", post_weight), bytes_of("gate", gate), bytes_of("pre_weight", pre_weight)}));
    if (n.rows == 0 || n.D == 0) return EVKHIP_OK;
    ResidualNormArgs a = norm_args(n, x, y, post_weight, gate, pre_weight, residual_scale, post_norm, eps);
    a.s = out_of(s);
    a.h = out_of(h);
    return residual_norm_forward(a, as_stream(stream));
}

uint64_t evkhip_residual_norm_backward_workspace(uint64_t rows, uint64_t gates, uint32_t d) {
    if (rows == 0 || gates == 0 || d == 0 || rows > kMaxRows || gates > rows || d > (uint32_t)RESIDUAL_NORM_MOST) return 0;
    return residual_norm_bwd_workspace(rows, gates, (int)d);
}

int evkhip_residual_norm_backward(const evkhip_tensor* x, const evkhip_tensor* y, const evkhip_tensor* post_weight, const evkhip_tensor* gate,
                                  const evkhip_tensor* pre_weight, const evkhip_tensor* ds, const evkhip_tensor* dh, const evkhip_tensor* dx,
                                  const evkhip_tensor* dy, const evkhip_tensor* dpost_weight, const evkhip_tensor* dgate,
                                  const evkhip_tensor* dpre_weight, float residual_scale, int post_norm, float eps, int accumulate,
                                  void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* op = "residual_norm_backward";
    Norm n;
    CHECK(norm_shapes(op, x, y, post_weight, gate, pre_weight, residual_scale, post_norm, eps, &n));
    EVK_RETURN_IF(!dy != !y, EVKHIP_ERR_INVALID_ARG, "%s: %s", op, dy ? "dy without y" : "null dy");
    for (const evkhip_tensor* t : {dh, dx}) CHECK(check_tensor(t, op, 1, EVKHIP_MAX_DIMS));
    for (const evkhip_tensor* t : {ds, dy})
        if (t) CHECK(check_tensor(t, op, 1, EVKHIP_MAX_DIMS));
    for (const evkhip_tensor* t : {ds, dh, dx, dy})
        EVK_RETURN_IF(t && !same_dims(x, t), EVKHIP_ERR_SHAPE, "%s: ds, dh, dx and dy must match x", op);
    EVK_RETURN_IF((dpost_weight && !post_weight) || (dgate && !gate) || (dpre_weight && !pre_weight), EVKHIP_ERR_INVALID_ARG,
                  "%s: the gradient of a weight or gate that is not there", op);
    CHECK(check_weight(op, "dpost_weight", dpost_weight, n.D));
    CHECK(check_weight(op, "dpre_weight", dpre_weight, n.D));
    if (dgate) {
        CHECK(check_tensor(dgate, op, 1, 2));
        EVK_RETURN_IF(!same_dims(gate, dgate), EVKHIP_ERR_SHAPE, "%s: dgate must match gate", op);
    }
    const bool sums = dpost_weight || dgate || dpre_weight;
    const uint64_t need = sums ? evkhip_residual_norm_backward_workspace(n.rows, n.gates, n.D) : 0;
    CHECK(check_workspace(op, workspace, workspace_bytes, need));
    CHECK(check_apart(op,
                      {bytes_of("dx", dx), bytes_of("dy", dy), bytes_of("dpost_weight", dpost_weight), bytes_of("dgate", dgate),
                       bytes_of("dpre_weight", dpre_weight), {"the workspace", workspace, need}},
                      {bytes_of("x", x), bytes_of("y", y), bytes_of("post_weight", post_weight), bytes_of("gate", gate),
                       bytes_of("pre_weight", pre_weight), bytes_of("ds", ds), bytes_of("dh", dh)}));
    if (n.D == 0) return EVKHIP_OK;
    if (n.rows == 0) {  // sums over nothing
        for (const evkhip_tensor* w : {dpost_weight, dgate, dpre_weight})
            if (w && !accumulate) CHECK(fill_launch(w->data, 0u, (int64_t)numel(w), aligned16(w->data), as_stream(stream)));
        return EVKHIP_OK;
    }
    ResidualNormArgs a = norm_args(n, x, y, post_weight, gate, pre_weight, residual_scale, post_norm, eps);
    a.ds = data_of(ds);
    a.dh = data_of(dh);
    a.dx = out_of(dx);
    a.dy = out_of(dy);
    a.dwo = out_of(dpost_weight);
    a.dgate = out_of(dgate);
    a.dwi = out_of(dpre_weight);
    a.accumulate = accumulate ? 1 : 0;
    return residual_norm_backward(a, sums ? (float*)workspace : nullptr, as_stream(stream));
}

uint64_t evkhip_prefix_attention_workspace(uint32_t batch, uint32_t n, uint32_t prefix, uint32_t rows, uint32_t heads, uint32_t kv_heads,
                                           uint32_t head_dim) {
    if (!prefix_sizes(batch, n, prefix, rows, heads, kv_heads, head_dim)) return 0;
    return prefix_workspace((int)batch, (int)n, (int)prefix, (int)rows, (int)heads, (int)kv_heads, (int)head_dim);
}

int evkhip_prefix_attention(const evkhip_tensor* q, const evkhip_tensor* prefix_k, const evkhip_tensor* prefix_v, const evkhip_tensor* k,
                            const evkhip_tensor* v, const evkhip_tensor* o, uint32_t head_dim, uint32_t position_offset, const int32_t* offsets,
                            float* lse, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* op = "prefix_attention";
    Heads s;
    CHECK(head_shapes(op, q, k, v, head_dim, &s));
    CHECK(check_tensor(prefix_k, op, 2, 2));
    CHECK(check_tensor(prefix_v, op, 2, 2));
    CHECK(check_tensor(o, op, 3, 3));
    EVK_RETURN_IF(!same_dims(q, o), EVKHIP_ERR_SHAPE, "%s: o must match q", op);
    EVK_RETURN_IF(!same_dims(prefix_k, prefix_v), EVKHIP_ERR_SHAPE, "%s: prefix_k and prefix_v differ", op);
    EVK_RETURN_IF(prefix_k->dims[1] != k->dims[2], EVKHIP_ERR_SHAPE, "%s: rows of %u values in the prefix, %u behind it", op, prefix_k->dims[1], k->dims[2]);
    const uint32_t P = prefix_k->dims[0];
    EVK_RETURN_IF(P > kMaxRows / s.KV || (uint64_t)P + s.R > kMaxRows, EVKHIP_ERR_UNSUPPORTED, "%s: more than 2^30 rows", op);
    CHECK(check_positions(op, s, position_offset, offsets));
    CHECK(check_floats(op, "lse", lse));
    const uint64_t need = evkhip_prefix_attention_workspace(s.B, s.N, P, s.R, s.H, s.KV, head_dim);
    CHECK(check_workspace(op, workspace, workspace_bytes, need));
    CHECK(check_apart(op, {bytes_of("o", o), {"lse", lse, (uint64_t)s.B * s.H * s.N * sizeof(float)}, {"the workspace", workspace, need}},
                      {bytes_of("q", q), bytes_of("prefix_k", prefix_k), bytes_of("prefix_v", prefix_v), bytes_of("k", k), bytes_of("v", v),
                       {"offsets", offsets, s.B * sizeof(int32_t)}}));
    if (s.B == 0 || s.N == 0) return EVKHIP_OK;
    PrefixArgs a{};
    a.q = data_of(q);
    a.pk = data_of(prefix_k);
    a.pv = data_of(prefix_v);
    a.k = data_of(k);
    a.v = data_of(v);
    a.out = out_of(o);
    a.lse = lse;
    a.offsets = offsets;
    a.B = (int)s.B;
    a.N = (int)s.N;
    a.H = (int)s.H;
    a.KV = (int)s.KV;
    a.P = (int)P;
    a.R = (int)s.R;
    a.dh = (int)head_dim;
    a.p0 = (int)position_offset;
    a.scale = 1.0f / sqrtf((float)head_dim);
    return prefix_forward(a, workspace, as_stream(stream));
}

int evkhip_token_logprobs(const evkhip_tensor* logits, const evkhip_tensor* tokens, float* logprobs, float* entropy, const evkhip_tensor* top_ids,
                          float* top_logprobs, float* stats, float input_scale, void* stream) {
    const char* op = "token_logprobs";
    uint64_t rows, top = 0;
    CHECK(logits_shapes(op, logits, tokens, input_scale, &rows));
    EVK_RETURN_IF(rows && !logprobs, EVKHIP_ERR_INVALID_ARG, "%s: null logprobs", op);
    if (top_ids) CHECK(check_tensor(top_ids, op, 1, EVKHIP_MAX_DIMS));
    EVK_RETURN_IF(!top_ids != !top_logprobs && !(top_ids && numel(top_ids) == 0), EVKHIP_ERR_INVALID_ARG,
                  "%s: top_ids and top_logprobs come together", op);
    CHECK(check_floats(op, "logprobs", logprobs));
    CHECK(check_floats(op, "entropy", entropy));
    CHECK(check_floats(op, "top_logprobs", top_logprobs));
    CHECK(check_floats(op, "stats", stats));
    if (top_ids) {
        uint64_t n;
        CHECK(rows_of(op, top_ids, &n));
        top = dim_at(top_ids, -1);
        EVK_RETURN_IF(top && n != rows, EVKHIP_ERR_SHAPE, "%s: alternatives of %llu rows, %llu are there", op, (unsigned long long)n,
                      (unsigned long long)rows);
        EVK_RETURN_IF(top > dim_at(logits, -1), EVKHIP_ERR_SHAPE, "%s: %llu alternatives among %u logits", op, (unsigned long long)top,
                      dim_at(logits, -1));
        EVK_RETURN_IF(top > LOGPROBS_TOP, EVKHIP_ERR_UNSUPPORTED, "%s: %llu alternatives, at most %u", op, (unsigned long long)top, LOGPROBS_TOP);
    }
    CHECK(check_apart(op,
                      {{"logprobs", logprobs, rows * sizeof(float)}, {"entropy", entropy, rows * sizeof(float)}, bytes_of("top_ids", top_ids),
                       {"top_logprobs", top_logprobs, rows * top * sizeof(float)}, {"stats", stats, rows * 2 * sizeof(float)}},
                      {bytes_of("logits", logits), bytes_of("tokens", tokens)}));
    if (rows == 0) return EVKHIP_OK;
    TokenLogprobsArgs a{};
    a.logits = data_of(logits);
    a.tokens = (const uint16_t*)tokens->data;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.stats = stats;
    a.top = (int)top;
    a.top_ids = top ? (uint16_t*)top_ids->data : nullptr;
    a.top_logprobs = top_logprobs;
    a.rows = (int64_t)rows;
    a.V = (int)dim_at(logits, -1);
    a.scale = input_scale;
    return token_logprobs_forward(a, as_stream(stream));
}

int evkhip_token_logprobs_backward(const evkhip_tensor* logits, const evkhip_tensor* tokens, const float* stats, const float* entropy,
                                   const float* dlogprobs, const float* dentropy, const evkhip_tensor* dlogits, float input_scale, void* stream) {
    const char* op = "token_logprobs_backward";
    uint64_t rows;
    CHECK(logits_shapes(op, logits, tokens, input_scale, &rows));
    CHECK(check_tensor(dlogits, op, 1, EVKHIP_MAX_DIMS));
    EVK_RETURN_IF(!same_dims(logits, dlogits), EVKHIP_ERR_SHAPE, "%s: dlogits must match logits", op);
    EVK_RETURN_IF(rows && !stats, EVKHIP_ERR_INVALID_ARG, "%s: null stats", op);
    EVK_RETURN_IF(rows && !dlogprobs && !dentropy, EVKHIP_ERR_INVALID_ARG, "%s: no gradient comes in", op);
    EVK_RETURN_IF(dentropy && !entropy, EVKHIP_ERR_INVALID_ARG, "%s: dentropy needs the forward's entropy", op);
    CHECK(check_floats(op, "stats", stats));
    CHECK(check_floats(op, "entropy", entropy));
    CHECK(check_floats(op, "dlogprobs", dlogprobs));
    CHECK(check_floats(op, "dentropy", dentropy));
    CHECK(check_apart(op, {bytes_of("dlogits", dlogits)},
                      {bytes_of("logits", logits), bytes_of("tokens", tokens), {"stats", stats, rows * 2 * sizeof(float)},
                       {"entropy", entropy, rows * sizeof(float)}, {"dlogprobs", dlogprobs, rows * sizeof(float)},
                       {"dentropy", dentropy, rows * sizeof(float)}}));
    if (rows == 0) return EVKHIP_OK;
    TokenLogprobsArgs a{};
    a.logits = data_of(logits);
    a.tokens = (const uint16_t*)tokens->data;
    a.stats = const_cast<float*>(stats);
    a.entropy = const_cast<float*>(entropy);
    a.dlogprobs = dlogprobs;
    a.dentropy = dentropy;
    a.dlogits = out_of(dlogits);
    a.rows = (int64_t)rows;
    a.V = (int)dim_at(logits, -1);
    a.scale = input_scale;
    return token_logprobs_backward(a, as_stream(stream));
}

}  // extern "C"

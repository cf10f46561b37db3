// C ABI entry points of the grouped-query block's operators (include/evkhip.h):
// every check happens on the host before any HIP call.
#include "kernels.h"

#include <math.h>

#include <initializer_list>

using namespace evkhip;

#define CHECK(expr)          \
    do {                     \
        int _rc = (expr);    \
        if (_rc) return _rc; \
    } while (0)

namespace {

constexpr uint32_t kMaxRows = 1u << 30;  // positions, rows, tokens: 32-bit arithmetic with room
static_assert(kMaxRows <= WINDOW_MOST, "no window");

bool same_dims(const evkhip_tensor* a, const evkhip_tensor* b) {
    if (a->rank != b->rank) return false;
    for (uint32_t i = 0; i < a->rank; ++i)
        if (a->dims[i] != b->dims[i]) return false;
    return true;
}

struct Bytes {
    const char* name;
    const void* p;
    uint64_t n;
};
Bytes bytes_of(const char* name, const evkhip_tensor* t) {
    return {name, t ? t->data : nullptr, t ? numel(t) * sizeof(f16) : 0};
}
// Every output apart from every input, from the other outputs and the workspace.
int check_apart(const char* op, std::initializer_list<Bytes> outs, std::initializer_list<Bytes> ins) {
    auto meet = [](const Bytes& a, const Bytes& b) {
        const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
        return a.p && b.p && a.n && b.n && x < y + b.n && y < x + a.n;
    };
    for (const Bytes* o = outs.begin(); o != outs.end(); ++o) {
        for (const Bytes& i : ins)
            EVK_RETURN_IF(meet(*o, i), EVKHIP_ERR_INVALID_ARG, "%s: %s overlaps %s", op, o->name, i.name);
        for (const Bytes* q = o + 1; q != outs.end(); ++q)
            EVK_RETURN_IF(meet(*o, *q), EVKHIP_ERR_INVALID_ARG, "%s: %s overlaps %s", op, o->name, q->name);
    }
    return EVKHIP_OK;
}

int check_workspace(const char* op, const void* p, uint64_t have, uint64_t need) {
    EVK_RETURN_IF(need && (!p || have < need), EVKHIP_ERR_INVALID_ARG, "%s: the workspace holds %llu bytes, %llu are needed",
                  op, (unsigned long long)(p ? have : 0), (unsigned long long)need);
    EVK_RETURN_IF(need && !aligned16(p), EVKHIP_ERR_INVALID_ARG, "%s: the workspace is not 16-byte aligned", op);
    return EVKHIP_OK;
}

int check_weight(const char* op, const char* name, const evkhip_tensor* w, uint32_t head_dim) {
    if (!w) return EVKHIP_OK;
    CHECK(check_tensor(w, name, 1, 1));
    EVK_RETURN_IF(w->dims[0] != head_dim, EVKHIP_ERR_SHAPE, "%s: %s must hold head_dim = %u values", op, name, head_dim);
    return EVKHIP_OK;
}

struct Heads {
    uint32_t B, N, R, H, KV;
};
// q (B,N,H dh); k, v (B,R,KV dh)
int head_shapes(const char* op, const evkhip_tensor* q, const evkhip_tensor* k, const evkhip_tensor* v, uint32_t dh,
                Heads* s) {
    CHECK(check_tensor(q, op, 3, 3));
    CHECK(check_tensor(k, op, 3, 3));
    CHECK(check_tensor(v, op, 3, 3));
    EVK_RETURN_IF(dh == 0, EVKHIP_ERR_INVALID_ARG, "%s: head_dim is 0", op);
    EVK_RETURN_IF(dh > 256, EVKHIP_ERR_UNSUPPORTED, "%s: head_dim %u > 256", op, dh);
    EVK_RETURN_IF(!same_dims(k, v), EVKHIP_ERR_SHAPE, "%s: k and v differ", op);
    EVK_RETURN_IF(k->dims[0] != q->dims[0], EVKHIP_ERR_SHAPE, "%s: %u sequences of q, %u of k", op, q->dims[0], k->dims[0]);
    EVK_RETURN_IF(q->dims[2] == 0 || k->dims[2] == 0 || q->dims[2] % dh || k->dims[2] % dh, EVKHIP_ERR_SHAPE,
                  "%s: rows of %u and %u values are no heads of %u", op, q->dims[2], k->dims[2], dh);
    *s = {q->dims[0], q->dims[1], k->dims[1], q->dims[2] / dh, k->dims[2] / dh};
    EVK_RETURN_IF(s->H % s->KV, EVKHIP_ERR_SHAPE, "%s: %u query heads do not share %u key heads evenly", op, s->H, s->KV);
    EVK_RETURN_IF((uint64_t)s->B * s->N * s->H > kMaxRows || (uint64_t)s->B * s->R * s->KV > kMaxRows || s->R > kMaxRows ||
                      s->N > kMaxRows || (uint64_t)s->H + 2 * s->KV > kMaxRows,
                  EVKHIP_ERR_UNSUPPORTED, "%s: more than 2^30 rows", op);
    return EVKHIP_OK;
}

// Positions of N tokens among R rows
int check_positions(const char* op, const Heads& s, uint32_t offset, const int32_t* offsets) {
    EVK_RETURN_IF(offsets && offset, EVKHIP_ERR_INVALID_ARG, "%s: position_offset %u besides offsets", op, offset);
    EVK_RETURN_IF(offsets && ((uintptr_t)offsets & 3), EVKHIP_ERR_INVALID_ARG, "%s: offsets are not 4-byte aligned", op);
    EVK_RETURN_IF(!offsets && (uint64_t)offset + s.N > s.R, EVKHIP_ERR_SHAPE, "%s: positions %u..%llu exceed the %u rows", op,
                  offset, (unsigned long long)offset + s.N, s.R);
    return EVKHIP_OK;
}

int check_norm(const char* op, float eps, float base) {
    EVK_RETURN_IF(!(eps >= 0.0f) || isinf(eps), EVKHIP_ERR_INVALID_ARG, "%s: eps %g", op, eps);
    EVK_RETURN_IF(!(base > 0.0f) || isinf(base), EVKHIP_ERR_INVALID_ARG, "%s: rotary_base %g", op, base);
    return EVKHIP_OK;
}

int clamp_int(uint32_t v) { return v > (uint32_t)INT32_MAX ? INT32_MAX : (int)v; }
int window_rows(uint32_t window) { return (int)(window && window < WINDOW_MOST ? window : WINDOW_MOST); }

// Whether the call takes these sizes; those that it refuses need no workspace.
bool window_sizes(uint32_t B, uint32_t N, uint32_t R, uint32_t H, uint32_t KV, uint32_t dh) {
    return B && N && R && H && KV && H % KV == 0 && dh && dh <= 256 && N <= kMaxRows && R <= kMaxRows &&
           (uint64_t)B * N <= kMaxRows / H && (uint64_t)B * R <= kMaxRows / KV;
}

WindowArgs window_args(const Heads& s, uint32_t dh, uint32_t window, uint32_t sinks) {
    WindowArgs a{};
    a.B = (int)s.B;
    a.N = (int)s.N;
    a.H = (int)s.H;
    a.KV = (int)s.KV;
    a.R = (int)s.R;
    a.dh = (int)dh;
    a.window = window_rows(window);
    a.far = window ? (int64_t)window - a.window : 1LL << 40;
    a.sinks = clamp_int(sinks);
    a.scale = 1.0f / sqrtf((float)dh);
    return a;
}

struct Gated {
    uint64_t T;
    uint32_t D, F;
};
// x (...,D), w (2,D,F), h (...,F), gate_up (2,...,F)
int gated_shapes(const char* op, const evkhip_tensor* x, const evkhip_tensor* w, const evkhip_tensor* h,
                 const evkhip_tensor* gate_up, int act, Gated* s) {
    CHECK(check_tensor(x, op, 1, EVKHIP_MAX_DIMS));
    CHECK(check_tensor(w, op, 3, 3));
    CHECK(check_tensor(h, op, 1, EVKHIP_MAX_DIMS));
    EVK_RETURN_IF(act < EVKHIP_ACT_SILU || act > EVKHIP_ACT_RELU, EVKHIP_ERR_INVALID_ARG, "%s: activation %d", op, act);
    EVK_RETURN_IF(w->dims[0] != 2, EVKHIP_ERR_SHAPE, "%s: w must be (2,D,F), its first dimension is %u", op, w->dims[0]);
    *s = {batch_of(x, 1), w->dims[1], w->dims[2]};
    EVK_RETURN_IF(dim_at(x, -1) != s->D, EVKHIP_ERR_SHAPE, "%s: rows of %u values, w takes %u", op, dim_at(x, -1), s->D);
    EVK_RETURN_IF(dim_at(h, -1) != s->F || batch_of(h, 1) != s->T, EVKHIP_ERR_SHAPE, "%s: h must be (%llu,%u)", op,
                  (unsigned long long)s->T, s->F);
    if (gate_up) {
        CHECK(check_tensor(gate_up, op, 2, EVKHIP_MAX_DIMS));
        EVK_RETURN_IF(gate_up->dims[0] != 2 || dim_at(gate_up, -1) != s->F || numel(gate_up) != 2 * s->T * s->F,
                      EVKHIP_ERR_SHAPE, "%s: gate_up must be (2,%llu,%u)", op, (unsigned long long)s->T, s->F);
    }
    EVK_RETURN_IF(s->T > kMaxRows || s->D > kMaxRows || s->F > kMaxRows / 2, EVKHIP_ERR_UNSUPPORTED, "%s: more than 2^30 rows", op);
    return EVKHIP_OK;
}

}  // namespace

extern "C" {

int evkhip_qkv_norm_rope(const evkhip_tensor* qkv, const evkhip_tensor* q_weight, const evkhip_tensor* k_weight,
                         const evkhip_tensor* q, const evkhip_tensor* k, const evkhip_tensor* v, uint32_t head_dim,
                         float eps, float rotary_base, uint32_t position_offset, const int32_t* offsets,
                         void* stream) {
    const char* op = "qkv_norm_rope";
    Heads s;
    CHECK(check_tensor(qkv, op, 3, 3));
    CHECK(head_shapes(op, q, k, v, head_dim, &s));
    EVK_RETURN_IF(head_dim % 2, EVKHIP_ERR_SHAPE, "%s: head_dim %u must be even", op, head_dim);
    EVK_RETURN_IF(qkv->dims[0] != s.B || qkv->dims[1] != s.N || (uint64_t)qkv->dims[2] != ((uint64_t)s.H + 2 * s.KV) * head_dim,
                  EVKHIP_ERR_SHAPE, "%s: qkv must be (%u,%u,%llu)", op, s.B, s.N,
                  (unsigned long long)((uint64_t)s.H + 2 * s.KV) * head_dim);
    CHECK(check_weight(op, "q_weight", q_weight, head_dim));
    CHECK(check_weight(op, "k_weight", k_weight, head_dim));
    CHECK(check_norm(op, eps, rotary_base));
    CHECK(check_positions(op, s, position_offset, offsets));
    CHECK(check_apart(op, {bytes_of("q", q), bytes_of("k", k), bytes_of("v", v)},
                      {bytes_of("qkv", qkv), bytes_of("q_weight", q_weight), bytes_of("k_weight", k_weight),
                       {"offsets", offsets, s.B * sizeof(int32_t)}}));
    if (s.B == 0 || s.N == 0) return EVKHIP_OK;
    QkvRopeArgs a{};
    a.qkv = (const f16*)qkv->data;
    a.wq = q_weight ? (const f16*)q_weight->data : nullptr;
    a.wk = k_weight ? (const f16*)k_weight->data : nullptr;
    a.q = (f16*)q->data;
    a.k = (f16*)k->data;
    a.v = (f16*)v->data;
    a.offsets = offsets;
    a.B = (int)s.B;
    a.N = (int)s.N;
    a.H = (int)s.H;
    a.KV = (int)s.KV;
    a.R = (int)s.R;
    a.dh = (int)head_dim;
    a.p0 = (int)position_offset;
    a.eps = eps;
    a.base = rotary_base;
    return qkv_rope_forward(a, as_stream(stream));
}

uint64_t evkhip_qkv_norm_rope_backward_workspace(uint64_t tokens, uint32_t head_dim) {
    return tokens == 0 || head_dim > 256 ? 0 : qkv_rope_bwd_workspace(tokens, (int)head_dim);
}

int evkhip_qkv_norm_rope_backward(const evkhip_tensor* qkv, const evkhip_tensor* q_weight,
                                  const evkhip_tensor* k_weight, const evkhip_tensor* dq, const evkhip_tensor* dk,
                                  const evkhip_tensor* dv, const evkhip_tensor* dqkv, const evkhip_tensor* dq_weight,
                                  const evkhip_tensor* dk_weight, uint32_t head_dim, float eps, float rotary_base,
                                  uint32_t position_offset, int accumulate, void* workspace,
                                  uint64_t workspace_bytes, void* stream) {
    const char* op = "qkv_norm_rope_backward";
    Heads s;
    CHECK(check_tensor(qkv, op, 3, 3));
    CHECK(check_tensor(dqkv, op, 3, 3));
    CHECK(head_shapes(op, dq, dk, dv, head_dim, &s));
    EVK_RETURN_IF(head_dim % 2, EVKHIP_ERR_SHAPE, "%s: head_dim %u must be even", op, head_dim);
    EVK_RETURN_IF(s.R != s.N, EVKHIP_ERR_SHAPE, "%s: dk and dv must hold %u rows", op, s.N);
    EVK_RETURN_IF(qkv->dims[0] != s.B || qkv->dims[1] != s.N || (uint64_t)qkv->dims[2] != ((uint64_t)s.H + 2 * s.KV) * head_dim,
                  EVKHIP_ERR_SHAPE, "%s: qkv must be (%u,%u,%llu)", op, s.B, s.N,
                  (unsigned long long)((uint64_t)s.H + 2 * s.KV) * head_dim);
    EVK_RETURN_IF(!same_dims(qkv, dqkv), EVKHIP_ERR_SHAPE, "%s: dqkv must match qkv", op);
    CHECK(check_weight(op, "q_weight", q_weight, head_dim));
    CHECK(check_weight(op, "k_weight", k_weight, head_dim));
    CHECK(check_weight(op, "dq_weight", dq_weight, head_dim));
    CHECK(check_weight(op, "dk_weight", dk_weight, head_dim));
    EVK_RETURN_IF((dq_weight && !q_weight) || (dk_weight && !k_weight), EVKHIP_ERR_INVALID_ARG,
                  "%s: the gradient of a weight that is not there", op);
    CHECK(check_norm(op, eps, rotary_base));
    EVK_RETURN_IF((uint64_t)position_offset + s.N > kMaxRows, EVKHIP_ERR_UNSUPPORTED, "%s: positions past 2^30", op);
    const uint64_t need = dq_weight || dk_weight
                              ? evkhip_qkv_norm_rope_backward_workspace((uint64_t)s.B * s.N, head_dim) : 0;
    CHECK(check_workspace(op, workspace, workspace_bytes, need));
    CHECK(check_apart(op, {bytes_of("dqkv", dqkv), bytes_of("dq_weight", dq_weight), bytes_of("dk_weight", dk_weight),
                           {"the workspace", workspace, need}},
                      {bytes_of("qkv", qkv), bytes_of("q_weight", q_weight), bytes_of("k_weight", k_weight),
                       bytes_of("dq", dq), bytes_of("dk", dk), bytes_of("dv", dv)}));
    if (s.B == 0 || s.N == 0) {  // sums over nothing
        for (const evkhip_tensor* w : {dq_weight, dk_weight})
            if (w && !accumulate) CHECK(fill_launch(w->data, 0u, head_dim, aligned16(w->data), as_stream(stream)));
        return EVKHIP_OK;
    }
    QkvRopeArgs a{};
    a.qkv = (const f16*)qkv->data;
    a.wq = q_weight ? (const f16*)q_weight->data : nullptr;
    a.wk = k_weight ? (const f16*)k_weight->data : nullptr;
    a.dq = (const f16*)dq->data;
    a.dk = (const f16*)dk->data;
    a.dv = (const f16*)dv->data;
    a.dqkv = (f16*)dqkv->data;
    a.dwq = dq_weight ? (f16*)dq_weight->data : nullptr;
    a.dwk = dk_weight ? (f16*)dk_weight->data : nullptr;
    a.B = (int)s.B;
    a.N = (int)s.N;
    a.H = (int)s.H;
    a.KV = (int)s.KV;
    a.R = (int)s.N;
    a.dh = (int)head_dim;
    a.p0 = (int)position_offset;
    a.eps = eps;
    a.base = rotary_base;
    a.accumulate = accumulate ? 1 : 0;
    return qkv_rope_backward(a, need ? (float*)workspace : nullptr, as_stream(stream));
}

uint64_t evkhip_window_attention_workspace(uint32_t batch, uint32_t n, uint32_t rows, uint32_t heads,
                                           uint32_t kv_heads, uint32_t head_dim, uint32_t window, uint32_t sinks) {
    if (!window_sizes(batch, n, rows, heads, kv_heads, head_dim)) return 0;
    return window_fwd_workspace((int)batch, (int)n, (int)rows, (int)heads, (int)kv_heads, (int)head_dim,
                                window_rows(window), clamp_int(sinks));
}

int evkhip_window_attention(const evkhip_tensor* q, const evkhip_tensor* k, const evkhip_tensor* v,
                            const evkhip_tensor* o, uint32_t head_dim, uint32_t window, uint32_t sinks,
                            uint32_t position_offset, const int32_t* offsets, float* lse, void* workspace,
                            uint64_t workspace_bytes, void* stream) {
    const char* op = "window_attention";
    Heads s;
    CHECK(head_shapes(op, q, k, v, head_dim, &s));
    CHECK(check_tensor(o, op, 3, 3));
    EVK_RETURN_IF(!same_dims(q, o), EVKHIP_ERR_SHAPE, "%s: o must match q", op);
    CHECK(check_positions(op, s, position_offset, offsets));
    EVK_RETURN_IF((uintptr_t)lse & 3, EVKHIP_ERR_INVALID_ARG, "%s: lse is not 4-byte aligned", op);
    const uint64_t need = evkhip_window_attention_workspace(s.B, s.N, s.R, s.H, s.KV, head_dim, window, sinks);
    CHECK(check_workspace(op, workspace, workspace_bytes, need));
    CHECK(check_apart(op, {bytes_of("o", o), {"lse", lse, (uint64_t)s.B * s.H * s.N * sizeof(float)}, {"the workspace", workspace, need}},
                      {bytes_of("q", q), bytes_of("k", k), bytes_of("v", v), {"offsets", offsets, s.B * sizeof(int32_t)}}));
    if (s.B == 0 || s.N == 0) return EVKHIP_OK;
    WindowArgs a = window_args(s, head_dim, window, sinks);
    a.q = (const f16*)q->data;
    a.k = (const f16*)k->data;
    a.v = (const f16*)v->data;
    a.out = (f16*)o->data;
    a.lse = lse;
    a.offsets = offsets;
    a.p0 = (int)position_offset;
    return window_forward(a, workspace, as_stream(stream));
}

uint64_t evkhip_window_attention_bwd_workspace(uint32_t batch, uint32_t n, uint32_t heads, uint32_t kv_heads,
                                               uint32_t head_dim, uint32_t window, uint32_t sinks) {
    if (!window_sizes(batch, n, n, heads, kv_heads, head_dim)) return 0;
    return window_bwd_workspace((int)batch, (int)n, (int)heads, (int)kv_heads, (int)head_dim,
                                window_rows(window), clamp_int(sinks));
}

int evkhip_window_attention_bwd(const evkhip_tensor* q, const evkhip_tensor* k, const evkhip_tensor* v,
                                const evkhip_tensor* o, const evkhip_tensor* dO, const evkhip_tensor* dQ,
                                const evkhip_tensor* dK, const evkhip_tensor* dV, const float* lse,
                                uint32_t head_dim, uint32_t window, uint32_t sinks, void* workspace,
                                uint64_t workspace_bytes, void* stream) {
    const char* op = "window_attention_bwd";
    Heads s;
    CHECK(head_shapes(op, q, k, v, head_dim, &s));
    for (const evkhip_tensor* t : {o, dO, dQ}) {
        CHECK(check_tensor(t, op, 3, 3));
        EVK_RETURN_IF(!same_dims(q, t), EVKHIP_ERR_SHAPE, "%s: o, dO and dQ must match q", op);
    }
    for (const evkhip_tensor* t : {dK, dV}) {
        CHECK(check_tensor(t, op, 3, 3));
        EVK_RETURN_IF(!same_dims(k, t), EVKHIP_ERR_SHAPE, "%s: dK and dV must match k", op);
    }
    EVK_RETURN_IF(s.R != s.N, EVKHIP_ERR_SHAPE, "%s: %u queries over %u rows; the gradient takes a whole sequence", op, s.N, s.R);
    EVK_RETURN_IF(!lse && s.B && s.N, EVKHIP_ERR_INVALID_ARG, "%s: null lse", op);
    EVK_RETURN_IF((uintptr_t)lse & 3, EVKHIP_ERR_INVALID_ARG, "%s: lse is not 4-byte aligned", op);
    const uint64_t need = evkhip_window_attention_bwd_workspace(s.B, s.N, s.H, s.KV, head_dim, window, sinks);
    CHECK(check_workspace(op, workspace, workspace_bytes, need));
    CHECK(check_apart(op, {bytes_of("dQ", dQ), bytes_of("dK", dK), bytes_of("dV", dV), {"the workspace", workspace, need}},
                      {bytes_of("q", q), bytes_of("k", k), bytes_of("v", v), bytes_of("o", o), bytes_of("dO", dO),
                       {"lse", lse, (uint64_t)s.B * s.H * s.N * sizeof(float)}}));
    if (s.B == 0 || s.N == 0) return EVKHIP_OK;
    WindowArgs a = window_args(s, head_dim, window, sinks);
    a.q = (const f16*)q->data;
    a.k = (const f16*)k->data;
    a.v = (const f16*)v->data;
    a.o = (const f16*)o->data;
    a.dO = (const f16*)dO->data;
    a.out = (f16*)dQ->data;
    a.dK = (f16*)dK->data;
    a.dV = (f16*)dV->data;
    a.lse = const_cast<float*>(lse);
    return window_backward(a, workspace, as_stream(stream));
}

int evkhip_gated_linear(const evkhip_tensor* x, const evkhip_tensor* w, const evkhip_tensor* h,
                        const evkhip_tensor* gate_up, int activation, void* stream) {
    const char* op = "gated_linear";
    Gated s;
    CHECK(gated_shapes(op, x, w, h, gate_up, activation, &s));
    CHECK(check_apart(op, {bytes_of("h", h), bytes_of("gate_up", gate_up)}, {bytes_of("x", x), bytes_of("w", w)}));
    if (s.T == 0 || s.F == 0) return EVKHIP_OK;
    if (s.D == 0) {  // products of nothing: act(0) * 0
        CHECK(fill_launch(h->data, 0u, (int64_t)numel(h), aligned16(h->data), as_stream(stream)));
        if (gate_up) CHECK(fill_launch(gate_up->data, 0u, (int64_t)numel(gate_up), aligned16(gate_up->data), as_stream(stream)));
        return EVKHIP_OK;
    }
    GemmArgs a{};
    a.A = (const f16*)x->data;
    a.B = (const f16*)w->data;
    a.C = (f16*)h->data;
    a.M = (int)s.T;
    a.N = (int)s.F;
    a.K = (int)s.D;
    a.act = activation;
    a.gate_up = gate_up ? (f16*)gate_up->data : nullptr;
    const bool vec_ok = aligned16(x->data) && aligned16(w->data) && aligned16(h->data) &&
                        (!gate_up || aligned16(gate_up->data)) && s.D % 8 == 0 && s.F % 8 == 0;
    return glu_dispatch(a, vec_ok, as_stream(stream));
}

uint64_t evkhip_gated_linear_backward_workspace(uint64_t tokens, uint32_t d, uint32_t f) {
    (void)d;
    return glu_bwd_workspace(tokens * f);
}

int evkhip_gated_linear_backward(const evkhip_tensor* x, const evkhip_tensor* w, const evkhip_tensor* gate_up,
                                 const evkhip_tensor* dh, const evkhip_tensor* dx, const evkhip_tensor* dw,
                                 int activation, int accumulate, void* workspace, uint64_t workspace_bytes,
                                 void* stream) {
    const char* op = "gated_linear_backward";
    Gated s;
    EVK_RETURN_IF(!gate_up, EVKHIP_ERR_INVALID_ARG, "%s: null gate_up", op);
    CHECK(gated_shapes(op, x, w, dh, gate_up, activation, &s));
    if (dx) {
        CHECK(check_tensor(dx, op, 1, EVKHIP_MAX_DIMS));
        EVK_RETURN_IF(!same_dims(x, dx), EVKHIP_ERR_SHAPE, "%s: dx must match x", op);
    }
    if (dw) {
        CHECK(check_tensor(dw, op, 3, 3));
        EVK_RETURN_IF(!same_dims(w, dw), EVKHIP_ERR_SHAPE, "%s: dw must match w", op);
    }
    const uint64_t need = evkhip_gated_linear_backward_workspace(s.T, s.D, s.F);
    CHECK(check_workspace(op, workspace, workspace_bytes, need));
    CHECK(check_apart(op, {bytes_of("dx", dx), bytes_of("dw", dw), {"the workspace", workspace, need}},
                      {bytes_of("x", x), bytes_of("w", w), bytes_of("gate_up", gate_up), bytes_of("dh", dh)}));
    hipStream_t st = as_stream(stream);
    if (s.D == 0) return EVKHIP_OK;  // dx and dw hold nothing
    if (s.T == 0 || s.F == 0) {      // sums over nothing
        if (dx) CHECK(fill_launch(dx->data, 0u, (int64_t)numel(dx), aligned16(dx->data), st));
        if (dw && !accumulate) CHECK(fill_launch(dw->data, 0u, (int64_t)numel(dw), aligned16(dw->data), st));
        return EVKHIP_OK;
    }
    f16* dgu = (f16*)workspace;
    const bool rows_ok = s.D % 8 == 0 && s.F % 8 == 0;
    GemmArgs gw{}, gx{};
    const bool gw_ok = rows_ok && aligned16(x->data) && dw && aligned16(dw->data);
    const bool gx_ok = rows_ok && aligned16(w->data) && dx && aligned16(dx->data);
    if (dw) {  // dw[i] (+)= x^T dgu[i]
        gw.A = (const f16*)x->data;
        gw.B = dgu;
        gw.C = (f16*)dw->data;
        gw.M = (int)s.D;
        gw.N = (int)s.F;
        gw.K = (int)s.T;
        gw.sB = (int64_t)(s.T * s.F);
        gw.sC = (int64_t)s.D * s.F;
        gw.acc = accumulate ? 1 : 0;
        CHECK(scaled_dispatch(gw, 2, gw_ok, st, true));
    }
    if (dx) {  // dx = dgu[0] w[0]^T + dgu[1] w[1]^T
        gx.A = dgu;
        gx.B = (const f16*)w->data;
        gx.C = (f16*)dx->data;
        gx.M = (int)s.T;
        gx.N = (int)s.D;
        gx.K = (int)s.F;
        CHECK(pair_dispatch(gx, gx_ok, st, true));
    }
    CHECK(glu_bwd_launch((const f16*)gate_up->data, (const f16*)dh->data, dgu, (int64_t)(s.T * s.F), activation, &gw.back, st));
    gx.back = gw.back;
    if (dw) CHECK(scaled_dispatch(gw, 2, gw_ok, st));
    if (dx) CHECK(pair_dispatch(gx, gx_ok, st));
    return EVKHIP_OK;
}

}  // extern "C"

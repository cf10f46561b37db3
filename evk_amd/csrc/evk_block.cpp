// evk::ai's operators of a grouped-query block (no reference counterparts)
// over the C ABI.  Workspaces are buffers of the runtime, released once the
// stream has passed the call.
#include <evk_ai.h>
#include <evkhip.h>

namespace evk::ai {
namespace {

evkhip_tensor desc(Tensor& t) {
    evkhip_tensor d{};
    d.data = t.device_ptr();
    d.rank = t.shape.rank();
    for (uint32_t i = 0; i < d.rank; ++i) d.dims[i] = t.shape.values[i];
    return d;
}
struct Opt {  // descriptor of a tensor that may be left out
    evkhip_tensor d{};
    const evkhip_tensor* p = nullptr;
    explicit Opt(Tensor* t) {
        if (t) {
            d = desc(*t);
            p = &d;
        }
    }
};

void check(int status, const char* op) {
    if (status != EVKHIP_OK) {
        std::fprintf(stderr, "evk::ai::%s failed (status %d): %s\n", op, status, evkhip_last_error());
        std::abort();
    }
}
void* stream() {
    return GetCmd().stream();
}

// Address of `count` 32-bit values in the storage of an fp16 tensor.
void* words(Tensor* t, uint64_t count, const char* op, const char* name) {
    if (!t) return nullptr;
    if (uint64_t(t->shape.count()) != 2 * count) {
        std::fprintf(stderr, "evk::ai::%s: %s holds %u fp16 slots, needs %llu (%llu 32-bit values)\n", op, name, t->shape.count(),
                     (unsigned long long)(2 * count), (unsigned long long)count);
        std::abort();
    }
    return t->device_ptr();
}
uint64_t rows_of(Tensor& q, uint32_t head_dim) {
    return head_dim ? uint64_t(q.shape.count()) / head_dim : 0;
}

struct Workspace {
    evk::Buffer buffer;
    uint64_t bytes;
    explicit Workspace(uint64_t n) : bytes(n) {
        if (n) buffer = evk::CreateBuffer({.size = n, .usage = evk::BufferUsage::Storage});
    }
    void* ptr() { return bytes ? reinterpret_cast<void*>(buffer.GetReference()) : nullptr; }
};

}  // namespace

void qkv_norm_rope(Tensor& qkv, Tensor& q, Tensor& k, Tensor& v, uint32_t head_dim, Tensor* q_weight, Tensor* k_weight,
                   float eps, float rotary_base, uint32_t position_offset, Tensor* offsets) {
    evkhip_tensor X = desc(qkv), Q = desc(q), K = desc(k), V = desc(v);
    Opt wq(q_weight), wk(k_weight);
    const int32_t* off = static_cast<const int32_t*>(words(offsets, qkv.shape[0], "qkv_norm_rope", "offsets"));
    check(evkhip_qkv_norm_rope(&X, wq.p, wk.p, &Q, &K, &V, head_dim, eps, rotary_base, position_offset, off, stream()),
          "qkv_norm_rope");
}

void qkv_norm_rope_backward(Tensor& qkv, Tensor& dq, Tensor& dk, Tensor& dv, Tensor& dqkv, uint32_t head_dim, Tensor* q_weight,
                            Tensor* k_weight, Tensor* dq_weight, Tensor* dk_weight, float eps, float rotary_base,
                            uint32_t position_offset, bool accumulate) {
    evkhip_tensor X = desc(qkv), Q = desc(dq), K = desc(dk), V = desc(dv), D = desc(dqkv);
    Opt wq(q_weight), wk(k_weight), gq(dq_weight), gk(dk_weight);
    uint64_t need = 0;
    if (qkv.shape.rank() == 3 && (dq_weight || dk_weight))
        need = evkhip_qkv_norm_rope_backward_workspace(uint64_t(qkv.shape[0]) * qkv.shape[1], head_dim);
    Workspace ws(need);
    check(evkhip_qkv_norm_rope_backward(&X, wq.p, wk.p, &Q, &K, &V, &D, gq.p, gk.p, head_dim, eps, rotary_base, position_offset,
                                        accumulate, ws.ptr(), ws.bytes, stream()),
          "qkv_norm_rope_backward");
}

void window_attention(Tensor& q, Tensor& k, Tensor& v, Tensor& o, uint32_t head_dim, uint32_t window, uint32_t sinks,
                      uint32_t position_offset, Tensor* offsets, Tensor* lse) {
    evkhip_tensor Q = desc(q), K = desc(k), V = desc(v), O = desc(o);
    const int32_t* off = static_cast<const int32_t*>(words(offsets, q.shape[0], "window_attention", "offsets"));
    float* L = static_cast<float*>(words(lse, rows_of(q, head_dim), "window_attention", "lse"));
    uint64_t need = 0;
    if (head_dim && q.shape.rank() == 3 && k.shape.rank() == 3)
        need = evkhip_window_attention_workspace(q.shape[0], q.shape[1], k.shape[1], q.shape[2] / head_dim, k.shape[2] / head_dim,
                                                 head_dim, window, sinks);
    Workspace ws(need);
    check(evkhip_window_attention(&Q, &K, &V, &O, head_dim, window, sinks, position_offset, off, L, ws.ptr(), ws.bytes, stream()),
          "window_attention");
}

void window_attention_bwd(Tensor& q, Tensor& k, Tensor& v, Tensor& o, Tensor& dO, Tensor& dQ, Tensor& dK, Tensor& dV, Tensor& lse,
                          uint32_t head_dim, uint32_t window, uint32_t sinks) {
    evkhip_tensor Q = desc(q), K = desc(k), V = desc(v), O = desc(o), G = desc(dO);
    evkhip_tensor DQ = desc(dQ), DK = desc(dK), DV = desc(dV);
    const float* L = static_cast<const float*>(words(&lse, rows_of(q, head_dim), "window_attention_bwd", "lse"));
    uint64_t need = 0;
    if (head_dim && q.shape.rank() == 3 && k.shape.rank() == 3)
        need = evkhip_window_attention_bwd_workspace(q.shape[0], q.shape[1], q.shape[2] / head_dim, k.shape[2] / head_dim, head_dim,
                                                     window, sinks);
    Workspace ws(need);
    check(evkhip_window_attention_bwd(&Q, &K, &V, &O, &G, &DQ, &DK, &DV, L, head_dim, window, sinks, ws.ptr(), ws.bytes, stream()),
          "window_attention_bwd");
}

void gated_linear(Tensor& x, Tensor& w, Tensor& h, Tensor* gate_up, Activation activation) {
    evkhip_tensor X = desc(x), W = desc(w), H = desc(h);
    Opt gu(gate_up);
    check(evkhip_gated_linear(&X, &W, &H, gu.p, int(activation), stream()), "gated_linear");
}

void gated_linear_backward(Tensor& x, Tensor& w, Tensor& gate_up, Tensor& dh, Tensor* dx, Tensor* dw, Activation activation,
                           bool accumulate) {
    evkhip_tensor X = desc(x), W = desc(w), U = desc(gate_up), H = desc(dh);
    Opt gx(dx), gw(dw);
    uint64_t need = 0;
    if (w.shape.rank() == 3 && w.shape[1])
        need = evkhip_gated_linear_backward_workspace(x.shape.count() / w.shape[1], w.shape[1], w.shape[2]);
    Workspace ws(need);
    check(evkhip_gated_linear_backward(&X, &W, &U, &H, gx.p, gw.p, int(activation), accumulate, ws.ptr(), ws.bytes, stream()),
          "gated_linear_backward");
}

}  // namespace evk::ai

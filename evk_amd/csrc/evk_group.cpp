// evk::ai's operators of a group of continuations of one prompt (no reference
// counterparts) over the C ABI.
#include "evk_calls.h"

namespace evk::ai {
using namespace calls;

namespace {
// Address of 32-bit values in the storage of an fp16 tensor: `per` for each row of t.
float* floats(Tensor* t, uint64_t rows, uint64_t per, const char* op, const char* name) {
    return static_cast<float*>(words(t, rows * per, op, name));
}
uint64_t rows_by(Tensor& t) {  // rows of the last dimension
    const uint32_t d = t.shape.rank() ? t.shape[t.shape.rank() - 1] : 0;
    return d ? uint64_t(t.shape.count()) / d : 0;
}
}  // namespace

void residual_norm(Tensor& x, Tensor* y, Tensor* s, Tensor& h, Tensor* post_weight, Tensor* gate, Tensor* pre_weight,
                   float residual_scale, bool post_norm, float eps) {
    evkhip_tensor X = desc(x), H = desc(h);
    Opt Y(y), S(s), wo(post_weight), g(gate), wi(pre_weight);
    check(evkhip_residual_norm(&X, Y.p, wo.p, g.p, wi.p, S.p, &H, residual_scale, post_norm, eps, stream()), "residual_norm");
}

void residual_norm_backward(Tensor& x, Tensor* y, Tensor* ds, Tensor& dh, Tensor& dx, Tensor* dy, Tensor* post_weight, Tensor* gate,
                            Tensor* pre_weight, Tensor* dpost_weight, Tensor* dgate, Tensor* dpre_weight, float residual_scale,
                            bool post_norm, float eps, bool accumulate) {
    evkhip_tensor X = desc(x), DH = desc(dh), DX = desc(dx);
    Opt Y(y), DS(ds), DY(dy), wo(post_weight), g(gate), wi(pre_weight), dwo(dpost_weight), dg(dgate), dwi(dpre_weight);
    uint64_t need = 0;
    if ((dpost_weight || dgate || dpre_weight) && x.shape.rank())
        need = evkhip_residual_norm_backward_workspace(rows_by(x), gate && gate->shape.rank() == 2 ? gate->shape[0] : 1,
                                                       x.shape[x.shape.rank() - 1]);
    Workspace ws(need);
    check(evkhip_residual_norm_backward(&X, Y.p, wo.p, g.p, wi.p, DS.p, &DH, &DX, DY.p, dwo.p, dg.p, dwi.p, residual_scale, post_norm,
                                        eps, accumulate, ws.ptr(), ws.bytes, stream()),
          "residual_norm_backward");
}

void prefix_attention(Tensor& q, Tensor& prefix_k, Tensor& prefix_v, Tensor& k, Tensor& v, Tensor& o, uint32_t head_dim,
                      uint32_t position_offset, Tensor* offsets, Tensor* lse) {
    evkhip_tensor Q = desc(q), PK = desc(prefix_k), PV = desc(prefix_v), K = desc(k), V = desc(v), O = desc(o);
    const int32_t* off = static_cast<const int32_t*>(words(offsets, q.shape[0], "prefix_attention", "offsets"));
    float* L = static_cast<float*>(words(lse, rows_of(q, head_dim), "prefix_attention", "lse"));
    uint64_t need = 0;
    if (head_dim && q.shape.rank() == 3 && k.shape.rank() == 3 && prefix_k.shape.rank() == 2)
        need = evkhip_prefix_attention_workspace(q.shape[0], q.shape[1], prefix_k.shape[0], k.shape[1], q.shape[2] / head_dim,
                                                 k.shape[2] / head_dim, head_dim);
    Workspace ws(need);
    check(evkhip_prefix_attention(&Q, &PK, &PV, &K, &V, &O, head_dim, position_offset, off, L, ws.ptr(), ws.bytes, stream()),
          "prefix_attention");
}

void token_logprobs(Tensor& logits, Tensor& tokens, Tensor& logprobs, Tensor* entropy, Tensor* top_ids, Tensor* top_logprobs, Tensor* stats,
                    float input_scale) {
    const char* op = "token_logprobs";
    evkhip_tensor X = desc(logits), T = desc(tokens);
    Opt ids(top_ids);
    const uint64_t rows = rows_by(logits);
    check(evkhip_token_logprobs(&X, &T, floats(&logprobs, rows, 1, op, "logprobs"), floats(entropy, rows, 1, op, "entropy"), ids.p,
                                floats(top_logprobs, top_ids ? top_ids->shape.count() : 0, 1, op, "top_logprobs"),
                                floats(stats, rows, 2, op, "stats"), input_scale, stream()),
          op);
}

void token_logprobs_backward(Tensor& logits, Tensor& tokens, Tensor& stats, Tensor* dlogprobs, Tensor& dlogits, Tensor* entropy,
                             Tensor* dentropy, float input_scale) {
    const char* op = "token_logprobs_backward";
    evkhip_tensor X = desc(logits), T = desc(tokens), D = desc(dlogits);
    const uint64_t rows = rows_by(logits);
    check(evkhip_token_logprobs_backward(&X, &T, floats(&stats, rows, 2, op, "stats"), floats(entropy, rows, 1, op, "entropy"),
                                         floats(dlogprobs, rows, 1, op, "dlogprobs"), floats(dentropy, rows, 1, op, "dentropy"), &D,
                                         input_scale, stream()),
          op);
}

}  // namespace evk::ai

// Checks shared by the C ABI files of the block's and the group's operators.
#pragma once

#include "kernels.h"

#include <math.h>

#include <initializer_list>

#define CHECK(expr)          \
    do {                     \
        int _rc = (expr);    \
        if (_rc) return _rc; \
    } while (0)

namespace evkhip {

constexpr uint32_t kMaxRows = 1u << 30;  // positions, rows, tokens: 32-bit arithmetic with room

inline bool same_dims(const evkhip_tensor* a, const evkhip_tensor* b) {
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
inline Bytes bytes_of(const char* name, const evkhip_tensor* t) {
    return {name, t ? t->data : nullptr, t ? numel(t) * sizeof(f16) : 0};
}
// Every output apart from every input, from the other outputs and the workspace.
inline int check_apart(const char* op, std::initializer_list<Bytes> outs, std::initializer_list<Bytes> ins) {
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

inline int check_workspace(const char* op, const void* p, uint64_t have, uint64_t need) {
    EVK_RETURN_IF(need && (!p || have < need), EVKHIP_ERR_INVALID_ARG, "%s: the workspace holds %llu bytes, %llu are needed",
                  op, (unsigned long long)(p ? have : 0), (unsigned long long)need);
    EVK_RETURN_IF(need && !aligned16(p), EVKHIP_ERR_INVALID_ARG, "%s: the workspace is not 16-byte aligned", op);
    return EVKHIP_OK;
}

inline int check_weight(const char* op, const char* name, const evkhip_tensor* w, uint32_t values) {
    if (!w) return EVKHIP_OK;
    CHECK(check_tensor(w, name, 1, 1));
    EVK_RETURN_IF(w->dims[0] != values, EVKHIP_ERR_SHAPE, "%s: %s must hold %u values", op, name, values);
    return EVKHIP_OK;
}

struct Heads {
    uint32_t B, N, R, H, KV;
};
// q (B,N,H dh); k, v (B,R,KV dh)
inline int head_shapes(const char* op, const evkhip_tensor* q, const evkhip_tensor* k, const evkhip_tensor* v, uint32_t dh,
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
inline int check_positions(const char* op, const Heads& s, uint32_t offset, const int32_t* offsets) {
    EVK_RETURN_IF(offsets && offset, EVKHIP_ERR_INVALID_ARG, "%s: position_offset %u besides offsets", op, offset);
    EVK_RETURN_IF(offsets && ((uintptr_t)offsets & 3), EVKHIP_ERR_INVALID_ARG, "%s: offsets are not 4-byte aligned", op);
    EVK_RETURN_IF(!offsets && (uint64_t)offset + s.N > s.R, EVKHIP_ERR_SHAPE, "%s: positions %u..%llu exceed the %u rows", op,
                  offset, (unsigned long long)offset + s.N, s.R);
    return EVKHIP_OK;
}

}  // namespace evkhip

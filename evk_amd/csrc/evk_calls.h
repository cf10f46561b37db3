// What evk::ai's files of operators without reference counterparts share: their
// calls of the C ABI.  Workspaces are buffers of the runtime, released once the
// stream has passed the call.
#pragma once

#include <evk_ai.h>
#include <evkhip.h>

namespace evk::ai::calls {

inline evkhip_tensor desc(Tensor& t) {
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

inline void check(int status, const char* op) {
    if (status != EVKHIP_OK) {
        std::fprintf(stderr, "evk::ai::%s failed (status %d): %s\n", op, status, evkhip_last_error());
        std::abort();
    }
}
inline void* stream() {
    return GetCmd().stream();
}

// Address of `count` 32-bit values in the storage of an fp16 tensor.
inline void* words(Tensor* t, uint64_t count, const char* op, const char* name) {
    if (!t) return nullptr;
    if (uint64_t(t->shape.count()) != 2 * count) {
        std::fprintf(stderr, "evk::ai::%s: %s holds %u fp16 slots, needs %llu (%llu 32-bit values)\n", op, name, t->shape.count(),
                     (unsigned long long)(2 * count), (unsigned long long)count);
        std::abort();
    }
    return t->device_ptr();
}
inline uint64_t rows_of(Tensor& q, uint32_t head_dim) {
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

}  // namespace evk::ai::calls

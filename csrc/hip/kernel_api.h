// The transformer kernels as plain C functions, handed from `_hip` (hipcc)
// to `_nodes` (g++ with torch) in a capsule: neither is built with the
// other's headers. Functions return a HIP error code, 0 is success;
// `error` names one. Types: 0 f32, 1 bf16, 2 f16.
#pragma once
#include <cstdint>

#define KF_KERNELS_CAPSULE "kungfu_amd.kernels"

struct kf_kernels {
    const char *(*error)(int);
    // embedding.hip
    long long (*embed_ws)(long long N, long long V, int H);
    int (*embed_fwd)(const void *ids, int wide, const void *weight,
                     long long ldw, int wtype, void *out, int otype,
                     long long N, long long V, int H, float scale,
                     void *stream);
    int (*embed_bwd)(const void *ids, int wide, const void *dout, int otype,
                     void *dw, int wtype, long long N, long long V, int H,
                     long long padding, float scale, void *work,
                     void *stream);
    // qk_norm_rope.hip
    long long (*qk_ws)(int D, int heads);
    int (*qk_norm_rope)(const uintptr_t *ptrs, const long long *dims,
                        int dtype, float eps, int backward, void *stream);
    // window_attention.hip
    long long (*attn_ws)(const long long *dims, int backward);
    int (*attn_fwd)(const uintptr_t *ptrs, const long long *dims,
                    const long long *strides, float scale, int dtype,
                    void *stream);
    int (*attn_bwd)(const uintptr_t *ptrs, const long long *dims,
                    const long long *strides, float scale, int dtype,
                    void *stream);
};

// ops.h — launch interface of the operators around the encoder: the dense
// layer and its gradients (ops_linear.hip), the token-row lookup and its
// gradient (ops_rows.hip) and the AdamW step (ops_adamw.hip).  ops_api.cpp
// holds their C entry points (include/bert_amd.h) and checks every argument;
// the launchers below assume checked ones.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bert_amd.h"

namespace bertamd {

// the message bert_amd_last_error() returns on this thread (runtime.cpp)
void set_last_error(const char *msg);

// y = act(x W^T + b) + r and its kept pre-activation z; rows are `ld*` elements apart
struct LinearArgs {
    int type = 0, act = 0;
    int64_t M = 0;
    int N = 0, K = 0;
    const void *x = nullptr, *w = nullptr, *r = nullptr;
    const float *bias = nullptr;
    void *y = nullptr, *z = nullptr;
    int64_t ldx = 0, ldw = 0, ldr = 0, ldy = 0, ldz = 0;
    void *ws = nullptr;
};
// whether a matrix's address and row stride allow whole 16-byte pieces; `aligned` below: those of all inputs do
bool linear_aligned(const void *p, int64_t ld, int type);
int64_t linear_ws_bytes(int type, int64_t M, int N, int K, bool aligned);
hipError_t launch_linear(const LinearArgs &a, hipStream_t s);

// dx = dz W, dw = dz^T x, db = sum of dz over rows, dz = dy act'(z)
struct LinearGradArgs {
    int type = 0, act = 0;
    int64_t M = 0;
    int N = 0, K = 0;
    const void *dy = nullptr, *z = nullptr, *x = nullptr, *w = nullptr;
    void *dx = nullptr, *dw = nullptr;
    float *db = nullptr;
    int64_t lddy = 0, ldz = 0, ldx = 0, ldw = 0, lddx = 0, lddw = 0;
    void *ws = nullptr;
};
int64_t linear_grad_ws_bytes(int type, int act, int64_t M, int N, int K, bool aligned);
hipError_t launch_linear_grad(const LinearGradArgs &a, hipStream_t s);

struct LookupArgs {
    int type = 0, out_type = 0;
    int64_t n = 0;
    int V = 0, E = 0;
    const void *table = nullptr;
    int64_t ld_bytes = 0;  // bytes between the table's rows
    const int32_t *ids = nullptr;
    float scale = 1.f;
    void *out = nullptr;
    int64_t ldo = 0;
};
hipError_t launch_lookup(const LookupArgs &a, hipStream_t s);

struct LookupGradArgs {
    int type = 0;
    int64_t n = 0;
    int V = 0, E = 0;
    const void *dout = nullptr;
    int64_t ldd = 0;
    const int32_t *ids = nullptr;
    float scale = 1.f;
    int pad_id = -1;
    bool accumulate = false;
    float *dtable = nullptr;
    int64_t ldt = 0;
    void *ws = nullptr;
};
int64_t lookup_grad_ws_bytes(int64_t n, int V, int E);
hipError_t launch_lookup_grad(const LookupGradArgs &a, hipStream_t s);

struct AdamwArgs {
    int n_tensors = 0;
    const bert_amd_adamw_tensor *t = nullptr;
    int grad_type = 0, copy_type = 0, bits = 32;
    double lr = 0, beta1 = 0, beta2 = 0, eps = 0;
    int64_t step = 1;
    uint32_t seed = 0;
    const float *grad_scale = nullptr;
};
hipError_t launch_adamw(const AdamwArgs &a, hipStream_t s);
hipError_t launch_adamw_moments(int64_t n, const uint8_t *m, const float *ms, const uint8_t *v, const float *vs,
                                float *m_out, float *v_out, hipStream_t s);

}  // namespace bertamd

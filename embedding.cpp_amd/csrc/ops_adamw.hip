// ops_adamw.hip — one AdamW step over many tensors, moments in f32 or 8 bits.
//
//   m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - (lr / (1 - beta1^t)) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// in f32, each operation rounded by itself in the order written in step_one
// (the build contracts no products into fused adds), so that a plain program
// with the same order gets the same bits: 8-bit codes have no tolerance.
//
// 8-bit states keep m and r = sqrt(v) as small floats over a scale that 256
// consecutive elements share, scale = peak / (largest code's value): a sign, 4
// exponent and 3 mantissa bits for m; 4 and 4 for r.  The lowest octave is
// linear, down to 0.  Codes are rounded up or down at random in proportion
// (bits mixed from the seed, the tensor's number and the element's): a moment
// moves by a tenth (m) or a thousandth (v) of its gap to g a step, less than
// half a code's step, and rounded to the nearest code it would stay for good.
// r of a nonzero v is never stored as 0: it divides.
//
// Memory bound: 28 bytes an element with f32 states and gradients, 16 with
// 8-bit states.
#include "ops_common.h"

#include <algorithm>
#include <cmath>

namespace bertamd {

namespace {

constexpr int STATE_BLOCK = 256;       // elements of a scale: one wave, 4 each
constexpr int CHUNK = 4096;            // elements of a workgroup
constexpr int64_t MAX_CHUNKS = 1 << 23;  // per launch: its threads are counted in 32 bits
constexpr int TENSORS = 44;            // per launch: the table travels in the kernel's arguments (4 KB)
constexpr float M_TOP = 61440.f;       // (2 - 2^-3) 2^15
constexpr float R_TOP = 63488.f;       // (2 - 2^-4) 2^15

struct Tensor {
    float *p;
    const void *g;
    void *m, *v;
    float *ms, *vs;
    void *copy;
    int64_t n;
    float keep;         // 1 - lr decay
    uint32_t key;       // the seed and the tensor's number, mixed
    int64_t first;      // first chunk of this tensor in the launch
};
struct Table {
    Tensor t[TENSORS];
    int count;
    float b1, c1, b2, c2, step, root, eps;
    const float *grad_scale;
};
static_assert(sizeof(Table) <= 4096, "kernel arguments");

__host__ __device__ __forceinline__ uint32_t mix(uint32_t h) {
    h = (h ^ (h >> 16)) * 0x9E3779B9u;
    h = (h ^ (h >> 15)) * 0xBB67AE85u;
    return h ^ (h >> 16);
}

// what code c of a magnitude with MANT mantissa bits stands for, over its scale
template <int MANT>
__device__ __forceinline__ float code_value(uint32_t c) {
    constexpr uint32_t N = 1u << MANT;
    if (c < N) return (float)c * (2.f / N);
    return __uint_as_float((c + 127u * N) << (23 - MANT));
}
template <int MANT>
__device__ __forceinline__ uint32_t code_of(float y, uint32_t h) {
    constexpr uint32_t N = 1u << MANT, DROP = 23 - MANT;
    uint32_t c;
    if (y >= 2.f)
        c = ((__float_as_uint(y) + (h >> (32 - DROP))) >> DROP) - 127u * N;
    else
        c = (uint32_t)(y * (N / 2.f) + (float)(h >> 8) * 0x1p-24f);
    return min(c, 16u * N - 1u);
}

// scale of a block whose largest magnitude has the bits `peak`, and its
// inverse.  Peaks under 2^-100 are taken as zero (the inverse would overflow).
// The scale of a block that holds an infinity or NaN is one too: it reads back
// as NaN throughout.
__device__ __forceinline__ void block_scale(uint32_t peak, float top, float &scale, float &inv) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) peak = max(peak, (uint32_t)__shfl_xor((int)peak, d));
    const float a = __uint_as_float(peak);
    scale = a < 0x1p-100f ? 0.f : a / top;
    inv = scale > 0.f && peak < 0x7f800000u ? 1.f / scale : 0.f;
}

struct Moments {
    float m, v, r;
};
__device__ __forceinline__ Moments step_one(const Table &a, float keep, float g, float &p, float m, float v) {
    m = m * a.b1 + g * a.c1;
    v = v * a.b2 + (g * a.c2) * g;
    const float r = sqrtf(v);
    p = p * keep - (m * a.step) / (r * a.root + a.eps);
    return {m, v, r};
}

template <int GRAD, int COPY, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(Table a) {
    typedef typename Elem<GRAD>::T G;
    typedef typename Elem<COPY>::T C;
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {  // the tensor of this chunk
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].first <= (int64_t)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const Tensor &t = a.t[lo];
    const float gs = a.grad_scale ? *a.grad_scale : 1.f;
    const int64_t start = ((int64_t)blockIdx.x - t.first) * CHUNK;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t b = start + wave * STATE_BLOCK; b < min(t.n, start + CHUNK); b += 4 * STATE_BLOCK) {
        float mn[4], rn[4];
        float ms = 0.f, vs = 0.f;
        if constexpr (BITS == 8) ms = t.ms[b / STATE_BLOCK], vs = t.vs[b / STATE_BLOCK];
        uint32_t mpeak = 0, rpeak = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t i = b + 4 * lane + j;
            mn[j] = rn[j] = 0.f;
            if (i >= t.n) continue;
            float g = (float)((const G *)t.g)[i];
            if (a.grad_scale) g *= gs;
            float m, v, p = t.p[i];
            if constexpr (BITS == 8) {
                const uint32_t cm = ((const uint8_t *)t.m)[i], cv = ((const uint8_t *)t.v)[i];
                m = code_value<3>(cm & 127u) * ms;
                m = cm & 128u ? -m : m;
                const float r = code_value<4>(cv) * vs;
                v = r * r;
            } else {
                m = ((const float *)t.m)[i], v = ((const float *)t.v)[i];
            }
            const Moments o = step_one(a, t.keep, g, p, m, v);
            t.p[i] = p;
            if (t.copy) ((C *)t.copy)[i] = (C)p;
            if constexpr (BITS == 8) {
                mn[j] = o.m, rn[j] = o.r;
                mpeak = max(mpeak, __float_as_uint(o.m) & 0x7fffffffu);
                rpeak = max(rpeak, __float_as_uint(o.r) & 0x7fffffffu);
            } else {
                ((float *)t.m)[i] = o.m;
                ((float *)t.v)[i] = o.v;
            }
        }
        if constexpr (BITS == 8) {
            float minv, rinv;
            block_scale(mpeak, M_TOP, ms, minv);
            block_scale(rpeak, R_TOP, vs, rinv);
            if (lane == 0) t.ms[b / STATE_BLOCK] = ms, t.vs[b / STATE_BLOCK] = vs;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t i = b + 4 * lane + j;
                if (i >= t.n) continue;
                const uint32_t h = mix((uint32_t)i ^ t.key ^ ((uint32_t)(i >> 32) * 0x9E3779B9u));
                uint32_t cm = 0, cv = 0;
                if (minv > 0.f) cm = code_of<3>(fabsf(mn[j]) * minv, h) | (mn[j] < 0.f ? 128u : 0u);
                if (rinv > 0.f) cv = code_of<4>(rn[j] * rinv, mix(h ^ 0x9E3779B9u));
                if (cv == 0 && rinv > 0.f && rn[j] > 0.f) cv = 1;
                ((uint8_t *)t.m)[i] = (uint8_t)cm;
                ((uint8_t *)t.v)[i] = (uint8_t)cv;
            }
        }
    }
}

__global__ __launch_bounds__(256) void moments_kernel(int64_t n, const uint8_t *m, const float *ms, const uint8_t *v, const float *vs,
                                                      float *m_out, float *v_out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        if (m_out) {
            const uint32_t c = m[i];
            const float x = code_value<3>(c & 127u) * ms[i / STATE_BLOCK];
            m_out[i] = c & 128u ? -x : x;
        }
        if (v_out) {
            const float r = code_value<4>(v[i]) * vs[i / STATE_BLOCK];
            v_out[i] = r * r;
        }
    }
}

template <int GRAD, int COPY>
void launch_table(const Table &a, int64_t chunks, int bits, hipStream_t s) {
    if (bits == 8)
        hipLaunchKernelGGL((adamw_kernel<GRAD, COPY, 8>), dim3(chunks), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((adamw_kernel<GRAD, COPY, 32>), dim3(chunks), dim3(256), 0, s, a);
}
template <int GRAD>
void launch_table(const Table &a, int64_t chunks, int copy_type, int bits, hipStream_t s) {
    if (copy_type == BERT_AMD_F16)
        launch_table<GRAD, BERT_AMD_F16>(a, chunks, bits, s);
    else
        launch_table<GRAD, BERT_AMD_BF16>(a, chunks, bits, s);
}

}  // namespace

hipError_t launch_adamw(const AdamwArgs &a, hipStream_t s) {
    Table t = {};
    t.b1 = (float)a.beta1, t.c1 = (float)(1 - a.beta1);
    t.b2 = (float)a.beta2, t.c2 = (float)(1 - a.beta2);
    t.step = (float)(a.lr / (1 - std::pow(a.beta1, (double)a.step)));
    t.root = (float)(1 / std::sqrt(1 - std::pow(a.beta2, (double)a.step)));
    t.eps = (float)a.eps;
    t.grad_scale = a.grad_scale;
    int64_t chunks = 0;
    for (int i = 0; i <= a.n_tensors; i++) {
        const int64_t more = i < a.n_tensors ? ceil_div<int64_t>(a.t[i].n, CHUNK) : 0;
        if (t.count == TENSORS || (t.count && (i == a.n_tensors || chunks + more > MAX_CHUNKS))) {
            switch (a.grad_type) {
                case BERT_AMD_F32: launch_table<BERT_AMD_F32>(t, chunks, a.copy_type, a.bits, s); break;
                case BERT_AMD_F16: launch_table<BERT_AMD_F16>(t, chunks, a.copy_type, a.bits, s); break;
                default: launch_table<BERT_AMD_BF16>(t, chunks, a.copy_type, a.bits, s); break;
            }
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            t.count = 0, chunks = 0;
        }
        if (i == a.n_tensors) break;
        const bert_amd_adamw_tensor &o = a.t[i];
        if (!o.n) continue;
        t.t[t.count++] = {o.p, o.grad, o.m, o.v, o.m_scale, o.v_scale, o.copy, o.n, (float)(1 - a.lr * o.weight_decay),
                          mix((uint32_t)i * 0x9E3779B9u ^ a.seed), chunks};
        chunks += more;
    }
    return hipSuccess;
}

hipError_t launch_adamw_moments(int64_t n, const uint8_t *m, const float *ms, const uint8_t *v, const float *vs, float *m_out,
                                float *v_out, hipStream_t s) {
    hipLaunchKernelGGL(moments_kernel, dim3(std::min<int64_t>(1 << 16, ceil_div<int64_t>(n, 256))), dim3(256), 0, s, n, m, ms, v, vs, m_out, v_out);
    return hipGetLastError();
}

}  // namespace bertamd

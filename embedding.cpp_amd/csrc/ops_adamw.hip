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
// Memory bound: 28 bytes an element with f32 states and gradients, 14 to 16
// with 8-bit states.  A wave takes 256 elements, four a lane in whole 16-byte
// pieces: 22.6 M weights in 101 tensors (f32 states, bf16 copies) 151 us, 4.5
// TB/s, three launches; 192 M weights with 8-bit states and bf16 gradients 625
// us, 4.3 TB/s (single elements a lane took 1.7 times as long).
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
    int32_t first;      // first chunk of this tensor in the launch
    int32_t vec;        // every pointer is aligned to four of its elements
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
        if (a.t[mid].first <= (int)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const Tensor &t = a.t[lo];
    const float gs = a.grad_scale ? *a.grad_scale : 1.f;
    const int64_t start = (int64_t)((int)blockIdx.x - t.first) * CHUNK;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t b = start + wave * STATE_BLOCK; b < min(t.n, start + CHUNK); b += 4 * STATE_BLOCK) {
        const int64_t i = b + 4 * lane;
        const int count = (int)min((int64_t)4, t.n - i);  // this lane's elements; none past the end
        const bool whole = t.vec && count == 4;
        float p[4] = {}, g[4] = {}, m[4] = {}, v[4] = {}, r[4] = {};
        uint32_t cm[4] = {}, cv[4] = {};
        float ms = 0.f, vs = 0.f;
        if constexpr (BITS == 8) ms = t.ms[b / STATE_BLOCK], vs = t.vs[b / STATE_BLOCK];
        if (whole) {
            get_n<float, 4>(t.p + i, p);
            get_n<G, 4>((const G *)t.g + i, g);
            if constexpr (BITS == 8) {
                get_n<uint8_t, 4>((const uint8_t *)t.m + i, cm);
                get_n<uint8_t, 4>((const uint8_t *)t.v + i, cv);
            } else {
                get_n<float, 4>((const float *)t.m + i, m);
                get_n<float, 4>((const float *)t.v + i, v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j >= count) continue;
                p[j] = t.p[i + j];
                g[j] = (float)((const G *)t.g)[i + j];
                if constexpr (BITS == 8) cm[j] = ((const uint8_t *)t.m)[i + j], cv[j] = ((const uint8_t *)t.v)[i + j];
                else m[j] = ((const float *)t.m)[i + j], v[j] = ((const float *)t.v)[i + j];
            }
        }
        uint32_t mpeak = 0, rpeak = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (BITS == 8) {
                m[j] = code_value<3>(cm[j] & 127u) * ms;
                m[j] = cm[j] & 128u ? -m[j] : m[j];
                const float old = code_value<4>(cv[j]) * vs;
                v[j] = old * old;
            }
            if (a.grad_scale) g[j] *= gs;
            const Moments o = step_one(a, t.keep, g[j], p[j], m[j], v[j]);
            m[j] = o.m, v[j] = o.v, r[j] = o.r;
            if (BITS == 8 && j < count) {
                mpeak = max(mpeak, __float_as_uint(o.m) & 0x7fffffffu);
                rpeak = max(rpeak, __float_as_uint(o.r) & 0x7fffffffu);
            }
        }
        if constexpr (BITS == 8) {
            float minv, rinv;
            block_scale(mpeak, M_TOP, ms, minv);
            block_scale(rpeak, R_TOP, vs, rinv);
            if (lane == 0) t.ms[b / STATE_BLOCK] = ms, t.vs[b / STATE_BLOCK] = vs;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t h = mix((uint32_t)(i + j) ^ t.key ^ ((uint32_t)((i + j) >> 32) * 0x9E3779B9u));
                cm[j] = minv > 0.f ? code_of<3>(fabsf(m[j]) * minv, h) | (m[j] < 0.f ? 128u : 0u) : 0u;
                cv[j] = rinv > 0.f ? code_of<4>(r[j] * rinv, mix(h ^ 0x9E3779B9u)) : 0u;
                if (cv[j] == 0 && rinv > 0.f && r[j] > 0.f) cv[j] = 1;
            }
        }
        if (whole) {
            put_n<float, 4>(t.p + i, p);
            if (t.copy) put_n<C, 4>((C *)t.copy + i, p);
            if constexpr (BITS == 8) {
                put_n<uint8_t, 4>((uint8_t *)t.m + i, cm);
                put_n<uint8_t, 4>((uint8_t *)t.v + i, cv);
            } else {
                put_n<float, 4>((float *)t.m + i, m);
                put_n<float, 4>((float *)t.v + i, v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j >= count) continue;
                t.p[i + j] = p[j];
                if (t.copy) ((C *)t.copy)[i + j] = (C)p[j];
                if constexpr (BITS == 8) ((uint8_t *)t.m)[i + j] = (uint8_t)cm[j], ((uint8_t *)t.v)[i + j] = (uint8_t)cv[j];
                else ((float *)t.m)[i + j] = m[j], ((float *)t.v)[i + j] = v[j];
            }
        }
    }
}

// 8-bit moments as values, four of an element's place a thread
__global__ __launch_bounds__(256) void moments_kernel(int64_t n, const uint8_t *m, const float *ms, const uint8_t *v, const float *vs,
                                                      float *m_out, float *v_out, bool vec) {
    for (int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x); i < n; i += (int64_t)gridDim.x * 1024) {
        const int count = (int)min((int64_t)4, n - i);
        if (m_out) {
            uint32_t c[4] = {};
            float x[4];
            if (vec && count == 4) get_n<uint8_t, 4>(m + i, c);
            else for (int j = 0; j < count; j++) c[j] = m[i + j];
            const float scale = ms[i / STATE_BLOCK];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = code_value<3>(c[j] & 127u) * scale, x[j] = c[j] & 128u ? -x[j] : x[j];
            if (vec && count == 4) put_n<float, 4>(m_out + i, x);
            else for (int j = 0; j < count; j++) m_out[i + j] = x[j];
        }
        if (v_out) {
            uint32_t c[4] = {};
            float x[4];
            if (vec && count == 4) get_n<uint8_t, 4>(v + i, c);
            else for (int j = 0; j < count; j++) c[j] = v[i + j];
            const float scale = vs[i / STATE_BLOCK];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float r = code_value<4>(c[j]) * scale;
                x[j] = r * r;
            }
            if (vec && count == 4) put_n<float, 4>(v_out + i, x);
            else for (int j = 0; j < count; j++) v_out[i + j] = x[j];
        }
    }
}

template <int GRAD, int COPY>
hipError_t launch_table(const Table &a, int64_t chunks, int bits, hipStream_t s) {
    return launch(bits == 8 ? adamw_kernel<GRAD, COPY, 8> : adamw_kernel<GRAD, COPY, 32>, dim3(chunks), dim3(256), 0, s, a);
}
template <int GRAD>
hipError_t launch_table(const Table &a, int64_t chunks, int copy_type, int bits, hipStream_t s) {
    return copy_type == BERT_AMD_F16 ? launch_table<GRAD, BERT_AMD_F16>(a, chunks, bits, s) : launch_table<GRAD, BERT_AMD_BF16>(a, chunks, bits, s);
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
            const hipError_t e = a.grad_type == BERT_AMD_F32   ? launch_table<BERT_AMD_F32>(t, chunks, a.copy_type, a.bits, s)
                                 : a.grad_type == BERT_AMD_F16 ? launch_table<BERT_AMD_F16>(t, chunks, a.copy_type, a.bits, s)
                                                               : launch_table<BERT_AMD_BF16>(t, chunks, a.copy_type, a.bits, s);
            if (e != hipSuccess) return e;
            t.count = 0, chunks = 0;
        }
        if (i == a.n_tensors) break;
        const bert_amd_adamw_tensor &o = a.t[i];
        if (!o.n) continue;
        const auto off = [](const void *p, int bytes) { return (uintptr_t)p & (4 * bytes - 1); };
        const int state = a.bits == 8 ? 1 : 4;
        const bool vec = !(off(o.p, 4) | off(o.grad, elem_size(a.grad_type)) | off(o.m, state) | off(o.v, state) | off(o.copy, 2));
        t.t[t.count++] = {o.p, o.grad, o.m, o.v, o.m_scale, o.v_scale, o.copy, o.n, (float)(1 - a.lr * o.weight_decay),
                          mix((uint32_t)i * 0x9E3779B9u ^ a.seed), (int32_t)chunks, vec};
        chunks += more;
    }
    return hipSuccess;
}

hipError_t launch_adamw_moments(int64_t n, const uint8_t *m, const float *ms, const uint8_t *v, const float *vs, float *m_out,
                                float *v_out, hipStream_t s) {
    const bool vec = !(((uintptr_t)m | (uintptr_t)v) & 3) && !(((uintptr_t)m_out | (uintptr_t)v_out) & 15);
    return launch(moments_kernel, dim3(std::min<int64_t>(1 << 16, ceil_div<int64_t>(n, 1024))), dim3(256), 0, s, n, m, ms, v, vs, m_out, v_out,
                  vec);
}

}  // namespace bertamd

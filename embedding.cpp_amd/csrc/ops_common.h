// ops_common.h — device helpers shared by the operator kernels (ops_*.hip).
#pragma once
#include "ops.h"

namespace bertamd {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// what each element type of bert_amd.h is on the device; 16 bytes hold CH of them
template <int TYPE> struct Elem;
template <> struct Elem<BERT_AMD_F32> { typedef float T; static constexpr int CH = 4; };
template <> struct Elem<BERT_AMD_F16> { typedef _Float16 T; static constexpr int CH = 8; };
template <> struct Elem<BERT_AMD_BF16> { typedef __bf16 T; static constexpr int CH = 8; };

inline int elem_size(int type) { return type == BERT_AMD_F32 ? 4 : 2; }
inline bool aligned16(const void *p, int64_t stride_bytes) {
    return ((uintptr_t)p & 15) == 0 && (stride_bytes & 15) == 0;
}
template <typename T>
constexpr T ceil_div(T a, T b) { return (a + b - 1) / b; }

// A kernel's launch and its own status: hipGetLastError() behind a launch would
// also give what an earlier call on this thread, anyone's, has left there.
template <typename T> struct AsIs { typedef T type; };
template <typename... P>
hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, uint32_t lds, hipStream_t s, typename AsIs<P>::type... args) {
    void *each[] = {&args...};
    return hipLaunchKernel((const void *)kernel, grid, block, each, lds, s);
}

// orders the LDS accesses of a wave's lanes before and after it (no instruction: they run in order)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 16 bytes of elements
template <typename T, int CH>
struct Chunk {
    T v[CH];
};

// 8 elements in the type to or from an aligned row piece
template <typename T>
__device__ __forceinline__ void put8(T *p, const float *v) {
    constexpr int CH = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += CH) {
        Chunk<T, CH> o;
#pragma unroll
        for (int j = 0; j < CH; j++) o.v[j] = (T)v[i + j];
        *(u32x4 *)(p + i) = __builtin_bit_cast(u32x4, o);
    }
}
template <typename T>
__device__ __forceinline__ void add8(const T *p, float *v) {
    constexpr int CH = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += CH) {
        const auto o = __builtin_bit_cast(Chunk<T, CH>, *(const u32x4 *)(p + i));
#pragma unroll
        for (int j = 0; j < CH; j++) v[i + j] += (float)o.v[j];
    }
}

// N elements at p, aligned to as many bytes as they take, as values and back
template <typename T, int N, typename V>
__device__ __forceinline__ void get_n(const T *p, V *v) {
    struct __attribute__((aligned(N * sizeof(T)))) Some { T v[N]; };
    const Some f = *(const Some *)p;
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = (V)f.v[j];
}
template <typename T, int N, typename V>
__device__ __forceinline__ void put_n(T *p, const V *v) {
    struct __attribute__((aligned(N * sizeof(T)))) Some { T v[N]; } f;
#pragma unroll
    for (int j = 0; j < N; j++) f.v[j] = (T)v[j];
    *(Some *)p = f;
}

// Activations and their slopes in f32.  gelu is the tanh form that the
// encoder's feed-forward layer uses, written z * sigmoid(2u): no cancellation
// in its lower tail.
// the exponential never overflows: a far tail fades out through the subnormals
__device__ __forceinline__ float sigmoid_f(float v) {
    const float t = expf(-fabsf(v));
    return (v < 0.f ? t : 1.f) / (1.f + t);
}
constexpr float GELU_C = 0.7978845608028654f, GELU_K = 0.044715f;

__device__ __forceinline__ float act_f(float z, int act) {
    switch (act) {
        case BERT_AMD_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        case BERT_AMD_ACT_GELU: return z * sigmoid_f(2.f * GELU_C * (z + GELU_K * z * z * z));
        case BERT_AMD_ACT_GELU_ERF: return 0.5f * z * erfcf(-z * 0.70710678118654752f);
        case BERT_AMD_ACT_SILU: return z * sigmoid_f(z);
        case BERT_AMD_ACT_TANH: return tanhf(z);
    }
    return z;
}
// Past |z| = 90 every slope is 0 or 1 in f32: z is held there, so that no
// product of an infinite factor and a vanished one makes a NaN (a NaN stays).
__device__ __forceinline__ float act_slope_f(float z, int act) {
    z = z > 90.f ? 90.f : z < -90.f ? -90.f : z;
    switch (act) {
        case BERT_AMD_ACT_RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
        case BERT_AMD_ACT_GELU: {
            const float s = sigmoid_f(2.f * GELU_C * (z + GELU_K * z * z * z));
            return s + z * s * (1.f - s) * 2.f * GELU_C * (1.f + 3.f * GELU_K * z * z);
        }
        case BERT_AMD_ACT_GELU_ERF:
            return 0.5f * erfcf(-z * 0.70710678118654752f) + z * 0.3989422804014327f * expf(-0.5f * z * z);
        case BERT_AMD_ACT_SILU: {
            const float s = sigmoid_f(z);
            return s + z * s * (1.f - s);
        }
        case BERT_AMD_ACT_TANH: {
            const float t = tanhf(z);
            return (1.f - t) * (1.f + t);
        }
    }
    return 1.f;
}

// The same for results of 16 bits, in fewer instructions: v_exp_f32 and
// v_rcp_f32 are within a few 2^-24 of the value, 2^-11 and more are kept.
__device__ __forceinline__ float sigmoid_16(float v) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}
// z sigmoid(v).  v_rcp_f32 gives 0 for what is under 2^-126, where z times it is still
// one of bf16's values: both factors carry 2^14 that cancels, which takes the
// product down to 2^-133, bf16's smallest.
__device__ __forceinline__ float z_sigmoid_16(float z, float v) {
    return z * 0x1p-14f * __builtin_amdgcn_rcpf(0x1p-14f + __builtin_amdgcn_exp2f(__builtin_fmaf(v, -1.4426950408889634f, -14.f)));
}
template <int ACT, bool WIDE>
__device__ __forceinline__ float act_t(float z) {
    if constexpr (!WIDE && ACT == BERT_AMD_ACT_GELU) return z_sigmoid_16(z, 2.f * GELU_C * (z + GELU_K * z * z * z));
    else if constexpr (!WIDE && ACT == BERT_AMD_ACT_SILU) return z_sigmoid_16(z, z);
    else if constexpr (!WIDE && ACT == BERT_AMD_ACT_TANH) {
        const float q = z * z, far = 1.f - 2.f * sigmoid_16(-2.f * z);
        const float near = z * (1.f + q * (-1.f / 3 + q * (2.f / 15 - q * (17.f / 315))));  // next to zero, where `far` cancels
        return q < 0.0625f ? near : far;
    } else return act_f(z, ACT);
}

template <int ACT, bool WIDE>
__device__ __forceinline__ float act_slope_t(float z) {
    if constexpr (!WIDE && (ACT == BERT_AMD_ACT_GELU || ACT == BERT_AMD_ACT_SILU)) {
        z = z > 90.f ? 90.f : z < -90.f ? -90.f : z;
        constexpr bool G = ACT == BERT_AMD_ACT_GELU;
        const float q = z * z, s = sigmoid_16(G ? 2.f * GELU_C * z * (1.f + GELU_K * q) : z);
        return s + z * s * (1.f - s) * (G ? 2.f * GELU_C * (1.f + 3.f * GELU_K * q) : 1.f);
    } else if constexpr (!WIDE && ACT == BERT_AMD_ACT_TANH) {
        const float t = act_t<ACT, false>(z);
        return (1.f - t) * (1.f + t);
    } else {
        return act_slope_f(z, ACT);
    }
}

}  // namespace bertamd

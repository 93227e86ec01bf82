// ops_linear.hip — the dense layer y = act(x W^T + b) + r and its gradients
// dx = dz W, dw = dz^T x, db = sum of dz over rows, with dz = dy act'(z).
//
// Sums run in f32 on the matrix units.  A 16-bit layer's dz is rounded to its
// type before the two products, as the matrix units take 16-bit operands: an
// error of half a step in each term, where the result is rounded by half a
// step once more; db sums the unrounded dz.
#include "ops_common.h"

#include <algorithm>

namespace bertamd {

namespace {

// ---- the tile kernel for any size, stride and alignment --------------------
//
// C[m][n] = sum over k of A(m, k) B(n, k) in 64 x 64 tiles, four waves of
// 32 x 32 each; A(m, k) is at A[m lda + k], or at A[k lda + m] where TA.
// Chunks of 16 bytes are loaded along the contiguous axis, whole where they are
// inside and aligned, else by element with zeros outside.  gridDim.z splits k:
// split sums go to `part` and split_join_kernel adds them in order.
struct Operand {
    const void *p = nullptr;
    int64_t ld = 0;
    bool vec = false;  // p and ld allow 16-byte loads
};
struct Epilogue {
    int act = 0;
    const float *bias = nullptr;
    const void *r = nullptr;
    void *y = nullptr, *z = nullptr;
    int64_t ldr = 0, ldy = 0, ldz = 0;
};

template <typename T>
__device__ __forceinline__ void epilogue_store(const Epilogue &e, int64_t m, int64_t n, float v) {
    if (e.bias) v += e.bias[n];
    if (e.z) ((T *)e.z)[m * e.ldz + n] = (T)v;
    v = act_f(v, e.act);
    if (e.r) v += (float)((const T *)e.r)[m * e.ldr + n];
    ((T *)e.y)[m * e.ldy + n] = (T)v;
}

template <typename T, int CH>
struct Chunk {
    T v[CH];
};

// CH elements of row r from column c of a [nr][nc] matrix
template <typename T, int CH>
__device__ __forceinline__ Chunk<T, CH> load_chunk(const T *p, int64_t ld, bool vec, int64_t r, int64_t c, int64_t nr, int64_t nc) {
    Chunk<T, CH> o;
    if (r < nr && vec && c + CH <= nc) {
        o = __builtin_bit_cast(Chunk<T, CH>, *(const u32x4 *)(p + r * ld + c));
    } else {
#pragma unroll
        for (int j = 0; j < CH; j++) o.v[j] = r < nr && c + j < nc ? p[r * ld + c + j] : (T)0.f;
    }
    return o;
}

constexpr int TB = 64;  // tile rows and columns
template <int TYPE> constexpr int tile_k() { return TYPE == BERT_AMD_F32 ? 16 : 32; }
// LDS row length: one float or 16 bytes more than the tile, so that the lanes
// of an operand read start in different banks
template <int TYPE> constexpr int tile_ld() { return TYPE == BERT_AMD_F32 ? 17 : 40; }

template <int TYPE, bool TRANS>
__device__ __forceinline__ void stage_tile(const Operand &o, int64_t row0, int64_t rows, int64_t k0, int64_t k1,
                                           typename Elem<TYPE>::T *lds) {
    typedef typename Elem<TYPE>::T T;
    constexpr int CH = Elem<TYPE>::CH, BK = tile_k<TYPE>(), LD = tile_ld<TYPE>();
    const int t = threadIdx.x;
    if constexpr (!TRANS) {
        const int r = t / (BK / CH), c = t % (BK / CH) * CH;
        const auto v = load_chunk<T, CH>((const T *)o.p, o.ld, o.vec, row0 + r, k0 + c, rows, k1);
#pragma unroll
        for (int j = 0; j < CH; j++) lds[r * LD + c + j] = v.v[j];
    } else {
        const int r = t / (TB / CH), c = t % (TB / CH) * CH;
        const auto v = load_chunk<T, CH>((const T *)o.p, o.ld, o.vec, k0 + r, row0 + c, k1, rows);
#pragma unroll
        for (int j = 0; j < CH; j++) lds[(c + j) * LD + r] = v.v[j];
    }
}

template <int TYPE, bool TA, bool TBT>
__global__ __launch_bounds__(256) void tile_gemm_kernel(Operand A, Operand B, int64_t M, int64_t N, int64_t K,
                                                        int64_t k_per_split, float *part, Epilogue e) {
    typedef typename Elem<TYPE>::T T;
    constexpr int BK = tile_k<TYPE>(), LD = tile_ld<TYPE>();
    __shared__ T sa[TB * LD], sb[TB * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave & 1, wn = wave >> 1, r = lane & 31, h = lane >> 5;
    const int64_t tiles_n = ceil_div<int64_t>(N, TB);
    const int64_t m0 = blockIdx.x / tiles_n * TB, n0 = blockIdx.x % tiles_n * TB;
    const int64_t ka = (int64_t)blockIdx.z * k_per_split, kb = min(K, ka + k_per_split);
    f32x16 acc = {};
    for (int64_t k0 = ka; k0 < kb; k0 += BK) {
        stage_tile<TYPE, TA>(A, m0, M, k0, kb, sa);
        stage_tile<TYPE, TBT>(B, n0, N, k0, kb, sb);
        __syncthreads();
        const T *pa = sa + (32 * wm + r) * LD, *pb = sb + (32 * wn + r) * LD;
        if constexpr (TYPE == BERT_AMD_F32) {
#pragma unroll
            for (int k = 0; k < BK; k += 2) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(pa[k + h], pb[k + h], acc, 0, 0, 0);
        } else {
#pragma unroll
            for (int k = 0; k < BK; k += 16) {
                const u32x4 a = *(const u32x4 *)(pa + k + 8 * h), b = *(const u32x4 *)(pb + k + 8 * h);
                if constexpr (TYPE == BERT_AMD_F16)
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
                else
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
            }
        }
        __syncthreads();
    }
    const int64_t n = n0 + 32 * wn + r;
    if (n >= N) return;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int64_t m = m0 + 32 * wm + 8 * (i >> 2) + 4 * h + (i & 3);
        if (m >= M) continue;
        if (part)
            part[((int64_t)blockIdx.z * M + m) * N + n] = acc[i];
        else
            epilogue_store<T>(e, m, n, acc[i]);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void split_join_kernel(const float *part, int splits, int64_t M, int64_t N, Epilogue e) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < M * N; i += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < splits; s++) v += part[s * M * N + i];
        epilogue_store<T>(e, i / N, i % N, v);
    }
}

// dz = dy act'(z) in the layer's type, and its sums over 64 rows at a time
constexpr int DB_ROWS = 64;
template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const T *dy, int64_t lddy, const T *z, int64_t ldz, int act, int64_t M, int64_t N,
                                                 T *dz, float *part) {
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    for (int64_t b = blockIdx.y; b * DB_ROWS < M; b += gridDim.y) {
        const int64_t m1 = min(M, (b + 1) * DB_ROWS);
        float sum = 0.f;
        for (int64_t m = b * DB_ROWS; m < m1; m++) {
            float v = (float)dy[m * lddy + n];
            if (act) v *= act_slope_f((float)z[m * ldz + n], act);
            if (dz) dz[m * N + n] = (T)v;
            sum += v;
        }
        if (part) part[b * N + n] = sum;
    }
}

__global__ __launch_bounds__(256) void column_sum_kernel(const float *part, int64_t rows, int64_t N, float *out) {
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    float v = 0.f;
    for (int64_t b = 0; b < rows; b++) v += part[b * N + n];
    out[n] = v;
}

// k is split where the tiles alone leave most of the 256 CUs idle
int splits_for(int64_t M, int64_t N, int64_t K) {
    const int64_t tiles = ceil_div<int64_t>(M, TB) * ceil_div<int64_t>(N, TB);
    if (tiles >= 256 || tiles == 0) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(512 / tiles, K / 256));
}
int64_t split_bytes(int64_t M, int64_t N, int64_t K) {
    const int s = splits_for(M, N, K);
    return s > 1 ? s * M * N * 4 : 0;
}
int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

template <int TYPE, bool TA, bool TBT>
hipError_t tile_gemm(const Operand &A, const Operand &B, int64_t M, int64_t N, int64_t K, void *ws, const Epilogue &e, hipStream_t s) {
    typedef typename Elem<TYPE>::T T;
    const int splits = splits_for(M, N, K);
    const int64_t per = ceil_div(ceil_div<int64_t>(K, splits), (int64_t)tile_k<TYPE>()) * tile_k<TYPE>();
    const int64_t tiles = ceil_div<int64_t>(M, TB) * ceil_div<int64_t>(N, TB);
    float *part = splits > 1 ? (float *)ws : nullptr;
    hipLaunchKernelGGL((tile_gemm_kernel<TYPE, TA, TBT>), dim3(tiles, 1, splits), dim3(256), 0, s, A, B, M, N, K, per, part, e);
    if (part)
        hipLaunchKernelGGL((split_join_kernel<T>), dim3(std::min<int64_t>(1024, ceil_div<int64_t>(M * N, 256))), dim3(256), 0, s, part, splits, M, N, e);
    return hipGetLastError();
}

Operand operand(const void *p, int64_t ld, int type) { return {p, ld, aligned16(p, ld * elem_size(type))}; }

template <int TYPE>
hipError_t linear_t(const LinearArgs &a, hipStream_t s) {
    return tile_gemm<TYPE, false, false>(operand(a.x, a.ldx, TYPE), operand(a.w, a.ldw, TYPE), a.M, a.N, a.K, a.ws,
                                         {a.act, a.bias, a.r, a.y, a.z, a.ldr, a.ldy, a.ldz}, s);
}

template <int TYPE>
hipError_t linear_grad_t(const LinearGradArgs &a, hipStream_t s) {
    typedef typename Elem<TYPE>::T T;
    char *ws = (char *)a.ws;
    Operand dz = operand(a.dy, a.lddy, TYPE);
    T *kept = nullptr;
    if (a.act) {
        kept = (T *)ws;
        ws += round256(a.M * a.N * sizeof(T));
        dz = operand(kept, a.N, TYPE);
    }
    if (kept || a.db) {
        const int64_t blocks = ceil_div<int64_t>(a.M, DB_ROWS);
        float *part = a.db ? (float *)ws : nullptr;
        if (blocks)
            hipLaunchKernelGGL((dz_kernel<T>), dim3(ceil_div(a.N, 256), std::min<int64_t>(blocks, 65535)), dim3(256), 0, s, (const T *)a.dy,
                           a.lddy, (const T *)a.z, a.ldz, a.act, a.M, (int64_t)a.N, kept, part);
        if (a.db) {
            hipLaunchKernelGGL(column_sum_kernel, dim3(ceil_div(a.N, 256)), dim3(256), 0, s, part, blocks, (int64_t)a.N, a.db);
            ws += round256(blocks * a.N * 4);
        }
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if (a.dx && a.M) {
        Epilogue e;
        e.y = a.dx;
        e.ldy = a.lddx;
        if (hipError_t r = tile_gemm<TYPE, false, true>(dz, operand(a.w, a.ldw, TYPE), a.M, a.K, a.N, ws, e, s); r != hipSuccess) return r;
    }
    if (a.dw) {
        Epilogue e;
        e.y = a.dw;
        e.ldy = a.lddw;
        if (hipError_t r = tile_gemm<TYPE, true, true>(dz, operand(a.x, a.ldx, TYPE), a.N, a.K, a.M, ws, e, s); r != hipSuccess) return r;
    }
    return hipSuccess;
}

}  // namespace

int64_t linear_ws_bytes(int, int64_t M, int N, int K) { return split_bytes(M, N, K); }

hipError_t launch_linear(const LinearArgs &a, hipStream_t s) {
    switch (a.type) {
        case BERT_AMD_F32: return linear_t<BERT_AMD_F32>(a, s);
        case BERT_AMD_F16: return linear_t<BERT_AMD_F16>(a, s);
        default: return linear_t<BERT_AMD_BF16>(a, s);
    }
}

int64_t linear_grad_ws_bytes(int type, int act, int64_t M, int N, int K) {
    return (act ? round256(M * N * elem_size(type)) : 0) + round256(ceil_div<int64_t>(M, DB_ROWS) * N * 4) +
           std::max(split_bytes(M, K, N), split_bytes(N, K, M));
}

hipError_t launch_linear_grad(const LinearGradArgs &a, hipStream_t s) {
    switch (a.type) {
        case BERT_AMD_F32: return linear_grad_t<BERT_AMD_F32>(a, s);
        case BERT_AMD_F16: return linear_grad_t<BERT_AMD_F16>(a, s);
        default: return linear_grad_t<BERT_AMD_BF16>(a, s);
    }
}

}  // namespace bertamd

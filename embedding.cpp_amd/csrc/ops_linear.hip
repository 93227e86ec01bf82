// ops_linear.hip — the dense layer y = act(x W^T + b) + r and its gradients
// dx = dz W, dw = dz^T x, db = sum of dz over rows, with dz = dy act'(z).
//
// Sums run in f32 on the matrix units.  Past 8 rows a 16-bit layer's dz is rounded
// to its type before the two products, as the matrix units take 16-bit operands: an
// error of half a step in each term, where the result is rounded by half a
// step once more (bf16 16384 x 1024 x 4096 with gelu: dx and dw are 2.34e-3 off in
// the mean square, of which the result's own rounding is 1.66e-3 and f32 sums
// 1.4e-4); db sums the unrounded dz.  Small layers go without that rounding, dz in
// two 16-bit halves (dz_passes): up to twice the products' time.
#include "ops_common.h"

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

namespace bertamd {

namespace {

// v *= act'(z), 8 at a time: one choice of the activation
template <typename T>
__device__ __forceinline__ void slope8(float *v, const float *z, int act) {
    const auto each = [&](auto a) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= act_slope_t<decltype(a)::value, sizeof(T) == 4>(z[i]);
    };
    switch (act) {
        case BERT_AMD_ACT_RELU: each(std::integral_constant<int, BERT_AMD_ACT_RELU>()); break;
        case BERT_AMD_ACT_GELU: each(std::integral_constant<int, BERT_AMD_ACT_GELU>()); break;
        case BERT_AMD_ACT_GELU_ERF: each(std::integral_constant<int, BERT_AMD_ACT_GELU_ERF>()); break;
        case BERT_AMD_ACT_SILU: each(std::integral_constant<int, BERT_AMD_ACT_SILU>()); break;
        case BERT_AMD_ACT_TANH: each(std::integral_constant<int, BERT_AMD_ACT_TANH>()); break;
    }
}

struct Operand {
    const void *p = nullptr;
    int64_t ld = 0;
    bool vec = false;  // p and ld allow 16-byte loads
    bool padded = false;  // zeros follow a row up to a multiple of 16 bytes
    int64_t rest = 0;     // dz in two halves: bytes from the first to the second
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

// ---- few rows ------------------------------------------------------------------
//
// Up to 8 rows of x, as a server's single requests have them: bound by reading
// W once, so no tile and no second launch.  A wave takes COLS rows of W, its
// lanes 16 bytes each of them at a time, and every row of x with them, in f32
// on the vector units; the lanes' sums are joined by a butterfly.  f32 1 x 384
// x 384: 3.6 us, a launch's own length (in 64 x 64 tiles and parts of k: two
// launches, 19 us a call instead of 10).
constexpr int FEW_ROWS = 8;

template <int TYPE, int ROWS, int COLS>
__global__ __launch_bounds__(256) void few_rows_kernel(Operand X, Operand W, int M, int64_t N, int64_t K, Epilogue e) {
    typedef typename Elem<TYPE>::T T;
    constexpr int CH = Elem<TYPE>::CH;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * COLS;
    if (n0 >= N) return;
    float acc[ROWS][COLS] = {};
#pragma unroll 2
    for (int64_t k = CH * lane; k < K; k += 64 * CH) {
        Chunk<T, CH> w[COLS];
#pragma unroll
        for (int c = 0; c < COLS; c++) w[c] = load_chunk<T, CH>((const T *)W.p, W.ld, W.vec, n0 + c, k, N, K);
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            const auto x = load_chunk<T, CH>((const T *)X.p, X.ld, X.vec, r, k, M, K);
#pragma unroll
            for (int c = 0; c < COLS; c++)
#pragma unroll
                for (int j = 0; j < CH; j++) acc[r][c] = __builtin_fmaf((float)x.v[j], (float)w[c].v[j], acc[r][c]);
        }
    }
    float v = 0.f;  // lane r COLS + c: the sum of row r and column c
#pragma unroll
    for (int r = 0; r < ROWS; r++)
#pragma unroll
        for (int c = 0; c < COLS; c++) {
            float a = acc[r][c];
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) a += __shfl_xor(a, d);
            if (lane == r * COLS + c) v = a;
        }
    const int64_t n = n0 + lane % COLS;
    if (lane < ROWS * COLS && lane / COLS < M && n < N) epilogue_store<T>(e, lane / COLS, n, v);
}

// The gradients for as few rows: bound by reading W and writing dw once each, so
// one kernel does both, with dz in f32 throughout (no rounding between).  A wave
// takes 4 rows of W at a time, each lane one of the 8 x 4 dz that belong to
// them, then 4 elements of each row: a rank-ROWS dw leaves at once, dx stays in
// registers, is joined over the workgroup's waves in LDS and over the
// workgroups along N by split_join_kernel, in order.  All three gradients with
// tanh, us a call (in tiles: dz, both products and a join): f32 1 x 384 x 384 8
// (13), 8 x 1024 x 1024 13 (16), 8 x 4096 x 4096 36 (62); bf16 14 (11.4) and 40
// (33) for the latter two, kept for the dz, as over so few terms its rounding
// showed (up to 1.67 times the error of the result's own).
struct FewGrads {
    const void *dy, *z;
    int64_t lddy, ldz;
    int act, M;
    int64_t N, K, rows;  // rows: of W in a workgroup, a multiple of 32
    Operand x, w;
    void *dw;            // or null: not wanted
    int64_t lddw;
    bool vec;            // dw's rows are aligned
    float *db, *part;    // or null
};
constexpr int FEW_COLS = 4;
// FEW_COLS elements of row r from column c of a [nr][nc] matrix
template <typename T>
__device__ __forceinline__ void load_few(const Operand &o, int64_t r, int64_t c, int64_t nr, int64_t nc, T *v) {
    const T *p = (const T *)o.p + r * o.ld + c;
    if (r < nr && o.vec && c + FEW_COLS <= nc) {
        get_n<T, FEW_COLS>(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < FEW_COLS; j++) v[j] = r < nr && c + j < nc ? p[j] : (T)0.f;
    }
}
template <int TYPE, int ROWS>
__global__ __launch_bounds__(512) void few_rows_grad_kernel(FewGrads a) {
    typedef typename Elem<TYPE>::T T;
    constexpr int CH = FEW_COLS, EACH = ROWS * CH;
    __shared__ float sums[4][EACH][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t k = ((int64_t)blockIdx.x * 64 + lane) * CH, end = min(a.N, (int64_t)(blockIdx.y + 1) * a.rows);
    float x[ROWS][CH] = {}, dx[ROWS][CH] = {};
    if (a.dw)
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            T v[CH];
            load_few(a.x, r, k, a.M, a.K, v);
#pragma unroll
            for (int c = 0; c < CH; c++) x[r][c] = (float)v[c];
        }
    for (int64_t n0 = (int64_t)blockIdx.y * a.rows + 4 * wave; n0 < end; n0 += 32) {
        T w[4][CH] = {};
        if (a.part)
#pragma unroll
            for (int j = 0; j < 4; j++) load_few(a.w, n0 + j, k, a.N, a.K, w[j]);
        const int m = lane >> 2;
        const int64_t n = n0 + (lane & 3);
        float dz = 0.f;
        if (m < a.M && n < a.N) {
            dz = (float)((const T *)a.dy)[m * a.lddy + n];
            if (a.act) dz *= act_slope_f((float)((const T *)a.z)[m * a.ldz + n], a.act);
        }
        if (a.db && blockIdx.x == 0) {
            float v = dz;
#pragma unroll
            for (int d = 4; d < 64; d <<= 1) v += __shfl_xor(v, d);
            if (lane < 4 && n < a.N) a.db[n] = v;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float g[ROWS], v[CH] = {};
#pragma unroll
            for (int r = 0; r < ROWS; r++) g[r] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(dz), 4 * r + j));
#pragma unroll
            for (int r = 0; r < ROWS; r++)
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    v[c] = __builtin_fmaf(g[r], x[r][c], v[c]);
                    dx[r][c] = __builtin_fmaf(g[r], (float)w[j][c], dx[r][c]);
                }
            if (!a.dw || n0 + j >= a.N) continue;
            T *to = (T *)a.dw + (n0 + j) * a.lddw + k;
            if (a.vec && k + CH <= a.K) {
                put_n<T, CH>(to, v);
            } else {
#pragma unroll
                for (int c = 0; c < CH; c++)
                    if (k + c < a.K) to[c] = (T)v[c];
            }
        }
    }
    if (!a.part) return;
    const auto leave = [&](int at) {
#pragma unroll
        for (int i = 0; i < EACH; i++) sums[at][i][lane] = dx[i / CH][i % CH];
    };
    const auto take = [&](int at) {
#pragma unroll
        for (int i = 0; i < EACH; i++) dx[i / CH][i % CH] += sums[at][i][lane];
    };
#pragma unroll 1
    for (int half = 4; half; half >>= 1) {
        if (wave >= half && wave < 2 * half) leave(wave - half);
        __syncthreads();
        if (wave < half) take(wave);
        __syncthreads();
    }
    if (wave) return;
#pragma unroll
    for (int r = 0; r < ROWS; r++)
#pragma unroll
        for (int c = 0; c < CH; c++)
            if (r < a.M && k + c < a.K) a.part[((int64_t)blockIdx.y * a.M + r) * a.K + k + c] = dx[r][c];
}

// ---- rows in whole chunks -------------------------------------------------------
//
// A matrix whose rows are not aligned, or no whole chunks long, is copied into
// the workspace with zeros up to the next chunk: one more pass over it, where
// loads of single elements would slow the whole product down (f16 777 x 1001 x
// 513: 5.6 us for both copies and 15 for the product, 26 with single loads in
// the product).
struct Packing {
    const void *from = nullptr;
    void *to = nullptr;
    int64_t ld = 0, rows = 0, cols = 0, ldt = 0;
};
// one or two matrices (blockIdx.y)
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(Packing a, Packing b) {
    constexpr int CH = 16 / sizeof(T);
    const Packing &p = blockIdx.y ? b : a;
    const int64_t chunks = p.ldt / CH;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.rows * chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / chunks, c = (i - r * chunks) * CH;
        *(u32x4 *)((T *)p.to + r * p.ldt + c) = __builtin_bit_cast(u32x4, load_chunk<T, CH>((const T *)p.from, p.ld, false, r, c, p.rows, p.cols));
    }
}

// ---- the tile kernel for operands in whole chunks ---------------------------
//
// The same products from operands whose rows are 16-byte aligned and whose
// contiguous axis is a multiple of 16 bytes long.  BM x BN tiles, k in stages
// of 128 bytes (64 k, in f32 32), two stages of both operands in LDS, loaded
// from memory straight into it (16 bytes a lane, no registers).  One barrier a
// stage: behind it all of the next stage has landed (each wave has waited for
// its own loads) and all waves have taken this stage's last operands, so that
// its buffer is free.
//
// Loads go through a buffer descriptor at the stage's start; a lane whose chunk
// lies outside its matrix gives an offset past the descriptor's range, for
// which the hardware writes zeros, so k and both tile edges need no branch.
//
// An operand stored along k has 128 bytes of a row's k side by side in LDS, 8
// chunks permuted by the row so that the rows of an operand read lie in
// different banks.  An operand stored along m (the gradients' W, dz and x)
// stays so in LDS; ds_read_b64_tr_b16 transposes 4 k x 16 m as it is read, and
// f32 reads its 4 k one by one: no transposed copy is made in memory.
//
// The second matrix is the matrix instruction's row operand, so that a lane
// holds 4 consecutive columns of one row of C at a time.  The finished sums go
// through LDS, 64 columns of each wave's tile at a time, for whole 128-byte
// row pieces on the way out.  One or two waves a SIMD have little to hide
// latencies behind there, so inside the matrix several rows' reads, loads and
// stores go together without a branch between them.
//
// Measured (us): bf16 8192 x 8192 x 8192 861 (1.28 PFLOP/s; all-zero operands
// run a fifth faster: the chip's power bounds it with the LDS reads, 96 of 128
// bytes a clock at the full rate); 32768 x 1024 x 4096 270, 198 of them
// the main loop's and 72 around it, with the matrix units idle: eight rounds of first
// loads and the way out, 33 its LDS passes and 15 its stores; four waves of 128 x 128 each instead
// of eight of 128 x 64 took 5 % longer.  f32 65536 x 1536 x 384 590 (131
// TFLOP/s, the matrix units busy 9 parts in 10).  With one workgroup on a CU a
// wave's LDS reads bound a 128 x 128 stage (0.7 us, its products take 0.25);
// three or four stages in LDS, or 16 waves, did not change that.
constexpr uint32_t OUTSIDE = 0x80000000u;       // an offset past every descriptor's range (2^31 bytes)

// until at most LEFT of this wave's loads are on their way
template <int LEFT>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() { asm volatile("s_barrier" ::: "memory"); }

// 16 bytes a lane from the descriptor's base + off to LDS bytes lds .. lds + 1023.
// The compiler sees neither the load nor what M0 means to it: a write of M0 has to
// be one wait state ahead of a load that reads it, and M0 is named as overwritten
// (clang warns that it keeps no values there itself), so that no write and use of it
// by other instructions end up on both sides of this.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(u32x4 rsrc, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop
// A buffer descriptor of 2^31 bytes from `base` on.  Scalar registers that the
// vector unit has written have to be five wait states old when a load reads
// them, and here the compiler does not know of the load.
__device__ __forceinline__ u32x4 descriptor(const char *base) {
    const uint64_t b = (uint64_t)base;
    u32x4 d = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(b >> 32) & 0xffffu)), OUTSIDE, 0x00020000u};
    asm volatile("s_nop 4" : "+s"(d));
    return d;
}

template <int TYPE> constexpr int stage_k() { return TYPE == BERT_AMD_F32 ? 32 : 64; }

// one operand's tile of R rows (of the product; its contiguous axis if TRANS)
template <int TYPE, bool TRANS, int R, int NT>
struct Tile {
    typedef typename Elem<TYPE>::T T;
    static constexpr int SK = stage_k<TYPE>(), CH = Elem<TYPE>::CH, S = sizeof(T);
    static constexpr int BYTES = R * 128, LOADS = BYTES / 16 / NT;  // 16-byte chunks a thread loads per stage
    static constexpr int CHUNKS = R / CH;                           // of a k row, if TRANS
    const char *base;     // of the stage to load next
    int64_t step;         // bytes from a stage to the next
    int64_t jump = 0;     // and, once `until` stages are loaded, to the first one of a second pass over k
    int until = 0;
    uint32_t off[LOADS];  // from base
    int at[LOADS];        // the chunk's k within the stage

    // the place of k chunk c (of 8) in row r's 128 bytes
    static __device__ __forceinline__ int spread(int r, int c) { return c ^ (r & 7); }
    // the place of column chunk c in k row k: what a read takes at once (4 k of 32 columns; in f32 2 k, 4 apart) in different banks
    static __device__ __forceinline__ int spread_t(int k, int c) { return c ^ ((TYPE == BERT_AMD_F32 ? 2 * (k & 4) : 4 * (k & 3)) & (CHUNKS - 1)); }

    __device__ __forceinline__ void init(const Operand &o, int64_t row0, int64_t rows, int64_t k0) {
        const int t = threadIdx.x;
        if constexpr (!TRANS) {
            base = (const char *)o.p + (row0 * o.ld + k0) * S;
            step = SK * S;
        } else {
            base = (const char *)o.p + (k0 * o.ld + row0) * S;
            step = SK * o.ld * S;
        }
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int q = i * NT + t;
            if constexpr (!TRANS) {
                const int r = q >> 3, c = spread(r, q & 7);
                at[i] = CH * c;
                off[i] = row0 + r < rows ? (uint32_t)(r * o.ld * S) + 16 * c : OUTSIDE;
            } else {
                const int k = q / CHUNKS, c = spread_t(k, q % CHUNKS);
                at[i] = k;
                off[i] = row0 + CH * c < rows ? (uint32_t)(k * o.ld * S) + 16 * c : OUTSIDE;
            }
        }
    }
    // a second pass over the same `stages`, `rest` bytes further on
    __device__ __forceinline__ void again(int stages, int64_t rest) { until = stages, jump = rest - stages * step; }
    // the descriptor of the next stage to load
    template <bool TWO>
    __device__ __forceinline__ u32x4 next_stage() {
        const u32x4 d = descriptor(base);
        base += step;
        if (TWO && --until == 0) base += jump;
        return d;
    }
    // loads FROM .. TO - 1 of a stage to `lds`; `left`: k from the stage's start to the end
    template <int FROM, int TO>
    __device__ __forceinline__ void load(u32x4 d, uint32_t lds, int left) const {
        const uint32_t w = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x >> 6) * 1024);
#pragma unroll
        for (int i = FROM; i < TO; i++) load_to_lds(d, at[i] < left ? off[i] : OUTSIDE, w + i * NT * 16);
    }
    // operand registers of rows r0 .. r0 + 31 and chunks 2 ks, 2 ks + 1 of the stage at `lds`: lane half h has chunk 2 ks + h's k
    static __device__ __forceinline__ u32x4 read(const char *lds, int r0, int ks) {
        const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31;
        if constexpr (!TRANS) {
            return *(const u32x4 *)(lds + (r0 + c) * 128 + spread(c, 2 * ks + h) * 16);
        } else if constexpr (TYPE == BERT_AMD_F32) {
            const int col = r0 + c;
            const char *p = lds + (8 * ks + 4 * h) * (R * 4) + spread_t(4 * h, col >> 2) * 16 + (col & 3) * 4;
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = *(const uint32_t *)(p + i * R * 4);
            return v;
        } else {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
            // lane i of each 16 gives the address of k row i / 4's columns 4 (i % 4) .. + 3 and gets column i of the 4 rows
            const int col = r0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            const int k = 16 * ks + 8 * h + ((lane & 15) >> 2);
            const char *p0 = lds + k * (R * 2) + spread_t(k, col >> 3) * 16 + (col & 7) * 2;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p0);
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p0 + 4 * R * 2));
            struct { s16x4 a, b; } both = {a, b};
            return __builtin_bit_cast(u32x4, both);
        }
    }
};

template <int... I, typename F>
__device__ __forceinline__ void for_const_(std::integer_sequence<int, I...>, const F &f) { (f(std::integral_constant<int, I>()), ...); }
// f(0), .. f(N - 1), each number a constant
template <int N, typename F>
__device__ __forceinline__ void for_const(const F &f) { for_const_(std::make_integer_sequence<int, N>(), f); }

// c += the products of two operands' 32 rows over the 16 (f32: 8) k that `read` gave
template <int TYPE>
__device__ __forceinline__ f32x16 multiply(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (TYPE == BERT_AMD_F16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else if constexpr (TYPE == BERT_AMD_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)  // k and k + 4 at a time, the same order in both operands
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    }
}

// v = act(v), N at a time: one choice of the activation
template <typename T, int N>
__device__ __forceinline__ void act_n(float *v, int act) {
    constexpr bool WIDE = sizeof(T) == 4;
    const auto each = [&](auto a) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = act_t<decltype(a)::value, WIDE>(v[i]);
    };
    switch (act) {
        case BERT_AMD_ACT_RELU: each(std::integral_constant<int, BERT_AMD_ACT_RELU>()); break;
        case BERT_AMD_ACT_GELU: each(std::integral_constant<int, BERT_AMD_ACT_GELU>()); break;
        case BERT_AMD_ACT_GELU_ERF: each(std::integral_constant<int, BERT_AMD_ACT_GELU_ERF>()); break;
        case BERT_AMD_ACT_SILU: each(std::integral_constant<int, BERT_AMD_ACT_SILU>()); break;
        case BERT_AMD_ACT_TANH: each(std::integral_constant<int, BERT_AMD_ACT_TANH>()); break;
    }
}

// LDS row of the epilogue: a wave's 64 columns and 16 bytes more, so that the rows of a write start in different banks
constexpr int OUT_LD = 68;

// C = A B^T as a launch has it: tiles times parts of k workgroups
struct Product {
    Operand A, B;
    int64_t M = 0, N = 0, K = 0, per = 0;  // per: k of a part
    int tiles = 0, parts = 1;
    float *part = nullptr;                 // where the parts' sums go; else through `e`
    Epilogue e;
    bool vec = false;                      // the epilogue's rows are aligned
};

// `block` of p.tiles, part `split` of k; TWO: A is the sum of two matrices, A.rest apart, k is gone over twice
template <int TYPE, bool TA, bool TBT, int BM, int BN, int WM, int WN, bool TWO>
__device__ __forceinline__ void stage_product(const Product &p, char *smem, int block, int split) {
    typedef typename Elem<TYPE>::T T;
    const Operand A = p.A, B = p.B;
    const int64_t M = p.M, N = p.N, K = p.K;
    float *part = p.part;
    const Epilogue e = p.e;
    const bool vec = p.vec;
    constexpr int NT = WM * WN * 64, TM = BM / WM / 32, TN = BN / WN / 32;
    static_assert(BN / WN % 64 == 0, "the epilogue takes 64 columns of a wave's tile at a time");
    typedef Tile<TYPE, TA, BM, NT> TileA;
    typedef Tile<TYPE, TBT, BN, NT> TileB;
    constexpr int STAGE = TileA::BYTES + TileB::BYTES;
    // workgroups of one XCD take neighbouring tiles, 8 tile rows at a time: they share operand rows in its L2
    const int tm = (int)ceil_div<int64_t>(M, BM), tn = (int)ceil_div<int64_t>(N, BN), all = tm * tn;
    const int xcd = block & 7, slot = block >> 3;
    const int tile = xcd * (all >> 3) + min(xcd, all & 7) + slot;
    const int group = tile / (8 * tn), in_group = tile - group * 8 * tn, high = min(8, tm - 8 * group);
    const int64_t m0 = (int64_t)(8 * group + in_group % high) * BM, n0 = (int64_t)(in_group / high) * BN;
    const int64_t ka = split * p.per, kb = min(K, ka + p.per);
    TileA ta;
    TileB tb;
    ta.init(A, m0, M, ka);
    tb.init(B, n0, N, ka);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
    const int wave = threadIdx.x >> 6, wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    // this lane's columns' bias, on its way from here (none: zeros; past the end: the last one, not used)
    const int lane = threadIdx.x & 63;
    float biases[TN / 2][8] = {};
    if (e.bias && !part)
#pragma unroll
        for (int h = 0; h < TN / 2; h++)
#pragma unroll
            for (int i = 0; i < 8; i++) biases[h][i] = e.bias[min(n0 + wn + 64 * h + 8 * (lane & 7) + i, N - 1)];
    f32x16 acc[TM][TN] = {};
    constexpr int SK = stage_k<TYPE>(), KS = 4;
    const int64_t span = ceil_div(kb - ka, (int64_t)SK) * SK, end = TWO ? ka + 2 * span : kb;
    if constexpr (TWO) ta.again((int)(span / SK), A.rest), tb.again((int)(span / SK), 0);
    u32x4 a[2][TM], b[2][TN];
    const auto read_a = [&](int set, int i, int from, int ks) { a[set][i] = TileA::read(smem + from * STAGE, wm + 32 * i, ks); };
    const auto read_b = [&](int set, int i, int from, int ks) { b[set][i] = TileB::read(smem + from * STAGE + TileA::BYTES, wn + 32 * i, ks); };
    const auto left_at = [&](int64_t k0) {
        if (TWO && k0 >= ka + span) k0 -= span;
        return (int)max((int64_t)0, min((int64_t)SK, kb - k0));
    };
#pragma unroll
    for (int i = 0; i < 2; i++) {
        ta.template load<0, TileA::LOADS>(ta.template next_stage<TWO>(), lds + i * STAGE, left_at(ka + i * SK));
        tb.template load<0, TileB::LOADS>(tb.template next_stage<TWO>(), lds + i * STAGE + TileA::BYTES, left_at(ka + i * SK));
    }
    wait_loads<TileA::LOADS + TileB::LOADS>();
    barrier();
#pragma unroll
    for (int i = 0; i < TN; i++) read_b(0, i, 0, 0);
#pragma unroll
    for (int i = 0; i < TM; i++) read_a(0, i, 0, 0);
    int buf = 0;
    u32x4 stage = {};
    for (int64_t k0 = ka; k0 < end; k0 += SK, buf ^= 1) {
        // The loads of the stage after the next go out between the products of
        // this stage's last quarter (its second matrix, once the barrier has freed
        // the buffer) and the next stage's first (its first matrix): a burst of them would hold up
        // the products behind it, and they have half a stage left to arrive in.
        // Past the end they write zeros, and the last reads take what nothing multiplies.
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int set = ks & 1, next = set ^ 1, from = ks < KS - 1 ? buf : buf ^ 1, kn = (ks + 1) % KS;
            if (ks == KS - 1) {
                wait_reads();
                wait_loads<0>();
                barrier();
                stage = tb.template next_stage<TWO>();
            }
            if (ks == 0 && k0 > ka) stage = ta.template next_stage<TWO>();
            for_const<TM>([&](auto ic) {
                constexpr int i = ic.value;
                if (ks == KS - 1) tb.template load<i * TileB::LOADS / TM, (i + 1) * TileB::LOADS / TM>(stage, lds + buf * STAGE + TileA::BYTES, left_at(k0 + 2 * SK));
                if (ks == 0 && k0 > ka) ta.template load<i * TileA::LOADS / TM, (i + 1) * TileA::LOADS / TM>(stage, lds + (buf ^ 1) * STAGE, left_at(k0 + SK));
#pragma unroll
                for (int j = i * TN / TM; j < (i + 1) * TN / TM; j++) read_b(next, j, from, kn);
                read_a(next, i, from, kn);
#pragma unroll
                for (int j = 0; j < TN; j++) acc[i][j] = multiply<TYPE>(b[set][j], a[set][i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    }
    wait_reads();
    wait_loads<0>();
    barrier();  // the stages' last loads and reads are done: the LDS is the epilogue's
    constexpr int WR = std::min(BM / WM, 64), PARTS = BM / WM / WR, G = std::min(WR / 8, sizeof(T) == 4 ? 2 : 4);
    float *out = (float *)smem + wave * WR * OUT_LD;
    const int row0 = lane >> 3, col = 8 * (lane & 7);
#pragma unroll 1
    for (int pass = 0; pass < TN / 2 * PARTS; pass++) {
        const int half = pass / PARTS, rows = pass % PARTS;
        const int64_t n = n0 + wn + 64 * half + col, m = m0 + wm + WR * rows + row0;
        float bias[8];
#pragma unroll
        for (int i = 0; i < 8; i++) bias[i] = half ? biases[1 % (TN / 2)][i] : biases[0][i];
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int i = 0; i < TM; i++)
                if (j / 2 == half && 32 * i / WR == rows)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        *(f32x4 *)(out + (32 * i % WR + (lane & 31)) * OUT_LD + 32 * (j & 1) + 8 * c + 4 * (lane >> 5)) =
                            f32x4{acc[i][j][4 * c], acc[i][j][4 * c + 1], acc[i][j][4 * c + 2], acc[i][j][4 * c + 3]};
        wave_sync();
        if (vec && !part && m0 + BM <= M && n0 + BN <= N) {
            const T *r = (const T *)e.r + m * e.ldr + n;
            T *y = (T *)e.y + m * e.ldy + n, *z = (T *)e.z + m * e.ldz + n;
#pragma unroll 1
            for (int g = 0; g < WR; g += 8 * G) {
                float v[8 * G];
#pragma unroll
                for (int i = 0; i < G; i++)
#pragma unroll
                    for (int c = 0; c < 8; c++) v[8 * i + c] = out[(g + 8 * i + row0) * OUT_LD + col + c] + bias[c];
                if (e.z)
#pragma unroll
                    for (int i = 0; i < G; i++) put8(z + (g + 8 * i) * e.ldz, v + 8 * i);
                act_n<T, 8 * G>(v, e.act);
                if (e.r)
#pragma unroll
                    for (int i = 0; i < G; i++) add8(r + (g + 8 * i) * e.ldr, v + 8 * i);
#pragma unroll
                for (int i = 0; i < G; i++) put8(y + (g + 8 * i) * e.ldy, v + 8 * i);
            }
        } else {  // an edge of the matrix, rows that are not aligned, or parts: a lane a column, four rows at a time
            const int64_t n1 = n0 + wn + 64 * half + lane, m1 = m0 + wm + WR * rows;
            const float bias1 = e.bias && !part ? e.bias[min(n1, N - 1)] : 0.f;
            const int there = (int)min((int64_t)WR, M - m1);
            if (n1 < N)
#pragma unroll 1
                for (int g = 0; g < there; g += 4) {
                    float v[4], add[4] = {};
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = out[(g + i) * OUT_LD + lane] + bias1;
                    if (part) {
                        float *q = part + (split * M + m1 + g) * N + n1;
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (g + i < there) q[i * N] = v[i];
                        continue;
                    }
                    const T *r = (const T *)e.r + (m1 + g) * e.ldr + n1;
                    T *y = (T *)e.y + (m1 + g) * e.ldy + n1, *z = (T *)e.z + (m1 + g) * e.ldz + n1;
                    if (e.r)
#pragma unroll
                        for (int i = 0; i < 4; i++) add[i] = (float)r[min(i, there - g - 1) * e.ldr];
                    if (e.z)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (g + i < there) z[i * e.ldz] = (T)v[i];
                    act_n<T, 4>(v, e.act);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (g + i < there) y[i * e.ldy] = (T)(v[i] + add[i]);
                }
        }
        wave_sync();
    }
}

template <int TYPE, bool TA, bool TBT, int BM, int BN, int WM, int WN, bool TWO>
__global__ __launch_bounds__(WM *WN * 64, 2) void stage_gemm_kernel(Product p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    stage_product<TYPE, TA, TBT, BM, BN, WM, WN, TWO>(p, smem, blockIdx.x, blockIdx.z);
}

// Both products of a small layer's gradients at once, in tiles of 64 x BN: each
// alone leaves most of the chip idle, and a launch less counts there.
template <int TYPE, int BN, int WN, bool TWO>
__global__ __launch_bounds__(128 * WN, 2) void pair_gemm_kernel(Product dx, Product dw) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int first = dx.tiles * dx.parts, b = blockIdx.x;
    if (b < first)
        stage_product<TYPE, false, true, 64, BN, 2, WN, TWO>(dx, smem, b % dx.tiles, b / dx.tiles);
    else
        stage_product<TYPE, true, true, 64, BN, 2, WN, TWO>(dw, smem, (b - first) % dw.tiles, (b - first) / dw.tiles);
}

// The parts of one or two products (blockIdx.y) added in order, COLS columns a
// thread: bound by memory (four parts of 4096 x 1024: 75 MB in 14.5 us).  A product in parts has under 2^31 elements (plan_for).
template <typename T, int COLS>
__global__ __launch_bounds__(256) void split_join_kernel(Product a, Product b) {
    const Product &p = blockIdx.y ? b : a;
    if (!p.part) return;
    const uint32_t across = (uint32_t)p.N / COLS, all = (uint32_t)p.M * across;
    const int64_t size = p.M * p.N;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < all; i += gridDim.x * 256) {
        const uint32_t m = i / across, n = (i - m * across) * COLS;
        const float *from = p.part + (int64_t)m * p.N + n;
        float v[COLS] = {};
#pragma unroll 4
        for (int s = 0; s < p.parts; s++) {
            float w[COLS];
            get_n<float, COLS>(from + s * size, w);
#pragma unroll
            for (int c = 0; c < COLS; c++) v[c] += w[c];
        }
        const Epilogue &e = p.e;
#pragma unroll
        for (int c = 0; c < COLS; c++) v[c] += e.bias ? e.bias[n + c] : 0.f;
        if (e.z) put_n<T, COLS>((T *)e.z + m * e.ldz + n, v);
        act_n<T, COLS>(v, e.act);
        if (e.r) {
            float w[COLS];
            get_n<T, COLS>((const T *)e.r + m * e.ldr + n, w);
#pragma unroll
            for (int c = 0; c < COLS; c++) v[c] += w[c];
        }
        put_n<T, COLS>((T *)e.y + m * e.ldy + n, v);
    }
}

// dz = dy act'(z) in the layer's type, rows `lddz` apart with zeros past their
// end (`rest`: and there what that rounding left, a finite dz past the type's largest
// value with it), and the unrounded dz's column sums over `rows` rows at a time: CT
// threads of 8 columns each, 256 / CT rows side by side, their sums joined in
// LDS in a fixed order.
template <typename T>
__device__ __forceinline__ void halves(float v, float &high, float &low) {
    constexpr float MOST = std::is_same<T, _Float16>::value ? 65504.f : 0x1.fep127f;
    high = (float)(T)v;
    if (fabsf(high) > MOST && fabsf(v) <= 0x1.fffffep127f) high = v > 0.f ? MOST : -MOST;
    low = fabsf(high) <= MOST ? v - high : 0.f;
}
template <typename T, int CT>
__global__ __launch_bounds__(256) void dz_kernel(const T *dy, int64_t lddy, const T *z, int64_t ldz, int act, int64_t M, int64_t N,
                                                 int64_t rows, T *dz, T *rest, int64_t lddz, float *part, bool vec) {
    constexpr int RT = 256 / CT;
    __shared__ float sums[RT][CT][9];
    const int c = threadIdx.x % CT, r = threadIdx.x / CT;
    const int64_t n = ((int64_t)blockIdx.x * CT + c) * 8, m1 = min(M, (int64_t)(blockIdx.y + 1) * rows);
    const bool whole = vec && n + 8 <= N;
    float sum[8] = {};
#pragma unroll 2
    for (int64_t m = (int64_t)blockIdx.y * rows + r; m < m1; m += RT) {
        float v[8] = {}, s[8] = {};
        if (whole) {
            add8(dy + m * lddy + n, v);
            if (act) add8(z + m * ldz + n, s);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (n + i < N) {
                    v[i] = (float)dy[m * lddy + n + i];
                    if (act) s[i] = (float)z[m * ldz + n + i];
                }
        }
        if (act) slope8<T>(v, s, act);
        if (dz) {
            const auto keep = [&](T *to, const float *from) {
                if (n + 8 <= lddz) {
                    put8(to + m * lddz + n, from);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (n + i < lddz) to[m * lddz + n + i] = (T)from[i];
                }
            };
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (n + i >= N) v[i] = 0.f;
            if (!rest) {
                keep(dz, v);
            } else {
                float high[8], low[8];
#pragma unroll
                for (int i = 0; i < 8; i++) halves<T>(v[i], high[i], low[i]);
                keep(dz, high);
                keep(rest, low);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] += v[i];
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < 8; i++) sums[r][c][i] = sum[i];
    __syncthreads();
    // eight rows' sums a thread, then (one column of threads: 32 such) those
    constexpr int COLS = CT * 8, GROUPS = 256 / COLS;
    const int mine = threadIdx.x % COLS, group = threadIdx.x / COLS;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) v += sums[8 * group + i][mine >> 3][mine & 7];
    if constexpr (GROUPS > 1) {
        __syncthreads();
        float *joined = &sums[0][0][0];
        joined[threadIdx.x] = v;
        __syncthreads();
        v = 0.f;
        if (group == 0)
#pragma unroll
            for (int i = 0; i < GROUPS; i++) v += joined[i * COLS + mine];
    }
    const int64_t col = (int64_t)blockIdx.x * COLS + mine;
    if (group == 0 && col < N) part[blockIdx.y * N + col] = v;
}

// the column sums of `part`: 16 columns, 64 rows side by side (256 rows of 4096: 5.3 us, one dependent chain of loads)
__global__ __launch_bounds__(1024) void column_sum_kernel(const float *part, int64_t rows, int64_t N, float *out) {
    __shared__ float sums[64][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const int64_t n = (int64_t)blockIdx.x * 16 + c;
    float v = 0.f;
    if (n < N)
#pragma unroll 4
        for (int64_t b = r; b < rows; b += 64) v += part[b * N + n];
    sums[r][c] = v;
    __syncthreads();
    if (r || n >= N) return;
#pragma unroll 16
    for (int i = 1; i < 64; i++) v += sums[i][c];
    out[n] = v;
}

// How dz_kernel goes over its matrix.  Up to 1024 rows and 2^21 elements: 8
// columns wide, all rows, and the sums are the bias's gradient at once.  Else 8 or,
// past 128 columns, 256 columns wide, whole pieces of rows, about 2048 workgroups
// (16384 x 4096 in bf16: 403 MB in 75 us), and the sums take a launch more.  The
// bias's gradient alone, us, 8 and 256 columns wide: bf16 256 x 384 4.0 and 11.3,
// 1024 x 1024 6.2 and 10.6, 512 x 4096 13.3 and 10.8, 1024 x 4096 23 and 11; f32
// 3.8 and 13.9, 8.0 and 13.1, 14.1 and 13.2, 24 and 15.  With dx 512 x 4096 comes
// out even (bf16 29.7 and 30.9), 1000 x 2500 takes 52 and 37: past that many
// elements the few bytes of a row cost whole cache lines of several L2s.
struct DzPlan {
    bool narrow;
    int64_t rows;
};
DzPlan dz_plan(int64_t M, int64_t N) {
    if (M <= 1024 && M * N <= 1 << 21) return {true, std::max<int64_t>(M, 1)};
    const bool narrow = N <= 128;
    const int64_t across = ceil_div<int64_t>(N, narrow ? 8 : 256);
    int64_t rows = narrow ? 256 : 64;
    while (rows < M && ceil_div(M, rows) * across > 2048) rows *= 2;
    return {narrow, rows};
}

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// How a product runs: its tile and in how many parts k is split.
struct Plan {
    int rows = 64, cols = 64;  // of a tile
    int splits = 1;
    int64_t per = 0;           // k of a split
};
// The tile and split whose estimated time is least.  A CU's share of the
// workgroups runs in rounds of as many as it holds; a round takes its stages'
// time and a time around them, and where k is split its parts are joined by
// another pass.  A stage takes `alone` us where a CU has one workgroup, and
// `more` for each other one.
// The numbers are fitted to products of 16 .. 65536 rows, 384 .. 4096 wide, in
// every tile and up to 64 parts (us a call): f32 4096 x 1024 x 1024 75 in 128
// wide tiles, 76 in 64 wide, 92 in two parts of k; bf16 16384 x 1024 x 1024 37
// in 256 wide, 40 in 128, 59 in 64; bf16 1536 x 384 over k = 65536 123 in 21
// parts of 256 wide tiles, 549 unsplit in 64 wide.  The choice was on average
// 1 % off the best measured, at most 9 %.
Plan plan_for(int type, int64_t M, int64_t N, int64_t K, int passes = 1) {
    struct Form {
        int rows, cols;
        double alone, more, around;
        int holds;
    };
    static const Form half[] = {{256, 256, 1.8, 0, 7, 1}, {128, 128, .72, .33, 4, 2}, {64, 64, .5, .11, 3, 4}};
    static const Form f32[] = {{128, 128, 2.15, 1.72, 4.5, 2}, {64, 128, 1.18, .89, 3, 3}, {64, 64, 1.3, .42, 2.7, 4}};
    const bool wide = type == BERT_AMD_F32;
    const int sk = wide ? 32 : 64;
    Plan best;
    best.per = 64;
    double least = 1e30;
    for (int i = 0; i < 3; i++) {
        const Form &f = wide ? f32[i] : half[i];
        const int64_t tiles = ceil_div<int64_t>(M, f.rows) * ceil_div<int64_t>(N, f.cols);
        if (!tiles) continue;
        const int64_t splits[] = {1, 2, 4, 6, 8, 12, 16, 256 / tiles, 512 / tiles, 768 / tiles};
        for (const int64_t n : splits) {
            if (n < 1 || (n > 1 && (n > 64 || K < n * sk * 2 || tiles * n > 1600))) continue;
            const int64_t per = std::max<int64_t>(64, ceil_div(ceil_div(K, n), (int64_t)64) * 64), parts = ceil_div(K, per);
            const int64_t each = ceil_div(tiles * parts, (int64_t)256), left = each % f.holds;
            const double stages = (double)passes * ceil_div(per, (int64_t)sk);
            const auto round = [&](int64_t wgs) { return stages * (f.alone + (wgs - 1) * f.more) + f.around; };
            const double t = each / f.holds * round(f.holds) + (left ? round(left) : 0) + (parts > 1 ? 3.7 + 1.6e-6 * parts * M * N : 0);
            if (t < least) least = t, best = {f.rows, f.cols, (int)parts, per};
        }
    }
    best.splits = std::max(1, best.splits);
    return best;
}
// bytes of a product's split sums
int64_t split_bytes(int type, int64_t M, int64_t N, int64_t K, int passes = 1) {
    const Plan p = plan_for(type, M, N, K, passes);
    return p.splits > 1 ? round256(p.splits * M * N * 4) : 0;
}

// whether a layer's two gradient products share a launch: both in the same
// small tiles (256 x 384 x 384 in f32 29 -> 22 us for all three gradients)
bool gradients_in_pair(int type, int64_t M, int64_t N, int64_t K, int passes) {
    const Plan dx = plan_for(type, M, K, N, passes), dw = plan_for(type, N, K, M, passes);
    return M > 0 && dx.rows == 64 && dw.rows == 64 && dx.cols == dw.cols;
}

// Passes over dz in the gradients' products: two, of its two halves, where dz, dx or
// dw has few elements.  With dz rounded dx and dw are 1.41 times as far off as their own
// rounding in the mean square, give or take about 1.2 over the root of the least of
// the three sizes (f16 1065 x 20 x 11: up to 1.66, bf16 11 x 605 x 11 1.52); in two
// halves 1.00.  us for all three gradients, rounded and in halves: bf16 9 x 64 x 64 7.8
// and 8.7, 64 x 4096 x 64 7.5 and 8.5, 1065 x 20 x 11 16.7 and 17.5, but 256 x 384 x
// 384 10.4 and 14.6, 1024 x 1024 x 1024 25 and 38, 16384 x 1024 x 4096 354 and 610.
constexpr int64_t FEW_ELEMENTS = 4096;
int dz_passes(int type, int act, int64_t M, int64_t N, int64_t K) {
    return type != BERT_AMD_F32 && act != BERT_AMD_ACT_NONE && std::min({M * N, M * K, N * K}) <= FEW_ELEMENTS ? 2 : 1;
}

// Up to 8 rows, and no more than 8192 columns of dz: with more the tiles' workgroups
// win (bf16 1 x 768 x 65536: 67 us, 134 here) and dz's roundings average out.
bool few_grads(int64_t M, int64_t N) { return M > 0 && M <= FEW_ROWS && N <= 8192; }
// workgroups along N, at most 64, as their sums are joined one after the other
int64_t few_grad_parts(int64_t N, int64_t K) {
    const int64_t across = ceil_div<int64_t>(K, 64 * FEW_COLS);
    return std::min(ceil_div(N, (int64_t)32), std::max((int64_t)8, std::min((int64_t)64, 256 / across)));
}

int64_t padded(int type, int64_t n) {
    const int64_t ch = 16 / elem_size(type);
    return (n + ch - 1) / ch * ch;
}
int64_t packed_bytes(int type, int64_t rows, int64_t cols) { return round256(rows * padded(type, cols) * elem_size(type)); }

// whether the stage kernel takes a matrix with rows of `cols` as it is: whole aligned chunks, offsets within a tile under 2^31
bool whole_rows(const Operand &o, int type, int64_t cols) {
    return o.padded || (o.vec && cols % (16 / elem_size(type)) == 0 && o.ld < (1 << 21));
}

// one or two matrices with rows of `cols` as the stage kernel takes them; copies go to `ws`, which moves on
template <typename T>
hipError_t pack(int type, Operand *o, const int64_t *rows, int n, int64_t cols, char *&ws, hipStream_t s) {
    Packing p[2];
    int64_t most = 0;
    int count = 0;
    for (int i = 0; i < n; i++) {
        if (whole_rows(o[i], type, cols)) continue;
        const int64_t ld = padded(type, cols);
        p[count++] = {o[i].p, ws, o[i].ld, rows[i], cols, ld};
        o[i] = {ws, ld, true, true};
        most = std::max(most, rows[i] * ld * (int64_t)sizeof(T) / 16);
        ws += packed_bytes(type, rows[i], cols);
    }
    if (!most) return hipSuccess;
    return launch(pack_kernel<T>, dim3(std::min<int64_t>(1 << 14, ceil_div<int64_t>(most, 256)), count), dim3(256), 0, s, p[0], p[1]);
}

template <int TYPE>
Product product(const Operand &A, const Operand &B, int64_t M, int64_t N, int64_t K, const Plan &plan, void *ws, const Epilogue &e) {
    const auto ok = [](const void *q, int64_t ld) { return !q || aligned16(q, ld * (int64_t)sizeof(typename Elem<TYPE>::T)); };
    Product p;
    p.A = A, p.B = B, p.M = M, p.N = N, p.K = K, p.per = plan.per, p.parts = plan.splits;
    p.tiles = (int)(ceil_div<int64_t>(M, plan.rows) * ceil_div<int64_t>(N, plan.cols));
    p.part = plan.splits > 1 ? (float *)ws : nullptr;
    p.e = e;
    p.vec = ok(e.y, e.ldy) && ok(e.z, e.ldz) && ok(e.r, e.ldr);
    return p;
}

constexpr int stage_lds(int BM, int BN, int WM, int WN) {
    return std::max(2 * (BM + BN) * 128, std::min(BM / WM, 64) * WM * WN * OUT_LD * 4);
}

template <int TYPE, bool TA, bool TBT, int BM, int BN, int WM, int WN, bool TWO>
hipError_t launch_stage(const Product &p, hipStream_t s) {
    constexpr int lds = stage_lds(BM, BN, WM, WN);
    const auto k = stage_gemm_kernel<TYPE, TA, TBT, BM, BN, WM, WN, TWO>;
    if (lds > 65536) {  // beyond a launch's default: asked for once on each device
        static std::atomic<uint64_t> asked{0};
        int dev = 0;
        if (hipError_t r = hipGetDevice(&dev); r != hipSuccess) return r;
        const uint64_t bit = 1ull << (dev & 63);
        if (!(asked.load(std::memory_order_relaxed) & bit) || dev > 63) {
            if (hipError_t r = hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds); r != hipSuccess) return r;
            asked.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    return launch(k, dim3(p.tiles, 1, p.parts), dim3(WM * WN * 64), lds, s, p);
}

template <typename T>
hipError_t join(const Product &a, const Product &b, hipStream_t s) {
    const int64_t most = std::max(a.part ? a.M * a.N : 0, b.part ? b.M * b.N : 0);
    if (!most) return hipSuccess;
    const auto four = [](const Product &p) { return !p.part || (p.vec && p.N % 4 == 0); };
    const int two = b.part ? 2 : 1;
    if (four(a) && four(b))
        return launch(split_join_kernel<T, 4>, dim3(std::min<int64_t>(4096, ceil_div<int64_t>(most, 1024)), two), dim3(256), 0, s, a, b);
    return launch(split_join_kernel<T, 1>, dim3(std::min<int64_t>(4096, ceil_div<int64_t>(most, 256)), two), dim3(256), 0, s, a, b);
}

// C = A B^T of two matrices in whole chunks
template <int TYPE, bool TA, bool TBT, bool TWO = false>
hipError_t gemm(const Operand &A, const Operand &B, int64_t M, int64_t N, int64_t K, void *ws, const Epilogue &e, hipStream_t s) {
    const Plan plan = plan_for(TYPE, M, N, K, TWO ? 2 : 1);
    const Product p = product<TYPE>(A, B, M, N, K, plan, ws, e);
    hipError_t r = hipSuccess;
    if (plan.cols == 64) r = launch_stage<TYPE, TA, TBT, 64, 64, 2, 1, TWO>(p, s);
    else if (plan.rows == 128) r = launch_stage<TYPE, TA, TBT, 128, 128, 2, 2, TWO>(p, s);
    else if constexpr (TYPE == BERT_AMD_F32) r = launch_stage<TYPE, TA, TBT, 64, 128, 2, 2, TWO>(p, s);
    else r = launch_stage<TYPE, TA, TBT, 256, 256, 2, 4, TWO>(p, s);
    return r != hipSuccess ? r : join<typename Elem<TYPE>::T>(p, Product(), s);
}

Operand operand(const void *p, int64_t ld, int type) { return {p, ld, aligned16(p, ld * elem_size(type))}; }

template <int TYPE, int COLS>
hipError_t few_rows(const Operand &x, const Operand &w, const LinearArgs &a, const Epilogue &e, hipStream_t s) {
    const dim3 grid(ceil_div(a.N, 4 * COLS));
    const int M = (int)a.M;
    if (M == 1) return launch(few_rows_kernel<TYPE, 1, COLS>, grid, dim3(256), 0, s, x, w, M, a.N, a.K, e);
    if (M == 2) return launch(few_rows_kernel<TYPE, 2, COLS>, grid, dim3(256), 0, s, x, w, M, a.N, a.K, e);
    if (M <= 4) return launch(few_rows_kernel<TYPE, 4, COLS>, grid, dim3(256), 0, s, x, w, M, a.N, a.K, e);
    return launch(few_rows_kernel<TYPE, 8, COLS>, grid, dim3(256), 0, s, x, w, M, a.N, a.K, e);
}

template <int TYPE>
hipError_t linear_t(const LinearArgs &a, hipStream_t s) {
    typedef typename Elem<TYPE>::T T;
    const Operand x = operand(a.x, a.ldx, TYPE), w = operand(a.w, a.ldw, TYPE);
    const Epilogue e = {a.act, a.bias, a.r, a.y, a.z, a.ldr, a.ldy, a.ldz};
    if (a.M <= FEW_ROWS)  // one column a wave fills the chip sooner, four read x a quarter as often
        return a.N < 4096 ? few_rows<TYPE, 1>(x, w, a, e, s) : few_rows<TYPE, 4>(x, w, a, e, s);
    char *ws = (char *)a.ws;
    Operand both[] = {x, w};
    const int64_t rows[] = {a.M, a.N};
    if (hipError_t r = pack<T>(TYPE, both, rows, 2, a.K, ws, s); r != hipSuccess) return r;
    return gemm<TYPE, false, false>(both[0], both[1], a.M, a.N, a.K, ws, e, s);
}

template <int TYPE>
hipError_t few_rows_grad(const LinearGradArgs &a, hipStream_t s) {
    typedef typename Elem<TYPE>::T T;
    const int64_t e = sizeof(T), parts = few_grad_parts(a.N, a.K);
    FewGrads f = {};
    f.dy = a.dy, f.z = a.z, f.lddy = a.lddy, f.ldz = a.ldz, f.act = a.act, f.M = (int)a.M, f.N = a.N, f.K = a.K;
    f.rows = ceil_div(ceil_div<int64_t>(a.N, parts), (int64_t)32) * 32;
    f.x = operand(a.x, a.ldx, TYPE), f.w = operand(a.w, a.ldw, TYPE);
    f.dw = a.dw, f.lddw = a.lddw, f.vec = aligned16(a.dw, a.lddw * e), f.db = a.db;
    f.part = a.dx ? (float *)a.ws : nullptr;
    const dim3 grid(a.dx || a.dw ? ceil_div(a.K, 64 * FEW_COLS) : 1, ceil_div<int64_t>(a.N, f.rows));
    const auto kernel = a.M == 1   ? few_rows_grad_kernel<TYPE, 1>
                        : a.M == 2 ? few_rows_grad_kernel<TYPE, 2>
                        : a.M <= 4 ? few_rows_grad_kernel<TYPE, 4>
                                   : few_rows_grad_kernel<TYPE, 8>;
    if (hipError_t r = launch(kernel, grid, dim3(512), 0, s, f); r != hipSuccess) return r;
    Product dx;
    dx.M = a.M, dx.N = a.K, dx.parts = (int)grid.y, dx.part = f.part;
    dx.e.y = a.dx, dx.e.ldy = a.lddx, dx.vec = aligned16(a.dx, a.lddx * e);
    return join<T>(dx, Product(), s);
}

// dx = dz W and dw = dz^T x
template <int TYPE, bool TWO>
hipError_t grad_products(const LinearGradArgs &a, const Operand &dz, char *ws, hipStream_t s) {
    typedef typename Elem<TYPE>::T T;
    constexpr int PASSES = TWO ? 2 : 1;
    Epilogue ex, ew;
    ex.y = a.dx, ex.ldy = a.lddx;
    ew.y = a.dw, ew.ldy = a.lddw;
    if (a.dx && a.dw && gradients_in_pair(TYPE, a.M, a.N, a.K, PASSES)) {
        Operand wx[] = {operand(a.w, a.ldw, TYPE), operand(a.x, a.ldx, TYPE)};
        const int64_t rows[] = {a.N, a.M};
        if (hipError_t r = pack<T>(TYPE, wx, rows, 2, a.K, ws, s); r != hipSuccess) return r;
        const Plan plan = plan_for(TYPE, a.M, a.K, a.N, PASSES);
        const Product dx = product<TYPE>(dz, wx[0], a.M, a.K, a.N, plan, ws, ex);
        ws += split_bytes(TYPE, a.M, a.K, a.N, PASSES);
        const Product dw = product<TYPE>(dz, wx[1], a.N, a.K, a.M, plan_for(TYPE, a.N, a.K, a.M, PASSES), ws, ew);
        const dim3 grid(dx.tiles * dx.parts + dw.tiles * dw.parts);
        hipError_t r = hipErrorInvalidValue;
        if (plan.cols == 64)
            r = launch(pair_gemm_kernel<TYPE, 64, 1, TWO>, grid, dim3(128), stage_lds(64, 64, 2, 1), s, dx, dw);
        else if constexpr (TYPE == BERT_AMD_F32)
            r = launch(pair_gemm_kernel<TYPE, 128, 2, TWO>, grid, dim3(256), stage_lds(64, 128, 2, 2), s, dx, dw);
        return r != hipSuccess ? r : join<T>(dx, dw, s);
    }
    if (a.dx && a.M) {
        char *rest = ws;
        Operand w = operand(a.w, a.ldw, TYPE);
        const int64_t rows = a.N;
        if (hipError_t r = pack<T>(TYPE, &w, &rows, 1, a.K, rest, s); r != hipSuccess) return r;
        if (hipError_t r = gemm<TYPE, false, true, TWO>(dz, w, a.M, a.K, a.N, rest, ex, s); r != hipSuccess) return r;
    }
    if (a.dw) {
        char *rest = ws;
        Operand x = operand(a.x, a.ldx, TYPE);
        if (hipError_t r = pack<T>(TYPE, &x, &a.M, 1, a.K, rest, s); r != hipSuccess) return r;
        if (hipError_t r = gemm<TYPE, true, true, TWO>(dz, x, a.N, a.K, a.M, rest, ew, s); r != hipSuccess) return r;
    }
    return hipSuccess;
}

template <int TYPE>
hipError_t linear_grad_t(const LinearGradArgs &a, hipStream_t s) {
    typedef typename Elem<TYPE>::T T;
    if (few_grads(a.M, a.N)) return few_rows_grad<TYPE>(a, s);
    char *ws = (char *)a.ws;
    Operand dz = operand(a.dy, a.lddy, TYPE);
    T *kept = nullptr;
    const int64_t lddz = padded(TYPE, a.N);
    const int passes = dz_passes(TYPE, a.act, a.M, a.N, a.K);
    T *rest = nullptr;
    if ((a.dx || a.dw) && (a.act || !whole_rows(dz, TYPE, a.N))) {
        const int64_t bytes = packed_bytes(TYPE, a.M, a.N);
        kept = (T *)ws;
        if (passes == 2) rest = (T *)(ws + bytes);
        ws += passes * bytes;
        dz = {kept, lddz, true, true, bytes};
    }
    if ((kept || a.db) && a.M) {
        const DzPlan plan = dz_plan(a.M, a.N);
        const int64_t rows = plan.rows, blocks = ceil_div<int64_t>(a.M, rows);
        float *part = !a.db || blocks == 1 ? a.db : (float *)ws;
        const bool vec = aligned16(a.dy, a.lddy * (int64_t)sizeof(T)) && (!a.act || aligned16(a.z, a.ldz * (int64_t)sizeof(T)));
        const auto kernel = plan.narrow ? dz_kernel<T, 1> : dz_kernel<T, 32>;
        const dim3 grid(ceil_div(a.N, plan.narrow ? 8 : 256), blocks);
        if (hipError_t r = launch(kernel, grid, dim3(256), 0, s, (const T *)a.dy, a.lddy, (const T *)a.z, a.ldz, a.act, a.M, a.N, rows, kept,
                                  rest, lddz, part, vec);
            r != hipSuccess)
            return r;
        if (a.db && blocks > 1) {
            if (hipError_t r = launch(column_sum_kernel, dim3(ceil_div(a.N, 16)), dim3(1024), 0, s, part, blocks, a.N, a.db); r != hipSuccess) return r;
            ws += round256(blocks * a.N * 4);
        }
    } else if (a.db) {
        if (hipError_t r = launch(column_sum_kernel, dim3(ceil_div(a.N, 16)), dim3(1024), 0, s, nullptr, 0, a.N, a.db); r != hipSuccess) return r;
    }
    if constexpr (TYPE != BERT_AMD_F32)
        if (passes == 2) return grad_products<TYPE, true>(a, dz, ws, s);
    return grad_products<TYPE, false>(a, dz, ws, s);
}

}  // namespace

int64_t linear_ws_bytes(int type, int64_t M, int N, int K, bool aligned) {
    if (M <= FEW_ROWS) return 0;
    const bool whole = aligned && padded(type, K) == K;
    return (whole ? 0 : packed_bytes(type, M, K) + packed_bytes(type, N, K)) + split_bytes(type, M, N, K);
}

hipError_t launch_linear(const LinearArgs &a, hipStream_t s) {
    switch (a.type) {
        case BERT_AMD_F32: return linear_t<BERT_AMD_F32>(a, s);
        case BERT_AMD_F16: return linear_t<BERT_AMD_F16>(a, s);
        default: return linear_t<BERT_AMD_BF16>(a, s);
    }
}

int64_t linear_grad_ws_bytes(int type, int act, int64_t M, int N, int K, bool aligned) {
    if (few_grads(M, N)) return round256(few_grad_parts(N, K) * M * K * 4);
    const bool whole_n = aligned && padded(type, N) == N, whole_k = aligned && padded(type, K) == K;
    const int passes = dz_passes(type, act, M, N, K);
    const int64_t for_dx = (whole_k ? 0 : packed_bytes(type, N, K)) + split_bytes(type, M, K, N, passes);
    const int64_t for_dw = (whole_k ? 0 : packed_bytes(type, M, K)) + split_bytes(type, N, K, M, passes);
    return (act || !whole_n ? passes * packed_bytes(type, M, N) : 0) + round256(ceil_div<int64_t>(M, dz_plan(M, N).rows) * N * 4) +
           (gradients_in_pair(type, M, N, K, passes) ? for_dx + for_dw : std::max(for_dx, for_dw));
}

hipError_t launch_linear_grad(const LinearGradArgs &a, hipStream_t s) {
    switch (a.type) {
        case BERT_AMD_F32: return linear_grad_t<BERT_AMD_F32>(a, s);
        case BERT_AMD_F16: return linear_grad_t<BERT_AMD_F16>(a, s);
        default: return linear_grad_t<BERT_AMD_BF16>(a, s);
    }
}

// whether rows of type `type`, `ld` elements apart, are whole aligned chunks as far as address and stride go
bool linear_aligned(const void *p, int64_t ld, int type) { return aligned16(p, ld * elem_size(type)) && ld < (1 << 21); }

}  // namespace bertamd

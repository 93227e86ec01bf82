// ops_rows.hip — token rows out of a table, and the table's gradient.
//
//   lookup:      out[i] = scale * table[ids[i]], a zero row where ids[i] names none
//   lookup_grad: dtable[v] (+)= scale * sum of dout[i] over the i with ids[i] = v
#include "ops_common.h"

#include <algorithm>

namespace bertamd {

namespace {

template <int TYPE> struct RowType { static constexpr bool BLOCKS = false; };
template <> struct RowType<BERT_AMD_Q4_0> { static constexpr bool BLOCKS = true; static constexpr int SIZE = 18, HEAD = 2; };
template <> struct RowType<BERT_AMD_Q4_1> { static constexpr bool BLOCKS = true; static constexpr int SIZE = 20, HEAD = 4; };

// element e of a row: ggml's get_rows values (d (q - 8), d q + m; both products exact in f32)
template <int TYPE>
__device__ __forceinline__ float row_value(const char *row, int e) {
    if constexpr (RowType<TYPE>::BLOCKS) {
        const uint8_t *b = (const uint8_t *)row + (int64_t)(e >> 5) * RowType<TYPE>::SIZE;
        const float d = (float)*(const _Float16 *)b;
        const int j = e & 31, byte = b[RowType<TYPE>::HEAD + (j & 15)], q = j < 16 ? byte & 15 : byte >> 4;
        if constexpr (TYPE == BERT_AMD_Q4_0)
            return d * (float)(q - 8);
        else
            return d * (float)q + (float)*(const _Float16 *)(b + 2);
    } else {
        return (float)((const typename Elem<TYPE>::T *)row)[e];
    }
}

template <int TYPE, int OUT>
__global__ __launch_bounds__(256) void lookup_kernel(LookupArgs a) {
    const int64_t total = a.n * a.E;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / a.E;
        const int e = (int)(i - row * a.E), id = a.ids[row];
        const float v = id >= 0 && id < a.V ? a.scale * row_value<TYPE>((const char *)a.table + id * a.ld_bytes, e) : 0.f;
        ((typename Elem<OUT>::T *)a.out)[row * a.ldo + e] = (typename Elem<OUT>::T)v;
    }
}

template <int TYPE>
hipError_t lookup_t(const LookupArgs &a, hipStream_t s) {
    const dim3 grid(std::min<int64_t>(1 << 20, ceil_div<int64_t>(a.n * a.E, 256)));
    switch (a.out_type) {
        case BERT_AMD_F32: hipLaunchKernelGGL((lookup_kernel<TYPE, BERT_AMD_F32>), grid, dim3(256), 0, s, a); break;
        case BERT_AMD_F16: hipLaunchKernelGGL((lookup_kernel<TYPE, BERT_AMD_F16>), grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((lookup_kernel<TYPE, BERT_AMD_BF16>), grid, dim3(256), 0, s, a); break;
    }
    return hipGetLastError();
}

// ---- the places sorted by token --------------------------------------------
//
// A stable radix sort of (token, place) by digits of up to 9 bits: per digit a
// histogram of each tile of 2048 places, each digit value's exclusive scan
// over the tiles, and a scatter in which every place's rank counts the places
// before it in its tile with the same digit.  No atomic's order enters the
// result, so the sums below have one order.  Places without a gradient (ids
// outside the table, the padding token) get the key V and sort last.
constexpr int TILE = 2048, BINS = 512;

__device__ __forceinline__ int sort_key(int id, int V, int pad) { return id >= 0 && id < V && id != pad ? id : V; }

struct SortPass {
    const int32_t *ids;                // first pass: the caller's ids, else null
    const int32_t *key_in, *place_in;
    int32_t *key_out, *place_out;
    int32_t *hist, *total;             // [BINS][tiles], [BINS]
    int n, V, pad, tiles, shift, bits;
};

__global__ __launch_bounds__(256) void sort_hist_kernel(SortPass p) {
    __shared__ int h[BINS];
    for (int i = threadIdx.x; i < BINS; i += 256) h[i] = 0;
    __syncthreads();
    const int mask = (1 << p.bits) - 1, base = blockIdx.x * TILE;
    for (int j = threadIdx.x; j < TILE; j += 256)
        if (base + j < p.n) {
            const int k = p.ids ? sort_key(p.ids[base + j], p.V, p.pad) : p.key_in[base + j];
            atomicAdd(&h[(k >> p.shift) & mask], 1);
        }
    __syncthreads();
    for (int i = threadIdx.x; i <= mask; i += 256) p.hist[(int64_t)i * p.tiles + blockIdx.x] = h[i];
}

// inclusive sum over the 256 threads of a workgroup; `sums` has one place per wave
__device__ __forceinline__ int block_scan(int v, int *sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; w++) v += sums[w];
    __syncthreads();
    return v;
}

__global__ __launch_bounds__(256) void sort_scan_kernel(SortPass p) {
    __shared__ int sums[4], carry;
    int32_t *h = p.hist + (int64_t)blockIdx.x * p.tiles;
    if (threadIdx.x == 0) carry = 0;
    __syncthreads();
    for (int base = 0; base < p.tiles; base += 256) {
        const int i = base + threadIdx.x, own = i < p.tiles ? h[i] : 0;
        const int upto = block_scan(own, sums) + carry;
        __syncthreads();
        if (i < p.tiles) h[i] = upto - own;
        if (threadIdx.x == 255) carry = upto;
        __syncthreads();
    }
    if (threadIdx.x == 0) p.total[blockIdx.x] = carry;
}

__global__ __launch_bounds__(256) void sort_scatter_kernel(SortPass p) {
    __shared__ int first[BINS];       // where this tile's places of each digit value start
    __shared__ int seen[4][BINS];     // per wave: places of each digit value so far
    __shared__ int sums[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mask = (1 << p.bits) - 1, bins = 1 << p.bits;
    for (int i = threadIdx.x; i < 4 * BINS; i += 256) (&seen[0][0])[i] = 0;
    {   // totals of the digit values before each: thread t owns values 2t and 2t + 1
        const int t = 2 * threadIdx.x, a = t < bins ? p.total[t] : 0, b = t + 1 < bins ? p.total[t + 1] : 0;
        const int upto = block_scan(a + b, sums);
        if (t < bins) first[t] = upto - a - b + p.hist[(int64_t)t * p.tiles + blockIdx.x];
        if (t + 1 < bins) first[t + 1] = upto - b + p.hist[(int64_t)(t + 1) * p.tiles + blockIdx.x];
    }
    __syncthreads();
    const int base = blockIdx.x * TILE + wave * (TILE / 4);
    int key[TILE / 256], place[TILE / 256], rank[TILE / 256];
#pragma unroll
    for (int j = 0; j < TILE / 256; j++) {
        const int i = base + 64 * j + lane;
        const bool in = i < p.n;
        key[j] = !in ? 0 : p.ids ? sort_key(p.ids[i], p.V, p.pad) : p.key_in[i];
        place[j] = !in ? 0 : p.ids ? i : p.place_in[i];
        const int d = (key[j] >> p.shift) & mask;
        uint64_t same = __ballot(in);
        for (int b = 0; b < p.bits; b++) {
            const uint64_t set = __ballot((d >> b) & 1);
            same &= (d >> b) & 1 ? set : ~set;
        }
        const int before = __popcll(same & ((1ull << lane) - 1)), so_far = seen[wave][d];
        rank[j] = so_far + before;
        __builtin_amdgcn_wave_barrier();  // the wave's reads stay before the count's update by one lane per value
        if (in && before == 0) seen[wave][d] = so_far + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TILE / 256; j++) {
        const int i = base + 64 * j + lane;
        if (i >= p.n) continue;
        const int d = (key[j] >> p.shift) & mask;
        int at = first[d] + rank[j];
        for (int w = 0; w < wave; w++) at += seen[w][d];
        p.key_out[at] = key[j];
        p.place_out[at] = place[j];
    }
}

__global__ __launch_bounds__(256) void fill_kernel(int32_t *p, int64_t n, int32_t v) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = v;
}

__global__ __launch_bounds__(256) void starts_kernel(const int32_t *key, int n, int V, int32_t *start) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n && key[i] < V && (i == 0 || key[i - 1] != key[i])) start[key[i]] = i;
}

template <int TYPE>
__global__ __launch_bounds__(256) void lookup_grad_kernel(LookupGradArgs a, const int32_t *key, const int32_t *place, const int32_t *start) {
    for (int v = blockIdx.x; v < a.V; v += gridDim.x) {
        const int first = start[v];
        if (first < 0 && a.accumulate) continue;
        for (int e = threadIdx.x; e < a.E; e += 256) {
            float sum = 0.f;
            if (first >= 0)
                for (int i = first; i < a.n && key[i] == v; i++)
                    sum += (float)((const typename Elem<TYPE>::T *)a.dout)[place[i] * a.ldd + e];
            float *o = a.dtable + (int64_t)v * a.ldt + e;
            *o = a.accumulate ? *o + a.scale * sum : a.scale * sum;
        }
    }
}

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

hipError_t launch_lookup(const LookupArgs &a, hipStream_t s) {
    switch (a.type) {
        case BERT_AMD_F32: return lookup_t<BERT_AMD_F32>(a, s);
        case BERT_AMD_F16: return lookup_t<BERT_AMD_F16>(a, s);
        case BERT_AMD_BF16: return lookup_t<BERT_AMD_BF16>(a, s);
        case BERT_AMD_Q4_0: return lookup_t<BERT_AMD_Q4_0>(a, s);
        default: return lookup_t<BERT_AMD_Q4_1>(a, s);
    }
}

int64_t lookup_grad_ws_bytes(int64_t n, int V, int) {
    const int64_t tiles = ceil_div<int64_t>(n, TILE);
    return 4 * round256(n * 4) + round256(BINS * tiles * 4) + round256(BINS * 4) + round256((int64_t)V * 4);
}

hipError_t launch_lookup_grad(const LookupGradArgs &a, hipStream_t s) {
    char *ws = (char *)a.ws;
    const auto take = [&](int64_t ints) {
        int32_t *p = (int32_t *)ws;
        ws += round256(ints * 4);
        return p;
    };
    const int tiles = (int)ceil_div<int64_t>(a.n, TILE);
    int32_t *key[2], *place[2];
    for (int i = 0; i < 2; i++) key[i] = take(a.n), place[i] = take(a.n);
    SortPass p = {};
    p.hist = take((int64_t)BINS * tiles);
    p.total = take(BINS);
    int32_t *start = take(a.V);
    hipLaunchKernelGGL(fill_kernel, dim3(std::min<int64_t>(1024, ceil_div(a.V, 256))), dim3(256), 0, s, start, (int64_t)a.V, -1);
    int at = 0;
    if (a.n) {
        int key_bits = 1;
        while ((int64_t)a.V >> key_bits) key_bits++;
        const int passes = ceil_div(key_bits, 9);
        p.n = (int)a.n, p.V = a.V, p.pad = a.pad_id, p.tiles = tiles;
        p.bits = ceil_div(key_bits, passes);
        for (int i = 0; i < passes; i++) {
            p.ids = i ? nullptr : a.ids;
            p.key_in = key[at], p.place_in = place[at];
            p.key_out = key[at ^ 1], p.place_out = place[at ^ 1];
            p.shift = i * p.bits;
            hipLaunchKernelGGL(sort_hist_kernel, dim3(tiles), dim3(256), 0, s, p);
            hipLaunchKernelGGL(sort_scan_kernel, dim3(1 << p.bits), dim3(256), 0, s, p);
            hipLaunchKernelGGL(sort_scatter_kernel, dim3(tiles), dim3(256), 0, s, p);
            at ^= 1;
        }
        hipLaunchKernelGGL(starts_kernel, dim3(ceil_div<int64_t>(a.n, 256)), dim3(256), 0, s, key[at], (int)a.n, a.V, start);
    }
    const int rows = std::min(a.V, 1 << 22);
    switch (a.type) {
        case BERT_AMD_F32: hipLaunchKernelGGL((lookup_grad_kernel<BERT_AMD_F32>), dim3(rows), dim3(256), 0, s, a, key[at], place[at], start); break;
        case BERT_AMD_F16: hipLaunchKernelGGL((lookup_grad_kernel<BERT_AMD_F16>), dim3(rows), dim3(256), 0, s, a, key[at], place[at], start); break;
        default: hipLaunchKernelGGL((lookup_grad_kernel<BERT_AMD_BF16>), dim3(rows), dim3(256), 0, s, a, key[at], place[at], start); break;
    }
    return hipGetLastError();
}

}  // namespace bertamd

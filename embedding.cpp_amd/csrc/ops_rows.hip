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

// elements 8 c .. 8 c + 7 of a row whose float elements are 16-byte aligned (Q4 blocks: 2-byte)
template <int TYPE>
__device__ __forceinline__ void row_values8(const char *row, int c, float *v) {
    if constexpr (RowType<TYPE>::BLOCKS) {
        const char *b = row + (int64_t)(c >> 2) * RowType<TYPE>::SIZE;
        const float d = (float)*(const _Float16 *)b;
        const uint16_t *q = (const uint16_t *)(b + RowType<TYPE>::HEAD) + 4 * (c & 1);
        const int shift = (c & 2) << 1;  // the block's second half is in the high nibbles
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const int two = q[i / 2] >> shift, lo = two & 15, hi = (two >> 8) & 15;
            if constexpr (TYPE == BERT_AMD_Q4_0) {
                v[i] = d * (float)(lo - 8), v[i + 1] = d * (float)(hi - 8);
            } else {
                const float m = (float)*(const _Float16 *)(b + 2);
                v[i] = d * (float)lo + m, v[i + 1] = d * (float)hi + m;
            }
        }
    } else {
        typedef typename Elem<TYPE>::T T;
        constexpr int CH = Elem<TYPE>::CH;
#pragma unroll
        for (int i = 0; i < 8; i += CH) {
            const Chunk<T, CH> o = __builtin_bit_cast(Chunk<T, CH>, *(const u32x4 *)(row + (8 * c + i) * sizeof(T)));
#pragma unroll
            for (int j = 0; j < CH; j++) v[i + j] = (float)o.v[j];
        }
    }
}

// One thread an element: any width, stride and alignment.
template <int TYPE, int OUT>
__global__ __launch_bounds__(256) void lookup_any_kernel(LookupArgs a) {
    const int64_t total = a.n * a.E;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / a.E;
        const int e = (int)(i - row * a.E), id = a.ids[row];
        const float v = id >= 0 && id < a.V ? a.scale * row_value<TYPE>((const char *)a.table + id * a.ld_bytes, e) : 0.f;
        ((typename Elem<OUT>::T *)a.out)[row * a.ldo + e] = (typename Elem<OUT>::T)v;
    }
}

// Eight elements a thread, `lanes` (8 .. 64) neighbours side by side on a row,
// chosen so that they come out even: bound by memory, and enough rows are on
// their way at once with no more than that (131072 x 768 f16 rows of a 250002
// row table: 62 us, 403 MB read and written at 6.4 TB/s with the rows that
// caches repeat; one element a thread took 270).
template <int TYPE, int OUT>
__global__ __launch_bounds__(256) void lookup_kernel(LookupArgs a, int lanes_log2) {
    const int lanes = 1 << lanes_log2, per = 256 >> lanes_log2, chunks = a.E / 8;
    const int64_t row = (int64_t)blockIdx.x * per + (threadIdx.x >> lanes_log2);
    if (row >= a.n) return;
    const int id = a.ids[row];
    const bool there = id >= 0 && id < a.V;
    const char *from = (const char *)a.table + (there ? id : 0) * a.ld_bytes;
    typename Elem<OUT>::T *to = (typename Elem<OUT>::T *)a.out + row * a.ldo;
#pragma unroll 4
    for (int c = threadIdx.x & (lanes - 1); c < chunks; c += lanes) {
        float v[8] = {};
        if (there) row_values8<TYPE>(from, c, v);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= there ? a.scale : 0.f;
        if (!there)
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.f;
        put8(to + 8 * c, v);
    }
}

// lanes side by side on a row of `chunks`: the most, of those that leave the fewest without work
int row_lanes_log2(int chunks) {
    int best = 3;
    for (int l = 3; l <= 6; l++)
        if (ceil_div(chunks, 1 << l) << l <= ceil_div(chunks, 1 << best) << best) best = l;
    return best;
}

template <int TYPE, int OUT>
hipError_t lookup_tt(const LookupArgs &a, hipStream_t s) {
    constexpr bool BLOCKS = RowType<TYPE>::BLOCKS;
    const bool whole = a.E % 8 == 0 && (BLOCKS || aligned16(a.table, a.ld_bytes)) && aligned16(a.out, a.ldo * (int64_t)sizeof(typename Elem<OUT>::T));
    const int l = row_lanes_log2(a.E / 8);
    const int64_t groups = ceil_div<int64_t>(a.n, 256 >> l);
    if (whole && groups <= 1 << 23) return launch(lookup_kernel<TYPE, OUT>, dim3(groups), dim3(256), 0, s, a, l);
    return launch(lookup_any_kernel<TYPE, OUT>, dim3(std::min<int64_t>(1 << 20, ceil_div<int64_t>(a.n * a.E, 256))), dim3(256), 0, s, a);
}

template <int TYPE>
hipError_t lookup_t(const LookupArgs &a, hipStream_t s) {
    switch (a.out_type) {
        case BERT_AMD_F32: return lookup_tt<TYPE, BERT_AMD_F32>(a, s);
        case BERT_AMD_F16: return lookup_tt<TYPE, BERT_AMD_F16>(a, s);
        default: return lookup_tt<TYPE, BERT_AMD_BF16>(a, s);
    }
}

// ---- the places sorted by token --------------------------------------------
//
// A stable radix sort of (token, place) by digits of up to 9 bits: per digit a
// histogram of each tile of 1024 places, each digit value's exclusive scan
// over the tiles, and a scatter in which every place's rank counts the places
// before it in its tile with the same digit.  No atomic's order enters the
// result, so the sums below have one order.  Places without a gradient (ids
// outside the table, the padding token) get the key V and sort last.
//
// These launches wait for memory more than they move, so other workgroups of
// theirs write the zeros of the rows that have no place (most of a table's
// gradient): the first one clears the rows' marks, the second one's others set
// them from the ids, the following ones' write.  131072 places by 18 bits: 5 +
// 5 + 9 us a digit without the zeros.
constexpr int TILE = 1024, BINS = 512;

__device__ __forceinline__ int sort_key(int id, int V, int pad) { return id >= 0 && id < V && id != pad ? id : V; }

// Rows first .. end - 1 of the gradient that no place belongs to, as zeros, by
// `groups` workgroups of which this is number `g`; `used` marks the others.
struct ZeroPart {
    float *dtable = nullptr;
    int64_t ldt = 0;
    int E = 0, first = 0, end = 0;
    const uint8_t *used = nullptr;
    bool four = false;  // rows are whole aligned float4s
};
constexpr int ZERO_ROWS = 16;

template <int ROWS>
__device__ __forceinline__ void zero_rows(const ZeroPart &z, int first, const uint8_t *used /* of row `first` on */) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    static_assert(ROWS <= 64, "a lane looks at one row's mark");
    const bool mine = lane < ROWS && first + lane < z.end;
    const uint64_t unused = __ballot(mine && !used[mine ? lane : 0]);
    for (int v = first + wave; v < min(z.end, first + ROWS); v += blockDim.x >> 6) {
        if (!(unused >> (v - first) & 1)) continue;
        float *row = z.dtable + (int64_t)v * z.ldt;
        if (z.four)
            for (int e = 4 * lane; e < z.E; e += 256) *(f32x4 *)(row + e) = f32x4{0.f, 0.f, 0.f, 0.f};
        else
            for (int e = lane; e < z.E; e += 64) row[e] = 0.f;
    }
}
__device__ __forceinline__ void zero_part(const ZeroPart &z, int g, int groups) {
    for (int64_t v = z.first + (int64_t)g * ZERO_ROWS; v < z.end; v += (int64_t)groups * ZERO_ROWS) zero_rows<ZERO_ROWS>(z, (int)v, z.used + v);
}
inline int zero_groups(const ZeroPart &z, int rows = ZERO_ROWS) { return std::min(1 << 20, ceil_div(std::max(0, z.end - z.first), rows)); }

struct SortPass {
    const int32_t *ids;                // first pass: the caller's ids, else null
    const int32_t *key_in, *place_in;
    int32_t *key_out, *place_out;
    int32_t *hist, *total;             // [BINS][tiles], [BINS]
    uint8_t *used;                     // marks of the rows that have a place: cleared and set in the first pass
    ZeroPart zero;                     // what this launch's other workgroups write
    int n, V, pad, tiles, shift, bits;
};

__global__ __launch_bounds__(256) void sort_hist_kernel(SortPass p) {
    __shared__ int h[BINS];
    if ((int)blockIdx.x >= p.tiles) return zero_part(p.zero, blockIdx.x - p.tiles, gridDim.x - p.tiles);
    if (p.ids)
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < ceil_div(p.V, 16); i += (int64_t)gridDim.x * 256)
            ((u32x4 *)p.used)[i] = u32x4{0, 0, 0, 0};
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
    const int bins = 1 << p.bits;
    if ((int)blockIdx.x >= bins) {
        if (!p.ids) return zero_part(p.zero, blockIdx.x - bins, gridDim.x - bins);
        for (int64_t i = (int64_t)(blockIdx.x - bins) * 256 + threadIdx.x; i < p.n; i += (int64_t)(gridDim.x - bins) * 256) {
            const int k = sort_key(p.ids[i], p.V, p.pad);
            if (k < p.V) p.used[k] = 1;
        }
        return;
    }
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
    if ((int)blockIdx.x >= p.tiles) return zero_part(p.zero, blockIdx.x - p.tiles, gridDim.x - p.tiles);
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
        wave_sync();  // the wave's reads stay before the count's update by one lane per value
        if (in && before == 0) seen[wave][d] = so_far + __popcll(same);
        wave_sync();
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

// ---- the sums ---------------------------------------------------------------
//
// A workgroup sums SUM_TILE sorted places, a thread COLS columns of them in
// order, eight rows' loads on their way at a time, and writes the row of each
// token whose places end within the tile.  A token whose places go on past a
// tile's end leaves its sums, one row for each tile it has places in, to
// join_kernel, which adds them in order: a frequent token's long sum is spread
// over many workgroups.  131072 x 768 bf16 places of 67705 tokens: 115 us, 409
// MB read and written at 3.6 TB/s, and 10 us of joins (a workgroup a token
// instead took 1.6 ms: a token 1200 times in the batch is one chain of loads).
constexpr int SUM_TILE = 64, AHEAD = 8;

// a finished sum into its row of the table
template <int COLS>
__device__ __forceinline__ void store_row(const LookupGradArgs &a, int v, int e, const float *sum) {
    float *p = a.dtable + (int64_t)v * a.ldt + e, o[COLS];
    if (a.accumulate) get_n<float, COLS>(p, o);
#pragma unroll
    for (int i = 0; i < COLS; i++) o[i] = a.accumulate ? o[i] + a.scale * sum[i] : a.scale * sum[i];
    put_n<float, COLS>(p, o);
}
struct SumArgs {
    const int32_t *key, *place;
    float *part;  // [tiles][2][E]: of the token that goes on from the tile before; of the one that goes on past the end
    int tiles;
};

template <int TYPE, int COLS>
__global__ __launch_bounds__(256) void sum_kernel(LookupGradArgs a, SumArgs s) {
    typedef typename Elem<TYPE>::T T;
    static_assert(SUM_TILE == 64, "a lane holds one place");
    const int lane = threadIdx.x & 63, n = (int)a.n, i = blockIdx.x * SUM_TILE + lane;
    const int key = i < n ? s.key[i] : a.V, next = i + 1 < n ? s.key[i + 1] : a.V, place = i < n ? s.place[i] : 0;
    const int before = blockIdx.x ? s.key[blockIdx.x * SUM_TILE - 1] : -1;
    const int count = __popcll(__ballot(key < a.V));  // the places without a gradient are the last ones
    const uint64_t ends = __ballot(key != next) | 1ull << (SUM_TILE - 1);
    if (!count) return;
    // Every lane stays on: a lane past the row's end holds a place that the others
    // read, so it sums the row's last columns again and stores nothing.
    const int own = (blockIdx.y * blockDim.x + threadIdx.x) * COLS, e = min(own, a.E - COLS);
    const bool there = own < a.E;
    const T *from = (const T *)a.dout + e;
    float *part = s.part + (int64_t)blockIdx.x * 2 * a.E + e;
    float sum[COLS] = {};
    bool from_before = before == __builtin_amdgcn_readlane(key, 0);
    float now[AHEAD][COLS], then[AHEAD][COLS];
    const auto load = [&](float (&v)[AHEAD][COLS], int at) {  // past the last place: its row again, not used
#pragma unroll
        for (int j = 0; j < AHEAD; j++) get_n<T, COLS>(from + __builtin_amdgcn_readlane(place, min(at + j, count - 1)) * a.ldd, v[j]);
    };
    load(now, 0);
    for (int at = 0; at < count; at += AHEAD) {
        if (at + AHEAD < count) load(then, at + AHEAD);
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            if (at + j >= count) break;
#pragma unroll
            for (int c = 0; c < COLS; c++) sum[c] += now[j][c];
            if (ends >> (at + j) & 1) {
                const int k = __builtin_amdgcn_readlane(key, at + j), after = __builtin_amdgcn_readlane(next, at + j);
                if (there) {
                    if (from_before) put_n<float, COLS>(part, sum);
                    else if (after == k) put_n<float, COLS>(part + a.E, sum);
                    else store_row<COLS>(a, k, e, sum);
                }
                from_before = false;
#pragma unroll
                for (int c = 0; c < COLS; c++) sum[c] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
#pragma unroll
            for (int c = 0; c < COLS; c++) now[j][c] = then[j][c];
    }
}

// The token that starts in this tile and goes on past its end: its sums of this
// tile and the following ones, 64 columns' threads in four groups that take a
// quarter of the tiles each.
template <int COLS>
__global__ __launch_bounds__(256) void join_kernel(LookupGradArgs a, SumArgs s) {
    const int t = blockIdx.x, last = (t + 1) * SUM_TILE - 1, n = (int)a.n;
    if (last + 1 >= n) return;
    const int k = s.key[last];
    if (k >= a.V || s.key[last + 1] != k) return;
    if (s.key[t * SUM_TILE] == k && t > 0 && s.key[t * SUM_TILE - 1] == k) return;  // it started before this tile
    int lo = t + 1, hi = s.tiles;  // the tiles after this one that begin with k end at lo
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s.key[mid * SUM_TILE] == k) lo = mid + 1;
        else hi = mid;
    }
    __shared__ float sums[4][64][COLS + 1];
    const int c = threadIdx.x & 63, g = threadIdx.x >> 6, e = (blockIdx.y * 64 + c) * COLS;
    const int rows = lo - t - 1, per = ceil_div(rows, 4);
    float sum[COLS] = {};
    if (e < a.E) {
        const float *head = s.part + (int64_t)(t + 1) * 2 * a.E + e;
#pragma unroll 8
        for (int i = g * per; i < min(rows, (g + 1) * per); i++) {
            float v[COLS];
            get_n<float, COLS>(head + (int64_t)i * 2 * a.E, v);
#pragma unroll
            for (int j = 0; j < COLS; j++) sum[j] += v[j];
        }
    }
#pragma unroll
    for (int j = 0; j < COLS; j++) sums[g][c][j] = sum[j];
    __syncthreads();
    if (g || e >= a.E) return;
    float v[COLS];
    get_n<float, COLS>(s.part + ((int64_t)t * 2 + 1) * a.E + e, v);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < COLS; j++) v[j] += sums[i][c][j];
    store_row<COLS>(a, k, e, v);
}

// Few places (at most FEW): no sort.  A workgroup for each place looks through
// all ids; its waves find the token's places among at most 512 ids each, sum
// those in order, and the waves' sums are added in order.  A token's r-th place
// takes the columns' slices r, r + its places, ..: a rare token's first place
// does it all, a frequent one's sums are spread over as many workgroups as there
// are slices, so that none walks along a wide row place by place.  Again the other
// workgroups write the zeros, and find out from the ids which rows are in use.
// f32 of a 30522 row table, us, here and sorted: 2048 x 384 places of tokens as
// text has them 14.1 and 48, all of one token 58 and 38; 4096 x 384 25 and 49, of
// one token 61 and 40; 4096 x 1023 (a column a lane) 60 and 59, of one token 93
// and 52.  The looking grows with the places' square.  Eight waves for 2048 places
// too take 15.7 and 33, four for 4096 x 384 22 and 111; the first place alone at work
// took 307 us for 4096 x 768 of one token and 2302 for 4096 x 1023.
constexpr int FEW = 4096, FEW_EACH = 512;

template <int TYPE, int COLS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_kernel(LookupGradArgs a, ZeroPart z) {
    typedef typename Elem<TYPE>::T T;
    constexpr int ZEROS = 4 * WAVES;
    const int n = (int)a.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = blockIdx.x;
    if (at >= n) {
        __shared__ uint8_t used[ZEROS];
        static_assert(ZEROS <= 64 * WAVES, "one thread clears one row's mark");
        for (int64_t b = at - n; b * ZEROS < a.V; b += gridDim.x - n) {
            const int first = (int)b * ZEROS;
            __syncthreads();
            if (threadIdx.x < ZEROS) used[threadIdx.x] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += 64 * WAVES) {
                const int id = a.ids[i];
                if (id >= first && id < first + ZEROS && id != a.pad_id) used[id - first] = 1;
            }
            __syncthreads();
            zero_rows<ZEROS>(z, first, used);
        }
        return;
    }
    const int k = sort_key(a.ids[at], a.V, a.pad_id);
    if (k == a.V) return;
    __shared__ uint16_t list[WAVES][FEW_EACH];
    __shared__ int counts[WAVES], before[WAVES];
    __shared__ float sums[WAVES - 1][64][COLS + 1];
    const int share = ceil_div(n, 64 * WAVES) * 64, from = wave * share;
    int count = 0, earlier = 0;
    for (int i = from; i < min(n, from + share); i += 64) {
        const bool same = i + lane < n && a.ids[i + lane] == k;
        const uint64_t mask = __ballot(same);
        if (same) list[wave][count + __popcll(mask & ((1ull << lane) - 1))] = (uint16_t)(i + lane);
        earlier += __popcll(__ballot(same && i + lane < at));
        count += __popcll(mask);
    }
    counts[wave] = count, before[wave] = earlier;
    __syncthreads();
    int rank = 0, places = 0;  // of this place among its token's
#pragma unroll
    for (int w = 0; w < WAVES; w++) rank += before[w], places += counts[w];
    for (int e0 = rank * 64 * COLS; e0 < a.E; e0 += places * 64 * COLS) {
        const int e = e0 + lane * COLS;
        float sum[COLS] = {};
        if (e < a.E)
            for (int i = 0; i < count; i += AHEAD) {
                float v[AHEAD][COLS] = {};
#pragma unroll
                for (int j = 0; j < AHEAD; j++)
                    if (i + j < count) get_n<T, COLS>((const T *)a.dout + list[wave][i + j] * a.ldd + e, v[j]);
#pragma unroll
                for (int j = 0; j < AHEAD; j++)
#pragma unroll
                    for (int c = 0; c < COLS; c++) sum[c] += v[j][c];
            }
        if (wave)
#pragma unroll
            for (int c = 0; c < COLS; c++) sums[wave - 1][lane][c] = sum[c];
        __syncthreads();
        if (!wave && e < a.E) {
#pragma unroll
            for (int w = 0; w < WAVES - 1; w++)
#pragma unroll
                for (int c = 0; c < COLS; c++) sum[c] += sums[w][lane][c];
            store_row<COLS>(a, k, e, sum);
        }
        __syncthreads();
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

int64_t lookup_grad_ws_bytes(int64_t n, int V, int E) {
    if (n <= FEW) return 0;
    return 4 * round256(n * 4) + round256(BINS * ceil_div<int64_t>(n, TILE) * 4) + round256(BINS * 4) + round256((int64_t)V + 16) +
           round256(ceil_div<int64_t>(n, SUM_TILE) * 2 * E * 4);
}

namespace {

template <int TYPE, int COLS>
hipError_t sum_t(const LookupGradArgs &a, const SumArgs &p, hipStream_t s) {
    const int threads = std::min(256, ceil_div(ceil_div(a.E, COLS), 64) * 64);
    const int across = ceil_div(ceil_div(a.E, COLS), threads);
    if (hipError_t e = launch(sum_kernel<TYPE, COLS>, dim3(p.tiles, across), dim3(threads), 0, s, a, p); e != hipSuccess) return e;
    return launch(join_kernel<COLS>, dim3(p.tiles, ceil_div(a.E, 64 * COLS)), dim3(256), 0, s, a, p);
}
template <int TYPE, int COLS, int WAVES>
hipError_t few_w(const LookupGradArgs &a, const ZeroPart &z, hipStream_t s) {
    const int groups = (int)a.n + zero_groups(z, 4 * WAVES);
    return groups ? launch(few_kernel<TYPE, COLS, WAVES>, dim3(groups), dim3(64 * WAVES), 0, s, a, z) : hipSuccess;
}
template <int TYPE, int COLS>
hipError_t few_t(const LookupGradArgs &a, const ZeroPart &z, hipStream_t s) {
    static_assert(8 * FEW_EACH == FEW, "eight waves take all places");
    return a.n <= 4 * FEW_EACH ? few_w<TYPE, COLS, 4>(a, z, s) : few_w<TYPE, COLS, 8>(a, z, s);
}
// four columns a thread where rows and places allow it
bool four_columns(const LookupGradArgs &a) {
    const int64_t e = elem_size(a.type);
    return a.E % 4 == 0 && a.ldd % 4 == 0 && ((uintptr_t)a.dout & (4 * e - 1)) == 0 && aligned16(a.dtable, a.ldt * 4);
}

}  // namespace

hipError_t launch_lookup_grad(const LookupGradArgs &a, hipStream_t s) {
    const bool four = four_columns(a);
    ZeroPart zero;
    zero.dtable = a.dtable, zero.ldt = a.ldt, zero.E = a.E, zero.end = a.accumulate ? 0 : a.V;
    zero.four = a.E % 4 == 0 && aligned16(a.dtable, a.ldt * 4);
    if (a.n <= FEW) {
        switch (a.type) {
            case BERT_AMD_F32: return four ? few_t<BERT_AMD_F32, 4>(a, zero, s) : few_t<BERT_AMD_F32, 1>(a, zero, s);
            case BERT_AMD_F16: return four ? few_t<BERT_AMD_F16, 4>(a, zero, s) : few_t<BERT_AMD_F16, 1>(a, zero, s);
            default: return four ? few_t<BERT_AMD_BF16, 4>(a, zero, s) : few_t<BERT_AMD_BF16, 1>(a, zero, s);
        }
    }
    char *ws = (char *)a.ws;
    const auto take = [&](int64_t bytes) {
        char *p = ws;
        ws += round256(bytes);
        return p;
    };
    const int tiles = (int)ceil_div<int64_t>(a.n, TILE);
    int32_t *key[2], *place[2];
    for (int i = 0; i < 2; i++) key[i] = (int32_t *)take(a.n * 4), place[i] = (int32_t *)take(a.n * 4);
    SortPass p = {};
    p.hist = (int32_t *)take((int64_t)BINS * tiles * 4);
    p.total = (int32_t *)take(BINS * 4);
    p.used = (uint8_t *)take((int64_t)a.V + 16);
    SumArgs q = {};
    q.part = (float *)take(ceil_div<int64_t>(a.n, SUM_TILE) * 2 * a.E * 4);
    q.tiles = (int)ceil_div<int64_t>(a.n, SUM_TILE);
    int key_bits = 1;
    while ((int64_t)a.V >> key_bits) key_bits++;
    const int passes = ceil_div(key_bits, 9);
    p.n = (int)a.n, p.V = a.V, p.pad = a.pad_id, p.tiles = tiles;
    p.bits = ceil_div(key_bits, passes);
    // The zeros' rows over the launches after the marks, in proportion to what
    // each can take beside its own work: scatter 4, histogram 1, scan 1.
    zero.used = p.used;
    const int rows = zero.end, shares = 6 * passes - 2;
    int given = 0;
    const auto share = [&](int n) {
        p.zero = zero;
        p.zero.first = (int)((int64_t)rows * given / shares);
        p.zero.end = (int)((int64_t)rows * (given + n) / shares);
        given += n;
        return zero_groups(p.zero);
    };
    int at = 0;
    for (int i = 0; i < passes; i++) {
        p.ids = i ? nullptr : a.ids;
        p.key_in = key[at], p.place_in = place[at];
        p.key_out = key[at ^ 1], p.place_out = place[at ^ 1];
        p.shift = i * p.bits;
        const int hist = i ? share(1) : 0;
        if (hipError_t e = launch(sort_hist_kernel, dim3(tiles + hist), dim3(256), 0, s, p); e != hipSuccess) return e;
        const int scan = i ? share(1) : std::min(1024, tiles * 4);  // first pass: the marks
        if (hipError_t e = launch(sort_scan_kernel, dim3((1 << p.bits) + scan), dim3(256), 0, s, p); e != hipSuccess) return e;
        const int scatter = share(4);
        if (hipError_t e = launch(sort_scatter_kernel, dim3(tiles + scatter), dim3(256), 0, s, p); e != hipSuccess) return e;
        at ^= 1;
    }
    q.key = key[at], q.place = place[at];
    switch (a.type) {
        case BERT_AMD_F32: return four ? sum_t<BERT_AMD_F32, 4>(a, q, s) : sum_t<BERT_AMD_F32, 1>(a, q, s);
        case BERT_AMD_F16: return four ? sum_t<BERT_AMD_F16, 4>(a, q, s) : sum_t<BERT_AMD_F16, 1>(a, q, s);
        default: return four ? sum_t<BERT_AMD_BF16, 4>(a, q, s) : sum_t<BERT_AMD_BF16, 1>(a, q, s);
    }
}

}  // namespace bertamd

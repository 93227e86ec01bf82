// ops_api.cpp — the C entry points of the operators around the encoder
// (include/bert_amd.h): argument checks, the device, and the launch.  Nothing
// throws across them and nothing is launched for a refused call.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <utility>
#include <vector>

#include "ggml_formats.h"
#include "ops.h"

using namespace bertamd;

namespace {

int refuse(const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_last_error(buf);
    return -1;
}

// runs `launch` with `device` current and puts the caller's device back
template <typename F>
int32_t on_device(const char *who, int32_t device, const F &launch) {
    int before = 0;
    hipError_t e = hipGetDevice(&before);
    if (e == hipSuccess && before != device) e = hipSetDevice(device);
    if (e == hipSuccess) {
        e = launch();
        if (before != device) (void)hipSetDevice(before);
    }
    if (e == hipSuccess) return 0;
    (void)hipGetLastError();  // reported here: not left for the thread's next caller to find
    refuse("%s: %s", who, hipGetErrorString(e));
    return -3;
}

bool is_float(int32_t t) { return t == BERT_AMD_F32 || t == BERT_AMD_F16 || t == BERT_AMD_BF16; }
int size_of(int32_t t) { return t == BERT_AMD_F32 ? 4 : 2; }
bool off(const void *p, int64_t size) { return ((uintptr_t)p & (size - 1)) != 0; }

struct Matrix {
    const char *name;
    const void *p;
    int64_t ld;
    int64_t width;
    bool input;
    int size;
};
// null, misaligned or overlapping rows: the matrix's name, else null
const char *bad_matrix(const Matrix &m) {
    if (!m.p || off(m.p, m.size) || m.ld > (int64_t)1 << 40) return m.name;
    return m.ld >= m.width || (m.input && m.ld == 0) ? nullptr : m.name;
}

// Whether any byte belongs to a row of both.  Rows of the same stride may lie
// side by side, as columns of one wider matrix do; with different strides,
// spans that meet count as overlapping.
bool overlap(const Matrix &a, int64_t a_rows, const Matrix &b, int64_t b_rows) {
    if (!a.p || !b.p || a_rows < 1 || b_rows < 1) return false;
    const int64_t wa = a.width * a.size, wb = b.width * b.size, la = a.ld * a.size, lb = b.ld * b.size;
    const char *pa = (const char *)a.p, *pb = (const char *)b.p;
    if (pa + (a_rows - 1) * la + wa <= pb || pb + (b_rows - 1) * lb + wb <= pa) return false;
    if (la != lb || la == 0) return true;
    int64_t d = (pb - pa) % la;
    if (d < 0) d += la;
    return d < wa || d + wb > la;
}

constexpr int64_t MAX_M = (int64_t)1 << 30;
constexpr int32_t MAX_SIDE = (1 << 22) - 1, MAX_WIDTH = (1 << 20) - 1, MAX_IDS = 1 << 28, MAX_ROWS = 1 << 30;

// the largest product's 64 x 64 tiles fit a launch (under 2^32 threads)
constexpr int64_t MAX_AREA = (int64_t)1 << 34;

bool linear_shape_ok(int32_t type, int64_t M, int32_t N, int32_t K) {
    return is_float(type) && M >= 0 && M <= MAX_M && N >= 1 && N <= MAX_SIDE && K >= 1 && K <= MAX_SIDE &&
           M * N <= MAX_AREA && M * K <= MAX_AREA && (int64_t)N * K <= MAX_AREA;
}
// The memory of an optimizer step: what is written must be disjoint, and what is
// read must not lie in it.  Tensors usually follow each other in buffers of
// their own, which one look at each tells; else the spans are sorted.
struct Spans {
    static constexpr int READ = 6;  // kinds 0 .. 5 are written
    typedef std::pair<const char *, const char *> Span;
    std::vector<Span> of[READ + 1];
    void add(int kind, const void *p, int64_t bytes) { of[kind].emplace_back((const char *)p, (const char *)p + bytes); }
    bool empty() const { return of[0].empty(); }
    bool clash() {
        std::vector<Span> whole;  // from each kind's first byte to its last
        bool ordered = true;
        for (int k = 0; k <= READ; k++) {
            if (of[k].empty()) continue;
            Span w = of[k][0];
            for (size_t i = 1; i < of[k].size(); i++) {
                ordered = ordered && (k == READ || of[k][i].first >= of[k][i - 1].second);
                w.first = std::min(w.first, of[k][i].first), w.second = std::max(w.second, of[k][i].second);
            }
            for (const Span &o : whole) ordered = ordered && (w.first >= o.second || o.first >= w.second);
            whole.push_back(w);
        }
        if (ordered) return false;
        std::vector<Span> written;
        for (int k = 0; k < READ; k++) written.insert(written.end(), of[k].begin(), of[k].end());
        std::sort(written.begin(), written.end());
        for (size_t i = 1; i < written.size(); i++)
            if (written[i].first < written[i - 1].second) return true;
        for (const Span &r : of[READ]) {  // the last written span that begins before r's end
            auto at = std::lower_bound(written.begin(), written.end(), Span(r.second, nullptr));
            if (at != written.begin() && (--at)->second > r.first) return true;
        }
        return false;
    }
};
bool workspace_ok(const void *p, int64_t bytes, int64_t need) {
    return need == 0 || (p && bytes >= need && !off(p, 16));
}

}  // namespace

extern "C" {

int64_t bert_amd_linear_workspace(int32_t type, int64_t M, int32_t N, int32_t K, int32_t aligned) {
    if (!linear_shape_ok(type, M, N, K)) return refuse("bert_amd_linear_workspace: invalid type or size");
    return linear_ws_bytes(type, M, N, K, aligned != 0);
}

int32_t bert_amd_linear(int32_t device, int32_t type, int32_t act, int64_t M, int32_t N, int32_t K, const void *x, int64_t ldx,
                        const void *w, int64_t ldw, const float *bias, const void *residual, int64_t ldr, void *y, int64_t ldy,
                        void *z, int64_t ldz, void *workspace, int64_t workspace_bytes, void *hip_stream) {
    if (!linear_shape_ok(type, M, N, K)) return refuse("bert_amd_linear: invalid type or size (type %d, M %lld, N %d, K %d)", type, (long long)M, N, K);
    if (act < BERT_AMD_ACT_NONE || act > BERT_AMD_ACT_TANH) return refuse("bert_amd_linear: unknown activation %d", act);
    if (M == 0) return 0;
    const int e = size_of(type);
    const Matrix all[] = {{"x", x, ldx, K, true, e}, {"w", w, ldw, K, true, e}, {"y", y, ldy, N, false, e},
                          {"residual", residual, ldr, N, true, e}, {"z", z, ldz, N, false, e}};
    for (const Matrix &m : all)
        if (m.p || (m.name[0] != 'r' && m.name[0] != 'z'))
            if (const char *bad = bad_matrix(m)) return refuse("bert_amd_linear: %s is null, misaligned or has too short rows", bad);
    if (bias && off(bias, 4)) return refuse("bert_amd_linear: bias is misaligned");
    const Matrix vector = {"bias", bias, N, N, true, 4};
    const int64_t rows[] = {M, N, M, M, M};
    for (int out : {2, 4})
        for (int in = 0; in < 5; in++) {
            const bool same = out == 2 && in == 3 && residual == y && (ldr == ldy || M == 1);  // each element read before it is written
            if (in != out && !same && overlap(all[out], M, all[in], rows[in]))
                return refuse("bert_amd_linear: %s overlaps %s", all[out].name, all[in].name);
            if (overlap(all[out], M, vector, 1)) return refuse("bert_amd_linear: %s overlaps bias", all[out].name);
        }
    const int64_t need = linear_ws_bytes(type, M, N, K, linear_aligned(x, ldx, type) && linear_aligned(w, ldw, type));
    if (!workspace_ok(workspace, workspace_bytes, need))
        return refuse("bert_amd_linear: workspace is null, misaligned or under %lld bytes", (long long)need);
    const Matrix room = {"workspace", need ? workspace : nullptr, need, need, false, 1};
    for (int i = 0; i < 5; i++)
        if (overlap(room, 1, all[i], rows[i])) return refuse("bert_amd_linear: the workspace overlaps %s", all[i].name);
    if (overlap(room, 1, vector, 1)) return refuse("bert_amd_linear: the workspace overlaps bias");
    LinearArgs a;
    a.type = type, a.act = act, a.M = M, a.N = N, a.K = K;
    a.x = x, a.w = w, a.r = residual, a.bias = bias, a.y = y, a.z = z, a.ws = workspace;
    a.ldx = ldx, a.ldw = ldw, a.ldr = ldr, a.ldy = ldy, a.ldz = ldz;
    return on_device("bert_amd_linear", device, [&] { return launch_linear(a, (hipStream_t)hip_stream); });
}

int64_t bert_amd_linear_backward_workspace(int32_t type, int32_t act, int64_t M, int32_t N, int32_t K, int32_t aligned) {
    if (!linear_shape_ok(type, M, N, K)) return refuse("bert_amd_linear_backward_workspace: invalid type or size");
    return linear_grad_ws_bytes(type, act, M, N, K, aligned != 0);
}

int32_t bert_amd_linear_backward(int32_t device, int32_t type, int32_t act, int64_t M, int32_t N, int32_t K, const void *dy,
                                 int64_t lddy, const void *z, int64_t ldz, const void *x, int64_t ldx, const void *w, int64_t ldw,
                                 void *dx, int64_t lddx, void *dw, int64_t lddw, float *dbias, void *workspace,
                                 int64_t workspace_bytes, void *hip_stream) {
    if (!linear_shape_ok(type, M, N, K))
        return refuse("bert_amd_linear_backward: invalid type or size (type %d, M %lld, N %d, K %d)", type, (long long)M, N, K);
    if (act < BERT_AMD_ACT_NONE || act > BERT_AMD_ACT_TANH) return refuse("bert_amd_linear_backward: unknown activation %d", act);
    const int e = size_of(type);
    const Matrix ins[] = {{"dy", dy, lddy, N, true, e}, {"z", z, ldz, N, true, e}, {"x", x, ldx, K, true, e}, {"w", w, ldw, K, true, e}};
    const bool reads[] = {true, act != BERT_AMD_ACT_NONE, dw != nullptr, dx != nullptr};
    for (int i = 0; i < 4; i++)
        if (reads[i] && M > 0)
            if (const char *bad = bad_matrix(ins[i])) return refuse("bert_amd_linear_backward: %s is null, misaligned or has too short rows", bad);
    const Matrix outs[] = {{"dx", dx, lddx, K, false, e}, {"dw", dw, lddw, K, false, e}, {"dbias", dbias, N, N, false, 4}};
    for (const Matrix &m : outs)
        if (m.p)
            if (const char *bad = bad_matrix(m)) return refuse("bert_amd_linear_backward: %s is misaligned or has too short rows", bad);
    if (!dx && !dw && !dbias) return 0;
    const int64_t in_rows[] = {M, M, M, N}, out_rows[] = {M, N, 1};
    for (int o = 0; o < 3; o++) {
        for (int i = 0; i < 4; i++)
            if (reads[i] && overlap(outs[o], out_rows[o], ins[i], in_rows[i]))
                return refuse("bert_amd_linear_backward: %s overlaps %s", outs[o].name, ins[i].name);
        for (int i = 0; i < o; i++)
            if (overlap(outs[o], out_rows[o], outs[i], out_rows[i]))
                return refuse("bert_amd_linear_backward: %s overlaps %s", outs[o].name, outs[i].name);
    }
    const bool aligned = linear_aligned(dy, lddy, type) && (!dw || linear_aligned(x, ldx, type)) && (!dx || linear_aligned(w, ldw, type));
    const int64_t need = linear_grad_ws_bytes(type, act, M, N, K, aligned);
    if (!workspace_ok(workspace, workspace_bytes, need))
        return refuse("bert_amd_linear_backward: workspace is null, misaligned or under %lld bytes", (long long)need);
    const Matrix room = {"workspace", need ? workspace : nullptr, need, need, false, 1};
    for (int i = 0; i < 4; i++)
        if (reads[i] && overlap(room, 1, ins[i], in_rows[i])) return refuse("bert_amd_linear_backward: the workspace overlaps %s", ins[i].name);
    for (int o = 0; o < 3; o++)
        if (overlap(room, 1, outs[o], out_rows[o])) return refuse("bert_amd_linear_backward: the workspace overlaps %s", outs[o].name);
    LinearGradArgs a;
    a.type = type, a.act = act, a.M = M, a.N = N, a.K = K;
    a.dy = dy, a.z = z, a.x = x, a.w = w, a.dx = dx, a.dw = dw, a.db = dbias, a.ws = workspace;
    a.lddy = lddy, a.ldz = ldz, a.ldx = ldx, a.ldw = ldw, a.lddx = lddx, a.lddw = lddw;
    return on_device("bert_amd_linear_backward", device, [&] { return launch_linear_grad(a, (hipStream_t)hip_stream); });
}

int32_t bert_amd_lookup(int32_t device, int32_t table_type, int32_t out_type, int64_t n, int32_t n_rows, int32_t width,
                        const void *table, int64_t ld_table_bytes, const int32_t *ids, float scale, void *out, int64_t ldo,
                        void *hip_stream) {
    const bool blocks = table_type == BERT_AMD_Q4_0 || table_type == BERT_AMD_Q4_1;
    if (!(is_float(table_type) || blocks) || !is_float(out_type)) return refuse("bert_amd_lookup: types %d, %d are not supported", table_type, out_type);
    if (n < 0 || n > MAX_M || n_rows < 1 || width < 1 || width > MAX_SIDE || (blocks && width % QK))
        return refuse("bert_amd_lookup: invalid size (n %lld, n_rows %d, width %d)", (long long)n, n_rows, width);
    if (n == 0) return 0;
    const int e = is_float(table_type) ? size_of(table_type) : 2;
    const int64_t row = blocks ? (int64_t)ggml_row_bytes(table_type, width) : (int64_t)width * e;
    if (!table || off(table, e) || (ld_table_bytes != 0 && ld_table_bytes < row) || ld_table_bytes % e || ld_table_bytes > (int64_t)1 << 40)
        return refuse("bert_amd_lookup: table is null, misaligned or has too short rows");
    if (!ids || off(ids, 4)) return refuse("bert_amd_lookup: ids are null or misaligned");
    if (const char *bad = bad_matrix({"out", out, ldo, width, false, size_of(out_type)}))
        return refuse("bert_amd_lookup: %s is null, misaligned or has too short rows", bad);
    const Matrix written = {"out", out, ldo, width, false, size_of(out_type)};
    if (overlap(written, n, {"table", table, ld_table_bytes, row, true, 1}, n_rows) || overlap(written, n, {"ids", ids, n, n, true, 4}, 1))
        return refuse("bert_amd_lookup: out overlaps the table or the ids");
    LookupArgs a;
    a.type = table_type, a.out_type = out_type, a.n = n, a.V = n_rows, a.E = width;
    a.table = table, a.ld_bytes = ld_table_bytes, a.ids = ids, a.scale = scale, a.out = out, a.ldo = ldo;
    return on_device("bert_amd_lookup", device, [&] { return launch_lookup(a, (hipStream_t)hip_stream); });
}

int64_t bert_amd_lookup_grad_workspace(int64_t n, int32_t n_rows, int32_t width) {
    if (n < 0 || n > MAX_IDS || n_rows < 1 || n_rows > MAX_ROWS || width < 1 || width > MAX_WIDTH)
        return refuse("bert_amd_lookup_grad_workspace: invalid size");
    return lookup_grad_ws_bytes(n, n_rows, width);
}

int32_t bert_amd_lookup_grad(int32_t device, int32_t type, int64_t n, int32_t n_rows, int32_t width, const void *dout, int64_t ldd,
                             const int32_t *ids, float scale, int32_t pad_id, int32_t accumulate, float *dtable, int64_t ldt,
                             void *workspace, int64_t workspace_bytes, void *hip_stream) {
    if (!is_float(type)) return refuse("bert_amd_lookup_grad: type %d is not supported", type);
    if (n < 0 || n > MAX_IDS || n_rows < 1 || n_rows > MAX_ROWS || width < 1 || width > MAX_WIDTH)
        return refuse("bert_amd_lookup_grad: invalid size (n %lld, n_rows %d, width %d)", (long long)n, n_rows, width);
    if (n > 0) {
        if (const char *bad = bad_matrix({"dout", dout, ldd, width, true, size_of(type)}))
            return refuse("bert_amd_lookup_grad: %s is null, misaligned or has too short rows", bad);
        if (!ids || off(ids, 4)) return refuse("bert_amd_lookup_grad: ids are null or misaligned");
    }
    if (const char *bad = bad_matrix({"dtable", dtable, ldt, width, false, 4}))
        return refuse("bert_amd_lookup_grad: %s is null, misaligned or has too short rows", bad);
    const Matrix written = {"dtable", dtable, ldt, width, false, 4};
    if (overlap(written, n_rows, {"dout", dout, ldd, width, true, size_of(type)}, n) || overlap(written, n_rows, {"ids", ids, n, n, true, 4}, 1))
        return refuse("bert_amd_lookup_grad: dtable overlaps dout or the ids");
    const int64_t need = lookup_grad_ws_bytes(n, n_rows, width);
    if (!workspace_ok(workspace, workspace_bytes, need))
        return refuse("bert_amd_lookup_grad: workspace is null, misaligned or under %lld bytes", (long long)need);
    const Matrix room = {"workspace", need ? workspace : nullptr, need, need, false, 1};
    if (overlap(room, 1, written, n_rows) || overlap(room, 1, {"dout", dout, ldd, width, true, size_of(type)}, n) ||
        overlap(room, 1, {"ids", ids, n, n, true, 4}, 1))
        return refuse("bert_amd_lookup_grad: the workspace overlaps dtable, dout or the ids");
    LookupGradArgs a;
    a.type = type, a.n = n, a.V = n_rows, a.E = width, a.dout = dout, a.ldd = ldd, a.ids = ids, a.scale = scale;
    a.pad_id = pad_id, a.accumulate = accumulate != 0, a.dtable = dtable, a.ldt = ldt, a.ws = workspace;
    return on_device("bert_amd_lookup_grad", device, [&] { return launch_lookup_grad(a, (hipStream_t)hip_stream); });
}

int32_t bert_amd_adamw(int32_t device, int32_t n_tensors, const bert_amd_adamw_tensor *tensors, int32_t state_bits,
                       int32_t grad_type, int32_t copy_type, double lr, double beta1, double beta2, double eps, int64_t step,
                       uint32_t seed, const float *grad_scale, void *hip_stream) {
    if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return refuse("bert_amd_adamw: no tensors");
    if (state_bits != 32 && state_bits != 8) return refuse("bert_amd_adamw: states of %d bits are not supported", state_bits);
    if (!is_float(grad_type)) return refuse("bert_amd_adamw: gradients of type %d are not supported", grad_type);
    if (!(lr >= 0 && std::isfinite(lr)) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) ||
        !((float)eps > 0 && std::isfinite((float)eps)) || step < 1)
        return refuse("bert_amd_adamw: lr >= 0, 0 <= beta < 1, eps > 0 and step >= 1 are required");
    if (off(grad_scale, 4)) return refuse("bert_amd_adamw: grad_scale is misaligned");
    try {
        Spans spans;
        for (int i = 0; i < n_tensors; i++) {
            const bert_amd_adamw_tensor &t = tensors[i];
            if (t.n < 0 || t.n > MAX_AREA || !(t.weight_decay >= 0 && std::isfinite(t.weight_decay)))
                return refuse("bert_amd_adamw: tensor %d has an invalid size or weight decay", i);
            if (!t.n) continue;
            const int64_t s = state_bits == 32 ? 4 : 1;
            if (!t.p || off(t.p, 4) || !t.grad || off(t.grad, size_of(grad_type)) || !t.m || off(t.m, s) || !t.v || off(t.v, s) ||
                (state_bits == 8 && (!t.m_scale || off(t.m_scale, 4) || !t.v_scale || off(t.v_scale, 4))))
                return refuse("bert_amd_adamw: tensor %d has a null or misaligned pointer", i);
            if (t.copy && (copy_type != BERT_AMD_F16 && copy_type != BERT_AMD_BF16))
                return refuse("bert_amd_adamw: copies of type %d are not supported", copy_type);
            if (t.copy && off(t.copy, 2)) return refuse("bert_amd_adamw: tensor %d has a misaligned copy", i);
            const int64_t blocks = state_bits == 8 ? (t.n + 255) / 256 * 4 : 0;
            spans.add(0, t.p, t.n * 4), spans.add(1, t.m, t.n * s), spans.add(2, t.v, t.n * s);
            if (blocks) spans.add(3, t.m_scale, blocks), spans.add(4, t.v_scale, blocks);
            if (t.copy) spans.add(5, t.copy, t.n * 2);
            spans.add(Spans::READ, t.grad, t.n * size_of(grad_type));
        }
        if (spans.empty()) return 0;
        if (grad_scale) spans.add(Spans::READ, grad_scale, 4);
        if (spans.clash()) return refuse("bert_amd_adamw: two tensors share memory, or a gradient lies in what is written");
    } catch (const std::exception &e) {
        return refuse("bert_amd_adamw: %s", e.what());
    }
    AdamwArgs a;
    a.n_tensors = n_tensors, a.t = tensors, a.bits = state_bits, a.grad_type = grad_type, a.copy_type = copy_type;
    a.lr = lr, a.beta1 = beta1, a.beta2 = beta2, a.eps = eps, a.step = step, a.seed = seed, a.grad_scale = grad_scale;
    return on_device("bert_amd_adamw", device, [&] { return launch_adamw(a, (hipStream_t)hip_stream); });
}

int32_t bert_amd_adamw_moments(int32_t device, int64_t n, const void *m, const float *m_scale, const void *v, const float *v_scale,
                               float *m_out, float *v_out, void *hip_stream) {
    if (n < 0 || n > (int64_t)1 << 40) return refuse("bert_amd_adamw_moments: invalid size");
    if (n == 0 || (!m_out && !v_out)) return 0;
    if ((m_out && (!m || !m_scale || off(m_scale, 4) || off(m_out, 4))) || (v_out && (!v || !v_scale || off(v_scale, 4) || off(v_out, 4))))
        return refuse("bert_amd_adamw_moments: a null or misaligned pointer");
    const int64_t blocks = (n + 255) / 256;
    const Matrix ins[] = {{"m", m_out ? m : nullptr, n, n, true, 1}, {"m_scale", m_out ? m_scale : nullptr, blocks, blocks, true, 4},
                          {"v", v_out ? v : nullptr, n, n, true, 1}, {"v_scale", v_out ? v_scale : nullptr, blocks, blocks, true, 4}};
    const Matrix outs[] = {{"m_out", m_out, n, n, false, 4}, {"v_out", v_out, n, n, false, 4}};
    for (const Matrix &o : outs)
        for (const Matrix &i : ins)
            if (overlap(o, 1, i, 1)) return refuse("bert_amd_adamw_moments: %s overlaps %s", o.name, i.name);
    if (overlap(outs[0], 1, outs[1], 1)) return refuse("bert_amd_adamw_moments: m_out overlaps v_out");
    return on_device("bert_amd_adamw_moments", device, [&] {
        return launch_adamw_moments(n, (const uint8_t *)m, m_scale, (const uint8_t *)v, v_scale, m_out, v_out, (hipStream_t)hip_stream);
    });
}

}  // extern "C"

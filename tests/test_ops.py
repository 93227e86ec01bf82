"""The operators around the encoder (include/bert_amd.h, bertops.py) against plain implementations in
64 bits, and what they refuse.

Tolerances: a result rounded to type t is off by at most u(t) = finfo(t).eps / 2 of its value; a sum of n
terms held in f32, in any order, by at most n 2^-24 of the sum of the terms' magnitudes; f32 operands may be
taken as two 16-bit halves, 22 bits or more of them, which three products leave at most 3 * 2^-22 = 12 * 2^-24
off; f32 evaluations of the activations by a few 2^-24 of the largest term in them (SLACK of them).
"""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import bertlib

torch = pytest.importorskip("torch")
import bertops  # noqa: E402

gpu = pytest.mark.gpu
F64 = torch.float64
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U32 = 2.0**-24
SLACK = 32


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the spacing of the smallest values: what rounding is off by next to zero."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, dtype=F64) * std


def act64(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "gelu":
        return z * torch.sigmoid(2 * (2 / np.pi) ** 0.5 * (z + 0.044715 * z**3))
    if act == "gelu_erf":
        return 0.5 * z * torch.special.erfc(-z * 0.5**0.5)  # its lower tail has no cancellation
    if act == "silu":
        return z * torch.sigmoid(z)
    return torch.tanh(z) if act == "tanh" else z


def strided(t, pad):
    """The same values with rows `pad` elements further apart, the space between filled with NaN."""
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    wide[:, : t.shape[1]] = t
    return wide[:, : t.shape[1]]


def close(got, want, tol, what):
    got = got.detach().to("cpu", F64)
    off = (got - want).abs() - tol
    assert torch.isfinite(got).all(), what
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum())} of {off.numel()} too far, worst {float(off.max()):.3g} over its bound"


# ---- the dense layer

ODD = [(1, 1, 1), (1, 384, 384), (3, 5, 7), (17, 33, 65), (64, 64, 64), (130, 200, 72), (257, 128, 96), (5, 4100, 31), (300, 31, 1030), (8, 70, 4100), (2, 1026, 4096), (9, 1000, 300), (1, 8, 5000)]


def make_layer(M, K, N, dtype, seed=0):
    g = gen(seed)
    return [t.to(dtype) for t in (normal(g, M, K), normal(g, N, K, std=K**-0.5), normal(g, M, N))] + [normal(g, N).float()]


def check_linear(x, w, b, r, act, y, z=None):
    """y and z against 64 bits; the arguments on the CPU."""
    dt, K = x.dtype, x.shape[1]
    terms = x.to(F64).abs() @ w.to(F64).abs().t() + (0 if b is None else b.to(F64).abs())
    zz = x.to(F64) @ w.to(F64).t() + (0 if b is None else b.to(F64))
    off = (K + 2 + 12) * U32 * terms
    if z is not None:
        close(z, zz, off + u(dt) * (zz.abs() + off) + tiny(dt), "z")
    want = act64(zz, act)
    off = 1.13 * off + SLACK * U32 * zz.abs()  # no activation is steeper than 1.13
    if r is not None:
        want = want + r.to(F64)
        off = off + U32 * (want.abs() + off)
    close(y, want, off + u(dt) * (want.abs() + off) + tiny(dt), "y")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", ODD)
def test_linear(M, K, N, dtype):
    x, w, r, b = make_layer(M, K, N, DTYPES[dtype])
    X, W, R, B = (t.cuda() for t in (x, w, r, b))
    for i, act in enumerate(bertops.ACTS):
        res, bias = (i & 1) == 0, i != 3
        y, z = bertops.linear(X, W, B if bias else None, residual=R if res else None, act=act, save_z=True)
        check_linear(x, w, b if bias else None, r if res else None, act, y, z)
    again = bertops.linear(X, W, B, residual=R, act=act)
    assert torch.equal(again, bertops.linear(X, W, B, residual=R, act=act))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 768, 384), (2, 1024, 1024), (16, 384, 1536), (100, 1024, 768), (1024, 384, 384), (2050, 768, 520), (1100, 1000, 1100), (6200, 136, 2056), (6199, 72, 2063)])
def test_linear_wide(M, K, N, dtype):
    """Sizes of whole layers: every tile form, ends of rows and columns inside a tile."""
    x, w, r, b = make_layer(M, K, N, DTYPES[dtype], seed=1)
    y, z = bertops.linear(x.cuda(), w.cuda(), b.cuda(), residual=r.cuda(), act="gelu", save_z=True)
    check_linear(x, w, b, r, "gelu", y, z)
    check_linear(x, w, None, None, "none", bertops.linear(x.cuda(), w.cuda()))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_linear_strides(pad, dtype):
    """Rows further apart than their width, at every alignment; nothing is read or written between them."""
    M, K, N = 70, 96, 130
    x, w, r, b = make_layer(M, K, N, DTYPES[dtype], seed=2)
    out = strided(torch.zeros(M, N, dtype=DTYPES[dtype], device="cuda"), pad)
    y = bertops.linear(strided(x.cuda(), pad), strided(w.cuda(), pad), b.cuda(), residual=strided(r.cuda(), pad), act="silu", out=out)
    assert y.data_ptr() == out.data_ptr()
    check_linear(x, w, b, r, "silu", y)
    assert torch.isnan(out._base[:, N:]).all()
    y = bertops.linear(x.cuda()[:1].expand(M, K), w.cuda(), b.cuda())  # one row for all
    check_linear(x[:1].expand(M, K), w, b, None, "none", y)
    got = r.cuda()
    bertops.linear(x.cuda(), w.cuda(), b.cuda(), residual=got, out=got)  # in place on the residual
    check_linear(x, w, b, r, "none", got)


@gpu
def test_linear_large_values_and_nonfinite():
    """f32 rows of any size keep their precision; an infinity or NaN stays in its row."""
    x, w, _, b = make_layer(40, 256, 64, torch.float32, seed=3)
    size = torch.logspace(-30, 30, 40, dtype=F64)[:, None].float()
    y = bertops.linear((x * size).cuda(), w.cuda())
    check_linear(x * size, w, None, None, "none", y)
    mixed = x.clone()
    mixed[:, ::3] *= 1e-6
    check_linear(mixed, w, None, None, "none", bertops.linear(mixed.cuda(), w.cuda()))
    for bad in (float("inf"), float("nan")):
        for rows in (40, 1):
            xb = x[:rows].clone()
            xb[0, 5] = bad
            y = bertops.linear(xb.cuda(), w.cuda(), b.cuda()).cpu()
            assert not torch.isfinite(y[0]).any()
            assert torch.isfinite(y[1:]).all()


@gpu
@pytest.mark.parametrize("act", bertops.ACTS)
def test_activations_far_out(act):
    """One column, weight 1: every activation and slope over the whole range, tails and extremes."""
    z = torch.cat([torch.linspace(-30, 30, 4001, dtype=F64), torch.tensor([-1e4, -88.8, -1e-8, 0.0, 1e-30, 1e-8, 89.5, 1e4, 3e18, -3e18, 1e30, -1e30], dtype=F64)]).float()
    one = torch.ones(1, 1, device="cuda")
    y = bertops.linear(z[:, None].cuda(), one, act=act)
    want = act64(z.to(F64), act)
    # the tanh form's argument u, cubic in z, is rounded to a few 2^-24 of itself and enters an exponential
    steep = 1 + (2 * z.to(F64).abs() ** 3).clamp(max=200) if act == "gelu" else 1 + z.to(F64).abs().clamp(max=200) ** (2 if act == "gelu_erf" else 1)
    close(y[:, 0], want, SLACK * U32 * steep * want.abs() + 2.0**-126, "y")
    dx, dw, db = bertops.linear_backward(torch.ones(len(z), 1, device="cuda"), z[:, None].cuda(), one, z=z[:, None].cuda(), act=act)
    at = z.to(F64).clone().requires_grad_(True)
    (slope,) = torch.autograd.grad(act64(at, act).sum(), at)
    slope = torch.nan_to_num(slope, nan=0.0)
    far = z.abs() > 100  # the reference's own products of 0 and infinity
    slope[far] = 0.0 if act == "tanh" else 1.0
    slope[far & (z < 0)] = 1.0 if act == "none" else 0.0
    close(dx[:, 0], slope, SLACK * U32 * (1 + z.to(F64).abs().clamp(max=30)), "slope")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N,pad", [(1, 1, 1, 0), (1, 384, 384, 0), (3, 5, 7, 0), (65, 130, 33, 3), (200, 64, 96, 8), (1000, 72, 40, 0), (1030, 384, 256, 0), (513, 520, 768, 0), (0, 48, 24, 0), (6201, 2056, 136, 0), (101, 3592, 3600, 0)])
def test_linear_backward(M, K, N, pad, dtype):
    dt = DTYPES[dtype]
    x, w, dy, _ = make_layer(M, K, N, dt, seed=4)
    z = normal(gen(5), M, N).to(dt)
    dev = (lambda t: strided(t.cuda(), pad)) if pad else (lambda t: t.cuda())
    for act in bertops.ACTS:
        dx, dw, db = bertops.linear_backward(dev(dy), dev(x), dev(w), z=dev(z), act=act)
        at = z.to(F64).clone().requires_grad_(True)
        (dz,) = torch.autograd.grad(act64(at, act), at, dy.to(F64))
        # the slope's own error, and in 16 bits the rounding of dz
        off = SLACK * U32 * (1 + z.to(F64).abs()) * dy.to(F64).abs() * (act != "none")
        offr = off + (u(dt) * dz.abs() + tiny(dt) if dt != torch.float32 else 0)
        terms = dz.abs() + offr
        for got, a, b, n, what in ((dx, terms, w.to(F64).abs(), N, "dx"), (dw, terms.t(), x.to(F64).abs(), M, "dw")):
            want = dz @ w.to(F64) if what == "dx" else dz.t() @ x.to(F64)
            o = (offr if what == "dx" else offr.t()) @ b + (n + 12) * U32 * (a @ b)
            close(got, want, o + u(dt) * (want.abs() + o) + tiny(dt), f"{what} {act}")
        o = off.sum(0) + (M + 1) * U32 * (dz.abs() + off).sum(0)
        close(db, dz.sum(0), o, f"db {act}")
        if M * N * K > 1e9 and act == "relu":
            break  # the large ones: two activations
        for need in ((True, False, False), (False, True, False), (False, False, True)):
            part = bertops.linear_backward(dev(dy), dev(x), dev(w), z=dev(z), act=act, need=need)
            for a, b, n in zip(part, (dx, dw, db), need):
                assert (a is None) if not n else torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N,pad", [(1, 25, 133, 0), (1, 768, 1, 0), (2, 32, 32, 3), (4, 2144, 33, 8), (5, 513, 2100, 0), (7, 8, 8192, 0), (8, 1000, 777, 5), (8, 4096, 4096, 0)])
def test_few_rows_backward(M, K, N, pad, dtype):
    """Up to 8 rows dz is not rounded before the products: only sums in f32 and each result's own rounding remain."""
    dt = DTYPES[dtype]
    x, w, dy, _ = make_layer(M, K, N, dt, seed=23)
    z = normal(gen(24), M, N).to(dt)
    dev = (lambda t: strided(t.cuda(), pad)) if pad else (lambda t: t.cuda())
    for act in bertops.ACTS:
        dx, dw, db = bertops.linear_backward(dev(dy), dev(x), dev(w), z=dev(z), act=act)
        at = z.to(F64).clone().requires_grad_(True)
        (dz,) = torch.autograd.grad(act64(at, act), at, dy.to(F64))
        off = SLACK * U32 * (1 + z.to(F64).abs()) * dy.to(F64).abs() * (act != "none")
        for got, a, o, b, n, what in ((dx, dz, off, w, N, "dx"), (dw, dz.t(), off.t(), x, M, "dw")):
            want, far = a @ b.to(F64), (o + (n + 1) * U32 * (a.abs() + o)) @ b.to(F64).abs()
            close(got, want, far + u(dt) * (want.abs() + far) + tiny(dt), f"{what} {act}")
        close(db, dz.sum(0), off.sum(0) + (M + 1) * U32 * (dz.abs() + off).sum(0), f"db {act}")


@gpu
def test_linear_backward_by_differences():
    """The loss sum(c y) changes along each input as its gradient says."""
    M, K, N = 6, 11, 9
    g = gen(6)
    x, w, r, c = (normal(g, *s).float() for s in ((M, K), (N, K), (M, N), (M, N)))
    b = normal(g, N).float()
    for act in ("gelu", "gelu_erf", "silu", "tanh"):
        y, z = bertops.linear(x.cuda(), w.cuda(), b.cuda(), residual=r.cuda(), act=act, save_z=True)
        grads = dict(zip("xwb", bertops.linear_backward(c.cuda(), x.cuda(), w.cuda(), z=z, act=act)))
        for name, t in (("x", x), ("w", w), ("b", b)):
            d = normal(gen(7), *t.shape)
            h = 1e-6
            loss = lambda s: float((c.to(F64) * act64((x.to(F64) + (s * d if name == "x" else 0)) @ (w.to(F64) + (s * d if name == "w" else 0)).t() + b.to(F64) + (s * d if name == "b" else 0), act)).sum())  # noqa: E731, B023
            want = (loss(h) - loss(-h)) / (2 * h)
            got = float((grads[name].cpu().to(F64) * d).sum())
            size = float((grads[name].cpu().to(F64) * d).abs().sum())
            # the difference is off by h^2 times third derivatives and by 64-bit rounding over h; the gradient by f32 sums
            assert abs(got - want) <= 1e-8 * (1 + size) * 10 + (max(M, K, N) + SLACK + 12) * U32 * size * 4, (name, act, got, want)


# ---- token rows


def make_table(t, V, E, seed=0):
    g = gen(seed)
    if t in DTYPES:
        v = normal(g, V, E).to(DTYPES[t])
        return v, v.to(F64)
    nb = E // 32
    qs = torch.randint(0, 256, (V, nb, 16), generator=g, dtype=torch.uint8)
    head = (normal(g, V, nb, 1 if t == "q4_0" else 2) * 0.1).half()
    raw = torch.cat([head.view(torch.uint8), qs], 2).reshape(V, -1).contiguous()
    q = torch.cat([qs & 15, qs >> 4], 2).to(F64)
    d = head[..., :1].to(F64)
    return raw, ((q - 8) * d if t == "q4_0" else q * d + head[..., 1:].to(F64)).reshape(V, E)


@gpu
@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("kind,E,pad", [("f32", 1, 0), ("f32", 384, 0), ("f16", 7, 0), ("f16", 768, 8), ("bf16", 129, 3), ("bf16", 1024, 0), ("q4_0", 32, 0), ("q4_0", 384, 2), ("q4_1", 96, 0), ("q4_1", 1024, 4), ("f16", 100, 4), ("f32", 2050, 2)])
def test_lookup(kind, E, pad, out):
    V = 50
    table, values = make_table(kind, V, E)
    dev = strided(table.cuda(), pad) if pad and kind in DTYPES else table.cuda()
    if pad and kind not in DTYPES:
        wide = torch.full((V, table.shape[1] + pad), 255, dtype=torch.uint8, device="cuda")
        wide[:, : table.shape[1]] = table.cuda()
        dev = wide[:, : table.shape[1]]
    for ids in ([0], [V - 1, -1, 3, 3, V, 2**31 - 1, -(2**31), 0], list(range(V)) * 41):
        ids = torch.tensor(ids, dtype=torch.int32)
        for scale in (1.0, E**0.5):
            got = bertops.lookup(dev, ids.cuda(), scale=scale, table_type=kind, out_dtype=DTYPES[out])
            there = (ids >= 0) & (ids < V)
            want = torch.where(there[:, None], values[ids.clamp(0, V - 1).long()], torch.zeros((), dtype=F64)) * scale
            off = 3 * U32 * (want.abs() + (values.abs().max() * scale if kind == "q4_1" else 0))  # the scale's rounding, the product's, q4_1's sum
            close(got, want, off + u(DTYPES[out]) * (want.abs() + off) + tiny(DTYPES[out]), f"{kind} {out}")
            assert (got[~there.cuda()] == 0).all()
    assert bertops.lookup(dev, torch.zeros(0, dtype=torch.int32, device="cuda"), table_type=kind).shape[0] == 0
    grid = torch.tensor([[1, 2, 3], [4, 5, 6]], dtype=torch.int32)
    assert torch.equal(bertops.lookup(dev, grid.cuda(), table_type=kind).reshape(6, E), bertops.lookup(dev, grid.flatten().cuda(), table_type=kind))


@gpu
def test_lookup_past_32_bits():
    """Rows that begin over 2^32 bytes into the table, and an output over 2^31 elements."""
    V, E = 1_500_000, 1024
    table = torch.empty(V, E, dtype=torch.float32, device="cuda")
    at = torch.tensor([0, 1_048_575, 1_048_576, 1_048_577, V - 1], dtype=torch.int32, device="cuda")
    for i in at.tolist():
        table[i] = torch.arange(E, device="cuda") + i
    assert torch.equal(bertops.lookup(table, at), table[at.long()])
    del table
    small = normal(gen(8), 3, E).half().cuda()
    ids = torch.zeros((1 << 21) + 5, dtype=torch.int32, device="cuda")
    ids[-3:] = torch.tensor([1, -1, 2])
    out = bertops.lookup(small, ids)
    assert torch.equal(out[-3], small[1]) and (out[-2] == 0).all() and torch.equal(out[-1], small[2]) and torch.equal(out[1 << 20], small[0])


def check_grad(got, dout, ids, V, scale, pad, base=None):
    there = (ids >= 0) & (ids < V) & (ids != pad)
    at, rows = ids[there].long(), dout[there].to(F64)
    E = dout.shape[1]
    want = torch.zeros(V, E, dtype=F64).index_add_(0, at, rows)
    size = torch.zeros(V, E, dtype=F64).index_add_(0, at, rows.abs())
    count = torch.bincount(at, minlength=V).to(F64)[:, None]
    off = (count + 2) * U32 * size * abs(scale)
    want = want * scale
    if base is not None:
        want = want + base.to(F64)
        off = off + U32 * want.abs()
        assert torch.equal(got.cpu()[count[:, 0] == 0], base[count[:, 0] == 0])
    close(got, want, off + 2.0**-149, "dtable")
    if base is None:
        assert (got.cpu()[count[:, 0] == 0] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,E,pad_ld", [(0, 5, 8, 0), (1, 1, 1, 0), (1, 30522, 384, 0), (7, 3, 33, 3), (64, 10, 384, 0), (1000, 100, 130, 8), (2048, 30522, 64, 0), (4095, 517, 96, 0), (4096, 60, 30, 0), (4097, 511, 130, 0), (5000, 2, 40, 0), (40000, 70000, 32, 0), (66000, 300000, 20, 0), (9000, 1, 300, 1), (30000, 900, 768, 0)])
def test_lookup_grad(n, V, E, pad_ld, dtype):
    g = gen(9)
    dout = normal(g, n, E).to(DTYPES[dtype])
    ids = (V * torch.rand(n, generator=g, dtype=F64) ** 4).to(torch.int32)
    if n > 4:
        ids[1], ids[3] = -1, V
    dev = strided(dout.cuda(), pad_ld) if pad_ld and n else dout.cuda()
    for scale, pad in ((1.0, -1), (-2.5, 0)):
        out = strided(torch.zeros(V, E, device="cuda"), pad_ld) if pad_ld else torch.full((V, E), float("nan"), device="cuda")
        got = bertops.lookup_grad(dev, ids.cuda(), V, scale=scale, pad_id=pad, out=out)
        check_grad(got, dout, ids, V, scale, pad)
        if pad_ld:
            assert torch.isnan(out._base[:, E:]).all()
        assert torch.equal(got, bertops.lookup_grad(dev, ids.cuda(), V, scale=scale, pad_id=pad))  # the same bits
        base = normal(g, V, E).float()
        got = bertops.lookup_grad(dev, ids.cuda(), V, scale=scale, pad_id=pad, out=base.cuda(), accumulate=True)
        check_grad(got, dout, ids, V, scale, pad, base)


@gpu
def test_lookup_grad_one_token():
    """Every place the same token, and one gradient row broadcast to all places."""
    n, E = 70000, 48
    dout = normal(gen(10), 1, E).half()
    ids = torch.full((n,), 2, dtype=torch.int32)
    got = bertops.lookup_grad(dout.cuda().expand(n, E), ids.cuda(), 4)
    check_grad(got, dout.expand(n, E), ids, 4, 1.0, -1)
    got = bertops.lookup_grad(dout.cuda().expand(n, E), torch.full_like(ids, -1).cuda(), 4)
    assert (got == 0).all()


@gpu
def test_lookup_grad_by_differences():
    """The loss sum(c out) is linear in the table: its change along any direction is the gradient's product with it."""
    V, E, n = 20, 24, 60
    g = gen(11)
    d, c = normal(g, V, E), normal(g, n, E)
    ids = torch.randint(-1, V, (n,), generator=g, dtype=torch.int32)
    grad = bertops.lookup_grad(c.float().cuda(), ids.cuda(), V, scale=3.0)
    moved = bertops.lookup(d.float().cuda(), ids.cuda(), scale=3.0).cpu().to(F64)
    size = float((moved * c).abs().sum())
    assert abs(float((grad.cpu().to(F64) * d.float().to(F64)).sum()) - float((moved * c.float().to(F64)).sum())) <= (n + 4) * 2 * U32 * size


# ---- AdamW


def mix(h):
    h = np.asarray(h, np.uint32)
    h = (h ^ (h >> np.uint32(16))) * np.uint32(0x9E3779B9)
    h = (h ^ (h >> np.uint32(15))) * np.uint32(0xBB67AE85)
    return h ^ (h >> np.uint32(16))


def code_values(mant):
    n = 1 << mant
    c = np.arange(16 * n)
    e, f = c >> mant, c & (n - 1)
    return np.where(e == 0, f * (2.0 / n), (1 + f / n) * 2.0**e).astype(np.float32)


def encode(a, mant, h):
    """Codes and scales of f32 magnitudes, block by block, rounded at random by the bits h."""
    n, codes, scales = 1 << mant, np.zeros(len(a), np.int64), []
    drop = 23 - mant
    top = np.float32((2 - 2.0**-mant) * 2.0**15)
    for s in range(0, len(a), 256):
        x, bits = a[s : s + 256], h[s : s + 256]
        peak = x.max() if not np.isnan(x).any() else np.float32(np.nan)
        scale = np.float32(0) if peak < 2.0**-100 else np.float32(peak / top)
        scales.append(scale)
        if not (scale > 0 and np.isfinite(scale)):
            continue
        y = x * (np.float32(1) / scale)
        far = ((y.view(np.uint32).astype(np.int64) + (bits >> np.uint32(32 - drop))) >> drop) - 127 * n
        near = np.floor(y * np.float32(n / 2) + (bits >> np.uint32(8)).astype(np.float32) * np.float32(2.0**-24)).astype(np.int64)
        codes[s : s + 256] = np.minimum(np.where(y >= 2, far, near), 16 * n - 1)
    return codes, np.asarray(scales, np.float32)


class PlainAdamW:
    """The step on numpy f32 arrays in the order the header gives, every operation rounded by itself."""

    def __init__(self, ps, bits, lr, betas, eps, decay, seed):
        self.ps = [p.copy() for p in ps]
        self.m, self.v = [np.zeros_like(p) for p in ps], [np.zeros_like(p) for p in ps]
        self.bits, self.lr, self.betas, self.eps, self.decay, self.seed, self.t = bits, lr, betas, eps, decay, seed, 0

    def step(self, gs, scale=None):
        f = np.float32
        self.t += 1
        (b1, b2), t = self.betas, self.t
        k, root = f(self.lr / (1 - b1**t)), f(1 / (1 - b2**t) ** 0.5)
        with np.errstate(over="ignore", invalid="ignore", under="ignore"):
            for i, g in enumerate(gs):
                g = g.astype(f) * (f(scale) if scale is not None else f(1))
                m = self.m[i] * f(b1) + g * f(1 - b1)
                v = self.v[i] * f(b2) + (g * f(1 - b2)) * g
                r = np.sqrt(v)
                self.ps[i] = self.ps[i] * f(1 - self.lr * self.decay[i]) - (m * k) / (r * root + f(self.eps))
                if self.bits == 8:
                    seed = np.uint32((self.seed + t) & 0xFFFFFFFF)
                    with np.errstate(over="ignore"):
                        h = mix(np.arange(len(g), dtype=np.uint32) ^ mix(np.uint32(i) * np.uint32(0x9E3779B9) ^ seed))
                    c, s = encode(np.abs(m), 3, h)
                    each = np.repeat(s, 256)[: len(g)]
                    m = code_values(3)[c] * each * np.where(m < 0, f(-1), f(1))
                    c, s = encode(r, 4, mix(h ^ np.uint32(0x9E3779B9)))
                    each = np.repeat(s, 256)[: len(g)]
                    c = np.where((r > 0) & (c == 0) & (each > 0) & np.isfinite(each), 1, c)
                    r = code_values(4)[c] * each
                    v = r * r
                self.m[i], self.v[i] = m, v


@gpu
@pytest.mark.parametrize("grad", DTYPES)
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(bits, grad):
    """Four steps over tensors of every odd size: the same bits as the plain step, which rounds in the same order."""
    sizes = [1, 3, 255, 256, 257, 1000, 4096, 4097, 70001] + [5, 600] * 30  # more than one launch's table
    g = gen(12)
    ps = [normal(g, n, std=0.1).float() for n in sizes]
    decay = [0.1 * (i % 3) for i in range(len(sizes))]
    dev = [p.cuda() for p in ps]
    copies = [torch.zeros_like(p, dtype=torch.float16) for p in dev]
    opt = bertops.AdamW(dev, lr=3e-3, betas=(0.8, 0.99), eps=1e-7, weight_decay=decay, bits=bits, copies=copies, seed=0xFFFFFFFE)
    plain = PlainAdamW([p.numpy() for p in ps], bits, 3e-3, (0.8, 0.99), 1e-7, decay, 0xFFFFFFFE)
    for step in range(4):
        gs = [(normal(g, n, std=0.01) * torch.logspace(-6, 0, n, dtype=F64)).to(DTYPES[grad]) for n in sizes]
        for x in gs:
            x[::7] = 0
        scale = None if step < 2 else 0.37
        opt.step([x.cuda() for x in gs], None if scale is None else torch.tensor([scale], device="cuda"))
        plain.step([x.float().numpy() for x in gs], scale)
        m, v = opt.moments()
        for i, n in enumerate(sizes):
            a = opt.where[i]
            for got, want, what in ((dev[i], plain.ps[i], "p"), (m[a : a + n], plain.m[i], "m"), (v[a : a + n], plain.v[i], "v")):
                assert np.array_equal(got.cpu().numpy(), want), (what, i, n, step)
            assert torch.equal(copies[i], dev[i].half())


@gpu
def test_adamw_against_64_bits():
    """f32 states stay within the f32 error of each operation of the same step in 64 bits."""
    n = 5000
    g = gen(13)
    p = normal(g, n).float()
    dev = p.cuda()
    opt = bertops.AdamW([dev], lr=1e-2, weight_decay=0.1)
    q, m, v = p.to(F64), torch.zeros(n, dtype=F64), torch.zeros(n, dtype=F64)
    moved = torch.zeros(n, dtype=F64)
    for t in range(1, 6):
        gr = normal(g, n).float()
        opt.step([gr.cuda()])
        m, v = 0.9 * m + 0.1 * gr.to(F64), 0.999 * v + 0.001 * gr.to(F64) ** 2
        d = 1e-2 / (1 - 0.9**t) * m / (v.sqrt() / (1 - 0.999**t) ** 0.5 + 1e-8)
        q = q * (1 - 1e-2 * 0.1) - d
        moved += 1e-2 / (1 - 0.9**t) * (0.1 * 5 * 4) / (v.sqrt() / (1 - 0.999**t) ** 0.5 + 1e-8)  # |m| of gradients of at most 4 sigma
    got_m, got_v = opt.moments()
    close(got_v[:n], v, 5 * 6 * U32 * v, "v")
    close(got_m[:n], m, 5 * 4 * U32 * 6.0, "m")
    close(dev, q, 5 * 4 * U32 * (q.abs() + 1) + 40 * U32 * moved, "p")


@gpu
def test_adamw_8_bit_states_follow_the_32_bit_ones():
    """Rounding up or down at random has no drift: over blocks of equal values the stored moments average to the exact ones."""
    n, steps = 256 * 64, 40
    g = torch.logspace(-3, 0, 64, dtype=F64).repeat_interleave(256).float()  # one size a block
    a = bertops.AdamW([torch.zeros(n, device="cuda")], bits=8, seed=1)
    for _ in range(steps):
        a.step([g.cuda()])
    m, v = a.moments()
    want_m, want_r = g.to(F64) * (1 - 0.9**steps), g.to(F64) * (1 - 0.999**steps) ** 0.5
    got_m, got_r = (x.cpu().to(F64).reshape(64, 256).mean(1) for x in (m, v.sqrt()))
    # each step's rounding is within one code's step (2^-3 of m, 2^-4 of r) of the value, and the scale follows the
    # block's largest: a mean over 256 elements of a sum of such roundings, forgotten at rate 1 - beta, stays within one step
    assert ((got_m / want_m[::256] - 1).abs() < 2.0**-3).all()
    assert ((got_r / want_r[::256] - 1).abs() < 2.0**-2).all()


@gpu
def test_adamw_nonfinite_and_tiny():
    n = 700
    p = normal(gen(14), n).float().cuda()
    g = torch.zeros(n)
    g[300] = float("inf")
    for bits in (32, 8):
        w = p.clone()
        opt = bertops.AdamW([w], bits=bits, weight_decay=0.0)
        opt.step([g.cuda()])
        m, v = opt.moments()
        assert not torch.isfinite(w[300]) and torch.isfinite(w[:300]).all() and torch.isfinite(w[301:]).all()
        hurt = slice(300, 301) if bits == 32 else slice(256, 512)
        assert not torch.isfinite(m[hurt]).any() and not torch.isfinite(v[hurt]).any()
        assert torch.isfinite(m[:256]).all() and torch.isfinite(v[512:n]).all()
    w = p.clone()
    opt = bertops.AdamW([w], bits=8, weight_decay=0.0)
    opt.step([torch.full((n,), 1e-44).cuda()])  # moments under any scale: stored as zero, and the weights are sound
    assert (opt.moments()[0] == 0).all() and torch.isfinite(w).all()
    opt.step([torch.zeros(n, device="cuda")])
    assert torch.isfinite(w).all()


# ---- together: streams, graphs, other shapes of use


def train_once(table, w, b, ids, target, opts, copies=None):
    """Rows, a layer on their mean over each sentence, and one step of both: every operator, as they are used together."""
    rows = bertops.lookup(table, ids, scale=2.0)
    e = rows.mean(1)
    y, z = bertops.linear(e, w, b, residual=e, act="tanh", save_z=True)
    dy = (y - target) / len(y)
    de, dw, db = bertops.linear_backward(dy, e, w, z=z, act="tanh")
    de = de + dy
    dt = bertops.lookup_grad((de / ids.shape[1])[:, None, :].expand(rows.shape).contiguous(), ids, table.shape[0], scale=2.0, pad_id=0)
    return y, [dt, dw, db]


def training_inputs(V=300, E=64, n=40, L=12):
    g = gen(15)
    table, w, b = normal(g, V, E, std=0.5).float().cuda(), normal(g, E, E, std=0.1).float().cuda(), torch.zeros(E, device="cuda")
    ids = torch.randint(0, V, (n, L), generator=g, dtype=torch.int32).cuda()
    return table, w, b, ids, normal(g, n, E).float().cuda()


@gpu
def test_together_against_autograd():
    """One pass through lookup, layer and both gradients against torch's own gradients in 64 bits."""
    table, w, b, ids, target = training_inputs()
    y, (dt, dw, db) = train_once(table, w, b, ids, target, None)
    T, W, B = (t.cpu().to(F64).requires_grad_(True) for t in (table, w, b))
    rows = torch.where((ids.cpu() != 0)[..., None], T[ids.cpu().long()], T[ids.cpu().long()].detach()) * 2.0
    e = rows.mean(1)
    yy = torch.tanh(e @ W.t() + B) + e
    loss = (0.5 * (yy - target.cpu().to(F64)) ** 2).sum() / len(yy)
    loss.backward()
    # f32 through about ten sums of at most 64 terms: every value within 2^-24 times 1000 of the largest one around it
    for got, want in ((y, yy.detach()), (dt, T.grad), (dw, W.grad), (db, B.grad)):
        close(got, want, 1000 * U32 * want.abs().max() * torch.ones_like(want), "gradient")


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_together_in_a_graph(bits):
    """A whole training step captured once and replayed, with eager work and synchronisation between the replays."""
    table, w, b, ids, target = training_inputs()
    opts = [bertops.AdamW([t.clone() for t in (table, w, b)], bits=bits, seed=3) for _ in range(2)]
    static = [t.clone() for t in (ids, target)]

    def grads(opt):
        y, g = train_once(*opt.params, *static, None)
        return y, g

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        grads(opts[1])
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, g = grads(opts[1])
    for k in range(4):
        static[0].copy_((ids + k) % table.shape[0])
        static[1].copy_(target * (k + 1))
        graph.replay()
        want_y, want_g = grads(opts[0])
        torch.cuda.synchronize()
        assert torch.equal(y, want_y) and all(torch.equal(a, c) for a, c in zip(g, want_g)), k
        for o, gr in ((opts[0], want_g), (opts[1], g)):
            o.step(gr)
        assert all(torch.equal(a, c) for a, c in zip(opts[0].params, opts[1].params))


FIRST_CALLS = """
import sys
sys.path[:0] = sys.argv[1:]
import torch, bertops
g = torch.Generator(device="cuda").manual_seed(22)
def normal(*s, t=torch.float32): return torch.randn(*s, generator=g, device="cuda").to(t)
x, w, r, b = normal(4100, 520, t=torch.float16), normal(2056, 520, t=torch.float16), normal(4100, 2056, t=torch.float16), normal(2056)
xs, ws = normal(300, 77), normal(50, 77)
ids = torch.randint(-1, 700, (9000,), generator=g, device="cuda").int()
dout = normal(9000, 96, t=torch.bfloat16)
params = [normal(5000), normal(300, 7)]
grads = [normal(5000), normal(300, 7)]
opts = [bertops.AdamW([p.clone() for p in params], bits=bits) for bits in (32, 8) for _ in range(2)]
def calls(which):
    out = [bertops.linear(x, w, b, residual=r, act="gelu"), bertops.linear(x[:1], w, b), bertops.linear(xs, ws)]
    out += bertops.linear_backward(r, x, w, z=r, act="silu")
    out += [bertops.lookup(w, ids), bertops.lookup_grad(dout, ids, 700), bertops.lookup_grad(dout[:900], ids[:900], 700)]
    for o in (opts[which], opts[2 + which]):
        o.t = 4
        o.step(grads)
    return out
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls(0)
for k in range(4):
    graph.replay()
    want = calls(1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want)), k
    assert all(torch.equal(a, c) for i in (0, 2) for a, c in zip(opts[i].params + list(opts[i].moments()), opts[i + 1].params + list(opts[i + 1].moments()))), k
    for t in (x, r, dout, grads[0]): t.mul_(-0.75)
    ids.add_(1)
    torch.cuda.synchronize()
print("four replays")
"""


@gpu
def test_first_calls_are_captured():
    """A process whose first call of every kernel is recorded into a graph; the replays see new values."""
    paths = [os.path.dirname(bertops.__file__)]
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS, *paths], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "four replays" in done.stdout, done.stderr[-2000:]


@gpu
def test_adamw_refuses_what_has_moved():
    """Weights, copies and states that got other memory after the optimizer was made."""
    def made():
        p = torch.ones(600, device="cuda")
        return bertops.AdamW([p], bits=8, copies=[p.bfloat16()]), torch.ones(600, device="cuda")

    def move_weights(o):
        o.params[0].data = torch.ones(600, device="cuda")

    def move_copy(o):
        o.copies[0] = o.copies[0].clone()

    def move_state(o):
        o.v_scale = o.v_scale.clone()

    for move in (move_weights, move_copy, move_state):
        o, g = made()
        o.step([g])
        before = [t.clone() for t in (*o.params, *o.copies, o.m, o.v)]
        move(o)
        with pytest.raises(ValueError, match="no longer"):
            o.step([g])
        torch.cuda.synchronize()
        assert o.t == 1 and all(torch.equal(a, c) for a, c in zip(before[2:], (o.m, o.v)))


@gpu
def test_two_streams_at_once():
    """The same calls on two streams at a time give what each gives alone."""
    x, w, r, b = (t.cuda() for t in make_layer(700, 384, 384, torch.bfloat16, seed=16))
    g = gen(17)
    ids = [torch.randint(0, 5000, (20000,), generator=g, dtype=torch.int32).cuda() for _ in range(2)]
    dout = [normal(g, 20000, 96).half().cuda() for _ in range(2)]
    alone = [(bertops.lookup_grad(d, i, 5000), bertops.linear_backward(r, x, w, z=r, act="gelu")) for d, i in zip(dout, ids)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, d, i in zip(streams, dout, ids):
            with torch.cuda.stream(s):
                got.append((bertops.lookup_grad(d, i, 5000), bertops.linear_backward(r, x, w, z=r, act="gelu")))
        torch.cuda.synchronize()
        for (a, b1), (c, d1) in zip(got, alone):
            assert torch.equal(a, c) and all(torch.equal(p, q) for p, q in zip(b1, d1))


@gpu
def test_adapter_and_token_table(model_dir):
    """An adapter on a model's embeddings and its word rows made trainable: the framework's own users of the operators."""
    import os

    path = os.path.join(model_dir, "ops_minilm_q4_0.gguf")
    if not os.path.exists(path):
        bertlib.synth_model(path, "minilm", "q4_0", n_layer=1)
    for options, kind in ((None, "q4_0"), ({"emb_raw": 0}, "f32")):
        model = bertlib.BertModel(path, devices=[0], options=options)
        rows = bertops.word_rows(model)
        assert rows.shape == (30522, 384) and model.word_table()[1] == bertops.TABLE_TYPES[kind]
        from gguf_reader import GGUF

        want = torch.from_numpy(GGUF(path).f32("embeddings.word_embeddings.weight").reshape(30522, 384).copy())
        assert torch.equal(rows.cpu(), want)
        ids = torch.tensor([[101, 7, 102], [-1, 30522, 30521]], dtype=torch.int32)
        some = bertops.word_rows(model, ids.cuda(), scale=2.0).cpu()
        assert torch.equal(some[0], want[ids[0].long()] * 2) and (some[1, :2] == 0).all()
        sentences = ["hello world", "a second sentence", "x"]
        e = model.encode(sentences)
        adapter = bertops.Adapter(384, lr=1e-2)
        assert np.allclose(adapter.encode(model, sentences), e, atol=4 * 2.0**-23)  # zero weights: the embeddings themselves
        E = torch.from_numpy(e).cuda()
        y = adapter.forward(E)
        assert torch.equal(y, E)
        de = adapter.backward(y - 1.0, need_input=True)
        assert torch.equal(de, y - 1.0)  # through zero weights only the residual passes
        before = adapter.b.clone()
        adapter.step()
        assert (adapter.b > before).all()  # each bias's gradient is a sum of negative values
        table = bertops.TokenTable(model, lr=1e-2)
        out = table.forward(torch.tensor([5, 5, 9], dtype=torch.int32, device="cuda"))
        table.backward(torch.ones_like(out))
        table.backward(torch.ones_like(out))
        table.step()
        moved = (table.rows.cpu() != want * (1 - 1e-2 * 0.01)).any(1).nonzero()[:, 0].tolist()
        assert 5 in moved and 9 in moved and (table.rows.cpu()[5] < want[5]).all()
        model.close()


# ---- refusals: no GPU is needed, none is launched


def test_refusals_of_the_library():
    """Every bad argument of the C entry points is refused with a message before any device call."""
    L = bertlib.lib()
    P, NULL = 1 << 20, None  # an aligned address that nothing dereferences
    big = 1 << 40

    def refused(rc, word):
        assert rc == -1 and word in bertlib.last_error(), (rc, bertlib.last_error())

    ok = dict(device=0, type=0, act=0, M=4, N=8, K=8, x=P, ldx=8, w=P, ldw=8, bias=P, r=P, ldr=8, y=P + 4096, ldy=8, z=NULL, ldz=8, ws=2 * P, nws=big, s=NULL)
    for change, word in ((dict(type=2), "type"), (dict(type=7), "type"), (dict(act=6), "activation"), (dict(act=-1), "activation"), (dict(M=-1), "size"), (dict(M=(1 << 30) + 1), "size"), (dict(N=0), "size"), (dict(K=0), "size"), (dict(N=1 << 22), "size"), (dict(M=1 << 30, N=1 << 10), "size"), (dict(x=NULL), "x"), (dict(x=P + 2), "x"), (dict(ldx=7), "x"), (dict(ldx=-8), "x"), (dict(w=NULL), "w"), (dict(y=NULL), "y"), (dict(ldy=0), "y"), (dict(ldy=7), "y"), (dict(r=P + 1), "residual"), (dict(z=P, ldz=0), "z"), (dict(bias=P + 1), "bias"), (dict(r=P + 4096, ldr=9), "residual"), (dict(y=P), "overlaps x"), (dict(y=P + 32 * 3 + 28), "overlaps x"), (dict(x=P + 4096, ldx=16), "overlaps x"), (dict(y=P + 64, ldx=32, ldy=32, ldw=4096), "overlaps w"), (dict(r=P + 4096 + 4), "overlaps residual"), (dict(z=P + 4096 + 16), "overlaps"), (dict(bias=P + 4096 + 8), "overlaps bias")):
        refused(L.bert_amd_linear(*{**ok, **change}.values()), word)
    assert L.bert_amd_linear_workspace(5, 4, 8, 8, 1) == -1
    for K in (100000, 100001):  # parts of k; copies in whole pieces
        need = L.bert_amd_linear_workspace(0, 40, 8, K, 1)
        assert need > 0
        for change in (dict(ws=NULL), dict(nws=need - 1), dict(ws=P + 8)):
            refused(L.bert_amd_linear(*{**ok, "M": 40, "K": K, "ldx": K, "ldw": K, "y": 64 * P, **change}.values()), "workspace")
    need = L.bert_amd_linear_workspace(0, 40, 8, 100000, 1)
    for change in (dict(x=P + 4), dict(ldw=100001)):  # asked for as aligned, given otherwise
        refused(L.bert_amd_linear(*{**ok, "M": 40, "K": 100000, "ldx": 100000, "ldw": 100000, "y": 64 * P, "nws": need, **change}.values()), "workspace")
    assert L.bert_amd_linear(*{**ok, "M": 0, "x": NULL}.values()) == 0

    ok = dict(device=0, type=1, act=2, M=4, N=8, K=8, dy=P, lddy=8, z=P, ldz=8, x=P, ldx=8, w=P, ldw=8, dx=P + 4096, lddx=8, dw=P + 8192, lddw=8, db=P + 16384, ws=2 * P, nws=big, s=NULL)
    for change, word in ((dict(type=3), "type"), (dict(act=9), "activation"), (dict(M=-1), "size"), (dict(dy=NULL), "dy"), (dict(dy=P + 1), "dy"), (dict(z=NULL), "z"), (dict(ldz=4), "z"), (dict(x=NULL), "x"), (dict(w=NULL), "w"), (dict(lddx=0), "dx"), (dict(lddw=7), "dw"), (dict(db=P + 2), "dbias"), (dict(ws=NULL), "workspace"), (dict(nws=1), "workspace"), (dict(dx=P), "overlaps"), (dict(dw=P + 4096 + 16), "overlaps"), (dict(db=P + 8192 + 64), "overlaps"), (dict(db=P + 16), "overlaps")):
        refused(L.bert_amd_linear_backward(*{**ok, **change}.values()), word)
    assert L.bert_amd_linear_backward(*{**ok, "dx": NULL, "dw": NULL, "db": NULL}.values()) == 0
    assert L.bert_amd_linear_backward_workspace(1, 2, -1, 8, 8, 1) == -1

    ok = dict(device=0, type=2, out=0, n=4, V=10, E=64, table=P, ld=36, ids=P, scale=1.0, o=P + 4096, ldo=64, s=NULL)
    for change, word in ((dict(type=8), "types"), (dict(out=2), "types"), (dict(n=-1), "size"), (dict(V=0), "size"), (dict(E=0), "size"), (dict(E=40), "size"), (dict(table=NULL), "table"), (dict(table=P + 1), "table"), (dict(ld=35), "table"), (dict(ld=37), "table"), (dict(ids=NULL), "ids"), (dict(ids=P + 2), "ids"), (dict(o=NULL), "out"), (dict(ldo=63), "out"), (dict(ldo=0), "out"), (dict(o=P + 352), "overlaps"), (dict(table=2 * P, o=P + 8), "overlaps")):
        refused(L.bert_amd_lookup(*{**ok, **change}.values()), word)
    assert L.bert_amd_lookup(*{**ok, "n": 0, "ids": NULL}.values()) == 0

    ok = dict(device=0, type=0, n=4, V=10, E=8, dout=P, ldd=8, ids=P, scale=1.0, pad=-1, acc=0, dt=P + 4096, ldt=8, ws=2 * P, nws=big, s=NULL)
    for change, word in ((dict(type=2), "type"), (dict(n=-1), "size"), (dict(n=(1 << 28) + 1), "size"), (dict(V=0), "size"), (dict(E=0), "size"), (dict(dout=NULL), "dout"), (dict(ldd=7), "dout"), (dict(ids=NULL), "ids"), (dict(dt=NULL), "dtable"), (dict(ldt=7), "dtable"), (dict(n=5000, ws=NULL, dt=3 * P), "workspace"), (dict(n=5000, nws=16, dt=3 * P), "workspace"), (dict(n=5000, ws=2 * P + 8, dt=3 * P), "workspace"), (dict(dt=P + 64), "overlaps"), (dict(dout=2 * P, dt=P + 12), "overlaps"), (dict(E=1 << 20, ldd=1 << 20, ldt=1 << 20), "size")):
        refused(L.bert_amd_lookup_grad(*{**ok, **change}.values()), word)
    assert L.bert_amd_lookup_grad_workspace(-1, 10, 8) == -1

    row = np.zeros(2, bertops.AdamW._ROW)
    for i, k in enumerate(("p", "g", "m", "v", "ms", "vs")):
        row[k] = [(2 + i) * P, (2 + i) * P + (1 << 16)]
    row["n"] = 100

    def adamw(rows=row, n=2, bits=32, grad=0, copy=30, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, step=1, scale=NULL):
        return L.bert_amd_adamw(0, n, rows.ctypes.data if rows is not None else NULL, bits, grad, copy, lr, b1, b2, eps, step, 0, scale, NULL)

    nan = float("nan")
    for change, word in ((dict(rows=None), "tensors"), (dict(n=-1), "tensors"), (dict(bits=16), "bits"), (dict(grad=2), "type"), (dict(lr=-1.0), "lr"), (dict(lr=nan), "lr"), (dict(b1=1.0), "beta"), (dict(b2=-0.1), "beta"), (dict(b2=nan), "beta"), (dict(eps=0.0), "eps"), (dict(eps=1e-60), "eps"), (dict(step=0), "step"), (dict(scale=P + 1), "grad_scale")):
        refused(adamw(**change), word)

    def with_(**kw):
        r = row.copy()
        for k, v in kw.items():
            r[k][1] = v
        return r

    for kw, word in ((dict(n=-1), "size"), (dict(n=(1 << 34) + 1), "size"), (dict(decay=nan), "decay"), (dict(decay=-1.0), "decay"), (dict(p=0), "pointer"), (dict(g=0), "pointer"), (dict(m=P + 2), "pointer"), (dict(copy=P + 1), "copy"), (dict(p=2 * P + 396), "share"), (dict(m=5 * P + 8), "share"), (dict(v=5 * P), "share"), (dict(g=2 * P + 100), "share"), (dict(g=4 * P - 396), "share"), (dict(copy=3 * P - 200 + 400, g=3 * P), "share")):
        refused(adamw(with_(**kw)), word)
    refused(adamw(with_(copy=P), copy=0), "copies")
    refused(adamw(with_(ms=0), bits=8), "pointer")
    assert adamw(n=0) == 0
    same = row.copy()  # in any order, one gradient for both: nothing is wrong, and only the missing GPU can refuse it
    same["p"][1], same["g"][1], same["m"][1] = 2 * P - 4000, 3 * P, 4 * P - 400
    if not torch.cuda.is_available():
        assert adamw(same) == -3 and adamw(row) == -3
    refused(L.bert_amd_adamw_moments(0, -1, P, P, P, P, P, P, NULL), "size")
    refused(L.bert_amd_adamw_moments(0, 4, NULL, P, P, P, P, P, NULL), "pointer")
    out = [ctypes.c_void_p()] + [ctypes.c_int32() for _ in range(4)]
    refused(L.bert_amd_word_table(None, 0, *(ctypes.byref(t) for t in out)), "invalid")


def test_workspace_sizes():
    """Bytes for every size, zero rows among them."""
    L = bertlib.lib()
    for t in (0, 1, 30):
        for N, K in ((1, 1), (384, 384), (31, 4097), ((1 << 22) - 1, 4)):
            for M in (0, 1, 63, 64, 1000, 4096):
                assert 0 <= L.bert_amd_linear_workspace(t, M, N, K, 1) <= L.bert_amd_linear_workspace(t, M, N, K, 0)
                for act in (0, 2):
                    least = M * N * (4 if t == 0 else 2) if act else 0
                    assert least <= L.bert_amd_linear_backward_workspace(t, act, M, N, K, 1) <= L.bert_amd_linear_backward_workspace(t, act, M, N, K, 0)
    for n in (0, 1, 4096, 4097, 1 << 28):
        for V in (1, 511, 512, 1 << 30):
            assert L.bert_amd_lookup_grad_workspace(n, V, 8) >= 0


def test_refusals_of_shared_workspace():
    """A workspace that lies in what a call reads or writes, and moments that are written over each other."""
    L, P, NULL = bertlib.lib(), 1 << 24, None

    def refused(rc, word):
        assert rc == -1 and word in bertlib.last_error(), (rc, bertlib.last_error())

    K = 100000  # parts of k
    ok = dict(device=0, type=0, act=0, M=40, N=8, K=K, x=P, ldx=K, w=3 * P, ldw=K, bias=5 * P, r=6 * P, ldr=8, y=7 * P, ldy=8, z=8 * P, ldz=8, ws=9 * P, nws=P, s=NULL)
    need = L.bert_amd_linear_workspace(0, 40, 8, K, 1)
    for ws, word in ((P, "overlaps x"), (P + 16 * K - 16, "overlaps x"), (3 * P - need + 16, "overlaps w"), (5 * P + 16, "overlaps bias"), (6 * P, "overlaps residual"), (7 * P + 1264, "overlaps y"), (8 * P - need + 16, "overlaps z")):
        refused(L.bert_amd_linear(*{**ok, "ws": ws}.values()), word)
    ok = dict(device=0, type=1, act=2, M=40, N=8, K=8, dy=P, lddy=8, z=2 * P, ldz=8, x=3 * P, ldx=8, w=4 * P, ldw=8, dx=5 * P, lddx=8, dw=6 * P, lddw=8, db=7 * P, ws=8 * P, nws=P, s=NULL)
    for i, word in enumerate(("dy", "z", "x", "w", "dx", "dw", "dbias"), 1):
        refused(L.bert_amd_linear_backward(*{**ok, "ws": i * P + 16}.values()), "overlaps " + word)
    ok = dict(device=0, type=0, n=5000, V=10, E=8, dout=P, ldd=8, ids=2 * P, scale=1.0, pad=-1, acc=0, dt=3 * P, ldt=8, ws=4 * P, nws=P, s=NULL)
    for i in (1, 2, 3):
        refused(L.bert_amd_lookup_grad(*{**ok, "ws": i * P + 16}.values()), "workspace overlaps")
    for m_out, v_out, word in ((P, 6 * P, "m_out overlaps m"), (6 * P, 3 * P + 96, "v_out overlaps v"), (2 * P, 6 * P, "m_out overlaps m_scale"), (6 * P, P, "v_out overlaps m"), (6 * P, 6 * P + 396, "overlaps v_out")):
        refused(L.bert_amd_adamw_moments(0, 100, P, 2 * P, 3 * P, 4 * P, m_out, v_out, NULL), word)


def test_workspace_of_wide_layers():
    """A layer so wide that one pass over its columns fills the chip: the bias gradient's sums have their room."""
    L = bertlib.lib()
    M, N = 1025, 600000  # parts of k take at most 64 M 4 floats here
    assert L.bert_amd_linear_backward_workspace(0, 0, M, N, 4, 1) >= 4 * N > 4 * 64 * M * 4


@gpu
def test_wide_layer_backward():
    """More columns than 2048 workgroups take; small integers, so that every f32 sum is exact in any order."""
    M, N, K = 1100, 530000, 4
    g = torch.Generator(device="cuda").manual_seed(21)
    dy, x, w = (torch.randint(-2, 3, shape, generator=g, device="cuda").float() for shape in ((M, N), (M, K), (N, K)))
    for act in ("none", "relu"):
        dx, dw, db = bertops.linear_backward(dy, x, w, z=dy, act=act)
        dz = dy.relu() if act == "relu" else dy
        assert torch.equal(db, dz.sum(0)) and torch.equal(dw, dz.t() @ x) and torch.equal(dx, dz @ w)


def test_refusals_on_tensors():
    """bertops refuses tensors of the wrong kind before it calls the library."""
    x = torch.zeros(4, 8)
    for call in (lambda: bertops.linear(x, x), lambda: bertops.linear_backward(x, x, x), lambda: bertops.lookup(x, torch.zeros(3, dtype=torch.int32)),
                 lambda: bertops.lookup_grad(x, torch.zeros(4, dtype=torch.int32), 5), lambda: bertops.AdamW([x]), lambda: bertops.AdamW([]),
                 lambda: bertops._act("swish"), lambda: bertops._matrix("m", x.t(), torch.float32, x.device, 8, 4),
                 lambda: bertops._matrix("m", x, torch.float16, x.device, 4, 8), lambda: bertops._matrix("m", x, torch.float32, x.device, 4, 7),
                 lambda: bertops._ids(torch.zeros(3, dtype=torch.int64), x.device), lambda: bertops._ids(torch.zeros(6, dtype=torch.int32)[::2], x.device)):
        with pytest.raises(ValueError):
            call()


@gpu
def test_columns_of_one_matrix():
    """Inputs and outputs side by side in one wider matrix do not overlap; shifted into each other they are refused."""
    x, w, r, b = make_layer(50, 64, 64, torch.float32, seed=20)
    wide = torch.zeros(50, 192, device="cuda")
    wide[:, :64], wide[:, 64:128] = x.cuda(), r.cuda()
    bertops.linear(wide[:, :64], w.cuda(), b.cuda(), residual=wide[:, 64:128], act="gelu", out=wide[:, 128:])
    check_linear(x, w, b, r, "gelu", wide[:, 128:])
    assert torch.equal(wide[:, :64].cpu(), x) and torch.equal(wide[:, 64:128].cpu(), r)
    for out in (wide[:, :64], wide[:, 32:96], wide[1:, :64]):
        with pytest.raises(ValueError):
            bertops.linear(wide[: len(out), :64], w.cuda(), out=out)


@gpu
def test_refusals_on_the_gpu():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    z = torch.zeros(4, 6, device="cuda")
    for call in (lambda: bertops.linear(x, w[:, :7]), lambda: bertops.linear(x, w.half()), lambda: bertops.linear(x.int(), w), lambda: bertops.linear(x, w, torch.zeros(6)),
                 lambda: bertops.linear(x, w, torch.zeros(6, device="cuda").half()), lambda: bertops.linear(x, w, residual=x), lambda: bertops.linear(x, w, out=torch.zeros(1, 6, device="cuda").expand(4, 6)),
                 lambda: bertops.linear(x, w, act="swish"), lambda: bertops.linear(x.t(), w[:, :4]), lambda: bertops.linear_backward(z, x, w, act="gelu"),
                 lambda: bertops.lookup(w, torch.zeros(2, dtype=torch.int64, device="cuda")), lambda: bertops.lookup(w, torch.zeros(2, dtype=torch.int32)),
                 lambda: bertops.lookup(w, torch.zeros(2, dtype=torch.int32, device="cuda"), table_type="q4_0"), lambda: bertops.lookup(w, torch.zeros(2, dtype=torch.int32, device="cuda"), table_type="f16"),
                 lambda: bertops.lookup_grad(x, torch.zeros(3, dtype=torch.int32, device="cuda"), 5), lambda: bertops.lookup_grad(x, torch.zeros(4, dtype=torch.int32, device="cuda"), 5, accumulate=True),
                 lambda: bertops.lookup_grad(x, torch.zeros(4, dtype=torch.int32, device="cuda"), 0), lambda: bertops.AdamW([x.half()]), lambda: bertops.AdamW([x.t()]), lambda: bertops.AdamW([x], bits=16),
                 lambda: bertops.AdamW([x], copies=[x]), lambda: bertops.AdamW([x], weight_decay=[0.1, 0.1]), lambda: bertops.AdamW([x, x[1:]]).step([x, x[1:]]), lambda: bertops.AdamW([x]).step([w]),
                 lambda: bertops.AdamW([x]).step([x], torch.ones(2, device="cuda")), lambda: bertops.Adapter(4).step(), lambda: bertops.Adapter(4).backward(x)):
        with pytest.raises(ValueError):
            call()


# ---- the dense layer's bounds without room to spare


def rounded_between(v, off, dtype):
    """v rounded to `dtype` in 64 bits, and how far apart the roundings of v - off and v + off are."""
    lo, hi = ((v + s * off).to(dtype).to(F64) for s in (-1, 1))
    return v.to(dtype).to(F64), hi - lo


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N,pad", [(1, 40, 9000, 0), (5, 72, 8200, 3), (8, 8, 9001, 0), (9, 96, 130, 0), (12, 1000, 48, 1), (40, 384, 384, 0), (63, 130, 257, 8), (64, 512, 64, 0), (700, 256, 512, 0), (9, 64, 64, 0), (64, 64, 64, 0), (1065, 20, 11, 5), (9, 455, 300, 0), (130, 31, 132, 0), (131, 33, 124, 1), (20000, 8, 12, 0), (3000, 1, 4096, 0), (4000, 3, 1366, 0), (11, 605, 11, 0), (64, 2056, 64, 0), (64, 300, 65, 0)])
def test_linear_backward_rounds_dz_once(M, K, N, pad, dtype):
    """Past 8 rows or 8192 columns: dz rounded to the layer's type (f32 and where dz, dx or dw has few elements: not
    at all), and from there on nothing is lost but sums in f32 and each result's own rounding.  f32 operands are taken whole."""
    dt = DTYPES[dtype]
    x, w, dy, _ = make_layer(M, K, N, dt, seed=30)
    z = normal(gen(31), M, N).to(dt)
    dev = (lambda t: strided(t.cuda(), pad)) if pad else (lambda t: t.cuda())
    for act in bertops.ACTS:
        dx, dw, db = bertops.linear_backward(dev(dy), dev(x), dev(w), z=dev(z), act=act)
        at = z.to(F64).clone().requires_grad_(True)
        (dz,) = torch.autograd.grad(act64(at, act), at, dy.to(F64))
        off = SLACK * U32 * (1 + z.to(F64).abs()) * dy.to(F64).abs() * (act != "none")
        kept, apart = rounded_between(dz, off, dt)
        if dt == torch.float32:
            kept, apart = dz, off
        elif act != "none" and min(M * N, M * K, N * K) <= 4096:  # two halves: the second is what the first left, rounded
            kept, apart = dz, off + 2 * u(dt) ** 2 * dz.abs() + tiny(dt)
        for got, a, o, b, n, what in ((dx, kept, apart, w, N, "dx"), (dw, kept.t(), apart.t(), x, M, "dw")):
            want, far = a @ b.to(F64), (o + (n + 1) * U32 * (a.abs() + o)) @ b.to(F64).abs()
            close(got, want, far + u(dt) * (want.abs() + far) + tiny(dt), f"{what} {act}")
        close(db, dz.sum(0), off.sum(0) + (M + 1) * U32 * (dz.abs() + off).sum(0), f"db {act}")


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 1000, 300), (8, 384, 384), (9, 130, 70), (300, 384, 384), (1030, 520, 260)])
def test_linear_f32_operands_are_taken_whole(M, K, N):
    """f32 sums: at most K + 2 roundings of the terms' magnitudes, none for the operands."""
    x, w, _, b = make_layer(M, K, N, torch.float32, seed=32)
    y = bertops.linear(x.cuda(), w.cuda(), b.cuda())
    terms = x.to(F64).abs() @ w.to(F64).abs().t() + b.to(F64).abs()
    close(y, x.to(F64) @ w.to(F64).t() + b.to(F64), (K + 2) * U32 * terms, "y")


# ---- errors of the device


def every_operator():
    """One small call of each operator, as functions without arguments."""
    g = gen(40)
    x, w, table = normal(g, 20, 64).float().cuda(), normal(g, 48, 64).float().cuda(), normal(g, 30, 48).float().cuda()
    dy = normal(g, 20, 48).float().cuda()
    ids, many = torch.arange(20, dtype=torch.int32, device="cuda"), torch.arange(6000, dtype=torch.int32, device="cuda") % 30
    rows = table[many.long()]
    opt = bertops.AdamW([table.clone(), w.clone()], bits=8)
    return [lambda: bertops.linear(x, w), lambda: bertops.linear(x[:1], w), lambda: bertops.linear(x[:, :63], w[:, :63]),
            lambda: bertops.linear_backward(dy, x, w, z=dy, act="gelu"), lambda: bertops.linear_backward(dy[:2], x[:2], w),
            lambda: bertops.lookup(table, ids), lambda: bertops.lookup_grad(dy, ids, 30),
            lambda: bertops.lookup_grad(rows, many, 30), lambda: opt.step([table, w]), opt.moments]


@gpu
def test_a_failed_call_leaves_no_error_behind():
    """A device that is not there: this call fails, the next ones, the library's and torch's, do not."""
    L, x = bertlib.lib(), torch.ones(4, 8, device="cuda")
    y = torch.empty(4, 4, device="cuda")
    for call in every_operator():
        rc = L.bert_amd_linear(torch.cuda.device_count() + 5, 0, 0, 4, 4, 8, x.data_ptr(), 8, x.data_ptr(), 8, None, None, 0, y.data_ptr(), 4, None, 4, None, 0, None)
        assert rc == -3 and bertlib.last_error()
        call()
        (x + 1).sum().item()


@gpu
def test_an_error_of_an_earlier_call_is_not_the_operators():
    """An error that another HIP call of this thread left and nobody took: the operators run and say so."""
    with open("/proc/self/maps") as f:
        runtimes = [ctypes.CDLL(p) for p in sorted({line.split()[-1] for line in f if "libamdhip64" in line})]
    calls = every_operator()
    for call in calls:
        call()  # memory from torch's cache from here on
    torch.cuda.synchronize()
    assert runtimes
    for call in calls:
        for r in runtimes:
            assert r.hipSetDevice(1000) != 0
        try:
            call()
        finally:
            for r in runtimes:
                r.hipGetLastError()
    torch.cuda.synchronize()


@gpu
def test_adamw_refuses_after_a_failed_step(monkeypatch):
    """A step that the device failed may have moved some tensors: no second one over them.  A refused one moved none."""
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = bertops.AdamW([p])
    opt.lr = -1.0
    with pytest.raises(ValueError):
        opt.step([g])
    opt.lr = 1e-3
    opt.step([g])
    real = bertlib.lib()

    class Failing:
        def __getattr__(self, name):
            return (lambda *a: -3) if name == "bert_amd_adamw" else getattr(real, name)

    monkeypatch.setattr(bertlib, "lib", lambda: Failing())
    with pytest.raises(RuntimeError):
        opt.step([g])
    monkeypatch.undo()
    before = p.clone()
    with pytest.raises(RuntimeError, match="undefined"):
        opt.step([g])
    torch.cuda.synchronize()
    assert opt.t == 1 and torch.equal(p, before)


# ---- frequent tokens among few places


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 63, 513, 2000, 4096])
@pytest.mark.parametrize("E", [1, 65, 129, 260, 1023, 2052])
def test_lookup_grad_frequent_tokens(n, E, dtype):
    """Tokens with fewer and with more places than a row has slices of columns, up to every place the same one."""
    g = gen(50)
    dout = normal(g, n, E).to(DTYPES[dtype])
    D = dout.cuda()
    for V, ids in ((3, torch.zeros(n)), (70, torch.full((n,), 69)), (40, torch.rand(n, generator=g) ** 6 * 40), (9, torch.where(torch.arange(n) % 3 == 0, -1, 4))):
        ids = ids.to(torch.int32)
        out = torch.full((V, E), float("nan"), device="cuda")
        got = bertops.lookup_grad(D, ids.cuda(), V, scale=0.5, out=out)
        check_grad(got, dout, ids, V, 0.5, -1)
        assert torch.equal(got, bertops.lookup_grad(D, ids.cuda(), V, scale=0.5))
        base = normal(g, V, E).float()
        check_grad(bertops.lookup_grad(D, ids.cuda(), V, out=base.cuda(), accumulate=True), dout, ids, V, 1.0, -1, base)


@gpu
def test_lookup_grad_of_one_token_is_spread():
    """All places one token: with 4096 of them, which are not sorted, not ten times as long as with one more, which are."""
    def time_of(n, E=1023):
        dout, ids, out = torch.ones(n, E, device="cuda"), torch.full((n,), 7, dtype=torch.int32, device="cuda"), torch.empty(100, E, device="cuda")
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        for k in range(12):
            if k == 2:
                start.record()
            bertops.lookup_grad(dout, ids, 100, out=out)
        end.record()
        end.synchronize()
        return start.elapsed_time(end)

    assert min(time_of(4096) for _ in range(3)) < 10 * min(time_of(4097) for _ in range(3))


# ---- the two ways over a layer's dz


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(1024, 2048), (1024, 2049), (1023, 2056), (517, 4104), (64, 33000), (16, 131080), (9, 240001)])
def test_backward_dz_forms(M, N, dtype):
    """Up to 1024 rows, with as many and with more columns than the narrow form takes."""
    dt, K = DTYPES[dtype], 8
    x, w, dy, _ = make_layer(M, K, N, dt, seed=60)
    z = normal(gen(61), M, N).to(dt)
    dx, dw, db = bertops.linear_backward(dy.cuda(), x.cuda(), w.cuda(), z=z.cuda(), act="relu")  # its dz needs no rounding
    dz = torch.where(z > 0, dy, torch.zeros_like(dy)).to(F64)
    for got, a, b, n, what in ((dx, dz, w, N, "dx"), (dw, dz.t(), x, M, "dw")):
        far = (n + 1) * U32 * (a.abs() @ b.to(F64).abs())
        want = a @ b.to(F64)
        close(got, want, far + u(dt) * (want.abs() + far) + tiny(dt), what)
    close(db, dz.sum(0), (M + 1) * U32 * dz.abs().sum(0), "db")
    (alone,) = (t for t in bertops.linear_backward(dy.cuda(), x.cuda(), w.cuda(), z=z.cuda(), act="relu", need=(False, False, True)) if t is not None)
    assert torch.equal(alone, db)


@gpu
def test_backward_of_wide_layers_takes_whole_lines():
    """A wide layer's bias gradient over 1000 rows takes no more than twice the time of 1040."""
    def time_of(M, N=65536):
        x, w, dy = (torch.ones(*s, device="cuda").bfloat16() for s in ((M, 8), (N, 8), (M, N)))
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        for k in range(12):
            if k == 2:
                start.record()
            bertops.linear_backward(dy, x, w, z=dy, act="gelu", need=(False, False, True))
        end.record()
        end.synchronize()
        return start.elapsed_time(end)

    assert min(time_of(1000) for _ in range(4)) < 2 * min(time_of(1040) for _ in range(4))


# ---- what Adapter and TokenTable keep between their calls


class FewRows:
    """A model's word rows as bert_amd_word_table gives them, without a model."""

    def __init__(self, rows):
        self.rows = rows

    def word_table(self, slot=0):
        return self.rows.data_ptr(), 0, *self.rows.shape, self.rows.device.index


def token_table(V=20, E=32, **kw):
    return bertops.TokenTable(FewRows(normal(gen(70), V, E).float().cuda()), pad_id=-1, **kw)


@gpu
def test_trained_layers_refuse_mixed_and_stale_backwards():
    """Two forwards before a backward, and a backward of weights that have moved since."""
    a, t = bertops.Adapter(32, lr=1e-2), token_table()
    e, f = (normal(gen(s), 6, 32).float().cuda() for s in (71, 72))
    i, j = torch.arange(6, dtype=torch.int32, device="cuda"), torch.arange(6, 12, dtype=torch.int32, device="cuda")
    for o, one, two, dy in ((a, e, f, e), (t, i, j, f)):
        with pytest.raises(ValueError, match="follows"):
            o.backward(dy)
        o.forward(one)
        o.forward(two)
        with pytest.raises(ValueError, match="two forwards"):
            o.backward(dy)
        with pytest.raises(ValueError, match="follows"):  # neither is meant from here on
            o.backward(dy)
        with pytest.raises(ValueError):
            o.step()
        o.forward(one)
        o.forward(two, train=False)
        o.backward(dy)
        o.step()
        with pytest.raises(ValueError, match="follows"):
            o.backward(dy)
        o.forward(two)
        o.backward(dy)
        o.forward(one)
        o.step()
        with pytest.raises(ValueError, match="follows"):  # the weights that forward used are gone
            o.backward(dy)
        o.forward(one)
        o.backward(dy)
        o.step()
    assert a.opt.t == 3 and t.opt.t == 3


@gpu
def test_pairs_through_one_forward():
    """The two sides of a pair in one batch: the gradients of both against 64 bits."""
    a = bertops.Adapter(16, act="gelu_erf", lr=1e-2)
    a.w.copy_(normal(gen(73), 16, 16, std=0.2))
    e, dy = (normal(gen(s), 10, 16).float() for s in (74, 75))
    a.forward(e.cuda())
    de = a.backward(dy.cuda(), need_input=True)
    E, W, B = e.to(F64).requires_grad_(True), a.w.cpu().to(F64).requires_grad_(True), torch.zeros(16, dtype=F64, requires_grad=True)
    (act64(E @ W.t() + B, "gelu_erf") + E).backward(dy.to(F64))
    for got, want in (*zip(a._grads.use(), (W.grad, B.grad)), (de, E.grad)):
        close(got, want, 200 * U32 * want.abs().max() * torch.ones_like(want), "pair")  # f32 sums of at most 16 terms, each within some 2^-24


@gpu
def test_gradients_add_up_until_the_step():
    """Two forwards and backwards before one step: the sum of both gradients moves the weights, as TokenTable's does."""
    e, f = (normal(gen(s), 12, 24).float().cuda() for s in (76, 77))
    both, lone = bertops.Adapter(24, lr=1e-2), [bertops.Adapter(24, lr=1e-2) for _ in range(2)]
    for x, o in zip((e, f), lone):
        both.backward(both.forward(x) - 1.0)
        o.backward(o.forward(x) - 1.0)
    assert all(torch.equal(s, p + q) for s, p, q in zip(*(o._grads.use() for o in (both, *lone))))
    both.step()
    both.backward(both.forward(e) - 1.0)
    assert not torch.equal(both._grads.use()[0], lone[0]._grads.use()[0])  # a new sum of the moved weights
    table = token_table()
    rows = table.rows.clone()
    ids = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([3, 4, 3], [4, 4, 9])]
    dout = normal(gen(78), 3, 32).float().cuda()
    for i in ids:
        table.forward(i)
        table.backward(dout)
    want = sum(bertops.lookup_grad(dout, i, 20) for i in ids)
    assert torch.equal(table._grad.use()[0], want)
    table.step()
    opt = bertops.AdamW([rows])
    opt.step([want])
    assert torch.equal(table.rows, rows)


@gpu
def test_steps_on_another_stream():
    """Forward, backward and step on a stream each: what a call drops is not given out while another stream reads it."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()

    x = normal(gen(79), 64, 384).float().cuda()
    ids = torch.arange(64, dtype=torch.int32, device="cuda") % 20
    for made, inputs in ((lambda: bertops.Adapter(384, lr=1e-2), x), (lambda: token_table(E=384, lr=1e-2), ids)):
        here, there = made(), made()
        weights = lambda o: o.opt.params  # noqa: E731
        here.forward(inputs)
        here.backward(x)
        here.backward(x)
        here.step()
        s0, s1, s2 = (torch.cuda.Stream() for _ in range(3))

        def given_out(stream, like, taken):
            with torch.cuda.stream(stream):
                new = [span(torch.empty_like(t)) for t in like]
            return any(a < d and c < b for a, b in new for c, d in taken)

        s0.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s0):
            there.forward(inputs.clone())
        s1.wait_stream(s0)
        with torch.cuda.stream(s1):
            torch.cuda._sleep(50_000_000)  # the backward is not done when what it reads is dropped
            there.backward(x)
            there.backward(x)
        kept = [span(t) for t in there._kept._what._tensors]
        there._kept.drop()
        assert not given_out(s0, [inputs, x], kept)
        grads = there._grads if hasattr(there, "_grads") else there._grad
        sums = [span(t) for t in grads._tensors]
        del grads
        s2.wait_stream(s1)
        with torch.cuda.stream(s2):
            torch.cuda._sleep(50_000_000)
            there.step()
        s1.synchronize()
        assert not given_out(s1, weights(there), sums)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(weights(here), weights(there)))


# ---- beside torch's autograd


@gpu
def test_written_tensors_count_as_changed():
    """A graph that saved a weight, a copy or an output notices that an operator has written it since."""
    def stale(t, change):
        w = torch.ones_like(t, requires_grad=True)
        y = (w * t).sum()  # saves t
        change()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()

    p = torch.nn.Parameter(torch.ones(8, 8, device="cuda"))
    copy = p.detach().bfloat16()
    opt = bertops.AdamW([p], copies=[copy])
    for t in (p, copy):
        stale(t, lambda: opt.step([torch.ones(8, 8, device="cuda")]))
    x, out = torch.ones(8, 8, device="cuda"), torch.ones(8, 8, device="cuda")
    stale(out, lambda: bertops.linear(x, x, out=out))
    ids = torch.zeros(8, dtype=torch.int32, device="cuda")
    stale(out, lambda: bertops.lookup_grad(x, ids, 8, out=out))
    opt.lr = -1.0
    w = torch.ones(8, 8, device="cuda", requires_grad=True)
    y = (w * p).sum()
    with pytest.raises(ValueError):
        opt.step([x])
    y.backward()  # a refused step has written nothing
    with torch.inference_mode():
        bertops.linear(x, x, out=torch.ones(8, 8, device="cuda"))


@gpu
def test_lost_gradients_are_said():
    """linear and lookup of tensors that require a gradient warn, but not where a wrapper takes care of it."""
    import warnings

    x, w, b = (torch.ones(*s, device="cuda") for s in ((4, 8), (6, 8), (6,)))
    r, ids = torch.ones(4, 6, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")

    class Layer(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, b):
            y, z = bertops.linear(x, w, b, act="tanh", save_z=True)
            ctx.save_for_backward(x, w, z)
            return y

        @staticmethod
        def backward(ctx, dy):
            x, w, z = ctx.saved_tensors
            return bertops.linear_backward(dy.contiguous(), x, w, z=z, act="tanh")  # a sum hands a broadcast one back

    for t in (x, w, b, r):
        t.requires_grad_(True)
        with pytest.warns(UserWarning, match="requires a gradient"):
            y = bertops.linear(x, w, b, residual=r)
        assert not y.requires_grad
        t.requires_grad_(False)
    w.requires_grad_(True)
    with pytest.warns(UserWarning, match="requires a gradient"):
        bertops.lookup(w, ids)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with torch.no_grad():
            bertops.linear(x, w, b)
            bertops.lookup(w, ids)
        bertops.linear(x, w.detach(), b)
        y = Layer.apply(x, w, b)
        y.sum().backward()
    want = torch.tanh(x @ w.detach().t() + b)
    slope = (1 - want.to(F64) ** 2).cpu()
    # eight ones and a bias of one: z is 9 exactly, and 1 - tanh(9)^2 is off by some 2^-24 of 1
    close(w.grad, slope.t() @ x.cpu().to(F64), 4 * SLACK * U32 * torch.ones(6, 8, dtype=F64), "dw")


# ---- sizes past 32 bits


def test_sizes_in_32_bits():
    for ok in (0, -1, 2**31 - 1, -(2**31)):
        bertops._int32("n", ok)
    for bad in (2**31, 2**32 + 5, -(2**31) - 1):
        with pytest.raises(ValueError, match="32 bits"):
            bertops._int32("n", 3, bad)


@gpu
def test_sizes_past_32_bits_are_refused():
    """Widths, rows and padding tokens whose low 32 bits would name others."""
    long = torch.empty(1, 2**32 + 8, dtype=torch.float16, device="cuda")
    ids, dout = torch.arange(6, dtype=torch.int32, device="cuda"), torch.ones(6, 1, device="cuda")
    one = torch.ones(1, 1, dtype=torch.float16, device="cuda")
    tall = long.view(-1, 1)
    for call in (lambda: bertops.linear(long, long), lambda: bertops.linear_backward(one, long, long),
                 lambda: bertops.linear(one, tall), lambda: bertops.lookup(tall, ids), lambda: bertops.lookup(long, ids),
                 lambda: bertops.lookup_grad(dout, ids, 2**32 + 8), lambda: bertops.lookup_grad(dout, ids, 6, pad_id=2**32 + 5)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    assert bertops.lookup_grad(dout, ids, 6, pad_id=5)[:, 0].tolist() == [1.0] * 5 + [0.0]
    assert bertops.lookup_grad(dout, ids, 6, pad_id=-(2**31))[:, 0].tolist() == [1.0] * 6


def test_hand_written_m0_is_named_as_overwritten():
    """Every asm statement of the kernels that writes M0 says so to the compiler."""
    import glob
    import re

    found = 0
    for path in glob.glob(os.path.join(os.path.dirname(bertops.__file__), "csrc", "*.h*")):
        with open(path) as f:
            for statement in re.findall(r"\basm\b[^;]*;", f.read()):
                if re.search(r"s_mov_b32\s+m0", statement):
                    found += 1
                    assert statement.rsplit(":", 1)[1].count('"m0"') == 1, (path, statement)
    assert found


# ---- the activations of 16-bit layers


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act", bertops.ACTS)
@pytest.mark.parametrize("K,N", [(1, 1), (8, 64)])
def test_activations_far_out_in_16_bits(act, dtype, K, N):
    """Every activation over its whole range, down to the type's smallest values: in tiles, inside and at an edge, and few rows."""
    dt = DTYPES[dtype]
    z = torch.cat([torch.linspace(-110, 40, 4076, dtype=F64), torch.tensor([-6e4, -300, 0.0, 1e-4, -1e-4, 300, 6e4, 3e4], dtype=F64), torch.linspace(-12, -4, 12, dtype=F64)]).to(dt)
    x, w = torch.zeros(len(z), K, dtype=dt), torch.zeros(N, K, dtype=dt)
    x[:, 0], w[:, 0] = z, 1.0
    d = z.to(F64)
    want = act64(d, act)
    steep = 1 + (2 * d.abs() ** 3).clamp(max=2400) if act == "gelu" else 1 + d.abs().clamp(max=200) ** (2 if act == "gelu_erf" else 1)
    off = SLACK * U32 * steep * want.abs()
    # off by half a step, and as much again where f32's own smallest values round next to the type's
    tol = off + u(dt) * (want.abs() + off) + 2 * tiny(dt)
    for rows in (slice(None), slice(4080, 4088), slice(0, 8), slice(1500, 1508)):
        y = bertops.linear(x[rows].cuda(), w.cuda(), act=act)
        assert N == 1 or torch.equal(y, y[:, :1].expand_as(y))
        close(y[:, 0], want[rows], tol[rows], f"{act} {rows}")


# ---- 8-bit states: no drift


SIZES_IN_A_BLOCK = np.logspace(-3, 0, 256).astype(np.float32)  # many magnitudes beside the peak, none under the lowest octave
DRIFT_STEPS, DRIFT_BLOCKS = 40, 4096
# A code is at most 2^-3 (m) or 2^-4 (r = sqrt v) of its value from the next one, and rounding between two at random
# varies by at most half of that.  m forgets at 0.9 a step: its standard deviation is at most 2^-4 / sqrt(1 - 0.81), the
# blocks' mean's by sqrt(blocks) less.  v grows evenly, so that step s of T is left in r with weight s / T:
# 2^-5 sqrt(T / 3); and r^2 is on average larger than the square of r's mean by the variance, in all at most
# 2^-10 T / 2 of v, half of it in r.  Five deviations.
M_LIMIT = 5 * 2.0**-4 / (1 - 0.81) ** 0.5 / DRIFT_BLOCKS**0.5
R_LIMIT = 5 * 2.0**-5 * (DRIFT_STEPS / 3) ** 0.5 / DRIFT_BLOCKS**0.5 + 2.0**-10 * DRIFT_STEPS / 4


def drift(m, v):
    """How far the blocks' means of m and v are from what constant gradients give, at worst, as parts of it."""
    g = SIZES_IN_A_BLOCK.astype(np.float64)
    want_m, want_r = g * (1 - 0.9**DRIFT_STEPS), g * (1 - 0.999**DRIFT_STEPS) ** 0.5
    m, v = (np.asarray(x, np.float64).reshape(-1, 256).mean(0) for x in (m, v))
    return abs(m / want_m - 1).max(), abs(np.sqrt(v) / want_r - 1).max()


def test_drift_limits_tell_other_roundings():
    """Rounding to the nearest code, up or down, the same in every block, is over both limits."""
    f, g = np.float32, SIZES_IN_A_BLOCK
    for bits in (0x80000000, 0xFFFFFFFF, 0):
        h = np.full(256, bits, np.uint32)
        m, v = np.zeros(256, f), np.zeros(256, f)
        for _ in range(DRIFT_STEPS):
            m, v = m * f(0.9) + g * f(0.1), v * f(0.999) + (g * f(1 - 0.999)) * g
            c, s = encode(m, 3, h)
            m = code_values(3)[c] * s[0]
            c, s = encode(np.sqrt(v), 4, h)
            v = (code_values(4)[np.maximum(c, 1)] * s[0]) ** 2
        far_m, far_r = drift(m, v)
        assert far_m > 2 * M_LIMIT and far_r > 1.4 * R_LIMIT, (hex(bits), far_m, far_r)


@gpu
@pytest.mark.parametrize("seed", [1, 2**31])
def test_adamw_8_bit_states_have_no_drift(seed):
    """The same 256 magnitudes in every block: each place's stored moments average to the exact ones over the blocks."""
    g = torch.from_numpy(np.tile(SIZES_IN_A_BLOCK, DRIFT_BLOCKS)).cuda()
    opt = bertops.AdamW([torch.zeros_like(g)], bits=8, seed=seed)
    for _ in range(DRIFT_STEPS):
        opt.step([g])
    far_m, far_r = drift(*(x.cpu().numpy() for x in opt.moments()))
    assert far_m < M_LIMIT and far_r < R_LIMIT, (far_m, far_r)


# ---- outputs with rows further apart than their width, through the C entry points


def wider(rows, cols, pad, dtype):
    return strided(torch.zeros(rows, cols, dtype=dtype, device="cuda"), pad)


def gap_is_untouched(t):
    return bool(torch.isnan(t._base[:, t.shape[1]:]).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("M,K,N", [(1, 36, 20), (5, 264, 130), (8, 1000, 777), (20, 2000, 24), (70, 96, 130), (300, 384, 384), (1100, 130, 264)])
def test_strided_outputs(M, K, N, pad, dtype):
    """y, z, dx and dw into wider rows: the same bits as into contiguous ones, and nothing between the rows."""
    L, dt = bertlib.lib(), DTYPES[dtype]
    x, w, dy, b = (t.cuda() for t in make_layer(M, K, N, dt, seed=80))
    typ, stream = bertops.TYPES[dt], torch.cuda.current_stream().cuda_stream
    room = torch.empty(max(L.bert_amd_linear_workspace(typ, M, N, K, 0), L.bert_amd_linear_backward_workspace(typ, 2, M, N, K, 0), 16), dtype=torch.uint8, device="cuda")
    ws = (room.data_ptr(), room.numel())
    for act in ("none", "gelu", "tanh"):
        a = bertops.ACTS[act]
        want_y, want_z = bertops.linear(x, w, b, residual=dy, act=act, save_z=True)
        y, z = wider(M, N, pad, dt), wider(M, N, pad, dt)
        assert L.bert_amd_linear(0, typ, a, M, N, K, x.data_ptr(), K, w.data_ptr(), K, b.data_ptr(), dy.data_ptr(), N, y.data_ptr(), N + pad, z.data_ptr(), N + pad, *ws, stream) == 0
        want = bertops.linear_backward(dy, x, w, z=want_z, act=act)
        dx, dw, db = wider(M, K, pad, dt), wider(N, K, pad, dt), torch.empty(N, device="cuda")
        assert L.bert_amd_linear_backward(0, typ, a, M, N, K, dy.data_ptr(), N, z.data_ptr(), N + pad, x.data_ptr(), K, w.data_ptr(), K, dx.data_ptr(), K + pad, dw.data_ptr(), K + pad, db.data_ptr(), *ws, stream) == 0
        for got, expected in ((y, want_y), (z, want_z), (dx, want[0]), (dw, want[1])):
            assert torch.equal(got, expected) and gap_is_untouched(got), act
        assert torch.equal(db, want[2])


FIRST_GRADIENTS = """
import sys
sys.path[:0] = sys.argv[1:]
import torch, bertops
g = torch.Generator(device="cuda").manual_seed(90)
def normal(*s, t=torch.float32): return torch.randn(*s, generator=g, device="cuda").to(t)
layers = [(normal(M, K, t=t), normal(N, K, t=t), normal(M, N, t=t)) for M, K, N, t in
          ((1, 384, 384, torch.float32), (7, 130, 77, torch.bfloat16), (300, 384, 384, torch.float32), (200, 64, 96, torch.float16), (1000, 72, 2500, torch.bfloat16))]
ids = torch.randint(-1, 50, (900,), generator=g, device="cuda").int()
dout = normal(900, 1023)
into = normal(50, 1023)
def calls():
    out = []
    for x, w, dy in layers:
        out += bertops.linear(x, w, act="gelu_erf", save_z=True)
        out += bertops.linear_backward(dy, x, w, z=dy, act="silu")
    out += [bertops.lookup_grad(dout, ids, 50), bertops.lookup_grad(dout, ids, 50, out=into.clone(), accumulate=True)]
    out += [bertops.lookup(into, ids, scale=3.0, out_dtype=torch.float16)]
    return out
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls()
for k in range(4):
    graph.replay()
    want = calls()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want)), k
    for x, w, dy in layers:
        x.mul_(-0.75)
        dy.add_(0.25)
    ids.add_(1)
    into.mul_(0.5)
    torch.cuda.synchronize()
print("four replays")
"""


@gpu
def test_first_gradients_are_captured():
    """As test_first_calls_are_captured, for the gradients of few rows, of small layers in a pair and of wide ones, and few places."""
    done = subprocess.run([sys.executable, "-c", FIRST_GRADIENTS, os.path.dirname(bertops.__file__)], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "four replays" in done.stdout, done.stderr[-2000:]


@gpu
def test_f16_dz_past_its_largest_value():
    """dy next to f16's largest value times a slope over 1, in a layer small enough for halves: gradients are finite."""
    M, K, N = 40, 16, 24
    x, w, _, _ = make_layer(M, K, N, torch.float16, seed=95)
    dy, z = torch.full((M, N), 65504.0).half(), torch.full((M, N), 1.5).half()  # GELU's slope there is 1.13
    w, x = w / 64, x / 1024
    dx, dw, db = bertops.linear_backward(dy.cuda(), x.cuda(), w.cuda(), z=z.cuda(), act="gelu")
    at = z.to(F64).clone().requires_grad_(True)
    (dz,) = torch.autograd.grad(act64(at, "gelu"), at, dy.to(F64))
    assert (dz > 65520).all()
    far = dz * SLACK * U32 + 2 * u(torch.float16) ** 2 * dz
    for got, a, b, o in ((dx, dz, w, far), (dw, dz.t(), x, far.t())):
        want, o = a @ b.to(F64), (o + 50 * U32 * a) @ b.to(F64).abs()
        close(got, want, o + u(torch.float16) * (want.abs() + o) + tiny(torch.float16), "gradient")
    dy[0, 0] = float("inf")
    dx, dw, db = bertops.linear_backward(dy.cuda(), x.cuda(), w.cuda(), z=z.cuda(), act="gelu")
    assert not torch.isfinite(dx[0]).any() and torch.isfinite(dx[1:]).all() and not torch.isnan(db).any()


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(4096, 20000, 1), (1024, 20000, 4), (16, 30000, 256)])
def test_few_dz_of_wide_inputs(M, K, N, dtype):
    """dz of few elements in two halves where dx or dw is large: the large tiles go over k twice, too."""
    dt = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(96)
    x, w, dy, z = (torch.randn(*s, generator=g, device="cuda").to(dt) for s in ((M, K), (N, K), (M, N), (M, N)))
    dx, dw, db = bertops.linear_backward(dy, x, w, z=z, act="silu")
    zz = z.to(F64)
    s = torch.sigmoid(zz)
    dz = dy.to(F64) * (s + zz * s * (1 - s))
    off = SLACK * U32 * (1 + zz.abs()) * dy.to(F64).abs() + 2 * u(dt) ** 2 * dz.abs() + tiny(dt)
    for got, a, o, b, n in ((dx, dz, off, w.to(F64), N), (dw, dz.t().contiguous(), off.t().contiguous(), x.to(F64), M)):
        want, far = a @ b, (o + (n + 1) * U32 * (a.abs() + o)) @ b.abs()
        assert ((got.to(F64) - want).abs() <= far + u(dt) * (want.abs() + far) + tiny(dt)).all()


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "q4_0"])
def test_lookup_in_one_row(kind):
    """A table whose rows are the same one again, as every input's may be: 0 elements apart."""
    table, values = make_table(kind, 1, 96)
    ids = torch.tensor([0, 4, 5, -1], dtype=torch.int32)
    got = bertops.lookup(table.cuda().expand(5, -1), ids.cuda(), scale=2.0, table_type=kind, out_dtype=torch.float32).cpu()
    assert torch.equal(got, (values * 2.0).float().expand(4, 96) * torch.tensor([1.0, 1.0, 0.0, 0.0])[:, None])


def test_rows_of_a_table_that_are_one():
    """0 bytes between rows pass the library's checks; without a GPU only the device call refuses them."""
    L, P = bertlib.lib(), 1 << 20
    args = dict(device=0, type=2, out=0, n=4, V=10, E=64, table=P, ld=0, ids=P, scale=1.0, o=P + 4096, ldo=64, s=None)
    if not torch.cuda.is_available():
        assert L.bert_amd_lookup(*args.values()) == -3
    assert L.bert_amd_lookup(*{**args, "ld": -36}.values()) == -1
    assert L.bert_amd_lookup(*{**args, "o": P + 16}.values()) == -1


@gpu
def test_trained_layers_refuse_changed_inputs():
    """Embeddings or ids overwritten between forward and backward; fresh ones, and inference tensors, pass."""
    a, t = bertops.Adapter(32), token_table()
    e, dy = (normal(gen(s), 6, 32).float().cuda() for s in (97, 98))
    ids = torch.arange(6, dtype=torch.int32, device="cuda")
    for o, x in ((a, e), (t, ids)):
        o.forward(x)
        x.add_(1)
        with pytest.raises(ValueError, match="changed in place"):
            o.backward(dy)
        o.forward(x)
        o.backward(dy)
        o.step()
        with torch.inference_mode():
            o.forward(x.clone())
            o.backward(dy)
            o.step()

"""The operators around the encoder, as they are measured: a dense layer with its epilogue and its
gradients, the lookup of token rows with its gradient, and the AdamW step.

`run` computes one of them, in plain torch operations where `own` is false and through the library's
entry points (embedding.cpp_amd/bertops.py) where it is true.  Sizes are those of the encoders this
library evaluates (rows of 384, 768 or 1024, feed-forward widths 1536 and 4096, vocabularies of 30522
and 250002, sentences of 128 and 256 tokens) or generic ones.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ROW_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "q4_0": 18 / 32, "q4_1": 20 / 32}
ACTS = ("none", "relu", "gelu", "gelu_erf", "silu", "tanh")
LR, BETA1, BETA2, EPS = 1e-3, 0.9, 0.999, 1e-8
BLOCK = 256  # elements that share a scale in 8-bit states


def _ops():
    p = os.path.join(ROOT, "embedding.cpp_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import bertops

    return bertops


def listed():
    return [
        # one sentence's embedding through a trained adapter (the server's single request)
        dict(name="linear_one", op="linear", type="f32", M=1, K=384, N=384, act="tanh", residual=True, save_z=False, pad=0),
        # a ragged batch of pooled rows through a head of odd width, no dimension a multiple of anything
        dict(name="linear_odd", op="linear", type="f16", M=777, K=1001, N=513, act="silu", residual=False, save_z=False, pad=0),
        # the widest feed-forward layer's up projection over 256 x 128 tokens, its pre-activation kept for training
        dict(name="linear_up", op="linear", type="bf16", M=32768, K=1024, N=4096, act="gelu", residual=False, save_z=True, pad=0),
        # the small encoder's down projection with its residual over 512 x 128 tokens, in full precision
        dict(name="linear_down", op="linear", type="f32", M=65536, K=1536, N=384, act="none", residual=True, save_z=False, pad=0),
        # one training step's gradients of an adapter on a batch of 256 embeddings
        dict(name="linear_grad_adapter", op="linear_backward", type="f32", M=256, K=384, N=384, act="tanh", pad=0),
        # the gradients of the wide up projection over 128 x 128 tokens
        dict(name="linear_grad_up", op="linear_backward", type="bf16", M=16384, K=1024, N=4096, act="gelu", pad=0),
        # one sentence's rows out of the quantised word table
        dict(name="lookup_one", op="lookup", type="q4_0", out="f32", n=128, V=30522, E=384, scale=1.0),
        # 512 x 256 tokens out of the multilingual word table, scaled by sqrt(E)
        dict(name="lookup_batch", op="lookup", type="f16", out="f16", n=131072, V=250002, E=768, scale=math.sqrt(768.0)),
        # the word table's gradient for a small batch: nearly every row of it is zero
        dict(name="lookup_grad_small", op="lookup_grad", type="f32", n=2048, V=30522, E=384, scale=1.0, accumulate=False),
        # the multilingual table's gradient for 512 x 256 tokens
        dict(name="lookup_grad_batch", op="lookup_grad", type="bf16", n=131072, V=250002, E=768, scale=math.sqrt(768.0), accumulate=False),
        # every weight of the small encoder, states in 32 bits, and the bf16 copy that the products read
        dict(name="adamw_32", op="adamw", V=30522, E=384, I=1536, layers=6, grad="f32", bits=32, copy=True),
        # every weight of the multilingual base encoder, states in 8 bits, gradients in bf16
        dict(name="adamw_8", op="adamw", V=250002, E=768, I=2048, layers=12, grad="bf16", bits=8, copy=False),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("linear", "linear_backward", "lookup", "lookup_grad", "adamw"))
    if op in ("linear", "linear_backward"):
        K, N = log(8, 4096), log(8, 4096)
        if rng.random() < 0.6:  # most layers are multiples of 32 wide
            K, N = -(-K // 32) * 32, -(-N // 32) * 32
        M = max(1, min(log(1, 32768), int(6e10 / (K * N))))
        c = dict(op=op, type=rng.choice(("f32", "f16", "bf16")), M=M, K=K, N=N, act=rng.choice(ACTS), pad=rng.choice((0, 0, 0, 8, 5)))
        if op == "linear":
            c.update(residual=rng.random() < 0.5, save_z=rng.random() < 0.3)
        return c
    if op == "lookup":
        t = rng.choice(("f32", "f16", "bf16", "q4_0", "q4_1"))
        E = log(32, 1024)
        E = -(-E // 32) * 32 if t in ("q4_0", "q4_1") or rng.random() < 0.6 else E
        return dict(op=op, type=t, out=rng.choice(("f32", "f16", "bf16")), n=log(1, 131072), V=log(100, 250002), E=E, scale=rng.choice((1.0, math.sqrt(E))))
    if op == "lookup_grad":
        E = log(32, 768)
        E = -(-E // 32) * 32 if rng.random() < 0.6 else E
        return dict(op=op, type=rng.choice(("f32", "f16", "bf16")), n=log(1, 131072), V=log(100, 250002), E=E, scale=rng.choice((1.0, math.sqrt(E))), accumulate=rng.random() < 0.4)
    E = log(16, 512)
    return dict(op=op, V=log(100, 30522), E=E, I=4 * E, layers=rng.randint(0, 6), grad=rng.choice(("f32", "f16", "bf16")), bits=rng.choice((32, 8)), copy=rng.random() < 0.5)


def _shapes(c):
    """The tensors of an encoder and whether each decays (vectors do not)."""
    V, E, I = c["V"], c["E"], c["I"]
    one = [(E, E), (E,)] * 4 + [(E,), (E,), (I, E), (I,), (E, I), (E,), (E,), (E,)]
    return [(V, E), (512, E), (2, E), (E,), (E,)] + one * c["layers"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _rows(t, dtype, pad):
    """`t` in `dtype` as a view whose row stride is `pad` more than its width."""
    if not pad:
        return t.to(dtype)
    wide = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=dtype, device="cuda")
    wide[:, : t.shape[1]] = t
    return wide[:, : t.shape[1]]


def _ids(g, n, V):
    """Token ids as text has them: few frequent ones, [CLS] at every 128th place, some places without a token (-1)."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (V * u**4).to(torch.int32).clamp_(0, V - 1)
    ids[::128] = min(101, V - 1)
    hole = torch.rand(n, generator=g, device="cuda") < 0.01
    return torch.where(hole, torch.full_like(ids, -1), ids)


def _table(g, c):
    """Word rows in the file's types: 18- or 20-byte blocks of 32 for q4_0 and q4_1, as bytes."""
    V, E, t = c["V"], c["E"], c["type"]
    if t in DTYPES:
        return _normal(g, V, E, std=0.05).to(DTYPES[t])
    nb = E // 32
    qs = torch.randint(0, 256, (V, nb, 16), generator=g, device="cuda", dtype=torch.uint8)
    d = (torch.rand(V, nb, 1, generator=g, device="cuda") * 0.02 + 0.002).half()
    m = torch.zeros(V, nb, 0, dtype=torch.float16, device="cuda") if t == "q4_0" else -8 * d
    head = torch.cat([d, m], 2).contiguous().view(torch.uint8)
    return torch.cat([head, qs], 2).reshape(V, -1).contiguous()


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=c)
    if c["op"] in ("linear", "linear_backward"):
        M, K, N, t, pad = c["M"], c["K"], c["N"], DTYPES[c["type"]], c["pad"]
        s["x"] = _rows(_normal(g, M, K), t, pad)
        s["w"] = _rows(_normal(g, N, K, std=1 / math.sqrt(K)), t, pad)
        s["b"] = _normal(g, N, std=0.1)
        if c["op"] == "linear":
            s["r"] = _rows(_normal(g, M, N), t, pad) if c["residual"] else None
        else:
            s["dy"] = _rows(_normal(g, M, N, std=0.01), t, pad)
            z = torch.addmm(s["b"], s["x"].float(), s["w"].float().t())
            s["z"] = None if c["act"] == "none" else _rows(z, t, pad)
    elif c["op"] == "lookup":
        s["table"], s["ids"] = _table(g, c), _ids(g, c["n"], c["V"])
    elif c["op"] == "lookup_grad":
        s["dout"] = _normal(g, c["n"], c["E"], std=0.01).to(DTYPES[c["type"]])
        s["ids"] = _ids(g, c["n"], c["V"])
        s["dtable"] = _normal(g, c["V"], c["E"], std=0.01) if c["accumulate"] else torch.empty(c["V"], c["E"], device="cuda")
    else:
        shapes = _shapes(c)
        sizes = [math.prod(x) for x in shapes]
        starts, total = [], 0
        for n in sizes:  # each tensor starts at a whole block of its buffer
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        used = torch.zeros(total, dtype=torch.bool, device="cuda")
        for a, n in zip(starts, sizes):
            used[a : a + n] = True
        s["p"] = _normal(g, total, std=0.05) * used
        s["g"] = (_normal(g, total, std=0.01) * used).to(DTYPES[c["grad"]])
        s["copy"] = torch.zeros(total, dtype=torch.bfloat16, device="cuda") if c["copy"] else None
        s["shapes"], s["sizes"], s["starts"] = shapes, sizes, starts
        s["decay"] = [0.01 if len(x) > 1 else 0.0 for x in shapes]
        at = torch.tensor(starts, device="cuda", dtype=torch.int32)  # of each block: its tensor, that one's first element and decay
        which = torch.bucketize(torch.arange(0, total, BLOCK, device="cuda", dtype=torch.int32), at, right=True) - 1
        s["which"], s["first"] = which.to(torch.int32), at[which]
        s["decay_of"] = torch.tensor(s["decay"], device="cuda", dtype=torch.float64)[which]
        s["seed"] = seed
    torch.cuda.synchronize()
    return s


# ---- the plain forms


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "gelu_erf":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "tanh":
        return torch.tanh(z)
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    if act == "gelu_erf":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "tanh":
        t = torch.tanh(z)
        return 1 - t * t
    return torch.ones_like(z)


def _linear(s):
    c = s["case"]
    if own:
        return _ops().linear(s["x"], s["w"], s["b"], residual=s["r"], act=c["act"], save_z=c["save_z"])
    z = s["x"].float() @ s["w"].float().t() + s["b"]
    y = _act(z, c["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    t = s["x"].dtype
    return (y.to(t), z.to(t)) if c["save_z"] else y.to(t)


def _linear_backward(s):
    c = s["case"]
    if own:
        return _ops().linear_backward(s["dy"], s["x"], s["w"], z=s["z"], act=c["act"])
    t = s["x"].dtype
    dz = s["dy"].float()
    if c["act"] != "none":
        dz = dz * _act_slope(s["z"].float(), c["act"])
    return (dz @ s["w"].float()).to(t), (dz.t() @ s["x"].float()).to(t), dz.sum(0)


def _dequant(rows, t):
    """The values of q4_0 or q4_1 rows given as bytes: low halves are the block's first 16 values."""
    blocks = rows.reshape(rows.shape[0], -1, 18 if t == "q4_0" else 20)
    head = blocks[:, :, : (2 if t == "q4_0" else 4)].contiguous().view(torch.float16).float()
    q = blocks[:, :, (2 if t == "q4_0" else 4) :]
    q = torch.cat([q & 15, q >> 4], 2).float()
    v = (q - 8) * head[:, :, :1] if t == "q4_0" else q * head[:, :, :1] + head[:, :, 1:2]
    return v.reshape(rows.shape[0], -1)


def _lookup(s):
    c = s["case"]
    if own:
        return _ops().lookup(s["table"], s["ids"], scale=c["scale"], table_type=c["type"], out_dtype=DTYPES[c["out"]])
    there = (s["ids"] >= 0) & (s["ids"] < c["V"])
    rows = s["table"][torch.where(there, s["ids"], torch.zeros_like(s["ids"])).long()]
    v = rows.float() if c["type"] in DTYPES else _dequant(rows, c["type"])
    return torch.where(there[:, None], v * c["scale"], torch.zeros_like(v)).to(DTYPES[c["out"]])


def _lookup_grad(s):
    c, d = s["case"], s["dtable"]
    if own:
        return _ops().lookup_grad(s["dout"], s["ids"], c["V"], scale=c["scale"], pad_id=0, out=d, accumulate=c["accumulate"])
    there = (s["ids"] > 0) & (s["ids"] < c["V"])  # row 0 is the padding token's: it has no gradient
    rows = torch.where(there[:, None], s["dout"].float(), torch.zeros_like(s["dout"], dtype=torch.float32))
    total = torch.zeros_like(d).index_add_(0, torch.where(there, s["ids"], torch.zeros_like(s["ids"])).long(), rows) * c["scale"]
    if c["accumulate"]:
        d += total
    else:
        d.copy_(total)
    return d


def _mix(h):
    """Mixes 32 bits by two rounds of a shift, an exclusive or and an odd product; int32 products wrap."""
    h = (h ^ ((h >> 16) & 0xFFFF)) * (0x9E3779B9 - 2**32)
    h = (h ^ ((h >> 15) & 0x1FFFF)) * (0xBB67AE85 - 2**32)
    return h ^ ((h >> 16) & 0xFFFF)


def _codes(mant):
    """What the codes of a magnitude with `mant` bits after the point stand for: linear in the lowest octave, then 15 octaves."""
    n = 1 << mant
    c = torch.arange(16 * n, device="cuda")
    e, f = (c >> mant).float(), (c & (n - 1)).float()
    return torch.where(e == 0, f * (2 / n), (1 + f / n) * torch.exp2(e))


def _encode(a, mant, h):
    """Magnitudes as codes and their block's scales, rounded up or down at random by the bits `h`."""
    n, top = 1 << mant, (2 - 2.0**-mant) * 2.0**15
    top_value = torch.full((), top, device="cuda")
    peak = a.reshape(-1, BLOCK).amax(1, keepdim=True)
    scale = torch.where(peak < 2.0**-100, torch.zeros_like(peak), peak / top_value)
    inv = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    y = (a.reshape(-1, BLOCK) * inv).reshape(-1)
    drop = 23 - mant
    far = ((y.view(torch.int32) + ((h >> (32 - drop)) & ((1 << drop) - 1))) >> drop) - 127 * n
    near = (y * (n / 2) + ((h >> 8) & 0xFFFFFF).float() * 2.0**-24).to(torch.int32)
    return torch.where(y >= 2, far, near).clamp_(max=16 * n - 1), scale


def _keys(s):
    """Each element's place in its tensor, mixed with its tensor's number and the step's seed."""
    seed = (s["seed"] + s["t"]) & 0xFFFFFFFF
    key = _mix(s["which"] * (0x9E3779B9 - 2**32) ^ (seed - 2**32 if seed >= 2**31 else seed))
    first = torch.arange(len(s["which"]), device="cuda", dtype=torch.int32) * BLOCK - s["first"]
    place = first[:, None] + torch.arange(BLOCK, device="cuda", dtype=torch.int32)
    return _mix(place ^ key[:, None]).reshape(-1)


def _adamw(s):
    c = s["case"]
    if own:
        ops = _ops()
        if "opt" not in s:
            views = lambda flat: [flat[a : a + n].view(x) for a, n, x in zip(s["starts"], s["sizes"], s["shapes"])]  # noqa: E731
            s["opt"] = ops.AdamW(views(s["p"]), lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=s["decay"], bits=c["bits"],
                                 copies=views(s["copy"]) if c["copy"] else None, seed=s["seed"])
            s["views"] = views(s["g"])
        s["opt"].step(s["views"])
        m, v = s["opt"].moments()
    else:
        if "m" not in s:
            s["t"] = 0
            s["m"], s["v"] = torch.zeros_like(s["p"]), torch.zeros_like(s["p"])
        s["t"] += 1
        bc1, bc2 = 1 - BETA1 ** s["t"], 1 - BETA2 ** s["t"]
        keep = (1 - LR * s["decay_of"]).float()[:, None]
        g = s["g"].float()
        m = s["m"] * BETA1 + g * (1 - BETA1)
        v = s["v"] * BETA2 + (g * (1 - BETA2)) * g
        root = v.sqrt()
        s["p"].copy_((s["p"].reshape(-1, BLOCK) * keep).reshape(-1) - (m * (LR / bc1)) / (root * (1 / math.sqrt(bc2)) + EPS))
        if c["bits"] == 8:
            h = _keys(s)
            k, scale = _encode(m.abs(), 3, h)
            m = (_codes(3)[k.long()].reshape(-1, BLOCK) * scale).reshape(-1) * m.sign()
            k, scale = _encode(root, 4, _mix(h ^ (0x9E3779B9 - 2**32)))
            k = torch.where((root > 0) & (k == 0), torch.ones_like(k), k)  # a second moment never vanishes
            root = (_codes(4)[k.long()].reshape(-1, BLOCK) * scale).reshape(-1)
            v = root * root
        s["m"].copy_(m)
        s["v"].copy_(v)
        if c["copy"]:
            s["copy"].copy_(s["p"])
        m, v = s["m"], s["v"]
    return dict(p=s["p"], m=m, v=v, copy=s["copy"]) if c["copy"] else dict(p=s["p"], m=m, v=v)


def run(state):
    return {"linear": _linear, "linear_backward": _linear_backward, "lookup": _lookup, "lookup_grad": _lookup_grad, "adamw": _adamw}[state["case"]["op"]](state)


# ---- the work that a pass cannot do without, and its results in 64 bits


def work(case):
    c = case
    if c["op"] in ("linear", "linear_backward"):
        M, K, N, e = c["M"], c["K"], c["N"], SIZE[c["type"]]
        if c["op"] == "linear":
            return dict(bytes=e * (M * K + N * K + M * N * (1 + c["residual"] + c["save_z"])) + 4 * N, flops=2 * M * N * K)
        return dict(bytes=e * (M * N * (1 if c["act"] == "none" else 2) + 2 * M * K + 2 * N * K) + 4 * N, flops=4 * M * N * K)
    if c["op"] == "lookup":
        return dict(bytes=4 * c["n"] + c["E"] * (min(c["n"], c["V"]) * ROW_BYTES[c["type"]] + c["n"] * SIZE[c["out"]]), flops=c["n"] * c["E"])
    if c["op"] == "lookup_grad":
        rows = 2 * min(c["n"], c["V"]) if c["accumulate"] else c["V"]
        return dict(bytes=4 * c["n"] + c["E"] * (c["n"] * SIZE[c["type"]] + 4 * rows), flops=c["n"] * c["E"])
    n = sum(math.prod(x) for x in _shapes(c))
    # weights and states read and written, the gradient read; 8-bit states are read back as values too
    each = 8 + SIZE[c["grad"]] + (16 if c["bits"] == 32 else 4 + 2 + 8) + (2 if c["copy"] else 0)
    return dict(bytes=n * each, flops=12 * n)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    f64 = torch.float64
    if c["op"] == "linear":
        z = torch.addmm(s["b"].to(f64), s["x"].to(f64), s["w"].to(f64).t())
        y = _definition(z, c["act"])
        y = y if s["r"] is None else y + s["r"].to(f64)
        return (y, z) if c["save_z"] else y
    if c["op"] == "linear_backward":
        dz = s["dy"].to(f64)
        if c["act"] != "none":
            z = s["z"].to(f64).clone().requires_grad_(True)
            (dz,) = torch.autograd.grad(_definition(z, c["act"]), z, dz)
        return dz.mm(s["w"].to(f64)), dz.t().contiguous().mm(s["x"].to(f64)), dz.sum(0)
    if c["op"] == "lookup":
        out = torch.zeros(c["n"], c["E"], dtype=f64, device="cuda")
        at = torch.nonzero((s["ids"] >= 0) & (s["ids"] < c["V"]))[:, 0]
        rows = s["table"][s["ids"][at].long()]
        if c["type"] not in DTYPES:
            nb, size = c["E"] // 32, 18 if c["type"] == "q4_0" else 20
            blocks = rows.view(-1, nb, size)
            d = blocks[..., 0:2].contiguous().view(torch.float16).to(f64)
            low = d * -8 if size == 18 else blocks[..., 2:4].contiguous().view(torch.float16).to(f64)
            q = blocks[..., size - 16 :].to(f64)
            high = torch.floor(q / 16)
            rows = (torch.cat([q - 16 * high, high], -1) * d + low).view(len(at), -1)
        out[at] = rows.to(f64) * c["scale"]
        return out
    if c["op"] == "lookup_grad":
        out = s["dtable"].to(f64) if c["accumulate"] else torch.zeros(c["V"], c["E"], dtype=f64, device="cuda")
        at = torch.nonzero((s["ids"] >= 1) & (s["ids"] < c["V"]))[:, 0]
        return out.index_put_((s["ids"][at].long(),), s["dout"][at].to(f64) * c["scale"], accumulate=True)
    # the first step from zero states: both moments are the gradient's, and their corrections cancel
    g, p = s["g"].to(f64), s["p"].to(f64)
    for a, n, d in zip(s["starts"], s["sizes"], s["decay"]):
        p[a : a + n] *= 1 - LR * d
    p -= LR * g / (g.abs() + EPS)
    plain = c["bits"] == 32  # what 8-bit states hold depends on the order of the roundings before theirs
    out = dict(p=p, m=(1 - BETA1) * g if plain else None, v=(1 - BETA2) * g**2 if plain else None)
    return dict(out, copy=p) if c["copy"] else out


def _definition(z, act):
    """The activations in 64 bits."""
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))
    if act == "gelu_erf":
        return z * torch.special.ndtr(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    return torch.tanh(z) if act == "tanh" else z

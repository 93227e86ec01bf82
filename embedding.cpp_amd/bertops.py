"""The operators around the encoder on torch tensors (include/bert_amd.h, second part).

`linear` / `linear_backward` are a dense layer with its epilogue, `lookup` / `lookup_grad` the rows of a
token table, `AdamW` the step that trains both.  Tensors stay on their device; every call is enqueued on
torch's current stream of that device and returns at once.  Arguments are checked here and in the
library: a bad one raises before anything is launched.  Results have no autograd nodes: `linear` and
`lookup` warn where torch would have made one, outside of torch.no_grad() and of an autograd.Function.

`Adapter` is a trained layer on a BertModel's embeddings and `TokenTable` a trainable copy of its word
rows; both are what a user builds from the operators.
"""
from __future__ import annotations

import ctypes
import warnings
from typing import List, Optional, Sequence

import numpy as np
import torch

import bertlib

ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_erf": 3, "silu": 4, "tanh": 5}
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
TABLE_TYPES = {"f32": 0, "f16": 1, "q4_0": 2, "q4_1": 3, "bf16": 30}
BLOCK_BYTES = {"q4_0": 18, "q4_1": 20}  # of 32 values
STATE_BLOCK = 256  # elements that share a scale in 8-bit states


def _check(rc: int) -> None:
    if rc < 0:
        raise (RuntimeError if rc == -3 else ValueError)(bertlib.last_error())


# a tensor that the library has written: what autograd saved of it is not its value any more
_written = torch.autograd.graph.increment_version

# the current stream's handle without the Stream object around it (2 us of a 10 us call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: torch.device) -> int:
    return _raw_stream(device.index) if _raw_stream else torch.cuda.current_stream(device).cuda_stream


def _room(nbytes: int, device: torch.device):
    """Workspace on the current stream: (tensor to keep until the call is enqueued, pointer, bytes)."""
    if nbytes < 0:
        _check(-1)
    if nbytes == 0:
        return None, None, 0
    t = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), nbytes


def _matrix(name: str, t: torch.Tensor, dtype, device, rows: int, cols: int) -> int:
    """The row stride of a [rows][cols] matrix in row order."""
    if t.dtype is dtype and t.device == device and t.shape == (rows, cols):
        s0, s1 = t.stride()
        if s1 == 1 or cols == 1:
            return s0 if rows > 1 else max(s0, cols)
        raise ValueError(f"{name}'s columns are {s1} elements apart: rows have to be contiguous")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}: {dtype} on {device} is needed")
    raise ValueError(f"{name} has shape {tuple(t.shape)}: {(rows, cols)} is needed")


def _first(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: a GPU tensor is needed")
    if t.dtype not in TYPES:
        raise ValueError(f"{name} is {t.dtype}: float32, float16 or bfloat16 is needed")
    if t.dim() != 2:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: two dimensions are needed")


def _no_node(name: str) -> None:
    """Says that the results of tensors that require a gradient have none, where torch would have given them one."""
    if torch.is_grad_enabled():
        warnings.warn(f"{name}() of a tensor that requires a gradient: its results have none.  Call it under torch.no_grad(), "
                      "or in a torch.autograd.Function", stacklevel=3)


def _act(act: str) -> int:
    if act not in ACTS:
        raise ValueError(f"unknown activation {act!r}: one of {', '.join(ACTS)}")
    return ACTS[act]


def _vector(name: str, t: torch.Tensor, device, n: int) -> int:
    if t.dtype != torch.float32 or t.device != device or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} has to be a contiguous float32 vector of {n} on {device}")
    return t.data_ptr()


def _int32(name: str, a: int, b: int = 0) -> None:
    """The library takes these in 32 bits, and ctypes would cut them off without a word."""
    if not -(1 << 31) <= a < 1 << 31 or not -(1 << 31) <= b < 1 << 31:
        raise ValueError(f"{name} {a if b == 0 else (a, b)} is over 32 bits")


def _aligned(size: int, *matrices) -> int:
    """Whether all (address, row stride) allow 16-byte pieces."""
    bits = 0
    for p, ld in matrices:
        if ld >= 1 << 21:
            return 0
        bits |= p | ld * size
    return int(bits & 15 == 0)


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
           act: str = "none", save_z: bool = False, out: Optional[torch.Tensor] = None):
    """act(x w^T + bias) + residual for x [M, K] and w [N, K] of one type; bias is float32.

    save_z: also returns the pre-activation, (y, z), which linear_backward takes.  out: where y goes (may
    be `residual`)."""
    _first("x", x)
    if x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad) or (residual is not None and residual.requires_grad):
        _no_node("linear")
    (M, K), N, dt, dev, a = x.shape, w.shape[0], x.dtype, x.device, _act(act)
    _int32("a width of", N, K)
    ldx, ldw = _matrix("x", x, dt, dev, M, K), _matrix("w", w, dt, dev, N, K)
    b = None if bias is None else _vector("bias", bias, dev, N)
    r, ldr = (None, 0) if residual is None else (residual.data_ptr(), _matrix("residual", residual, dt, dev, M, N))
    y = torch.empty(M, N, dtype=dt, device=dev) if out is None else out
    ldy = N if out is None else _matrix("out", out, dt, dev, M, N)
    z = torch.empty(M, N, dtype=dt, device=dev) if save_z else None
    L, px, pw, typ = bertlib.lib(), x.data_ptr(), w.data_ptr(), TYPES[dt]
    keep, ws, nws = _room(L.bert_amd_linear_workspace(typ, M, N, K, _aligned(x.element_size(), (px, ldx), (pw, ldw))), dev)
    _check(L.bert_amd_linear(dev.index, typ, a, M, N, K, px, ldx, pw, ldw, b, r, ldr, y.data_ptr(), ldy,
                             z.data_ptr() if save_z else None, N, ws, nws, _stream(dev)))
    if out is not None:
        _written(out)
    return (y, z) if save_z else y


def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, *, z: Optional[torch.Tensor] = None, act: str = "none",
                    need: Sequence[bool] = (True, True, True)):
    """(dx, dw, dbias) of linear() from dy [M, N]; None where `need` says so.  The residual's gradient is dy."""
    _first("x", x)
    (M, K), N, dt, dev, a = x.shape, w.shape[0], x.dtype, x.device, _act(act)
    _int32("a width of", N, K)
    ldx, ldw, lddy = _matrix("x", x, dt, dev, M, K), _matrix("w", w, dt, dev, N, K), _matrix("dy", dy, dt, dev, M, N)
    if a and z is None:
        raise ValueError(f"the gradient of {act!r} needs z: linear(..., save_z=True)")
    pz, ldz = (z.data_ptr(), _matrix("z", z, dt, dev, M, N)) if a else (None, 0)
    dx = torch.empty(M, K, dtype=dt, device=dev) if need[0] else None
    dw = torch.empty(N, K, dtype=dt, device=dev) if need[1] else None
    db = torch.empty(N, dtype=torch.float32, device=dev) if need[2] else None
    L = bertlib.lib()
    aligned = _aligned(x.element_size(), (x.data_ptr(), ldx), (w.data_ptr(), ldw), (dy.data_ptr(), lddy))
    keep, ws, nws = _room(L.bert_amd_linear_backward_workspace(TYPES[dt], a, M, N, K, aligned), dev)
    _check(L.bert_amd_linear_backward(dev.index, TYPES[dt], a, M, N, K, dy.data_ptr(), lddy, pz, ldz, x.data_ptr(), ldx,
                                      w.data_ptr(), ldw, dx.data_ptr() if need[0] else None, K,
                                      dw.data_ptr() if need[1] else None, K, db.data_ptr() if need[2] else None, ws, nws,
                                      _stream(dev)))
    return dx, dw, db


def _ids(ids: torch.Tensor, device) -> int:
    if ids.dtype != torch.int32 or ids.device != device or not ids.is_contiguous():
        raise ValueError(f"ids have to be contiguous int32 on {device}")
    return ids.data_ptr()


def lookup(table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0, table_type: Optional[str] = None,
           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """scale * table[ids], shape ids.shape + (width,); zeros where an id names no row.

    table: [rows, width] of a float type, or with table_type "q4_0" / "q4_1" the rows' bytes (uint8) as in
    a model file.  out_dtype: float32 for those, the table's own type otherwise, unless given."""
    if not table.is_cuda or table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError("the table has to be a GPU tensor [rows, width]")
    if table.requires_grad:
        _no_node("lookup")
    blocks = table_type in BLOCK_BYTES
    if blocks:
        if table.dtype != torch.uint8 or table.shape[1] % BLOCK_BYTES[table_type]:
            raise ValueError(f"a {table_type} table is uint8 rows of whole blocks of {BLOCK_BYTES[table_type]} bytes")
        width, typ = table.shape[1] // BLOCK_BYTES[table_type] * 32, TABLE_TYPES[table_type]
    else:
        if table.dtype not in TYPES or (table_type is not None and TABLE_TYPES.get(table_type) != TYPES[table.dtype]):
            raise ValueError(f"a {table.dtype} table is not of type {table_type!r}")
        width, typ = table.shape[1], TYPES[table.dtype]
    _int32("a table of", table.shape[0], width)
    out_dtype = out_dtype or (torch.float32 if blocks else table.dtype)
    if out_dtype not in TYPES:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    dev = table.device
    ld = _matrix("table", table, table.dtype, dev, *table.shape) * table.element_size()
    out = torch.empty(*ids.shape, width, dtype=out_dtype, device=dev)
    _check(bertlib.lib().bert_amd_lookup(dev.index, typ, TYPES[out_dtype], ids.numel(), table.shape[0], width, table.data_ptr(),
                                         ld, _ids(ids, dev), scale, out.data_ptr(), width, _stream(dev)))
    return out


def lookup_grad(dout: torch.Tensor, ids: torch.Tensor, n_rows: int, *, scale: float = 1.0, pad_id: int = -1,
                out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """The table's gradient [n_rows, width] in float32 from dout, ids.shape + (width,): every row written, or
    with `accumulate` added to `out`.  Ids that name no row and pad_id have none."""
    dev, width = dout.device, dout.shape[-1]
    if tuple(dout.shape[:-1]) != tuple(ids.shape):
        raise ValueError(f"dout has shape {tuple(dout.shape)} for ids {tuple(ids.shape)}")
    _int32("a table of", n_rows, width)
    _int32("pad_id", pad_id)
    if dout.dim() != 2:
        dout = dout.reshape(-1, width)
    _first("dout", dout)
    ldd = _matrix("dout", dout, dout.dtype, dev, *dout.shape)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty(n_rows, width, dtype=torch.float32, device=dev)
    ldt = _matrix("out", out, torch.float32, dev, n_rows, width)
    L = bertlib.lib()
    keep, ws, nws = _room(L.bert_amd_lookup_grad_workspace(ids.numel(), n_rows, width), dev)
    _check(L.bert_amd_lookup_grad(dev.index, TYPES[dout.dtype], ids.numel(), n_rows, width, dout.data_ptr(), ldd, _ids(ids, dev),
                                  scale, pad_id, int(accumulate), out.data_ptr(), ldt, ws, nws, _stream(dev)))
    _written(out)
    return out


class AdamW:
    """AdamW over `params` (float32, contiguous), updated in place; moments in 32 or 8 bits.

    weight_decay: one value, or one for each tensor.  copies: for each tensor a float16 / bfloat16 tensor
    that gets its updated values rounded (None: none).  seed: what 8-bit states are rounded by, with the
    step's number added.  The moments are buffers of their own, laid out once: tensor i's begin at
    where[i], a multiple of 256; load saved ones with copy_.  Tensors, copies and states stay where they
    are: step() refuses to run once one has moved.  A step that fails on the device may have moved some of the
    weights and moments: step() refuses from then on, too.  A step captured in a graph repeats its own number,
    learning rate and rounding."""

    _ROW = np.dtype([("p", "u8"), ("g", "u8"), ("m", "u8"), ("v", "u8"), ("ms", "u8"), ("vs", "u8"), ("copy", "u8"), ("n", "i8"),
                     ("decay", "f8")])

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01,
                 bits: int = 32, copies: Optional[Sequence[torch.Tensor]] = None, seed: int = 0):
        self.params: List[torch.Tensor] = list(params)
        if not self.params:
            raise ValueError("no tensors")
        if bits not in (8, 32):
            raise ValueError(f"states of {bits} bits are not supported")
        dev = self.params[0].device
        for i, t in enumerate(self.params):
            if not t.is_cuda or t.device != dev or t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError(f"tensor {i} has to be contiguous float32 on {dev}, a GPU")
        self.copies = list(copies) if copies is not None else None
        self._copy_type = TYPES[torch.bfloat16]
        if self.copies is not None:
            kinds = {t.dtype for t in self.copies}
            if len(self.copies) != len(self.params) or len(kinds) != 1 or not kinds <= {torch.float16, torch.bfloat16}:
                raise ValueError("copies: one float16 or bfloat16 tensor for each, all of one type")
            for t, c in zip(self.params, self.copies):
                if c.device != dev or c.shape != t.shape or not c.is_contiguous():
                    raise ValueError("a copy has another shape or device than its tensor, or is not contiguous")
            self._copy_type = TYPES[self.copies[0].dtype]
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * len(self.params)
        if len(decay) != len(self.params):
            raise ValueError("weight_decay: one value, or one for each tensor")
        self.device, self.bits, self.seed, self.t, self._failed = dev, bits, int(seed), 0, False
        self.lr, self.betas, self.eps = lr, betas, eps
        sizes = [t.numel() for t in self.params]
        room = [-(-n // STATE_BLOCK) * STATE_BLOCK for n in sizes]
        self.where = [0] + list(np.cumsum(room)[:-1].tolist())
        total = int(sum(room))
        kind = torch.float32 if bits == 32 else torch.uint8
        self.m, self.v = (torch.zeros(total, dtype=kind, device=dev) for _ in range(2))
        self.m_scale, self.v_scale = ((torch.zeros(total // STATE_BLOCK, device=dev) for _ in range(2)) if bits == 8 else (None, None))
        rows = np.zeros(len(sizes), self._ROW)
        at = np.asarray(self.where, np.uint64)
        rows["p"] = [t.data_ptr() for t in self.params]
        rows["m"] = self.m.data_ptr() + at * self.m.element_size()
        rows["v"] = self.v.data_ptr() + at * self.v.element_size()
        if bits == 8:
            rows["ms"] = self.m_scale.data_ptr() + at // STATE_BLOCK * 4
            rows["vs"] = self.v_scale.data_ptr() + at // STATE_BLOCK * 4
        if self.copies is not None:
            rows["copy"] = [t.data_ptr() for t in self.copies]
        rows["n"], rows["decay"] = sizes, decay
        self._rows, self._shapes, self._at = rows, [t.shape for t in self.params], self._addresses()

    def _addresses(self) -> List[int]:
        states = [self.m, self.v] + ([self.m_scale, self.v_scale] if self.bits == 8 else [])
        return [t.data_ptr() for t in (*self.params, *(self.copies or ()), *states)]

    def step(self, grads: Sequence[torch.Tensor], grad_scale: Optional[torch.Tensor] = None) -> None:
        """One step; grads: one for each tensor, all of one float type.  grad_scale: one float32 on the device
        (a clipping factor) that multiplies them."""
        if self._failed:
            raise RuntimeError("an earlier step failed on the device: weights and moments are undefined")
        dt, dev = grads[0].dtype, self.device
        if dt not in TYPES or len(grads) != len(self._shapes):
            raise ValueError("grads: one float tensor for each parameter")
        for g, s in zip(grads, self._shapes):
            if g.dtype != dt or g.shape != s or g.device != dev or not g.is_contiguous():
                raise ValueError("a gradient has another type, shape or device than the others or its tensor, or is not contiguous")
        if self._addresses() != self._at:
            raise ValueError("a tensor, copy or state is no longer where it was when the optimizer was made")
        if grad_scale is not None and (grad_scale.dtype != torch.float32 or grad_scale.device != dev or grad_scale.numel() != 1):
            raise ValueError(f"grad_scale has to be one float32 on {dev}")
        self._rows["g"] = [g.data_ptr() for g in grads]
        rc = bertlib.lib().bert_amd_adamw(dev.index, len(self._rows), self._rows.ctypes.data, self.bits, TYPES[dt], self._copy_type,
                                          self.lr, self.betas[0], self.betas[1], self.eps, self.t + 1,
                                          (self.seed + self.t + 1) & 0xFFFFFFFF,
                                          grad_scale.data_ptr() if grad_scale is not None else None, _stream(dev))
        self._failed = rc == -3
        if rc != -1:
            _written([*self.params, *(self.copies or ())])
        _check(rc)
        self.t += 1

    def moments(self):
        """(m, v) in float32, laid out by `where`: the states themselves, or what 8-bit ones stand for."""
        if self.bits == 32:
            return self.m, self.v
        m, v = torch.empty(self.m.shape, device=self.device), torch.empty(self.v.shape, device=self.device)
        _check(bertlib.lib().bert_amd_adamw_moments(self.device.index, m.numel(), self.m.data_ptr(), self.m_scale.data_ptr(),
                                                    self.v.data_ptr(), self.v_scale.data_ptr(), m.data_ptr(), v.data_ptr(),
                                                    _stream(self.device)))
        return m, v


class _Own:
    """Tensors made on one stream that calls on others may use and drop: their memory is not given out again
    before those are done with it."""

    def __init__(self, *tensors: torch.Tensor):
        self._tensors, self._stream = tensors, _stream(tensors[0].device)

    def use(self):
        dev = self._tensors[0].device
        if _stream(dev) != self._stream:
            for t in self._tensors:
                t.record_stream(torch.cuda.current_stream(dev))
        return self._tensors


def _version(t: torch.Tensor) -> int:
    return 0 if t.is_inference() else t._version


class _Kept:
    """What a training forward keeps for its backward: one forward at a time, until the weights move."""

    def __init__(self):
        self._what, self._open = None, 0  # the newest forward's; forwards since the last backward
        self._versions = []

    def put(self, *tensors: torch.Tensor) -> None:
        self._what, self._open, self._versions = _Own(*tensors), self._open + 1, [_version(t) for t in tensors]

    def get(self):
        if self._what is None:
            raise ValueError("backward() follows forward(), before step()")
        if self._open > 1:
            self.drop()
            raise ValueError("two forwards before a backward, whose gradient is meant? Take both batches in one forward, "
                             "and forwards without a backward with train=False")
        self._open = 0
        tensors = self._what.use()
        if [_version(t) for t in tensors] != self._versions:
            raise ValueError("an input of forward() has been changed in place since: its backward needs it as it was")
        return tensors

    def drop(self) -> None:
        self._what, self._open = None, 0


class Adapter:
    """A trained layer on embeddings: y = act(W e + b) + e, W and b starting at zero.

    Trained by the caller's loss: y = forward(e), backward(dy), step().  A backward is its newest forward's;
    pairs and triplets of a loss go through one forward, side by side in a batch.  Gradients add up over backwards until step()."""

    def __init__(self, n_embd: int, act: str = "tanh", device="cuda:0", **optimizer):
        _act(act)
        device = torch.device(device)
        self.act = act
        self.w, self.b = torch.zeros(n_embd, n_embd, device=device), torch.zeros(n_embd, device=device)
        self.opt = AdamW([self.w, self.b], **{"weight_decay": [0.01, 0.0], **optimizer})
        self._kept, self._grads = _Kept(), None

    def forward(self, e: torch.Tensor, train: bool = True) -> torch.Tensor:
        if not train:
            return linear(e, self.w, self.b, residual=e, act=self.act)
        y, z = linear(e, self.w, self.b, residual=e, act=self.act, save_z=True)
        self._kept.put(e, z)
        return y

    def backward(self, dy: torch.Tensor, need_input: bool = False) -> Optional[torch.Tensor]:
        """Adds to the weights' gradients until step(); gives the embeddings' own where asked for."""
        e, z = self._kept.get()
        de, dw, db = linear_backward(dy, e, self.w, z=z, act=self.act, need=(need_input, True, True))
        if self._grads is None:
            self._grads = _Own(dw, db)
        else:
            for kept, new in zip(self._grads.use(), (dw, db)):
                kept.add_(new)
        return de + dy if need_input else None

    def step(self) -> None:
        if self._grads is None:
            raise ValueError("step() follows backward()")
        self.opt.step(self._grads.use())
        self._grads = None
        self._kept.drop()  # z is of the weights as they were

    def encode(self, model: "bertlib.BertModel", sentences, batch_size: int = 16) -> np.ndarray:
        """The model's embeddings of `sentences` through the adapter, L2-normalised again."""
        single = isinstance(sentences, str)
        e = torch.from_numpy(model.encode([sentences] if single else sentences, batch_size)).to(self.w.device)
        y = self.forward(e, train=False)
        y = (y / y.norm(dim=1, keepdim=True)).cpu().numpy()
        return y[0] if single else y


class TokenTable:
    """A trainable float32 copy of a model's word rows: static embeddings of tokens.

    forward(ids), backward(dout), step(), as Adapter."""

    def __init__(self, model: "bertlib.BertModel", slot: int = 0, pad_id: int = 0, **optimizer):
        self.rows = word_rows(model, slot=slot)
        self.pad_id = pad_id
        self.opt = AdamW([self.rows], **optimizer)
        self._kept, self._scale, self._grad = _Kept(), 1.0, None

    def forward(self, ids: torch.Tensor, scale: float = 1.0, train: bool = True) -> torch.Tensor:
        out = lookup(self.rows, ids, scale=scale)
        if train:
            self._kept.put(ids)
            self._scale = scale
        return out

    def backward(self, dout: torch.Tensor) -> None:
        """Adds to the table's gradient until step()."""
        (ids,) = self._kept.get()
        (out,) = (None,) if self._grad is None else self._grad.use()
        grad = lookup_grad(dout, ids, self.rows.shape[0], scale=self._scale, pad_id=self.pad_id, out=out, accumulate=out is not None)
        if out is None:
            self._grad = _Own(grad)

    def step(self) -> None:
        if self._grad is None:
            raise ValueError("step() follows backward()")
        self.opt.step(self._grad.use())
        self._grad = None
        self._kept.drop()


def word_rows(model: "bertlib.BertModel", ids: Optional[torch.Tensor] = None, *, slot: int = 0, scale: float = 1.0,
              out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Rows of the model's own word-embedding table (all of them without ids), out of the type the model file has."""
    ptr, typ, n_rows, width, dev = model.word_table(slot)
    device = torch.device("cuda", dev)
    if ids is None:
        ids = torch.arange(n_rows, dtype=torch.int32, device=device)
    if out_dtype not in TYPES:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    names = {v: k for k, v in TABLE_TYPES.items()}
    ld = width // 32 * BLOCK_BYTES[names[typ]] if names[typ] in BLOCK_BYTES else width * (4 if typ == 0 else 2)
    out = torch.empty(*ids.shape, width, dtype=out_dtype, device=device)
    _check(bertlib.lib().bert_amd_lookup(dev, typ, TYPES[out_dtype], ids.numel(), n_rows, width, ctypes.c_void_p(ptr), ld,
                                         _ids(ids, device), scale, out.data_ptr(), width, _stream(device)))
    return out

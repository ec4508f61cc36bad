"""Row-selection operators on torch tensors: embedding lookup, routing to
experts and the exchange of rows with them, and gradient clipping (the C
entry points spmvb_embedding_*, spmvb_router_* and spmvb_clip_*).

They are the sparse products of a language model's step. Tokens select rows
of a table (one entry per row) or experts (k entries per row); the matrix is
made on the device in every step, so nothing is uploaded. Every method
enqueues its kernels on `stream` (default: torch's current stream of the
context's device) and returns; outputs are tensors the caller passes in. A
handle holds scratch memory and is used by one stream at a time. Calls do not
allocate or synchronize and can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
from operator import index as _as_int

from . import _lib
from ._lib import BF16, F16, F32, F64, call, load

_MOST = 2 ** 31 - 1  # rows, entries: the C side counts in int32
SCORES = {"softmax": 0, "sigmoid": 1}
_CODES: dict = {}
_raw_stream = None


def _torch_names() -> None:
    """What the checks need of torch, looked up once (the package imports
    without it)."""
    global _raw_stream
    import torch
    _CODES.update({torch.float32: F32, torch.float64: F64, torch.float16: F16, torch.bfloat16: BF16,
                   torch.int32: "int32"})
    # The current stream's handle, without a Stream object around it.
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda device: torch.cuda.current_stream(device).cuda_stream)


def _int32(v, what: str) -> int:
    """An integer for the C side, which would take what int32 does not hold
    modulo 2^32."""
    n = _as_int(v)
    if not -_MOST - 1 <= n <= _MOST:
        raise ValueError(f"{what} = {n} does not fit int32")
    return n


def _stream(stream, device: int) -> int:
    if stream is None:
        return _raw_stream(device)
    if stream.device_index != device:
        raise ValueError(f"the stream belongs to cuda:{stream.device_index}, the handle to cuda:{device}")
    return stream.cuda_stream


def _on(t, device: int, what: str) -> None:
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.get_device() != device:
        raise ValueError(f"{what} is on cuda:{t.get_device()}, the handle on cuda:{device}")


def _code(t, codes, device: int, what: str):
    """The library's code of t's type, which must be one of `codes`; t must
    be a CUDA tensor of `device`."""
    if not _CODES:
        _torch_names()
    try:
        code, at = _CODES.get(t.dtype), t.get_device()
    except (AttributeError, RuntimeError):
        code, at = None, -1
    if at != device:
        _on(t, device, what)
    if code not in codes:
        raise ValueError(f"{what} cannot be {t.dtype}")
    return code


def _rows(t, rows, width: int, device: int, what: str, codes=(F32, F16, BF16)):
    """Checks a rows x width tensor (rows None: any number) with unit column
    stride; returns (dtype code, row stride, address)."""
    code = _code(t, codes, device, what)
    shape = t.shape
    if len(shape) != 2 or shape[1] != width or (rows is not None and shape[0] != rows) or shape[0] > _MOST or width > _MOST:
        raise ValueError(f"{what} has shape {tuple(shape)}; ({'any' if rows is None else rows}, {width}) is needed")
    ld, unit = t.stride()
    if unit != 1 or ld < width:
        if (unit != 1 and width > 1) or (ld < width and shape[0] > 1):
            raise ValueError(f"{what} must have rows of unit stride that do not overlap (strides {t.stride()})")
        ld = max(ld, width)
    return code, ld, t.data_ptr()


def _flat(t, code, count: int, device: int, what: str) -> int:
    """Checks a contiguous tensor of `count` entries; returns its address."""
    _code(t, (code,), device, what)
    if t.numel() != count or count > _MOST:
        raise ValueError(f"{what} holds {t.numel()} entries; {count} are needed")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return t.data_ptr()


I32 = "int32"
_ALL = (F32, F64, F16, BF16)


class _Handle:
    _destroy = ""
    handle = None

    def close(self) -> None:
        if self.handle:
            getattr(load(), self._destroy)(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Embedding(_Handle):
    """Rows of a `rows` x `width` table selected by tokens, and the gradient
    (spmvb_embedding). float32, float16, bfloat16 and float64; scratch for
    the gradient of up to `max_tokens` tokens."""

    _destroy = "spmvb_embedding_destroy"

    def __init__(self, ctx, rows: int, width: int, max_tokens: int):
        rows, width, max_tokens = _int32(rows, "rows"), _int32(width, "width"), _int32(max_tokens, "max_tokens")
        h = C.c_void_p()
        call("spmvb_embedding_create", ctx.handle, rows, width, max_tokens, C.byref(h))
        self.handle, self.ctx = h, ctx
        self.rows, self.width, self.max_tokens = rows, width, max_tokens

    def lookup(self, tokens, table, out, scale: float = 1.0, stream=None) -> None:
        """out[t] = scale * table[tokens[t]]; a negative token gives a row of
        zeros. tokens: int32, any shape, `count` entries; out: count x width."""
        dev, width = self.ctx.device, self.width
        count = tokens.numel()
        code, ld, table_at = _rows(table, self.rows, width, dev, "table", _ALL)
        _, ldo, out_at = _rows(out, count, width, dev, "out", (code,))
        call("spmvb_embedding_lookup", self.handle, code, count, _flat(tokens, I32, count, dev, "tokens"), scale,
             table_at, ld, out_at, ldo, _stream(stream, dev))

    def lookup_grad(self, tokens, dout, dtable, scale: float = 1.0, accumulate: bool = False, stream=None) -> None:
        """dtable[r] = scale * sum of dout[t] over the tokens that name r, 0
        where none does; `accumulate` adds to dtable instead. dtable has
        dout's type or is float32."""
        dev, width = self.ctx.device, self.width
        count = tokens.numel()
        code, ldo, dout_at = _rows(dout, count, width, dev, "dout", _ALL)
        grad_code, ld, dtable_at = _rows(dtable, self.rows, width, dev, "dtable", (code,) if code == F64 else (code, F32))
        call("spmvb_embedding_lookup_grad", self.handle, code, count, _flat(tokens, I32, count, dev, "tokens"), scale,
             dout_at, ldo, grad_code, dtable_at, ld, int(accumulate), _stream(stream, dev))


class Router(_Handle):
    """Routing of tokens to `k` of `experts` and the exchange of rows with
    them (spmvb_router). `score` is "softmax" or "sigmoid"; with `groups` > 1
    only the `groups_kept` best groups of neighbouring experts can be chosen
    from, a group's value being the sum of its `group_top` best; weights are
    the chosen scores, divided by their sum if `renormalise`, times `scale`.
    float32, float16 and bfloat16; weights are float32, indices int32. Scratch
    for plans of up to `max_tokens` tokens."""

    _destroy = "spmvb_router_destroy"

    def __init__(self, ctx, experts: int, k: int, max_tokens: int, score: str = "softmax", renormalise: bool = True,
                 scale: float = 1.0, groups: int = 1, groups_kept: int | None = None, group_top: int = 1):
        spec = router_spec(experts, k, score, renormalise, scale, groups, groups_kept, group_top)
        max_tokens = _int32(max_tokens, "max_tokens")
        h = C.c_void_p()
        call("spmvb_router_create", ctx.handle, C.byref(spec), max_tokens, C.byref(h))
        self.handle, self.ctx = h, ctx
        self.experts, self.k, self.max_tokens = spec.experts, spec.k, max_tokens

    def route(self, logits, indices, weights, bias=None, offsets=None, order=None, position=None, stream=None) -> None:
        """The chosen experts of each row of logits (tokens x experts), best
        first, into indices and weights (tokens x k): ranked by score + bias
        (float32, one per expert), or by the logits without a bias; equal
        ones go to the lowest index; -1 with weight 0 where fewer than k are
        available (logit -inf or NaN). With offsets, order and position, also
        their plan (see plan)."""
        dev, k = self.ctx.device, self.k
        code, ld, logits_at = _rows(logits, None, self.experts, dev, "logits")
        tokens = logits.shape[0]
        n = tokens * k
        b = None if bias is None else _flat(bias, F32, self.experts, dev, "bias")
        if offsets is None and order is None and position is None:
            plan = (None, None, None)
        elif offsets is None or order is None or position is None:
            raise ValueError("offsets, order and position come together")
        else:
            plan = (_flat(offsets, I32, self.experts + 1, dev, "offsets"), _flat(order, I32, n, dev, "order"),
                    _flat(position, I32, n, dev, "position"))
        call("spmvb_router_route", self.handle, code, tokens, logits_at, ld, b,
             _flat(indices, I32, n, dev, "indices"), _flat(weights, F32, n, dev, "weights"), *plan,
             _stream(stream, dev))

    def route_grad(self, logits, indices, dweights, dlogits, stream=None) -> None:
        """dlogits (all of it) from the weights' gradient, the choice in
        `indices` held fixed."""
        dev = self.ctx.device
        code, ld, logits_at = _rows(logits, None, self.experts, dev, "logits")
        tokens = logits.shape[0]
        _, ldd, dlogits_at = _rows(dlogits, tokens, self.experts, dev, "dlogits", (code,))
        n = tokens * self.k
        call("spmvb_router_route_grad", self.handle, code, tokens, logits_at, ld,
             _flat(indices, I32, n, dev, "indices"), _flat(dweights, F32, n, dev, "dweights"), dlogits_at, ldd,
             _stream(stream, dev))

    def plan(self, indices, offsets, order, position, stream=None) -> None:
        """The choice by expert: expert e's rows are offsets[e] ..
        offsets[e + 1] - 1, row r is entry order[r] (token order[r] // k), and
        position (tokens x k) is the row of each entry, -1 for none. order is
        written up to offsets[experts]."""
        dev = self.ctx.device
        n = indices.numel()
        if n % self.k:
            raise ValueError(f"indices holds {n} entries; a multiple of k = {self.k} is needed")
        call("spmvb_router_plan", self.handle, n // self.k, _flat(indices, I32, n, dev, "indices"),
             _flat(offsets, I32, self.experts + 1, dev, "offsets"), _flat(order, I32, n, dev, "order"),
             _flat(position, I32, n, dev, "position"), _stream(stream, dev))

    def _exchange(self, position, by_token, by_row, by_token_name: str, by_row_name: str):
        """Checks the two row sets of an exchange; returns (code, tokens,
        width, position, by_token, its stride, rows, by_row, its stride)."""
        dev = self.ctx.device
        if len(getattr(by_token, "shape", ())) != 2:
            raise ValueError(f"{by_token_name} must be a matrix")
        tokens, width = by_token.shape
        code, ld, at = _rows(by_token, tokens, width, dev, by_token_name)
        _, ldr, row_at = _rows(by_row, None, width, dev, by_row_name, (code,))
        return code, tokens, width, _flat(position, I32, tokens * self.k, dev, "position"), at, ld, by_row.shape[0], row_at, ldr

    def dispatch(self, position, X, out, stream=None) -> None:
        """out[position[t, j]] = X[t]; rows that no position names are left."""
        code, tokens, width, pos, at, ld, rows, row_at, ldr = self._exchange(position, X, out, "X", "out")
        call("spmvb_router_dispatch", self.handle, code, tokens, width, pos, at, ld, rows, row_at, ldr,
             _stream(stream, self.ctx.device))

    def dispatch_grad(self, position, dout, dX, stream=None) -> None:
        """dX[t] = sum over j of dout[position[t, j]]."""
        code, tokens, width, pos, at, ld, rows, row_at, ldr = self._exchange(position, dX, dout, "dX", "dout")
        call("spmvb_router_dispatch_grad", self.handle, code, tokens, width, pos, rows, row_at, ldr, at, ld,
             _stream(stream, self.ctx.device))

    def combine(self, position, weights, Y, out, stream=None) -> None:
        """out[t] = sum over j of weights[t, j] * Y[position[t, j]]."""
        code, tokens, width, pos, at, ld, rows, row_at, ldr = self._exchange(position, out, Y, "out", "Y")
        dev = self.ctx.device
        call("spmvb_router_combine", self.handle, code, tokens, width, pos,
             _flat(weights, F32, tokens * self.k, dev, "weights"), rows, row_at, ldr, at, ld, _stream(stream, dev))

    def combine_grad(self, position, weights, Y, dout, dY, dweights, stream=None) -> None:
        """dY[position[t, j]] = weights[t, j] * dout[t] (rows that no position
        names are left; positions are distinct) and dweights[t, j] = the
        inner product of dout[t] and Y[position[t, j]]."""
        code, tokens, width, pos, at, ld, rows, row_at, ldr = self._exchange(position, dout, Y, "dout", "Y")
        dev = self.ctx.device
        n = tokens * self.k
        _, ldd, dY_at = _rows(dY, rows, width, dev, "dY", (code,))
        call("spmvb_router_combine_grad", self.handle, code, tokens, width, pos,
             _flat(weights, F32, n, dev, "weights"), rows, row_at, ldr, at, ld, dY_at, ldd,
             _flat(dweights, F32, n, dev, "dweights"), _stream(stream, dev))


def router_spec(experts: int, k: int, score: str = "softmax", renormalise: bool = True, scale: float = 1.0,
                groups: int = 1, groups_kept: int | None = None, group_top: int = 1) -> _lib.RouterSpec:
    """The checked description of a Router (no device needed)."""
    if score not in SCORES:
        raise ValueError(f"score must be one of {sorted(SCORES)}")
    kept = groups if groups_kept is None else groups_kept
    spec = _lib.RouterSpec(_int32(experts, "experts"), _int32(k, "k"), SCORES[score], int(bool(renormalise)),
                           _int32(groups, "groups"), _int32(kept, "groups_kept"), _int32(group_top, "group_top"), scale)
    call("spmvb_router_check", C.byref(spec))
    return spec


class GradClip(_Handle):
    """The 2-norm over all of `tensors`, and their scaling in place by
    min(1, max_norm / (norm + eps)) (spmvb_clip). float32, float16, bfloat16
    and float64, contiguous, none overlapping another.

    The handle keeps the tensors and works on their memory: they have to keep
    their storage (a replaced one is refused) and their sizes. A parameter's
    gradient is another tensor after zero_grad(set_to_none=True), which is
    torch's default: the handle then still holds the old ones, which nobody
    else does. Zero gradients in place, or make a new handle. With
    `parameters`, the tensors' owners, one each, a call is refused where a
    parameter's .grad is no longer its tensor."""

    _destroy = "spmvb_clip_destroy"

    def __init__(self, ctx, tensors, parameters=None):
        tensors = list(tensors)
        owners = [] if parameters is None else list(parameters)
        if parameters is not None and len(owners) != len(tensors):
            raise ValueError(f"{len(tensors)} tensors of {len(owners)} parameters")
        dev, codes = ctx.device, []
        for i, t in enumerate(tensors):
            codes.append(_code(t, _ALL, dev, f"tensor {i}"))
            if not t.is_contiguous():
                raise ValueError(f"tensor {i} must be contiguous")
        n = len(tensors)
        self._tensors, self._places, self._owners = tensors, [t.data_ptr() for t in tensors], owners
        self._check_owners()
        h = C.c_void_p()
        call("spmvb_clip_create", ctx.handle, n, (C.c_void_p * n)(*self._places),
             (C.c_int64 * n)(*[t.numel() for t in tensors]), (C.c_int * n)(*codes),
             C.byref(h))
        self.handle, self.ctx = h, ctx

    def _check_owners(self) -> None:
        for i, (p, t) in enumerate(zip(self._owners, self._tensors)):
            if p.grad is not t:
                raise ValueError(f"the gradient of parameter {i} is another tensor: make a new GradClip")

    def _check(self, norm) -> int:
        if self._owners:
            self._check_owners()
        if [t.data_ptr() for t in self._tensors] != self._places:
            raise ValueError("a tensor's storage has been replaced: make a new GradClip")
        return _flat(norm, F32, 1, self.ctx.device, "norm")

    def norm(self, norm, stream=None) -> None:
        """The norm into `norm` (one float32 on the device)."""
        call("spmvb_clip_norm", self.handle, self._check(norm), _stream(stream, self.ctx.device))

    def clip(self, max_norm: float, norm, eps: float = 1e-6, stream=None) -> None:
        """The norm before clipping into `norm`, then the scaling."""
        call("spmvb_clip_run", self.handle, max_norm, eps, self._check(norm), _stream(stream, self.ctx.device))

"""Low-rank adapters of many samples beside a trained VAE's layers, and 8-bit activation checkpoints (``csrc/adapt*.hip``).

One VAE is trained on the contigs of many samples (``vamb_amd.encode.VAE``); an adapter is a small correction of a layer for the
contigs of ONE sample -- a batch effect of its library, its depth, its host.  A batch holds contigs of many samples, so every call
serves all adapters at once.  With ``x [rows, k]``, the shared weight ``W [n, k]`` and bias ``b``, ``down = A [groups, rank, k]``, ``up = B
[groups, n, rank]`` and the group ``g`` of a row (a row whose group is outside ``[0, groups)``, -1 say, has no adapter)::

    u = x A_g^T     y = f(x W^T + b + scale u B_g^T)          f: identity, or LeakyReLU(negative_slope)
    p = dy f'(y)    v = scale p B_g     dx = p W + v A_g      dA_g = sum v^T x     dB_g = scale sum p^T u     dW = p^T x     db = sum p

What the backward pass needs of the forward pass waits as a :class:`Checkpoint8`: one byte per activation.

The functions take and return tensors of one GPU (float32 or bfloat16, all tensors of a call in one type; ``u`` is always float32), run on the current
stream of that GPU, do not synchronise and may be captured into a graph.  Memory comes from torch's allocator, so a tensor (a plan, a
packed weight, a checkpoint) that is used on another stream than the one that made it has to be ordered as any other
tensor has.  They stand outside of autograd: gradients come from :func:`adapted_linear_backward` and :func:`checkpoint_weight_grad`, for what
:func:`adapted_linear_train` returns; :func:`adapted_linear`, which keeps nothing for them, refuses tensors that require a gradient.
Sums are float32; gradients have the type of their parameters.  Of bf16 tensors ``u`` and ``v`` are multiplied in 24 bits, ``p`` in 16 where the slope
applies; of float32 tensors the products of the last bits are dropped (2^-21 of a product at most).  Equal inputs give equal bits.

:class:`VAEAdapters` trains adapters for a VAE's encoder and encodes with them.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Optional, Union

import torch as _torch

from . import _lib

MAX_RANK = 64
MAX_GROUPS = 16384
BLOCK = 32   # columns of a checkpoint that share an exponent
# Up to this cost adapted_linear goes without a plan: one launch, in which each workgroup (16 rows, 16 columns) reads the adapters of its rows.
# Cost = (adapters that 16 rows can have x pieces of 16 ranks x k + 1000) x rounds of 256 workgroups.  Times of a call, that launch against
# plan and projection: bf16 304 -> 512, rank 8, 64 rows of 200 groups 10 us / 16 (cost 5900); 1104 -> 512, rank 16, 8 rows of 200 groups 13 / 16 (9800), 16 rows
# 23 / 16 (18700); 32 -> 512, rank 1, 5000 rows of 200 groups 54 / 16 (59000); float32 (six products for one) 512 -> 512, rank 1, 8 rows of 200 groups 15 / 17
# (5100), 17 rows 27 / 17 (9200).  Over 420 drawn calls this takes 1.004 of the faster way's time in the mean, 1.54 at worst.  One or two rows always
# (512 -> 512, rank 64, one row: bf16 9.3 / 15, float32 12 / 29).
_FEW = {_torch.bfloat16: 12_000, _torch.float32: 8_000}


def _few_cost(rows: int, n: int, k: int, rank: int, groups: int) -> float:
    return (min(16, rows, groups) * -(-rank // 16) * k + 1000) * max(1.0, -(-rows // 16) * -(-n // 16) / 256)


_DTYPES = {_torch.float32: 0, _torch.bfloat16: 1}
# the current stream's handle without a Stream object around it (a call here is a few microseconds in all)
_raw_stream = getattr(_torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: _torch.cuda.current_stream(index).cuda_stream)


def _dtype_of(t: _torch.Tensor, what: str) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise ValueError(f"{what} must be float32 or bfloat16, not {t.dtype}") from None


def _matrix(t, what: str, rows: Optional[int] = None, cols: Optional[int] = None) -> int:
    """Check a [rows, cols] tensor whose rows are contiguous; returns its row stride."""
    if not isinstance(t, _torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{what} must be a two-dimensional tensor")
    n, m = t.shape
    if (rows is not None and n != rows) or (cols is not None and m != cols):
        raise ValueError(f"{what} must be [{'rows' if rows is None else rows}, {'columns' if cols is None else cols}], not {[n, m]}")
    ld, step = t.stride()
    if m > 1 and step != 1:
        raise ValueError(f"the rows of {what} must be contiguous")
    if n <= 1:
        return m
    if ld < m:
        raise ValueError(f"the rows of {what} overlap (row stride {ld}, {m} columns)")
    return ld


def _dense(t, what: str, shape) -> None:
    if not isinstance(t, _torch.Tensor) or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be {list(shape)}, not {list(getattr(t, 'shape', ()))}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _enter(first, *others):
    """The library's side of a call: all tensors on one GPU, that GPU current; ``(its stream, the device to go back to or None)``."""
    index = first.get_device()
    if index < 0:
        raise ValueError(f"the tensors must be on a GPU, not on {first.device}")
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"the tensors of a call must be on one device: {first.device} and {t.device}")
    before = _torch.cuda.current_device()
    if before == index:
        return _raw_stream(index), None
    _torch.cuda.set_device(index)
    return _raw_stream(index), before


def _leave(before) -> None:
    if before is not None:
        _torch.cuda.set_device(before)


@lru_cache(maxsize=4096)
def _plan_words(rows: int, groups: int):
    a, b = ctypes.c_int64(), ctypes.c_int64()
    _lib.check(_lib.load().vh_rows_plan_size(rows, groups, ctypes.byref(a), ctypes.byref(b)))
    return a.value, b.value


@lru_cache(maxsize=4096)
def _backward_words(rows: int, groups: int, n: int, k: int, rank: int, dtype: int) -> int:
    a = ctypes.c_int64()
    _lib.check(_lib.load().vh_adapt_backward_size(rows, groups, n, k, rank, dtype, ctypes.byref(a)))
    return a.value


@lru_cache(maxsize=4096)
def _weight_grad_words(rows: int, n: int, k: int) -> int:
    a = ctypes.c_int64()
    _lib.check(_lib.load().vh_checkpoint8_weight_grad_size(rows, n, k, ctypes.byref(a)))
    return a.value


# ---- which rows an adapter serves -----------------------------------------------------------------------------------------------
class RowGroups:
    """The rows of a batch sorted by group (:func:`group_rows`): made once per batch, read by every layer's forward and backward."""

    __slots__ = ("rows", "groups", "plan")

    def __init__(self, rows: int, groups: int, plan: Optional[_torch.Tensor]):
        self.rows, self.groups, self.plan = rows, groups, plan


def _check_groups(groups, n_groups: int) -> None:
    if not isinstance(groups, _torch.Tensor) or groups.dim() != 1 or groups.dtype != _torch.int32:
        raise ValueError("groups must be a one-dimensional int32 tensor (or what group_rows made of one)")
    if not groups.is_contiguous():
        raise ValueError("groups must be contiguous")
    if not 1 <= n_groups <= MAX_GROUPS:
        raise ValueError(f"the number of groups must be in [1, {MAX_GROUPS}], not {n_groups}")


def group_rows(groups: _torch.Tensor, n_groups: int) -> RowGroups:
    """Sort the rows of a batch by their group: ``groups`` int32 ``[rows]``; values outside ``[0, n_groups)`` are rows without an adapter."""
    _check_groups(groups, n_groups)
    rows = groups.shape[0]
    if rows == 0:
        return RowGroups(0, n_groups, None)
    lib = _lib.load()
    stream, before = _enter(groups)
    try:
        words, scratch_words = _plan_words(rows, n_groups)
        plan = _torch.empty(words, dtype=_torch.int32, device=groups.device)
        scratch = _torch.empty(scratch_words, dtype=_torch.int32, device=groups.device) if scratch_words else None
        _lib.check(lib.vh_rows_plan(groups.data_ptr(), rows, n_groups, plan.data_ptr(), scratch.data_ptr() if scratch is not None else None, stream))
    finally:
        _leave(before)
    return RowGroups(rows, n_groups, plan)


# ---- the shared projection ------------------------------------------------------------------------------------------------------
class SharedProjection:
    """``weight [n, k]`` and ``bias [n]`` of a layer that all adapters share, laid out once for both directions (a copy: later
    changes of ``weight`` are not seen; make another)."""

    def __init__(self, weight: _torch.Tensor, bias: Optional[_torch.Tensor] = None):
        ld = _matrix(weight, "weight")
        self.dtype = weight.dtype
        code = _dtype_of(weight, "weight")
        self.n, self.k = weight.shape
        if self.n < 1 or self.k < 1:
            raise ValueError("weight must not be empty")
        if bias is not None:
            _dense(bias, "bias", (self.n,))
            if bias.dtype != weight.dtype:
                raise ValueError(f"bias must have the weight's type {weight.dtype}, not {bias.dtype}")
        self.device = weight.device
        lib = _lib.load()
        stream, before = _enter(weight, bias)
        try:
            size = ctypes.c_int64()
            _lib.check(lib.vh_adapt_weight_size(self.n, self.k, code, ctypes.byref(size)))
            self.packed = _torch.empty(size.value, dtype=_torch.uint8, device=weight.device)
            _lib.check(lib.vh_adapt_weight_pack(weight.data_ptr(), ld, bias.data_ptr() if bias is not None else None, self.n, self.k, code,
                                                self.packed.data_ptr(), stream))
        finally:
            _leave(before)


def _layer(shared, down, up, n_groups, scale, negative_slope):
    """Check a layer's adapters and describe it to the library."""
    if not isinstance(shared, SharedProjection):
        raise ValueError("shared must be a SharedProjection")
    if not isinstance(down, _torch.Tensor) or down.dim() != 3:
        raise ValueError("down must be a tensor [groups, rank, k]")
    groups, rank = down.shape[:2]
    if groups != n_groups:
        raise ValueError(f"down holds {groups} adapters, the rows' groups are {n_groups}")
    if not 1 <= rank <= MAX_RANK:
        raise ValueError(f"the rank must be in [1, {MAX_RANK}], not {rank}")
    _dense(down, "down", (groups, rank, shared.k))
    _dense(up, "up", (groups, shared.n, rank))
    if down.dtype != shared.dtype or up.dtype != shared.dtype:
        raise ValueError(f"down and up must have the weight's type {shared.dtype}, not {down.dtype} and {up.dtype}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, not {scale}")
    _check_slope(negative_slope)
    return _lib.AdaptLayer(_DTYPES[shared.dtype], int(negative_slope is not None), shared.n, shared.k, rank, groups, shared.packed.data_ptr(),
                           down.data_ptr(), up.data_ptr(), scale, 0.0 if negative_slope is None else negative_slope)


def _check_slope(negative_slope) -> None:
    if negative_slope is not None and not 0.0 <= negative_slope < math.inf:
        raise ValueError(f"negative_slope must be finite and >= 0 (the derivative is read from the sign of the result), not {negative_slope}")


def _input(x, shared) -> int:
    if not isinstance(shared, SharedProjection):
        raise ValueError("shared must be a SharedProjection")
    ld = _matrix(x, "x", None, shared.k)
    if x.dtype != shared.dtype:
        raise ValueError(f"x must have the weight's type {shared.dtype}, not {x.dtype}")
    return ld


def adapted_linear(x, shared: SharedProjection, down, up, groups: Union[_torch.Tensor, RowGroups], scale: float = 1.0,
                   negative_slope: Optional[float] = None) -> _torch.Tensor:
    """``f(x W^T + b + scale u B_g^T)``, ``[rows, n]``: the layer with every row's own adapter.

    ``groups``: an int32 tensor ``[rows]``, or the :class:`RowGroups` of these rows where several layers use it.  ``x`` may have any row stride.
    For inference: where autograd is on, tensors that require a gradient are refused (the result would have none)."""
    ld = _input(x, shared)
    rows = x.shape[0]
    planned = isinstance(groups, RowGroups)
    n_groups = groups.groups if planned else (down.shape[0] if isinstance(down, _torch.Tensor) and down.dim() == 3 else 0)
    layer = _layer(shared, down, up, n_groups, scale, negative_slope)
    if _torch.is_grad_enabled() and (x.requires_grad or down.requires_grad or up.requires_grad):
        raise ValueError("adapted_linear gives no gradients: call it under torch.no_grad() or on detached tensors, or use adapted_linear_train "
                         "with adapted_linear_backward")
    if not planned:
        _check_groups(groups, n_groups)
    if (groups.rows if planned else groups.shape[0]) != rows:
        raise ValueError(f"x has {rows} rows, groups {groups.rows if planned else groups.shape[0]}")
    lib = _lib.load()
    stream, before = _enter(x, shared.packed, down, up, groups.plan if planned else groups)
    try:
        y = x.new_empty((rows, shared.n))
        if rows == 0:
            return y
        if not planned and (rows <= 2 or _few_cost(rows, shared.n, shared.k, down.shape[1], n_groups) <= _FEW[x.dtype]):
            _lib.check(lib.vh_adapt_forward_few(layer, x.data_ptr(), ld, rows, groups.data_ptr(), y.data_ptr(), shared.n, stream))
            return y
        if not planned:
            groups = group_rows(groups, n_groups)
        _lib.check(lib.vh_adapt_forward(layer, x.data_ptr(), ld, rows, groups.plan.data_ptr(), y.data_ptr(), shared.n, None, None, None, stream))
    finally:
        _leave(before)
    return y


def adapted_linear_train(x, shared: SharedProjection, down, up, groups: RowGroups, scale: float = 1.0, negative_slope: Optional[float] = None):
    """``(y, u, checkpoint of y)``: :func:`adapted_linear` with what the backward pass needs -- the small product ``u [rows, rank]`` in
    float32, and ``y`` as a :class:`Checkpoint8`, written by the same launch."""
    ld = _input(x, shared)
    rows = x.shape[0]
    if not isinstance(groups, RowGroups):
        raise ValueError("groups must come from group_rows")
    layer = _layer(shared, down, up, groups.groups, scale, negative_slope)
    if groups.rows != rows:
        raise ValueError(f"x has {rows} rows, groups {groups.rows}")
    lib = _lib.load()
    stream, before = _enter(x, shared.packed, down, up, groups.plan)
    try:
        y = x.new_empty((rows, shared.n))
        low = _torch.empty((rows, down.shape[1]), dtype=_torch.float32, device=x.device)
        held = Checkpoint8._empty(rows, shared.n, x.device)
        if rows:
            _lib.check(lib.vh_adapt_forward(layer, x.data_ptr(), ld, rows, groups.plan.data_ptr(), y.data_ptr(), shared.n, low.data_ptr(),
                                            *held._at, stream))
    finally:
        _leave(before)
    return y, low, held


def adapted_linear_backward(dy, x, y, low, shared: SharedProjection, down, up, groups: RowGroups, scale: float = 1.0,
                            negative_slope: Optional[float] = None, need_dx: bool = True):
    """``(dx, ddown, dup)`` of :func:`adapted_linear_train`; ``dx`` is None with ``need_dx=False`` (a first layer), the
    others are the same bits.

    ``x`` and ``y`` are the layer's input and output, as tensors or checkpoints (``y`` may be None without an activation: it gives
    the derivative); ``low`` is its ``u``.  The gradients of a group without rows are zero."""
    if not isinstance(groups, RowGroups):
        raise ValueError("groups must come from group_rows")
    layer = _layer(shared, down, up, groups.groups, scale, negative_slope)
    ld = _matrix(dy, "dy", groups.rows, shared.n)
    rows, rank = groups.rows, down.shape[1]
    if dy.dtype != shared.dtype:
        raise ValueError(f"dy must have the weight's type {shared.dtype}, not {dy.dtype}")
    if negative_slope is not None and y is None:
        raise ValueError("y is needed for the derivative of the activation")
    held_x, tx = _held(x, "x", rows, shared.k, dy.dtype)
    held_y, ty = _held(y, "y", rows, shared.n, dy.dtype) if y is not None else (None, None)
    _dense(low, "low", (rows, rank))
    if low.dtype != _torch.float32:
        raise ValueError(f"low must be float32, not {low.dtype}")
    lib = _lib.load()
    stream, before = _enter(dy, shared.packed, down, up, groups.plan, tx, ty, low)
    try:
        dx = dy.new_empty((rows, shared.k)) if need_dx else None
        if rows == 0:
            return dx, _torch.zeros_like(down), _torch.zeros_like(up)
        ddown, dup = _torch.empty_like(down), _torch.empty_like(up)
        scratch = _torch.empty(_backward_words(rows, groups.groups, shared.n, shared.k, rank, layer.dtype), dtype=_torch.float32, device=dy.device)
        _lib.check(lib.vh_adapt_backward(layer, dy.data_ptr(), ld, held_x, held_y, low.data_ptr(), rows, groups.plan.data_ptr(),
                                         dx.data_ptr() if need_dx else None, shared.k, ddown.data_ptr(), dup.data_ptr(), scratch.data_ptr(), stream))
    finally:
        _leave(before)
    return dx, ddown, dup


# ---- checkpoints ----------------------------------------------------------------------------------------------------------------
class Checkpoint8:
    """A matrix ``[rows, columns]`` held in one byte per element: ``codes`` uint8 ``[rows, columns rounded up to 32]``, e4m3 bits of
    ``x 2^-e``, and ``exponents`` uint8 ``[rows, columns / 32 rounded up]``, ``e + 127`` of every 32 columns.  Those made by hand keep to
    what is written here: exponent bytes in [10, 247], and codes of value zero behind the last column.

    ``e`` is the least with ``amax <= 448 * 2^e`` over the block's finite magnitudes, kept in [-117, 120]; codes are rounded to nearest even
    (2^-4 relative to the value, 2^-10 of the block's scale near zero), their sign bit is set where ``x > 0`` does not hold (the derivative
    of LeakyReLU can be read from it), a non-finite element is NaN, and magnitudes that would round to
    2^128 become 240 * 2^120.  Every value is exact in bfloat16."""

    __slots__ = ("columns", "_rows", "_memory", "_codes", "_exponents", "_at")

    def __init__(self, codes: _torch.Tensor, exponents: _torch.Tensor, columns: int):
        if columns < 1:
            raise ValueError(f"a checkpoint has at least one column, not {columns}")
        if not isinstance(codes, _torch.Tensor) or codes.dim() != 2 or codes.dtype != _torch.uint8:
            raise ValueError("codes must be a uint8 tensor [rows, columns rounded up to 32]")
        blocks = -(-columns // BLOCK)
        _dense(codes, "codes", (codes.shape[0], BLOCK * blocks))
        _dense(exponents, "exponents", (codes.shape[0], blocks))
        if exponents.dtype != _torch.uint8:
            raise ValueError("exponents must be uint8")
        if exponents.device != codes.device:
            raise ValueError("codes and exponents must be on one device")
        if codes.numel() and codes.data_ptr() % 8:
            raise ValueError("codes must be 8-byte aligned")
        self.columns, self._rows = columns, codes.shape[0]
        self._memory = self._codes = codes
        self._exponents = exponents
        self._at = codes.data_ptr(), exponents.data_ptr()   # what the library is given

    @classmethod
    def _empty(cls, rows: int, columns: int, device):
        """Memory for a checkpoint: one allocation, codes before exponents (the tensors of both are made when somebody asks)."""
        blocks = -(-columns // BLOCK)
        self = cls.__new__(cls)
        self.columns, self._rows = columns, rows
        self._memory = _torch.empty(rows * blocks * (BLOCK + 1), dtype=_torch.uint8, device=device)
        self._codes = self._exponents = None
        at = self._memory.data_ptr()
        self._at = at, at + rows * blocks * BLOCK
        return self

    @property
    def codes(self) -> _torch.Tensor:
        if self._codes is None:
            width = BLOCK * -(-self.columns // BLOCK)
            self._codes = self._memory[:self._rows * width].view(self._rows, width)
        return self._codes

    @property
    def exponents(self) -> _torch.Tensor:
        if self._exponents is None:
            blocks = -(-self.columns // BLOCK)
            self._exponents = self._memory[self._rows * blocks * BLOCK:].view(self._rows, blocks)
        return self._exponents

    @property
    def shape(self):
        return _torch.Size((self._rows, self.columns))

    def restore(self, dtype: _torch.dtype = _torch.float32) -> _torch.Tensor:
        """The values that the codes stand for, ``[rows, columns]`` (exact in either type)."""
        if dtype not in _DTYPES:
            raise ValueError(f"a checkpoint is restored to float32 or bfloat16, not {dtype}")
        rows = self._rows
        lib = _lib.load()
        stream, before = _enter(self._memory)
        try:
            out = self._memory.new_empty((rows, self.columns), dtype=dtype)
            if rows:
                _lib.check(lib.vh_checkpoint8_restore(*self._at, rows, self.columns, _DTYPES[dtype],
                                                      out.data_ptr(), stream))
        finally:
            _leave(before)
        return out


def checkpoint8(x: _torch.Tensor) -> Checkpoint8:
    """Hold ``x [rows, columns]`` for the backward pass in one byte per element."""
    ld = _matrix(x, "x")
    code = _dtype_of(x, "x")
    rows, columns = x.shape
    if columns < 1:
        raise ValueError("x must have at least one column")
    lib = _lib.load()
    stream, before = _enter(x)
    try:
        held = Checkpoint8._empty(rows, columns, x.device)
        if rows:
            _lib.check(lib.vh_checkpoint8(x.data_ptr(), ld, rows, columns, code, *held._at, stream))
    finally:
        _leave(before)
    return held


def _held(t, what: str, rows: int, cols: int, dtype):
    if isinstance(t, Checkpoint8):
        if t._rows != rows or t.columns != cols:
            raise ValueError(f"the checkpoint {what} must be [{rows}, {cols}], not {list(t.shape)}")
        return _lib.Held(None, 0, *t._at), t._memory
    ld = _matrix(t, what, rows, cols)
    if t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, not {t.dtype}")
    return _lib.Held(t.data_ptr(), ld, None, None), t


def checkpoint_weight_grad(dy, x: Checkpoint8, y=None, negative_slope: Optional[float] = None):
    """``(dW, db)`` of a layer whose input waited as a checkpoint: ``p^T x [n, k]`` and ``sum p [n]`` with ``p = dy f'(y)``.

    ``y`` (tensor or checkpoint) and ``negative_slope`` come together for a layer with LeakyReLU; without them ``p = dy``."""
    if not isinstance(x, Checkpoint8):
        raise ValueError("x must be a Checkpoint8")
    rows, k = x.shape
    ld = _matrix(dy, "dy", rows)
    code = _dtype_of(dy, "dy")
    n = dy.shape[1]
    if n < 1:
        raise ValueError("dy must have at least one column")
    _check_slope(negative_slope)
    if negative_slope is not None and y is None:
        raise ValueError("y is needed for the derivative of the activation")
    held_x, tx = _held(x, "x", rows, k, dy.dtype)
    # (without an activation y plays no part, as in adapted_linear_backward)
    held_y, ty = _held(y, "y", rows, n, dy.dtype) if y is not None else (None, None)
    lib = _lib.load()
    stream, before = _enter(dy, tx, ty)
    try:
        if rows == 0:
            return _torch.zeros((n, k), dtype=dy.dtype, device=dy.device), _torch.zeros(n, dtype=dy.dtype, device=dy.device)
        dweight = dy.new_empty((n, k))
        dbias = dy.new_empty(n)
        scratch = _torch.empty(_weight_grad_words(rows, n, k), dtype=_torch.float32, device=dy.device)
        _lib.check(lib.vh_checkpoint8_weight_grad(dy.data_ptr(), ld, held_x, held_y if negative_slope is not None else None,
                                                  negative_slope or 0.0, rows, n, k, code, dweight.data_ptr(), dbias.data_ptr(), scratch.data_ptr(), stream))
    finally:
        _leave(before)
    return dweight, dbias


# ---- adapters of a trained VAE --------------------------------------------------------------------------------------------------
_SLOPE = 0.01       # torch.nn.LeakyReLU's default (encode.py:264)
_BN_EPS = 1e-5


class VAEAdapters:
    """Low-rank adapters of a trained :class:`vamb_amd.encode.VAE`, one set per sample: trained on the VAE's own loss with the VAE's weights
    and BatchNorm statistics as they are, and used to encode.  (The reference has no counterpart: its VAE treats all samples alike.)

    Every Linear of the encoder (the hidden layers and ``mu``) has an adapter of ``rank`` per group; the decoder is as it was trained.  The
    BatchNorm of a layer (eval mode, encode.py:264) is folded into the Linear behind it, so an adapter reads the layer's input in front of that BatchNorm.
    A new adapter changes nothing (``up`` is zero).  Arithmetic in ``dtype`` (default: the VAE's compute type), ``mu`` always
    in float32; parameters and their optimiser (torch's Adam) in float32.  Activations wait for the backward pass as 8-bit checkpoints (a byte
    each; the inputs in the gradients of ``down`` and of ``mu`` are then within 2^-4 of their values, whatever ``dtype`` is), or, with
    ``checkpoints=False``, as they are.

    ``groups``: the sample of each contig of the data set, integers; a value outside ``[0, n_groups)`` stands for a contig without an adapter."""

    def __init__(self, vae, n_groups: int, rank: int = 8, scale: float = 1.0, seed: int = 0, dtype: Optional[_torch.dtype] = None,
                 device: Union[str, _torch.device] = "cuda", checkpoints: bool = True):
        from . import encode as _encode
        if type(vae) is not _encode.VAE:
            raise ValueError("adapters are made for a plain VAE")
        if not 1 <= n_groups <= MAX_GROUPS:
            raise ValueError(f"the number of groups must be in [1, {MAX_GROUPS}], not {n_groups}")
        if not 1 <= rank <= MAX_RANK:
            raise ValueError(f"the rank must be in [1, {MAX_RANK}], not {rank}")
        if not math.isfinite(scale):
            raise ValueError(f"scale must be finite, not {scale}")
        if dtype is None:
            dtype = _torch.bfloat16 if vae.compute_dtype == "bf16" else _torch.float32
        if dtype not in _DTYPES:
            raise ValueError(f"dtype must be float32 or bfloat16, not {dtype}")
        self.nsamples, self.nlatent, self.alpha, self.beta = vae.nsamples, vae.nlatent, vae.alpha, vae.beta
        self.ntnf = vae.ntnf
        self.n_groups, self.rank, self.scale, self.dtype = n_groups, rank, float(scale), dtype
        self.checkpoints = bool(checkpoints)
        device = _torch.device(device)
        self.device = _torch.device("cuda", _torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device
        state = {k: v.double() for k, v in vae.state_dict().items()}
        self._mu_weight = self._mu_bias = None
        n = len(vae.nhiddens)
        self._encoder = self._folded(state, "encoder", n, "mu")
        self._decoder = self._folded(state, "decoder", n, "outputlayer")
        g = _torch.Generator(device="cpu").manual_seed(seed)
        self.down, self.up = [], []
        for s in self._encoder:
            bound = s.k ** -0.5
            d = (_torch.rand((n_groups, rank, s.k), generator=g) * 2 - 1) * bound
            self.down.append(d.to(self.device))
            self.up.append(_torch.zeros((n_groups, s.n, rank), device=self.device))
        self._generator = _torch.Generator(device=self.device).manual_seed(seed)
        # the decoder's layers have no adapters: no row asks for this one
        self._none = [(_torch.zeros((1, 1, s.k), dtype=s.dtype, device=self.device), _torch.zeros((1, s.n, 1), dtype=s.dtype, device=self.device))
                      for s in self._decoder]

    def _folded(self, state, kind: str, n: int, last: str):
        """The layers' weights with the BatchNorm in front of each folded in: W (a x + c) + b = (W a) x + (W c + b)."""
        layers, a, c = [], None, None
        for i, name in enumerate([f"{kind}layers.{i}" for i in range(n)] + [last]):
            w, b = state[name + ".weight"], state[name + ".bias"]
            if a is not None:
                w, b = w * a, w @ c + b
            dtype = _torch.float32 if name == "mu" else self.dtype
            w, b = (t.float().to(self.device, dtype).contiguous() for t in (w, b))
            if name == "mu":
                self._mu_weight, self._mu_bias = w, b
            layers.append(SharedProjection(w, b))
            if i < n:
                norm = f"{kind}norms.{i}"
                a = state[norm + ".weight"] / (state[norm + ".running_var"] + _BN_EPS).sqrt()
                c = state[norm + ".bias"] - state[norm + ".running_mean"] * a
        return layers

    def _pairs(self):
        """The adapters in the types that the layers compute in."""
        return [(d.to(s.dtype), u.to(s.dtype)) for d, u, s in zip(self.down, self.up, self._encoder)]

    # ---- data -------------------------------------------------------------------------------------------------------------------
    def _features(self, data_loader):
        tensors = data_loader.dataset.tensors
        if len(tensors) != 4:
            raise ValueError("expected a DataLoader made by make_dataloader (4 tensors)")
        parts = [_torch.as_tensor(t[:]) for t in tensors]
        n = len(parts[0])
        if parts[0].shape != (n, self.nsamples) or parts[1].shape != (n, self.ntnf) or parts[2].shape != (n, 1) or parts[3].shape != (n, 1):
            raise ValueError("dataset tensors do not match this VAE (nsamples / 103 TNF / 1 / 1 columns)")
        return _torch.cat(parts[:3], dim=1).to(self.device), parts[3].to(self.device)

    def _groups(self, groups, n: int) -> _torch.Tensor:
        g = _torch.as_tensor(groups)
        if g.dim() != 1 or len(g) != n or g.dtype.is_floating_point or g.dtype in (_torch.bool, _torch.complex64, _torch.complex128):
            raise ValueError(f"groups must be {n} integers, one per contig")
        g = g.to(self.device, _torch.int64)
        return _torch.where((g >= 0) & (g < self.n_groups), g, -1).to(_torch.int32)

    # ---- encode -----------------------------------------------------------------------------------------------------------------
    @_torch.no_grad()
    def encode(self, data_loader, groups, batchsize: int = 262144):
        """Latents ``[n, nlatent]`` like ``VAE.encode`` (float32, the low 12 mantissa bits cleared, vambtools.py:324-330)."""
        if batchsize < 1:
            raise ValueError(f"batchsize must be at least 1, not {batchsize}")
        x, _ = self._features(data_loader)
        g = self._groups(groups, len(x))
        pairs = self._pairs()
        out = []
        for at in range(0, len(x), batchsize):
            plan = group_rows(g[at:at + batchsize], self.n_groups)
            h = x[at:at + batchsize].to(self.dtype)
            for i, (s, (d, u)) in enumerate(zip(self._encoder, pairs)):
                last = i == len(pairs) - 1
                h = adapted_linear(h.to(s.dtype), s, d, u, plan, self.scale, None if last else _SLOPE)
            out.append((h.view(_torch.int32) & ~0xfff).view(_torch.float32))
        if not out:
            return _torch.empty((0, self.nlatent)).numpy()
        return _torch.cat(out).cpu().numpy()

    # ---- training ---------------------------------------------------------------------------------------------------------------
    def gradients(self, x, weights, groups, noise, mu_too: bool = False):
        """``(loss, gradients of down, gradients of up, gradients of mu's weight and bias or None)`` of one batch: ``x`` float32 ``[rows, columns]``,
        ``weights`` ``[rows, 1]``, ``groups`` int32 ``[rows]``, ``noise`` the reparameterisation noise ``[rows, nlatent]``.  The loss is
        ``VAE.calc_loss`` (encode.py:316-357), whose ``[rows] * [rows, 1]`` means the product of two means."""
        rows = len(x)
        plan, alone = group_rows(groups, self.n_groups), group_rows(_torch.full_like(groups, -1), 1)
        pairs = self._pairs()
        last = len(pairs) - 1
        # forward: every layer leaves its input and its output (whose signs are the derivative), as checkpoints or as they are
        h, held, low = x.to(self.dtype), [], []
        c = checkpoint8(h) if self.checkpoints else None
        for i, (s, (d, u)) in enumerate(zip(self._encoder, pairs)):
            below, h = c, h.to(s.dtype)
            y, l, c = adapted_linear_train(h, s, d, u, plan, self.scale, None if i == last else _SLOPE)
            held.append((below, c) if self.checkpoints else (h, y))
            low.append(l)
            h = y
        mu = h
        h = (mu + noise).to(self.dtype)
        kept = []
        c = checkpoint8(h) if self.checkpoints else None
        for i, (s, (d, u)) in enumerate(zip(self._decoder, self._none)):
            below = c
            y, zero, c = adapted_linear_train(h, s, d, u, alone, 0.0, None if i == len(self._decoder) - 1 else _SLOPE)
            kept.append((below, c, zero) if self.checkpoints else (h, y, zero))
            h = y
        out = h.float()
        # loss and its gradient
        ns, nt = self.nsamples, self.ntnf
        mean_w = weights.mean()
        per = mean_w / rows
        do = _torch.empty_like(out)
        ab_w, sse_w, kld_w = (1 - self.alpha) / ns, self.alpha / nt, 1 / (self.nlatent * self.beta)
        diff = out[:, ns:] - x[:, ns:]
        loss = (diff[:, :nt].square().sum(1) * sse_w + diff[:, nt:].square().sum(1) * ab_w + 0.5 * mu.square().sum(1) * kld_w)
        do[:, ns:ns + nt] = diff[:, :nt] * (2 * sse_w * per)
        do[:, ns + nt:] = diff[:, nt:] * (2 * ab_w * per)
        if ns > 1:
            ce_w = (1 - self.alpha) * (ns - 1) / (ns * math.log(ns))
            p = _torch.softmax(out[:, :ns], dim=1)
            loss = loss - ((p + 1e-9).log() * x[:, :ns]).sum(1) * ce_w
            dp = x[:, :ns] / (p + 1e-9)
            do[:, :ns] = p * ((dp * p).sum(1, keepdim=True) - dp) * (ce_w * per)
        else:
            do[:, :ns] = 0.0
        loss = loss.mean() * mean_w
        # backward
        dh = do.to(self.dtype)
        for i in range(len(self._decoder) - 1, -1, -1):
            below, c, zero = kept[i]
            dh, _, _ = adapted_linear_backward(dh, below, c, zero, self._decoder[i], *self._none[i], alone, 0.0,
                                               None if i == len(self._decoder) - 1 else _SLOPE)
        dh = dh.float() + mu * (kld_w * per)
        downs, ups, shared = [None] * (last + 1), [None] * (last + 1), None
        for i in range(last, -1, -1):
            s, (d, u) = self._encoder[i], pairs[i]
            slope = None if i == last else _SLOPE
            below, c = held[i]
            if i == last and mu_too:   # (of tensors as they are: a product of nlatent columns, torch's)
                shared = checkpoint_weight_grad(dh, below) if self.checkpoints else (dh.t() @ below, dh.sum(0))
            dh, dd, du = adapted_linear_backward(dh.to(s.dtype), below, c, low[i], s, d, u, plan, self.scale, slope, need_dx=i > 0)
            downs[i], ups[i] = dd.float(), du.float()
        return loss, downs, ups, shared

    def train(self, data_loader, groups, nepochs: int = 10, batchsize: int = 4096, lrate: float = 1e-3, mu_too: bool = False):
        """Train the adapters (Adam) for ``nepochs`` epochs over shuffled batches; ``mu_too``: the shared ``mu`` layer with them.  Returns
        the mean loss of every epoch."""
        if nepochs < 1:
            raise ValueError(f"Minimum 1 epoch, not {nepochs}")
        if batchsize < 1:
            raise ValueError(f"batchsize must be at least 1, not {batchsize}")
        if not lrate > 0:
            raise ValueError(f"lrate must be > 0, not {lrate}")
        x, w = self._features(data_loader)
        g = self._groups(groups, len(x))
        n = len(x)
        if n < 1:
            raise ValueError("cannot train on a dataset without sequences")
        batch = min(batchsize, n)
        shared = [self._mu_weight, self._mu_bias] if mu_too else []
        params = [*self.down, *self.up, *shared]
        optimizer = _torch.optim.Adam(params, lr=lrate)
        losses = []
        for _ in range(nepochs):
            order = _torch.randperm(n, generator=self._generator, device=self.device)
            total = []
            for at in range(0, n - batch + 1, batch):     # the ragged tail is dropped, as by make_dataloader's loader
                rows = order[at:at + batch]
                noise = _torch.randn((batch, self.nlatent), generator=self._generator, device=self.device)
                loss, downs, ups, mu_grads = self.gradients(x[rows], w[rows], g[rows], noise, mu_too)
                for p, grad in zip(params, [*downs, *ups, *(mu_grads or ())]):
                    p.grad = grad
                optimizer.step()
                optimizer.zero_grad(set_to_none=True)
                if mu_too:
                    self._encoder[-1] = SharedProjection(self._mu_weight, self._mu_bias)
                total.append(loss)
            losses.append(float(_torch.stack(total).mean()))
        return losses

    # ---- files ------------------------------------------------------------------------------------------------------------------
    def save(self, file) -> None:
        _torch.save({"n_groups": self.n_groups, "rank": self.rank, "scale": self.scale, "down": [t.cpu() for t in self.down],
                     "up": [t.cpu() for t in self.up], "mu": [self._mu_weight.cpu(), self._mu_bias.cpu()]}, file)

    @classmethod
    def load(cls, file, vae, dtype: Optional[_torch.dtype] = None, device: Union[str, _torch.device] = "cuda", checkpoints: bool = True):
        """Adapters that :meth:`save` wrote, on the VAE that they were made for."""
        d = _torch.load(file, map_location="cpu", weights_only=True)
        self = cls(vae, d["n_groups"], d["rank"], d["scale"], dtype=dtype, device=device, checkpoints=checkpoints)
        for mine, saved in ((self.down, d["down"]), (self.up, d["up"])):
            if [tuple(t.shape) for t in mine] != [tuple(t.shape) for t in saved]:
                raise ValueError("the saved adapters do not match this VAE")
            for m, t in zip(mine, saved):
                m.copy_(t)
        self._mu_weight, self._mu_bias = (t.to(self.device) for t in d["mu"])
        self._encoder[-1] = SharedProjection(self._mu_weight, self._mu_bias)
        return self

"""The fine-tuning operators of a ParamStore: losses over logits with their gradient, activations
kept in 8 bits and the gradients made from them.

They take and give torch tensors on the store's device.  Results are new tensors unless given;
work is queued on the store's stream, ordered with torch's current stream as the store's other
device work is.  Where both share one stream (ParamStore.set_stream) nothing waits; a store on a
stream of its own, the default, waits for torch's stream before a call's work and for that work
after it.
While the store captures a graph, every result has to be given (an earlier call's, `out=`), and
the graph reads and writes the tensors in place at every launch.

Autograd does not follow the operators: no result requires a gradient, whatever the inputs do (a
loss's gradient goes on by logits.backward(r.grad)).  A given result counts as changed in place:
where torch's backward still needs its old contents (the result of a tanh, an exp or a softmax) it
refuses.  What a captured graph writes at its launches is not seen, as with torch's own graphs.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Any, NamedTuple, Optional

from . import _lib as L

try:
    import torch
except ImportError:  # the optimizers do without it; the operators take its tensors
    torch = None
else:
    _ROW_TYPES = (torch.bfloat16, torch.float32)


class PreferenceLoss(NamedTuple):
    """loss (), margins (pairs,) and logps (rows,) in float32, and the logits' gradient (or
    None)."""
    loss: Any
    margins: Any
    logps: Any
    grad: Optional[Any]


class PolicyLoss(NamedTuple):
    """loss (), kl () and logps (rows,) in float32, and the logits' gradient (or None)."""
    loss: Any
    kl: Any
    logps: Any
    grad: Optional[Any]


class Checkpoint8:
    """An activation kept in 8 bits (ttp_checkpoint8): `values` (rows, cols rounded up to 32) and
    `scales` (rows, that / 32), both uint8; element i of a row is values[i] (int8, or fp8 e4m3)
    times 2^(scales[i // 32] - 127).  `shape` and `dtype` are the activation's own."""

    __slots__ = ("values", "scales", "shape", "dtype", "format", "rows", "cols")

    def __init__(self, values, scales, shape, dtype, fmt):
        _choice(_FORMATS, fmt, "fmt")
        self._set(values, scales, shape, dtype, fmt)
        blocks = -(-self.cols // L.CHECKPOINT_BLOCK)
        for t, width in ((values, blocks * L.CHECKPOINT_BLOCK), (scales, blocks)):
            if t.dtype != torch.uint8 or t.shape != (self.rows, width) or not t.is_contiguous():
                raise ValueError(f"a checkpoint of shape {self.shape} has contiguous uint8 values "
                                 f"and scales of {(self.rows, blocks * L.CHECKPOINT_BLOCK)} and "
                                 f"{(self.rows, blocks)} elements")

    def _set(self, values, scales, shape, dtype, fmt):
        self.values, self.scales = values, scales
        self.shape, self.dtype, self.format = tuple(shape), dtype, fmt
        self.cols = self.shape[-1]
        self.rows = math.prod(self.shape[:-1])
        return self

    def _c(self):
        return L.Checkpoint8(self.values.data_ptr(), self.scales.data_ptr(), self.rows, self.cols,
                             _FORMATS[self.format], 0)


_FORMATS = {"int8": L.CHECKPOINT_INT8, "e4m3": L.CHECKPOINT_E4M3}
_APPROXIMATE = {"none": L.GELU_ERF, "tanh": L.GELU_TANH}


def _choice(table, key, what):
    if key not in table:
        raise ValueError(f"{what} must be one of {', '.join(map(repr, table))}")
    return table[key]


def _matrix(t):
    """The C view of a 2-D tensor whose rows are contiguous."""
    rows, cols = t.shape
    return L.Matrix(t.data_ptr(), rows, cols, t.stride(0) if rows > 1 else cols,
                    L.DTYPE_BF16 if t.element_size() == 2 else L.DTYPE_F32, 0)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _cuts(shape):
    """Where rows in C order begin a new index of a leading dimension, by their counts: the
    elements behind each dimension.  A shape that splits or merges another's dimensions has a
    superset or a subset of its cuts."""
    n, cuts = 1, set()
    for d in reversed(shape):
        cuts.add(n)
        n *= d
    return cuts - {1, n}


def _check_row_order(logits, *per_row):
    """Refuses tensors of one element per row (checked to be as many) whose shape is not the
    others' with some dimensions split or merged (flat: all merged): (T, B) targets of (B, T)
    rows would be paired in another order."""
    rows = logits.shape[:-1]
    finest = _cuts(rows)
    for t in per_row:
        if t is None or t.shape == rows or not t.numel():
            continue
        cuts = _cuts(t.shape)
        if cuts >= finest:
            finest = cuts
        elif not cuts <= finest:
            raise ValueError(f"a tensor of shape {tuple(t.shape)} has its rows in another order "
                             f"than the others (the logits' rows: {tuple(rows)})")


class Operators:
    """Mixed into ParamStore.  (What runs on every call asks as little as it can: a call over one
    row takes 10.5 us of host time: 4.1 the library, 2.9 the streams and sources, 1.7 each new
    tensor.)"""

    def _rows_of(self, t, what):
        """A 2-D view of a float32 or bfloat16 device tensor: all but its last dimension are
        rows (a tensor of one dimension is one row).  Nothing is copied: a layout that is no
        matrix of contiguous rows is refused."""
        if not isinstance(t, torch.Tensor) or t.dtype not in _ROW_TYPES or not t.is_cuda:
            raise ValueError(f"{what} must be a float32 or bfloat16 tensor on the GPU")
        if t.get_device() != self.device:
            raise ValueError(f"{what} is on {t.device}, the store on cuda:{self.device}")
        shape = t.shape
        if not shape or shape[-1] == 0:
            raise ValueError(f"{what} has no columns")
        if len(shape) != 2:
            try:
                t = t.detach().view(-1, shape[-1])
            except RuntimeError:
                raise ValueError(f"{what} must be a matrix of contiguous rows (or a view as "
                                 "one): make it contiguous first") from None
        if not t.is_contiguous():
            (rows, cols), (pitch, one) = t.shape, t.stride()
            if (cols > 1 and one != 1) or (rows > 1 and pitch < cols):
                raise ValueError(f"{what} must have contiguous rows that do not overlap: make it "
                                 "contiguous first")
        return t

    def _vector_of(self, t, n, dtype, what):
        """A contiguous device tensor of n elements of `dtype` (a copy where it is not)."""
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or not t.is_cuda:
            raise ValueError(f"{what} must be a {str(dtype)[6:]} tensor on the GPU")
        if t.get_device() != self.device:
            raise ValueError(f"{what} is on {t.device}, the store on cuda:{self.device}")
        if t.numel() != n:
            raise ValueError(f"{what}: expected {n} elements, got {t.numel()}")
        if t.is_contiguous():
            return t
        if self._in_capture:
            raise ValueError(f"{what} must be contiguous while capturing")
        return t.detach().contiguous()

    def _result(self, given, like, shape, dtype, what):
        """The tensor to write: `given`, checked, or a new one on the device of `like`."""
        if given is None:
            if self._in_capture:
                raise ValueError(f"{what} has to be given while capturing")
            return like.new_empty(shape, dtype=dtype)
        if not isinstance(given, torch.Tensor) or given.dtype != dtype or not given.is_cuda or \
                given.get_device() != self.device or given.shape != torch.Size(shape) or \
                not given.is_contiguous():
            raise ValueError(f"{what} must be a contiguous {str(dtype)[6:]} tensor of shape "
                             f"{tuple(shape)} on cuda:{self.device}")
        return given

    def _queue(self, tensors, written, call, *args):
        """Queue the library's `call` behind torch's work on `tensors`: what it reads, and the
        results that were given (a new one is torch's on its current stream already).  `written`:
        those results, whose versions it raises as torch's own in-place operations do: a backward
        that saved one of them refuses rather than use what is there now."""
        if self._in_capture:
            L.check(call(self._h, *args))
        else:
            kept = self._before_device_sources(tensors)
            L.check(call(self._h, *args))
            self._after_device_sources(kept)
        if written:
            torch.autograd.graph.increment_version(written)

    def _gradient(self, grad, logits, want):
        """(what the caller gets back, its matrix) of a loss's gradient: `grad` True for a new
        tensor like the logits, a tensor to write it to (the logits themselves too), False for
        none."""
        if grad is False or grad is None:
            return None, None
        if grad is True:
            if want is not None:
                grad = want
            else:
                if self._in_capture:
                    raise ValueError("the gradient has to be given while capturing")
                grad = logits.new_empty(logits.shape)
        if not isinstance(grad, torch.Tensor) or grad.dtype != logits.dtype or \
                grad.shape != logits.shape:
            raise ValueError("the gradient must be a tensor of the logits' shape and type")
        return grad, self._rows_of(grad, "the gradient")

    @staticmethod
    def _given_results(grad, given, out):
        """Of a loss's results, those that the caller gave (`given`: the gradient's tensor)."""
        if out is None:
            return [] if given is None or grad is True else [given]
        return [*out[:3]] if given is None else [*out[:3], given]

    def token_logprobs(self, logits, targets, *, out=None):
        """Each row's log-probability of its token under softmax(logits): float32, of targets'
        shape.  logits: (..., V) float32 or bfloat16; targets: int64, of the logits' rows (or flat,
        or with dimensions split or merged), a negative one masks its row (0).  A token past the
        vocabulary gives NaN.  (ttp_token_logprobs)"""
        z = self._rows_of(logits, "the logits")
        y = self._vector_of(targets, z.shape[0], torch.int64, "the targets")
        if targets.dim() > 1:
            _check_row_order(logits, targets)
        result = self._result(out, z, targets.shape, torch.float32, "out")
        given = () if out is None else (out,)
        self._queue((z, y) + given, given, L.lib.ttp_token_logprobs, _matrix(z), y.data_ptr(),
                    result.data_ptr())
        return result

    def preference_loss(self, logits, targets, starts, ref_logps=None, *, beta=0.1,
                        label_smoothing=0.0, grad=True, out=None):
        """The preference loss of P pairs of sequences, and its gradient for the logits.

        Sequence s is rows starts[s] to starts[s + 1] (starts: int64, 2 P + 1 of them on the GPU,
        not decreasing); the first P sequences are the chosen ones, sequence P + p the one
        rejected against p.  With d the sum of logps - ref_logps over a sequence's unmasked rows
        (targets < 0: masked) and margins = beta (d_chosen - d_rejected):

            loss = mean(-(1 - eps) log sigmoid(margins) - eps log sigmoid(-margins))

        grad: True (a new tensor), False (none), or the tensor to write it to, which may be
        `logits` itself.  While loss scaling is on the gradient is the scaled loss's, by the
        store's own scale; the loss is not scaled.  logits.backward(r.grad) continues in torch.
        out: an earlier call's result, whose tensors are written again.  (ttp_preference_loss)"""
        z = self._rows_of(logits, "the logits")
        rows = z.shape[0]
        y = self._vector_of(targets, rows, torch.int64, "the targets")
        if not isinstance(starts, torch.Tensor) or starts.numel() < 3 or starts.numel() % 2 == 0:
            raise ValueError("starts must hold 2 * pairs + 1 row numbers")
        pairs = starts.numel() // 2
        at = self._vector_of(starts, 2 * pairs + 1, torch.int64, "starts")
        ref = None if ref_logps is None else self._vector_of(
            ref_logps, rows, torch.float32, "ref_logps")
        if targets.dim() > 1 or (ref is not None and ref_logps.dim() > 1):
            _check_row_order(logits, targets, ref_logps)
        loss = self._result(out and out.loss, z, (), torch.float32, "the loss")
        margins = self._result(out and out.margins, z, (pairs,), torch.float32, "the margins")
        logps = self._result(out and out.logps, z, targets.shape, torch.float32, "the logps")
        given, g = self._gradient(grad, logits, out and out.grad)
        m, gm = _matrix(z), None if g is None else _matrix(g)
        args = L.PreferenceArgs(
            C.addressof(m), y.data_ptr(), at.data_ptr(), _ptr(ref), pairs, beta, label_smoothing,
            None if gm is None else C.addressof(gm), logps.data_ptr(), margins.data_ptr(),
            loss.data_ptr())
        used = [t for t in (z, y, at, ref) if t is not None]
        written = () if out is None and grad is True else self._given_results(grad, given, out)
        self._queue([*used, *written], written, L.lib.ttp_preference_loss, args)
        return PreferenceLoss(loss, margins, logps, given)

    def policy_loss(self, logits, targets, old_logps, advantages, ref_logps=None, *, clip=0.2,
                    kl_coef=0.0, denominator=None, grad=True, out=None):
        """The clipped policy loss over single tokens, and its gradient for the logits.

        With r = exp(logp - old_logps), A = advantages, g = ref_logps - logp of each unmasked row
        (targets < 0: masked), k = exp(g) - g - 1 (0 without ref_logps):

            loss = sum(-min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef k) / D
            kl   = sum(k) / D

        clip: one number or (low, high).  denominator: D; None: the number of unmasked rows (at
        least 1).  grad and out as in preference_loss.  (ttp_policy_loss)"""
        low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
        if denominator is not None and not denominator > 0:
            raise ValueError("denominator must be positive")
        z = self._rows_of(logits, "the logits")
        rows = z.shape[0]
        y = self._vector_of(targets, rows, torch.int64, "the targets")
        old = self._vector_of(old_logps, rows, torch.float32, "old_logps")
        adv = self._vector_of(advantages, rows, torch.float32, "advantages")
        ref = None if ref_logps is None else self._vector_of(
            ref_logps, rows, torch.float32, "ref_logps")
        if targets.dim() > 1 or old_logps.dim() > 1 or advantages.dim() > 1 or \
                (ref is not None and ref_logps.dim() > 1):
            _check_row_order(logits, targets, old_logps, advantages, ref_logps)
        loss = self._result(out and out.loss, z, (), torch.float32, "the loss")
        kl = self._result(out and out.kl, z, (), torch.float32, "kl")
        logps = self._result(out and out.logps, z, targets.shape, torch.float32, "the logps")
        given, g = self._gradient(grad, logits, out and out.grad)
        m, gm = _matrix(z), None if g is None else _matrix(g)
        args = L.PolicyArgs(
            C.addressof(m), y.data_ptr(), old.data_ptr(), adv.data_ptr(), _ptr(ref), low, high,
            kl_coef, denominator or 0.0, None if gm is None else C.addressof(gm),
            logps.data_ptr(), loss.data_ptr(), kl.data_ptr())
        used = [t for t in (z, y, old, adv, ref) if t is not None]
        written = () if out is None and grad is True else self._given_results(grad, given, out)
        self._queue([*used, *written], written, L.lib.ttp_policy_loss, args)
        return PolicyLoss(loss, kl, logps, given)

    # ---- activations kept in 8 bits ------------------------------------------------------------
    def _kept_of(self, x, fmt, out, shape):
        """The checkpoint to write for the matrix `x`: `out`, checked, or a new one."""
        _choice(_FORMATS, fmt, "fmt")
        rows, cols = x.shape
        blocks = -(-cols // L.CHECKPOINT_BLOCK)
        if out is not None and (not isinstance(out, Checkpoint8) or out.format != fmt or
                                out.shape != tuple(shape) or out.dtype != x.dtype):
            raise ValueError(f"out must be a checkpoint of shape {tuple(shape)} in {fmt}, of a "
                             f"{str(x.dtype)[6:]} activation")
        values = self._result(out and out.values, x, (rows, blocks * L.CHECKPOINT_BLOCK),
                              torch.uint8, "the checkpoint")
        scales = self._result(out and out.scales, x, (rows, blocks), torch.uint8,
                              "the checkpoint")
        return out or Checkpoint8.__new__(Checkpoint8)._set(values, scales, shape, x.dtype, fmt)

    @staticmethod
    def _check_kept(kept):
        if not isinstance(kept, Checkpoint8):
            raise ValueError("a Checkpoint8 is needed (checkpoint8, gelu_checkpoint8)")

    def checkpoint8(self, x, *, fmt="int8", out=None):
        """x (..., cols), float32 or bfloat16, kept in 8 bits: a Checkpoint8.  Blocks of 32 columns
        share a power of two; fmt "int8" keeps 7 bits beside the sign of a block's largest value,
        "e4m3" 4 significant bits of every value.  A block with an infinity or a NaN stands for
        NaN.  out: a Checkpoint8 to write again.  (ttp_checkpoint8_pack)"""
        m = self._rows_of(x, "the activation")
        kept = self._kept_of(m, fmt, out, x.shape)
        given = () if out is None else (out.values, out.scales)
        self._queue((m,) + given, given, L.lib.ttp_checkpoint8_pack, _matrix(m), kept._c())
        return kept

    def restore8(self, kept, *, dtype=None, out=None):
        """The values a Checkpoint8 stands for, in its activation's shape and type (or `dtype`:
        float32 or bfloat16; exact in both).  (ttp_checkpoint8_restore)"""
        self._check_kept(kept)
        dtype = dtype or (kept.dtype if out is None else out.dtype)
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("dtype must be torch.float32 or torch.bfloat16")
        result = self._result(out, kept.values, kept.shape, dtype, "out")
        m = self._rows_of(result, "out")
        given = () if out is None else (out,)
        self._queue((kept.values, kept.scales) + given, given, L.lib.ttp_checkpoint8_restore,
                    kept._c(), _matrix(m))
        return result

    def gelu_checkpoint8(self, x, *, fmt="int8", approximate="none", out=None, kept=None):
        """(gelu(x), x as a Checkpoint8) in one pass.  approximate: "none" (x Phi(x)) or "tanh"
        (GPT-2's), as torch.nn.functional.gelu.  out: where to put gelu(x), x itself too; kept: a
        Checkpoint8 to write again.  (ttp_gelu_checkpoint8)"""
        approx = _choice(_APPROXIMATE, approximate, "approximate")
        m = self._rows_of(x, "the input")
        given = []
        if kept is not None:
            self._check_kept(kept)
            given += [kept.values, kept.scales]
        if out is None:
            out = self._result(None, x, x.shape, x.dtype, "out")
        else:
            given.append(out)
        y = self._like(out, x, "out")
        kept = self._kept_of(m, fmt, kept, x.shape)
        self._queue([m] + given, given, L.lib.ttp_gelu_checkpoint8, _matrix(m), approx, _matrix(y),
                    kept._c())
        return out, kept

    def gelu_backward8(self, kept, dy, *, approximate="none", out=None):
        """dy gelu'(x) from the x that gelu_checkpoint8 kept.  out: where to put it, dy itself
        too.  (ttp_gelu_backward8)"""
        approx = _choice(_APPROXIMATE, approximate, "approximate")
        self._check_kept(kept)
        g = self._rows_of(dy, "dy")
        if tuple(dy.shape) != kept.shape:
            raise ValueError(f"dy has shape {tuple(dy.shape)}, the checkpoint {kept.shape}")
        given = () if out is None else (out,)
        if out is None:
            out = self._result(None, dy, dy.shape, dy.dtype, "out")
        d = self._like(out, dy, "out")
        self._queue((kept.values, kept.scales, g) + given, given, L.lib.ttp_gelu_backward8,
                    kept._c(), approx, _matrix(g), _matrix(d))
        return out

    def accumulate_linear_grad8(self, index, kept, dy, *, bias=None, transposed=False):
        """Add a linear layer's gradients to the store's: tensor `index` receives xhat^T dy
        (cols x outs, the layout of py/nn.py:36; transposed=True: outs x cols, torch.nn.Linear's)
        and tensor `bias` the sum of dy's rows, with xhat what the Checkpoint8 `kept` of the
        layer's input stands for and dy (..., outs), float32 or bfloat16.  As accumulate_grad: the
        first gradient of a tensor is assigned, a further one added in fp32 and rounded once.
        (ttp_accumulate_linear_grad8)"""
        self._check_kept(kept)
        g = self._rows_of(dy, "dy")
        if tuple(dy.shape[:-1]) != kept.shape[:-1]:
            raise ValueError(f"dy has shape {tuple(dy.shape)}, the checkpoint {kept.shape}")
        if bias is None:
            bias = L.NO_TENSOR
        # (here: the library has 32 bits of an index, and -1 would be no bias)
        for i in (index,) if bias == L.NO_TENSOR else (index, bias):
            if not 0 <= i < len(self.tensors):
                raise ValueError(f"tensor index {i} out of range (the store has "
                                 f"{len(self.tensors)} tensors)")
        self._queue((kept.values, kept.scales, g), (), L.lib.ttp_accumulate_linear_grad8, index,
                    bias, kept._c(), _matrix(g), 1 if transposed else 0)

    def _like(self, out, x, what):
        """The matrix of a result that has x's shape and type."""
        if not isinstance(out, torch.Tensor) or out.dtype != x.dtype or out.shape != x.shape:
            raise ValueError(f"{what} must be a tensor of the input's shape and type")
        return self._rows_of(out, what)

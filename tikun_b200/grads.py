"""Gradients between backward and step, on the B200 engine: the norm over many
tensors, clipping by it, and the sum over micro-batches.

The optimizers clip by themselves (``max_norm``): they form the global L2 norm
and fold the scale into their update, so that neither the norm nor a clipped
gradient ever reaches memory.  The functions here are for programs that need
those: a norm for the log (of the whole model, or of each tensor), clipped
gradients for a consumer that does not clip, one norm over the gradients of
several optimizers (``clip_scale``), or f32 sums of bf16 or f16 micro-batch
gradients.

Gradients are a PyTree (as ``UniversalOptimizer`` takes it) of CUDA tensors of
one device, f32, bf16 or f16, in any mix and any number.  A ``Parameter``
stands for its ``.grad``, so ``model.parameters()`` may be given; a parameter
without a gradient, and ``None``, are left out.  A gradient may be any dense
view without gaps (a transposed weight's gradient is one).  A program whose
gradient buffers stand (``arena=True``, or ``zero_grad(set_to_none=False)``)
builds a ``GradTable`` of them once and gives that in their place: checking and
laying out 150 tensors takes 0.1 ms of host time, a call on a table 8 us.

Every call runs on torch's current stream of the gradients' device and does not
wait for it (``error_if_nonfinite=True`` does).  A call may be captured into a
CUDA graph.  No call is seen by autograd, and what is written in place keeps its
version counter, as under the optimizers' steps: a tensor that a later backward
pass still needs is not to be clipped.
"""
from __future__ import annotations

import array
import ctypes
import math

import torch

from . import _native
from .universal import flatten_leaves

_NORMS = {2.0: _native.TK_NORM_L2, 1.0: _native.TK_NORM_L1, math.inf: _native.TK_NORM_MAX}
_DTYPES = {torch.float32: _native.TK_F32, torch.bfloat16: _native.TK_BF16,
           torch.float16: _native.TK_F16}


def _norm_code(norm_type) -> int:
    code = _NORMS.get(norm_type)
    if code is None:
        raise ValueError(f"norm_type is 2, 1 or inf, got {norm_type!r}")
    return code


def _positive(max_norm) -> float:
    """max_norm as the f32 number that the kernels take."""
    value = ctypes.c_float(max_norm).value
    if not value > 0:  # also where it is so small that it rounds to 0: no limit, there
        raise ValueError(f"max_norm is positive as a float32, got {max_norm!r}")
    return value


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one stretch of memory, in whatever order."""
    if t.is_contiguous():
        return True
    span = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != span:
            return False
        span *= size
    return True


def _refuse(t, what: str) -> None:
    """Raises for what is not a dense CUDA tensor of one of the types."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a torch tensor, got {type(t).__name__}")
    if t.layout != torch.strided or not t.is_cuda:
        raise ValueError(f"{what}: expected a dense CUDA tensor, got {t.layout} on {t.device}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{what} is float32, bfloat16 or float16, got {t.dtype}")
    if t.is_neg():
        raise ValueError(f"{what} is a lazily negated view: its memory holds the negative")
    if t.numel() and not _dense(t):
        raise ValueError(f"{what}: its elements do not fill one stretch of memory (shape "
                         f"{tuple(t.shape)}, strides {t.stride()})")


def _columns(ts: list, what: str) -> tuple[list, list, list, set, bool]:
    """Addresses, element counts and type codes of checked tensors, their
    device indices, and whether all are contiguous.  One attribute of all
    tensors at a time: a third of the time of one tensor at a time."""
    at = None
    try:
        at, codes = [t.data_ptr() for t in ts], [_DTYPES[t.dtype] for t in ts]
        devices = {t.get_device() for t in ts}  # -1 on the host
        plain = min(devices, default=0) >= 0 and all([t.is_contiguous() for t in ts]) and \
            not any([t.is_neg() for t in ts])
    except (AttributeError, KeyError, RuntimeError):  # no tensor, its type, no memory of its own
        plain = False
    if not plain:
        for i, t in enumerate(ts):
            _refuse(t, f"{what} {i}")
        if at is None:
            raise TypeError(f"the {what} tensors have no memory of their own")
    return at, [t.numel() for t in ts], codes, devices, plain


# what current_stream().cuda_stream gives, at a fortieth of its 3 us
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(index: int) -> int:
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def _on_device(t: "GradTable", call):
    """call(stream) with the table's device current."""
    index = t.device.index
    if torch.cuda.current_device() == index:
        return call(_stream(index))
    with torch.cuda.device(index):
        return call(_stream(index))


def _leaves(tree) -> list:
    """flatten_leaves, without its walk for a plain list of tensors."""
    if not isinstance(tree, (list, tuple, dict, torch.Tensor)) and hasattr(tree, "__iter__"):
        tree = list(tree)  # model.parameters()
    if isinstance(tree, (list, tuple)) and all([isinstance(t, torch.Tensor) for t in tree]):
        return list(tree)
    return flatten_leaves(tree)


class GradTable:
    """The gradients of one or many calls, checked and laid out once.

    ``out`` (a PyTree of as many CUDA tensors, element i of the size and the
    strides of gradient i) is where ``clip_grad_norm_`` and
    ``accumulate_grads_`` write; without it they work in place.  The table reads
    and writes the memory that the tensors have now, and keeps it.  For
    parameters it is their ``.grad`` of now: a call raises ``RuntimeError`` once
    one of them has another (as after ``zero_grad(set_to_none=True)``), or has
    its first."""

    def __init__(self, grads, out=None):
        self._build(grads, out)
        self._like = torch.empty((), dtype=torch.float32, device=self.device)
        # a tensor may be given other memory (.data, set_): this one stays
        self._memory = [t.untyped_storage() for t in self.grads + (self.out or [])]

    def _build(self, grads, out):
        self._handle = None
        self._like = None
        self._params = []
        self.grads = _leaves(grads)
        # a plain tensor is no Parameter (whose isinstance costs ten times as much)
        if not all([type(t) is torch.Tensor for t in self.grads]):
            leaves, self.grads = self.grads, []
            for leaf in leaves:
                if isinstance(leaf, torch.nn.Parameter):
                    g = leaf.grad
                    self._params.append((leaf, g))  # without one too: it may get its first
                    if g is not None:
                        self.grads.append(g)
                elif leaf is not None:
                    self.grads.append(leaf)
        n = len(self.grads)
        at, sizes, codes, devices, plain = _columns(self.grads, "gradient")
        out_at = [0] * n
        self.out = None
        if out is not None:
            self.out = _leaves(out)
            if any([type(t) is not torch.Tensor and isinstance(t, torch.nn.Parameter)
                    for t in self.out]):
                raise TypeError("out holds tensors to write, not parameters")
            if len(self.out) != n:
                raise ValueError(f"{len(self.out)} out tensors for {n} gradients")
            out_at, out_sizes, out_codes, out_devices, out_plain = _columns(self.out, "out")
            devices |= out_devices
            codes = [g | o << 32 for g, o in zip(codes, out_codes)]  # the C struct's two int32
            if out_sizes != sizes or not (plain and out_plain):
                for i, (g, o) in enumerate(zip(self.grads, self.out)):
                    if g.numel() != o.numel() or not (g.is_contiguous() and o.is_contiguous() or
                                                      o.stride() == g.stride()):
                        raise ValueError(f"out {i} has shape {tuple(o.shape)} and strides "
                                         f"{o.stride()}, its gradient {tuple(g.shape)} and "
                                         f"{g.stride()}")
        if len(devices) > 1:
            raise ValueError(f"the tensors of one call are on one device, got {sorted(devices)}")
        self.device = torch.device("cuda", devices.pop() if devices else torch.cuda.current_device())
        words = array.array("Q", [w for row in zip(at, out_at, sizes, codes) for w in row])
        entries = ctypes.cast(words.buffer_info()[0], ctypes.POINTER(_native.TkGrad))
        handle = ctypes.c_void_p()
        _on_device(self, lambda _: _native.check(
            _native.lib().tk_grad_table_create(entries, n, ctypes.byref(handle))))
        self._destroy = _native.lib().tk_grad_table_destroy
        self._handle = handle
        sizes = _native._U64(), _native._U64()
        _native.check(_native.lib().tk_grad_workspace(handle, *map(ctypes.byref, sizes)))
        self._scratch, self._scratch_each = (s.value for s in sizes)

    def __reduce_ex__(self, protocol):
        raise TypeError("a GradTable is of this process's memory: build another")

    def __len__(self) -> int:
        return len(self.grads)

    def __del__(self):
        if getattr(self, "_handle", None) is not None:
            self._destroy(self._handle)
            self._handle = None

    def _result(self) -> torch.Tensor:
        """A 0-dim f32 tensor for a call's result."""
        if self._like is None:
            return torch.empty((), dtype=torch.float32, device=self.device)
        return torch.empty_like(self._like)  # a microsecond less

    def _workspace(self, size: int):
        """(tensor, address) of a call's scratch from torch's allocator, which
        gives it to no other stream's work and to each captured graph its own."""
        if not size:
            return None, None
        ws = torch.empty(size // 8, dtype=torch.float64, device=self.device)
        return ws, ws.data_ptr()

    def _standing(self) -> "GradTable":
        for p, g in self._params:
            if p.grad is not g:
                raise RuntimeError("a parameter of this GradTable has another gradient tensor "
                                   "now: build the table anew")
        return self


def _table(grads, out=None) -> GradTable:
    if isinstance(grads, GradTable):
        if out is not None:
            raise ValueError("a GradTable has its out tensors already")
        return grads._standing()
    table = GradTable.__new__(GradTable)  # for this call: its tensors stand that long
    table._build(grads, out)
    return table


def _finite(norm: torch.Tensor, norm_type) -> None:
    v = norm.item()
    if not math.isfinite(v):
        raise RuntimeError(f"the gradients' norm of order {norm_type} is {v}")


def grad_norm(grads, norm_type: float = 2.0, per_tensor: bool = False,
              error_if_nonfinite: bool = False):
    """The norm of all gradients' elements as one vector, a 0-dim f32 tensor:
    sqrt(sum x^2) (2), sum |x| (1) or max |x| (``inf``); 0 without elements,
    NaN with a NaN among them.  Sums are formed in f64 (of bf16 and f16 values
    first by eights in f32) in a fixed order and rounded once.

    ``per_tensor=True``: (norm, norms), ``norms`` the f32 norms of the
    gradients, one each."""
    code = _norm_code(norm_type)
    t = _table(grads)
    norm = t._result()
    each = torch.empty(len(t), dtype=torch.float32, device=t.device) if per_tensor else None
    each_ptr = each.data_ptr() if per_tensor and len(t) else None
    _ws, ws = t._workspace(t._scratch_each if per_tensor else t._scratch)
    _on_device(t, lambda stream: _native.check(_native.lib().tk_grad_norm(
        t._handle, code, 0.0, norm.data_ptr(), each_ptr, None, ws, stream)))
    if error_if_nonfinite:
        _finite(norm, norm_type)
    return (norm, each) if per_tensor else norm


def clip_scale(grads, max_norm: float, norm_type: float = 2.0):
    """(norm, scale): the norm of ``grad_norm`` and the scale that
    ``clip_grad_norm_`` would multiply by, both 0-dim f32 tensors on the device
    that no later call or step writes.
    The optimizers' ``step(clip_scale=scale)`` folds it into their updates, so
    that several of them clip by one norm and no gradient is written."""
    code = _norm_code(norm_type)
    max_norm = _positive(max_norm)
    t = _table(grads)
    norm = t._result()
    scale = t._result()
    _ws, ws = t._workspace(t._scratch)
    _on_device(t, lambda stream: _native.check(_native.lib().tk_grad_norm(
        t._handle, code, max_norm, norm.data_ptr(), None, scale.data_ptr(), ws, stream)))
    return norm, scale


def clip_grad_norm_(grads, max_norm: float, norm_type: float = 2.0, out=None,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the gradients by ``max_norm / (norm + 1e-6)`` if their norm (see
    ``grad_norm``) exceeds ``max_norm``, in place or into ``out``, and returns
    the norm from before.  Each product is formed in f32 and rounded once to its
    target's type.  The scale is formed as an optimizer with this ``max_norm``
    forms the one that it folds into its update, so clipping f32 gradients here
    and stepping without ``max_norm`` gives the same bits.  Of bf16 gradients the
    two norms, and so the scales, may differ in their last bits: the optimizer
    adds each square in f64, ``grad_norm`` eight of them in f32 first.

    A norm of NaN leaves the gradients as they are (in place) or copies them
    (``out``), as the optimizers do; an infinite one makes the scale 0.
    ``error_if_nonfinite=True`` raises ``RuntimeError`` for both before
    anything is written, and waits for the norm to know."""
    code = _norm_code(norm_type)
    max_norm = _positive(max_norm)
    t = _table(grads, out)
    if error_if_nonfinite:
        grad_norm(t, norm_type, error_if_nonfinite=True)
    norm = t._result()
    _ws, ws = t._workspace(t._scratch)
    _on_device(t, lambda stream: _native.check(_native.lib().tk_clip_grad_norm(
        t._handle, code, max_norm, norm.data_ptr(), None, ws, stream)))
    return norm


def accumulate_grads_(grads, acc=None, alpha: float = 1.0, overwrite: bool = False,
                      norm_type: float | None = None) -> torch.Tensor | None:
    """``acc += alpha * grad`` for every gradient, or ``acc = alpha * grad``
    with ``overwrite`` (the first micro-batch: ``acc`` need not be cleared).
    ``acc`` (the ``out`` of a ``GradTable``) is f32 whatever the gradients are:
    sums of micro-batches in bf16 lose the small ones.  ``alpha`` is a host
    number, such as one over the micro-batches or over a loss scale.

    ``norm_type``: returns the norm of the new ``acc`` (see ``grad_norm``),
    formed as it is written; otherwise None."""
    code = _native.TK_NORM_NONE if norm_type is None else _norm_code(norm_type)
    if not isinstance(grads, GradTable) and acc is None:
        raise ValueError("accumulate_grads_ needs acc")
    t = _table(grads, acc)
    norm = t._result() if norm_type is not None else None
    norm_ptr = norm.data_ptr() if norm is not None else None
    _ws, ws = t._workspace(t._scratch if norm is not None else 0)
    _on_device(t, lambda stream: _native.check(_native.lib().tk_accumulate_grads(
        t._handle, float(alpha), 1 if overwrite else 0, code, norm_ptr, ws, stream)))
    return norm


__all__ = ["GradTable", "grad_norm", "clip_scale", "clip_grad_norm_", "accumulate_grads_"]

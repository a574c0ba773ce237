"""What lies between a backward pass and the quantisers: the global gradient norm, clipping by it and the AdamW update.

The trainer's loop around a weight sync is backward -> norm -> clip -> update -> quantise -> ship, and everything here works
like the quantisers do: over whole lists of tensors, a few launches per list, nothing read back to the host.  The update takes
the clip as a factor (no pass of its own) and writes the bf16 / fp16 weight that ``Fp8QuantPlan``, ``Int4PackPlan`` or
``BucketConverter`` then read.

``get_total_norm``, ``clip_grad_norm_`` and ``clip_grads_with_norm_`` have the names and arguments of ``torch.nn.utils`` and take
whatever gradients a call presents; ``GradNormPlan``, ``GradClipPlan`` and ``AdamWPlan`` take a fixed list (gradient buffers that
stay where they are) and can be captured into a HIP graph.  Norms are fp32, whatever the gradients' type: sums of squares are
formed in 64 bits, so they do not overflow (a norm beyond fp32's range is infinite), and in an order that depends on the list, on where
its tensors start and on the kind of call or plan, but not on the run.

Norm of a model that is sharded over ranks, for ``total_norm=`` of the clip or the update: of 2-norms
``total = plan.run().double().square(); all_reduce(total); total_norm = total.sqrt().float()`` (fp32 squares would be infinite for a
norm above 1.8e19 and zero below 2.6e-23); of infinity norms ``total_norm = plan.run(); all_reduce(total_norm.view(torch.int32),
op=MAX)`` (the bits of magnitudes have their order, and a NaN on one rank is above infinity; of floats a maximum may drop it).
"""

from __future__ import annotations

import math
import numbers
import operator
from array import array
from bisect import bisect_left
from contextlib import nullcontext
from typing import Iterable, Sequence

import numpy as np
import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
_NORMS = {2.0: _lib.NORM_2, math.inf: _lib.NORM_INF}

# Lists of hundreds of tensors are looked at by passes that stay in C, map() over these (40 ns a tensor); only where something is
# out of the ordinary are they looked at one by one.
_data_ptr, _numel, _is_contiguous, _get_device, _is_neg = (getattr(torch.Tensor, n) for n in ("data_ptr", "numel", "is_contiguous", "get_device", "is_neg"))
_dtype, _layout, _shape, _nbytes, _grad = (getattr(torch.Tensor, n).__get__ for n in ("dtype", "layout", "shape", "nbytes", "grad"))
_PLAIN_TYPES = {torch.Tensor, torch.nn.Parameter}
_F32_MAX = float(np.finfo(np.float32).max)      # what the kernels take as fp32 has to be finite there


def _norm_selector(norm_type, what: str) -> int:
    norm = _NORMS.get(float(norm_type))
    if norm is None:
        raise ValueError(f"{what}: norm_type {norm_type} is not supported (2 and inf are)")
    return norm


def _check_max_norm(max_norm, what: str) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: max_norm must not be negative or NaN, got {max_norm}")
    return max_norm


def _check_tensor(t, what: str, dtypes=_DTYPES) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    if t.layout != torch.strided or hasattr(t, "to_local"):
        raise TypeError(f"{what}: only plain strided tensors are supported (of a sharded one, pass the local part)")
    if t.dtype not in dtypes or t.is_neg():
        raise TypeError(f"{what}: dtype {t.dtype}{' with a pending negation' * t.is_neg()} is not supported "
                        f"({', '.join(str(d) for d in dtypes)})")


def _check_tensors(tensors, what: str, dtypes=_DTYPES) -> None:
    if set(map(type, tensors)) <= _PLAIN_TYPES and set(map(_layout, tensors)) <= {torch.strided} and \
            set(map(_dtype, tensors)) <= set(dtypes) and not any(map(_is_neg, tensors)):
        return
    for t in tensors:
        _check_tensor(t, what, dtypes)


def _strides(t):
    """(stride, size) of the dimensions that have a stride, smallest first."""
    return sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1)


def _is_dense(t) -> bool:
    """Whether the elements fill one run of memory, in any order of dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for st, n in _strides(t):
        if st != expected:
            return False
        expected *= n
    return True


def _check_no_self_overlap(t, what: str) -> None:
    reach = 0
    for st, n in _strides(t):
        if st <= reach:
            raise ValueError(f"{what}: elements of a gradient share memory (strides {tuple(t.stride())}); it cannot be written")
        reach += st * (n - 1)


class _Elements:
    """What numpy needs to know of a tensor's elements to tell whether they share memory with others'; it follows no address."""

    def __init__(self, t):
        size = t.element_size()
        self.__array_interface__ = {"version": 3, "data": (t.data_ptr(), False), "shape": tuple(t.shape), "typestr": f"|V{size}",
                                    "strides": tuple(st * size for st in t.stride())}


def _run_and_pitch(t):
    """-> (bytes of the runs of memory that the elements form, greatest common divisor of the distances between runs; 0 for one)"""
    run, pitch, size = 1, 0, t.element_size()
    for st, n in _strides(t):
        if st == run and not pitch:
            run *= n
        else:
            pitch = math.gcd(pitch, st)
    return run * size, pitch * size


def _share_memory(tensors) -> bool:
    """Whether two of the tensors share an element, exactly: slices that interleave do not.  Tensors whose byte ranges meet are
    compared in pairs, first by where their runs lie modulo the common pitch (0.4 us: slices of one buffer), then by numpy; the
    few pairs of strides that would take that milliseconds count as sharing."""
    spans = sorted((t.data_ptr(), t.data_ptr() + (1 + sum(st * (n - 1) for st, n in zip(t.stride(), t.shape))) * t.element_size(),
                    *_run_and_pitch(t), i) for i, t in enumerate(tensors) if t.numel())
    arrays, meeting = {}, []
    for span in spans:
        start, _, run, pitch, i = span
        meeting = [other for other in meeting if other[1] > start]
        for from_, _, other_run, other_pitch, j in meeting:
            common = math.gcd(pitch, other_pitch)
            if not common:
                return True
            at = (start - from_) % common
            if at >= other_run and at + run <= common:
                continue
            for k in (i, j):
                if k not in arrays:
                    arrays[k] = np.asarray(_Elements(tensors[k]))
            try:
                if np.shares_memory(arrays[i], arrays[j], max_work=100_000):
                    return True
            except np.exceptions.TooHardError:
                return True
        meeting.append(span)
    return False


def _same_layout(a, b) -> bool:
    return a.shape == b.shape and (a.stride() == b.stride() or a.numel() == 0 or
                                   all(n == 1 or x == y for x, y, n in zip(a.stride(), b.stride(), a.shape)))


def _same_layouts(tensors, others) -> bool:
    if all(map(_is_contiguous, tensors)) and all(map(_is_contiguous, others)):
        return all(map(torch.Size.__eq__, map(_shape, tensors), map(_shape, others)))
    return all(map(_same_layout, tensors, others))


def _one_device(tensors, what: str) -> torch.device:
    indices = set(map(_get_device, tensors))
    if len(indices) == 1 and min(indices) >= 0:
        return tensors[0].device
    for t in tensors:
        _lib.require_gpu(t, what)
    raise ValueError(f"{what}: all tensors must be on one device (got {sorted(set(str(t.device) for t in tensors))})")


def _column(f, tensors) -> np.ndarray:
    return np.fromiter(map(f, tensors), dtype=np.int64, count=len(tensors))


def _refuse_overlaps(written, read, what: str) -> None:
    """Ranges that are written share no byte with each other or with one that is read."""
    tensors = [*written, *read]
    start, size = _column(_data_ptr, tensors), _column(_nbytes, tensors)
    w = np.arange(len(tensors)) < len(written)
    order = np.argsort(start[size > 0], kind="stable")
    start, end, w = (x[size > 0][order] for x in (start, start + size, w))
    any_end = np.maximum.accumulate(end)[:-1]
    written_end = np.maximum.accumulate(np.where(w, end, 0))[:-1]
    if ((start[1:] < written_end) | (w[1:] & (start[1:] < any_end))).any():
        raise ValueError(f"{what}: tensors that are written share memory with others of the call (the same tensor twice?)")


def _lies_in(address: int, starts, ends) -> bool:
    """Whether an fp32 value at the address shares a byte with one of the ranges (disjoint, ascending)."""
    i = bisect_left(starts, address + 4) - 1
    return i >= 0 and address < ends[i]


def _scalar_on_device(value, device, what: str, number: str = "") -> int:
    """The address of a scalar argument; a sharded or wrapped tensor has none (0, which the kernels take for "not given")."""
    if not isinstance(value, torch.Tensor) or value.dtype != torch.float32 or value.numel() != 1 or value.device != device or \
            value.layout != torch.strided or value.is_neg() or not (address := value.data_ptr()):
        raise ValueError(f"{what} must be {number}one float32 value on {device} (of a sharded tensor, the full one)")
    return address


def _scale_args(scale, device, what: str):
    """-> (factor, address of a factor on the device or None)"""
    if isinstance(scale, torch.Tensor):
        return 1.0, _scalar_on_device(scale, device, what, "a number or ")
    scale = float(scale)
    if not 0.0 <= scale <= _F32_MAX:
        raise ValueError(f"{what} must be a finite number (in fp32) that is not negative, got {scale}")
    return scale, None


def _launch(device: torch.device, entry: str, what: str, *args) -> None:
    fn = getattr(_lib.load(), entry)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, _lib.raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _lib.raw_stream(device.index))
    if rc:
        _lib.check(rc, what)


def _bump(tensors) -> None:
    """Tell autograd that a kernel wrote into these tensors, as torch's in-place operations do."""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:                    # inference tensors have no version
        torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def _workspace(n_items: int, device) -> torch.Tensor:
    return torch.empty(_lib.load().wq_grad_workspace_bytes(n_items) // 8, dtype=torch.int64, device=device)


def _grad_rows(grads, outs) -> np.ndarray:
    kind = _column(_DTYPES.get, list(map(_dtype, grads))) | _column(_DTYPES.get, list(map(_dtype, outs))) << 32
    return np.stack([_column(_data_ptr, grads), _column(_data_ptr, outs), _column(_numel, grads), kind], axis=1)


def _cuts(rows: np.ndarray):
    """-> (elements of a piece, elements by which the first is shorter) per row: pieces are cut at 128-byte lines of the fp32
    weight of an update, of the wider stream of a clip."""
    if rows.shape[1] == 8:
        return _lib.ADAMW_ITEM, rows[:, 4] % 128 // 4
    g, o = (np.where(d == _lib.DTYPE_F32, 4, 2) for d in (rows[:, 3] & 0xFFFFFFFF, rows[:, 3] >> 32))
    return _lib.GRAD_ITEM_BYTES // g, np.where((rows[:, 1] != 0) & (o >= g), rows[:, 1] % 128 // o, rows[:, 0] % 128 // g)


def _refuse_no_memory(addresses: np.ndarray, what: str) -> None:
    if (addresses == 0).any():
        raise ValueError(f"{what}: a tensor has no memory (a wrapper, or storage that was released)")


def _item_table(rows: np.ndarray, device, what: str):
    """Per-tensor rows (int64 [n, 4 or 8], the fields of wq_grad_desc / wq_adamw_desc) -> (item table on the device, starts
    of the tensors in it, number of items)."""
    n = rows[:, 2]
    g, out = (np.where(d == _lib.DTYPE_F32, 4, 2) for d in (rows[:, 3] & 0xFFFFFFFF, rows[:, 3] >> 32))
    if (rows[:, 0] % g).any() or (rows[:, 1] % out).any() or (rows[:, 4:7] % 4).any():
        raise ValueError(f"{what}: a tensor does not start at a multiple of its element size")
    _refuse_no_memory(rows[n > 0][:, [0, 4, 5, 6] if rows.shape[1] == 8 else [0, 1]], what)
    starts = np.zeros(len(rows) + 1, dtype=np.int64)
    per, phase = _cuts(rows)
    np.cumsum(np.where(n > 0, -(-(n + phase) // per), 0), out=starts[1:])
    table = torch.from_numpy(np.concatenate([rows.reshape(-1), starts])).to(device)
    n_items, words = int(starts[-1]), rows.shape[1]
    items = torch.empty((max(n_items, 1), words), dtype=torch.int64, device=device)
    start_t = table[rows.size:]
    _launch(device, "wq_grad_make_items", what, table.data_ptr(), start_t.data_ptr(), len(rows), n_items, words, items.data_ptr())
    return items, start_t, n_items


class _Plan:
    """Tables and workspace of a fixed list.  One plan's runs - captured ones too - must be ordered on one stream (or by
    events): they share the workspace and the result.  The stream need not be the one the plan was built on.  The plan reads
    and writes the tensors it was given, wherever their contents come from; one that moves needs a new plan.  A graph that
    captured a run needs the plan for as long as it is replayed."""

    # Tensors that a run writes while others of its workgroups may still read the run's device scalars (an AdamW run has read its
    # scalars before it writes any).
    _written_beside_reads: Sequence[torch.Tensor] = ()
    _spans = None

    def _build(self, rows, device, what: str) -> None:
        self.device, self._what = device, what
        with torch.cuda.device(device):
            self._items, self._starts, self._n_items = _item_table(rows, device, what)
            self._workspace = _workspace(self._n_items, device)
            self.total_norm = torch.zeros((), dtype=torch.float32, device=device)
            self._stream = torch.cuda.current_stream(device)
            self._owned = [self._items, self._starts, self._workspace, self.total_norm]

    def _built(self) -> None:
        self._stream.synchronize()      # a run on another stream finds the tables ready

    def _run(self, entry: str, *args) -> None:
        if _lib.raw_stream(self.device.index) != self._stream.cuda_stream and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(self.device)
            for t in self._owned:       # the allocator must not hand them out while this stream may still use them
                t.record_stream(stream)
        _launch(self.device, entry, self._what, *args)

    def _factor(self, value, what: str):
        factor, address = _scale_args(value, self.device, f"{self._what}: {what}")
        if address is not None and address == self.total_norm.data_ptr():
            raise ValueError(f"{self._what}: {what} must not be the plan's own total_norm, which the run overwrites")
        self._refuse_written(address, what)
        return factor, address

    def _given(self, total_norm):
        address = None if total_norm is None else _scalar_on_device(total_norm, self.device, f"{self._what}: total_norm")
        self._refuse_written(address, "total_norm")
        return address

    def _refuse_written(self, address, what: str) -> None:
        if address is None or not self._written_beside_reads:
            return
        if self._spans is None:             # they share no memory
            spans = sorted((t.data_ptr(), t.data_ptr() + t.nbytes) for t in self._written_beside_reads if t.numel())
            self._spans = [s for s, _ in spans], [e for _, e in spans]
        if _lies_in(address, *self._spans):
            raise ValueError(f"{self._what}: {what} must not lie in a tensor that the run writes")


def _check_grads(grads, what: str):
    grads = list(grads)
    if not grads:
        raise ValueError(f"{what}: empty gradient list")
    _check_tensors(grads, what)
    for g in grads if not all(map(_is_contiguous, grads)) else ():
        if not _is_dense(g):
            raise ValueError(f"{what}: tensors of a plan must fill one run of memory (a copy would be read instead of the live "
                             f"gradient); got shape {tuple(g.shape)}, strides {tuple(g.stride())}")
    return grads


class GradNormPlan(_Plan):
    """The global norm (2 or inf) of a fixed list of bf16 / fp16 / fp32 gradients, and with ``per_tensor`` the norm of each.

    ``run(grad_scale=1.0)`` returns ``total_norm``, a 0-d fp32 tensor that the next run overwrites, or ``(total_norm, norms)``
    with ``norms`` fp32 ``[len(grads)]``.  grad_scale (a number or one fp32 value on the device: an inverse loss scale, one over
    the number of tokens; not a value that the run writes) multiplies the gradients.  A gradient may be in the list twice and then
    counts twice."""

    def __init__(self, grads: Sequence[torch.Tensor], norm_type: float = 2.0, per_tensor: bool = False):
        self._norm = _norm_selector(norm_type, "GradNormPlan")
        self.grads = _check_grads(grads, "GradNormPlan")
        self._build(_grad_rows(self.grads, self.grads), _one_device(self.grads, "GradNormPlan"), "GradNormPlan")
        self.norms = torch.zeros(len(self.grads), dtype=torch.float32, device=self.device) if per_tensor else None
        if per_tensor:
            self._owned.append(self.norms)
            self._written_beside_reads = [self.norms]
        self._built()

    def run(self, grad_scale=1.0):
        scale, scale_dev = self._factor(grad_scale, "grad_scale")
        each = self.norms
        self._run("wq_grad_norm_items", self._items.data_ptr(), self._n_items, 4, self._starts.data_ptr(), len(self.grads),
                  self._norm, scale, scale_dev, self._workspace.data_ptr(), self.total_norm.data_ptr(),
                  None if each is None else each.data_ptr())
        return self.total_norm if each is None else (self.total_norm, each)


class GradClipPlan(_Plan):
    """Clip a fixed list of gradients by their global norm: ``g * grad_scale * min(1, max_norm / (norm + 1e-6))``, in place or,
    with ``out``, into other tensors of the same shapes and layouts (bf16 gradients into fp32 main gradients, say), rounded
    once.  In place, gradients that need no change are not rewritten.

    ``run(max_norm, grad_scale=1.0, total_norm=None)`` returns the norm before the clip: a 0-d fp32 tensor that the next run
    overwrites.  ``total_norm`` (one fp32 value on the device, of the gradients times grad_scale) is taken for the norm, and
    returned, if it is given.  Device scalars must not lie in the tensors that are written."""

    def __init__(self, grads: Sequence[torch.Tensor], norm_type: float = 2.0, out: Sequence[torch.Tensor] | None = None):
        self._norm = _norm_selector(norm_type, "GradClipPlan")
        self.grads = _check_grads(grads, "GradClipPlan")
        self.out = self.grads if out is None else list(out)
        if len(self.out) != len(self.grads):
            raise ValueError("GradClipPlan: need one output per gradient")
        _check_tensors(self.out, "GradClipPlan")
        if not _same_layouts(self.grads, self.out):
            g, o = next((g, o) for g, o in zip(self.grads, self.out) if not _same_layout(g, o))
            raise ValueError(f"GradClipPlan: output of shape {tuple(o.shape)}, strides {tuple(o.stride())} for a gradient of "
                             f"shape {tuple(g.shape)}, strides {tuple(g.stride())}")
        apart = [g for g, o in zip(self.grads, self.out) if g is not o and (g.data_ptr() != o.data_ptr() or g.dtype != o.dtype)]
        _refuse_overlaps(self.out, apart, "GradClipPlan")
        self._build(_grad_rows(self.grads, self.out), _one_device(self.grads + self.out, "GradClipPlan"), "GradClipPlan")
        self._written_beside_reads = self.out
        self._built()

    def run(self, max_norm: float, grad_scale=1.0, total_norm: torch.Tensor | None = None) -> torch.Tensor:
        max_norm = _check_max_norm(max_norm, "GradClipPlan")
        scale, scale_dev = self._factor(grad_scale, "grad_scale")
        self._run("wq_grad_clip_items", self._items.data_ptr(), self._n_items, self._norm, max_norm, scale, scale_dev,
                  self._given(total_norm), self._workspace.data_ptr(), self.total_norm.data_ptr())
        _bump(self.out)
        return self.total_norm if total_norm is None else total_norm


def _address(t):
    return t.data_ptr() if t.layout == torch.strided else None


def _per_tensor(value, n: int, what: str):
    values = [float(value)] * n if isinstance(value, numbers.Real) else [float(v) for v in value]
    if len(values) != n:
        raise ValueError(f"AdamWPlan: need one {what} per parameter")
    for v in values:
        if not 0.0 <= v <= _F32_MAX:
            raise ValueError(f"AdamWPlan: {what} must be finite (in fp32) and not negative, got {v}")
    return values


class AdamWPlan(_Plan):
    """One AdamW step (decoupled weight decay) over a fixed list of fp32 parameters per ``run()``: with t = ``step`` + 1 and
    g = gradient * grad_scale * min(1, max_norm / (norm + 1e-6)),

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        p = p - lr w p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps);  weight = round(p)

    ``weights``: bf16 / fp16 copies of the parameters (None, or None for single ones), written by the same pass.
    ``exp_avgs`` / ``exp_avg_sqs``: fp32 moments (fresh zeros by default).  All tensors of one parameter have its shape and
    layout.  ``weight_decay`` (w) and ``lr_scale`` (multiplies lr): one number or one per parameter.  ``step`` counts the steps
    done, in a 0-d int64 tensor on the device (``plan.step``; start at another one with ``step=``), so a captured run counts its
    replays.  With ``skip_nonfinite`` a step whose gradient norm is infinite or NaN changes nothing and is not counted.

    ``run(lr, max_norm=None, grad_scale=1.0, total_norm=None)``: lr is a number or one fp32 value on the device (a number is
    fixed in a captured run).  Parameters with other betas are a plan of their own; the norm over several plans comes from one
    ``GradNormPlan`` as their ``total_norm``.  The gradients are read where they were when the plan was built; if they were the
    parameters' ``.grad`` and a parameter has another one now (``zero_grad()`` drops them unless ``set_to_none=False``), the run is
    refused.  Returns the gradient norm before the clip where it is needed (max_norm or skip_nonfinite; a 0-d
    fp32 tensor that the next run overwrites, or the ``total_norm`` given), else None."""

    def __init__(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], weights: Sequence | None = None,
                 exp_avgs: Sequence[torch.Tensor] | None = None, exp_avg_sqs: Sequence[torch.Tensor] | None = None,
                 betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01, lr_scale=1.0, norm_type: float = 2.0,
                 skip_nonfinite: bool = False, step: int = 0):
        self._norm = _norm_selector(norm_type, "AdamWPlan")
        self.betas, self.eps = (float(betas[0]), float(betas[1])), float(eps)
        if not all(0.0 <= b < 1.0 for b in self.betas) or not 0.0 <= self.eps < math.inf:
            raise ValueError(f"AdamWPlan: betas must be in [0, 1) and eps finite and not negative, got {betas}, {eps}")
        if 0.0 < self.eps <= 2.0 ** -150:       # 0 in fp32: elements without a gradient so far would become NaN
            raise ValueError(f"AdamWPlan: eps must be 0 or above 2^-150, half of fp32's smallest number, got {eps}")
        if int(step) < 0:
            raise ValueError(f"AdamWPlan: step must not be negative, got {step}")
        self.grads, self.params = _check_grads(grads, "AdamWPlan"), list(params)
        n = len(self.params)
        self.weights, *moments = ([None] * n if x is None else list(x) for x in (weights, exp_avgs, exp_avg_sqs))
        if any(len(x) != n for x in (self.grads, self.weights, *moments)):
            raise ValueError("AdamWPlan: need equally many parameters, gradients, weights and moments")
        decay, lr_scales = _per_tensor(weight_decay, n, "weight_decay"), _per_tensor(lr_scale, n, "lr_scale")
        _check_tensors(self.params, "AdamWPlan: parameters", (torch.float32,))
        given = {"moments": ((torch.float32,), moments), "weights": ((torch.bfloat16, torch.float16), [self.weights])}
        for name, (dtypes, lists) in given.items():
            for xs in lists:
                _check_tensors([x for x in xs if x is not None], f"AdamWPlan: {name}", dtypes)
        for xs in (self.grads, self.weights, *moments):
            pairs = [(p, x) for p, x in zip(self.params, xs) if x is not None]
            if pairs and not _same_layouts(*zip(*pairs)):
                p, x = next(pair for pair in pairs if not _same_layout(*pair))
                raise ValueError(f"AdamWPlan: gradient, weight and moments must have the shape and strides of their parameter "
                                 f"(got {tuple(x.shape)}, {tuple(x.stride())} for {tuple(p.shape)}, {tuple(p.stride())})")
        self._written = self.params + [w for w in self.weights if w is not None]
        state = [x for xs in moments for x in xs if x is not None]
        _refuse_overlaps(self._written + state, self.grads, "AdamWPlan")
        device = _one_device(self.params + self.grads + self._written + state, "AdamWPlan")
        fresh = []
        for xs in moments:
            for i, p in enumerate(self.params):
                if xs[i] is None:           # in the parameter's layout
                    xs[i] = torch.empty_strided(p.shape, p.stride(), dtype=torch.float32, device=device).zero_()
                    fresh.append(xs[i])
        self.exp_avgs, self.exp_avg_sqs = moments
        rows = np.zeros((n, 8), dtype=np.int64)
        rows[:, :4] = _grad_rows(self.grads, self.grads)
        has = np.array([w is not None for w in self.weights])
        rows[:, 1], rows[:, 3] = 0, rows[:, 3] & 0xFFFFFFFF
        rows[has, 1] = _column(_data_ptr, [w for w in self.weights if w is not None])
        _refuse_no_memory(rows[has & (rows[:, 2] > 0), 1], "AdamWPlan")      # further on a 0 stands for "no copy"
        rows[has, 3] |= _column(_DTYPES.get, [w.dtype for w in self.weights if w is not None]) << 32
        for k, xs in enumerate((self.params, self.exp_avgs, self.exp_avg_sqs)):
            rows[:, 4 + k] = _column(_data_ptr, xs)
        rows[:, 7] = np.array([lr_scales, decay], dtype=np.float32).T.copy().view(np.int64)[:, 0]
        self._build(rows, device, "AdamWPlan")
        self.skip_nonfinite = bool(skip_nonfinite)
        self.step = torch.full((), int(step), dtype=torch.int64, device=device)
        self._owned += [self.step, *fresh]
        leaves = [p for p, g in zip(self.params, self.grads) if p.is_leaf and p.grad is not None and _address(p.grad) == g.data_ptr()]
        self._leaves = leaves, [p.grad for p in leaves]
        self._hyper = _lib.AdamWHyper(self.betas[0], self.betas[1], self.eps, 0.0, None, None, None, self.total_norm.data_ptr(),
                                      self.step.data_ptr(), 1.0, -1.0, self._norm, self.skip_nonfinite)
        self._built()

    def _refuse_moved_grads(self) -> None:
        for p, g in zip(*self._leaves):
            if p.grad is not None and _address(p.grad) != g.data_ptr():
                raise RuntimeError(f"AdamWPlan: a parameter of shape {tuple(p.shape)} has another gradient tensor than the plan was built over; "
                                   "keep gradients in place (zero_grad(set_to_none=False)) or build a new plan")

    def run(self, lr, max_norm: float | None = None, grad_scale=1.0, total_norm: torch.Tensor | None = None):
        if any(map(operator.is_not, map(_grad, self._leaves[0]), self._leaves[1])):
            self._refuse_moved_grads()
        max_norm = -1.0 if max_norm is None else _check_max_norm(max_norm, "AdamWPlan")
        h = self._hyper
        h.lr, h.lr_dev = self._factor(lr, "lr")
        h.grad_scale, h.grad_scale_dev = self._factor(grad_scale, "grad_scale")
        h.total_given, h.max_norm = self._given(total_norm), max_norm
        self._run("wq_adamw_items", self._items.data_ptr(), self._n_items, h, self._workspace.data_ptr())
        _bump(self._written)
        if max_norm < 0.0 and not self.skip_nonfinite:
            return None
        return self.total_norm if total_norm is None else total_norm


# ---- the torch.nn.utils forms ---------------------------------------------------------------------------------------

def _grads_of(parameters) -> list:
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return [g for p in parameters if (g := p.grad) is not None]


_SHARED = "gradients share memory (the same tensor twice?); they cannot be clipped in place"


class _List:
    """Tensors as the list entry points take them: host arrays of addresses, element counts and types.  The common case -
    contiguous tensors of one GPU - is found out by passes that stay in C (0.2 us a tensor; with the gathering of gradients, the
    check for shared memory and the version counters of a clip 0.35); anything else is looked at one by one, for the message or
    for the copies that other strides need."""

    def __init__(self, tensors, what: str, written: bool):
        self.copies, given = [], tensors
        selectors = None
        if set(map(type, tensors)) <= _PLAIN_TYPES:
            try:
                index = set(map(_get_device, tensors))
                if len(index) == 1 and all(map(_is_contiguous, tensors)):
                    self.index = index.pop()
                    selectors = list(map(_DTYPES.get, map(_dtype, tensors)))
            except RuntimeError:            # a layout without strides
                pass
        if selectors is None or None in selectors or self.index < 0:
            tensors, selectors = self._one_by_one(tensors, what, written)
        self.tensors, self.device = tensors, torch.device("cuda", self.index)
        self.ptr, self.n = array("q", map(_data_ptr, tensors)), array("q", map(_numel, tensors))
        self.dtype = array("i", selectors)
        if written:
            self._refuse_overlaps(what)
            if self.copies and _share_memory(given):      # of the originals: the copies lie apart
                raise ValueError(f"{what}: {_SHARED}")
        self.args = (self.ptr.buffer_info()[0], self.n.buffer_info()[0], self.dtype.buffer_info()[0], len(tensors))

    def _one_by_one(self, tensors, what: str, written: bool):
        _check_tensors(tensors, what)
        self.index = _one_device(tensors, what).index
        dense = []
        for t in tensors:
            if _is_dense(t):
                dense.append(t)
                continue
            if written:
                _check_no_self_overlap(t, what)
            copy = t.contiguous()
            dense.append(copy)
            self.copies.append((t, copy))
        return dense, [_DTYPES[t.dtype] for t in dense]

    def _refuse_overlaps(self, what: str) -> None:
        if len(self.ptr) <= 16:             # the arrays below cost 8 us however short they are
            spans = sorted((p, p + n * (4 if d == _lib.DTYPE_F32 else 2)) for p, n, d in zip(self.ptr, self.n, self.dtype) if n)
            start, end = [s for s, _ in spans], [e for _, e in spans]
            overlap = any(map(int.__lt__, start[1:], end))
        else:
            at, n = np.frombuffer(self.ptr, np.int64), np.frombuffer(self.n, np.int64)
            order = np.argsort(at[n > 0], kind="stable")
            start = at[n > 0][order]
            end = start + (n * np.where(np.frombuffer(self.dtype, np.int32) == _lib.DTYPE_F32, 4, 2))[n > 0][order]
            overlap = (start[1:] < end[:-1]).any()
        if overlap:
            raise ValueError(f"{what}: {_SHARED}")
        self.spans = start, end

    def writes(self, address: int) -> bool:
        """Whether the fp32 value there lies in a tensor of the list."""
        return _lies_in(address, *self.spans)

    def workspace(self) -> torch.Tensor:
        """Kept by the caller until the launches are out; what comes after them on the stream may reuse it.  Large enough for
        any list of these sizes: as many pieces as fp32 has, and two more per tensor for where it starts."""
        return _workspace(sum(self.n) * 4 // _lib.GRAD_ITEM_BYTES + 2 * len(self.n), self.device)


def _refuse_nonfinite(total: torch.Tensor, norm_type) -> None:
    if not torch.isfinite(total):
        raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients is non-finite, so it cannot be clipped. "
                           "To disable this error and scale the gradients by the non-finite norm anyway, set "
                           "`error_if_nonfinite=False`")


def _total_norm(tensors: _List, norm: int, what: str) -> torch.Tensor:
    device = tensors.device
    total, workspace = torch.empty((), dtype=torch.float32, device=device), tensors.workspace()
    _launch(device, "wq_grad_norm_list", what, *tensors.args, norm, 1.0, workspace.data_ptr(), total.data_ptr())
    return total


def get_total_norm(tensors: torch.Tensor | Iterable[torch.Tensor], norm_type: float = 2.0, error_if_nonfinite: bool = False,
                   foreach: bool | None = None) -> torch.Tensor:
    """``torch.nn.utils.get_total_norm`` for bf16 / fp16 / fp32 tensors on one GPU: the norm (2 or inf) over all elements as a
    0-d fp32 tensor (torch rounds it to the tensors' type).  ``foreach`` is accepted and has no effect."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    norm = _norm_selector(norm_type, "get_total_norm")
    if not tensors:
        return torch.tensor(0.0)
    total = _total_norm(_List(tensors, "get_total_norm", written=False), norm, "get_total_norm")
    if error_if_nonfinite:
        _refuse_nonfinite(total, norm_type)
    return total


def _clip(grads: _List, max_norm: float, norm: int, total_norm, what: str) -> torch.Tensor:
    device = grads.device
    if total_norm is None:
        total, workspace = torch.empty((), dtype=torch.float32, device=device), grads.workspace()
        _launch(device, "wq_grad_clip_list", what, *grads.args, norm, max_norm, 1.0, None, workspace.data_ptr(), total.data_ptr())
    else:
        total = total_norm.detach().resolve_neg().to(device=device, dtype=torch.float32)
        if grads.writes(total.data_ptr()):  # one workgroup would scale it while others read it
            total = total.clone()
        _launch(device, "wq_grad_clip_list", what, *grads.args, norm, max_norm, 1.0, total.data_ptr(), None, None)
    _bump(grads.tensors)
    with torch.no_grad() if grads.copies else nullcontext():
        for t, copy in grads.copies:
            t.copy_(copy)
    return total


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for bf16 / fp16 / fp32 gradients on one GPU: scales the gradients in place by
    ``min(1, max_norm / (norm + 1e-6))`` and returns the norm before the clip as a 0-d fp32 tensor.  Nothing is read back
    unless ``error_if_nonfinite``.  The gradients must not share memory.  ``foreach`` is accepted and has no effect."""
    norm, max_norm = _norm_selector(norm_type, "clip_grad_norm_"), _check_max_norm(max_norm, "clip_grad_norm_")
    grads = _grads_of(parameters)
    if not grads:
        return torch.tensor(0.0)
    grads, total = _List(grads, "clip_grad_norm_", written=True), None
    if error_if_nonfinite:
        total = _total_norm(grads, norm, "clip_grad_norm_")
        _refuse_nonfinite(total, norm_type)
    return _clip(grads, max_norm, norm, total, "clip_grad_norm_")


def clip_grads_with_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, total_norm: torch.Tensor,
                          foreach: bool | None = None) -> None:
    """``torch.nn.utils.clip_grads_with_norm_``: the clip alone, by a norm that the caller has (reduced over ranks, say)."""
    max_norm = _check_max_norm(max_norm, "clip_grads_with_norm_")
    if not isinstance(total_norm, torch.Tensor) or total_norm.numel() != 1:
        raise TypeError("clip_grads_with_norm_: total_norm must be a tensor of one value")
    if hasattr(total_norm, "to_local"):
        raise TypeError("clip_grads_with_norm_: total_norm must be a plain tensor (of a sharded one, pass the full tensor)")
    grads = _grads_of(parameters)
    if grads:
        what = "clip_grads_with_norm_"
        _clip(_List(grads, what, written=True), max_norm, _lib.NORM_2, total_norm, what)

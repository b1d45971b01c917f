"""AdamW over many separate tensors on B200: ``FusedAdamW`` and ``clip_gradients``.

``FusedMLXAdam`` updates the pooled Gaussian slabs of the trainer; a program
that trains a scene through autograd (``rasterize_gaussians_mlx`` on leaf
tensors, or slab views of a pool) with other parameters beside it (appearance
embeddings, pose deltas, exposure, a small network) has a list of tensors of
all sizes instead.  ``FusedAdamW`` steps all of them in one launch:

* decoupled weight decay, per-tensor learning-rate and decay factors;
* parameters and gradients in float32, bfloat16 or float16, optionally with
  float32 master copies of the 16-bit parameters;
* moments in 32 bits, or in 8 (``state_bits=8``: 2.02 bytes a parameter instead
  of 8): 256 neighbours share a scale, and values are rounded without bias over
  steps.  Gradients below 1.1e-5 of the largest among the 256 are damped: their
  second moment has reached the form's lowest step (``moments8.cuh``);
* clipping by the global gradient norm inside the step (``max_norm``), and
  skipping of a step whose gradients are not all finite, without a host sync;
* the step counts on the device, so that ``step`` can be captured into a CUDA
  graph and replayed (``lr`` may be a device tensor; ``grad_scale`` is a number
  of the host, fixed in a graph).

``clip_gradients`` clips a set of gradients on its own, for other optimizers.
"""
from __future__ import annotations

import ctypes
import math
from collections.abc import Mapping
from functools import partial
from operator import attrgetter, is_
from typing import Dict, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib

TYPES = {torch.float32: _lib.GS_F32, torch.bfloat16: _lib.GS_BF16, torch.float16: _lib.GS_F16}
BLOCK = _lib.GS_MOMENT_BLOCK
_F32_MAX = 3.4028234663852886e38
_ENTRY = np.dtype([("param", np.uint64), ("grad", np.uint64), ("n", np.int64), ("state", np.int64),
                   ("cols", np.int64), ("param_stride", np.int64), ("grad_stride", np.int64),
                   ("param_type", np.int32), ("grad_type", np.int32), ("lr_scale", np.float64),
                   ("decay", np.float64)], align=True)
_data_ptr = torch.Tensor.data_ptr
_is_contiguous = torch.Tensor.is_contiguous
_is_neg = torch.Tensor.is_neg
_device_index = torch.Tensor.get_device
_dtype = attrgetter("dtype")
_shape = attrgetter("shape")
_stride = torch.Tensor.stride
_is_none = partial(is_, None)


def rows_of(t: torch.Tensor) -> Optional[Tuple[int, int]]:
    """``(cols, stride)`` of a tensor whose elements, in order, are rows of
    ``cols`` adjacent ones ``stride`` apart (``(n, n)`` when it is dense), or
    None when it has no such form (transposed, broadcast, two strides)."""
    n = t.numel()
    if t.is_contiguous():
        return max(n, 1), max(n, 1)
    dims = [(s, d) for s, d in zip(t.stride(), t.shape) if d != 1]
    cols = 1
    while dims and dims[-1][0] == cols:
        cols *= dims.pop()[1]
    if not dims:
        return n, n
    stride, rows = dims.pop()
    if stride < cols:
        return None
    reach = stride * rows
    while dims:
        s, d = dims.pop()
        if s != reach:
            return None
        reach *= d
    return cols, stride


def _span(t: torch.Tensor, rows: Tuple[int, int]) -> Tuple[int, int]:
    cols, stride = rows
    last = (t.numel() // cols - 1) * stride + cols
    return t.data_ptr(), t.data_ptr() + last * t.element_size()


def overlapping(tensors: Sequence[torch.Tensor], rows: Sequence[Tuple[int, int]]) -> Optional[Tuple[int, int]]:
    """Two of the tensors that share an element, or None.  Columns of one slab
    interleave without sharing; what cannot be told apart counts as shared."""
    items = sorted(((*_span(t, r), k) for k, (t, r) in enumerate(zip(tensors, rows)) if t.numel()))
    group: List[Tuple[int, int, int]] = []
    reach = -1
    for lo, hi, k in items:
        if lo >= reach:
            group = []
        for lo2, hi2, j in group:
            if hi2 <= lo:
                continue
            # two sets of rows share nothing when their columns lie apart modulo a distance that divides both pitches
            (cj, sj), (ck, sk) = rows[j], rows[k]
            bj, bk = tensors[j].element_size(), tensors[k].element_size()
            pitch = math.gcd(sj * bj, sk * bk)
            at = (lo - lo2) % pitch
            if not (sj > cj and sk > ck and cj * bj <= at and at + ck * bk <= pitch):
                return j, k
        group.append((lo, hi, k))
        reach = max(reach, hi)
    return None


def _check_tensor(what: str, t) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    if t.layout != torch.strided:
        raise ValueError(f"{what}: sparse tensors are not supported")
    if t.dtype not in TYPES:
        raise ValueError(f"{what}: {t.dtype} is not float32, bfloat16 or float16")


def _check_written(what: str, t) -> None:
    _check_tensor(what, t)
    if t.is_neg():
        raise ValueError(f"{what}: a view that reads as the negative of its memory cannot be written")


def _check_cuda(tensors: Sequence[torch.Tensor]) -> torch.device:
    index = set(map(_device_index, tensors))
    if len(index) == 1 and index != {-1}:
        return torch.device("cuda", index.pop())
    devices = {t.device for t in tensors}
    if len(devices) != 1:
        raise ValueError(f"all tensors must be on one device, got {sorted(map(str, devices))}")
    device = devices.pop()
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, not {device}")
    return device


class _on_device:
    """Makes a device the current one where it is not (launches go to the
    current device's context)."""

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.prev != self.index:
            torch.cuda.set_device(self.prev)


def _copied(entries: np.ndarray) -> np.ndarray:
    return entries.view(np.uint8).copy().view(_ENTRY)  # (a copy of bytes: field by field it takes 7 us)


def _changed(tensors: List[torch.Tensor]) -> None:
    """Tells autograd that the tensors were written."""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:  # inference tensors have no version
        torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def _dense(tensors: List) -> List:
    """Dense tensors in the place of strided ones (anything else is left to the
    checks)."""
    return [t if not isinstance(t, torch.Tensor) or t.layout != torch.strided or t.is_contiguous() else t.contiguous()
            for t in tensors]


def _norm_partials(lib, entries: int, n: int, buffer: torch.Tensor, stream: int) -> int:
    count = ctypes.c_int64(0)
    _lib.check(lib.gs_grad_norm_partials(entries, n, buffer.data_ptr(), buffer.numel(), ctypes.byref(count), stream),
               "gradient norm")
    return count.value


class FusedAdamW:
    """AdamW over the tensors of ``params`` (name -> tensor, updated in place).

    ``lr``: a float, or a one-element float32 tensor on the parameters' device
    that each step reads there.  ``lr_scales`` / ``decay_scales``: per-name
    factors of ``lr`` and ``weight_decay`` (1 where a name is missing).
    ``state_bits``: 32 or 8.  ``master_weights``: keep float32 copies of the
    16-bit parameters and round the parameters from them (call
    ``sync_master`` after changing such parameters elsewhere; the slab of
    copies has room for every parameter, 4 bytes an element, also where only
    some have 16 bits).  ``max_norm``: clip the gradients to this global norm
    inside the step.
    ``skip_nonfinite``: leave parameters, moments and the step count as they
    are when a gradient is not finite (a step with ``max_norm`` always does).

    A parameter without a gradient in a step keeps its values and moments and
    does not count the step: its bias corrections are those of the steps that
    it took itself.

    Parameters may be strided rows (a pool's columns) but not permuted ones
    (transposed, channels last); they may not overlap, and gradients may not
    lie in their memory.
    ``lr``, ``weight_decay``, ``beta1``, ``beta2``, ``eps``, ``max_norm`` and
    ``skip_nonfinite`` may be changed between steps (a captured step keeps the
    values it was captured with, but for a tensor ``lr``).  The optimizer
    belongs to one stream at a time, as its parameters do."""

    def __init__(self, params: Dict[str, torch.Tensor], lr: Union[float, torch.Tensor] = 1e-3,
                 betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 lr_scales: Optional[Dict[str, float]] = None, decay_scales: Optional[Dict[str, float]] = None,
                 state_bits: int = 32, master_weights: bool = False, max_norm: Optional[float] = None,
                 skip_nonfinite: bool = False):
        if not params:
            raise ValueError("no parameters")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must be in [0, 1): {betas}")
        if not (math.isfinite(eps) and eps >= 2.0 ** -126):
            raise ValueError(f"eps must be positive (a normal float32): {eps}")
        if not (math.isfinite(weight_decay) and weight_decay >= 0.0):
            raise ValueError(f"weight_decay must not be negative: {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32: {state_bits}")
        for what, scales in (("lr_scales", lr_scales), ("decay_scales", decay_scales)):
            unknown = set(scales or ()) - set(params)
            if unknown:
                raise ValueError(f"{what}: no parameter named {sorted(unknown)}")
            if not all(math.isfinite(x) for x in (scales or {}).values()):
                raise ValueError(f"{what} must be finite")
        self.names = list(params)
        self._params = [params[k] for k in self.names]
        self._rows = []
        for name, p in params.items():
            _check_written(f"parameter {name!r}", p)
            rows = rows_of(p)
            if rows is None:
                raise ValueError(f"parameter {name!r}: strides {tuple(p.stride())} of shape {tuple(p.shape)} are "
                                 "neither dense nor rows at one distance")
            self._rows.append(rows)
        both = overlapping(self._params, self._rows)
        if both is not None:
            raise ValueError(f"parameters {self.names[both[0]]!r} and {self.names[both[1]]!r} share memory")
        self.device = _check_cuda(self._params)
        self.beta1, self.beta2 = float(betas[0]), float(betas[1])
        self.eps = float(eps)
        self.state_bits = state_bits
        self.skip_nonfinite = bool(skip_nonfinite)
        self.lr = lr
        self.max_norm = max_norm
        self._lr_value()
        self._norm_limit()
        self._shapes = list(map(_shape, self._params))
        self._take_memory()
        n = len(self._params)
        sizes = [p.numel() for p in self._params]
        room = [-(-s // BLOCK) * BLOCK for s in sizes]
        self.offsets = {k: o for k, o in zip(self.names, np.cumsum([0] + room[:-1]).tolist())}
        self.slab_elements = sum(room)
        e = np.zeros(n, _ENTRY)
        e["param"], e["n"] = self._ptrs, sizes
        e["state"] = [self.offsets[k] for k in self.names]
        e["cols"] = [c for c, _ in self._rows]
        e["param_stride"] = [s for _, s in self._rows]
        e["param_type"] = [TYPES[p.dtype] for p in self._params]
        e["lr_scale"] = [float((lr_scales or {}).get(k, 1.0)) for k in self.names]
        self._entries, self._at = e, e.ctypes.data
        self._decay_scales = np.array([float((decay_scales or {}).get(k, 1.0)) for k in self.names])
        self.weight_decay = weight_decay
        dt = torch.float32 if state_bits == 32 else torch.uint8
        self.m = torch.zeros(self.slab_elements, dtype=dt, device=self.device)
        self.v = torch.zeros(self.slab_elements, dtype=dt, device=self.device)
        blocks = self.slab_elements // BLOCK if state_bits == 8 else 0
        self.m_exp = torch.zeros(blocks, dtype=torch.uint8, device=self.device)
        self.v_exp = torch.zeros(blocks, dtype=torch.uint8, device=self.device)
        # steps taken, the kernel's own (upper half: look at what follows), per parameter the steps without its gradient
        self._control = torch.zeros(2 + n, dtype=torch.int64, device=self.device)
        self._count, self._missed = self._control[0], self._control[2:]
        self._any_missed = False  # whether any call so far left a parameter out
        self._found = (ctypes.c_ssize_t * 2)()
        self.master_slab: Optional[torch.Tensor] = None
        if master_weights and any(p.dtype != torch.float32 for p in self._params):
            self.master_slab = torch.zeros(self.slab_elements, dtype=torch.float32, device=self.device)
            self.sync_master()
        self._state = _lib.GsAdamWState(_lib.ptr(self.m), _lib.ptr(self.v), _lib.ptr(self.m_exp),
                                        _lib.ptr(self.v_exp), _lib.ptr(self.master_slab), _lib.ptr(self._control),
                                        state_bits, 1)
        self._partials: Optional[torch.Tensor] = None
        if max_norm is not None or skip_nonfinite:
            self._partials_buffer(_lib.lib())

    @property
    def weight_decay(self) -> float:
        return self._weight_decay

    @weight_decay.setter
    def weight_decay(self, value: float) -> None:
        if not (math.isfinite(value) and value >= 0.0):
            raise ValueError(f"weight_decay must not be negative: {value}")
        self._weight_decay = float(value)
        self._entries["decay"] = self._weight_decay * self._decay_scales

    # ------------------------------------------------------------------ checks
    def _lr_value(self) -> Tuple[float, Optional[int]]:
        lr = self.lr
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != self.device:
                raise ValueError("a tensor lr is one float32 on the parameters' device")
            if lr.is_neg():
                raise ValueError("a tensor lr may not be a view that reads as the negative of its memory")
            return 0.0, lr.data_ptr()
        lr = float(lr)
        if not (math.isfinite(lr) and lr >= 0.0):
            raise ValueError(f"lr must not be negative: {lr}")
        return lr, None

    def _norm_limit(self) -> float:
        if self.max_norm is None:
            return math.inf
        limit = float(self.max_norm)
        if not limit > 0.0:
            raise ValueError(f"max_norm must be positive: {self.max_norm}")
        return limit

    def _partials_buffer(self, lib) -> torch.Tensor:
        if self._partials is None:
            with _on_device(self.device):
                size = lib.gs_grad_norm_max_partials(len(self._params))
            self._partials = torch.empty(size, dtype=torch.float64, device=self.device)
        return self._partials

    def _take_memory(self) -> None:
        # aliases keep the memory that the entries point to alive, and its layout, whatever happens to the caller's
        # tensors
        self._aliases = [p.detach() for p in self._params]
        self._ptrs = list(map(_data_ptr, self._params))
        self._types = list(map(_dtype, self._params))
        self._strides = list(map(_stride, self._params))

    def _as_taken(self) -> bool:
        """Whether the parameters are the memory, types and layouts of the entries."""
        ps = self._params
        native = _lib.tensors()
        if native is not None:
            return not native.gst_params_as_taken(ps, self._aliases, self._at, len(ps))
        return list(map(_data_ptr, ps)) == self._ptrs and list(map(_dtype, ps)) == self._types and \
            list(map(_shape, ps)) == self._shapes and list(map(_stride, ps)) == self._strides and \
            not any(map(_is_neg, ps))

    def _refresh(self) -> None:
        """The parameters' memory was replaced (``p.data = ...``): takes the new
        memory when it has the old form."""
        for k, (name, p) in enumerate(zip(self.names, self._params)):
            if p.layout != torch.strided or p.dtype != self._types[k] or p.shape != self._shapes[k] or \
                    p.device != self.device or rows_of(p) != self._rows[k] or p.is_neg():
                raise ValueError(f"parameter {name!r} no longer has the type, shape, strides or device it was "
                                 "given with")
        both = overlapping(self._params, self._rows)
        if both is not None:
            raise ValueError(f"parameters {self.names[both[0]]!r} and {self.names[both[1]]!r} share memory")
        self._take_memory()
        self._entries["param"] = self._ptrs

    def _elements_in(self, entries: np.ndarray) -> bool:
        return self.slab_elements > 0 if entries is self._entries else bool(entries["n"].any())

    def _with_grads(self, entries: np.ndarray, names: Sequence[str], shapes: Sequence[torch.Size],
                    grads: List[torch.Tensor], what: str = "gradient") -> Tuple[np.ndarray, List[torch.Tensor]]:
        """Fills the entries' second tensor from ``grads`` (checked against
        ``shapes``); returns the entries (a copy where their rows had to change)
        and the tensors that must outlive the launch."""
        try:
            if any(map(_is_neg, grads)):  # views that read as the negative of their memory (autograd makes some)
                grads = [g.resolve_neg() for g in grads]
            types = list(map(_dtype, grads))
            codes = list(map(TYPES.__getitem__, types)) if types.count(types[0]) != len(types) else TYPES[types[0]]
            same = list(map(_shape, grads)) == shapes
            here = set(map(_device_index, grads)) == {self.device.index}
            dense = all(map(_is_contiguous, grads))
            entries["grad"] = ptrs = list(map(_data_ptr, grads))
        except (KeyError, AttributeError, TypeError, RuntimeError):
            for name, g in zip(names, grads):
                _check_tensor(f"{what} of {name!r}", g)
            raise
        if not same:
            for name, s, g in zip(names, shapes, grads):
                if g.shape != s:
                    raise ValueError(f"{what} of {name!r} has shape {tuple(g.shape)}, not {tuple(s)}")
        if not here:
            raise ValueError(f"every {what} must be on {self.device}")
        if 0 in ptrs and ((entries["grad"] == 0) & (entries["n"] > 0)).any():
            raise ValueError(f"a {what} has no memory")
        entries["grad_type"] = codes
        entries["grad_stride"] = entries["cols"]
        if not dense:
            entries, grads = entries.copy(), list(grads)
            for k, g in enumerate(grads):
                if g.is_contiguous():
                    continue
                rows = rows_of(g)
                cols, stride = int(entries["cols"][k]), int(entries["param_stride"][k])
                if rows is not None and rows[0] == cols:
                    entries["grad_stride"][k] = rows[1]
                elif rows is not None and cols == stride:  # a dense parameter takes the gradient's rows
                    entries["cols"][k] = entries["param_stride"][k] = rows[0]
                    entries["grad_stride"][k] = rows[1]
                else:
                    grads[k] = g.contiguous()
                    entries["grad"][k] = grads[k].data_ptr()
        return entries, grads

    # ------------------------------------------------------------------ the step
    def step(self, grads: Optional[Dict[str, torch.Tensor]] = None, grad_scale: float = 1.0) -> Optional[torch.Tensor]:
        """One step on the current stream.  ``grads``: name -> gradient (default:
        the parameters' ``.grad``); a parameter without one keeps its values and
        moments and misses the step, and a step without any does nothing.
        ``grad_scale`` multiplies every gradient first (the inverse of a loss
        scale).  Returns the global norm of the scaled gradients before clipping
        as a device scalar when ``max_norm`` or ``skip_nonfinite`` asks for it,
        else None."""
        lib = _lib.lib()
        if grads is not None and not isinstance(grads, Mapping):
            raise TypeError(f"gradients are given by name, not as {type(grads).__name__}")
        grad_scale = float(grad_scale)
        if not abs(grad_scale) <= _F32_MAX:
            raise ValueError(f"grad_scale must be finite in float32: {grad_scale}")
        lr, lr_device = self._lr_value()
        limit = self._norm_limit()
        names, shapes, params, entries, on = self.names, self._shapes, self._params, self._entries, None
        native = _lib.tensors()
        # gradients dense and as expected, or missing: the table is filled natively
        filled = native is not None and not native.gst_step(grads, names, params, self._aliases, self._at, len(params),
                                                            self.device.index, self._found)
        if filled:
            elements = self._found[1] != 0
            self._any_missed |= self._found[0] != len(params)
        else:
            if grads is None:
                found = [p.grad for p in params]
            else:
                found = list(map(grads.get, names))
            if not self._as_taken():
                self._refresh()
            none = any(map(_is_none, found))
            if (none or (grads is not None and len(grads) != len(found))) and grads is not None and \
                    not grads.keys() <= self.offsets.keys():
                raise ValueError(f"no parameter named {sorted(set(grads) - set(names))}")
            if none:
                on = [k for k, g in enumerate(found) if g is not None]
                entries = entries[on]
                names, shapes, params, found = ([x[k] for k in on] for x in (names, shapes, params, found))
            elements = self._elements_in(entries)
        with_norm = self.max_norm is not None or self.skip_nonfinite
        norm = None
        with _on_device(self.device):
            if with_norm:
                norm = torch.empty((), dtype=torch.float32, device=self.device)
            if not elements:
                return norm.zero_() if with_norm else None
            if not filled:
                entries, keep = self._with_grads(entries, names, shapes, found)
            at, count = self._at if entries is self._entries else entries.ctypes.data, len(entries)
            stream = _lib.stream_ptr(self.device)
            s = _lib.GsAdamWSettings(lr, self.beta1, self.beta2, self.eps, grad_scale, lr_device, None, 0, limit, None)
            if with_norm:
                buffer = self._partials_buffer(lib)
                s.num_partials = _norm_partials(lib, at, count, buffer, stream)
                s.norm_partials = buffer.data_ptr()
                s.norm_out = norm.data_ptr()
            if on is not None:  # the step takes the whole list, those that miss it without a gradient
                every = _copied(self._entries)
                every["grad"] = 0
                every[on] = entries
                at, count, self._any_missed = every.ctypes.data, len(every), True
            _lib.check(lib.gs_adamw_step(at, count, self._state, s, stream), "adamw step")
        if not filled:
            del keep
            _changed(params)
        return norm

    # ------------------------------------------------------------------ state
    @property
    def t(self) -> int:
        """Steps taken (read from the device: a host sync).  Setting it makes
        every parameter one that took that many."""
        return int(self._count)

    @t.setter
    def t(self, value: int) -> None:
        if value < 0:
            raise ValueError(f"the step count must not be negative: {value}")
        self._set_steps(value)

    def _set_steps(self, value: int) -> None:
        self._count.fill_(int(value))
        if self._any_missed:
            self._control[1:].zero_()

    def _views(self, slab: torch.Tensor) -> Dict[str, torch.Tensor]:
        return {k: slab[self.offsets[k]:self.offsets[k] + s.numel()].view(s)
                for k, s in zip(self.names, self._shapes)}

    def moment_slabs(self, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """m and v as flat slabs (``offsets`` gives each tensor's place; the
        padding between them is zero).  The optimizer's own buffers when the
        moments are float32 and ``dtype`` is too, else new tensors; bfloat16
        holds every value of the 8-bit form exactly."""
        if self.state_bits == 32:
            return self.m.to(dtype), self.v.to(dtype)
        return _dequantize(self.m, self.v, self.m_exp, self.v_exp, dtype)

    def moments(self, dtype: torch.dtype = torch.float32) -> Tuple[Dict[str, torch.Tensor], Dict[str, torch.Tensor]]:
        """``moment_slabs`` as name -> tensor of the parameter's shape."""
        m, v = self.moment_slabs(dtype)
        return self._views(m), self._views(v)

    def load_moments(self, m: Dict[str, torch.Tensor], v: Dict[str, torch.Tensor], t: Optional[int] = None) -> None:
        """Sets every parameter's moments (tensors of the parameters' shapes on
        their device, any of the three types; v must not be negative) and the
        step count, which is then every parameter's (None: the counts stay).
        With 8-bit moments values that the form holds are kept exactly and
        others are rounded with the step count's offsets."""
        if m.keys() != self.offsets.keys() or v.keys() != self.offsets.keys():
            raise ValueError("moments for exactly the optimizer's parameters are needed")
        if t is not None and t < 0:
            raise ValueError(f"the step count must not be negative: {t}")
        ml, vl = list(map(m.__getitem__, self.names)), list(map(v.__getitem__, self.names))
        with _on_device(self.device):
            entries = _copied(self._entries)
            entries["cols"] = entries["param_stride"] = np.maximum(entries["n"], 1)
            # a tensor's first place takes its m, the second its v
            ml = self._fill_dense(entries, ml, "moment m")
            entries["param"], entries["param_type"] = entries["grad"], entries["grad_type"]
            vl = self._fill_dense(entries, vl, "moment v")
            if t is None:
                t = self.t if self.state_bits == 8 else None
            else:
                self._set_steps(t)
            if self.state_bits == 32:
                torch._foreach_copy_(list(self._views(self.m).values()) + list(self._views(self.v).values()),
                                     [x.detach() for x in ml + vl])
                return
            lib = _lib.lib()
            _lib.check(lib.gs_moments8_quantize(entries.ctypes.data, len(entries), self.m.data_ptr(),
                                                self.v.data_ptr(), self.m_exp.data_ptr(), self.v_exp.data_ptr(),
                                                int(t), _lib.stream_ptr(self.device)), "8-bit moments")

    def _fill_dense(self, entries: np.ndarray, tensors: List[torch.Tensor], what: str) -> List[torch.Tensor]:
        native = _lib.tensors()
        if native is None or native.gst_fill(tensors, None, None, self._aliases, entries.ctypes.data, len(tensors),
                                             self.device.index):
            _, tensors = self._with_grads(entries, self.names, self._shapes, _dense(tensors), what)
        return tensors

    def sync_master(self) -> None:
        """Takes the float32 master copies from the parameters again."""
        if self.master_slab is not None:
            torch._foreach_copy_(list(self._views(self.master_slab).values()), [p.detach() for p in self._params])

    def state_dict(self) -> Dict[str, object]:
        """A copy of the state: the moments in the form they are held in, the
        master copies, the step count, the steps that each parameter missed and
        the layout."""
        d = {"state_bits": self.state_bits, "t": self.t, "missed": self._missed.clone(),
             "shapes": {k: tuple(s) for k, s in zip(self.names, self._shapes)},
             "m": self.m.clone(), "v": self.v.clone(), "m_exp": self.m_exp.clone(), "v_exp": self.v_exp.clone()}
        if self.master_slab is not None:
            d["master"] = self.master_slab.clone()
        return d

    def load_state_dict(self, d: Dict[str, object]) -> None:
        """Restores a ``state_dict`` of the same parameters (names in the same
        order, and shapes); moments held in the other number of bits are
        converted."""
        if list(d["shapes"].items()) != [(k, tuple(s)) for k, s in zip(self.names, self._shapes)]:
            raise ValueError("the state belongs to other parameters")
        bits = d["state_bits"]
        m, v = d["m"].to(self.device), d["v"].to(self.device)
        if self.master_slab is not None:
            if "master" in d:
                self.master_slab.copy_(d["master"])
            else:
                self.sync_master()
        if bits == self.state_bits:
            for dst, src in ((self.m, m), (self.v, v), (self.m_exp, d["m_exp"]), (self.v_exp, d["v_exp"])):
                dst.copy_(src)
            self.t = d["t"]
        else:
            if bits == 8:
                m, v = _dequantize(m, v, d["m_exp"].to(self.device), d["v_exp"].to(self.device), torch.float32)
            self.load_moments(self._views(m), self._views(v), t=d["t"])
        if "missed" in d:
            self._missed.copy_(d["missed"])
            self._control[1].fill_(1 << 32)
            self._any_missed = True


def _dequantize(m, v, m_exp, v_exp, dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"8-bit moments are read as float32 or bfloat16, not {dtype}")
    lib = _lib.lib()
    with _on_device(m.device):
        mo = torch.empty(m.numel(), dtype=dtype, device=m.device)
        vo = torch.empty(v.numel(), dtype=dtype, device=v.device)
        _lib.check(lib.gs_moments8_dequantize(m.data_ptr(), v.data_ptr(), m_exp.data_ptr(), v_exp.data_ptr(),
                                              m.numel(), TYPES[dtype], mo.data_ptr(), vo.data_ptr(),
                                              _lib.stream_ptr(m.device)), "moment values")
    return mo, vo


Tensors = Union[Dict[str, torch.Tensor], Sequence[torch.Tensor]]


def clip_gradients(grads: Tensors, max_norm: float, out: Optional[Tensors] = None) -> torch.Tensor:
    """Scales the gradients (name -> tensor, or a sequence) by ``max_norm`` over
    their global norm where that exceeds ``max_norm``, in place, or into the
    tensors of ``out`` (same names and shapes, any of the three types; written
    in any case).  Returns the norm before as a device scalar; where it is not
    finite nothing is scaled.  Strided rows are taken as they are; written
    tensors may not overlap one another or other gradients."""
    max_norm = float(max_norm)
    if not max_norm > 0.0:
        raise ValueError(f"max_norm must be positive: {max_norm}")
    if isinstance(grads, dict):
        names, gl = list(grads), list(grads.values())
        if out is not None:
            if not isinstance(out, dict) or out.keys() != grads.keys():
                raise ValueError("out must have the gradients' names")
            ol = list(map(out.__getitem__, names))
    else:
        names, gl = range(len(grads)), list(grads)
        if out is not None:
            ol = list(out)
            if len(ol) != len(gl):
                raise ValueError(f"{len(ol)} tensors in out for {len(gl)} gradients")
    if not gl:
        raise ValueError("no gradients")
    if out is None:
        ol = gl
    n = len(gl)
    native = _lib.tensors()
    if native is not None:
        table, found = (ctypes.c_char * (_ENTRY.itemsize * n))(), (ctypes.c_int * 2)()
        at = ctypes.addressof(table)
    filled = native is not None and not native.gst_clip(gl, ol, at, n, found)
    if filled:
        device, elements = torch.device("cuda", found[0]), found[1]
    else:
        entries, gl = _clip_entries(names, gl, ol)
        device, elements, at = _check_cuda(gl + ol), entries["n"].any(), entries.ctypes.data
    lib = _lib.lib()
    with _on_device(device):
        norm = torch.empty((), dtype=torch.float32, device=device)
        if not elements:
            return norm.zero_()
        stream = _lib.stream_ptr(device)
        partials = torch.empty(lib.gs_grad_norm_max_partials(n), dtype=torch.float64, device=device)
        count = _norm_partials(lib, at, n, partials, stream)
        _lib.check(lib.gs_clip_gradients(at, n, partials.data_ptr(), count, max_norm, norm.data_ptr(), stream),
                   "clip gradients")
    if not filled:
        _changed(ol)
    return norm


def _clip_entries(names, gl: List[torch.Tensor], ol: List[torch.Tensor]) -> Tuple[np.ndarray, List[torch.Tensor]]:
    """The entries of any tensors, with the refusals; and the gradients, copies
    in the place of those that are not rows or read as the negative of their memory."""
    in_place = ol is gl
    for name, g, o in zip(names, gl, ol):
        _check_tensor(f"gradient {name!r}", g)
        _check_written(f"{'gradient' if in_place else 'out'} {name!r}", o)
        if o.shape != g.shape:
            raise ValueError(f"out {name!r} has shape {tuple(o.shape)}, not {tuple(g.shape)}")
    gl = [g.resolve_neg() for g in gl]
    g_rows, o_rows = list(map(rows_of, gl)), list(map(rows_of, ol))
    for name, o, rows in zip(names, ol, o_rows):
        if rows is None:
            raise ValueError(f"{'gradient' if in_place else 'out'} {name!r}: strides {tuple(o.stride())} of shape "
                             f"{tuple(o.shape)} are neither dense nor rows at one distance")
    if overlapping(ol, o_rows) is not None:
        raise ValueError("written tensors share memory")
    if not in_place:
        _check_apart(gl, ol, o_rows)
    entries = np.zeros(len(gl), _ENTRY)
    for k, (g, o) in enumerate(zip(gl, ol)):
        (o_cols, o_stride), rows = o_rows[k], g_rows[k]
        if rows is None or not (rows[0] == rows[1] or o_cols in (o_stride, rows[0])):
            g = gl[k] = g.contiguous()
            rows = rows_of(g)
        g_dense, o_dense = rows[0] == rows[1], o_cols == o_stride
        cols = o_cols if g_dense else rows[0]
        entries[k] = (o.data_ptr(), g.data_ptr(), g.numel(), 0, cols, cols if o_dense else o_stride,
                      cols if g_dense else rows[1], TYPES[o.dtype], TYPES[g.dtype], 1.0, 0.0)
    return entries, gl


def _check_apart(gl: List[torch.Tensor], ol: List[torch.Tensor], o_rows) -> None:
    """A written tensor may be its own gradient's memory, but no other's."""
    spans = sorted(_span(o, r) for o, r in zip(ol, o_rows) if o.numel())
    for g, o in zip(gl, ol):
        if not g.numel() or (g.data_ptr() == o.data_ptr() and g.dtype == o.dtype and g.stride() == o.stride()):
            continue
        lo = g.data_ptr()
        hi = lo + (sum((d - 1) * s for d, s in zip(g.shape, g.stride())) + 1) * g.element_size()
        if any(a < hi and b > lo for a, b in spans):
            raise ValueError("a written tensor shares memory with another gradient")

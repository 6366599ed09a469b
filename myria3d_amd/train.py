"""Training-step pieces that sit right behind the net: the reference's criterion and optimizer, MI355X-native.

* ``cross_entropy`` — ``torch.nn.CrossEntropyLoss(ignore_index=65)`` on the logits
  (``/root/reference/myria3d/models/model.py:118``, ``configs/model/criterion/CrossEntropyLoss.yaml:1-3``).
* ``FusedAdam`` — ``torch.optim.Adam`` (``/root/reference/configs/model/optimizer/Adam.yaml:1-4``) as ONE kernel
  launch over the flat parameter / gradient buffers of a ``HipRandLANet`` that has run ``flatten_parameters()``;
  stock torch runs ~250 small launches for the same update (141 parameter tensors).
* ``AdamW`` — ``torch.optim.AdamW`` over any list of parameter tensors (a net that is not flattened, ``HipPointNet2``, frozen
  parts, several groups, bf16 or fp16 parameters), 152 tensors a launch, its moments in 32 or in 8 bits, clipping included.
* ``clip_grad_norm_`` — ``torch.nn.utils.clip_grad_norm_`` (Lightning's ``gradient_clip_val``) in two passes over all gradients.
"""
from __future__ import annotations

import copy
import ctypes
import math
from array import array
from itertools import repeat
from operator import attrgetter, is_, is_not
from typing import Dict, Iterable, List, Optional, Tuple, Union

import torch
import torch.distributed as dist
from torch import Tensor

from . import _lib, ops
from ._lib import call
from .ops import cross_entropy  # noqa: F401  (re-export)


class FusedAdam(torch.optim.Optimizer):
    """Adam over ``net.flat_parameters`` / ``net.flat_grads`` (same update rule and defaults as ``torch.optim.Adam``,
    ``amsgrad=False``).  ``step()`` also clears the gradient buffer (``zero_grad`` is then free), and under
    ``torch.distributed`` all-reduces the flat gradient first when ``all_reduce=True`` — one RCCL collective on
    the 4.45 MB bucket, no packing copies.

    ``state_dict()`` / ``load_state_dict()`` speak ``torch.optim.Adam``'s format (per-parameter ``step`` /
    ``exp_avg`` / ``exp_avg_sq``), so Lightning checkpoints (``ckpt_path`` resume, ``/root/reference/myria3d/train.py:145``)
    keep the Adam moments and the bias-correction step, and a run started with the reference's ``torch.optim.Adam``
    can be resumed here (and the other way round).  One parameter group, every parameter trainable: the single
    launch updates the whole flat buffer."""

    def __init__(self, net, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                 all_reduce: bool = False, overlap_wgrad: bool = True, force_collective: bool = False):
        if net.flat_parameters is None:
            net.flatten_parameters()
        self.net = net
        params = list(net.parameters())
        if any(not p.requires_grad for p in params):
            raise ValueError("FusedAdam updates the whole flat parameter buffer: frozen parameters "
                             "(requires_grad=False) are not supported — use torch.optim.Adam for partial fine-tuning")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        flat = net.flat_parameters
        self.exp_avg = torch.zeros_like(flat)
        self.exp_avg_sq = torch.zeros_like(flat)
        # device-side state of m3d_adam_step: [0] the step counter (fp32), then the arrival tickets of the update's workgroups
        self._adam_state = torch.zeros(66, dtype=torch.float32, device=flat.device)  # (M3D_ADAM_STATE_WORDS)
        self.step_count = self._adam_state[:1]
        self.lr_dev: Optional[torch.Tensor] = None  # optional device-side learning rate (graph-replay safe)
        self.all_reduce = all_reduce
        # run the gradient all-reduce even on a 1-rank process group (exercises RCCL and its interplay with hipGraph
        # capture on a one-GPU box: tests, ``bench.py --force-collective``)
        self.force_collective = force_collective
        if overlap_wgrad and flat.is_cuda:  # weight-gradient GEMMs run beside the rest of the backward pass
            net.grad_side = ops.GradSideStream(flat.device)

    def add_param_group(self, param_group):
        if len(self.param_groups) >= 1:
            raise ValueError("FusedAdam supports exactly one parameter group (one launch over the flat buffer)")
        super().add_param_group(param_group)

    # ------------------------------------------------------------------------------------------
    def _slices(self):
        off = 0
        for p in self.net.parameters():
            n = p.numel()
            yield p, off, n
            off += (n + 3) // 4 * 4

    def state_dict(self):
        """``torch.optim.Adam``'s layout: ``state[i] = {step, exp_avg, exp_avg_sq}`` per parameter index."""
        step = self.step_count.detach().reshape(()).clone().cpu()
        state = {}
        for i, (p, off, n) in enumerate(self._slices()):
            state[i] = {"step": step.clone(),
                        "exp_avg": self.exp_avg[off:off + n].view(p.shape).clone(),
                        "exp_avg_sq": self.exp_avg_sq[off:off + n].view(p.shape).clone()}
        groups = [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]
        groups[0]["params"] = list(range(len(state)))
        return {"state": state, "param_groups": groups}

    def load_state_dict(self, state_dict):
        groups = state_dict["param_groups"]
        if len(groups) != 1:
            raise ValueError("FusedAdam supports exactly one parameter group")
        slices = list(self._slices())
        if len(groups[0]["params"]) != len(slices):
            raise ValueError("loaded state dict has a different number of parameters")
        if groups[0].get("amsgrad", False) or groups[0].get("maximize", False):
            raise ValueError("FusedAdam implements amsgrad=False, maximize=False only")
        state = state_dict["state"]
        steps = set()
        with torch.no_grad():
            self.exp_avg.zero_(), self.exp_avg_sq.zero_()
            for key, (p, off, n) in zip(groups[0]["params"], slices):
                st = state.get(key, state.get(str(key)))
                if st is None:  # torch.optim.Adam has no entry for a parameter that was never stepped
                    continue
                if tuple(st["exp_avg"].shape) != tuple(p.shape):
                    raise ValueError(f"optimizer state of parameter {key} has shape {tuple(st['exp_avg'].shape)}, "
                                     f"expected {tuple(p.shape)}")
                self.exp_avg[off:off + n].copy_(st["exp_avg"].reshape(-1))
                self.exp_avg_sq[off:off + n].copy_(st["exp_avg_sq"].reshape(-1))
                steps.add(float(st["step"]))
            if len(steps) > 1:
                raise ValueError(f"FusedAdam keeps ONE step counter; the loaded state has {sorted(steps)}")
            self.step_count.fill_(steps.pop() if steps else 0.0)
        for k, v in groups[0].items():
            if k != "params" and k in self.param_groups[0]:
                self.param_groups[0][k] = v

    # ------------------------------------------------------------------------------------------
    @torch.no_grad()
    def reduce_gradients(self) -> float:
        """Joins the weight-gradient side stream and, with ``all_reduce`` under ``torch.distributed``, sums the flat
        gradient bucket over the ranks with ONE collective.  Returns the scale (1 / world size) the update applies."""
        net = self.net
        if net.grad_side is not None:
            net.grad_side.join()  # the weight-gradient side stream has finished writing the flat gradient buffer
        if not net._flat_intact():
            net._check_flat()
        if self.uses_collective():
            dist.all_reduce(net.flat_grads, op=dist.ReduceOp.SUM)
            return 1.0 / dist.get_world_size()
        return 1.0

    def uses_collective(self) -> bool:
        """True when ``step()`` exchanges gradients: ``all_reduce`` under an initialised process group with more than
        one rank (or ``force_collective``)."""
        return bool(self.all_reduce and dist.is_available() and dist.is_initialized()
                    and (dist.get_world_size() > 1 or self.force_collective))

    @torch.no_grad()
    def step(self, closure=None, grad_scale: float = 1.0):
        """``grad_scale``: factor applied to the (all-reduced) gradient inside the update — ``1 / k`` after ``k`` micro-batches
        whose backward passes accumulated into the flat gradient buffer (the reference's production run uses
        ``accumulate_grad_batches: 3``, ``configs/experiment/RandLaNet_base_run_FR.yaml:18``; Lightning divides each
        micro-batch loss by ``k`` instead: the same mean)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        net = self.net
        scale = self.reduce_gradients() * float(grad_scale)
        flat_p, flat_g = net.flat_parameters, net.flat_grads
        if flat_p.data_ptr() != getattr(self, "_bound_ptr", flat_p.data_ptr()):
            raise RuntimeError("FusedAdam: the net was re-flattened after the optimizer was created")
        self._bound_ptr = flat_p.data_ptr()
        g = self.param_groups[0]
        call("m3d_adam_step", flat_p.data_ptr(), flat_g.data_ptr(), self.exp_avg.data_ptr(),
             self.exp_avg_sq.data_ptr(), self._adam_state.data_ptr(),
             None if self.lr_dev is None else self.lr_dev.data_ptr(), float(g["lr"]), float(g["betas"][0]),
             float(g["betas"][1]), float(g["eps"]), float(g["weight_decay"]), scale, 1, flat_p.numel(),
             torch.cuda.current_stream().cuda_stream)
        net.invalidate_eval_cache()  # the weights changed behind the module's back (raw-pointer update)
        return loss

    def zero_grad(self, set_to_none: bool = False):  # gradients are views of the flat buffer: never detach them
        self.net.flat_grads.zero_()


# --------------------------------------------------------------------------------------------------
# many tensors at once
# --------------------------------------------------------------------------------------------------
BLOCK = 256  # elements of a block of the flat moments (every tensor's slice starts at a multiple of it)
GRAD_NORM_PARTS = 2048  # M3D_GRAD_NORM_PARTS


def _dense(t: Tensor) -> bool:
    """Whether the elements of ``t`` fill one run of memory, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda d: (d[1], d[0])):
        if size == 1:
            continue
        if stride != expected:
            return False
        expected *= size
    return True


def _like(g: Tensor, p: Tensor) -> Tensor:
    """``g`` in the memory order of ``p`` (itself where it has that already)."""
    if g.stride() == p.stride() or (g.is_contiguous() and p.is_contiguous()):
        return g
    return torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)


# (one pass over a list of tensors each, without Python code per tensor: a step over small tensors is bound by the host)
_GRAD, _DTYPE, _SPARSE = attrgetter("grad"), attrgetter("dtype"), attrgetter("is_sparse")


def _pointers(tensors: List[Tensor]) -> array:
    return array("Q", list(map(Tensor.data_ptr, tensors)))  # (an array grows element by element from anything but a list)


def _sizes(tensors: List[Tensor]) -> array:
    return array("q", list(map(Tensor.numel, tensors)))


def _types(tensors: List[Tensor], who: str) -> array:
    """M3D_TYPE_* of every tensor."""
    kinds = set(map(_DTYPE, tensors))
    for kind in kinds:
        if kind not in ops.TYPES:
            raise TypeError(f"{who} must be float32, bfloat16 or float16, got {kind}")
    if len(kinds) == 1:
        return array("i", (ops.TYPES[kinds.pop()],)) * len(tensors)
    return array("i", map(ops.TYPES.__getitem__, map(_DTYPE, tensors)))


def _check_strided(tensors: List[Tensor]) -> None:
    """(of tensors that are not all contiguous: a sparse one never says that it is)"""
    if any(map(_SPARSE, tensors)):
        raise RuntimeError("sparse gradients are not supported")


def _check_apart(params: List[Tensor]) -> None:
    """Whether no two of these (dense) parameters share memory: both would be updated at once."""
    spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
    if any(stop > start for (_, stop), (start, _) in zip(spans, spans[1:])):
        raise ValueError("AdamW: two parameters of a group share memory")


def _at(a: array) -> int:
    return a.buffer_info()[0]


@torch.no_grad()
def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float) -> Tensor:
    """``torch.nn.utils.clip_grad_norm_(parameters, max_norm)`` for the 2-norm: scales all gradients in place by
    ``min(1, max_norm / (norm + 1e-6))`` and returns the norm they had together, a 0-dim fp32 tensor on their device (nothing is
    read back).  fp32, bf16 and fp16 gradients, mixed as they come, on one device; parameters without one are left out.  The norm
    is summed in 64 bits in a fixed order: the same gradients give the same bits.  Gradients that are not finite scale as in
    torch (an infinite norm: zeros, NaN for the infinite ones themselves; a NaN norm: NaN).  No two gradients may share memory."""
    params = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm must not be negative, got {max_norm}")
    grads = list(map(_GRAD, params))
    if not all(map(is_not, grads, repeat(None))):
        grads = [g for g in grads if g is not None]
    if not grads:
        return torch.zeros((), dtype=torch.float32, device=params[0].device if params else "cpu")
    types = _types(grads, "clip_grad_norm_: gradients")
    if len(set(map(Tensor.get_device, grads))) > 1:
        raise ValueError("clip_grad_norm_: all gradients must be on one device")
    dense = grads
    if not all(map(Tensor.is_contiguous, grads)):
        _check_strided(grads)
        if any(stride == 0 and size > 1 for g in grads for size, stride in zip(g.shape, g.stride())):
            raise RuntimeError("clip_grad_norm_: a gradient whose elements share memory cannot be scaled in place")
        dense = [g if _dense(g) else g.contiguous() for g in grads]
    ptrs, numel = _pointers(dense), _sizes(dense)
    if len(set(ptrs)) < len(ptrs) and len({g.data_ptr() for g in grads if g.numel()}) < sum(g.numel() > 0 for g in grads):
        raise ValueError("clip_grad_norm_: the same gradient twice")
    dev = grads[0].device
    if dev.type != "cuda":
        raise RuntimeError("clip_grad_norm_ runs on an MI355X only (no CPU fallback by design)")
    parts = torch.empty(GRAD_NORM_PARTS, dtype=torch.float64, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nparts = ctypes.c_int32(0)
    with ops.on_device(dev):
        st = ops._st()
        call("m3d_grad_norm", _at(ptrs), _at(numel), _at(types), len(ptrs), parts.data_ptr(), ctypes.addressof(nparts), st)
        call("m3d_clip_grads", _at(ptrs), _at(numel), _at(types), len(ptrs), parts.data_ptr(), nparts.value, max_norm, norm.data_ptr(), st)
    if dense is not grads:
        for g, d in zip(grads, dense):
            if d is not g:
                g.copy_(d)
    torch.autograd.graph.increment_version(grads)
    return norm


class _Group:
    """What one parameter group of ``AdamW`` keeps: sizes and types of its tensors, its moments (flat, in blocks of 256), counters."""

    def __init__(self, params: List[Tensor], bits: int, dev: torch.device):
        self.params, self.bits = params, bits
        self.numel, self.types = _sizes(params), _types(params, "AdamW: parameters")
        self.strides = [p.stride() for p in params]
        self.plain = all(map(Tensor.is_contiguous, params))
        self.starts, blocks = [], 0
        for p in params:
            self.starts.append(blocks * BLOCK)
            blocks += -(-p.numel() // BLOCK)
        self.blocks = blocks
        self.avg, self.avg_sq = (torch.zeros(blocks * BLOCK, dtype=torch.float32 if bits == 32 else torch.uint8, device=dev) for _ in range(2))
        self.scale = self.scale_sq = None
        if bits == 8:
            self.scale, self.scale_sq = (torch.zeros(blocks, dtype=torch.float32, device=dev) for _ in range(2))
        self.state = torch.zeros(66, dtype=torch.float32, device=dev)  # (M3D_ADAM_STATE_WORDS)
        self.missed = torch.zeros(len(params), dtype=torch.int32, device=dev)
        self.pointers, self.aliases = _pointers(params), [p.detach() for p in params]
        self.args = _lib.M3DAdamW(numel=_at(self.numel), types=_at(self.types), count=len(params), state_bits=bits, exp_avg=self.avg.data_ptr(),
                                  exp_avg_sq=self.avg_sq.data_ptr(), scale_avg=None if bits == 32 else self.scale.data_ptr(),
                                  scale_avg_sq=None if bits == 32 else self.scale_sq.data_ptr(), state=self.state.data_ptr(),
                                  missed=self.missed.data_ptr())

    def slice(self, flat: Tensor, i: int) -> Tensor:
        """Tensor ``i``'s part of a flat buffer, in its shape and memory order."""
        p = self.params[i]
        return flat[self.starts[i]:self.starts[i] + p.numel()].as_strided(p.shape, p.stride(), flat.storage_offset() + self.starts[i])

    def blocks_of(self, scale: Tensor, i: int) -> Tensor:
        a = self.starts[i] // BLOCK
        return scale[a:a + -(-self.params[i].numel() // BLOCK)]

    def decoded(self) -> Tuple[Tensor, Tensor]:
        if self.bits == 32:
            return self.avg, self.avg_sq
        m, v = torch.empty((2, self.blocks * BLOCK), dtype=torch.float32, device=self.avg.device).unbind(0)
        with ops.on_device(self.avg.device):
            call("m3d_moments_decode", self.avg.data_ptr(), self.avg_sq.data_ptr(), self.scale.data_ptr(), self.scale_sq.data_ptr(),
                 m.data_ptr(), v.data_ptr(), self.blocks, ops._st())
        return m, v

    def encode(self, m: Tensor, v: Tensor) -> None:
        with ops.on_device(self.avg.device):
            call("m3d_moments_encode", m.data_ptr(), v.data_ptr(), self.avg.data_ptr(), self.avg_sq.data_ptr(), self.scale.data_ptr(),
                 self.scale_sq.data_ptr(), self.blocks, ops._st())


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` (``amsgrad=False``, ``maximize=False``; with ``weight_decay=0`` also ``torch.optim.Adam``, the
    reference's optimizer) over any parameter tensors on one device: one launch updates up to 152 of them, one more in front of it
    where gradients are clipped.  fp32, bf16 and fp16 parameters, mixed as they come; the update is computed in 32 bits and rounded
    once to the parameter's type.  A parameter without a gradient is left out of a step and keeps its own count, as in torch.

    ``state_bits=8`` holds both moments in a byte an element (with one fp32 scale per 256 elements and moment): 2.03 instead of
    8 bytes an element.  ``exp_avg`` keeps 4 bits of exponent and 3 of fraction of its block's largest magnitude, ``exp_avg_sq`` 5
    and 3, so that an element may be 2^-17 of its block's largest gradient before it is lost; a positive second moment never
    becomes zero.  A value that is not finite is held as NaN, in its own element only.

    ``max_grad_norm``: the gradients of ALL parameters are taken as ``clip_grad_norm_`` would leave them (``p.grad`` itself is
    not written); ``grad_norm`` is then the norm they had, a 0-dim fp32 tensor on the device, which every step writes again
    (``clone()`` it to keep one).  A step whose norm is not finite changes nothing and is not counted.

    ``lr`` may be a 0-dim fp32 tensor on the device (a schedule under graph replay).  Nothing is read back and step counts live on the
    device: ``step()`` may be captured into a hipGraph (after one eager step) and replayed; the gradients must then be written in
    place.  ``state_dict()`` has torch's layout (``step``, ``exp_avg``, ``exp_avg_sq`` per parameter), and with 32 bits states travel
    to and from ``torch.optim.AdamW`` and, without a weight decay of its own kind, ``Adam``; with 8 bits the codes and scales are
    stored, and 32-bit states are taken in too."""

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, max_grad_norm: Optional[float] = None):
        if state_bits not in (32, 8):
            raise ValueError(f"AdamW: state_bits must be 32 or 8, got {state_bits}")
        if max_grad_norm is not None and not float(max_grad_norm) >= 0.0:
            raise ValueError(f"AdamW: max_grad_norm must not be negative, got {max_grad_norm}")
        self.state_bits, self.max_grad_norm = state_bits, None if max_grad_norm is None else float(max_grad_norm)
        self._groups: List[_Group] = []  # (None, until a device is known, for one without parameters)
        self._device = None
        self.grad_norm: Optional[Tensor] = None
        # (the last one is torch's mark of AdamW's decay, by which torch.optim.Adam goes on with that where it loads this state)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled_weight_decay=True))
        if self._device is None:
            raise ValueError("AdamW: no parameters")
        self._groups = [g if g is not None else _Group([], state_bits, self._device) for g in self._groups]
        if self.max_grad_norm is not None:
            self.grad_norm = torch.zeros((), dtype=torch.float32, device=self._device)
            self._parts = torch.empty(GRAD_NORM_PARTS, dtype=torch.float64, device=self._device)

    def _check_group(self, g: dict) -> None:
        lr, (b1, b2), eps, wd, bits = g["lr"], g["betas"], g["eps"], g["weight_decay"], self.state_bits
        if isinstance(lr, Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda or (self._device is not None and lr.device != self._device):
                raise ValueError("AdamW: a tensor lr must be one fp32 element on the parameters' device")
        elif not (float(lr) >= 0.0 and math.isfinite(lr)):
            raise ValueError(f"AdamW: lr must not be negative, got {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {(b1, b2)}")
        if not (eps >= 0.0 and wd >= 0.0):
            raise ValueError(f"AdamW: eps and weight_decay must not be negative, got {eps} and {wd}")
        if bits == 8 and not eps > 0.0:
            raise ValueError("AdamW: state_bits=8 needs eps > 0 (a second moment may be held as zero)")

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            params = group["params"]
            self._check_group(group)
            if len({id(p) for p in params}) < len(params):
                raise ValueError("AdamW: the same parameter twice in a group")
            dev = self._device or (params[0].device if params else None)
            if params and isinstance(group["lr"], Tensor) and group["lr"].device != dev:
                raise ValueError("AdamW: a tensor lr must be one fp32 element on the parameters' device")
            for p in params:
                if p.dtype not in ops.TYPES:
                    raise TypeError(f"AdamW: parameters must be float32, bfloat16 or float16, got {p.dtype}")
                if not _dense(p):
                    raise ValueError(f"AdamW: a parameter's elements must fill one run of memory, got strides {p.stride()} for {tuple(p.shape)}")
                if p.device != dev or p.device.type != "cuda":
                    raise RuntimeError(f"AdamW: all parameters must be on one MI355X (no CPU fallback by design), got {p.device} and {dev}")
            _check_apart(params)
        except Exception:
            self.param_groups.pop()
            raise
        self._device = dev
        self._groups.append(None if dev is None else _Group(list(params), self.state_bits, dev))

    # ------------------------------------------------------------------------------------------
    def _parameters(self, g: _Group) -> array:
        """Pointers of a group's parameters.  The aliases made with the group keep the memory that they were found in alive: where the
        pointers (and the order) are the same, the parameters are where they were; elsewhere everything about them is looked at again."""
        params = g.params
        ptrs = _pointers(params)
        if ptrs != g.pointers or not (all(map(Tensor.is_contiguous, params)) if g.plain else [p.stride() for p in params] == g.strides):
            if (_sizes(params) != g.numel or _types(params, "AdamW: parameters") != g.types or [p.stride() for p in params] != g.strides
                    or {p.get_device() for p in params} != {self._device.index}):
                raise RuntimeError("AdamW: a parameter changed its size, type, order or device after the optimizer was made")
            _check_apart(params)
            g.pointers, g.aliases = ptrs, [p.detach() for p in params]
        return ptrs

    def _gradients(self, g: _Group) -> Tuple[array, List[Tensor]]:
        """Pointers of a group's gradients (0: none), and the tensors that they point to."""
        grads = list(map(_GRAD, g.params))
        there, numel, types = grads, g.numel, g.types
        if not all(map(is_not, grads, repeat(None))):
            there = [x for x in grads if x is not None]
            numel, types = (array(a.typecode, (n for n, x in zip(a, grads) if x is not None)) for a in (numel, types))
        if _sizes(there) != numel or _types(there, "AdamW: gradients") != types or not set(map(Tensor.get_device, there)) <= {self._device.index}:
            raise RuntimeError("AdamW: a gradient must have its parameter's size, type and device")
        if not (g.plain and all(map(Tensor.is_contiguous, there))):
            _check_strided(there)
            grads = [None if x is None else _like(x, p) for x, p in zip(grads, g.params)]
            there = [x for x in grads if x is not None]
        if len(there) == len(grads):
            return _pointers(grads), there
        return array("Q", (0 if x is None else x.data_ptr() for x in grads)), there

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        pointers, keep = [], []
        for g, group in zip(self._groups, self.param_groups):
            self._check_group(group)
            if len(group["params"]) != len(g.params) or not all(map(is_, group["params"], g.params)):
                raise RuntimeError("AdamW: the parameters of a group were exchanged after the optimizer was made")
            params = self._parameters(g)
            ptrs, there = self._gradients(g)
            pointers.append((params, ptrs))
            keep.append(there)
        clip = self.max_grad_norm is not None
        with ops.on_device(self._device):
            st = ops._st()
            nparts = ctypes.c_int32(0)
            if clip:
                numel, types, grads = self._groups[0].numel, self._groups[0].types, pointers[0][1]
                for g, (_, ptrs) in zip(self._groups[1:], pointers[1:]):
                    numel, types, grads = numel + g.numel, types + g.types, grads + ptrs
                call("m3d_grad_norm", _at(grads), _at(numel), _at(types), len(grads), self._parts.data_ptr(), ctypes.addressof(nparts), st)
            for g, group, (params, ptrs), there in zip(self._groups, self.param_groups, pointers, keep):
                if not g.params:
                    continue
                lr, (b1, b2) = group["lr"], group["betas"]
                a = g.args
                a.params, a.grads = _at(params), _at(ptrs)
                if clip:
                    a.parts, a.nparts, a.max_norm, a.norm_out = self._parts.data_ptr(), nparts.value, self.max_grad_norm, self.grad_norm.data_ptr()
                if isinstance(lr, Tensor):
                    a.lr_dev, a.lr = lr.data_ptr(), 0.0
                else:
                    a.lr_dev, a.lr = None, lr
                a.beta1, a.beta2, a.eps, a.weight_decay = b1, b2, group["eps"], group["weight_decay"]
                call("m3d_adamw_step", ctypes.addressof(a), st)
                # (these parameters changed behind torch's back: graphs and caches that go by their version counters notice.  Whether a
                # clipped step was taken only the device knows: its parameters count as changed)
                torch.autograd.graph.increment_version(g.params if len(there) == len(ptrs) else [p for p, x in zip(g.params, ptrs) if x])
        return loss

    # ------------------------------------------------------------------------------------------
    def moments(self) -> List[Tuple[Tensor, Tensor]]:
        """``(exp_avg, exp_avg_sq)`` of every parameter group as flat fp32 buffers: the tensors in order, each from a multiple of 256
        elements on.  With 32 bits the optimizer's own buffers, with 8 bits the values that the codes stand for."""
        return [g.decoded() for g in self._groups]

    def state_dict(self):
        state: Dict[int, dict] = {}
        groups = []
        for g, group in zip(self._groups, self.param_groups):
            steps = (g.state[:1] - g.missed.to(torch.float32)).cpu()
            index = list(range(len(state), len(state) + len(g.params)))
            for i, key in enumerate(index):
                state[key] = {"step": steps[i].clone(), "exp_avg": g.slice(g.avg, i).clone(), "exp_avg_sq": g.slice(g.avg_sq, i).clone()}
                if g.bits == 8:
                    state[key] |= {"exp_avg_scale": g.blocks_of(g.scale, i).clone(), "exp_avg_sq_scale": g.blocks_of(g.scale_sq, i).clone()}
            groups.append({**{k: v for k, v in group.items() if k != "params"}, "params": index})
        return {"state": state, "param_groups": groups}

    @staticmethod
    def _check_entry(p: Tensor, e: dict, coded: bool) -> None:
        keys = {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if coded else set())
        if not keys <= set(e):
            raise ValueError(f"optimizer state lacks {sorted(keys - set(e))}")
        for key in ("exp_avg", "exp_avg_sq"):
            m = e[key]
            if tuple(m.shape) != tuple(p.shape):
                raise ValueError(f"optimizer state has shape {tuple(m.shape)}, expected {tuple(p.shape)}")
            if m.dtype != torch.uint8 if coded else not m.is_floating_point():
                raise ValueError(f"optimizer state {key} has type {m.dtype}, expected {'uint8' if coded else 'a floating-point type'}")
            if coded:
                if not (m.is_contiguous() and p.is_contiguous()) and m.stride() != p.stride():
                    raise ValueError("8-bit states belong to the memory order of the parameter that they were saved from")
                s, blocks = e[key + "_scale"], -(-p.numel() // BLOCK)
                if tuple(s.shape) != (blocks,) or not s.is_floating_point():
                    raise ValueError(f"optimizer state has {s.dtype} scales of shape {tuple(s.shape)}, expected {(blocks,)}")

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        groups, state = state_dict["param_groups"], state_dict["state"]
        if [len(g["params"]) for g in groups] != [len(g.params) for g in self._groups]:
            raise ValueError("loaded state dict has other parameter groups")
        todo = []  # (all of it is looked at before any of it is written)
        for g, group, mine in zip(self._groups, groups, self.param_groups):
            if group.get("amsgrad", False) or group.get("maximize", False):
                raise ValueError("AdamW implements amsgrad=False, maximize=False only")
            if not group.get("decoupled_weight_decay", True) and float(group.get("weight_decay", 0.0)) != 0.0:
                raise ValueError("the state of an optimizer whose weight decay goes through the gradient (Adam's) cannot go on with AdamW's")
            entries = [state.get(key, state.get(str(key))) for key in group["params"]]
            coded = {("exp_avg_scale" in e) for e in entries if e}
            if len(coded) > 1 or (True in coded and g.bits != 8):
                raise ValueError("8-bit states go into an optimizer with state_bits=8 only")
            for p, e in zip(g.params, entries):
                if e:
                    self._check_entry(p, e, True in coded)
            # (everything in the group, as torch does: a scheduler made after this looks for initial_lr)
            values = {k: tuple(map(float, v)) if k == "betas" else float(v) if isinstance(v, Tensor) and v.numel() == 1 else copy.deepcopy(v)
                      for k, v in group.items() if k not in ("params", "decoupled_weight_decay") and not (k == "param_names" and k in mine)}
            self._check_group({**mine, **values})
            todo.append((g, mine, values, entries, True in coded))
        for g, mine, values, entries, coded in todo:
            steps = [float(e["step"]) if e else 0.0 for e in entries]
            top = max(steps, default=0.0)
            if coded or g.bits == 32:
                flat = (g.avg, g.avg_sq)
            else:
                flat = tuple(torch.zeros(g.blocks * BLOCK, dtype=torch.float32, device=g.avg.device) for _ in range(2))
            for f in flat + ((g.scale, g.scale_sq) if coded else ()):
                f.zero_()
            for i, e in enumerate(entries):
                if not e:  # (torch has no entry for a parameter that was never stepped)
                    continue
                for f, key, scale in zip(flat, ("exp_avg", "exp_avg_sq"), (g.scale, g.scale_sq)):
                    g.slice(f, i).copy_(e[key])
                    if coded:
                        g.blocks_of(scale, i).copy_(e[key + "_scale"])
            if g.bits == 8 and not coded:
                g.encode(*flat)
            g.state.zero_()
            g.state[0] = top
            g.missed.copy_(torch.tensor([int(top - s) for s in steps], dtype=torch.int32))
            for k, v in values.items():
                if k == "lr" and isinstance(mine["lr"], Tensor):
                    mine["lr"].fill_(v)  # (the place that a captured step reads)
                else:
                    mine[k] = v

    def __getstate__(self):
        raise TypeError("AdamW cannot be copied or pickled: make another one and load state_dict()")

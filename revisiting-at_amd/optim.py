"""AdamW over all parameters in two launches, with moments in 32 or in 8 bits (``csrc/optim_kernels.hip``).

The reference steps ``torch.optim.AdamW`` (``main.py:395-459, 993``); ``train_step.create_optimizer`` builds that by default and
``FusedAdamW`` for ``state_bits=32 | 8``.  Per fp32 parameter a step moves 28 bytes with 32-bit moments and 16 with 8-bit ones, which also
keep 2 bytes instead of 8 in memory."""
from __future__ import annotations

import ctypes
import warnings

import numpy as np
import torch

from . import _lib, ops

__all__ = ["FusedAdamW"]

BLOCK, CHUNK, MAX_TENSORS, MAX_GROUPS = 256, 4096, 440, 8          # CNX_ADAMW_* of include/convnext_hip.h
SMALL = 4096                                                       # tensors with fewer elements keep 32-bit moments (norms, biases)

_TENSOR = np.dtype([("param", np.int64), ("numel", np.int64), ("state", np.int64), ("bits", np.int32), ("dtype", np.int32), ("group", np.int32),
                    ("step", np.int32)])                           # cnx_adamw_tensor
_CHUNK = np.dtype([("tensor", np.int32), ("part", np.int32)])      # cnx_adamw_chunk
_KEYS = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg_codes", "exp_avg_scales", "exp_avg_sq_codes", "exp_avg_sq_scales")}


def _dense(p):
    """Elements of ``p`` fill its memory, each once (any order of the dimensions: channels-last weights)."""
    need = 1
    for size, stride in sorted(((n, s) for n, s in zip(p.shape, p.stride()) if n > 1), key=lambda v: v[1]):
        if stride != need:
            return False
        need *= size
    return True


def _order(p):
    """Dimensions of more than one element, from the slowest to the fastest; empty where that is their own order."""
    dims = sorted((d for d, n in enumerate(p.shape) if n > 1), key=lambda d: -p.stride(d))
    return () if dims == sorted(dims) else tuple(dims)


# 8-bit moments outside the kernel (csrc/optim_kernels.hip): mantissa bits, code of 1.0, sign bit
_CODES = {"exp_avg": (3, 127, 128), "exp_avg_sq": (4, 255, 0)}


def _decode(codes, scales, kind):
    """The numbers that 8-bit moments stand for (of the second moment: its root)."""
    mant, top, sign = _CODES[kind]
    c = codes.to(torch.int32)
    x = ((c & top) + ((0x3f800000 >> (23 - mant)) - top) << (23 - mant)).view(torch.float32)
    x = torch.where(c & top > 0, x, 0.0)
    return (torch.where(c & sign > 0, -x, x).view(-1, BLOCK) * scales.unsqueeze(1)).view(-1)


def _encode(x, kind):
    """(codes, scales) of whole blocks of numbers, rounded as the kernel does."""
    mant, top, sign = _CODES[kind]
    shift = 23 - mant
    scales = x.view(torch.int32).bitwise_and(0x7fffffff).view(-1, BLOCK).amax(1).view(torch.float32)       # (patterns: a NaN is the largest)
    scales = torch.where(scales < torch.finfo(torch.float32).tiny, 0.0, scales)
    inv = torch.where(scales > 0, 1 / scales, 0.0).unsqueeze(1)
    b = (x.abs().view(-1, BLOCK) * inv).view(-1).view(torch.int32) & 0x7fffffff
    c = ((b + ((1 << (shift - 1)) - 1) + ((b >> shift) & 1) >> shift) - ((0x3f800000 >> shift) - top)).clamp_(0, top)
    if sign:
        c |= torch.where(x < 0, sign, 0).to(torch.int32)
    else:
        some = (x.view(-1, BLOCK) > 0) & (scales > 0).unsqueeze(1)
        c = torch.where(some.view(-1) & (c == 0), 1, c)
    return c.to(torch.uint8), scales


def _reorder(state, p):
    """The four 8-bit tensors of a state for the memory order of ``p``: where it was another one, blocks get other members, and the numbers are
    rounded again to the new blocks' scales."""
    old = state.get("exp_avg_order")
    old = _order(p) if old is None else tuple(torch.as_tensor(old).tolist())
    if old == _order(p):
        return state
    dims = old or tuple(d for d, n in enumerate(p.shape) if n > 1)
    strides, step = [0] * p.dim(), 1
    for d in reversed(dims):
        strides[d] = step
        step *= p.shape[d]
    n, out = p.numel(), dict(state)
    for kind in _CODES:
        codes, scales = (torch.as_tensor(state[f"{kind}_{k}"]) for k in ("codes", "scales"))
        was = _decode(codes, scales, kind)
        now = torch.zeros_like(was)
        now.as_strided(p.shape, p.stride()).copy_(was[:n].as_strided(p.shape, strides))
        out[f"{kind}_codes"], out[f"{kind}_scales"] = _encode(now, kind)
    return out


def _copy(pairs):
    """``dst.copy_(src)`` of each pair, those of one type and device together."""
    groups = {}
    for dst, src in pairs:
        src = torch.as_tensor(src)
        dsts, srcs = groups.setdefault((dst.dtype, src.dtype, src.device), ([], []))
        dsts.append(dst)
        srcs.append(src)
    for dsts, srcs in groups.values():
        torch._foreach_copy_(dsts, srcs)


class _Plan:
    """What does not change between steps: the moments' buffers, the device tables of tensors and chunks."""

    def __init__(self, params, groups, bits):
        dev = params[0].device
        self.layout = ops._host().Layout(params)
        self.groups = groups                                       # of each parameter
        self.grads = (ctypes.c_void_p * len(params))()
        self.bits = bits
        self.at, size = [], {32: 0, 8: 0}
        for p, b in zip(params, self.bits):
            self.at.append(size[b])
            size[b] += -(-p.numel() // BLOCK) * BLOCK
        self.size = size
        zeros = lambda n, dt: torch.zeros(n, device=dev, dtype=dt) if n else None                       # noqa: E731
        self.m, self.v = zeros(size[32], torch.float32), zeros(size[32], torch.float32)
        self.mc, self.vc = zeros(size[8], torch.uint8), zeros(size[8], torch.uint8)
        self.ms, self.vs = zeros(size[8] // BLOCK, torch.float32), zeros(size[8] // BLOCK, torch.float32)
        self.steps = torch.zeros(len(params), device=dev, dtype=torch.float32)
        self.coef = torch.empty(8 * len(params), device=dev, dtype=torch.float32)
        self.runs = []                                             # (first tensor, tensors, table, chunks)
        for first in range(0, len(params), MAX_TENSORS):
            rows, chunks = [], []
            for i in range(first, min(first + MAX_TENSORS, len(params))):
                p = params[i]
                rows.append((p.data_ptr(), p.numel(), self.at[i], self.bits[i], _lib.dtype_code(p.dtype), groups[i], i))
                part = np.arange(-(-p.numel() // CHUNK), dtype=np.int32)
                chunks.append(np.stack((np.full_like(part, i - first), part), 1))
            table = torch.from_numpy(np.array(rows, dtype=_TENSOR).view(np.uint8).copy()).to(dev)
            chunks = torch.from_numpy(np.concatenate(chunks)).to(dev)
            self.runs.append((first, len(rows), table, chunks))

    def moments(self, i, p):
        """Views of one tensor's moments, by the names they have in a state dict."""
        a, e = self.at[i], self.at[i] + -(-p.numel() // BLOCK) * BLOCK
        if self.bits[i] == 32:
            return {k: t.as_strided(p.shape, p.stride(), a) for k, t in zip(_KEYS[32], (self.m, self.v))}
        return {**dict(zip(_KEYS[8], (self.mc[a:e], self.ms[a // BLOCK:e // BLOCK], self.vc[a:e], self.vs[a // BLOCK:e // BLOCK]))),
                "exp_avg_order": torch.tensor(_order(p), dtype=torch.int64)}


class FusedAdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` (decoupled weight decay, bias correction) for fp32 or bf16 parameters on one device: one prepared launch updates
    them all (at most 8 parameter groups).  ``state_bits=8`` keeps the moments of tensors with 4096 or more elements in a byte each (a
    scale for every 256 elements; the second moment as its root), the others in 32 bits.  Codes are rounded to nearest up to betas of 31/32 (a
    moment then follows its gradients because they vary, to about 8 % of a root at 0.95) and, above, up or down by a hash of element and step
    (about 20 % at 0.999): a step of a moment is less than half a step of its code there.

    Step counters live on the device and ``lr`` may be a device tensor, so a step can be captured into a hipGraph after one eager step (or
    ``load_state_dict``) has built the tables.  ``load_state_dict`` writes into the buffers, counters and device learning rates that are there, so
    a captured step goes on from what was loaded; a parameter that moves, changes its type or joins needs new tables, and with them a new capture.
    Parameters without a gradient are left alone.  ``state_dict`` has torch's layout: ``step`` and
    ``exp_avg`` / ``exp_avg_sq`` (torch's AdamW loads and is loaded), or ``exp_avg_codes``, ``exp_avg_scales``, ``exp_avg_sq_codes``,
    ``exp_avg_sq_scales`` where the moments have 8 bits; those lie in the memory order of their parameter, which ``exp_avg_order`` tells (a state
    without it is taken to be in the present one), and are brought into another order's blocks when that changes.  ``moments()`` gives all moments as numbers.  The optimizer steps on the stream that
    is current; its buffers belong to one stream at a time, as the parameters do."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        if state_bits not in (32, 8):
            raise ValueError(f"FusedAdamW: state_bits={state_bits!r} is not 32 or 8")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"FusedAdamW: lr={lr!r}")
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"FusedAdamW: betas={betas!r}, eps={eps!r}, weight_decay={weight_decay!r}")
        self.state_bits, self._plan, self._captured = state_bits, None, []
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def add_param_group(self, group):
        super().add_param_group(group)
        if len(self.param_groups) > MAX_GROUPS:
            self.param_groups.pop()
            raise ValueError(f"FusedAdamW: more than {MAX_GROUPS} parameter groups")
        self._stale = True

    def _bits(self, p):
        return 8 if self.state_bits == 8 and p.numel() >= SMALL else 32

    def _shapes(self, p):
        """Names and shapes of a parameter's moments."""
        bits, blocks = self._bits(p), -(-p.numel() // BLOCK)
        return dict(zip(_KEYS[bits], [tuple(p.shape)] * 2 if bits == 32 else [(blocks * BLOCK,), (blocks,)] * 2))

    def _params(self):
        return [p for g in self.param_groups for p in g["params"]]

    def _groups(self):
        return [i for i, g in enumerate(self.param_groups) for _ in g["params"]]

    def _build(self):
        """Tables and buffers for the parameters as they are now; moments that exist are kept."""
        params = self._params()
        if not params:
            raise ValueError("FusedAdamW: no parameters")
        for p in params:
            if not p.is_cuda:
                raise _lib.ApgdHipError("FusedAdamW needs device parameters (no CPU path in the product)")
            if p.device != params[0].device:
                raise ValueError(f"FusedAdamW: parameters on {params[0].device} and {p.device}")
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError(f"FusedAdamW: no kernel for {p.dtype} parameters")
            if not _dense(p):
                raise ValueError(f"FusedAdamW: a parameter with strides {p.stride()} for {tuple(p.shape)} does not fill its memory")
            if p.numel() > CHUNK * (1 << 22):
                raise ValueError(f"FusedAdamW: a parameter of {p.numel()} elements")
        spans = sorted((p.data_ptr(), p.numel() * p.element_size()) for p in params if p.numel())
        if any(a + n > b for (a, n), (b, _) in zip(spans, spans[1:])):
            raise ValueError("FusedAdamW: two parameters share memory")                        # (their updates would race)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: the first step (and one after parameters were moved or added) has to run outside a graph capture")
        old = {p: dict(self.state[p]) for p in params if self.state.get(p)}
        for i, p in enumerate(params):                             # (before anything is changed)
            for k, shape in self._shapes(p).items() if p in old else ():
                if k not in old[p] or tuple(old[p][k].shape) != shape:
                    raise RuntimeError(f"FusedAdamW: the moments of parameter {i} do not go with its shape {tuple(p.shape)}")
        with ops._on_device(params[0]), torch.no_grad():
            plan = _Plan(params, self._groups(), [self._bits(p) for p in params])
            self._adopt(plan, params)
            old = {p: _reorder(s, p) if "exp_avg_codes" in s else s for p, s in old.items()}
            _copy([(t, old[p][k]) for p in params if p in old for k, t in self.state[p].items() if k != "exp_avg_order"])
        return plan

    def _adopt(self, plan, params):
        for i, (p, step) in enumerate(zip(params, plan.steps.unbind())):
            self.state[p] = {"step": step, **plan.moments(i, p)}
        self._plan, self._stale = plan, False

    def _ready(self, params):
        plan = self._plan
        if plan is None or self._stale or plan.groups != self._groups() or not plan.layout.matches(params) or params[0] not in self.state:
            plan = self._build()
        return plan

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        params = self._params()
        plan = self._ready(params)
        if torch.cuda.is_current_stream_capturing() and plan not in self._captured:
            self._captured.append(plan)                            # replays write into its buffers, also after tables have been built anew
        kept = plan.layout.gradients(params, ctypes.addressof(plan.grads))                     # copies that live until the launch
        n = len(self.param_groups)
        hyper, lr_dev = (ctypes.c_double * (5 * n))(), (ctypes.c_void_p * n)()
        for i, g in enumerate(self.param_groups):
            lr = g["lr"]
            if isinstance(lr, torch.Tensor):
                if lr.is_cuda:
                    if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != params[0].device:
                        raise ValueError("FusedAdamW: a learning rate in device memory has to be one float32 on the parameters' device")
                    lr_dev[i] = lr.data_ptr()
                lr = 0.0 if lr.is_cuda else float(lr)
            hyper[5 * i:5 * i + 5] = (lr, g["betas"][0], g["betas"][1], g["eps"], g["weight_decay"])
        if not any(plan.size.values()):                            # only empty parameters
            return loss
        lib = _lib.load()
        with ops._on_device(params[0]):
            for first, count, table, chunks in plan.runs:
                _lib.check(lib.cnx_adamw_step(table.data_ptr(), chunks.data_ptr(), chunks.shape[0], ctypes.byref(plan.grads, 8 * first), count,
                                              hyper, lr_dev, n, plan.steps.data_ptr(), plan.coef.data_ptr() + 32 * first, _lib.ptr(plan.m),
                                              _lib.ptr(plan.v), _lib.ptr(plan.mc), _lib.ptr(plan.ms), _lib.ptr(plan.vc), _lib.ptr(plan.vs),
                                              ops._stream()), "cnx_adamw_step")
        del kept
        return loss

    @torch.no_grad()
    def moments(self):
        """``{32: (exp_avg, exp_avg_sq)}`` and / or ``{8: ...}``: the moments as numbers, flat, the tensors of each width in the order of the
        groups, each padded with zeros to a multiple of 256 elements.  32 bits: the buffers themselves; 8 bits: bfloat16 copies (a code has
        4 or 5 significant bits)."""
        plan = self._ready(self._params())
        out = {}
        if plan.m is not None:
            out[32] = plan.m, plan.v
        if plan.mc is not None:
            n = plan.mc.numel()
            m, v = (torch.empty(n, device=plan.mc.device, dtype=torch.bfloat16) for _ in range(2))
            with ops._on_device(m):
                _lib.check(_lib.load().cnx_adamw_values(plan.mc.data_ptr(), plan.ms.data_ptr(), plan.vc.data_ptr(), plan.vs.data_ptr(), m.data_ptr(),
                                                        v.data_ptr(), n, ops._stream()), "cnx_adamw_values")
            out[8] = m, v
        return out

    def state_dict(self):
        if self._plan is not None:
            self._ready(self._params())
        return super().state_dict()

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """A state dict of this class, or (32-bit moments) of ``torch.optim.AdamW``; moments of another width are refused, before anything is
        changed."""
        params, ids = self._params(), [i for g in state_dict["param_groups"] for i in g["params"]]
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("FusedAdamW: no amsgrad, no maximize")
        for i, (p, at) in enumerate(zip(params, ids)):
            given = state_dict["state"].get(at)
            if given is None:                                                                  # never stepped
                continue
            bits, shapes = self._bits(p), self._shapes(p)
            if {"step", *shapes} - set(given):
                raise ValueError(f"FusedAdamW: the state of parameter {i} lacks {sorted({'step', *shapes} - set(given))} (state_bits="
                                 f"{self.state_bits} keeps its moments in {bits} bits)")
            for k, shape in shapes.items():
                if tuple(given[k].shape) != shape:
                    raise ValueError(f"FusedAdamW: {k} of parameter {i} is {tuple(given[k].shape)}, not {shape}")
            if bits == 8 and "exp_avg_order" not in given:
                if sum(n > 1 for n in p.shape) > 2:                                            # (memory formats)
                    warnings.warn(f"FusedAdamW: the 8-bit state of parameter {i} does not tell its memory order; it is taken to be the parameter's")
            elif bits == 8:
                order = torch.as_tensor(given["exp_avg_order"]).tolist()
                if order and sorted(order) != [d for d, n in enumerate(p.shape) if n > 1]:
                    raise ValueError(f"FusedAdamW: exp_avg_order of parameter {i} is {order} for {tuple(p.shape)}")
        plan = None if self._plan is None or self._stale or self._plan.groups != self._groups() or not self._plan.layout.matches(params) else self._plan
        if plan is not None and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: load_state_dict has to run outside a graph capture")
        rates = [g["lr"] for g in self.param_groups]
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})     # checks and takes the groups
        for g, lr in zip(self.param_groups, rates):
            if isinstance(lr, torch.Tensor) and lr.is_cuda:                                    # (a captured step reads this one)
                g["lr"] = lr.copy_(torch.as_tensor(g["lr"]).reshape(lr.shape))
        if plan is None:
            self._build()
        else:
            self._adopt(plan, params)
        mine = {t.untyped_storage().data_ptr() for s in self.state.values() for t in s.values()}
        pairs, never = [], []
        for p, at in zip(params, ids):
            given = state_dict["state"].get(at) or {}
            if "exp_avg_codes" in given:
                given = _reorder(given, p)
            for k, t in self.state[p].items():
                if k == "exp_avg_order":
                    continue
                if k in given:
                    x = torch.as_tensor(given[k])
                    pairs.append((t, x.clone() if x.untyped_storage().data_ptr() in mine else x))
                else:
                    never.append(t)
        with ops._on_device(params[0]):
            _copy(pairs)
            if never:
                torch._foreach_zero_(never)

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plan, self._stale = None, True
        self.__dict__.setdefault("_captured", [])

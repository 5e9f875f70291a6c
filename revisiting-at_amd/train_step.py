"""Outer adversarial-training step (``/root/reference/main.py:961-997``) and its DDP wiring
(``main.py:351-359, 889-890``): per-iteration LR, ``zero_grad(set_to_none)``, autocast forward
through ``WrappedModel`` (attack inside), loss, backward (RCCL gradient all-reduce fired by DDP's
hooks — the only collective of the path), AdamW step, EMA update.

Differences from the reference, all MI355X-motivated (SURVEY.md §7 "hard parts"):
  * bf16 autocast, no GradScaler (the reference uses fp16 + GradScaler, ``main.py:797, 992-994``);
  * the EMA copy lives on the device and is updated with one multi-tensor lerp instead of a
    per-step device->host copy of every parameter (``main.py:885, 996-997``).
"""
from __future__ import annotations

import math
import os
from typing import Optional

import numpy as np
import torch
import torch.nn as nn

from . import graphed, ops
from .config import AdvConfig, wrap_model_for_at
from .optim import FusedAdamW


def get_cosine_lr(epoch, lr, epochs, lr_peak_epoch):
    """Linear warm-up to ``lr`` then cosine to 5e-6 (``main.py:227-243``)."""
    if epoch <= lr_peak_epoch:
        return float(np.interp([epoch], [0, lr_peak_epoch], [1e-4 * lr, lr])[0])
    lr_min = 5e-6
    return lr_min + .5 * (lr - lr_min) * (1 + math.cos(math.pi * (epoch - lr_peak_epoch) / (epochs - lr_peak_epoch)))


def iteration_lrs(epoch, iters, **kw):
    """Per-iteration LR table of one epoch (``main.py:956-958``)."""
    return np.interp(np.arange(iters), [0, iters], [get_cosine_lr(epoch, **kw), get_cosine_lr(epoch + 1, **kw)])


def create_optimizer(model: nn.Module, arch: str, weight_decay: float = 0.05, capturable: bool = False, state_bits: Optional[int] = None):
    """AdamW(betas=(0.9, 0.95)) with the reference's two parameter groups (``main.py:395-459``):
    for convnext/resnet archs the names containing ``bn`` or ``.bias`` are not decayed (LayerNorm
    weights and gammas ARE); otherwise 1-D parameters and biases are not decayed.

    ``capturable``: step counters and the learning rate are device tensors, so the update can be part of a hipGraph
    (``ATTrainStep(graph_train=True)``); the arithmetic is the same.

    ``state_bits``: 32 or 8 - ``optim.FusedAdamW`` with moments of that many bits instead of torch's AdamW (None)."""
    named = [(k, v) for k, v in model.named_parameters() if v.requires_grad]
    if 'convnext' in arch or 'resnet' in arch:
        excluded = ['bn', '.bias']
        no_decay = [v for k, v in named if any(c in k for c in excluded)]
        decay = [v for k, v in named if not any(c in k for c in excluded)]
    else:
        no_decay = [v for k, v in named if v.ndim <= 1 or k.endswith('.bias')]
        decay = [v for k, v in named if not (v.ndim <= 1 or k.endswith('.bias'))]
    groups = [{'params': no_decay, 'weight_decay': 0.}, {'params': decay, 'weight_decay': weight_decay}]
    dev = decay[0].device
    if state_bits is not None:
        return FusedAdamW(groups, lr=torch.tensor(1e-3, dtype=torch.float32, device=dev) if capturable else 1e-3, betas=(0.9, 0.95),
                          state_bits=state_bits)
    if capturable:
        return torch.optim.AdamW(groups, lr=torch.tensor(1e-3, dtype=torch.float32, device=dev), betas=(0.9, 0.95), fused=True,
                                 capturable=True)
    return torch.optim.AdamW(groups, betas=(0.9, 0.95), fused=decay[0].is_cuda)


class DeviceEma:
    """``ModelEmaV2(decay)`` semantics (``ema = decay*ema + (1-decay)*model`` over the whole state dict,
    ``main.py:882-887, 996-997``) kept on the device and updated by one multi-tensor lerp.

    The copy keeps the model's state-dict keys (``base_model.*`` under ``WrappedModel``), which is what the
    reference saves as ``weights_ema_{epoch}.pt`` / ``state_dict_ema`` via ``get_state_dict(model_ema)``
    (``main.py:739-747``).  Non-floating entries (none in the LayerNorm models of this path, but e.g.
    ``num_batches_tracked`` elsewhere) are copied verbatim at every update."""

    def __init__(self, model: nn.Module, decay: float = 0.9999):
        self.decay = decay
        sd = model.state_dict()
        self.keys = list(sd.keys())
        self._model_sd = sd                                   # live views of the parameters / buffers
        self._ema_sd = {k: v.detach().clone() for k, v in sd.items()}
        self._fkeys = [k for k in self.keys if sd[k].is_floating_point()]
        self._ikeys = [k for k in self.keys if not sd[k].is_floating_point()]
        self.src = [sd[k] for k in self._fkeys]
        self.ema = [self._ema_sd[k] for k in self._fkeys]

    @torch.no_grad()
    def update(self):
        torch._foreach_lerp_(self.ema, [s.detach() for s in self.src], 1.0 - self.decay)
        for k in self._ikeys:
            self._ema_sd[k].copy_(self._model_sd[k])

    def state_dict(self):
        """``{key: ema tensor}`` with the wrapped model's own keys (timm ``get_state_dict(model_ema)``)."""
        return {k: self._ema_sd[k] for k in self.keys}

    @torch.no_grad()
    def load_state_dict(self, sd, strict: bool = True):
        missing = [k for k in self.keys if k not in sd]
        extra = [k for k in sd if k not in self._ema_sd]
        if strict and (missing or extra):
            raise KeyError(f"EMA state dict mismatch: missing {missing[:4]}, unexpected {extra[:4]}")
        for k in self.keys:
            if k in sd:
                self._ema_sd[k].copy_(sd[k])


def setup_distributed():
    """One process per GPU, RCCL via the "nccl" backend (``main.py:351-356``); reads the torchrun env."""
    import torch.distributed as dist
    # dmabuf IPC (the only mode the host driver of this pool supports): must be in the environment before the HIP runtime
    # starts in this process, or RCCL's buffer exchange fails with hipIpcGetMemHandle: invalid argument
    os.environ.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    if world > 1 and not dist.is_initialized():
        # RCCL ("nccl") on GPUs; APGD_DIST_BACKEND=gloo lets the same wiring be exercised with several ranks on ONE GPU
        # (RCCL refuses two ranks per device), which is how the 1-GPU test box covers DDP + the hand-written backward
        backend = os.environ.get("APGD_DIST_BACKEND") or ("nccl" if torch.cuda.is_available() else "gloo")
        if torch.cuda.is_available():
            local = local % max(1, torch.cuda.device_count())
            torch.cuda.set_device(local)
        dist.init_process_group(backend, rank=rank, world_size=world)
    return rank, local, world


class FlatGradSync:
    """The gradient exchange of the outer step (``main.py:889-890, 992``: DDP's bucketed all-reduce of the parameter gradients) without
    autograd hooks, so that the training pass of a rank can be replayed from hipGraphs like the single-GPU one.

    DDP fires its bucket reductions from hooks inside ``loss.backward()``; RCCL calls cannot sit inside a stream capture on this pool,
    which round 3 answered by leaving every N > 1 rank on the eager pass (~350 Python launches, 30 - 40 ms of host per step, eight
    ranks on one host).  Here the parameter gradients live in TWO flat fp32 buffers - ``late``: the parameters behind the model's
    cut point (ConvNeXt-T: stages 2, 3 and the head = 95 % of the bytes, whose gradients are complete after ~45 % of the backward),
    ``early``: the rest - every ``p.grad`` is a view into them, and the backward runs in two ``torch.autograd.grad`` calls split at the
    cut activation.  The training pass becomes three graph segments with the collectives issued eagerly BETWEEN them:

        [forward, loss, backward down to the cut]  -> all-reduce(late), asynchronous: runs on RCCL's stream under ...
        [... the backward of the early stages]     -> all-reduce(early); wait for both
        [AdamW, EMA]

    One exchange per step and rank, 4 bytes per parameter, none inside the attack - the traffic ``north_star`` / SURVEY.md section
    8e prescribe; the mean over ranks is RCCL's ``AVG`` (gloo: ``SUM`` then a division).  With one rank (or no process group) the
    reductions are no-ops and the same code is the single-GPU step."""

    def __init__(self, module: nn.Module, device):
        import torch.distributed as dist
        self.world = dist.get_world_size() if (dist.is_available() and dist.is_initialized()) else 1
        self.backend = dist.get_backend() if self.world > 1 else None
        params = [p for p in module.parameters() if p.requires_grad]
        cut, late_mods = None, []
        for m in module.modules():
            if hasattr(m, "ddp_cut"):
                cut, late_mods = m.ddp_cut()
                break
        late_ids = {id(p) for lm in late_mods for p in lm.parameters()}
        self.cut = cut if late_ids else None
        self.late = [p for p in params if id(p) in late_ids]
        self.early = [p for p in params if id(p) not in late_ids]
        self.flat, self.views = [], []
        for group in (self.late, self.early):
            n = sum(p.numel() for p in group)
            buf = torch.zeros(n, device=device, dtype=torch.float32)
            vs, o = [], 0
            for p in group:
                # the parameter's own layout (channels_last convolution weights): the fused AdamW wants params and grads alike
                dense = p.numel() > 0 and sum((sz - 1) * st for sz, st in zip(p.shape, p.stride())) + 1 == p.numel()
                vs.append(buf[o:o + p.numel()].as_strided(p.shape, p.stride()) if dense else buf[o:o + p.numel()].view(p.shape))
                o += p.numel()
            self.flat.append(buf)
            self.views.append(vs)
        for group, vs in zip((self.late, self.early), self.views):
            for p, v in zip(group, vs):
                if p.dtype != torch.float32:
                    raise TypeError("FlatGradSync keeps fp32 gradients (the path's parameters are fp32, main.py:797)")
                p.grad = v                                                 # for the optimizer; never set to None again
        self._works = []
        self.verified = self.cut is None                                   # split backward checked against the whole one (check_split)
        self.reduces = 0                                                   # collectives issued (tests, bench)
        self.bytes_per_step = 4 * sum(b.numel() for b in self.flat)

    @torch.no_grad()
    def broadcast_parameters(self, module: nn.Module):
        """Rank 0's parameters and buffers to every rank, once (what DDP's constructor does, ``main.py:889-890``)."""
        if self.world > 1:
            import torch.distributed as dist
            for t in list(module.parameters()) + list(module.buffers()):
                dist.broadcast(t.data, 0)

    @torch.no_grad()
    def store(self, which: int, grads):
        """Gradients of one group (``torch.autograd.grad`` output, None for an unused parameter) into its flat buffer."""
        vs = self.views[which]
        have = [(v, g) for v, g in zip(vs, grads) if g is not None]
        # torch._foreach_copy_ runs ONE multi-tensor kernel only if every pair qualifies (same dtype, same strides, dense); a single
        # odd pair (a permuted convolution-weight gradient) sends the whole list down the per-tensor path: 169 copy launches, 0.6 ms
        # per step on the headline model.  The qualifying pairs go together, the others one by one.
        fast = [(v, g) for v, g in have if g.dtype == v.dtype and g.stride() == v.stride() and g.shape == v.shape]
        slow = [(v, g) for v, g in have if not (g.dtype == v.dtype and g.stride() == v.stride() and g.shape == v.shape)]
        if fast:
            torch._foreach_copy_([v for v, _ in fast], [g for _, g in fast])
        for v, g in slow:
            v.copy_(g)
        for v, g in zip(vs, grads):
            if g is None:
                v.zero_()

    def check_split(self, loss, h):
        """First eager pass with a cut point: the two-call backward must reach every parameter the whole backward reaches.  A
        trainable parameter that lies downstream of the cut but is not listed in the model's late modules (or is shared across the
        cut) gets ``None`` from ``autograd.grad([h], early)`` and ``store`` would zero-fill it on every step without a sound - so the
        used-sets are compared once (one extra backward, graph retained); on a mismatch the cut is dropped with a warning and the
        exchange runs behind ONE whole backward (same gradients as ``loss.backward()``, no overlap of the first all-reduce)."""
        full = torch.autograd.grad([loss], self.late + self.early, allow_unused=True, retain_graph=True)
        g1 = torch.autograd.grad([loss], self.late + [h], allow_unused=True, retain_graph=True)
        dev = self.flat[0].device
        n_short = torch.zeros((), device=dev)
        if g1[-1] is None:
            # the cut activation is not on the loss path at all: every early parameter the whole backward reaches would be lost
            lost = [i for i, a in enumerate(full) if a is not None and (i >= len(self.late) or g1[i] is None)]
        else:
            g2 = torch.autograd.grad([h], self.early, grad_outputs=[g1[-1]], allow_unused=True, retain_graph=True)
            split = list(g1[:-1]) + list(g2)
            lost = [i for i, (a, b) in enumerate(zip(full, split)) if a is not None and b is None]
            both = [(a.float(), b.float()) for a, b in zip(full, split) if a is not None and b is not None]
            if both:
                # ONE device-side verdict (no host round trip per parameter): 5 % in norm - far above the run-to-run noise of the
                # library's split-K filter gradients
                ref = torch.stack(torch._foreach_norm([a for a, _ in both]))
                dif = torch.stack(torch._foreach_norm(torch._foreach_sub([a for a, _ in both], [b for _, b in both])))
                n_short = (dif > 0.05 * ref + 1e-12).sum().to(torch.float32)
        verdict = torch.stack([torch.tensor(float(len(lost)), device=dev), n_short.to(dev)])
        if self.world > 1:
            # the ranks decide TOGETHER (MAX over ranks): a data-dependent verdict of one rank's own batch must not leave the ranks
            # with different graph segmentations
            import torch.distributed as dist
            dist.all_reduce(verdict, op=dist.ReduceOp.MAX)
        n_lost, n_bad = (int(v) for v in verdict.tolist())
        self.verified = True
        if n_lost or n_bad:
            import warnings
            warnings.warn(f"FlatGradSync: the model's ddp_cut() does not partition its parameters ({n_lost} parameters would lose "
                          f"their gradient, {n_bad} would get a part of it; maximum over the ranks): cut point dropped, one whole "
                          "backward per step")
            self.cut = None

    def start_reduce(self, which: int):
        if self.world > 1 and self.flat[which].numel():
            import torch.distributed as dist
            op = dist.ReduceOp.AVG if self.backend == "nccl" else dist.ReduceOp.SUM
            self._works.append((dist.all_reduce(self.flat[which], op=op, async_op=True), which))
            self.reduces += 1

    def wait(self):
        for w, which in self._works:
            w.wait()
            if self.backend != "nccl":
                self.flat[which].div_(self.world)
        self._works = []


class _TrainPassGraph:
    """The training pass of one step - forward of the adversarial batch, loss, backward, AdamW, EMA (``main.py:985-997``) -
    captured once as hipGraph segments and replayed: ~350 kernel launches through Python autograd functions become one graph
    launch (three with the gradient exchange of ``FlatGradSync`` issued eagerly between them).  Same capture rules as
    ``graphed._Program``: parameters are read and written in place, derived weight copies are rebuilt inside the graph."""

    def __init__(self, step: "ATTrainStep", x, target, x_is_static: bool = False, attack_prog=None):
        # x_is_static: x is the static output of the attack's own graph (graphed.borrow_outputs) - the same tensor at every
        # step, read in place; anything else is copied into a buffer of this graph
        self.x = x if x_is_static else torch.empty_like(x)
        self.t = torch.empty_like(target)
        if not x_is_static:
            self.x.copy_(x)
        self.t.copy_(target)
        # attack_prog: the attack program whose replay ran in front of this capture and will run in front of every replay of this
        # graph (ATTrainStep._graph_step checks it): its derived weight copies - packed / bf16 weights, rebuilt by each of its replays
        # from the parameters the optimizer last wrote, unchanged until this graph's own optimizer step - are READ here instead of
        # being rebuilt (~75 five-microsecond kernels per step).  Entries keep their tensors (the attack graph's pool memory) alive;
        # segment -1: complete by stream order, never waited for (ops._cached).
        self.attack_prog = attack_prog
        self.derived = {} if attack_prog is None else {k: (v[0], v[1], None, None, -1) for k, v in attack_prog.derived.items()}
        self.shared_derived = len(self.derived)
        rec = graphed._Recorder()
        if step.sync is None:
            step.optimizer.zero_grad(set_to_none=True)         # the captured backward allocates every .grad in the graph's pool
        if rec.mode != "global":
            torch.cuda.synchronize()                           # nothing left for a communicator's watchdog thread to poll
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        prev = ops._CAPTURE_CACHE
        ops._CAPTURE_CACHE = self.derived
        try:
            with torch.cuda.stream(side):
                rec.begin()
                try:
                    self.loss = step._train_pass(self.x, self.t, rec=rec)
                except BaseException:
                    rec.abort()
                    raise
                rec.end()
        finally:
            ops._CAPTURE_CACHE = prev
        torch.cuda.current_stream().wait_stream(side)
        self.steps = rec.steps
        self.n_graphs = sum(isinstance(s, torch.cuda.CUDAGraph) for s in self.steps)

    def __call__(self, x, target):
        if x.data_ptr() != self.x.data_ptr():
            self.x.copy_(x)
        self.t.copy_(target)
        for s in self.steps:
            if isinstance(s, torch.cuda.CUDAGraph):
                s.replay()
            else:
                s()
        return self.loss.clone()


TRAIN_GRAPH_WARMUP = 3            # eager steps per batch shape before its training pass is captured (the attack's graphs: step 3)


class ATTrainStep:
    """Builds ``DDP(WrappedModel(model, apgd))`` + optimizer (+EMA) and runs single steps.

    ``graph_train`` (default: on when ``adv.graph`` is set): after ``TRAIN_GRAPH_WARMUP`` eager steps the training pass is
    replayed from hipGraphs (``_TrainPassGraph``); it needs static batch shapes - a batch of another shape runs eagerly.

    ``grad_sync`` - how the gradients of the ranks meet when ``distributed``: ``"flat"`` (default): ``FlatGradSync`` - flat
    gradient buffers, two asynchronous all-reduces issued between the graph segments of the training pass, so an N > 1 rank runs
    the same replayed step as the single GPU; ``"ddp"``: ``torch.nn.parallel.DistributedDataParallel`` around the wrapped model
    (``main.py:889-890`` literally; its hooks keep the training pass eager).  ``grad_sync="flat"`` with ``distributed=False`` runs
    the N > 1 code path on one GPU (``bench.py --ddp-path 1``).

    ``state_bits`` - the optimizer: None = torch's AdamW, 32 or 8 = ``optim.FusedAdamW`` with moments of that many bits."""

    # what captures and replays the training pass (a seam for the process-group tests: a rank whose capture failed runs the pass
    # eagerly next to ranks that replay - both issue the same two all-reduces per step, tests/test_ddp_gloo.py)
    _graph_cls = _TrainPassGraph

    def __init__(self, model: nn.Module, arch: str, adv: AdvConfig, device, lr: float = 1e-3,
                 weight_decay: float = 0.05, distributed: bool = False, channels_last: bool = True,
                 amp_dtype: Optional[torch.dtype] = torch.bfloat16, ema: bool = True, mixup=None,
                 soft_targets: bool = False, perturb=None, gemm_table: bool = False, ema_decay: float = 0.9999,
                 graph_train: Optional[bool] = None, grad_sync: Optional[str] = None, state_bits: Optional[int] = None):
        self.device = torch.device(device)
        self.distributed = bool(distributed)
        if grad_sync not in (None, "flat", "ddp"):
            raise ValueError(f"grad_sync={grad_sync!r}")
        if grad_sync is None and distributed:
            grad_sync = "flat"
        if graph_train is None:
            graph_train = bool(getattr(adv, "graph", 0)) and os.environ.get("APGD_GRAPH_TRAIN", "1") != "0"
        self.graph_train = bool(graph_train) and grad_sync != "ddp" and self.device.type == 'cuda'
        self._tg = {}                                                      # (shapes, dtypes, id of the attack program whose derived
        #                                                                    copies it reads | None) -> _TrainPassGraph | None (failed)
        self._tg_seen = {}                                                 # (shapes, dtypes) -> eager steps so far
        self._tg_attack = {}                                               # (shapes, dtypes) -> that attack program (None: none)
        self._tg_failed = set()                                            # (shapes, dtypes) whose capture failed: eager from then on
        if gemm_table and self.device.type == 'cuda':
            # opt-in: points PyTorch's process-wide TunableOp at the shipped, read-only hipBLASLt solution table
            ops.load_gemm_table()
        if channels_last:
            model = model.to(memory_format=torch.channels_last)            # main.py:815-817
        if perturb is not None:                                            # any callable(model, x, y), as main.py:844
            from .wrapped_model import WrappedModel
            wrapped = WrappedModel(model, perturb).to(self.device)
        else:
            wrapped = wrap_model_for_at(model, adv, mixup=mixup).to(self.device)  # main.py:831-844, 881
        self.ema = DeviceEma(wrapped, ema_decay) if ema else None                     # before DDP (main.py:882-887)
        self.perturb = adv.attack != 'none' or perturb is not None
        self.inner = wrapped
        self.sync = None
        if grad_sync == "flat":
            self.sync = FlatGradSync(wrapped, self.device)
            if distributed:
                self.sync.broadcast_parameters(wrapped)
        elif distributed:
            ids = [self.device.index] if self.device.type == 'cuda' else None
            # main.py:889-890.  The models of this path carry constant buffers only (ImageNormalizer mean / std), so the
            # per-forward buffer broadcast is dropped; gradients live in the all-reduce buckets (no copy in / out per step).
            wrapped = nn.parallel.DistributedDataParallel(wrapped, device_ids=ids, broadcast_buffers=False,
                                                          gradient_as_bucket_view=True)
        self.model = wrapped
        self.optimizer = create_optimizer(self.inner, arch, weight_decay, capturable=self.graph_train, state_bits=state_bits)
        self.loss = (lambda o, t: torch.sum(-t * torch.log_softmax(o.float(), dim=-1), dim=-1).mean()) \
            if soft_targets else nn.CrossEntropyLoss()                     # SoftTargetCrossEntropy / CE (main.py:461-466)
        self.amp_dtype = amp_dtype
        self.lr = lr
        self.mixup_fn = mixup if callable(mixup) else None                # timm-style Mixup object (main.py:599-607)
        if self.perturb:
            self.inner.set_perturb(True)                                   # main.py:950-954
        self.model.train()

    def state_dict(self):
        """The model's state dict with the keys the reference's ``self.model.state_dict()`` has (``main.py:738-754``): under N > 1
        ranks that is ``DDP(WrappedModel(model))`` = ``module.base_model.*``.  On the flat gradient path ``self.model`` is the bare
        ``WrappedModel`` (no DDP object: ``.module`` / ``register_comm_hook`` do not exist there), so the ``module.`` prefix is added
        here and ``weights_{epoch}.pt`` / ``full_model_{epoch}.pth`` keep the reference's on-disk layout byte for byte; the loaders
        (``checkpoint.load_weights``, ``main.py:858``) strip it either way."""
        sd = self.model.state_dict()
        if self.distributed and not isinstance(self.model, nn.parallel.DistributedDataParallel):
            sd = {f"module.{k}": v for k, v in sd.items()}
        return sd

    def _set_lr(self, lr):
        for g in self.optimizer.param_groups:                              # main.py:973-974
            if isinstance(g['lr'], torch.Tensor):
                g['lr'].fill_(lr)                                          # capturable optimizer: the graph reads this tensor
            else:
                g['lr'] = lr

    def _train_pass(self, x_adv, target, rec=None):
        """forward - loss - backward - (gradient exchange) - AdamW - EMA on an already perturbed batch: what ``_TrainPassGraph``
        captures (``rec``: its recorder; the collectives are handed to it as eager closures between graph segments)."""
        sync = self.sync
        stash = {}
        hook = None
        if sync is not None and sync.cut is not None:
            hook = sync.cut.register_forward_hook(lambda m, i, o: stash.__setitem__("h", o))
        try:
            with torch.autocast(self.device.type, dtype=self.amp_dtype, enabled=self.amp_dtype is not None):
                output = self.inner.base_model(x_adv)                      # main.py:293 (WrappedModel.forward after the attack)
                loss = self.loss(output, target)
        finally:
            if hook is not None:
                hook.remove()
        if sync is None:
            loss.backward()                                                # main.py:992
        else:
            def between(fn):
                if rec is not None:
                    rec.eager(fn)
                else:
                    fn()
            h = stash.get("h")
            if (rec is None and not sync.verified and isinstance(h, torch.Tensor) and h.requires_grad and sync.late and sync.early):
                sync.check_split(loss, h)                                  # once, on the first eager pass (never inside a capture)
            if sync.cut is not None and isinstance(h, torch.Tensor) and h.requires_grad and sync.late and sync.early:
                g1 = torch.autograd.grad([loss], sync.late + [h], allow_unused=True)
                sync.store(0, g1[:-1])
                between(lambda: sync.start_reduce(0))                      # ... runs under the backward of the early stages
                g2 = torch.autograd.grad([h], sync.early, grad_outputs=[g1[-1]], allow_unused=True)
                sync.store(1, g2)
                del g1, g2
            else:
                g = torch.autograd.grad([loss], sync.late + sync.early, allow_unused=True)
                sync.store(0, g[:len(sync.late)])
                sync.store(1, g[len(sync.late):])
                del g
                between(lambda: sync.start_reduce(0))

            def finish():
                sync.start_reduce(1)
                sync.wait()
            between(finish)
        self.optimizer.step()                                              # main.py:993
        if self.ema is not None:
            self.ema.update()                                              # main.py:996-997
        return loss.detach()

    def warm_libraries(self, images, target):
        """One LOCAL training forward / backward of the model on this batch shape - no attack, no optimizer step, no collective,
        ``.grad`` untouched - so that the libraries under the path (MIOpen's find for the convolutions it still serves, hipBLASLt's
        heuristics) meet every shape of the training pass.  ``bench.py`` runs it on rank 0 first and on the other ranks behind a
        barrier: the per-process search of eight ranks is serialised into one search + seven find-db hits."""
        was = self.inner.base_model.training
        self.inner.base_model.train()
        params = [p for p in self.inner.base_model.parameters() if p.requires_grad]
        with torch.autocast(self.device.type, dtype=self.amp_dtype, enabled=self.amp_dtype is not None):
            out = self.inner.base_model(images)
            loss = self.loss(out, target)
        torch.autograd.grad([loss], params, allow_unused=True)
        self.inner.base_model.train(was)

    def _perturbed(self, images, target, borrow=False):
        """The first half of ``WrappedModel.forward`` (``main.py:276-292``): the attack in eval mode, under the step's autocast as
        ``main.py:985`` has it; returns ``x_best`` (``borrow``: a replayed attack hands out its graph's static tensor itself)."""
        if not self.perturb:
            return images
        import contextlib
        base = self.inner.base_model
        base.eval()
        with torch.autocast(self.device.type, dtype=self.amp_dtype, enabled=self.amp_dtype is not None), \
                (graphed.borrow_outputs() if borrow else contextlib.nullcontext()):
            z = self.inner.perturb(base, images, target)
        base.train()
        if isinstance(z, (tuple, list)):
            z = z[0]
        return z

    def _graph_step(self, images, target):
        """The step with the training pass replayed from a hipGraph; None if this batch has to run eagerly."""
        shape = (tuple(images.shape), images.dtype, tuple(target.shape), target.dtype)
        if shape in self._tg_failed:
            return None
        if shape not in self._tg_attack and self._tg_seen.get(shape, 0) < TRAIN_GRAPH_WARMUP:
            self._tg_seen[shape] = self._tg_seen.get(shape, 0) + 1        # libraries meet every shape outside a capture first
            return None
        replays0 = graphed.STATS["replays"]
        graphed.LAST = None
        z = self._perturbed(images, target, borrow=True)
        replayed = graphed.STATS["replays"] > replays0
        # The attack program that just replayed.  The training-pass graph of a batch shape READS the derived weight copies of the FIRST
        # program it was captured behind (that program rebuilds them at every replay from the live parameters); behind any other
        # attack - another program (a new eps, an evicted program) or an eager attack - a second, self-contained graph of the same
        # pass runs: a graph never reads copies that were not rebuilt in front of it in THIS step.
        aprog = graphed.LAST if (replayed and ops.SHARE_DERIVED) else None
        if self._tg_attack.setdefault(shape, aprog) is None:
            self._tg_attack[shape] = aprog                                 # (captured behind an eager attack first: shares from now on)
        if self._tg_attack[shape] is not aprog:
            aprog = None
        key = shape + (None if aprog is None else id(aprog),)
        prog = self._tg.get(key)
        if prog is None:
            try:
                # (a replayed attack under borrow_outputs hands out its graph's own static tensor: stable address)
                kw = {} if aprog is None else {"attack_prog": aprog}
                prog = self._tg[key] = self._graph_cls(self, z, target, x_is_static=replayed, **kw)
            except Exception as e:                                         # noqa: BLE001 - any capture failure means "run eagerly"
                import warnings
                warnings.warn(f"training-pass graph capture failed ({type(e).__name__}: {e}); this batch shape runs eagerly")
                self._tg[key] = None
                self._tg_failed.add(shape)
                if self.device.type == 'cuda':
                    torch.cuda.synchronize()
                if self.sync is None:
                    self.optimizer.zero_grad(set_to_none=True)
                loss = self._train_pass(z, target)
                ops.invalidate_weight_cache()
                return loss
        loss = prog(z, target)
        ops.invalidate_weight_cache()                                      # eager consumers of packed / bf16 weight copies
        return loss

    def step(self, images, target, lr: Optional[float] = None):
        self._set_lr(self.lr if lr is None else lr)
        if self.mixup_fn is not None:
            images, target = self.mixup_fn(images, target)                 # main.py:965-966 (soft labels [B, n_cls])
        if self.graph_train and (images.is_cuda or self._graph_cls is not _TrainPassGraph):
            loss = self._graph_step(images, target)
            if loss is not None:
                return loss
        return self._eager_step(images, target)

    def _eager_step(self, images, target):
        if self.sync is not None:                                          # same pass as the replayed one, launched from Python
            loss = self._train_pass(self._perturbed(images, target), target)
            ops.invalidate_weight_cache()
            return loss
        self.optimizer.zero_grad(set_to_none=True)                         # main.py:984
        with torch.autocast(self.device.type, dtype=self.amp_dtype, enabled=self.amp_dtype is not None):
            output = self.model(images, target) if self.perturb else self.model(images)   # main.py:985-989
            loss = self.loss(output, target)                               # main.py:990
        loss.backward()                                                    # main.py:992 (DDP all-reduce inside)
        self.optimizer.step()                                              # main.py:993
        ops.invalidate_weight_cache()                                      # packed / bf16 weight copies follow the update
        if self.ema is not None:
            self.ema.update()                                              # main.py:996-997
        return loss.detach()

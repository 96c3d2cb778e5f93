"""`torch.optim.Adam` for the drop-in trainer as ONE kernel launch per parameter group.

The reference's loop builds `optim.Adam(model.parameters(), lr=...)` (train.py:166) and steps it once per iteration after `check_weights`
(training.py:559-574).  torch's foreach path is eleven multi-tensor launches over the 42 + 32 tensors of the May model plus their host-side
list handling (~0.5 ms of a 1.4-ms-per-frame step); `FusedAdam.step()` is one launch of `s2l_adam_step` (csrc/train.hip): torch's
`_single_tensor_adam` arithmetic operation for operation in fp32, every tensor of the group through a device table of pointers, and -- because
the pass reads every parameter anyway -- the NaN scan of `check_weights` (src/common.py:56-64) folded into it (`nan_flags`).

Same constructor arguments, same `state_dict()` layout (`step`, `exp_avg`, `exp_avg_sq` per parameter) as `torch.optim.Adam`: a checkpoint
written by either loads into the other (the reference's checkpoints carry `optimizer.state_dict()`, checkpoints.py:38-41).  fp32 CUDA
parameters with dense gradients; no amsgrad / maximize / capturable (the reference uses none of them; a step under capture is refused).  There is no CPU path.

`FusedMuon` is the same for `torch.optim.Muon` (the update of a weight matrix orthogonalised before it is applied; its arithmetic in 32 bits where
torch's is bf16), with an Adam of its own for the parameters that are no such matrix; `orthogonalize` is its Newton-Schulz iteration alone
(csrc/orthogonalize.hip: every matrix of a group in the same 2 + 3 * steps launches)."""
from __future__ import annotations

import ctypes
import functools
import itertools
import math
import struct

import torch

from . import _abi


def _refuse_capture(who, dev):
    """A captured step would go on writing its report to host memory that the next step gives back (and Adam's would repeat one bias correction)."""
    if dev.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise _abi.S2LError(f"{who}: a step is not for capture into a graph")


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, amsgrad=False):
        if amsgrad:
            raise NotImplementedError("FusedAdam: amsgrad is not part of the reference's optimizer (train.py:166)")
        if lr < 0 or eps < 0 or weight_decay < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("FusedAdam: invalid hyper-parameter")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, amsgrad=False))
        self._plans = {}           # per group index: the cached launch plan (block table, counts, pinned staging, device buffers)
        self.nan_flags = None      # [(parameter, bool)] of the last step(): which parameters held a NaN BEFORE the update (after `nan_report()`)
        self._flag_jobs = []

    # ---- launch plan of one group: everything that only depends on the tensors' sizes
    def _plan(self, gi, ps):
        key = tuple((p.numel(), p.device) for p in ps)
        plan = self._plans.get(gi)
        if plan is not None and plan["key"] == key:
            return plan
        lib = _abi.load()
        dev = ps[0].device
        chunk = int(lib.s2l_adam_chunk())
        blocks = []
        for t, p in enumerate(ps):
            blocks += [(t, off) for off in range(0, p.numel(), chunk)]
        plan = {"key": key, "n_blocks": len(blocks),
                "blocks": torch.tensor(blocks, dtype=torch.int32).reshape(-1, 2).to(dev),
                "counts": torch.tensor([p.numel() for p in ps], dtype=torch.int64).to(dev),
                "host": torch.empty(len(ps) * 4, dtype=torch.int64, pin_memory=True),          # {param, grad, exp_avg, exp_avg_sq} pointers
                "table": torch.empty(len(ps) * 4, dtype=torch.int64, device=dev),
                "ptrs": None, "copied": None}
        self._plans[gi] = plan
        return plan

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._flag_jobs = []
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group["params"] if p.grad is not None]
            if ps:
                self._step_group(gi, group, ps)
        return loss

    def _step_group(self, gi, group, ps):
        """One launch of s2l_adam_step for the parameters `ps` of group `gi`."""
        lib = _abi.load()
        dev = ps[0].device
        _refuse_capture("FusedAdam", dev)
        for p in ps:
            if p.device != dev or dev.type != "cuda" or p.dtype != torch.float32 or p.grad.is_sparse or not p.is_contiguous() or p.is_neg():
                raise _abi.S2LError("FusedAdam takes contiguous fp32 CUDA parameters of one device with dense gradients (no CPU path)")
            st = self.state[p]
            if not st:
                st["step"] = torch.tensor(0.0, dtype=torch.float32)          # (torch.optim.Adam's own layout: a host scalar tensor)
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        steps = {float(self.state[p]["step"]) for p in ps}
        if len(steps) != 1:
            raise _abi.S2LError("FusedAdam: the parameters of one group must share their step count (one launch has one bias correction)")
        step_no = int(steps.pop()) + 1
        plan = self._plan(gi, ps)
        grads = [p.grad if (p.grad.dtype == torch.float32 and p.grad.is_contiguous() and not p.grad.is_neg())
                 else p.grad.to(torch.float32).resolve_neg().contiguous() for p in ps]
        ptrs = []
        for p, g in zip(ps, grads):
            st = self.state[p]
            ptrs += [p.data_ptr(), g.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()]
        with torch.cuda.device(dev):
            stream = torch.cuda.current_stream()
            if ptrs != plan["ptrs"]:      # (gradients are fresh tensors every step in the fused trainer: 2.4 KB of pointers cross once per step)
                if plan["copied"] is not None:
                    plan["copied"].synchronize()      # the pinned staging block of the previous step has left
                plan["host"].copy_(torch.tensor(ptrs, dtype=torch.int64))
                plan["table"].copy_(plan["host"], non_blocking=True)
                plan["copied"] = torch.cuda.Event()
                plan["copied"].record(stream)
                plan["ptrs"] = ptrs
            # (flags per step, not per plan: a pipelined caller reads step k's report after step k + 1 has been queued; the pinned block
            #  comes from torch's caching host allocator)
            flags = torch.zeros(len(ps), dtype=torch.int32, device=dev)
            flags_host = torch.empty(len(ps), dtype=torch.int32, pin_memory=True)
            b1, b2 = group["betas"]
            _abi.check(lib.s2l_adam_step(ctypes.c_void_p(plan["table"].data_ptr()), ctypes.c_void_p(plan["blocks"].data_ptr()),
                                         ctypes.c_void_p(plan["counts"].data_ptr()), len(ps), plan["n_blocks"], float(group["lr"]), float(b1),
                                         float(b2), float(group["eps"]), float(group["weight_decay"]), step_no,
                                         ctypes.c_void_p(flags.data_ptr()), ctypes.c_void_p(stream.cuda_stream)), "s2l_adam_step")
            flags_host.copy_(flags, non_blocking=True)
            done = torch.cuda.Event()
            done.record(stream)
        self._flag_jobs.append((ps, flags_host, done, grads))      # (`grads` keeps converted copies alive until the launch has run)
        for p in ps:
            self.state[p]["step"] += 1
            # the kernel wrote through raw pointers: tell autograd the tensor changed in place, as torch's own in-place update would --
            # the model's packed-weight caches (TalkingFace.packed_weights, SimpleUnetLight.packed_weights*) key on the version counters
            torch.autograd.graph.increment_version(p)

    def take_nan_jobs(self):
        """The last `step()`'s flag transfers, handed over to the caller (Trainer keeps them with its pending step): pass to `nan_report`."""
        jobs, self._flag_jobs = self._flag_jobs, []
        return jobs

    def nan_report(self, jobs=None):
        """[(parameter, True / False)] for the parameters of the last `step()` (or of `jobs`): held a NaN before that update.  Waits for that
        step's flags (a few bytes behind the kernel) -- call it after the next piece of work has been queued."""
        out = []
        for ps, host, done, _ in (self._flag_jobs if jobs is None else jobs):
            done.synchronize()
            out += list(zip(ps, [bool(v) for v in host.tolist()]))
        if jobs is None:
            self._flag_jobs = [(ps, host, done, None) for ps, host, done, _ in self._flag_jobs]
        self.nan_flags = out
        return out

    def covers(self):
        """The parameters whose NaN state `nan_report()` answers for (ids), given the gradients present now."""
        return {id(p) for g in self.param_groups for p in g["params"] if p.grad is not None}


def _refuse_tracing(who):
    """NotImplementedError under what records a program (torch.jit.trace, make_fx, fake tensors): it would not see the launches."""
    if torch._C._get_tracing_state() is not None or (torch._C._len_torch_dispatch_stack() and any(
            torch._C._get_dispatch_mode(key) is not None for key in torch._C._TorchDispatchModeKey.__members__.values())):
        raise NotImplementedError(f"{who}: not under a tracer, which would not see its launches")


def _matrix_table(records):
    """s2l_matrix records (in, out, momentum, rows, cols, step) as one host block."""
    return ctypes.create_string_buffer(struct.pack("=" + "qqqiif4x" * len(records), *itertools.chain.from_iterable(records)))


@functools.lru_cache(maxsize=64, typed=True)      # (of what passed; 2048 samples a step are 0.5 ms)
def _check_iteration(who, steps, coefficients, eps):
    if not (isinstance(steps, int) and not isinstance(steps, bool) and 1 <= steps <= 100):
        raise ValueError(f"{who}: steps must be a whole number from 1 to 100: got {steps!r}")
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f"{who}: three finite coefficients (a, b, c): got {coefficients!r}")
    if not eps > 0:
        raise ValueError(f"{who}: eps must be above 0: got {eps!r}")
    a, b, c = coefficients
    top = 1.0      # the largest singular value so far (the Frobenius norm starts at 1): the same bound as the library's, checked there again
    for k in range(steps):
        s = [top * i / 2048 for i in range(2049)]
        q = [abs(a + b * x * x + c * x ** 4) for x in s]
        top = max(max(x * y for x, y in zip(s, q)) * 1.01, 1e-6)
        if max(q) > 16 or (k + 1 < steps and top > 4):
            raise ValueError(f"{who}: with the coefficients {coefficients!r} a singular value can grow past 4 (or its factor past 16) in step {k + 1}: "
                             "beyond the range of the iteration's halves")


_ORTH_DTYPES = {torch.float32: _abi.S2L_DTYPE_F32, torch.bfloat16: _abi.S2L_DTYPE_BF16, torch.float16: _abi.S2L_DTYPE_F16}


def _iteration(who, steps, coefficients, eps):
    coefficients = tuple(float(c) for c in coefficients)
    _check_iteration(who, steps, coefficients, float(eps))
    return coefficients


def _check_matrices(given):
    for t in given:
        if not isinstance(t, torch.Tensor):
            raise TypeError("orthogonalize: a tensor [..., rows, cols] or a list of them")
        if t.dim() < 2:
            raise ValueError(f"orthogonalize: matrices [..., rows, cols]: got {tuple(t.shape)}")
        if t.dtype not in _ORTH_DTYPES or t.dtype != given[0].dtype:
            raise ValueError(f"orthogonalize: all float32, all bfloat16 or all float16: got {t.dtype}")
        if max(t.shape[-2:]) > 131072:
            raise ValueError(f"orthogonalize: at most 131072 rows and columns: got {tuple(t.shape)}")


def _orthogonalize_all(given, steps, a, b, c, eps):
    """The matrices of `given` (one type, one GPU) in one set of launches."""
    sources = [t.resolve_neg().contiguous() for t in given]
    outs = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in sources]
    lib = _abi.load()
    records = []
    for src, out in zip(sources, outs):
        rows, cols = src.shape[-2:]
        stride = rows * cols * src.element_size()
        if stride:
            records += [(src.data_ptr() + i * stride, out.data_ptr() + i * stride, 0, rows, cols, 0.0) for i in range(src.numel() // (rows * cols))]
    if not records:
        return outs
    dev = sources[0].device
    table = _matrix_table(records)
    with torch.cuda.device(dev):
        work = torch.empty(lib.s2l_orthogonalize_work_bytes(table, len(records)), dtype=torch.uint8, device=dev)
        _abi.check(lib.s2l_orthogonalize(_ORTH_DTYPES[sources[0].dtype], table, len(records), a, b, c, eps, steps, work.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream), "s2l_orthogonalize")
    return outs


def _orthogonalize_operator(updates, steps, a, b, c, eps):
    _check_matrices(updates)
    _check_iteration("orthogonalize", steps, (a, b, c), eps)
    if any(t.device != updates[0].device for t in updates):
        raise _abi.S2LError("orthogonalize: every tensor must be on one GPU (no CPU fallback)")
    return _orthogonalize_all(updates, steps, a, b, c, eps)


# The same as an operator that torch knows, for what watches, records or replaces a call's operators (dispatch modes: make_fx, fake tensors, selective
# checkpoints, counters; subclasses that dispatch for themselves): it would see the allocation of the results and not the launches that write them.
_operators = torch.library.Library("speech2lip_amd", "FRAGMENT")
_operators.define("orthogonalize(Tensor[] updates, int steps, float a, float b, float c, float eps) -> Tensor[]")
_operators.impl("orthogonalize", _orthogonalize_operator, "CUDA")
_operators.impl("orthogonalize", lambda updates, *_: [torch.empty_like(t, memory_format=torch.contiguous_format) for t in updates], "Meta")
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter))


@torch.no_grad()
def orthogonalize(update, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315), eps: float = 1e-7):
    """The Newton-Schulz iteration of Muon: X0 = G / max(||G||_F, eps), then `steps` times X <- (a I + b A + c A A) X with A = X X^T of the shorter
    side.  With the default coefficients the singular values end in 0.7 .. 1.2 (but for the smallest): nearly U V^T.

    update [..., rows, cols], or a list of such tensors of any sizes, all float32, all bfloat16 or all float16 on one GPU -> the same shape(s) and type,
    in one set of launches.  Operands of 22 bits, sums in fp32, rounded once: an fp32 iteration's accuracy; bfloat16: its last two steps on
    half-precision products (relative error 1.8e-3 to 2.2e-3, of which its rounding is 1.7e-3).
    A matrix that holds a NaN or an infinity comes out all NaN, a zero matrix zero.  Not differentiable (an optimiser's step is not), not
    under torch.jit.trace."""
    many = isinstance(update, (list, tuple))
    given = list(update) if many else [update]
    _check_matrices(given)
    if torch._C._get_tracing_state() is not None:
        raise NotImplementedError("orthogonalize: not under torch.jit.trace, which would record the allocation of the result and not the launches that write it")
    a, b, c = _iteration("orthogonalize", steps, coefficients, eps)
    for t in given:
        if not t.is_cuda or t.device != given[0].device:
            raise _abi.S2LError("orthogonalize: every tensor must be on one GPU (no CPU fallback)")
    if torch._C._len_torch_dispatch_stack() or not _PLAIN.issuperset(map(type, given)):
        outs = torch.ops.speech2lip_amd.orthogonalize(given, steps, a, b, c, float(eps)) if given else []
    else:
        outs = _orthogonalize_all(given, steps, a, b, c, float(eps))
    return outs if many else outs[0]


class FusedMuon(FusedAdam):
    """`torch.optim.Muon` -- momentum, orthogonalisation of the update, decoupled weight decay -- for every matrix of a parameter group in one set of
    launches (s2l_muon_step), the Newton-Schulz products on operands of 22 bits, summed in fp32; the same constructor arguments and `state_dict()` layout
    (`momentum_buffer` per parameter).  Parameters of more than two dimensions (convolutions) are taken as [shape[0], everything else].

        m <- m + (1 - momentum) (g - m);  u = g + momentum (m - g) if nesterov else m
        p <- (1 - lr weight_decay) p - lr_p orth(u),  lr_p = lr sqrt(max(1, rows / cols))             adjust_lr_fn None or "original"
                                                            = lr 0.2 sqrt(max(rows, cols))               "match_rms_adamw"
    A group with `algorithm="adam"` is stepped by FusedAdam (its own lr 1e-3, betas, eps 1e-8, weight_decay 0 unless given): biases, embeddings, the
    output layer, whatever is no weight matrix -- so that a Trainer drives both through one optimiser (`muon_groups` splits a model).
    fp32 CUDA parameters, contiguous, dense gradients; NaN report as FusedAdam's.  No CPU path, not for capture into a graph."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, ns_coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, ns_steps=5,
                 adjust_lr_fn=None):
        self._plans, self.nan_flags, self._flag_jobs = {}, None, []
        torch.optim.Optimizer.__init__(self, params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                                          ns_coefficients=tuple(ns_coefficients), eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn,
                                                          algorithm="muon"))

    def add_param_group(self, param_group):
        g = dict(param_group)
        if g.get("algorithm", "muon") == "adam":
            for key, value in (("lr", 1e-3), ("betas", (0.9, 0.999)), ("eps", 1e-8), ("weight_decay", 0.0), ("amsgrad", False)):
                g.setdefault(key, value)
            if g["amsgrad"]:
                raise NotImplementedError("FusedMuon: amsgrad is not supported")
            if g["lr"] < 0 or g["eps"] < 0 or g["weight_decay"] < 0 or not all(0 <= v < 1 for v in g["betas"]):
                raise ValueError("FusedMuon: invalid hyper-parameter of an adam group")
        elif g.get("algorithm", "muon") != "muon":
            raise ValueError(f"FusedMuon: algorithm must be \"muon\" or \"adam\": got {g['algorithm']!r}")
        else:
            full = {**self.defaults, **g}
            if full["lr"] < 0 or full["weight_decay"] < 0 or not 0 <= full["momentum"] <= 1:
                raise ValueError("FusedMuon: invalid hyper-parameter (lr, weight_decay >= 0, momentum in 0 .. 1)")
            if full["adjust_lr_fn"] not in (None, "original", "match_rms_adamw"):
                raise ValueError(f"FusedMuon: adjust_lr_fn must be None, \"original\" or \"match_rms_adamw\": got {full['adjust_lr_fn']!r}")
            g["ns_coefficients"] = _iteration("FusedMuon", full["ns_steps"], full["ns_coefficients"], full["eps"])
            g["params"] = [g["params"]] if isinstance(g["params"], torch.Tensor) else list(g["params"])
            for p in g["params"]:
                t = p[1] if isinstance(p, tuple) else p
                if isinstance(t, torch.Tensor) and (t.dim() < 2 or t.numel() == 0 or max(t.shape[0], t.numel() // t.shape[0]) > 131072):
                    raise ValueError(f"FusedMuon: a muon group takes matrices of 1 .. 131072 rows and columns (others: a group with algorithm=\"adam\"): "
                                     f"got {tuple(t.shape)}")
        super().add_param_group(g)

    def _step_group(self, gi, group, ps):
        if group.get("algorithm", "muon") == "adam":
            return super()._step_group(gi, group, ps)
        _refuse_tracing("FusedMuon")
        _refuse_capture("FusedMuon", ps[0].device)
        lib = _abi.load()
        lr, mode = float(group["lr"]), group["adjust_lr_fn"]
        index, f32, state = ps[0].get_device(), torch.float32, self.state
        records, grads, buffers = [], [], []
        for p in ps:
            g = p.grad
            if p.get_device() != index or index < 0 or p.dtype != f32 or g.layout != torch.strided or not p.is_contiguous():
                raise _abi.S2LError("FusedMuon takes contiguous fp32 CUDA parameters of one device with dense gradients (no CPU path)")
            st = state[p]
            m = st.get("momentum_buffer")
            if m is None:
                if p.is_neg():
                    raise _abi.S2LError("FusedMuon: a parameter that is a lazily negated view")
                m = st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            elif m.shape != p.shape or m.dtype != f32 or m.get_device() != index or not m.is_contiguous():
                m = st["momentum_buffer"] = m.to(device=p.device, dtype=f32).reshape(p.shape).contiguous()
            if g.dtype != f32 or not g.is_contiguous() or g.is_neg():
                g = g.to(f32).resolve_neg().contiguous()
            rows, count = p.shape[0], p.numel()
            cols = count // rows
            scale = 0.2 * math.sqrt(max(rows, cols)) if mode == "match_rms_adamw" else math.sqrt(rows / cols) if rows > cols else 1.0
            records.append((g.data_ptr(), p.data_ptr(), m.data_ptr(), rows, cols, lr * scale))
            grads.append(g)
            buffers.append(m)
        table = _matrix_table(records)
        a, b, c = coefficients = tuple(group["ns_coefficients"])
        _check_iteration("FusedMuon", group["ns_steps"], coefficients, group["eps"])
        dev = ps[0].device
        with torch.cuda.device(dev):
            stream = torch.cuda.current_stream()
            flags = torch.zeros(len(ps), dtype=torch.int32, device=dev)
            flags_host = torch.empty(len(ps), dtype=torch.int32, pin_memory=True)
            work = torch.empty(lib.s2l_orthogonalize_work_bytes(table, len(ps)), dtype=torch.uint8, device=dev)
            _abi.check(lib.s2l_muon_step(table, len(ps), float(group["momentum"]), int(bool(group["nesterov"])), 1.0 - lr * float(group["weight_decay"]), a, b, c,
                                         float(group["eps"]), group["ns_steps"], flags.data_ptr(), work.data_ptr(), stream.cuda_stream), "s2l_muon_step")
            flags_host.copy_(flags, non_blocking=True)
            done = torch.cuda.Event()
            done.record(stream)
        self._flag_jobs.append((ps, flags_host, done, grads))
        torch.autograd.graph.increment_version(ps + buffers)      # written through raw pointers (see FusedAdam)


def muon_groups(model, adam_names=("output_linear.", "outc.", "canonical_depth_head"), muon=None, adam=None):
    """Parameter groups of `model` for FusedMuon: its weight matrices (two or more dimensions), and, stepped by Adam, everything else and whatever
    `adam_names` name by their beginning (the output layers, the depth image).  muon / adam: options of the two groups."""
    named = [(k, p) for k, p in model.named_parameters() if p.requires_grad]
    is_matrix = lambda k, p: p.dim() >= 2 and not any(part in "." + k for part in ("." + a for a in adam_names))  # noqa: E731
    groups = [{"params": [p for k, p in named if is_matrix(k, p)], **(muon or {}), "algorithm": "muon"},
              {"params": [p for k, p in named if not is_matrix(k, p)], **(adam or {}), "algorithm": "adam"}]
    return [g for g in groups if g["params"]]

"""AdamW on gfx950: the optimizer the reference builds (training/engine.py:10-16,
torch.optim.AdamW(groups, ..., foreach=False, fused=True)) with its step in the HIP kernel
ct_adamw_step.

`FusedAdamW` takes torch.optim.AdamW's arguments and keeps its state layout (per
parameter: a fp32 `step` tensor on the parameter's device, `exp_avg` and `exp_avg_sq` in
the parameter's dtype), so checkpoints written for the reference's fused optimizer load
unchanged (checkpointing/io.py:205-222 checks exactly these keys, shapes and dtypes).
Each step is one launch per parameter group and dtype: the step counters are incremented
and every tensor is updated from a device-side table of (param, grad, exp_avg,
exp_avg_sq, step, numel) rows and a list of fixed-size chunks. Parameters must live on
the HIP device in fp32 or bf16 with dense gradients of the same dtype; amsgrad is not
supported (the reference does not use it).

Beside it stands an optimizer for parameters that are all matrices, as LoRA adapters are:
`FusedMuon` takes torch.optim.Muon's arguments and keeps its state key (`momentum_buffer`; in
float32 whatever the parameter's type), and `orthogonalize` is its iteration alone. Both run
ct_muon: the Newton-Schulz steps in double on the short side's Gram matrix, all matrices of one
type in one set of launches, results rounded once (torch's runs the steps in bfloat16).
"""

import ctypes
import functools
import math

import torch

from .kernels import _native

_CHUNK = 1 << 16  # elements per workgroup


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False, *,
                 maximize=False, foreach=None, capturable=False, differentiable=False, fused=True):
        if not 0.0 <= float(lr):
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameters: {betas}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if amsgrad:
            raise NotImplementedError("FusedAdamW: amsgrad is not supported")
        if differentiable:
            raise NotImplementedError("FusedAdamW: differentiable updates are not supported")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False, maximize=maximize,
                        foreach=foreach, capturable=capturable, differentiable=False, fused=True)
        super().__init__(params, defaults)
        self._tables = {}

    def _state_of(self, p):
        state = self.state[p]
        if not state:
            state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            state["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        return state

    def _table(self, slot, rows, device):
        """Device copies of the tensor table and the chunk list of one (group, device,
        dtype) slot, reused while the same storages take part in the step."""
        key = tuple(rows)
        cached = self._tables.get(slot)
        if cached is not None and cached[0] == key:
            return cached[1], cached[2]
        table = torch.tensor([list(r) for r in rows], dtype=torch.int64).reshape(-1, 6)
        chunks = [(index, start) for index, r in enumerate(rows) for start in range(0, r[5], _CHUNK)]
        chunk_list = torch.tensor(chunks, dtype=torch.int64).reshape(-1, 2)
        # Pinned host copies go up asynchronously on the current stream (no host wait); the
        # pinned allocator keeps their blocks until the copies are done.
        entry = (key, table.pin_memory().to(device, non_blocking=True),
                 chunk_list.pin_memory().to(device, non_blocking=True))
        self._tables[slot] = entry
        return entry[1], entry[2]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _native.library()
        for index, group in enumerate(self.param_groups):
            beta1, beta2 = group["betas"]
            buckets = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("FusedAdamW does not support sparse gradients")
                if not p.is_cuda or p.dtype not in (torch.float32, torch.bfloat16):
                    raise NotImplementedError("FusedAdamW: parameters must be fp32 or bf16 device tensors")
                if p.grad.dtype != p.dtype or not p.is_contiguous() or not p.grad.is_contiguous():
                    raise NotImplementedError("FusedAdamW: contiguous gradients of the parameter's dtype required")
                state = self._state_of(p)
                buckets.setdefault((p.device, p.dtype), []).append((p, state))
            for (device, dtype), members in buckets.items():
                rows = [(p.data_ptr(), p.grad.data_ptr(), s["exp_avg"].data_ptr(), s["exp_avg_sq"].data_ptr(),
                         s["step"].data_ptr(), p.numel()) for p, s in members if p.numel()]
                if not rows:
                    for _, s in members:
                        s["step"] += 1
                    continue
                for p, s in members:
                    if not p.numel():
                        s["step"] += 1
                table, chunks = self._table((index, device, dtype), rows, device)
                with torch.cuda.device(device):
                    status = lib.ct_adamw_step(
                        _native.ptr(table), len(rows), _native.ptr(chunks), len(chunks), _CHUNK,
                        _native.dtype_code(dtype), float(group["lr"]), float(beta1), float(beta2),
                        float(group["eps"]), float(group["weight_decay"]), int(bool(group["maximize"])), 1,
                        _native.stream_of(members[0][0]))
                _native.check(status, "ct_adamw_step")
        return loss


_captured_plans = set()   # plans that a captured graph reads: never dropped


class _MuonPlan:
    """The shares of work of one list of shapes on one device: kept between steps."""

    def __init__(self, shapes, device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("orthogonalize/FusedMuon: the first call with a list of shapes makes its plan and cannot "
                               "be captured; run it once before the capture")
        lib = _native.library()
        table = (_native.MuonMatrix * len(shapes))()
        for row, (rows, cols) in zip(table, shapes):
            row.rows, row.cols = rows, cols
        self.counts, needed = (ctypes.c_int64 * _native.CT_MUON_KINDS)(), ctypes.c_int64()
        _native.check(lib.ct_muon_plan(table, len(shapes), None, 0, self.counts, ctypes.byref(needed)), "ct_muon_plan")
        size = sum(self.counts)
        entries = torch.empty(size, 8, dtype=torch.int32)
        _native.check(lib.ct_muon_plan(table, len(shapes), entries.data_ptr(), size, self.counts, ctypes.byref(needed)),
                      "ct_muon_plan")
        # A copy that the host waits for: complete for every stream.
        with torch.cuda.device(device):
            self.entries = entries.to(device)
            self.stream = _native.stream_of(self.entries)
        self.table, self.workspace = bytes(table), needed.value

    def run(self, matrices, dtype, options):
        """One call over `matrices`, a list of (param, grad, momentum) addresses and the factor on
        the learning rate, in the shapes' order."""
        device, stream = self.entries.device, _native.stream_of(self.entries)
        table = (_native.MuonMatrix * len(matrices)).from_buffer_copy(self.table)
        for row, (param, grad, momentum, adjust) in zip(table, matrices):
            row.param, row.grad, row.momentum, row.adjust = param, grad, momentum, adjust
        if torch.cuda.is_current_stream_capturing():
            _captured_plans.add(self)
        elif stream != self.stream:
            self.entries.record_stream(torch.cuda.current_stream(device))
        workspace = torch.empty(self.workspace, dtype=torch.uint8, device=device)
        with _native.device_of(self.entries):
            status = _native.library().ct_muon(
                table, len(matrices), self.entries.data_ptr(), self.counts, _native.dtype_code(dtype),
                ctypes.byref(options), workspace.data_ptr(), self.workspace, self.workspace, stream)
        _native.check(status, "ct_muon")


@functools.lru_cache(maxsize=64)
def _muon_plan(shapes, device):
    return _MuonPlan(shapes, device)


_MUON_SHORT, _MUON_LONG = 16384, 1 << 30   # sides of a matrix that ct_muon_plan takes


def _refuse_large(name, shape):
    if min(shape) > _MUON_SHORT or max(shape) > _MUON_LONG:
        raise NotImplementedError(f"{name}: the HIP kernels take matrices up to {_MUON_SHORT} x {_MUON_LONG}, "
                                  f"not {tuple(shape)}")


def _muon_numbers(coefficients, steps, eps):
    """Checked (a, b, c), steps and eps of the iteration."""
    a, b, c = (float(x) for x in coefficients)
    if not all(math.isfinite(x) for x in (a, b, c)):
        raise ValueError(f"Invalid Newton-Schulz coefficients: {coefficients}")
    if not 1 <= int(steps) <= 100 or int(steps) != steps:
        raise ValueError(f"Invalid number of Newton-Schulz steps: {steps}")
    if not float(eps) >= 0.0:
        raise ValueError(f"Invalid epsilon value: {eps}")
    return (a, b, c), int(steps), float(eps)


def _newton_schulz(matrix, coefficients, steps, eps):
    """The iteration in torch operations, in double: host tensors."""
    a, b, c = coefficients
    x = matrix.double()
    x = x.T if x.shape[0] > x.shape[1] else x
    x = x / x.norm().clamp(min=eps)
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.T if matrix.shape[0] > matrix.shape[1] else x).to(matrix.dtype).contiguous()


@torch.no_grad()
def orthogonalize(matrices, *, coefficients=(3.4445, -4.7750, 2.0315), steps=5, eps=1e-7):
    """Matrices with their singular values driven towards one by Newton-Schulz steps:
    X = M / max(|M|, eps), then `steps` times X = a X + (b A + c A^2) X with A = X X^T (of the
    transposed matrix where it has more rows than columns).

    `matrices` is a 2-D tensor or a list of them, float32 or bfloat16 on the device (any strides,
    types and devices mixed, shorter sides up to 16384, longer ones up to 2^30); returns new
    contiguous tensors of the same shapes and types, one or a list, that carry no gradient. Empty
    matrices come back empty, zero ones zero (where eps is not zero); device matrices need
    max(|M|, eps) of 1e-35, below which float32 factors 1 / |M| overflow.

    A direction that M does not have grows from rounding noise by a per step, as in any iteration
    in 32 bits: matrices of low rank are 2e-5 off after 5 steps of the default coefficients, 1e-2
    after 10 and about 0.1 however many follow; those of full rank stay within 2e-7."""
    coefficients, steps, eps = _muon_numbers(coefficients, steps, eps)
    single = isinstance(matrices, torch.Tensor)
    inputs = [matrices] if single else list(matrices)
    buckets, results = {}, []
    for index, m in enumerate(inputs):
        if m.dim() != 2:
            raise ValueError(f"orthogonalize: a tensor of shape {tuple(m.shape)} is not a matrix")
        if m.is_cuda and m.dtype not in (torch.float32, torch.bfloat16):
            raise NotImplementedError("orthogonalize: the HIP kernels take float32 or bfloat16")
        if not m.is_floating_point():
            raise ValueError("orthogonalize: matrices of a floating type required")
        if not m.is_cuda:
            results.append(_newton_schulz(m, coefficients, steps, eps) if m.numel() else m.clone())
            continue
        _native.refuse_tangents("orthogonalize", m)
        _refuse_large("orthogonalize", m.shape)
        results.append(torch.empty(m.shape, dtype=m.dtype, device=m.device))
        if m.numel():
            buckets.setdefault((m.device, m.dtype), []).append(index)
    options = _native.MuonOptions(a=coefficients[0], b=coefficients[1], c=coefficients[2], eps=eps, steps=steps)
    for (device, dtype), members in buckets.items():
        sources = [inputs[i].contiguous() for i in members]
        plan = _muon_plan(tuple(tuple(m.shape) for m in sources), device)
        plan.run([(results[i].data_ptr(), m.data_ptr(), None, 1.0) for i, m in zip(members, sources)], dtype, options)
    return results[0] if single else results


def _adjusted(adjust_lr_fn, rows, cols):
    """Factor on the learning rate of a [rows, cols] matrix."""
    if adjust_lr_fn == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    return math.sqrt(max(1.0, rows / cols))


class FusedMuon(torch.optim.Optimizer):
    """Muon over matrices on the device (shorter sides up to 16384); torch.optim.Muon's arguments.

    Each step: momentum = mu momentum + (1 - mu) grad, M = mu momentum + (1 - mu) grad (nesterov)
    or momentum, param = param (1 - lr weight_decay) - lr adjust orthogonalize(M), with adjust =
    sqrt(max(1, rows / cols)) ("original", the default) or 0.2 sqrt(max(rows, cols))
    ("match_rms_adamw"). A step can be captured into a graph after a first one outside; the
    graph keeps the learning rate and the other numbers that it was captured with."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True,
                 ns_coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, ns_steps=5, adjust_lr_fn=None):
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps,
                                      adjust_lr_fn=adjust_lr_fn))

    @staticmethod
    def _check_group(group):
        if not 0.0 <= float(group["lr"]):
            raise ValueError(f"Invalid learning rate: {group['lr']}")
        if not 0.0 <= group["momentum"] <= 1.0:
            raise ValueError(f"Invalid momentum value: {group['momentum']}")
        if not 0.0 <= group["weight_decay"]:
            raise ValueError(f"Invalid weight_decay value: {group['weight_decay']}")
        if group["adjust_lr_fn"] not in (None, "original", "match_rms_adamw"):
            raise ValueError(f"Invalid learning rate adjustment: {group['adjust_lr_fn']}")
        _muon_numbers(group["ns_coefficients"], group["ns_steps"], group["eps"])
        for p in group["params"]:
            if p.dim() != 2:
                raise ValueError(f"FusedMuon takes matrices only, not a parameter of shape {tuple(p.shape)}")

    def add_param_group(self, param_group):
        """Adds a group, or raises and leaves the optimizer as it was."""
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict):
        """Loads a state dict (this class's or torch.optim.Muon's); the buffers stay float32,
        which the base class would round to a bfloat16 parameter's type."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        for group, given in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], given["params"]):
                if "momentum_buffer" in saved.get(key, ()):
                    self.state[p]["momentum_buffer"] = saved[key]["momentum_buffer"].to(
                        device=p.device, dtype=torch.float32, copy=True).contiguous()

    def _buffer_of(self, p):
        state = self.state[p]
        if "momentum_buffer" not in state:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("FusedMuon: a parameter's first step makes its momentum_buffer and cannot be captured "
                                   "(every replay would clear it); run a step before the capture")
            state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        buffer = state["momentum_buffer"]
        if (buffer.dtype != torch.float32 or buffer.shape != p.shape or buffer.device != p.device
                or not buffer.is_contiguous()):
            raise RuntimeError("FusedMuon: momentum_buffer must be a contiguous float32 tensor of the parameter's shape")
        return buffer

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            coefficients, steps, eps = _muon_numbers(group["ns_coefficients"], group["ns_steps"], group["eps"])
            buckets = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("FusedMuon does not support sparse gradients")
                if not p.is_cuda or p.dtype not in (torch.float32, torch.bfloat16):
                    raise NotImplementedError("FusedMuon: parameters must be fp32 or bf16 device tensors")
                if p.grad.dtype != p.dtype or not p.is_contiguous() or not p.grad.is_contiguous():
                    raise NotImplementedError("FusedMuon: contiguous gradients of the parameter's dtype required")
                if p.numel():
                    _refuse_large("FusedMuon", p.shape)
                    buckets.setdefault((p.device, p.dtype), []).append((p, self._buffer_of(p)))
            options = _native.MuonOptions(
                lr=float(group["lr"]), weight_decay=float(group["weight_decay"]), momentum=float(group["momentum"]),
                a=coefficients[0], b=coefficients[1], c=coefficients[2], eps=eps,
                nesterov=int(bool(group["nesterov"])), steps=steps, update=1)
            for (device, dtype), members in buckets.items():
                plan = _muon_plan(tuple(tuple(p.shape) for p, _ in members), device)
                plan.run([(p.data_ptr(), p.grad.data_ptr(), m.data_ptr(), _adjusted(group["adjust_lr_fn"], *p.shape))
                          for p, m in members], dtype, options)
        return loss

"""GraphAdamW: AdamW over all tensors of a group at once, with a step that a CUDA graph can replay.

:class:`~adambridge_b200.optimizer.AdamBridge` hands the step count, the learning rate and the rounding seed to its
kernels from the host, so a captured update would repeat one step for ever.  ``GraphAdamW`` keeps what changes from
step to step on the device: step counts, optionally the learning rate, the clip coefficient, and whether to skip the
step.  Everything runs on the caller's current stream, with no host synchronization::

    opt = GraphAdamW(model.parameters(), lr=lr, precision="int8")
    ...                                             # warm-up steps on a side stream, as torch.cuda.graph wants
    with torch.cuda.graph(graph):
        loss = model(x).square().mean()
        loss.backward()
        opt.clip_grad_norm_(1.0)
        opt.step()
    graph.replay()                                  # the next step, every time

The state of a parameter group is one :class:`StateArena`: flat buffers in which each parameter starts on a
256-value boundary.  Moments are fp32 or 8-bit blocks: ``m = code * scale`` with int8 codes, ``v = (code * scale)**2``
with uint8 codes, one fp32 scale per 256 values, 2.03 bytes per parameter for both.  bf16 parameters have an fp32
master; fp32 parameters are updated in place.
"""

from __future__ import annotations

import ctypes
from typing import Any, Callable, Iterable

import torch

from . import native
from .clip import clip_coefficient
from .precision import StateBuffer

__all__ = ["GraphAdamW", "StateArena"]

BLOCK = native.I8_BLOCK
_PRECISIONS = ("fp32", "int8")
_CODES = {"m": torch.int8, "v": torch.uint8}


def _padded(n: int) -> int:
    return -(-n // BLOCK) * BLOCK


def _capturing() -> bool:
    return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()


class StateArena:
    """The optimizer state of one parameter group: flat device buffers, parameter ``i`` at ``offsets[i]``.

    ``m``, ``v``: fp32 values, or int8 / uint8 codes with ``m_scale``, ``v_scale`` (one per 256 values; else None);
    ``master``: the fp32 masters of the bf16 parameters, parameter ``i`` at ``master_offsets[i]`` (None for an fp32
    parameter; the buffer is None if the group has no bf16 one); ``steps``: steps taken, int64 per parameter.
    Values between a parameter's end and the next boundary are zero and stay zero (but for 8-bit moments whose block has a
    value that is not finite: the whole block reads back as NaN)."""

    def __init__(self, params: list[torch.Tensor], first_index: int, precision: str):
        for p in params:
            if not p.is_cuda:
                raise ValueError("adambridge_b200 updates CUDA parameters only (the state lives in GPU memory)")
            if p.device != params[0].device:
                raise ValueError("GraphAdamW needs all parameters of a group on one device")
            if not p.is_contiguous():
                raise ValueError("non-contiguous parameters are not supported")
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError(f"parameters must be float32 or bfloat16, got {p.dtype}")
        self.params, self.precision, self.first_index, self._ops = params, precision, first_index, native.torch_ops()
        dev = self.device = params[0].device
        self.numels, self.dtypes = [p.numel() for p in params], [p.dtype for p in params]
        self.offsets: list[int] = []
        self.master_offsets: list[int | None] = []
        total = masters = 0
        for n, dt in zip(self.numels, self.dtypes):
            self.offsets.append(total)
            self.master_offsets.append(masters if dt == torch.bfloat16 else None)
            total += _padded(n)
            masters += _padded(n) if dt == torch.bfloat16 else 0
        self.numel = total
        zeros = lambda n, dt: torch.zeros(n, dtype=dt, device=dev)   # noqa: E731
        int8 = precision == "int8"
        self.m = zeros(total, torch.int8 if int8 else torch.float32)
        self.v = zeros(total, torch.uint8 if int8 else torch.float32)
        self.m_scale = zeros(total // BLOCK, torch.float32) if int8 else None
        self.v_scale = zeros(total // BLOCK, torch.float32) if int8 else None
        self.steps = zeros(len(params), torch.int64)
        self.ticket = zeros(1, torch.int32)
        self.master = None
        if masters:
            self.master = zeros(masters, torch.float32)
            for p, n, at in zip(params, self.numels, self.master_offsets):
                if at is not None:
                    self.master[at:at + n].copy_(p.detach().reshape(-1))
        # one kernel description per parameter, as words: what a step changes is the weight's and gradient's address
        rows = []
        item = self.m.element_size()
        for i, (n, dt, at, mat) in enumerate(zip(self.numels, self.dtypes, self.offsets, self.master_offsets)):
            scale = at // BLOCK * 4
            rows.append([0, 0, 0 if mat is None else self.master.data_ptr() + 4 * mat,
                         self.m.data_ptr() + item * at, self.v.data_ptr() + item * at,
                         self.m_scale.data_ptr() + scale if int8 else 0, self.v_scale.data_ptr() + scale if int8 else 0,
                         self.steps.data_ptr() + 8 * i, n,
                         (first_index + i) | (native.dtype_code_of(dt) << 32)])
        self._table = torch.tensor(rows, dtype=torch.int64)

    def describe(self):
        """The kernel's descriptions of the parameters that have a gradient: parameters and gradients are checked and
        their addresses taken now."""
        return self._ops.describe_step(self.params, self._table, self.device.index)

    def launch(self, described, shared: native.GraphStep, max_ctas: int) -> None:
        """Enqueue the step of what :meth:`describe` returned, on the current stream."""
        self._ops.launch_step(described, ctypes.addressof(shared), self.ticket, max_ctas)

    # ------------------------------------------------------------------ reading and writing the moments

    def _plane(self, role: str) -> tuple[torch.Tensor, torch.Tensor | None]:
        return (self.m, self.m_scale) if role == "m" else (self.v, self.v_scale)

    def _values(self, role: str) -> torch.Tensor:
        plane, scales = self._plane(role)
        if scales is None:
            return plane
        return self._ops.i8_decode(plane, scales, self.numel, role == "v")

    def exp_avg(self) -> torch.Tensor:
        """The first moments as flat fp32 (``numel`` values, parameter ``i`` from ``offsets[i]``): the live buffer, or
        decoded from 8 bits into a new one."""
        return self._values("m")

    def exp_avg_sq(self) -> torch.Tensor:
        """The second moments, as :meth:`exp_avg` gives the first."""
        return self._values("v")

    def master_of(self, i: int) -> torch.Tensor:
        """Parameter ``i``'s fp32 master: a view of the buffer, or of the parameter if it is its own master."""
        at = self.master_offsets[i]
        return self.params[i].detach().view(-1) if at is None else self.master[at:at + self.numels[i]]

    def saved_moment(self, i: int, role: str, as_fp32: bool) -> dict[str, Any]:
        """Parameter ``i``'s moment as a checkpoint dict."""
        plane, scales = self._plane(role)
        at, n = self.offsets[i], self.numels[i]
        if scales is None:
            return {"precision": "fp32", "data": plane[at:at + n]}
        end = at + _padded(n)
        codes, scale = plane[at:end], scales[at // BLOCK:end // BLOCK]
        if not as_fp32:
            return {"precision": "int8", "role": role, "block": BLOCK, "q": codes, "scale": scale}
        return {"precision": "fp32", "data": self._ops.i8_decode(codes, scale, n, role == "v")}

    def reset_master(self, i: int) -> None:
        """Parameter ``i``'s master from its weight as it is now."""
        if self.master_offsets[i] is not None:
            self.master_of(i).copy_(self.params[i].detach().reshape(-1))

    def reset(self, i: int) -> None:
        """Parameter ``i``'s state as a new optimizer has it, in place."""
        at, end = self.offsets[i], self.offsets[i] + _padded(self.numels[i])
        self.m[at:end].zero_()
        self.v[at:end].zero_()
        if self.m_scale is not None:
            self.m_scale[at // BLOCK:end // BLOCK].zero_()
            self.v_scale[at // BLOCK:end // BLOCK].zero_()
        self.steps[i] = 0
        self.reset_master(i)

    def load_moment(self, i: int, role: str, saved: "dict | StateBuffer") -> None:
        """Write a checked checkpoint moment: int8 planes as they are, other formats by their values."""
        plane, scales = self._plane(role)
        at, n = self.offsets[i], self.numels[i]
        end = at + _padded(n)
        if isinstance(saved, dict) and scales is not None:
            plane[at:end].copy_(saved["q"].reshape(-1))
            scales[at // BLOCK:end // BLOCK].copy_(saved["scale"].reshape(-1))
            return
        if isinstance(saved, dict):
            q, scale = (saved[name].reshape(-1).to(self.device).contiguous() for name in ("q", "scale"))
            values = self._ops.i8_decode(q, scale, n, role == "v")
        else:
            values = saved.to_device(self.device).to_fp32()
        if scales is None:
            plane[at:at + n].copy_(values)
        else:
            self._ops.i8_encode(values, plane[at:end], scales[at // BLOCK:end // BLOCK], role == "v")

    @property
    def nbytes(self) -> dict[str, int]:
        size = lambda *ts: sum(t.nbytes for t in ts if t is not None)   # noqa: E731
        return {"master": size(self.master), "moments": size(self.m, self.v, self.m_scale, self.v_scale),
                "control": size(self.steps, self.ticket)}


def _check_int8(saved: dict, numel: int, role: str, what: str) -> dict:
    blocks = _padded(numel) // BLOCK
    if saved.get("block") != BLOCK or saved.get("role") != role:
        raise ValueError(f"checkpoint {what}: expected int8 blocks of {BLOCK} values of role {role!r}, found "
                         f"{saved.get('block')!r} and {saved.get('role')!r}")
    for name, dt, n in (("q", _CODES[role], blocks * BLOCK), ("scale", torch.float32, blocks)):
        t = saved.get(name)
        if not isinstance(t, torch.Tensor) or t.dtype != dt or t.numel() != n:
            raise ValueError(f"checkpoint {what}: {name} must be a {dt} tensor of {n} elements")
    return saved


class GraphAdamW(torch.optim.Optimizer):
    r"""AdamW (decoupled weight decay, bias correction) whose whole step is device work on the current stream.

    Arguments are AdamBridge's where they have its names.  ``precision`` is ``'int8'`` (8-bit blocks) or ``'fp32'``;
    ``stochastic_rounding`` rounds 8-bit moments at random, so that the expected moment is the moment to within 2^-16 of the
    gap between its neighbouring codes, by a hash of ``seed``, the parameter's index, its step and the element: the same run
    gives the same bits.  A second moment whose root is below one code of its block (1/255 of the block's largest) is the
    exception, with either rounding: it is stored as one code, so that it never reads as zero, and such an element moves less
    than its own moment would have it.  ``lr`` of a group may
    be a one-element float32 or float64 CUDA tensor, read by every replay of a captured step; a float is captured as
    it is.  ``max_ctas`` caps the CTAs of a launch (0: all).

    The arithmetic is fp32 with each operation rounded once (AdamBridge reproduces its reference's fused
    multiply-adds instead), and a gradient is scaled in fp32: the two optimizers agree to rounding, not bit for bit.

    A step makes the state of parameters that have none yet, which a graph cannot capture: take a step, or call
    :meth:`prepare`, before the capture.  Graphs that captured steps of one optimizer update the same state: replay them
    one after another.  As with any captured backward pass, drop what holds an earlier eager graph
    of the same parameters (its loss, its outputs) before capturing, and warm up on a side stream.
    """

    def __init__(self, params: Iterable[torch.Tensor] | Iterable[dict[str, Any]], lr: float | torch.Tensor = 1e-3,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 precision: str = "int8", stochastic_rounding: bool = True, seed: int = 0, max_ctas: int = 0):
        if precision not in _PRECISIONS:
            raise ValueError(f"unknown moment precision {precision!r}; expected one of {sorted(_PRECISIONS)}")
        if max_ctas < 0:
            raise ValueError("max_ctas must be >= 0")
        self.precision, self.stochastic, self.seed, self.max_ctas = precision, stochastic_rounding, seed, max_ctas
        self.arenas: list[StateArena] = []       # one per parameter group, once prepared
        self._native = native.load()
        # coefficient, norm, captured, the stream that they were made on
        self._clip: tuple[torch.Tensor, torch.Tensor, bool, torch.cuda.Stream] | None = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group: dict[str, Any]) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
            if not group["params"]:
                raise ValueError("a parameter group needs at least one parameter")
            if len({id(p) for p in group["params"]}) != len(group["params"]):
                raise ValueError("a parameter group holds a parameter twice")
            if any(p.is_sparse for p in group["params"]):
                raise ValueError("GraphAdamW does not support sparse parameters")
        except (ValueError, TypeError):
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(group: dict[str, Any]) -> None:
        lr, betas = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype not in (torch.float32, torch.float64):
                raise TypeError("lr must be a float or a one-element float32 or float64 tensor")
        elif not lr >= 0.0:
            raise ValueError(f"invalid learning rate: {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"invalid betas: {betas}")
        if not group["eps"] >= 0.0:
            raise ValueError(f"invalid epsilon: {group['eps']}")
        if not group["weight_decay"] >= 0.0:
            raise ValueError(f"invalid weight_decay: {group['weight_decay']}")

    @classmethod
    def _check_saved_group(cls, group: dict[str, Any], what: str) -> None:
        for name in ("lr", "betas", "eps", "weight_decay"):
            if name not in group:
                raise ValueError(f"{what} has no {name}")
        cls._check_group(group)
        for name in ("maximize", "amsgrad"):
            if group.get(name):
                raise ValueError(f"{what} has {name}=True, which GraphAdamW does not do")
        if group["weight_decay"] and not group.get("decoupled_weight_decay", True):
            raise ValueError(f"{what} adds its weight decay to the gradient; GraphAdamW's is decoupled")

    # ------------------------------------------------------------------ the step

    def prepare(self) -> "GraphAdamW":
        """Make the state (fp32 masters from the weights as they are now, zero moments) where there is none yet."""
        if len(self.arenas) < len(self.param_groups):
            if _capturing():
                raise RuntimeError("GraphAdamW: make the state before a capture (prepare(), or an uncaptured step)")
            first = sum(len(a.params) for a in self.arenas)
            for group in self.param_groups[len(self.arenas):]:
                self.arenas.append(StateArena(group["params"], first, self.precision))
                first += len(group["params"])
        return self

    @torch.no_grad()
    def step(self, closure: Callable[[], torch.Tensor] | None = None, grad_scale: torch.Tensor | None = None,
             found_inf: torch.Tensor | None = None):
        """Update every parameter that has a gradient, on the current stream.

        ``grad_scale`` and ``found_inf`` are one-element float32 CUDA tensors: every gradient is multiplied by the
        first inside the kernel, and where the second is not zero the step changes nothing, step counts included.
        After :meth:`clip_grad_norm_` the clip coefficient is the scale, and a step whose gradient norm is not finite
        changes nothing either.  For autograd the step is a change in place of the parameters that it describes."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        clip, self._clip = self._clip, None
        if clip is not None and grad_scale is not None:
            raise ValueError("step(grad_scale=...) after clip_grad_norm_(): the clip coefficient is the scale")
        if clip is not None and clip[2] != _capturing():
            raise RuntimeError("clip_grad_norm_() and its step() belong into one capture, or both outside: the other's "
                               "coefficient would be that of other gradients")
        coef, norm = clip[:2] if clip is not None else (grad_scale, None)
        self.prepare()
        # every group is described, and so checked, before any is launched
        work = [(arena, arena.describe(), self._shared(arena, group, coef, found_inf, norm))
                for arena, group in zip(self.arenas, self.param_groups)]
        for arena, described, shared in work:
            arena.launch(described, shared, self.max_ctas)
        if clip is not None:
            made, now = clip[3], torch.cuda.current_stream(clip[3].device)
            if now != made:   # the memory stays until this stream has read it
                for t in clip[:2]:
                    t.record_stream(now)
        return loss

    def _shared(self, arena: StateArena, group: dict[str, Any], coef, found_inf, norm) -> native.GraphStep:
        self._check_group(group)
        s = native.GraphStep(beta1=group["betas"][0], beta2=group["betas"][1], eps=group["eps"],
                             weight_decay=group["weight_decay"],
                             moments=native.DT_I8 if self.precision == "int8" else native.DT_F32,
                             stochastic=int(self.stochastic), seed=self.seed & 0xFFFFFFFF)
        lr = group["lr"]
        if isinstance(lr, torch.Tensor) and lr.is_cuda:
            if lr.device != arena.device:
                raise ValueError(f"lr is on {lr.device}, its parameters on {arena.device}")
            s.lr_ptr, s.lr_f64 = lr.data_ptr(), int(lr.dtype == torch.float64)
        else:
            s.lr = float(lr)
        for name, t in (("grad_scale", coef), ("found_inf", found_inf), ("the gradient norm", norm)):
            if t is None:
                continue
            if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float32 and t.numel() == 1):
                raise TypeError(f"{name} must be a one-element float32 CUDA tensor")
            if t.device != arena.device:
                raise ValueError(f"{name} is on {t.device}, the parameters on {arena.device}")
        s.g_scale = None if coef is None else coef.data_ptr()
        s.skip = None if found_inf is None else found_inf.data_ptr()
        s.norm = None if norm is None else norm.data_ptr()
        return s

    @torch.no_grad()
    def clip_grad_norm_(self, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
        """``torch.nn.utils.clip_grad_norm_`` over this optimizer's gradients, applied by the next :meth:`step` as it
        reads them (see :meth:`AdamBridge.clip_grad_norm_`); both are captured, or neither.  Returns the total norm; the
        step is skipped on the device if it is not finite."""
        if float(norm_type) != 2.0:
            raise ValueError("GraphAdamW.clip_grad_norm_ computes the L2 norm (norm_type=2) only")
        self._clip = None
        grads = [p.grad for group in self.param_groups for p in group["params"] if p.grad is not None]
        if not grads:
            return torch.tensor(0.0)
        if any(g.device != grads[0].device for g in grads):
            raise ValueError("clip_grad_norm_ needs gradients of one device")
        wide = [g for g in grads if g.dtype == torch.float32]
        if len(wide) in (0, len(grads)):
            total, coef, _ = clip_coefficient(grads, max_norm, kernels=self._native)
        else:
            # as clip_coefficient treats mixed gradients, in an order that needs no index on the device (a capture
            # cannot copy one there): each norm rounded to its gradient's dtype, the total in fp32
            parts = ([g for g in grads if g.dtype != torch.float32], wide)
            norms = [clip_coefficient(part, max_norm, kernels=self._native)[2] for part in parts]
            total = torch.linalg.vector_norm(torch.cat(norms))
            coef = torch.clamp(max_norm / (total + 1e-6), max=1.0).reshape(1)
        self._clip = (coef, total.float().reshape(1), _capturing(), torch.cuda.current_stream(grads[0].device))
        return total

    # ------------------------------------------------------------------ inspection

    def memory_report(self) -> dict[str, int]:
        """Device bytes the optimizer holds, by category."""
        report = {"master": 0, "moments": 0, "control": 0}
        for arena in self.arenas:
            for k, n in arena.nbytes.items():
                report[k] += n
        report["total"] = sum(report.values())
        return report

    def master_params(self) -> list[torch.Tensor]:
        """The fp32 master of each parameter, in optimizer order, as flat views (of the parameter itself where it is
        its own master); empty before the state is made."""
        return [a.master_of(i) for a in self.arenas for i in range(len(a.params))]

    # ------------------------------------------------------------------ checkpoints

    def state_dict(self, moments: str = "stored") -> dict[str, Any]:
        """AdamBridge's checkpoint dict, tensors left on the GPU (views of the live state).  8-bit moments are saved
        as they are stored, for this class; ``moments='fp32'`` saves their values, which AdamBridge loads too.
        Synchronizes, to read the step counts."""
        if moments not in ("stored", "fp32"):
            raise ValueError("moments must be 'stored' or 'fp32'")
        sd = super().state_dict()
        state = {}
        for arena in self.arenas:
            for i, step in enumerate(arena.steps.tolist()):
                if step:
                    state[arena.first_index + i] = {
                        "step": step, "master": arena.master_of(i),
                        "exp_avg": arena.saved_moment(i, "m", moments == "fp32"),
                        "exp_avg_sq": arena.saved_moment(i, "v", moments == "fp32")}
        sd["state"] = state
        sd["adambridge"] = {"precision": "fp32" if moments == "fp32" else self.precision, "master_precision": "fp32",
                            "format": 1, "algorithm": "adamw"}
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        """Load a GraphAdamW, AdamBridge or ``torch.optim.AdamW`` checkpoint.  Everything is checked before anything
        changes; moments in another format are re-encoded on the GPU (to the nearest codes).

        The checkpoint replaces the whole state, in the same buffers: a parameter that it does not list starts over, and
        an fp32 master that it does not hold is taken from the bf16 weight, so load the model's weights first."""
        where = [(arena, i) for arena in self.prepare().arenas for i in range(len(arena.params))]
        parsed = {}
        for key, entry in state_dict["state"].items():
            index = int(key) if isinstance(key, str) and key.isdigit() else key
            if isinstance(index, bool) or not isinstance(index, int) or not 0 <= index < len(where):
                raise ValueError(f"checkpoint state for parameter {key!r}: this optimizer has parameters "
                                 f"0..{len(where) - 1}")
            arena, i = where[index]
            n = arena.numels[i]
            missing = [name for name in ("exp_avg", "exp_avg_sq") if name not in entry]
            if missing:
                raise ValueError(f"checkpoint parameter {index} has no {' or '.join(missing)} (saved by LionBridge?): "
                                 "GraphAdamW needs 2 moments")
            master = None
            if entry.get("master") is not None:
                master = StateBuffer.master_from_checkpoint(entry["master"], n, f"master weights of parameter {index}")
            found = []
            for name, role in (("exp_avg", "m"), ("exp_avg_sq", "v")):
                saved, what = entry[name], f"{name} of parameter {index}"
                if isinstance(saved, dict) and saved.get("precision") == "int8":
                    found.append((role, _check_int8(saved, n, role, what)))
                else:
                    found.append((role, StateBuffer.from_checkpoint(saved, n, role, what)))
            step = entry["step"]
            step = int(step.item() if isinstance(step, torch.Tensor) else step)
            if step < 0:
                raise ValueError(f"checkpoint parameter {index} has taken {step} steps")
            parsed[index] = (step, master, found)
        for number, group in enumerate(state_dict["param_groups"]):
            self._check_saved_group(group, f"checkpoint parameter group {number}")
        rates = [group["lr"] for group in self.param_groups]
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        for group, lr in zip(self.param_groups, rates):
            if isinstance(lr, torch.Tensor):   # a captured step reads this tensor
                group["lr"] = lr.copy_(torch.as_tensor(group["lr"]).reshape(lr.shape))
        for index, (arena, i) in enumerate(where):
            if index not in parsed:
                arena.reset(i)
                continue
            step, master, found = parsed[index]
            arena.steps[i] = step
            if master is not None:
                arena.master_of(i).copy_(master.to_device(arena.device).to_fp32())
            else:
                arena.reset_master(i)
            for role, saved in found:
                arena.load_moment(i, role, saved)

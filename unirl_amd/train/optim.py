"""AdamW over all of a policy's parameters in a few launches.

The optimizer step of the reference's train stack (``unirl/train/stack.py:332``): the gradients' global
norm (``unirl/train/fsdp_utils.py:313``), the clip factor and the AdamW update.  The norm never leaves
the device, and the clipped gradients are never written: the update multiplies by the factor as it
reads them.
"""

from __future__ import annotations

import collections
import copy
from typing import Any, Dict, List, Optional, Tuple

import torch

from .. import _native as N
from .. import ops


def _placed(saved: torch.Tensor, held: Any, device: torch.device) -> torch.Tensor:
    """A copy of ``saved`` on ``device``, in the tensor ``held`` where that is of its kind."""
    if isinstance(held, torch.Tensor) and (held.shape, held.dtype, held.device) == (saved.shape, saved.dtype, device):
        return held.copy_(saved)
    return saved.detach().to(device, copy=True).contiguous()


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s update (decoupled weight decay) with fused kernels.

    ``state_bits``: moments in fp32 (32), or in one byte each with a power-of-two scale per 256
    elements (8; formats in :func:`unirl_amd.ops.adamw_moments`).  ``master_weights`` keeps an fp32 copy of
    16-bit parameters, without which updates below half a unit in the last place of a parameter are
    lost; it is made in a parameter's first step and leads from then on, so parameters written by
    hand (loaded weights) need :meth:`refresh_masters`.  Both may be set per parameter group.

    ``max_grad_norm`` clips by the global norm of all groups' gradients; ``step()`` leaves that norm in
    ``grad_norm`` (a device scalar; ``None`` without ``max_grad_norm`` and ``skip_nonfinite``).
    ``skip_nonfinite`` makes a step whose norm is Inf or NaN write nothing and not count.

    ``capturable`` keeps the count of steps on the device, one per group, so that ``step()`` can be
    captured into a graph and replayed (``lr`` as an fp32 device scalar may then change between replays);
    ``skip_nonfinite`` needs it.  The first step, which makes the state, has to run before the capture.
    Otherwise each parameter counts the steps in which it had a gradient.

    Parameters are contiguous fp32, bf16 or fp16 tensors on a HIP device, one per group (with clipping or
    ``skip_nonfinite``, one for all groups); sparse gradients are refused.
    """

    def __init__(
        self,
        params,
        lr=1e-3,
        betas: Tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 1e-2,
        *,
        state_bits: int = 32,
        master_weights: bool = False,
        max_grad_norm: Optional[float] = None,
        skip_nonfinite: bool = False,
        capturable: bool = False,
        seed: int = 0,
    ) -> None:
        if isinstance(lr, torch.Tensor):
            if not capturable:
                raise ValueError("a tensor lr needs capturable=True")
        elif not lr >= 0.0:
            raise ValueError(f"lr must not be negative; got {lr}")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError(f"max_grad_norm must not be negative; got {max_grad_norm}")
        if skip_nonfinite and not capturable:
            raise ValueError("skip_nonfinite needs capturable=True: whether a step counts is known on the device only")
        self.max_grad_norm = max_grad_norm
        self.skip_nonfinite = bool(skip_nonfinite)
        self.capturable = bool(capturable)
        self.grad_norm: Optional[torch.Tensor] = None
        self._next_base = 0
        self._controls: Dict[int, torch.Tensor] = {}
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                        master_weights=master_weights, seed=int(seed), step=None)
        super().__init__(params, defaults)

    def add_param_group(self, param_group: Dict[str, Any]) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            ops._adamw_hyper(group["betas"], group["eps"], group["weight_decay"])
            if group["state_bits"] not in (8, 32):
                raise ValueError(f"state_bits must be 8 or 32; got {group['state_bits']}")
            if len(set(group["params"])) != len(group["params"]):
                raise ValueError("a parameter appears more than once in its group")
            for p in group["params"]:
                N.dtype_code(p.dtype)
                if not p.is_contiguous():
                    raise ValueError(f"parameters must be contiguous; got strides {p.stride()} of {tuple(p.shape)}")
        except Exception:
            self.param_groups.pop()
            raise

    # -- copies and pickles: the base class keeps defaults, state and groups alone ---------------------
    _OPTIONS = ("max_grad_norm", "skip_nonfinite", "capturable", "_next_base")

    def __getstate__(self) -> Dict[str, Any]:
        return {**super().__getstate__(), **{k: getattr(self, k) for k in self._OPTIONS}}

    def __setstate__(self, state: Dict[str, Any]) -> None:
        super().__setstate__(state)
        self._controls = {}
        self.grad_norm = None

    # -- state -------------------------------------------------------------
    def _new_state(self, group: Dict[str, Any], p: torch.Tensor) -> Dict[str, Any]:
        N.require_device(p, "parameter")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: run one step before capturing: the state would be made anew by every replay")
        blocks = -(-p.numel() // ops.ADAMW_BLOCK)
        state: Dict[str, Any] = {"step": 0, "index_base": self._next_base}
        self._next_base += self._indices(p)
        dtype = torch.float32 if group["state_bits"] == 32 else torch.uint8
        for name in ("exp_avg", "exp_avg_sq"):
            state[name] = torch.zeros(p.shape, dtype=dtype, device=p.device)
            if dtype is torch.uint8:
                state[name + "_scale"] = torch.zeros(blocks, dtype=torch.uint8, device=p.device)
        if group["master_weights"] and p.dtype is not torch.float32:
            state["master"] = p.detach().to(torch.float32, copy=True)
        return state

    def moments(self, p: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(exp_avg, exp_avg_sq)`` of a parameter as fp32 values, whatever they are held in."""
        s = self.state.get(p)  # a look must not leave an entry behind
        if not s:
            raise ValueError("the parameter has no state: it had no gradient in any step so far")
        if "exp_avg_scale" not in s:
            return s["exp_avg"], s["exp_avg_sq"]
        return ops.adamw_moments(s["exp_avg"], s["exp_avg_sq"], s["exp_avg_scale"], s["exp_avg_sq_scale"])

    @torch.no_grad()
    def refresh_masters(self) -> None:
        """Take the fp32 masters anew from the parameters as they are."""
        for p, s in self.state.items():
            if "master" in s:
                s["master"].copy_(p)

    @torch.no_grad()
    def load_state_dict(self, state_dict: Dict[str, Any]) -> None:
        """The state of :meth:`state_dict`; what does not fit this optimizer (another optimizer's state, other
        shapes, moments in other bits, masters on one side only) raises ``ValueError`` and leaves it as it was.
        The groups take the saved rates and constants; how a state is held (``state_bits``,
        ``master_weights``) stays this optimizer's choice.  States, counts and tensor rates that are
        already there are written in place, so that a captured step goes on with what was loaded."""
        state_dict = state_dict.copy()
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        saved, groups = state_dict["state"], copy.deepcopy(state_dict["param_groups"])
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the saved parameter groups differ from this optimizer's in number or size")
        rates = [float(g["lr"]) for g in groups if "lr" in g]
        loaded: List[Tuple[torch.Tensor, Dict[str, Any], int]] = []
        for mine, group in zip(self.param_groups, groups):
            missing = [k for k in self._GROUP_KEYS if k not in group]
            if missing:
                raise ValueError(f"not a state of this optimizer: its parameter groups have no {', '.join(missing)}")
            ops._adamw_hyper(group["betas"], group["eps"], group["weight_decay"])
            for k in ("state_bits", "master_weights"):
                group[k] = mine[k]
            if isinstance(group["lr"], torch.Tensor):  # where the parameters are; a number where the host counts
                group["lr"] = (group["lr"].to(mine["params"][0].device if mine["params"] else None, torch.float32)
                               if self.capturable else float(group["lr"]))
            states = [(p, saved[i]) for p, i in zip(mine["params"], group["params"]) if saved.get(i)]
            for p, s in states:
                self._check_state(mine, p, s)
            counts = self._counts(mine, group, [s for _, s in states])
            loaded += [(p, s, n) for (p, s), n in zip(states, counts)]
        # from here on nothing is refused
        ids = {i for g in groups for i in g["params"]}
        state: Dict[Any, Any] = collections.defaultdict(dict)
        state.update((k, v) for k, v in saved.items() if k not in ids)
        # saved tensors that are this optimizer's own may be written before they are read
        own = {t.data_ptr() for s in self.state.values() for t in s.values() if isinstance(t, torch.Tensor)}
        loaded = [(p, {k: v.clone() if isinstance(v, torch.Tensor) and v.data_ptr() in own else v for k, v in s.items()}, n)
                  for p, s, n in loaded]
        self._next_base = 0
        for p, s, count in loaded:
            old = self.state.get(p, {})
            state[p] = {k: _placed(v, old.get(k), p.device) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
            state[p]["step"] = count
            self._next_base = max(self._next_base, s["index_base"] + self._indices(p))
        for mine, group, rate in zip(self.param_groups, groups, rates):
            for p in mine["params"]:
                if self.capturable and self.state.get(p) and p not in state:  # a captured step may hold it
                    state[p] = self.state[p]
                    for k, v in state[p].items():
                        if isinstance(v, torch.Tensor):
                            v.copy_(p) if k == "master" else v.zero_()
                    state[p]["index_base"] = self._next_base
                    self._next_base += self._indices(p)
            group["params"] = mine["params"]
            if "param_names" in mine:
                group.setdefault("param_names", mine["param_names"])
            if isinstance(group["step"], torch.Tensor):
                group["step"] = _placed(group["step"], mine["step"], group["step"].device)
            if self.capturable and isinstance(mine["lr"], torch.Tensor):  # may be the rate of several groups
                one = len({r for g, r in zip(self.param_groups, rates) if g["lr"] is mine["lr"]}) == 1
                group["lr"] = mine["lr"].fill_(rate) if one else torch.full_like(mine["lr"], rate)
        controls = self._controls
        self.__setstate__({"state": state, "param_groups": groups})
        self._controls = controls
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def _counts(self, mine: Dict[str, Any], group: Dict[str, Any], states: List[Dict[str, Any]]) -> List[int]:
        """Where this optimizer keeps the count of steps: ``group["step"]`` on the device with ``capturable`` (the
        states then hold 0), else one number per state.  A count saved in the other place moves over."""
        count, counts = group.setdefault("step", None), [int(s["step"]) for s in states]
        if not self.capturable:
            group["step"] = None
            return counts if count is None else [int(count)] * len(states)
        if count is None and counts:
            if len(set(counts)) > 1:
                raise ValueError(f"capturable=True counts one number of steps per group; the saved parameters have {sorted(set(counts))}")
            count = counts[0]
        if count is not None or mine["step"] is not None:
            device = mine["params"][0].device if mine["params"] else None
            group["step"] = torch.tensor(int(count or 0), dtype=torch.int64, device=device)
        return [0] * len(states)

    @staticmethod
    def _indices(p: torch.Tensor) -> int:
        """Dither positions of a parameter's elements: whole blocks."""
        return -(-p.numel() // ops.ADAMW_BLOCK) * ops.ADAMW_BLOCK

    _GROUP_KEYS = ("lr", "betas", "eps", "weight_decay", "state_bits", "master_weights", "seed")

    @staticmethod
    def _check_state(group: Dict[str, Any], p: torch.Tensor, s: Dict[str, Any]) -> None:
        missing = [k for k in ("step", "index_base", "exp_avg", "exp_avg_sq") if k not in s]
        if missing:
            raise ValueError(f"not a state of this optimizer: a parameter's state has no {', '.join(missing)}")
        blocks = -(-p.numel() // ops.ADAMW_BLOCK)
        dtype = torch.float32 if group["state_bits"] == 32 else torch.uint8
        want = {"exp_avg": (dtype, p.shape), "exp_avg_sq": (dtype, p.shape)}
        if dtype is torch.uint8:
            want.update({"exp_avg_scale": (dtype, (blocks,)), "exp_avg_sq_scale": (dtype, (blocks,))})
        if group["master_weights"] and p.dtype is not torch.float32:
            want["master"] = (torch.float32, p.shape)
        for name, (kind, shape) in want.items():
            t = s.get(name)
            if not isinstance(t, torch.Tensor) or t.dtype != kind or t.shape != torch.Size(shape):
                found = f"{t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else type(t).__name__
                raise ValueError(f"saved moments are unlike this optimizer's: {name} is {found}; it holds {kind} {tuple(shape)}")
        if "master" in s and "master" not in want:
            raise ValueError("the saved state has fp32 masters; this optimizer (master_weights=False) would lose them")
        if s["index_base"] < 0 or s["index_base"] % ops.ADAMW_BLOCK:
            raise ValueError(f"index_base must be a multiple of {ops.ADAMW_BLOCK}; got {s['index_base']}")

    # -- the step ------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        if capturing and not self.capturable:
            raise RuntimeError("AdamW: a captured step needs capturable=True (the count of steps would not move)")
        strided, state_of = torch.strided, self.state
        pairs = [[(p, p.grad) for p in group["params"] if p.grad is not None] for group in self.param_groups]
        if any(g.layout is not strided for group in pairs for _, g in group):
            raise RuntimeError("AdamW does not support sparse gradients")
        counted = not self.capturable
        # what shares a call: types, master, count of steps; all groups' before the first launch, so that a
        # state that cannot be made leaves every group as it was
        work: List[Dict[Any, List[Any]]] = []
        for group, with_grad in zip(self.param_groups, pairs):
            buckets: Dict[Any, List[Any]] = {}
            known = True
            for p, g in with_grad:
                s = state_of.get(p)
                if not s:
                    if known and len({q.device for q, _ in with_grad}) > 1:
                        raise ValueError("the parameters of a group that have gradients must share one device")
                    known = False
                    s = state_of[p] = self._new_state(group, p)
                buckets.setdefault((p.dtype, g.dtype, "master" in s, s["step"]), []).append((p, g, s))
            work.append(buckets)
        self.grad_norm = None
        clip: Dict[str, Any] = {}
        if self.max_grad_norm is not None or self.skip_nonfinite:
            grads = [g for group in pairs for _, g in group]
            if grads:
                self.grad_norm = ops.grad_norm(grads)
                clip = dict(grad_norm=self.grad_norm, max_norm=self.max_grad_norm, skip_nonfinite=self.skip_nonfinite)
        for index, (group, with_grad, buckets) in enumerate(zip(self.param_groups, pairs, work)):
            if not with_grad:
                continue
            how: Dict[str, Any] = {}
            if self.capturable:
                how["control"] = self._advance(index, group, with_grad[0][0].device, clip)
            else:
                how.update(lr=float(group["lr"]), weight_decay=group["weight_decay"], seed=group["seed"], **clip)
            small = group["state_bits"] == 8
            for (_, _, master, count), rows in buckets.items():
                ps, gs, states = zip(*rows)

                def column(name, wanted=True):
                    return [s[name] for s in states] if wanted else None

                if counted:
                    how["step"] = count + 1
                ops.adamw_step(
                    ps, gs, column("exp_avg"), column("exp_avg_sq"), betas=group["betas"], eps=group["eps"],
                    masters=column("master", master), exp_avg_scales=column("exp_avg_scale", small),
                    exp_avg_sq_scales=column("exp_avg_sq_scale", small), index_bases=column("index_base"), **how,
                )
                if counted:
                    for s in states:
                        s["step"] = count + 1
        return loss

    def _advance(self, index: int, group: Dict[str, Any], device: torch.device, clip: Dict[str, Any]) -> torch.Tensor:
        """The group's count of steps goes up on the device; the step's scalars."""
        count, control = group["step"], self._controls.get(index)
        if count is None or control is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: run one step before capturing: the state would be made anew by every replay")
            if count is None:
                count = group["step"] = torch.zeros((), dtype=torch.int64, device=device)
            elif count.device != device:
                count = group["step"] = count.to(device)
            control = self._controls[index] = torch.zeros(N.ADAMW_CONTROL_BYTES, dtype=torch.uint8, device=device)
        ops.adamw_advance(count, control, lr=group["lr"], betas=group["betas"], weight_decay=group["weight_decay"],
                          seed=group["seed"], **clip)
        return control


__all__ = ["AdamW"]

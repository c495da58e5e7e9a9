"""Single-launch optimizers for the training scripts' ``optimizer.step()``
(reference tests/gcn/graphcuda_impl.py:45,56).

``FusedAdam`` follows ``torch.optim.Adam`` (amsgrad / maximize off) and
``FusedSGD`` the momentum-free ``torch.optim.SGD`` the reference's script
builds (``FusedAdamW``, for deeper models, has its own notes below); both update every parameter of the model with one kernel
(``gc_adam_step_f32`` / ``gc_sgd_step_f32``).  The Adam step count lives on the
device, so ``step()`` can be recorded in a CUDA graph and replayed
(graphed.GraphedTrainStep); ``lr`` is read on the host when the launch is
issued -- or recorded -- so change it between captures, not between replays.
"""
from __future__ import annotations

import torch

from . import _lib

_MAX = 32  # tensors per launch (kMaxTensors in csrc/optim.cu)


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0):
        if lr < 0 or eps < 0 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1 or weight_decay < 0:
            raise ValueError("FusedAdam: invalid hyper-parameter")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def _group_state(self, group, device, chunk):
        key = f"_gc_state_{device.index}_{chunk}"
        if key not in group:
            # [steps taken, CTA arrival counter]; zero before the first step
            group[key] = torch.zeros(2, dtype=torch.int64, device=device)
        return group[key]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = self.state[p]
                if not st:
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                by_device.setdefault(p.device, []).append(p)
            for dev, all_ps in by_device.items():
                # one launch per 32 tensors; every launch keeps its own step count
                for chunk, i in enumerate(range(0, len(all_ps), _MAX)):
                    ps = all_ps[i:i + _MAX]
                    st = [self.state[p] for p in ps]
                    _lib.host.adam_step(ps, [p.grad for p in ps], [x["exp_avg"] for x in st],
                                        [x["exp_avg_sq"] for x in st], group["lr"], group["betas"][0],
                                        group["betas"][1], group["eps"], group["weight_decay"],
                                        self._group_state(group, dev, chunk))
        return loss

    def steps_taken(self) -> int:
        """Reads the device step count of the first group back (synchronises)."""
        for group in self.param_groups:
            for k, v in group.items():
                if k.startswith("_gc_state_"):
                    return int(v[0].item())
        return 0


class FusedSGD(torch.optim.Optimizer):
    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.0):
        if lr < 0 or weight_decay < 0:
            raise ValueError("FusedSGD: invalid hyper-parameter")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is not None:
                    by_device.setdefault(p.device, []).append(p)
            for ps in by_device.values():
                for i in range(0, len(ps), _MAX):
                    chunk = ps[i:i + _MAX]
                    _lib.host.sgd_step(chunk, [p.grad for p in chunk], group["lr"], group["weight_decay"])
        return loss


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, masters=None, scales=None, seed: int = 0, follow: bool = False) -> None:
    """One AdamW step over lists of tensors, in place; one launch for up to 449 tensors (688 in float32 alone).

    ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
    ``p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)``.

    ``params`` and ``grads`` are all float32, or all bfloat16 beside float32 ``masters``, which take the update: a parameter is
    its master's rounding, whatever it held before.  ``follow=True``: one that is not has been changed by others since the last
    step, and its master takes its value first.
    ``exp_avgs`` and ``exp_avg_sqs`` are float32; or uint8 (zeros at the start) with ``scales = (of exp_avgs, of
    exp_avg_sqs)``, float32 tensors of ceil(size / 256) elements each: 8 bits per value, rounded at random by a hash of
    (seed, step, position in the list, element).  ``step`` is a CUDA int64 tensor of two elements, zeros at the start; the
    kernel counts in it, so the call can be recorded in a CUDA graph."""
    of_m, of_v = scales if scales is not None else ((), ())
    _lib.host.adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, masters or (), of_m, of_v, lr, betas[0], betas[1], eps,
                         weight_decay, seed & 0xFFFFFFFF, follow)


def adamw_moments(exp_avgs, exp_avg_sqs, scales, out=None):
    """The values that moments in 8 bits stand for: two lists of float32 tensors (``out``, where given)."""
    if out is None:
        out = tuple([torch.empty(t.shape, dtype=torch.float32, device=t.device) for t in ts] for ts in (exp_avgs, exp_avg_sqs))
    _lib.host.adamw_moments(exp_avgs, exp_avg_sqs, scales[0], scales[1], out[0], out[1])
    return out


class FusedAdamW(torch.optim.Optimizer):
    """AdamW (``torch.optim.AdamW``, amsgrad and maximize off) for any number of tensors, up to 449 to a launch (688 in float32 alone).

    Float32 parameters are updated as they are; bfloat16 ones beside a float32 master in the optimizer's state, which follows a
    parameter that others have changed between steps (a state dict loaded, a copy, weights clipped; recorded or not).
    ``state_bits=8`` holds both moments in 8 bits with a float32 scale per 256 elements (see ``adamw_step``): 2 bytes per
    parameter instead of 8.  Tensors of 256 elements and fewer keep 32 bits: there is nothing to save in them.

    The lists are gathered in Python on every step, about a microsecond per tensor (480 tensors: 445 us to issue, whatever their
    size); recorded in a CUDA graph a step takes what its kernels take.  States are made at the first step, and a count of its
    own when a parameter has no gradient in some step: both before a step is recorded."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, seed: int = 0):
        if lr < 0 or eps < 0 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1 or weight_decay < 0:
            raise ValueError("FusedAdamW: invalid hyper-parameter")
        if state_bits not in (8, 32):
            raise ValueError("FusedAdamW: state_bits must be 8 or 32")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, seed=seed))

    @staticmethod
    def _not_recorded(device):
        """What is made while a stream is captured is made again, as it was, at every replay."""
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: take one step with the gradients of the recorded one before it is recorded "
                               "(states and step counts must exist by then)")

    def _new_state(self, p, bits):
        self._not_recorded(p.device)
        st, n = {}, p.numel()
        kind = torch.uint8 if bits == 8 and n > _lib.ADAMW_BLOCK else torch.float32
        for name in ("exp_avg", "exp_avg_sq"):
            st[name] = torch.zeros(p.shape, dtype=kind, device=p.device)
            if kind == torch.uint8:
                st[name + "_scale"] = torch.zeros(-(-n // _lib.ADAMW_BLOCK), dtype=torch.float32, device=p.device)
        if p.dtype == torch.bfloat16:
            st["master"] = p.detach().to(torch.float32, memory_format=torch.contiguous_format)
        return st

    def _together(self, group):
        """The group's parameters that have a gradient, as lists that one launch updates: of one device and type, and of one
        step count -- parameters that have always been updated together share the tensor that holds it."""
        fresh, launches, members = {}, {}, {}
        for p in group["params"]:
            st = self.state[p] if p.grad is not None else self.state.get(p)
            if p.grad is not None and not st:
                st.update(self._new_state(p, group["state_bits"]))
                key = (p.device, p.dtype, st["exp_avg"].dtype)
                if key not in fresh:
                    fresh[key] = torch.zeros(2, dtype=torch.int64, device=p.device)
                st["step"] = fresh[key]
            if not st:
                continue
            members[id(st["step"])] = members.get(id(st["step"]), 0) + 1
            if p.grad is not None:
                launches.setdefault(id(st["step"]), []).append(p)
        for key, ps in launches.items():
            if len(ps) < members[key]:  # the others keep the old count
                self._not_recorded(ps[0].device)
                step = self.state[ps[0]]["step"].clone()
                for p in ps:
                    self.state[p]["step"] = step
        return launches.values()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        number = 0  # of the 8-bit list within the step: each rounds by random bits of its own
        for group in self.param_groups:
            for ps in self._together(group):
                st = [self.state[p] for p in ps]
                of = lambda name: [x[name] for x in st]  # noqa: E731
                eight = st[0]["exp_avg"].dtype == torch.uint8
                adamw_step(ps, [p.grad for p in ps], of("exp_avg"), of("exp_avg_sq"), st[0]["step"], lr=group["lr"],
                           betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                           masters=of("master") if "master" in st[0] else None, follow="master" in st[0],
                           scales=(of("exp_avg_scale"), of("exp_avg_sq_scale")) if eight else None,
                           seed=group["seed"] + number * 0x632BE5AB)
                number += eight
        return loss

    def moments(self, p):
        """(exp_avg, exp_avg_sq) of a parameter as float32 tensors, whatever they are held in."""
        st = self.state[p]
        if st["exp_avg"].dtype != torch.uint8:
            return st["exp_avg"], st["exp_avg_sq"]
        m, v = adamw_moments([st["exp_avg"]], [st["exp_avg_sq"]], ([st["exp_avg_scale"]], [st["exp_avg_sq_scale"]]))
        return m[0], v[0]

    def steps_taken(self) -> int:
        """Reads the largest step count back (synchronises)."""
        return max((int(st["step"][0].item()) for st in self.state.values()), default=0)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # The base class casts states to the parameter's type: here their types are their own.
        saved = {i: st for i, st in state_dict["state"].items()}
        order = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        shared = {}
        for i, p in zip(order, params):
            if i not in saved:
                continue
            st = {k: v.detach().to(p.device, copy=True) for k, v in saved[i].items()}
            # Equal counts are shared again, within what one launch updates.
            group = next(n for n, g in enumerate(self.param_groups) if any(q is p for q in g["params"]))
            key = (group, p.device, p.dtype, st["exp_avg"].dtype, int(st["step"][0].item()))
            st["step"] = shared.setdefault(key, st["step"])
            self.state[p] = st

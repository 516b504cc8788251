"""AdamW as one kernel over all tensors of a group, with moments of 32 or 8 bits.

The reference's recipes configure ``torch.optim.AdamW(fused=True)`` (``recipes/configs/llama3_1/8B_qlora_single_device.yaml:60-64``)
or, to save memory, an optimizer of a third package with 8-bit states.  :class:`AdamW` stands in for either.
"""
from __future__ import annotations

import threading
from typing import Dict, List, Tuple

import torch

from .. import _host


def _order(t: torch.Tensor) -> List[int]:
    """The dimensions of more than one element, from the slowest to the fastest in memory."""
    return sorted((d for d in range(t.dim()) if t.shape[d] > 1), key=lambda d: -t.stride(d))


def _order_of_states(p: torch.Tensor) -> List[int]:
    """That of a parameter's states: as it lies itself, or row by row if it has gaps."""
    order, step = _order(p), 1
    for d in reversed(order):
        if p.stride(d) != step:
            return sorted(order)
        step *= p.shape[d]
    return order


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` (decoupled weight decay) for parameters on the GPU, bfloat16 or float32.

    A step is ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
    ``p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)``, in fp32 whatever the parameters' type, one pass over
    all of them.  The moments are held in fp32 or, with ``state_bits=8``, in a byte each and two bytes of exponents for 128
    elements (a quarter of the memory): the first with a sign, 4 bits of exponent and 3 of mantissa, the second with 4 and 4.
    They are rounded stochastically, since a change of ``1 - b2`` in a step is smaller than what rounding to the nearest would
    let through; the numbers are a function of ``seed``, the step, the parameter's place and the element's, so that a run can be
    repeated and continued.  A gradient that is not finite makes its element NaN for good, as in 32 bits; with 8 bits the 127
    others of its block lose their moments and stand still.  In 8 bits a block spans about 2^15: below that part of its block's largest a
    first moment is held as 0 and a second one, which goes with the gradients' squares, as that part, so that an element with so much
    smaller gradients than its neighbours' moves less than with 32 bits.  ``eps`` counts as at least 1.1e-19, so that with ``eps=0`` an
    element that never had a gradient stands still.

    Args:
        params: parameters or groups, as for any ``torch.optim.Optimizer``
        lr (float): learning rate. Default: 1e-3
        betas (Tuple[float, float]): decay of the moments. Default: (0.9, 0.999)
        eps (float): added to the denominator. Default: 1e-8
        weight_decay (float): Default: 1e-2
        state_bits (int): 32 or 8. Default: 32
        stochastic_rounding (bool): round bfloat16 parameters stochastically: updates of less than half a step of the format are
            then kept on average, as they would be with a float32 copy. Default: False
        seed (int): of the stochastic rounding. Default: 0

    Every option may be a group's own.  Loading a state dict takes its options over, as for any optimizer, ``seed`` and
    ``stochastic_rounding`` among them, so that a run goes on with the numbers that it would have had; ``state_bits`` stays, and states
    of the other width are refused.

    ``state[p]`` holds ``step``, ``exp_avg``, ``exp_avg_sq`` (and ``exp_avg_exponent``, ``exp_avg_sq_exponent`` with 8 bits), made when ``p``
    first has a gradient; they are parts of buffers that all parameters share, so write into them, or load a state dict, but do not put
    other tensors in their place.  A parameter whose entry is taken out of ``state`` begins anew.  A parameter's memory
    may be replaced (``p.data = ..``) by one of the same size, type and order.  A state dict of ``torch.optim.AdamW`` can be loaded
    with 32 bits.  Parameters that share memory are refused where one launch would step both.  Calls of several threads wait for each
    other.  A step cannot be recorded into a graph.
    """

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 *, state_bits: int = 32, stochastic_rounding: bool = False, seed: int = 0) -> None:
        if isinstance(lr, torch.Tensor):
            raise TypeError("AdamW: lr must be a number, not a tensor")
        if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"AdamW: lr, eps and weight_decay must not be negative, got {lr}, {eps}, {weight_decay}")
        if not all(0.0 <= b < 1.0 for b in betas) or len(betas) != 2:
            raise ValueError(f"AdamW: betas must be two numbers in [0, 1), got {betas}")
        self._lock = threading.RLock()  # of the plans and the states' dictionary: calls of several threads wait for each other
        self._taken = None  # states on their way from a state dict
        self._forget()
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      stochastic_rounding=bool(stochastic_rounding), seed=int(seed)))

    def add_param_group(self, param_group) -> None:
        if isinstance(param_group, dict):  # else the base class refuses it
            self._check_bits(param_group.get("state_bits", self.defaults["state_bits"]))
        with self._lock:
            super().add_param_group(param_group)

    @staticmethod
    def _check_bits(bits) -> None:
        if bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {bits}")

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        if "_lock" not in self.__dict__:  # unpickled or copied
            self._lock = threading.RLock()
            self._taken = None
        self._forget()
        if self._taken is not None:  # a state dict is being loaded
            self.state.update(self._taken)
            for index in range(len(self.param_groups)):
                self._plan(index, checked=True)

    def _forget(self) -> None:
        self._plans: Dict[int, tuple] = {}
        self._owned: Dict[torch.Tensor, dict] = {}  # the entries of the dictionary of states that show theirs
        self._seen = (None, 0)  # that dictionary and its length when the plans were right

    def _look(self) -> None:
        state, length = self._seen
        if state is self.state and length == len(state):
            return
        state, owned = self.state, self._owned
        if any(state.get(p) is not own for p, own in owned.items()) or any(held and p not in owned for p, held in state.items()):
            self._forget()  # states were taken out, or put in
        self._seen = (state, len(state))

    def _plan(self, index: int, checked: bool = False):
        """The group's native side; a new one takes over the states that are there already."""
        self._look()
        group = self.param_groups[index]
        params, bits = group["params"], group["state_bits"]
        known = self._plans.get(index)
        if known is not None and known[1] == bits and known[0].holds(params):
            return known[0]
        self._check_bits(bits)
        if len({id(p) for p in params}) != len(params):
            raise ValueError("AdamW: a parameter occurs twice in a group")
        first = sum(len(g["params"]) for g in self.param_groups[:index])
        plan = _host.load().AdamWGroup(params, first, bits)
        given = [i for i, p in enumerate(params) if self.state.get(p)]
        if not checked:
            for i in given:
                self._check_states(self.state[params[i]], params[i], bits)
        plan.make(given)
        states = {}
        for i in given:
            held, own = self.state[params[i]], self._shown(plan, i)
            for name, tensor in own.items():
                if name == "step":
                    tensor.fill_(int(held[name]))
                else:
                    tensor.copy_(held[name].reshape(tensor.shape))
            states[params[i]] = own
        self.state.update(states)  # all of them or, after an error, none
        if index in self._plans:  # entries that were its own and are gone keep nothing alive
            self._owned = {p: own for p, own in self._owned.items() if self.state.get(p) is own}
        self._owned.update(states)
        self._plans[index] = (plan, bits)
        self._seen = (self.state, len(self.state))
        return plan

    @staticmethod
    def _shown(plan, i: int) -> dict:
        return dict(zip(("step", "exp_avg", "exp_avg_sq", "exp_avg_exponent", "exp_avg_sq_exponent"), plan.state(i)))

    def step(self, closure=None):
        """One step; with ``closure``, which computes the loss again, its value is returned.  A step that is refused for one
        parameter or group changes none."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        with self._lock:
            self._step()
        return loss

    def _step(self) -> None:
        self._look()
        steps = []
        for index, group in enumerate(self.param_groups):
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("AdamW: amsgrad and maximize are not supported")
            params = group["params"]
            plan, bits = self._plans.get(index, (None, 0))
            fresh = plan.fresh(params) if bits == group["state_bits"] else None
            if fresh is None:  # no native side for these parameters and options
                plan = self._plan(index)
                fresh = plan.fresh(params)
            if fresh:
                plan.make(fresh)
                for i in fresh:
                    self.state[params[i]] = self._owned[params[i]] = self._shown(plan, i)
                self._seen = (self.state, len(self.state))
            beta1, beta2 = group["betas"]
            steps.append((plan, float(group["lr"]), beta1, beta2, group["eps"], group["weight_decay"], group["seed"], group["stochastic_rounding"]))
        native = _host.load().adamw_step
        native(*steps[0]) if len(steps) == 1 else native(steps)

    def moments(self):
        """``(exp_avg, exp_avg_sq)`` of all parameters that have states, one after another in their order (a parameter's elements as
        they lie in memory), as two flat tensors of numbers: the fp32 states themselves where they lie that way already, bfloat16
        (exact) for 8-bit states."""
        firsts, seconds = [], []
        with self._lock:
            for index in range(len(self.param_groups)):
                plan = self._plan(index)
                whole = plan.whole()
                for m, v in plan.moments() if whole is None else [whole]:
                    firsts.append(m)
                    seconds.append(v)
        if not firsts:
            raise RuntimeError("AdamW.moments: no parameter has taken a step yet")
        return (firsts[0], seconds[0]) if len(firsts) == 1 else (torch.cat(firsts), torch.cat(seconds))

    def state_dict(self):
        with self._lock:
            return super().state_dict()

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """What :meth:`state_dict` gave, of an optimizer with as many bits.  With 8 bits the parameters have to lie in memory in the order in
        which those of the saved states lay (of dense ones the states have the strides), since neighbours there share exponents."""
        with self._lock:
            # last of the hooks that see the dictionary before it is loaded
            hook = self.register_load_state_dict_pre_hook(AdamW._take)
            try:
                super().load_state_dict(state_dict)
            finally:
                hook.remove()
                self._taken = None

    def _take(self, state_dict):
        """The states, checked; the base class, which would cast them to the parameters' type, gets the groups alone."""
        saved, groups = state_dict["state"], state_dict["param_groups"]
        self._taken = {}
        if [len(g["params"]) for g in groups] == [len(g["params"]) for g in self.param_groups]:  # else the base class refuses it
            for theirs, ours in zip(groups, self.param_groups):
                for key, p in zip(theirs["params"], ours["params"]):
                    if key in saved:
                        self._check_states(saved[key], p, ours["state_bits"])
                        self._taken[p] = dict(saved[key])
            # the width stays; another AdamW's groups have no such options
            groups = [{"stochastic_rounding": ours["stochastic_rounding"], "seed": ours["seed"], **theirs, "state_bits": ours["state_bits"]}
                      for theirs, ours in zip(groups, self.param_groups)]
        return {**state_dict, "state": {}, "param_groups": groups}

    @staticmethod
    def _check_states(held, p, bits: int) -> None:
        eight = bits == 8
        names = {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_exponent", "exp_avg_sq_exponent"} if eight else set())
        if not names <= set(held):
            raise ValueError(f"AdamW: a state holds {sorted(held)}, expected {sorted(names)}")
        blocks = -(-p.numel() // 128)
        for name in names - {"step"}:
            t = held[name]
            if (t.dtype == torch.uint8) != eight:
                raise ValueError(f"AdamW: {name} is {t.dtype}, the states of this optimizer have {bits} bits")
            if t.numel() != (blocks if name.endswith("exponent") else p.numel()):
                raise ValueError(f"AdamW: {name} has {t.numel()} elements, the parameter {p.numel()}")
        if eight and not (p.is_contiguous() and held["exp_avg"].is_contiguous() and held["exp_avg_sq"].is_contiguous()):
            AdamW._check_order(held, p)

    @staticmethod
    def _check_order(held, p) -> None:
        """8 bits: the exponents are those of neighbours in memory, so codes in another order would meet others' exponents."""
        want = _order_of_states(p)
        for name in ("exp_avg", "exp_avg_sq"):
            t = held[name]
            have = _order(t)
            same = have == want if t.shape == p.shape else have == sorted(have) and want == sorted(want)
            if p.numel() and not same:
                raise ValueError(f"AdamW: the 8-bit {name} {tuple(t.shape)} of strides {t.stride()} lies in another order than its parameter "
                                 f"{tuple(p.shape)} of strides {p.stride()}")

"""AdamW over many tensors at once, with the moments in float32 or in 8 bits and the parameters in float32 or in
bfloat16.

`adamw_step` is one step over lists of tensors that the caller keeps; `FusedAdamW` is the optimizer around it, with
torch.optim.AdamW's parameter groups, state and state_dict (beside fdgs.adam.FusedAdam, which is plain Adam);
`pack8` / `unpack8` turn float32 moments into 8-bit ones and back.

8-bit moments take a quarter of the memory (2,000,000 Gaussians: 944 MB of moments become 239 MB) and of the bytes
that the step and the densification surgery move for them.  Their format and rounding are described in
include/fdgs.h.  bfloat16 parameters keep the 16 bits that bfloat16 drops in `residual`: parameter and residual
together are the float32 weight, so updates smaller than a bfloat16 step add up instead of vanishing, and a parameter
that is written from outside (a checkpoint, a mask) simply is the new weight, up to half a bfloat16 step."""
from typing import NamedTuple

import torch

from . import _host, _lib, _records
from .adam import GENERATION

BLOCK = _records.MOMENT8_BLOCK


class Moment8(NamedTuple):
    """A moment in 8 bits: one code per element, one exponent per block of 256 elements.  signed: a first moment."""
    codes: torch.Tensor
    exponents: torch.Tensor
    signed: bool

    @staticmethod
    def zeros_like(p, signed):
        return Moment8(torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.contiguous_format),
                       torch.zeros(-(-p.numel() // BLOCK), dtype=torch.uint8, device=p.device), signed)


def _each(value, n, what):
    if isinstance(value, (list, tuple)):
        if len(value) != n:
            raise ValueError(f"{what}: one value, or one for each of the {n} tensors")
        return value
    return [value] * n


def round_key(seed, index, step):
    """A 32-bit key for tensor `index` at `step`: what the rounding of its 8-bit moments is drawn with."""
    x = (seed * 0x9E3779B9 + index * 0xBB67AE85 + step * 0x6A09E667) & 0xFFFFFFFF
    x ^= x >> 15
    x = (x * 0x9E3779B9) & 0xFFFFFFFF
    return x ^ (x >> 16)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, steps, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               residuals=None, keys=None):
    """One AdamW step over lists of tensors, in place: params, their moments (contiguous float32 tensors, or Moment8),
    and for bfloat16 params `residuals` (int16), each of its parameter's shape or flat.  grads: the parameters' type and shape;
    contiguous, or column slices of wider row-major arrays (read in place), anything else is copied.  steps (1-based), lr
    and weight_decay: one value, or one for each tensor.  keys: for 8-bit moments, 32-bit numbers, one for each tensor,
    others at every step.  All tensors are on one GPU, have one type, and the step runs on its current stream; no tensor
    that it writes overlaps another one.  Tensors without elements are passed over.  The call reads steps, lr and keys on
    the host: a captured graph would replay the ones it was captured with, so a stream that is being captured is
    refused."""
    _host.adamw_step(params, grads, exp_avgs, exp_avg_sqs, residuals, steps, lr, weight_decay, keys, Moment8, *betas, eps)
    GENERATION[0] += 1


def unpack8(moments, dtype=torch.float32, out=None):
    """The values that a list of Moment8 stands for: float32 or bfloat16 tensors (both exact) of the codes' shapes,
    written into `out` (a list of contiguous tensors of one type, of the codes' shapes or flat, none of which
    overlaps another or the moments) where it is given."""
    moments = list(moments)
    if not moments:
        return []
    if out is None:
        out = [torch.empty(x.codes.shape, dtype=dtype, device=x.codes.device) for x in moments]
    _host.moment8(False, moments, out, None, Moment8)
    return list(out)


@torch.no_grad()
def pack8(values, signed, keys=None):
    """8-bit moments of a list of float32 tensors (signed: first moments; a bool, or one for each): to the nearest, or
    with the random numbers of `keys` (one for each)."""
    values = list(values)
    if not values:
        return []
    signed = _each(signed, len(values), "signed")
    device = values[0].device
    _lib.require_gpu(values[0])
    values = [t.resolve_neg().contiguous() for t in values]
    out = []
    for t, s in zip(values, signed):
        if t.dtype is not torch.float32 or t.device != device:
            raise ValueError("pack8 takes float32 tensors on one device")
        out.append(Moment8(torch.empty_like(t, dtype=torch.uint8),
                           torch.empty(-(-t.numel() // BLOCK), dtype=torch.uint8, device=device), bool(s)))
    _host.moment8(True, out, values, keys, Moment8)
    return out


class FusedAdamW:
    """AdamW with the surface of torch.optim.AdamW that fdgs.adam.FusedAdam has: parameter groups (dicts with `params`,
    `lr`, `weight_decay` and any other key; or a plain list of tensors), `step()`, `zero_grad()`, `state`, `state_dict()` and
    `load_state_dict()`; learning rates are read at every step.  A tensor without a gradient is skipped, and every tensor
    counts its own steps.

    state_bits 8 keeps both moments as Moment8 (state[p]["exp_avg"], ["exp_avg_sq"]); bfloat16 parameters have
    state[p]["residual"] beside them.  seed: of the 8-bit moments' rounding; replicas of a model have to have the same one
    (and the same order of parameters) to stay the same.  state_dict() holds tensors only, with the keys of
    torch.optim.AdamW where moments are in 32 bits; load_state_dict() takes a state in either width and converts it, also one
    of torch.optim.Adam (without weight decay, which means another thing there) or FusedAdam."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("state_bits is 8 or 32")
        self.state_bits, self.seed = state_bits, int(seed)
        params = list(params)
        if params and not isinstance(params[0], dict):
            params = [{"params": params}]
        self.param_groups = []
        for grp in params:
            g = dict(grp)
            g["params"] = list(g["params"])
            for k, v in (("lr", lr), ("betas", betas), ("eps", eps), ("weight_decay", weight_decay), ("amsgrad", False),
                         ("maximize", False), ("foreach", None), ("capturable", False), ("differentiable", False),
                         ("fused", None), ("decoupled_weight_decay", True)):
                g.setdefault(k, v)
            self.param_groups.append(g)
        self._check_groups(self.param_groups)
        seen = [p for g in self.param_groups for p in g["params"]]
        if len({id(p) for p in seen}) != len(seen):
            raise ValueError("a tensor is in the parameter groups twice")
        self.state = {}

    @staticmethod
    def _check_groups(groups):
        for g in groups:
            if g["amsgrad"] or g["maximize"] or not g["decoupled_weight_decay"]:
                raise ValueError("FusedAdamW implements decoupled weight decay, without amsgrad and maximize")
            if not (0 <= g["betas"][0] < 1 and 0 <= g["betas"][1] < 1 and g["eps"] >= 0):
                raise ValueError("betas are in [0, 1), eps is not negative")

    def zero_grad(self, set_to_none=True):
        for g in self.param_groups:
            for p in g["params"]:
                if set_to_none:
                    p.grad = None
                elif p.grad is not None:
                    p.grad.zero_()

    def _new_state(self, p):
        if p.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"FusedAdamW takes float32 and bfloat16 parameters, not {p.dtype}")
        zeros = lambda dtype: torch.zeros_like(p, dtype=dtype, memory_format=torch.contiguous_format)  # noqa: E731
        st = {"step": 0}
        if self.state_bits == 8:
            st["exp_avg"], st["exp_avg_sq"] = Moment8.zeros_like(p, True), Moment8.zeros_like(p, False)
        else:
            st["exp_avg"], st["exp_avg_sq"] = zeros(torch.float32), zeros(torch.float32)
        if p.dtype is torch.bfloat16:
            st["residual"] = zeros(torch.int16)
        return st

    def _fits(self, st, p):
        if st is None or "exp_avg" not in st:
            return False
        m = st["exp_avg"]
        return (m.codes if isinstance(m, Moment8) else m).shape == p.shape

    @torch.no_grad()
    def step(self):
        # one call for the tensors that share what a call has one of: type, device, betas and eps
        calls, index = {}, -1
        for g in self.param_groups:
            betas, eps, lr, wd = tuple(g["betas"]), g["eps"], g["lr"], g["weight_decay"]
            for p in g["params"]:
                index += 1
                grad = p.grad
                if grad is None:
                    continue
                if not p.is_cuda:
                    raise RuntimeError("libfdgs kernels run on the GPU only; got a tensor on " + str(p.device))
                st = self.state.get(p)
                if not self._fits(st, p):
                    st = self.state[p] = self._new_state(p)
                call = calls.get((p.dtype, p.device, betas, eps))
                if call is None:
                    call = calls[(p.dtype, p.device, betas, eps)] = ([], [], [], [], [], [], [], [], [], [])
                ps, gs, ms, vs, steps, lrs, wds, low, keys, states = call
                ps.append(p)
                gs.append(grad)
                ms.append(st["exp_avg"])
                vs.append(st["exp_avg_sq"])
                t = int(st["step"]) + 1
                steps.append(t)
                lrs.append(lr)
                wds.append(wd)
                states.append(st)
                if p.dtype is torch.bfloat16:
                    low.append(st["residual"])
                if self.state_bits == 8:
                    keys.append(round_key(self.seed, index, t))
        for (_, _, betas, eps), (ps, gs, ms, vs, steps, lrs, wds, low, keys, states) in calls.items():
            adamw_step(ps, gs, ms, vs, steps=steps, lr=lrs, betas=betas, eps=eps, weight_decay=wds, residuals=low or None,
                       keys=keys or None)
            for st, t in zip(states, steps):
                st["step"] = t

    # -- what the densification surgery (fdgs.densify) moves and puts back -----------------------------------------------
    def moments(self, p):
        """The moments of p as float32 tensors of its shape, or None where it has none yet."""
        st = self.state.get(p)
        if not self._fits(st, p):
            return None
        if "residual" in st:
            raise ValueError("the surgery moves float32 parameters")
        if self.state_bits == 8:
            return tuple(unpack8([st["exp_avg"], st["exp_avg_sq"]]))
        return st["exp_avg"], st["exp_avg_sq"]

    def set_moments(self, st, exp_avg, exp_avg_sq):
        """Puts float32 moments (the surgery's result) into the state `st`, to the nearest where they are kept in 8 bits:
        what comes from 8 bits lies on their grid and stays as it is, unless its new block of 256 has a largest value so
        much larger that it falls below that block's smallest code."""
        if self.state_bits == 8:
            exp_avg, exp_avg_sq = pack8([exp_avg, exp_avg_sq], [True, False])
        st["exp_avg"], st["exp_avg_sq"] = exp_avg, exp_avg_sq

    # -- torch.optim.Optimizer's serialisation layout ---------------------------------------------------------------------
    def state_dict(self):
        index, groups = {}, []
        for g in self.param_groups:
            ids = []
            for p in g["params"]:
                index[id(p)] = len(index)
                ids.append(index[id(p)])
            groups.append({**{k: v for k, v in g.items() if k != "params"}, "params": ids})
        state = {}
        for p, st in self.state.items():
            if id(p) not in index:
                continue
            out = {"step": torch.tensor(float(st["step"]))}
            for k in ("exp_avg", "exp_avg_sq"):
                if isinstance(st[k], Moment8):
                    out[k + "_codes"], out[k + "_exponents"] = st[k].codes, st[k].exponents
                else:
                    out[k] = st[k]
            if "residual" in st:
                out["residual"] = st["residual"]
            state[index[id(p)]] = out
        return {"state": state, "param_groups": groups}

    @torch.no_grad()
    def load_state_dict(self, sd):
        groups = sd["param_groups"]
        if len(groups) != len(self.param_groups) or any(len(a["params"]) != len(b["params"])
                                                        for a, b in zip(groups, self.param_groups)):
            raise ValueError("loaded state dict has different parameter groups")
        merged, by_index = [], {}
        for saved, g in zip(groups, self.param_groups):
            merged.append({**g, **{k: v for k, v in saved.items() if k not in ("params", "decoupled_weight_decay")}})
            for i, p in zip(saved["params"], g["params"]):
                by_index[int(i)] = p
        self._check_groups(merged)
        if any(saved.get("weight_decay") and saved.get("decoupled_weight_decay") is False for saved in groups):
            raise ValueError("the loaded state's weight decay is part of the gradient (torch.optim.Adam's), this optimizer's is not")
        state = {by_index[int(i)]: self._loaded(by_index[int(i)], st) for i, st in sd["state"].items()}
        for g, m in zip(self.param_groups, merged):
            g.update(m)
        self.state = state
        GENERATION[0] += 1

    def _loaded(self, p, saved):
        st = self._new_state(p)
        st["step"] = int(round(float(saved["step"])))
        if "residual" in st and "residual" in saved:
            st["residual"].copy_(saved["residual"].view(p.shape))
        for k, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            if k in saved:
                x = saved[k].to(device=p.device, dtype=torch.float32).reshape(p.shape).contiguous().clone()
                st[k] = pack8([x], signed)[0] if self.state_bits == 8 else x
            else:
                x = Moment8(saved[k + "_codes"].to(p.device).reshape(p.shape).contiguous().clone(),
                            saved[k + "_exponents"].to(p.device).contiguous().clone(), signed)
                if x.exponents.numel() != blocks_of(p):
                    raise ValueError("loaded 8-bit moments have another number of blocks")
                st[k] = x if self.state_bits == 8 else unpack8([x])[0]
        return st


def blocks_of(p):
    """Blocks, and so exponents, of an 8-bit moment of p."""
    return -(-p.numel() // BLOCK)

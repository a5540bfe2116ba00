"""AdamW over many tensors at once, with the moments in float32 or in 8 bits and the parameters in float32 or in
bfloat16.

`adamw_step` is one step over lists of tensors that the caller keeps; `FusedAdamW` is the optimizer around it, with
torch.optim.AdamW's parameter groups, state and state_dict (beside fdgs.adam.FusedAdam, which is plain Adam);
`pack8` / `unpack8` turn float32 moments into 8-bit ones and back.

8-bit moments take a quarter of the memory (2,000,000 Gaussians: 944 MB of moments become 239 MB) and of the bytes
that the step and the densification surgery move for them.  Their format and rounding are described in
include/fdgs.h.  bfloat16 parameters keep the 16 bits that bfloat16 drops in `residual`: parameter and residual
together are the float32 weight, so updates smaller than a bfloat16 step add up instead of vanishing, and a parameter
that is written from outside (a checkpoint) simply is the new weight, up to half a bfloat16 step."""
from typing import NamedTuple

import torch

from . import _lib, _records
from .adam import GENERATION, _row_slice

BLOCK = _records.MOMENT8_BLOCK
_TYPES = {torch.float32: _records.TYPE_F32, torch.bfloat16: _records.TYPE_BF16}


class Moment8(NamedTuple):
    """A moment in 8 bits: one code per element, one exponent per block of 256 elements.  signed: a first moment."""
    codes: torch.Tensor
    exponents: torch.Tensor
    signed: bool

    @staticmethod
    def zeros_like(p, signed):
        return Moment8(torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.contiguous_format),
                       torch.zeros(-(-p.numel() // BLOCK), dtype=torch.uint8, device=p.device), signed)


def _check_moment8(x, like, signed, what):
    if not isinstance(x, Moment8):
        raise ValueError(f"{what}: an 8-bit moment is an adamw.Moment8; do not mix moments in 8 and in 32 bits")
    c, e = x.codes, x.exponents
    if c.dtype is not torch.uint8 or e.dtype is not torch.uint8 or not c.is_contiguous() or not e.is_contiguous():
        raise ValueError(f"{what}: codes and exponents are contiguous uint8 tensors")
    if c.numel() != like.numel() or e.numel() != -(-like.numel() // BLOCK) or bool(x.signed) != signed:
        raise ValueError(f"{what}: one code per element, one exponent per {BLOCK} elements, signed for the first moment only")
    if c.device != like.device or e.device != like.device:
        raise ValueError(f"{what}: every tensor of a step is on one device")


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


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, steps, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               residuals=None, keys=None):
    """One AdamW step over lists of tensors, in place: params, their moments (contiguous float32 tensors, or Moment8),
    and for bfloat16 params `residuals` (int16).  grads: the parameters' type; contiguous, or column slices of wider
    row-major arrays (read in place), anything else is copied.  steps (1-based), lr and weight_decay: one value, or
    one for each tensor.  keys: for 8-bit moments, 32-bit numbers, one for each tensor, others at every step.
    All tensors are on one GPU, have one type, do not overlap, and the step runs on its current stream.  Tensors
    without elements are passed over.  The call reads steps, lr and keys on the host: a captured graph would replay
    the ones it was captured with, so a stream that is being captured is refused."""
    n = len(params)
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n):
        raise ValueError("params, grads and moments have to be lists of the same length")
    if n == 0:
        return
    steps, lrs, wds = _each(steps, n, "steps"), _each(lr, n, "lr"), _each(weight_decay, n, "weight_decay")
    dtype, device = params[0].dtype, params[0].device
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"adamw_step takes float32 and bfloat16 parameters, not {dtype}")
    bf16 = kind == _records.TYPE_BF16
    if not params[0].is_cuda:
        raise RuntimeError("libfdgs kernels run on the GPU only; got a tensor on " + str(device))
    if bf16 and (residuals is None or len(residuals) != n):
        raise ValueError("bfloat16 parameters need residuals: an int16 tensor for each")
    eight = isinstance(exp_avgs[0], Moment8)
    if eight and (keys is None or len(keys) != n):
        raise ValueError("8-bit moments need keys: a number for each tensor, others at every step")
    fields, seen, hold = [], set(), []
    for i in range(n):
        p, g, m, v = params[i], grads[i], exp_avgs[i], exp_avg_sqs[i]
        numel = p.numel()
        if p.dtype is not dtype or g.dtype is not dtype:
            raise ValueError(f"parameters and gradients of one step have one type: {dtype}, {p.dtype} and {g.dtype} given")
        if g.numel() != numel or not p.is_contiguous():
            raise ValueError("a parameter has to be contiguous, and its gradient of its size")
        if p.device != device or g.device != device:
            raise ValueError("every tensor of a step is on one device")
        row, stride = 0, 0
        if not g.is_contiguous():
            rs = _row_slice(g)                   # a column slice of a wider array is read in place
            if rs is None:
                g = g.contiguous()
                hold.append(g)
            else:
                row, stride = rs
        low = me = ve = 0
        if eight:
            _check_moment8(m, p, True, "exp_avgs")
            _check_moment8(v, p, False, "exp_avg_sqs")
            me, ve, m, v = m.exponents.data_ptr(), v.exponents.data_ptr(), m.codes, v.codes
        else:
            for x in (m, v):
                if isinstance(x, Moment8) or x.dtype is not torch.float32 or x.numel() != numel or not x.is_contiguous() \
                        or x.device != device:
                    raise ValueError("moments are contiguous float32 tensors of the parameter's size on its device, or "
                                     "all of them Moment8")
        if bf16:
            r = residuals[i]
            if r.dtype is not torch.int16 or r.numel() != numel or not r.is_contiguous() or r.device != device:
                raise ValueError("a residual is a contiguous int16 tensor of the parameter's size on its device")
            low = r.data_ptr()
        step = int(steps[i])
        if not 1 <= step <= 0x7FFFFFFF:
            raise ValueError("steps count from 1")
        pp, mp, vp = p.data_ptr(), m.data_ptr(), v.data_ptr()
        if numel:
            if pp in seen or mp in seen or vp in seen:
                raise ValueError("a tensor is in the lists twice")
            seen.update((pp, mp, vp))
        fields += (pp, g.data_ptr(), mp, vp, low, me, ve, numel, stride, row, step, float(lrs[i]), float(wds[i]),
                   (int(keys[i]) & 0xFFFFFFFF) if eight else 0, 0)
    _no_capture(device, "adamw_step")
    records = _records.pack(_records.ADAMW_TENSOR, n, fields)
    b1, b2 = betas
    _lib.call_on(device, "fdgs_adamw_step", _records.AdamWArgs(n, kind, 8 if eight else 32, 0, b1, b2, eps, records))
    GENERATION[0] += 1


def _no_capture(device, what):
    if device.index == torch.cuda.current_device():
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(device):
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError(f"{what} reads its step counts on the host and cannot be captured into a graph")


def _moment8_call(name, moments, values, value_type, nearest, keys):
    fields = []
    for i, (x, t) in enumerate(zip(moments, values)):
        fields += (x.codes.data_ptr(), x.exponents.data_ptr(), t.data_ptr(), t.numel(), 1 if x.signed else 0,
                   int(keys[i]) & 0xFFFFFFFF if keys is not None else 0)
    records = _records.pack(_records.MOMENT8_TENSOR, len(moments), fields)
    _lib.call_on(values[0].device, name, _records.Moment8Args(len(moments), value_type, 1 if nearest else 0, 0, records))


@torch.no_grad()
def unpack8(moments, dtype=torch.float32, out=None):
    """The values that a list of Moment8 stands for: float32 or bfloat16 tensors (both exact) of the codes' shapes,
    written into `out` (a list of contiguous tensors of one type) where it is given."""
    moments = list(moments)
    if not moments:
        return []
    if out is None:
        out = [torch.empty(x.codes.shape, dtype=dtype, device=x.codes.device) for x in moments]
    if len(out) != len(moments):
        raise ValueError("out has to have a tensor for each moment")
    dtype, device = out[0].dtype, out[0].device
    if dtype not in _TYPES:
        raise ValueError("unpack8 writes float32 or bfloat16")
    _lib.require_gpu(out[0])
    for x, t in zip(moments, out):
        _check_moment8(x, t, bool(x.signed), "moments")
        if t.dtype is not dtype or t.device != device or not t.is_contiguous():
            raise ValueError("the values go to contiguous tensors of one type on one device")
    _moment8_call("fdgs_moment8_unpack", moments, out, _TYPES[dtype], False, None)
    return list(out)


@torch.no_grad()
def pack8(values, signed, keys=None):
    """8-bit moments of a list of float32 tensors (signed: first moments; a bool, or one for each): to the nearest, or
    with the random numbers of `keys` (one for each)."""
    values = list(values)
    if not values:
        return []
    signed = _each(signed, len(values), "signed")
    if keys is not None and len(keys) != len(values):
        raise ValueError("keys has to have a number for each tensor")
    device = values[0].device
    _lib.require_gpu(values[0])
    values = [t.contiguous() for t in values]
    out = []
    for t, s in zip(values, signed):
        if t.dtype is not torch.float32 or t.device != device:
            raise ValueError("pack8 takes float32 tensors on one device")
        out.append(Moment8(torch.empty_like(t, dtype=torch.uint8),
                           torch.empty(-(-t.numel() // BLOCK), dtype=torch.uint8, device=device), bool(s)))
    _moment8_call("fdgs_moment8_pack", out, values, _records.TYPE_F32, keys is None, keys)
    return out

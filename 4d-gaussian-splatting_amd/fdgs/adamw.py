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
    and for bfloat16 params `residuals` (int16).  grads: the parameters' type; contiguous, or column slices of wider
    row-major arrays (read in place), anything else is copied.  steps (1-based), lr and weight_decay: one value, or
    one for each tensor.  keys: for 8-bit moments, 32-bit numbers, one for each tensor, others at every step.
    All tensors are on one GPU, have one type, do not overlap, and the step runs on its current stream.  Tensors
    without elements are passed over.  The call reads steps, lr and keys on the host: a captured graph would replay
    the ones it was captured with, so a stream that is being captured is refused."""
    if not len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs):
        raise ValueError("params, grads and moments have to be lists of the same length")
    if not len(params):
        return
    device = params[0].device
    if device.type == "cuda":
        _no_capture(device, "adamw_step")
    records, kind, bits, hold = _host.adamw_records(params, grads, exp_avgs, exp_avg_sqs, residuals, steps, lr, weight_decay,
                                                    keys, Moment8)
    b1, b2 = betas
    _lib.call_on(device, "fdgs_adamw_step", _records.AdamWArgs(len(params), kind, bits, 0, b1, b2, eps, records))
    GENERATION[0] += 1
    del hold                                     # copies of gradients: kept until the kernels were on the stream


def _no_capture(device, what):
    if device.index == torch.cuda.current_device():
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(device):
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError(f"{what} reads its step counts on the host and cannot be captured into a graph")


def _moment8_call(name, moments, values, nearest, keys):
    records, kind = _host.moment8_records(moments, values, keys, Moment8)
    _lib.call_on(values[0].device, name, _records.Moment8Args(len(moments), kind, 1 if nearest else 0, 0, records))


def unpack8(moments, dtype=torch.float32, out=None):
    """The values that a list of Moment8 stands for: float32 or bfloat16 tensors (both exact) of the codes' shapes,
    written into `out` (a list of contiguous tensors of one type) where it is given."""
    moments = list(moments)
    if not moments:
        return []
    if out is None:
        out = [torch.empty(x.codes.shape, dtype=dtype, device=x.codes.device) for x in moments]
    _moment8_call("fdgs_moment8_unpack", moments, out, False, None)
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
    values = [t.contiguous() for t in values]
    out = []
    for t, s in zip(values, signed):
        if t.dtype is not torch.float32 or t.device != device:
            raise ValueError("pack8 takes float32 tensors on one device")
        out.append(Moment8(torch.empty_like(t, dtype=torch.uint8),
                           torch.empty(-(-t.numel() // BLOCK), dtype=torch.uint8, device=device), bool(s)))
    _moment8_call("fdgs_moment8_pack", out, values, keys is None, keys)
    return out

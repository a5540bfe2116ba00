"""Table lookup with scaling, and its gradient by sorted tokens.

`embedding(ids, table, scale)` is scale * table[ids] with a gradient for the table: float32, bfloat16 or float16
tables of any width, int32 or int64 ids of any shape, padded batches.  `embedding_grad` is that gradient alone, and
`FeatureCodebook` a module around both for Gaussians whose SH coefficients come from a shared table: one id per
Gaussian and V rows of [16, 3] instead of 48 floats each (fdgs.renderer.render takes a model with a
`feature_codebook`)."""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib, _records
from ._lib import lib

_TYPES = {torch.float32: _records.TYPE_F32, torch.bfloat16: _records.TYPE_BF16, torch.float16: _records.TYPE_F16}
_IDS = {torch.int32: 4, torch.int64: 8}


def _ids(ids, device):
    if ids.dtype not in _IDS:
        raise ValueError(f"ids are int32 or int64, not {ids.dtype}")
    if ids.device != device:
        raise ValueError("ids and table have to be on one device")
    return ids if ids.is_contiguous() else ids.contiguous()


def _rows(t, lead):
    """(tensor, elements of a row, distance of the rows) of t [lead..., row...], copied where its rows are not contiguous
    runs a constant distance apart."""
    width = 1
    for d in t.shape[lead:]:
        width *= d
    if t.is_contiguous():
        return t, width, width
    row = t[(0,) * lead] if all(t.shape[:lead]) else t
    if lead == 1 and row.is_contiguous() and t.stride(0) >= 0:
        return t, width, t.stride(0)
    if lead > 1 and row.is_contiguous() and _one_stride(t, lead):
        return t, width, t.stride(lead - 1)
    return t.contiguous(), width, width


def _one_stride(t, lead):
    """Whether the leading dimensions are one run of rows a constant, not negative distance apart."""
    step = t.stride(lead - 1)
    if step < 0:
        return False
    for k in range(lead - 1):
        if t.shape[k] > 1 and t.stride(k) != t.stride(k + 1) * t.shape[k + 1]:
            return False
    return True


def _check_table(table):
    if table.dim() < 2 or table.dtype not in _TYPES:
        raise ValueError("the table is [rows, ...] in float32, bfloat16 or float16")


def _forward(ids, table, scale, padding_id):
    ids = _ids(ids, table.device)
    table, width, stride = _rows(table.detach(), 1)
    out = torch.empty(ids.shape + table.shape[1:], dtype=table.dtype, device=table.device)
    _lib.call_on(table.device, "fdgs_embedding_fwd", _records.EmbeddingFwdArgs(
        ids.numel(), table.shape[0], width, _TYPES[table.dtype], _IDS[ids.dtype], ids.data_ptr(), table.data_ptr(), stride,
        -1 if padding_id is None else padding_id, out.data_ptr(), scale))
    return out


@torch.no_grad()
def embedding_grad(grad_out, ids, num_rows, scale=1.0, padding_id=None):
    """The gradient of embedding() with respect to its table: [num_rows, ...] for grad_out [*ids.shape, ...], the sum
    of scale * grad_out over the tokens of each row, zeros for rows without one.  Sums are taken in float32 in an order
    that the ids alone decide."""
    if not grad_out.is_cuda:
        raise RuntimeError("libfdgs kernels run on the GPU only; got a tensor on " + str(grad_out.device))
    if grad_out.dtype not in _TYPES:
        raise ValueError("grad_out is float32, bfloat16 or float16")
    ids = _ids(ids, grad_out.device)
    lead = ids.dim()
    if tuple(grad_out.shape[:lead]) != tuple(ids.shape) or grad_out.dim() <= lead:
        raise ValueError("grad_out has to be [*ids.shape, ...]")
    if not 0 <= num_rows <= 0x7FFFFFFF:
        raise ValueError("num_rows is between 0 and 2^31 - 1")
    row_shape = grad_out.shape[lead:]
    if lead == 0:
        grad_out, lead = grad_out.unsqueeze(0), 1
    g, width, stride = _rows(grad_out, lead)
    grad_table = torch.empty((num_rows,) + tuple(row_shape), dtype=g.dtype, device=g.device)
    if num_rows == 0 or width == 0:
        return grad_table
    kind = _TYPES[g.dtype]
    size = lib.fdgs_embedding_bwd_workspace_bytes(ids.numel(), num_rows, width, kind)
    workspace = torch.empty(size, dtype=torch.uint8, device=g.device)
    _lib.call_on(g.device, "fdgs_embedding_bwd", _records.EmbeddingBwdArgs(
        ids.numel(), num_rows, width, kind, _IDS[ids.dtype], ids.data_ptr(), g.data_ptr(), stride,
        -1 if padding_id is None else padding_id, grad_table.data_ptr(), scale, workspace.data_ptr(), size))
    return grad_table


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding_id):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding_id = table.shape[0], scale, padding_id
        return _forward(ids, table, scale, padding_id)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        ids, = ctx.saved_tensors
        return embedding_grad(grad_out, ids, ctx.rows, ctx.scale, ctx.padding_id), None, None, None


def embedding(ids, table, scale=1.0, padding_id=None):
    """scale * table[ids]: ids [...] int32 or int64, table [V, ...] float32, bfloat16 or float16 (a slice of a wider
    table is read in place) -> [*ids.shape, *table.shape[1:]] in the table's type, rounded once.  Negative ids and
    `padding_id` give zeros and take no part in the gradient; an id of V or more - an error that only the GPU sees -
    gives a row of NaN.  The gradient of the table is dense, with the table's shape and type, and the same bits for the
    same inputs."""
    _check_table(table)
    if not table.is_cuda:
        raise RuntimeError("libfdgs kernels run on the GPU only; got a tensor on " + str(table.device))
    scale = float(scale)
    if padding_id is not None:
        padding_id = int(padding_id)
        if padding_id < 0:
            raise ValueError("padding_id is a row of the table; negative ids are padding always")
    if table.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(table, ids, scale, padding_id)
    return _forward(ids, table, scale, padding_id)


class FeatureCodebook(nn.Module):
    """SH coefficients of N Gaussians as rows of a shared table: `table` [V, 16, 3] (trained) and `ids` [N] (which row a
    Gaussian has).  Called without arguments it returns the [N, 16, 3] features; the gradient goes to the table."""

    def __init__(self, table, ids):
        super().__init__()
        _check_table(table)
        if ids.dim() != 1 or ids.dtype not in _IDS:
            raise ValueError("ids are one int32 or int64 number per Gaussian")
        self.table = nn.Parameter(table.detach().clone())
        self.register_buffer("ids", ids.detach().clone())

    def forward(self):
        return embedding(self.ids, self.table)

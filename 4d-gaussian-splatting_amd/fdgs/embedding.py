"""Table lookup with scaling, and its gradient by sorted tokens.

`embedding(ids, table, scale)` is scale * table[ids] with a gradient for the table: float32, bfloat16 or float16
tables of any width, int32 or int64 ids of any shape, padded batches.  `embedding_grad` is that gradient alone, and
`FeatureCodebook` a module around both for Gaussians whose SH coefficients come from a shared table: one id per
Gaussian and V rows of [16, 3] instead of 48 floats each (fdgs.renderer.render takes a model with a
`feature_codebook`)."""
import torch
from torch import nn

from . import _lib  # noqa: F401  (loads the library and gives it to _host)
from . import _host


def embedding(ids, table, scale=1.0, padding_id=None):
    """scale * table[ids]: ids [...] int32 or int64, table [V, ...] float32, bfloat16 or float16 (a slice of a wider
    table is read in place) -> [*ids.shape, *table.shape[1:]] in the table's type, rounded once.  Negative ids and
    `padding_id` give zeros and take no part in the gradient; an id of V or more - an error that only the GPU sees -
    gives a row of NaN.  The gradient of the table is dense, with the table's shape and type, and the same bits for the
    same inputs; it can be differentiated again, in reverse (a table with a forward-mode tangent is refused).  A call that
    is recorded for a gradient also sorts its tokens, which the backward pass needs (8 bytes a token until then); under
    torch.no_grad() it does not."""
    return _host.embedding(ids, table, scale, padding_id)


def embedding_grad(grad_out, ids, num_rows, scale=1.0, padding_id=None):
    """The gradient of embedding() with respect to its table: [num_rows, ...] for grad_out [*ids.shape, ...], the sum
    of scale * grad_out over the tokens of each row, zeros for rows without one.  Sums are taken in float32 in an order
    that the ids alone decide.  Not recorded by autograd itself."""
    return _host.embedding_grad(grad_out, ids, num_rows, scale, padding_id)


class FeatureCodebook(nn.Module):
    """SH coefficients of N Gaussians as rows of a shared table: `table` [V, 16, 3] (trained) and `ids` [N] (which row a
    Gaussian has).  Called without arguments it returns the [N, 16, 3] features; the gradient goes to the table."""

    def __init__(self, table, ids):
        super().__init__()
        if table.dim() < 2:
            raise ValueError("the table is [rows, ...]")
        if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
            raise ValueError("ids are one int32 or int64 number per Gaussian")
        self.table = nn.Parameter(table.detach().clone())
        self.register_buffer("ids", ids.detach().clone())

    def forward(self):
        return embedding(self.ids, self.table)

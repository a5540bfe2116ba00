"""GPU: fdgs_embedding_fwd / fdgs_embedding_bwd through fdgs.embedding against the definition in 64 bits.

Tolerances: the lookup rounds a product to float32 (u = 2^-24) and once to the table's type (half a step, h).  The
gradient adds up to n terms in float32: a share of up to 64 items, or (a row that no join is needed for) a share and 63
more, then n / 8 + 2 partial sums at most (a share holds at least 8 items) and those of up to 256 groups of a join: a term
passes through at most 128 additions without a join, 64 + n / 8 + 2 + 256 with one, and never more than n."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half a step at the small end, where a type's numbers are evenly spaced
SMALL = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ids(t, v, seed, dtype, spread="mixed"):
    g = torch.Generator().manual_seed(seed)
    if spread == "one":
        return torch.full((t,), v // 2, dtype=dtype)
    if spread == "distinct":
        return torch.randperm(max(t, v), generator=g)[:t].remainder(v).to(dtype)
    ids = (v * torch.rand(t, generator=g) ** 3).long().clamp(0, v - 1)
    if t > 4:
        ids[torch.rand(t, generator=g) < 0.1] = -1           # without a row
        ids[torch.rand(t, generator=g) < 0.05] = v           # beyond the table
        ids[0], ids[-1] = v - 1, 0
    return ids.to(dtype)


def _lookup64(ids, table, scale, padding=None):
    v = table.shape[0]
    ids = ids.long()
    none = (ids < 0) | (torch.zeros_like(ids, dtype=torch.bool) if padding is None else ids == padding)
    out = torch.zeros(ids.shape + table.shape[1:], dtype=torch.float64)
    if v:
        out = scale * table.double()[ids.clamp(0, v - 1)]
    out[none] = 0.0
    out[(ids >= v) & ~none] = float("nan")
    return out


def _grad64(gy, ids, v, scale, padding=None):
    flat = gy.reshape(ids.numel(), math.prod(gy.shape[ids.dim():])).double()
    ids = ids.reshape(-1).long()
    ok = (ids >= 0) & (ids < v)
    if padding is not None:
        ok &= ids != padding
    acc = torch.zeros(v, flat.shape[1], dtype=torch.float64)
    size = torch.zeros(v, flat.shape[1], dtype=torch.float64)
    acc.index_add_(0, ids[ok], flat[ok])
    size.index_add_(0, ids[ok], flat[ok].abs())
    count = torch.bincount(ids[ok], minlength=v).double()[:, None]
    return scale * acc, abs(scale) * size, count


def _check_lookup(y, want, dtype):
    y = y.cpu().double()
    assert torch.equal(y.isnan(), want.isnan())
    err = (y - want).abs().nan_to_num(0.0)
    assert (err <= want.abs().nan_to_num(0.0) * (HALF[dtype] * (1 + U) + U) + SMALL[dtype]).all(), float(err.max())


def _check_grad(got, gy, ids, scale, dtype, padding=None):
    want, size, count = _grad64(gy.cpu(), ids.cpu(), got.shape[0], scale, padding)
    got = got.reshape(want.shape).cpu().double()
    depth = torch.minimum(count, 322 + count / 8) + 1                    # additions a term passes, and the product
    err = (got - want).abs()
    tol = U * depth * size + (want.abs() + U * depth * size) * HALF[dtype] + SMALL[dtype]
    assert (err <= tol).all(), (float((err - tol).max()), int((err > tol).sum()))
    assert (got[(count == 0).view(-1)] == 0).all()


SHAPES = [  # tokens, rows, width
    (0, 5, 8), (1, 1, 1), (1, 7, 3), (3, 1, 4), (37, 101, 33), (63, 64, 5), (64, 3, 64), (65, 1000, 12), (300, 17, 48),
    (1000, 5000, 31), (4096, 300, 7), (4097, 11, 256), (5000, 2, 1), (700, 40000, 2), (129, 33, 2056), (40, 9, 9001),
    (16384, 500, 16), (16385, 500, 16), (50000, 70000, 6), (60000, 255, 48), (40001, 256, 9)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,v,d", SHAPES)
def test_lookup_and_gradient(t, v, d, dtype):
    from fdgs.embedding import embedding
    g = torch.Generator().manual_seed(t + v + d)
    idt = torch.int32 if (t + d) % 2 else torch.int64
    ids = _ids(t, v, t, idt)
    table = torch.randn(v, d, generator=g).to(dtype)
    gy = torch.randn(t, d, generator=g).to(dtype)
    scale = math.sqrt(d)
    x = table.cuda().requires_grad_(True)
    y = embedding(ids.cuda(), x, scale=scale)
    assert y.dtype is dtype and y.shape == (t, d)
    _check_lookup(y.detach(), _lookup64(ids, table, float(torch.tensor(scale)), None), dtype)
    grad, = torch.autograd.grad(y, x, gy.cuda())
    assert grad.dtype is dtype and grad.shape == x.shape
    _check_grad(grad, gy, ids, float(torch.tensor(scale)), dtype)
    # the same bits again
    again, = torch.autograd.grad(embedding(ids.cuda(), x, scale=scale), x, gy.cuda())
    assert torch.equal(grad, again)


@pytest.mark.parametrize("spread", ["one", "distinct"])
@pytest.mark.parametrize("t,v,d,dtype", [(20000, 3, 48, torch.float32), (9000, 5, 1000, torch.bfloat16), (33000, 4, 1, torch.float16),
                                         (2000, 2, 2500, torch.float32), (16000, 20000, 48, torch.float32), (100, 1 << 20, 5, torch.float32),
                                         (100, 3, 48, torch.float32), (128, 2, 1000, torch.bfloat16), (129, 2, 1000, torch.bfloat16),
                                         (4096, 9, 64, torch.float16), (4097, 9, 64, torch.float16), (300000, 2, 4, torch.float32)])
def test_one_row_for_all_and_a_row_for_each(t, v, d, dtype, spread):
    """A row with every token (its sum is cut over many shares) and none with more than one or two.  Small whole numbers: the
    sums are exact in float32, so the gradient is the rounded exact value, whatever the order."""
    from fdgs.embedding import embedding_grad
    g = torch.Generator().manual_seed(t)
    ids = _ids(t, v, 5, torch.int32, spread)
    gy = torch.randint(-4, 5, (t, d), generator=g).to(dtype)
    got = embedding_grad(gy.cuda(), ids.cuda(), v, scale=0.5).cpu()
    want, _, _ = _grad64(gy, ids, v, 0.5)
    assert torch.equal(got, want.to(torch.float32).to(dtype))


def test_padding_and_shapes_of_ids():
    from fdgs.embedding import embedding, embedding_grad
    g = torch.Generator().manual_seed(4)
    table = torch.randn(50, 16, 3, generator=g).cuda()
    ids = torch.randint(-2, 50, (6, 9, 4), generator=g)
    for use in (ids, ids.transpose(0, 2), ids[::2, 1:], ids[0, 0, 0], ids[:0]):
        dev = use.cuda() if use.is_contiguous() else ids.cuda().transpose(0, 2) if use.shape[0] == 4 else ids.cuda()[::2, 1:]
        assert dev.shape == use.shape
        for padding in (None, 7):
            x = table.clone().requires_grad_(True)
            y = embedding(dev, x, scale=2.0, padding_id=padding)
            assert y.shape == use.shape + (16, 3)
            _check_lookup(y.detach(), _lookup64(use, table.cpu(), 2.0, padding), torch.float32)
            gy = torch.randn(y.shape, generator=g)
            grad, = torch.autograd.grad(y, x, gy.cuda())
            _check_grad(grad, gy, use, 2.0, torch.float32, padding)
            assert torch.equal(grad, embedding_grad(gy.cuda(), dev, 50, scale=2.0, padding_id=padding))


@pytest.mark.parametrize("t", [60, 3000, 9000, 40000])
def test_what_padded_tokens_hold_does_not_matter(t):
    """NaN and infinities in the gradients of padded tokens, and in the padding row of the table."""
    from fdgs.embedding import embedding, embedding_grad
    g = torch.Generator().manual_seed(t)
    ids = torch.randint(0, 50, (t,), generator=g)
    ids[torch.rand(t, generator=g) < 0.4] = -1
    ids[torch.rand(t, generator=g) < 0.2] = 49
    none = (ids == -1) | (ids == 49)
    gy = torch.randint(-3, 4, (t, 24), generator=g).float()
    bad = gy.clone()
    bad[none] = float("nan")
    bad[none.nonzero()[::2, 0]] = float("inf")
    table = torch.randn(50, 24, generator=g)
    table[49] = float("nan")
    got = embedding_grad(bad.cuda(), ids.cuda(), 50, padding_id=49).cpu()
    assert torch.equal(got, _grad64(gy, ids, 50, 1.0, 49)[0].float()) and (got[49] == 0).all()
    assert (embedding(ids.cuda(), table.cuda(), padding_id=49).cpu()[none] == 0).all()
    assert (embedding_grad(bad.cuda(), torch.full_like(ids, -5).cuda(), 50).cpu() == 0).all()


def test_slices_of_tables_and_gradients_are_read_in_place():
    from fdgs.embedding import embedding, embedding_grad
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(40, 30, generator=g).cuda()
    ids = torch.randint(0, 40, (5, 21), generator=g).cuda()
    for table in (wide[:, 3:20], wide[:, 1:2], wide[::3], wide.t(), wide[:1].expand(40, 30)):
        ok = ids.remainder(table.shape[0])
        assert torch.equal(embedding(ok, table, scale=1.5), embedding(ok, table.contiguous(), scale=1.5))
    wide = torch.randn(5, 21, 64, generator=g).cuda()
    for gy in (wide[..., 5:20], wide[..., :1], wide[:, :1].expand(5, 21, 64), wide[:1, :1, :9].expand(5, 21, 9),
               torch.ones((), device="cuda").expand(5, 21, 33), wide.transpose(1, 2)[:, :21]):
        assert torch.equal(embedding_grad(gy, ids, 40), embedding_grad(gy.contiguous(), ids, 40))


def test_gradient_against_differences():
    """The lookup is linear: with whole numbers the difference of two lookups, weighted, is the gradient exactly."""
    from fdgs.embedding import embedding
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 30, (400,), generator=g).cuda()
    table = torch.randint(-8, 9, (30, 20), generator=g).float().cuda().requires_grad_(True)
    step = torch.randint(-3, 4, (30, 20), generator=g).float().cuda()
    gy = torch.randint(-3, 4, (400, 20), generator=g).float().cuda()
    y = embedding(ids, table, scale=2.0)
    grad, = torch.autograd.grad(y, table, gy)
    moved = embedding(ids, (table + step).detach(), scale=2.0)
    assert float(((moved - y.detach()) * gy).double().sum()) == float((grad * step).double().sum())


def test_second_derivatives():
    """sum(y^2 w) has the Hessian 2 scale^2 diag(sum of w): whole numbers, so exact."""
    from fdgs.embedding import embedding
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-1, 6, (50,), generator=g).cuda()
    table = torch.randint(-4, 5, (6, 5), generator=g).float().cuda().requires_grad_(True)
    w = torch.randint(-3, 4, (50, 5), generator=g).float().cuda()
    u = torch.randint(-3, 4, (6, 5), generator=g).float().cuda()
    y = embedding(ids, table, scale=2.0)
    first, = torch.autograd.grad((y * y * w).sum(), table, create_graph=True)
    second, = torch.autograd.grad((first * u).sum(), table, create_graph=True)
    sums = torch.zeros(6, 5, device="cuda").index_add_(0, ids.clamp_min(0), w * (ids >= 0)[:, None])
    assert torch.equal(first, 8 * sums * table) and torch.equal(second, 8 * sums * u)


def test_profiled_calls():
    """With _lib.PROFILE set the calls are bracketed with events, forward and backward."""
    from fdgs import _lib
    from fdgs.embedding import embedding
    table = torch.randn(9, 4, device="cuda", requires_grad=True)
    ids = torch.tensor([3, 3, 1], device="cuda")
    plain = embedding(ids, table)
    _lib.PROFILE = {}
    try:
        y = embedding(ids, table)
        y.sum().backward()
        seen = {k: len(v) for k, v in _lib.PROFILE.items()}
    finally:
        _lib.PROFILE = None
    assert seen == {"fdgs_embedding_fwd": 1, "fdgs_embedding_bwd": 1}
    assert torch.equal(y, plain) and table.grad.sum() == 12


def test_two_captured_graphs_with_workspaces_of_their_own():
    """Lookup and gradient captured twice, replayed in turn with new inputs and eager calls in between."""
    from fdgs.embedding import embedding, embedding_grad
    cases = []
    for t, v, d in ((20000, 300, 24), (500, 900, 40), (9000, 70, 16), (100, 30, 8)):
        cases.append([torch.zeros(t, dtype=torch.int32, device="cuda"), torch.zeros(v, d, device="cuda"),
                      torch.zeros(t, d, device="cuda"), None, None, torch.cuda.CUDAGraph()])
    for c in cases:
        ids, table, gy = c[:3]
        embedding_grad(gy, ids, table.shape[0])
        with torch.cuda.graph(c[5]):
            c[3], c[4] = embedding(ids, table, scale=3.0), embedding_grad(gy, ids, table.shape[0], scale=3.0)
    for k in range(4):
        for j, (ids, table, gy, y, grad, graph) in enumerate(cases):
            g = torch.Generator().manual_seed(10 * k + j)
            ids.copy_((table.shape[0] * torch.rand(ids.shape, generator=g) ** 2).int())
            table.copy_(torch.randn(table.shape, generator=g))
            gy.copy_(torch.randn(gy.shape, generator=g))
            graph.replay()
            eager = embedding(ids, table, scale=3.0), embedding_grad(gy, ids, table.shape[0], scale=3.0)
            torch.cuda.synchronize()
            assert torch.equal(y, eager[0]) and torch.equal(grad, eager[1])


def test_captured_training_pass():
    """Lookup and backward through autograd in one graph, replayed with other inputs and eager calls in between."""
    from fdgs.embedding import embedding, embedding_grad
    ids = torch.zeros(5000, dtype=torch.int64, device="cuda")
    table = torch.zeros(40, 12, device="cuda", requires_grad=True)
    gy = torch.zeros(5000, 12, device="cuda")

    def once():
        y = embedding(ids, table, scale=0.5)
        return y, torch.autograd.grad(y, table, gy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for k in range(3):
        g = torch.Generator().manual_seed(k)
        ids.copy_(torch.randint(-1, 40, (5000,), generator=g))
        with torch.no_grad():
            table.copy_(torch.randn(40, 12, generator=g))
        gy.copy_(torch.randn(5000, 12, generator=g))
        graph.replay()
        y = embedding(ids, table.detach(), scale=0.5)
        want = embedding_grad(gy, ids, 40, scale=0.5)
        torch.cuda.synchronize()
        assert torch.equal(out[0], y) and torch.equal(out[1], want)


def test_capture_beside_a_living_eager_graph_is_refused():
    """Such a backward pass would end the process; without gradients, or with the eager graph gone, the capture works."""
    from fdgs.embedding import embedding
    ids = torch.tensor([1, 0, 1], device="cuda")
    table = torch.randn(2, 8, device="cuda", requires_grad=True)
    eager = embedding(ids, table)
    first = torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        with pytest.raises(RuntimeError, match="outside the capture"):
            embedding(ids, table)
        plain = embedding(ids, table.detach())
    first.replay()
    torch.cuda.synchronize()
    assert torch.equal(plain, eager)
    want = eager.detach().clone()
    del eager
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        y = embedding(ids, table) + embedding(ids, table)        # twice in one capture
        grad, = torch.autograd.grad(y, table, torch.ones_like(y))
    for _ in range(3):
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, 2 * want) and torch.equal(grad, torch.tensor([[2.0], [4.0]], device="cuda").expand(2, 8))


def test_two_streams_at_once():
    from fdgs.embedding import embedding_grad
    g = torch.Generator().manual_seed(1)
    jobs = []
    for t, v, d in ((30000, 100, 64), (17000, 5000, 33)):
        ids, gy = torch.randint(0, v, (t,), generator=g).cuda(), torch.randn(t, d, generator=g).cuda()
        jobs.append((gy, ids, v, torch.cuda.Stream(), embedding_grad(gy, ids, v)))
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for gy, ids, v, stream, want in jobs:
            with torch.cuda.stream(stream):
                got.append((embedding_grad(gy, ids, v), want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)


def test_offsets_past_32_bits():
    """Outputs, tables and gradients of more than 2^31 elements: rows and tokens at both ends."""
    from fdgs.embedding import embedding, embedding_grad
    d, n = 2048, (1 << 20) + 77                  # 2^31 + 157,696 elements
    ids = torch.arange(n, device="cuda").flip(0).to(torch.int32)
    table = torch.zeros(n, d, dtype=torch.bfloat16, device="cuda")
    for r in (0, 1, n // 2, n - 2, n - 1):
        table[r] = float(r % 251 + 1)
    y = embedding(ids, table)
    for r in (0, 1, n // 2, n - 2, n - 1):
        assert (y[n - 1 - r] == float(r % 251 + 1)).all()
    assert int((y[:, 0] != 0).sum()) == 5 and int((y[:, d - 1] != 0).sum()) == 5
    del table
    grad = embedding_grad(y, ids, n, scale=2.0)
    for r in (0, 1, n // 2, n - 2, n - 1):
        assert (grad[r] == 2.0 * float(r % 251 + 1)).all()
    assert int((grad[:, 0] != 0).sum()) == 5 and int((grad[:, d - 1] != 0).sum()) == 5


def test_refusals_on_the_device():
    from fdgs.embedding import embedding, embedding_grad
    table = torch.zeros(4, 4, device="cuda")
    with pytest.raises(ValueError, match="one device"):
        embedding(torch.tensor([1]), table)
    with pytest.raises(ValueError, match="int32 or int64"):
        embedding(torch.tensor([1.0], device="cuda"), table)
    with pytest.raises(ValueError, match="float32, bfloat16"):
        embedding(torch.tensor([1], device="cuda"), table.double())
    with pytest.raises(TypeError, match="scale is a number"):
        embedding(torch.tensor([1], device="cuda"), table, scale=torch.ones(()))
    with pytest.raises(ValueError, match="row of the table"):
        embedding(torch.tensor([1], device="cuda"), table, padding_id=-1)
    ids = torch.tensor([1, 2], device="cuda")
    with pytest.raises(ValueError, match="ids.shape"):
        embedding_grad(torch.zeros(3, 4, device="cuda"), ids, 4)
    with pytest.raises(ValueError, match="ids.shape"):
        embedding_grad(torch.zeros(2, device="cuda"), ids, 4)
    with pytest.raises(ValueError, match="num_rows"):
        embedding_grad(torch.zeros(2, 4, device="cuda"), ids, -1)
    assert embedding_grad(torch.zeros(2, 4, device="cuda"), ids, 0).shape == (0, 4)
    assert embedding(torch.tensor([0, 1], device="cuda"), torch.zeros(0, 4, device="cuda")).isnan().all()
    assert embedding(ids, torch.zeros(4, 0, device="cuda")).shape == (2, 0)
    assert embedding_grad(torch.zeros(2, 0, device="cuda"), ids, 4).shape == (4, 0)


@pytest.mark.parametrize("tokens, rows, dim", [(128, 40, 7), (129, 40, 3), (2000, 17, 5), (4096, 300, 8), (4097, 300, 2), (9000, 5000, 4100),
                                               (16384, 40000, 33), (16385, 40000, 1), (70001, 90, 48), (300000, 8192, 12), (600001, 300000, 3), (20000, 1, 3)])
@pytest.mark.parametrize("dtype, idt", [(torch.float32, torch.int32), (torch.bfloat16, torch.int64), (torch.float16, torch.int32)])
def test_lookup_that_sorts_for_its_gradient(tokens, rows, dim, dtype, idt):
    """A lookup that is recorded sorts the tokens beside its own work: the output and the gradient have the bits of the plain
    lookup and of the gradient that sorts by itself, also when the pass is walked back twice."""
    from fdgs.embedding import embedding, embedding_grad
    gen = torch.Generator().manual_seed(tokens)
    table = torch.randn(rows, dim, generator=gen).to(dtype).cuda().requires_grad_(True)
    ids = torch.randint(-3, rows + 2, (tokens,), generator=gen)
    ids[torch.rand(tokens, generator=gen) < 0.3] = rows // 2     # a row with many tokens
    ids = ids.to(idt).cuda()
    gy = torch.randn(tokens, dim, generator=gen).to(dtype).cuda()
    y = embedding(ids, table, scale=0.75, padding_id=1)
    with torch.no_grad():
        assert torch.equal(y.view(torch.uint8), embedding(ids, table, scale=0.75, padding_id=1).view(torch.uint8))
    want = embedding_grad(gy, ids, rows, scale=0.75, padding_id=1)
    for _ in range(2):
        got, = torch.autograd.grad(y, table, gy, retain_graph=True)
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_ids_that_change_after_the_lookup_are_noticed():
    from fdgs.embedding import embedding
    table = torch.randn(50, 4, device="cuda", requires_grad=True)
    ids = torch.arange(50, device="cuda").repeat(5)
    y = embedding(ids, table)
    ids.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_capture_beside_a_living_eager_graph_of_a_leaf_behind_the_table():
    from fdgs.embedding import embedding
    ids = torch.tensor([1, 0, 1], device="cuda")
    leaf = torch.randn(2, 8, device="cuda", requires_grad=True)
    eager = leaf * 2
    first = torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        with pytest.raises(RuntimeError, match="outside the capture"):
            embedding(ids, (leaf + 1).bfloat16())
        plain = embedding(ids, (leaf + 1).detach())
    first.replay()
    torch.cuda.synchronize()
    assert torch.equal(plain, (leaf + 1)[ids])
    del eager
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        y = embedding(ids, 3 * leaf)
        grad, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    for _ in range(3):
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, (3 * leaf)[ids].detach()) and torch.equal(grad, torch.tensor([3.0, 6.0], device="cuda")[:, None].expand(2, 8))


def test_a_table_of_very_many_rows():
    """Keys of 28 bits: four digits.  Rows of one element, nearly all of them without a token."""
    from fdgs.embedding import embedding, embedding_grad
    rows, tokens = (1 << 27) + 5, 20000
    gen = torch.Generator().manual_seed(0)
    ids = torch.randint(0, rows, (tokens,), generator=gen)
    ids[:5000] = ids[5000]
    ids[5000:5003] = torch.tensor([rows - 1, 0, rows])           # the last one's is beyond the table
    gy = torch.randn(tokens, 1, generator=gen).half()
    got = embedding_grad(gy.cuda(), ids.cuda(), rows)
    there = ids < rows
    where, index = torch.unique(ids[there], return_inverse=True)
    want = torch.zeros(len(where), dtype=torch.float64).index_add_(0, index, gy[there, 0].double())
    size = torch.zeros(len(where), dtype=torch.float64).index_add_(0, index, gy[there, 0].double().abs())
    many = torch.bincount(index).double()
    # a sum of n terms in float32, then half a step of float16
    off = (got.cpu()[where, 0].double() - want).abs()
    assert (off <= many * 2.0 ** -24 * size + 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -25).all()
    assert int(got.count_nonzero()) == int((want.half() != 0).sum())
    table = torch.zeros(rows, 1, dtype=torch.float16, device="cuda", requires_grad=True)
    y = embedding(ids.cuda(), table)
    again, = torch.autograd.grad(y, table, gy.cuda())
    assert torch.equal(again, got) and int(y.isnan().sum()) == int((~there).sum())


@pytest.mark.parametrize("dim, dtype", [(1, torch.float32), (3, torch.bfloat16), (8, torch.float32), (48, torch.float32), (100, torch.float16),
                                        (1030, torch.float32), (2048, torch.bfloat16)])
@pytest.mark.parametrize("rows, where", [(1, "one"), (5000, "one"), (5000, "two"), (40, "even"), (5000, "half")])
def test_rows_with_very_many_tokens(dim, dtype, rows, where):
    """Rows that whole workgroups of the walk lie inside of, that begin and end anywhere, beside rows with few tokens or none."""
    from fdgs.embedding import embedding_grad
    tokens = 2000000 // max(dim, 20)
    gen = torch.Generator().manual_seed(dim + rows)
    ids = torch.randint(0, rows, (tokens,), generator=gen)
    if where == "one":
        ids[:] = rows // 2
    elif where == "two":
        ids = rows // 2 + (torch.rand(tokens, generator=gen) < 0.3).long()
    elif where == "half":
        ids[torch.rand(tokens, generator=gen) < 0.5] = rows - 1
        ids[torch.rand(tokens, generator=gen) < 0.1] = -1
    gy = torch.randn(tokens, dim, generator=gen).to(dtype)
    got = embedding_grad(gy.cuda(), ids.int().cuda(), rows).cpu().double()
    ok = ids >= 0
    want = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids[ok], gy[ok].double())
    size = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids[ok], gy[ok].double().abs())
    many = torch.bincount(ids[ok], minlength=rows).double()[:, None]
    # n additions in float32, each off by at most half a step of a partial sum that is at most the sum of the magnitudes
    assert ((got - want).abs() <= many * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + 2.0 ** -25).all()


@pytest.mark.parametrize("rows", [1, 2, 300, 511, 512, 70000, 262143, 262144, (1 << 27) + 1])
def test_every_sort_at_its_limits(rows):
    """Sums of whole numbers, exact in float32, at the numbers of tokens where one way to sort ends and the next begins."""
    from fdgs.embedding import embedding_grad
    gen = torch.Generator().manual_seed(rows)
    for tokens in (127, 128, 129, 767, 768, 769, 1536, 1537, 2304, 2305, 3072, 3073, 4095, 4096, 4097, 8192, 8193, 12289, 16384, 16385, 33000):
        even = torch.randint(0, rows, (tokens,), generator=gen)
        kinds = {"even": even, "skewed": (rows * torch.rand(tokens, generator=gen, dtype=torch.float64) ** 8).long(),
                 "one": torch.full((tokens,), rows - 1), "none": torch.full((tokens,), -1), "rising": even.sort()[0],
                 "falling": even.sort(descending=True)[0], "padded": torch.where(torch.rand(tokens, generator=gen) < 0.4, -1, even)}
        gy = torch.randint(-8, 9, (tokens, 1), generator=gen).float().cuda()
        for name, ids in kinds.items():
            ids = ids.int().cuda()
            got = embedding_grad(gy, ids, rows)
            ok = ids >= 0
            want = torch.zeros(rows, 1, device="cuda").index_add_(0, ids[ok].long(), gy[ok])     # whole numbers: in any order
            assert torch.equal(got, want), (tokens, name)


@pytest.mark.parametrize("scale", [-2.0, math.inf, math.nan])
@pytest.mark.parametrize("tokens, apart", [(3, 7), (100, 7), (5000, 7), (128, 6), (100, 11), (700, 13), (900, 17)])
def test_rows_without_tokens_are_zeros_whatever_the_scale(scale, tokens, apart):
    from fdgs.embedding import embedding_grad
    ids = apart * torch.arange(tokens, device="cuda") % 901
    got = embedding_grad(torch.ones(tokens, 6, device="cuda"), ids, 6000, scale=scale)
    none = torch.ones(6000, dtype=torch.bool, device="cuda")
    none[ids] = False
    assert int(none.sum()) > 5000 and (got[none].view(torch.int32) == 0).all()           # and no negative zero
    assert not torch.isfinite(got[~none]).any() if math.isinf(scale) or math.isnan(scale) else (got[~none] < 0).all()


def test_forward_derivatives_are_refused_on_the_device():
    import torch.autograd.forward_ad as forward_ad
    from fdgs.embedding import embedding, embedding_grad
    ids, table = torch.tensor([1, 2], device="cuda"), torch.randn(5, 4, device="cuda")
    tangent = torch.ones(2, 4, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            embedding(ids, forward_ad.make_dual(table, torch.ones_like(table)))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            embedding_grad(forward_ad.make_dual(table[:2], tangent), ids, 5)
        y = embedding(ids, table.requires_grad_(True))
        with pytest.raises(RuntimeError, match="forward-mode"):          # out of a backward pass
            torch.autograd.grad(y, table, forward_ad.make_dual(tangent, tangent))


def test_views_that_are_still_to_be_negated():
    from fdgs.embedding import embedding, embedding_grad
    z = torch.randn(6, 1, dtype=torch.complex64, device="cuda")
    ids = torch.tensor([5, 0, 3, 3], device="cuda")
    for x in (z.conj().imag, torch._neg_view(torch.randn(6, 4, device="cuda"))):
        assert x.is_neg()
        assert torch.equal(embedding(ids, x), embedding(ids, x.clone().resolve_neg()))
        assert torch.equal(embedding(ids, x), x[ids].resolve_neg())
        assert torch.equal(embedding_grad(x[:4], ids, 6), embedding_grad(x[:4].resolve_neg().contiguous(), ids, 6))
    assert torch.equal(embedding(torch._neg_view(-ids), z.imag), z.imag[ids])


def test_a_lookup_of_more_workgroups_than_a_launch_has():
    """73 tokens of 7 float16 numbers to a workgroup: 2^24 workgroups of 256 threads are one launch too many.  17 GB of output."""
    from fdgs.embedding import embedding
    tokens, rows = 73 * (1 << 24) + 500, 1000
    table = torch.randn(rows, 7, device="cuda").half()
    ids = (torch.arange(tokens, dtype=torch.int32, device="cuda") * 7 + 3) % (rows + 1) - 1
    y = embedding(ids, table, scale=0.5)
    half = torch.cat([table * 0.5, torch.zeros_like(table[:1])])            # -1: the last row; exact
    part = 1 << 26
    for at in range(0, tokens, part):
        assert torch.equal(y[at:at + part], half[ids[at:at + part].long()]), at


def test_a_recorded_lookup_of_more_workgroups_than_a_launch_has():
    """One token to a workgroup: the sort runs by itself, the lookup in two launches.  69 GB of output."""
    from fdgs.embedding import embedding
    tokens, rows, dim = (1 << 24) + 5, 500, 2056
    table = torch.randn(rows, dim, device="cuda").bfloat16().requires_grad_(True)
    ids = (torch.arange(tokens, device="cuda") * 7 + 3) % (rows + 1) - 1
    y = embedding(ids, table).detach()
    want = torch.cat([table.detach(), torch.zeros_like(table[:1])])
    part = 1 << 20
    for at in range(0, tokens, part):
        assert torch.equal(y[at:at + part], want[ids[at:at + part]]), at
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dim, dtype", [(1, torch.float32), (3, torch.bfloat16), (8, torch.float32), (48, torch.float32), (100, torch.float16),
                                        (1030, torch.float32), (2048, torch.bfloat16)])
@pytest.mark.parametrize("rows, where", [(1, "one"), (5000, "one"), (5000, "two"), (5000, "three"), (40, "even"), (5000, "half")])
def test_sums_of_rows_with_very_many_tokens_are_exact(dim, dtype, rows, where):
    """Gradients of whole numbers, the sums of which float32 holds whatever the order: a token that is left out, taken twice or added
    to another row shows.  Rows that begin and end inside workgroups of the walk and hold whole ones between."""
    from fdgs.embedding import embedding_grad
    tokens = 2000000 // max(dim, 20)
    gen = torch.Generator().manual_seed(dim + rows)
    ids = torch.randint(0, rows, (tokens,), generator=gen)
    if where == "one":
        ids[:] = rows // 2
    elif where == "two":
        ids = rows // 2 + (torch.rand(tokens, generator=gen) < 0.3).long()
    elif where == "three":
        ids[torch.rand(tokens, generator=gen) < 0.9] = rows // 3
        ids[torch.rand(tokens, generator=gen) < 0.5] = rows // 2
    elif where == "half":
        ids[torch.rand(tokens, generator=gen) < 0.5] = rows - 1
        ids[torch.rand(tokens, generator=gen) < 0.1] = -1
    gy = torch.randint(1, 8, (tokens, dim), generator=gen).to(dtype)         # none of them zero: every token counts
    got = embedding_grad(gy.cuda(), ids.int().cuda(), rows, scale=0.25).cpu()
    ok = ids >= 0
    want = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids[ok], gy[ok].double())
    assert want.max() < 2 ** 24 and torch.equal(got, (0.25 * want).float().to(dtype))


@pytest.mark.parametrize("tokens", [2097152, 2097153, 2100000, 5000000])
@pytest.mark.parametrize("rows, dim", [(300, 1), (511, 3), (70000, 1), (600000, 2)])
def test_sorts_whose_workgroups_take_several_tiles(tokens, rows, dim):
    """More than 1024 tiles of 2048 tokens: a workgroup of the sort goes on with a second and a third.  One to three digits, ids that are
    skewed, partly absent; by itself and beside the lookup.  Whole numbers: exact in any order."""
    from fdgs.embedding import embedding, embedding_grad
    gen = torch.Generator(device="cuda").manual_seed(tokens + rows)
    ids = (rows * torch.rand(tokens, generator=gen, device="cuda", dtype=torch.float64) ** 4).long()
    ids[torch.rand(tokens, generator=gen, device="cuda") < 0.05] = -1
    ids[torch.rand(tokens, generator=gen, device="cuda") < 0.02] = rows
    ids[-3:] = torch.tensor([rows - 1, 0, rows - 1], device="cuda")
    gy = torch.randint(-8, 9, (tokens, dim), generator=gen, device="cuda").float()
    ok = (ids >= 0) & (ids < rows)
    here = ids[ok].cpu()                                     # (the GPU's own sums wait for one another at a frequent row)
    want = torch.stack([torch.bincount(here, x, rows) for x in gy[ok].double().cpu().t()], 1).float().cuda()
    assert torch.equal(embedding_grad(gy, ids, rows), want)
    table = torch.randn(rows, dim, generator=gen, device="cuda", requires_grad=True)
    y = embedding(ids.int(), table)
    assert torch.equal(torch.autograd.grad(y, table, gy)[0], want)
    y = y.detach()
    assert torch.equal(y[ok], table.detach()[ids[ok]]) and (y[ids < 0] == 0).all() and y[ids == rows].isnan().all()


def test_as_many_tokens_as_a_gradient_takes():
    """2^30 tokens of one and the same gradient, every row's count known beforehand: sums exact below 2^24.  30 GB."""
    from fdgs.embedding import embedding_grad
    tokens, rows, often = 1 << 30, 1009, 1 << 23
    ids = torch.empty(tokens, dtype=torch.int32, device="cuda")
    part = 1 << 27
    for at in range(0, tokens, part):
        ids[at:at + part] = (torch.arange(at, at + part, device="cuda") * 787 % rows).int()
    count = torch.full((rows,), tokens // rows, dtype=torch.int64)
    count[torch.arange(tokens % rows) * 787 % rows] += 1
    place = torch.arange(often, device="cuda") * 127 + 5         # these change to one row
    count -= torch.bincount(ids[place].cpu(), minlength=rows)
    ids[place] = 500
    count[500] += often
    assert int(count.sum()) == tokens and int(count.max()) < 1 << 24
    got = embedding_grad(torch.ones((), device="cuda").expand(tokens, 1), ids, rows)
    assert torch.equal(got[:, 0].cpu(), count.float())


def test_a_table_of_nearly_2_to_the_31_rows():
    """Items past 2^31 in the walk, keys of 31 bits."""
    from fdgs.embedding import embedding, embedding_grad
    rows = (1 << 31) - 200000
    ids = torch.tensor([rows - 1, 0, rows - 1, 1 << 30, -1, rows, rows - 2, 0, 0] * 20, device="cuda")
    gy = torch.arange(1, 181, device="cuda").half()[:, None]
    got = embedding_grad(gy, ids, rows)
    where = torch.tensor([0, 1 << 30, rows - 2, rows - 1], device="cuda")
    want = torch.stack([gy[ids == r].double().sum() for r in where]).half()
    assert torch.equal(got[where, 0], want)
    assert sum(int(c.count_nonzero()) for c in got.view(-1).split(1 << 28)) == 4
    y = embedding(ids, got)
    assert torch.equal(y[(ids >= 0) & (ids < rows)], got[ids[(ids >= 0) & (ids < rows)]]) and (y[ids < 0] == 0).all() and y[ids == rows].isnan().all()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens", [20, 500, 20000])
def test_what_is_saved_may_be_kept_elsewhere_or_made_again(tokens):
    """Under saved-tensor hooks and activation checkpointing (whose recomputation ends by an exception out of such a hook)."""
    from fdgs.embedding import embedding
    from torch.utils.checkpoint import checkpoint
    ids = torch.randint(-1, 90, (tokens,), device="cuda")
    table = torch.randn(90, 12, device="cuda", requires_grad=True)
    gy = torch.randn(tokens, 12, device="cuda")
    want, = torch.autograd.grad(embedding(ids, table), table, gy)
    for pinned in (False, True):
        with torch.autograd.graph.save_on_cpu(pin_memory=pinned):
            y = embedding(ids, table)
        assert torch.equal(torch.autograd.grad(y, table, gy)[0], want)
    for reentrant in (False, True):
        table.grad = None
        (0.5 * checkpoint(lambda t: 2 * embedding(ids, t), table, use_reentrant=reentrant)).backward(gy)
        assert torch.equal(table.grad, want)


def test_an_exception_out_of_a_hook_stays_what_it_is():
    from fdgs.embedding import embedding

    class Stop(Exception):
        pass

    def pack(x):
        raise Stop(tuple(x.shape))
    ids, table = torch.tensor([1, 0, 1], device="cuda"), torch.randn(2, 8, device="cuda", requires_grad=True)
    with pytest.raises(Stop, match="(3,)"):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda x: x):
            embedding(ids, table)
    assert embedding(ids, table).shape == (3, 8)


def test_an_exception_in_a_profiled_call_stays_what_it_is():
    from fdgs import _lib
    from fdgs.embedding import embedding
    ids, table = torch.tensor([1, 0, 1], device="cuda"), torch.randn(2, 8, device="cuda", requires_grad=True)
    y = embedding(ids, table)
    _lib.PROFILE = ()                                        # not a dict
    try:
        for call in (lambda: embedding(ids, table), lambda: y.sum().backward()):
            with pytest.raises(AttributeError, match="setdefault"):
                call()
    finally:
        _lib.PROFILE = None
    embedding(ids, table).sum().backward()
    assert table.grad.sum() == 24

"""CPU: what the table lookup and its gradient refuse, and the sizes of the workspace."""
import ctypes as C

import pytest
import torch


def _fwd(**over):
    from fdgs import _lib, _records
    f = dict(num_tokens=2, num_rows=3, dim=4, type=0, id_bytes=4, ids=64, table=64, table_row_stride=4, padding_id=-1, out=64, scale=1.0)
    f.update(over)
    return _lib.lib.fdgs_embedding_fwd(C.byref(_records.EmbeddingFwdArgs(**f)), None)


def _bwd(**over):
    from fdgs import _lib, _records
    f = dict(num_tokens=2, num_rows=3, dim=4, type=0, id_bytes=8, ids=64, grad_out=64, grad_out_row_stride=4, padding_id=-1,
             grad_table=64, scale=1.0, workspace=64, workspace_bytes=1 << 30)
    f.update(over)
    return _lib.lib.fdgs_embedding_bwd(C.byref(_records.EmbeddingBwdArgs(**f)), None)


def test_library_refuses_before_any_launch():
    from fdgs import _lib
    assert _lib.lib.fdgs_embedding_fwd(None, None) == -1 and _lib.lib.fdgs_embedding_bwd(None, None) == -1
    for call in (_fwd, _bwd):
        for bad in (dict(num_tokens=-1), dict(num_rows=-1), dict(dim=-1), dict(type=3), dict(type=-1), dict(id_bytes=2), dict(ids=0)):
            assert call(**bad) == -1, bad
        assert call(dim=0) == 0 and call(dim=(1 << 22) + 1) == -4
    assert _fwd(table=0) == -1 and _fwd(out=0) == -1 and _fwd(table_row_stride=-1) == -1 and _fwd(num_tokens=0) == 0
    assert _fwd(num_tokens=1 << 31) == -4
    assert _bwd(grad_out=0) == -1 and _bwd(grad_table=0) == -1 and _bwd(grad_out_row_stride=-1) == -1 and _bwd(num_rows=0) == 0
    assert _bwd(num_tokens=(1 << 30) + 1) == -4
    assert _bwd(workspace=0) == -3 and _bwd(workspace_bytes=16) == -3


def test_sorted_tokens_need_a_workspace():
    from fdgs import _lib
    size = _lib.lib.fdgs_embedding_sort_workspace_bytes
    assert size(-1) == 0 and size((1 << 30) + 1) == 0 and size(4096) == 0 and size(4097) >= 8 * 4097 and size(1 << 30) >= 8 << 30
    for tokens in (5000, 20000):
        assert _fwd(num_tokens=tokens, sorted=64) == -3
        assert _fwd(num_tokens=tokens, sorted=64, workspace=64, workspace_bytes=size(tokens) - 1) == -3
        assert _fwd(num_tokens=tokens, sorted=64, workspace=0, workspace_bytes=size(tokens)) == -3
    assert _fwd(num_tokens=(1 << 30) + 1, sorted=64) == -4


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_workspace_grows_with_the_work(kind):
    from fdgs._lib import lib
    size = lib.fdgs_embedding_bwd_workspace_bytes
    assert size(-1, 4, 4, kind) == 0 and size(4, 4, 0, kind) == 0 and size(4, 4, 4, 7) == 0
    for v, d in ((1, 1), (100, 48), (65536, 48), (1000, 5000)):
        last = 0
        for t in (0, 1, 100, 16384, 16385, 300000):
            now = size(t, v, d, kind)
            assert now >= 8 * t and now >= last * 0.5
            last = now


def test_cpu_tensors_are_refused():
    from fdgs.embedding import FeatureCodebook, embedding, embedding_grad
    ids, table = torch.tensor([0, 1]), torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        embedding(ids, table)
    with pytest.raises(RuntimeError, match="GPU only"):
        embedding_grad(torch.zeros(2, 4), ids, 3)
    with pytest.raises(ValueError, match="rows, ..."):
        embedding(ids, torch.zeros(3))
    with pytest.raises(ValueError, match="per Gaussian"):
        FeatureCodebook(torch.zeros(3, 16, 3), ids.view(2, 1))
    book = FeatureCodebook(torch.zeros(3, 16, 3), ids)
    assert set(book.state_dict()) == {"table", "ids"} and book.table.requires_grad


def test_rows_of_strided_gradients():
    """Which tensors are read in place, and with what distance between their rows."""
    from fdgs._host import rows_layout
    base = torch.zeros(6, 5, 8)
    for t, lead, width, stride in ((base, 2, 8, 8), (base[..., 2:5], 2, 3, 8), (base[:, :1].expand(6, 5, 8), 2, 8, None),
                                   (base[:1, :1].expand(6, 5, 8), 2, 8, 0), (base[:, ::2, :4], 2, 4, None), (base[::2], 1, 40, 80),
                                   (base[:, 0], 1, 8, 40), (base.transpose(0, 1), 2, 8, None), (torch.zeros(()).expand(6, 5, 8), 2, 8, None)):
        assert rows_layout(t, lead) == (stride is not None, width, width if stride is None else stride), (t.shape, t.stride())


@pytest.mark.parametrize("ids, row", [(3, (16, 3)), (5, (16, 3)), (4, (48,)), (4, (15, 3))])
def test_render_refuses_a_codebook_that_does_not_fit(ids, row):
    """An id for each Gaussian and rows of 16 x 3, or the kernels behind would read past the looked-up rows."""
    from types import SimpleNamespace
    from fdgs.embedding import FeatureCodebook
    from fdgs.renderer import render
    eye = torch.eye(4)
    cam = SimpleNamespace(FoVx=1.0, FoVy=1.0, image_height=8, image_width=8, world_view_transform=eye, full_proj_transform=eye,
                          camera_center=torch.zeros(3), time=0.0)
    xyz = torch.zeros(4, 3)
    pc = SimpleNamespace(get_xyz=xyz, _xyz=xyz, _opacity=torch.zeros(4, 1), active_sh_degree=3, max_sh_degree=3,
                         feature_codebook=FeatureCodebook(torch.zeros(7, *row), torch.zeros(ids, dtype=torch.int32)))
    with pytest.raises(ValueError, match="an id each"):
        render(cam, pc, None, torch.zeros(3), stage="coarse")


def test_forward_derivatives_are_refused():
    """The kernels carry no tangent: a result without one would read as a derivative of zero."""
    import torch.autograd.forward_ad as forward_ad
    from fdgs.embedding import embedding, embedding_grad
    ids, x = torch.tensor([0, 1]), torch.ones(2, 4)
    with forward_ad.dual_level():
        for wants in (False, True):
            dual = forward_ad.make_dual(x.clone().requires_grad_(wants), x)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                embedding(ids, dual)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                embedding_grad(dual, ids, 3)
        with pytest.raises(RuntimeError, match="GPU only"):
            embedding(ids, x)


def test_rows_of_views_that_are_still_to_be_negated():
    """The imaginary part of a conjugate lies in memory with the other sign: it is never read in place."""
    from fdgs._host import rows_layout
    z = torch.zeros(6, 1, dtype=torch.complex64)
    assert z.conj().imag.is_neg()
    assert rows_layout(z.imag, 1) == (True, 1, 2) and rows_layout(z.conj().imag, 1) == (False, 1, 1)
    assert rows_layout(torch._neg_view(torch.zeros(3, 4)), 1) == (False, 4, 4)


def test_gradients_that_no_grid_holds_are_refused():
    """A launch has fewer than 2^32 threads: rows of one element, 128 rows and tokens to a workgroup of the join."""
    for rows, tokens in (((1 << 31) - 1, 1), ((1 << 31) - 129, 129), ((1 << 31) - 1, 1 << 30)):
        assert _bwd(num_rows=rows, num_tokens=tokens, dim=1) == -4
    for rows, tokens, dim in (((1 << 31) - 200000, 129, 1), ((1 << 31) - 1, 1 << 30, 2)):
        assert _bwd(num_rows=rows, num_tokens=tokens, dim=dim) == -3                    # as far as the workspace


def test_pipeline_refuses_a_codebook():
    """It reads _features_dc and _features_rest, which a model with a codebook may have beside it."""
    from types import SimpleNamespace
    from fdgs.embedding import FeatureCodebook
    from fdgs.pipeline import ViewPipeline
    model = SimpleNamespace(scaling_activation=torch.exp, opacity_activation=torch.sigmoid, rotation_activation=torch.nn.functional.normalize)
    pipe = ViewPipeline(model, None, torch.zeros(3))
    assert pipe.usable("coarse")
    model.feature_codebook = FeatureCodebook(torch.zeros(3, 16, 3), torch.tensor([0, 2]))
    assert not pipe.usable("coarse")
    with pytest.raises(ValueError, match="feature_codebook"):
        pipe.run(None, None, 1.0, "coarse")


def test_surgery_refuses_a_codebook_beside_the_groups_that_it_moves():
    """The ids would stay where they are while the Gaussians move."""
    from types import SimpleNamespace
    from fdgs.densify import PARAM_NAMES, GaussianSurgery
    from fdgs.embedding import FeatureCodebook
    model = SimpleNamespace(feature_codebook=FeatureCodebook(torch.zeros(3, 16, 3), torch.tensor([0, 2])))
    groups = [{"name": k, "params": [torch.zeros(2, 3, requires_grad=True)]} for k in PARAM_NAMES]
    surgery = GaussianSurgery(model, SimpleNamespace(param_groups=groups, state={}))
    with pytest.raises(ValueError, match="f_dc and f_rest"):
        surgery.apply_classes(torch.zeros(2, dtype=torch.uint8))

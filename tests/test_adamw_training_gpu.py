"""GPU: fdgs.adamw.FusedAdamW as an optimizer (groups, states, checkpoints), in the training step and under the densification
surgery; and a codebook's lookup, gradient and step together in a render."""
import math

import numpy as np
import pytest
import torch

import adamw_cases as ac

pytestmark = pytest.mark.gpu
U = ac.U


def _params(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    shapes = [(700, 3), (257,), (64, 48), (1,), (5, 16, 3)]
    return [torch.randn(s, generator=g).to(dtype).cuda().requires_grad_(True) for s in shapes]


def _groups(ps):
    return [{"params": ps[:2], "lr": 1e-2, "name": "a"}, {"params": ps[2:4], "lr": 3e-3, "weight_decay": 0.0, "name": "b"},
            {"params": ps[4:], "lr": 1e-3, "betas": (0.8, 0.99), "name": "c"}]


def _set_grads(ps, step, skip=()):
    g = torch.Generator().manual_seed(100 + step)
    for i, p in enumerate(ps):
        x = torch.randn(p.shape, generator=g).to(p.dtype).cuda()
        p.grad = None if i in skip else x


def _weights(opt, p):
    if p.dtype is torch.float32:
        return p.detach().cpu().numpy().astype(np.float64)
    low = opt.state[p]["residual"] if p in opt.state else torch.zeros_like(p, dtype=torch.int16)
    bits = (p.detach().view(torch.int16).to(torch.int32) << 16) + low.to(torch.int32)
    return bits.view(torch.float32).cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_of_groups_against_the_formula(dtype):
    """Five steps; one tensor joins at the third.  Errors add up: m keeps what the steps before left (3 u a step, less than
    30 u of its largest terms), v likewise (4 u a step for five steps), the weight 4 u a step; the update at most 60 u."""
    from fdgs.adamw import FusedAdamW
    ps = _params(dtype)
    opt = FusedAdamW(_groups(ps), weight_decay=0.1)
    want = [_weights(opt, p) for p in ps]
    m, v, t = ([np.zeros(p.shape) for p in ps] for _ in range(3))
    t = [0] * len(ps)
    hyper = [(1e-2, 0.1, 0.9, 0.999)] * 2 + [(3e-3, 0.0, 0.9, 0.999)] * 2 + [(1e-3, 0.1, 0.8, 0.99)]
    moved = [np.zeros(p.shape) for p in ps]
    for step in range(5):
        _set_grads(ps, step, skip=(1,) if step < 2 else ())
        opt.step()
        for i, p in enumerate(ps):
            if p.grad is None:
                continue
            lr, wd, b1, b2 = hyper[i]
            t[i] += 1
            before = want[i]
            want[i], m[i], v[i] = ac.adamw64(before, p.grad.float().cpu().numpy(), m[i], v[i], t[i], lr, wd, b1, b2, 1e-8)
            moved[i] = moved[i] + np.abs(want[i] - before * (1 - lr * wd))
            # |m| / sqrt(v) <= 1 / sqrt(1 - b2) times the roots' corrections: what m's error can move the weight by
            moved[i] = moved[i] + lr * (30.0 / 60.0) * np.sqrt((1 - b2 ** t[i]) / (1 - b2)) / (1 - b1 ** t[i])
    for i, p in enumerate(ps):
        assert opt.state[p]["step"] == t[i]
        off = np.abs(_weights(opt, p) - want[i])
        assert (off <= 60 * U * moved[i] + 5 * 4.04 * U * (np.abs(want[i]) + moved[i]) + 1e-38).all(), (i, off.max())
    opt.zero_grad()
    assert all(p.grad is None for p in ps)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_restored_optimizer_goes_on_with_the_same_bits(bits, dtype, tmp_path):
    from fdgs.adamw import FusedAdamW
    ps = _params(dtype)
    opt = FusedAdamW(_groups(ps), state_bits=bits, seed=7)
    for step in range(3):
        _set_grads(ps, step)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    other = FusedAdamW(_groups(qs), state_bits=bits, seed=7, lr=5.0)
    other.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    for step in range(3, 5):
        for xs, o in ((ps, opt), (qs, other)):
            _set_grads(xs, step)
            o.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        if bits == 8:
            assert torch.equal(opt.state[p]["exp_avg"].codes, other.state[q]["exp_avg"].codes)


def test_states_of_other_optimizers_are_taken():
    """A state of torch.optim.AdamW, of FusedAdam, and of the other width: the moments are those, to the nearest in 8 bits."""
    from fdgs.adam import FusedAdam
    from fdgs.adamw import FusedAdamW, pack8, unpack8
    for make in (lambda ps: torch.optim.AdamW(_groups(ps)),
                 lambda ps: FusedAdam([{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:4], "lr": 1e-2}, {"params": ps[4:], "lr": 1e-3}]),
                 lambda ps: FusedAdamW(_groups(ps))):
        ps = _params(torch.float32)
        src = make(ps)
        for step in range(2):
            _set_grads(ps, step)
            src.step()
        eight, wide = (FusedAdamW(_groups(_params(torch.float32)), state_bits=b) for b in (8, 32))
        eight.load_state_dict(src.state_dict())
        wide.load_state_dict(eight.state_dict())
        for p, a, b in zip(ps, (p for g in eight.param_groups for p in g["params"]), (p for g in wide.param_groups for p in g["params"])):
            for k, signed in (("exp_avg", True), ("exp_avg_sq", False)):
                packed = pack8([src.state[p][k]], signed)[0]
                assert torch.equal(packed.codes, eight.state[a][k].codes) and torch.equal(packed.exponents, eight.state[a][k].exponents)
                assert torch.equal(unpack8([packed])[0], wide.state[b][k])
            assert eight.state[a]["step"] == wide.state[b]["step"] == 2
    # and torch.optim.AdamW takes a 32-bit one
    theirs = torch.optim.AdamW(_groups(ps))
    theirs.load_state_dict(src.state_dict())
    assert all(torch.equal(theirs.state[p]["exp_avg"], src.state[p]["exp_avg"]) for p in ps)


def test_a_step_is_seen_by_saved_graphs():
    """A backward pass over a parameter that was stepped after its forward pass raises, as with torch's optimizers."""
    from fdgs.adamw import FusedAdamW
    p = torch.ones(8, device="cuda", requires_grad=True)
    opt = FusedAdamW([p])
    loss = (p * p).sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def _scene(n=3000, w=96, h=64):
    from fdgs import scene_synth as ss
    from fdgs.deformation import DeformationFields
    from fdgs.renderer import render
    from fdgs.train_step import DeformHolder
    dev = torch.device("cuda:0")
    g = ss.GaussianParams(n, device=dev, scale_mult=3.0)
    torch.manual_seed(ss.SEED)
    net = ss.perturb_deformation_(DeformationFields(ss.DYNERF_NET_KWARGS)).to(dev)
    net.deformation_net.set_aabb(list(ss.SCENE_MAX), list(ss.SCENE_MIN))
    deforms = DeformHolder(net)
    cams = ss.make_cameras(3, w, h, device=dev)
    bg = torch.ones(3, device=dev)
    other = ss.GaussianParams(n, seed=ss.SEED + 100, device=dev, requires_grad=False, scale_mult=3.0)
    with torch.no_grad():
        for cam in cams:
            cam.original_image = render(cam, other, deforms, bg, stage="coarse")["render"].clamp(0, 1).clone()
    return g, deforms, cams, bg


@pytest.mark.parametrize("bits", [32, 8])
def test_training_step_and_surgery(bits):
    """TrainStep with FusedAdamW on the direct route (gradients that are column slices), a densification and a pruning in
    between: the moments of the Gaussians that stay are what they were, new ones have none."""
    from fdgs.adamw import FusedAdamW
    from fdgs.train_step import TrainStep
    g, deforms, cams, bg = _scene()
    step = TrainStep(g, deforms, bg, adamw={"state_bits": bits, "weight_decay": 0.01})
    assert isinstance(step.optimizer, FusedAdamW) and step.optimizer.param_groups[0]["eps"] == 1e-15
    first = g._features_rest.detach().clone()
    for k in range(3):
        loss = step(cams, iteration=k + 1)
    assert torch.isfinite(loss) and not torch.equal(first, g._features_rest)
    groups = {gr["name"]: gr["params"][0] for gr in step.optimizer.param_groups if len(gr["params"]) == 1}
    before = {k: step.optimizer.moments(p) for k, p in groups.items()}
    n = g._xyz.shape[0]
    out = step.densify(float((step.xyz_gradient_accum / step.denom.clamp_min(1)).median()), 1.0)
    assert out["clones"] + out["splits"] > 0
    keep = out["survivors"]
    after = {gr["name"]: step.optimizer.moments(gr["params"][0]) for gr in step.optimizer.param_groups
             if len(gr["params"]) == 1 and gr["name"] in groups}
    for k in ("xyz", "f_rest", "opacity"):
        for i, (old, new) in enumerate(zip(before[k], after[k])):
            assert new.shape[0] == out["rows"] and (new[keep:] == 0).all()
            # the survivors in their old order: every row of theirs is among the old ones, and so are the sums.  In 8 bits a
            # new block's largest value may push a value below its smallest code: 2^-15 (2^-31) of that largest at most
            x, y = old.double().cpu(), new[:keep].double().cpu()
            if out["splits"] == 0:
                assert (x[:keep] - y).abs().max() <= (0 if bits == 32 else x.abs().max() * 2.0 ** (-15 if i == 0 else -31))
            assert y.abs().max() <= x.abs().max()
            assert y.abs().sum() <= x.abs().sum() + keep * x.abs().max() * (0 if bits == 32 else 2.0 ** -31)
    step(cams, iteration=4)
    step.prune(0.05, 1.0, None)
    step.reset_opacity()
    assert (step.optimizer.moments(g._opacity)[0] == 0).all()
    loss = step(cams, iteration=5)
    assert torch.isfinite(loss) and step.optimizer.state[g._xyz]["step"] >= 3 and g._xyz.shape[0] != n


class _CodebookModel:
    """A model whose SH coefficients are rows of a table, with the tensor layout render() asks for."""

    def __init__(self, g, table, ids):
        from fdgs.embedding import FeatureCodebook
        self._xyz, self._scaling, self._rotation, self._opacity = g._xyz, g._scaling, g._rotation, g._opacity
        self.feature_codebook = FeatureCodebook(table, ids).cuda()
        for k in ("max_sh_degree", "active_sh_degree", "scaling_activation", "opacity_activation", "rotation_activation"):
            setattr(self, k, getattr(g, k))

    @property
    def get_xyz(self):
        return self._xyz

    def parameters(self):
        return [self._xyz, self._scaling, self._rotation, self._opacity, self.feature_codebook.table]


@pytest.mark.parametrize("stage", ["coarse", "fine"])
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_codebook_in_a_render(stage, idt):
    """render() of a model with a codebook is render() of the model with the looked-up coefficients, and the table's gradient
    the sum of theirs (the rasterizer adds with atomics: 2e-5 of the largest, the bound the data-parallel test holds)."""
    from fdgs.renderer import render
    g, deforms, cams, bg = _scene()
    gen = torch.Generator().manual_seed(5)
    n, v = g._xyz.shape[0], 37
    table = torch.cat([torch.randn(v, 1, 3, generator=gen), 0.1 * torch.randn(v, 15, 3, generator=gen)], 1)
    ids = torch.randint(0, v - 1, (n,), generator=gen).to(idt)
    model = _CodebookModel(g, table, ids)
    flat = table.cuda()[ids.cuda().long()].requires_grad_(True)

    class Flat(_CodebookModel):
        feature_codebook = None

        def __init__(self):
            self.__dict__.update({k: x for k, x in model.__dict__.items() if k != "feature_codebook"})
        get_features = flat
    gy = torch.rand(3, 64, 96, generator=gen).cuda()
    ims = []
    for m in (model, Flat()):
        im = render(cams[0], m, deforms, bg, stage=stage)["render"]
        (im * gy).sum().backward()
        ims.append(im.detach())
    assert torch.equal(*ims)
    got = model.feature_codebook.table.grad.double().cpu()
    want = torch.zeros(v, 16, 3, dtype=torch.float64).index_add_(0, ids.long(), flat.grad.double().cpu())
    size = torch.zeros(v, 16, 3, dtype=torch.float64).index_add_(0, ids.long(), flat.grad.double().abs().cpu())
    assert (got - want).abs().max() <= 2e-5 * size.abs().max() and (got[v - 1] == 0).all() and want.abs().max() > 0
    with torch.no_grad():
        assert torch.equal(render(cams[0], model, deforms, bg, stage=stage)["render"], ims[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_lookup_gradient_and_step_together(bits):
    """A training step over a codebook: the table moves by the formula on the gradient that the lookup's backward gave."""
    from fdgs.train_step import TrainStep
    g, deforms, cams, bg = _scene()
    gen = torch.Generator().manual_seed(6)
    table = torch.cat([torch.randn(50, 1, 3, generator=gen), 0.1 * torch.randn(50, 15, 3, generator=gen)], 1)
    model = _CodebookModel(g, table, torch.randint(0, 50, (g._xyz.shape[0],), generator=gen))
    step = TrainStep(model, deforms, bg, adamw={"state_bits": bits, "weight_decay": 0.05})
    names = [gr["name"] for gr in step.optimizer.param_groups]
    assert "codebook" in names and "f_dc" not in names
    seen = {}
    p = model.feature_codebook.table
    loss = step(cams, iteration=1, before_optimizer_step=lambda s: seen.update(grad=p.grad.clone(), before=p.detach().clone()))
    assert torch.isfinite(loss) and seen["grad"].abs().max() > 0
    zero = np.zeros(p.shape)
    w64, m64, v64 = ac.adamw64(seen["before"].cpu().numpy(), seen["grad"].cpu().numpy(), zero, zero, 1, 0.0025, 0.05, 0.9, 0.999, 1e-15)
    update = np.abs(w64 - seen["before"].cpu().numpy().astype(np.float64) * (1 - 0.0025 * 0.05))
    off = np.abs(p.detach().cpu().numpy() - w64)
    # m three, v four roundings (the root halves v's), the update twelve, the weight four
    assert (off <= 15.3 * U * update + 4.04 * U * np.abs(w64) + 1e-12).all(), off.max()
    with pytest.raises(ValueError, match="f_dc"):
        step.densify(0.0, 1.0)
    assert math.isfinite(float(step(cams, iteration=2)))


@pytest.mark.parametrize("stage", ["coarse", "fine"])
def test_a_rank_without_views_exchanges_the_codebooks_gradient(stage, monkeypatch):
    """The exchange adds up the gradients that there are: the same tensors have one on a rank that has views and on one that has none,
    the codebook's table among them also where the model's parameters() does not name it."""
    from fdgs import dp
    from fdgs.embedding import FeatureCodebook
    from fdgs.train_step import TrainStep
    have = []
    for views in (True, False):
        g, deforms, cams, bg = _scene()
        gen = torch.Generator().manual_seed(7)
        g.feature_codebook = FeatureCodebook(0.1 * torch.randn(20, 16, 3, generator=gen), torch.randint(0, 20, (g._xyz.shape[0],), generator=gen)).cuda()
        assert all(p is not g.feature_codebook.table for p in g.parameters())
        step = TrainStep(g, deforms, bg, stage=stage)
        seen = {}
        with monkeypatch.context() as m:
            m.setattr(dp, "is_dist", lambda: True)
            m.setattr(dp, "all_reduce_", lambda *a, **k: None)
            if not views:
                m.setattr(dp, "shard_views", lambda v: [])
            step(cams, before_optimizer_step=lambda s: seen.update(grads=[p.grad is not None for p in s.params],
                                                                   table=g.feature_codebook.table.grad is not None))
        assert seen["table"]
        have.append(seen["grads"])
    assert have[0] == have[1]


@pytest.mark.parametrize("bits", [32, 8])
def test_surgery_moves_every_moment_with_its_gaussian(bits):
    """Known classes: the moments of those that stay follow them in their old order, clones and children begin with none.  In 8 bits the
    new blocks of 256 are the format's, to the nearest, of the old values."""
    from fdgs import _lib
    from fdgs.train_step import TrainStep
    g, deforms, cams, bg = _scene(n=1501)
    step = TrainStep(g, deforms, bg, adamw={"state_bits": bits})
    for k in range(2):
        step(cams, iteration=k + 1)
    names = ("xyz", "f_dc", "f_rest", "opacity", "scaling", "rotation")

    def moments():
        params = {gr["name"]: gr["params"][0] for gr in step.optimizer.param_groups if gr["name"] in names}
        return {k: [m.cpu().numpy() for m in step.optimizer.moments(params[k])] for k in names}

    def stored(x, signed):
        if bits == 32:
            return x
        flat = np.ascontiguousarray(x).reshape(-1)
        return ac.decode(*ac.encode(flat, 0x8000, signed), signed).reshape(x.shape)

    gen = torch.Generator().manual_seed(0)
    for kind in ("densify", "prune"):
        n = g._xyz.shape[0]
        before, steps = moments(), step.optimizer.state[g._xyz]["step"]
        draw = torch.rand(n, generator=gen)
        if kind == "densify":
            cls = torch.full((n,), _lib.CLS_KEEP, dtype=torch.uint8)
            cls[draw < 0.3], cls[draw < 0.2], cls[draw < 0.1] = _lib.CLS_CLONE, _lib.CLS_SPLIT, _lib.CLS_DROP
            stay = (cls == _lib.CLS_KEEP) | (cls == _lib.CLS_CLONE)
            out = step.surgery().apply_classes(cls.cuda())
            assert out["clones"] == int((cls == _lib.CLS_CLONE).sum()) > 0 and out["splits"] == int((cls == _lib.CLS_SPLIT).sum()) > 0
        else:
            stay = draw > 0.25
            out = step.surgery().prune_points((~stay).cuda())
        rows = g._xyz.shape[0]
        assert out["survivors"] == int(stay.sum()) < n and out["rows"] == rows
        after = moments()
        for k in names:
            for old, new, signed in zip(before[k], after[k], (True, False)):
                assert (old != 0).any()
                want = np.zeros((rows, *old.shape[1:]), np.float32)
                want[:out["survivors"]] = old[stay.numpy()]
                assert new.shape == want.shape and np.array_equal(new, stored(want, signed)), (kind, k, signed)
        assert step.optimizer.state[g._xyz]["step"] == steps

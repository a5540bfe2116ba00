"""GPU: fdgs_adamw_step and the 8-bit moments' conversions against the formula in 64 bits and the format in integers.

Tolerances count roundings (u = 2^-24, half a float32 step): of m three on each of its two terms, of v four, of the
update twelve beside what m is off by, of the weight four (constant, product, difference, and one to spare)."""
import math

import numpy as np
import pytest
import torch

import adamw_cases as ac

pytestmark = pytest.mark.gpu
U = ac.U


def _inputs(sizes, seed, spread=4.0):
    rng = np.random.default_rng(seed)
    out = []
    for n in sizes:
        scale = 10.0 ** rng.uniform(-spread, 0)
        g = (rng.standard_normal(n) * scale).astype(np.float32)
        g[rng.random(n) < 0.2] = 0.0
        m = (0.3 * g + 0.1 * scale * rng.standard_normal(n)).astype(np.float32)
        v = ((scale * rng.random(n)) ** 2).astype(np.float32)
        v[rng.random(n) < 0.1] = 0.0
        w = (0.1 * rng.standard_normal(n)).astype(np.float32)
        out.append((w, g, m, v))
    return out


def _bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16)


class Arena:
    """Tensors cut from one array, `skew` elements off its alignment, with a marked gap between them."""

    def __init__(self, arrays, dtype, skew, mark):
        at, self.at = skew, []
        for a in arrays:
            self.at.append(at)
            at += len(a) + 3
        self.flat = torch.full((at + 5,), mark, dtype=dtype)
        for o, a in zip(self.at, arrays):
            self.flat[o:o + len(a)] = torch.as_tensor(a).to(dtype)
        self.flat = self.flat.cuda()
        self.views = [self.flat[o:o + len(a)] for o, a in zip(self.at, arrays)]
        self.before = self.flat.clone()

    def gaps_untouched(self):
        inside = torch.zeros(self.flat.numel(), dtype=torch.bool)
        for o, v in zip(self.at, self.views):
            inside[o:o + v.numel()] = True
        return torch.equal(self.flat.cpu()[~inside], self.before.cpu()[~inside])


SIZES = [1, 3, 4, 63, 255, 256, 257, 511, 512, 513, 2047, 2048, 2049, 5001, 0, 70001]


def _within(got, want, tol, what):
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (what, float((err - tol).max()), int((err > tol).sum()))


@pytest.mark.parametrize("skew", [0, 1, 2, 3])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_against_the_formula(dtype, bits, skew):
    from fdgs import adamw
    b1, b2, eps = 0.9, 0.999, 1e-8
    data = _inputs(SIZES, 17 * skew + bits)
    bf16 = dtype is torch.bfloat16
    lrs = [1e-3 * (1 + i % 3) for i in range(len(data))]
    wds = [0.0 if i % 4 == 0 else 0.1 for i in range(len(data))]
    steps = [1 + 7 * i for i in range(len(data))]
    keys = [adamw.round_key(5, i, s) for i, s in enumerate(steps)]
    g_in = [(_bf16(d[1]).float().numpy() if bf16 else d[1]) for d in data]
    low = Arena([ac.split_bf16(d[0])[1] for d in data], torch.int16, skew, 77) if bf16 else None
    if bf16:
        p = Arena([np.zeros(len(d[0])) for d in data], dtype, skew, 9.0)
        for view, d in zip(p.views, data):
            view.copy_(torch.from_numpy(ac.split_bf16(d[0])[0].view(np.int16).copy()).view(torch.bfloat16).cuda())
    else:
        p = Arena([d[0] for d in data], dtype, skew, 9.0)
    g = Arena(g_in, dtype, skew, float("nan"))
    if bits == 32:
        m = Arena([d[2] for d in data], torch.float32, skew, 9.0)
        v = Arena([d[3] for d in data], torch.float32, skew, 9.0)
        old = [(d[2], d[3]) for d in data]
        adamw.adamw_step(p.views, g.views, m.views, v.views, steps=steps, lr=lrs, betas=(b1, b2), eps=eps, weight_decay=wds,
                         residuals=low.views if bf16 else None)
        new = [(a.cpu().numpy(), b.cpu().numpy()) for a, b in zip(m.views, v.views)]
        states = [m, v]
    else:
        em, ev = ([ac.encode(d[k], 0x8000, k == 2) for d in data] for k in (2, 3))
        old = [(ac.decode(*a, True), ac.decode(*b, False)) for a, b in zip(em, ev)]
        mc, vc = (Arena([x[0] for x in e], torch.uint8, skew, 201) for e in (em, ev))
        me, ve = (Arena([x[1] for x in e], torch.uint8, skew, 201) for e in (em, ev))
        adamw.adamw_step(p.views, g.views, [adamw.Moment8(a, b, True) for a, b in zip(mc.views, me.views)],
                         [adamw.Moment8(a, b, False) for a, b in zip(vc.views, ve.views)], steps=steps, lr=lrs, betas=(b1, b2),
                         eps=eps, weight_decay=wds, residuals=low.views if bf16 else None, keys=keys)
        states = [mc, vc, me, ve]
    for i, (d, (m0, v0)) in enumerate(zip(data, old)):
        w64, m64, v64 = ac.adamw64(d[0], g_in[i], m0, v0, steps[i], lrs[i], wds[i], b1, b2, eps)
        mtol = 3.03 * U * (b1 * np.abs(m0) + (1 - b1) * np.abs(g_in[i])) + 2.0 ** -149
        vtol = 4.04 * U * v64 + 2.0 ** -147
        if bits == 32:
            _within(new[i][0], m64, mtol, "m")
            _within(new[i][1], v64, vtol, "v")
        else:       # the codes are those of the format, bit by bit
            m32, v32 = ac.adamw32(g_in[i], m0, v0, b1, b2)
            h = ac.hash32(np.arange(len(m32)), keys[i])
            for got, e, want in ((mc, me, ac.encode(m32, h >> 16, True)), (vc, ve, ac.encode(v32, h & 0xFFFF, False))):
                assert np.array_equal(got.views[i].cpu().numpy(), want[0]) and np.array_equal(e.views[i].cpu().numpy(), want[1])
        if bf16:
            bits_p = p.views[i].cpu().view(torch.int16).numpy().astype(np.int64)
            w = ((bits_p << 16) + low.views[i].cpu().numpy()).astype(np.int32).view(np.float32)
            off = np.abs(w.astype(np.float64) - p.views[i].cpu().float().numpy())
            assert (off <= 2.0 ** -8 * np.abs(w) * (1 + 2.0 ** -8) + 2.0 ** -134).all()     # the parameter is the nearest one
        else:
            w = p.views[i].cpu().numpy()
        lr, bc1, bc2 = lrs[i], 1 - b1 ** steps[i], 1 - b2 ** steps[i]
        denom = np.sqrt(v64 / bc2) + eps
        update = np.abs(lr / bc1 * m64 / denom)
        tol = 12.2 * U * update + 1.01 * lr / bc1 * mtol / denom + 4.04 * U * np.abs(d[0]) + 2.0 ** -149
        # where v is below the normal numbers its own roundings count for more than u
        tol += update * np.where(v64 > 0, 2.0 ** -147 / np.maximum(v64, 2.0 ** -149), 0.0)
        _within(w, w64, tol, "w")
    for a in [p] + ([low] if bf16 else []) + states:
        assert a.gaps_untouched()
    assert torch.equal(g.flat.cpu().isnan(), g.before.cpu().isnan())


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_as_column_slices_and_other_orders(bits):
    """Gradients read from the columns of a wider array, expanded from one row or in another order give the bits that
    a contiguous copy gives."""
    from fdgs import adamw
    gen = torch.Generator().manual_seed(3)
    n = 1037
    wide = torch.randn(n, 48, generator=gen).cuda()
    grads = [wide[:, :3], wide[:, 3:], wide[:, 7:8], wide.t()[:5], wide[:1, :8].expand(n, 8), wide[::2, 5:9]]

    def run(copy):
        ps = [torch.linspace(-1, 1, g.numel(), device="cuda").view(g.shape) for g in grads]
        make = (lambda p, s: adamw.Moment8.zeros_like(p, s)) if bits == 8 else (lambda p, s: torch.zeros_like(p))
        ms, vs = [make(p, True) for p in ps], [make(p, False) for p in ps]
        for t in (1, 2):
            adamw.adamw_step(ps, [g.contiguous() if copy else g for g in grads], ms, vs, steps=t, lr=1e-2,
                             keys=[adamw.round_key(1, i, t) for i in range(len(ps))] if bits == 8 else None)
        return ps + [x for s in ms + vs for x in ((s.codes, s.exponents) if bits == 8 else (s,))]
    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("signed", [True, False])
def test_pack_and_unpack(signed):
    from fdgs import adamw
    rng = np.random.default_rng(8)
    arrays = []
    for n in (1, 255, 256, 257, 4099):
        x = (rng.standard_normal(n) * 10.0 ** rng.uniform(-12, 2, n)).astype(np.float32)
        arrays.append(np.where(rng.random(n) < 0.2, np.float32(0), x if signed else np.abs(x)).astype(np.float32))
    arrays.append(np.zeros(300, np.float32))
    arrays.append((rng.random(700) * 2.0 ** -140).astype(np.float32))            # below the normal numbers
    arrays.append(np.full(256, np.float32(1.9999999)))                           # rounds up into the next power of two
    arrays.append(np.where(np.arange(512) == 5, np.float32("inf"), np.float32(1)).astype(np.float32))
    arrays.append(np.where(np.arange(512) == 300, np.float32("nan"), np.float32(1)).astype(np.float32))
    arrays.append(np.full(256, np.float32(3e38)))
    dev = [torch.from_numpy(a).cuda() for a in arrays]
    keys = [adamw.round_key(2, i, 1) for i in range(len(arrays))]
    for ks in (None, keys):
        packed = adamw.pack8(dev, signed, ks)
        for i, (a, p) in enumerate(zip(arrays, packed)):
            h = ac.hash32(np.arange(a.size), keys[i])
            noise = 0x8000 if ks is None else (h >> 16 if signed else h & 0xFFFF)
            code, e = ac.encode(a, noise, signed)
            assert np.array_equal(p.codes.cpu().numpy(), code) and np.array_equal(p.exponents.cpu().numpy(), e), i
        values = adamw.unpack8(packed)
        halves = adamw.unpack8(packed, torch.bfloat16)
        for a, p, x, y in zip(arrays, packed, values, halves):
            want = ac.decode(p.codes.cpu().numpy(), p.exponents.cpu().numpy(), signed)
            assert np.array_equal(x.cpu().numpy(), want, equal_nan=True)
            assert np.array_equal(y.float().cpu().numpy(), want, equal_nan=True)           # bfloat16 holds them exactly
            ok = np.repeat(p.exponents.cpu().numpy() != 255, 256)[:a.size]
            a64, x64 = np.abs(a[ok].astype(np.float64)), np.abs(want[ok].astype(np.float64))
            if not signed:
                assert ((a64 > 0) == (x64 > 0)).all()          # a second moment that is not zero stays so
            # within one step of the grid (half of one to the nearest): an eighth of the power of two, the block's
            # largest times 2^-15 or 2^-31 at the small end
            top = np.repeat(2.0 ** (p.exponents.cpu().numpy().astype(np.float64) - 126), 256)[:a.size][ok]
            low = np.maximum(top * 2.0 ** (-15.6 if signed else -31.6), 2.0 ** -128.9)
            step = np.where(a64 > 0, 2.0 ** (np.floor(np.log2(np.maximum(a64, 2.0 ** -149))) - 3), 0)
            limit = (0.5 if ks is None else 1.0) * np.maximum(step, 2.0 ** -129)
            far = np.abs(a64 - x64) > limit * (1 + 2.0 ** -15)
            assert (~far | (a64 <= low)).all() and (np.abs(a64 - x64)[far] <= low[far]).all()
        again = adamw.pack8(values, signed)                    # what is on the grid stays where it is
        for x, p, q in zip(values, packed, again):             # (but for the smallest, where the largest has rounded up)
            same, x = adamw.unpack8([q])[0].cpu().numpy(), x.cpu().numpy()
            top = np.repeat(2.0 ** (q.exponents.cpu().numpy().astype(np.float64) - 126), 256)[:x.size]
            there = ~(np.abs(x) < top * 2.0 ** (-14.6 if signed else -30.6))
            assert np.array_equal(same[there], x[there], equal_nan=True)


def test_rounding_keeps_the_mean():
    """A value between two codes is stored as either, with the mean of what it is: 2^18 elements, five standard
    deviations of the mean of so many draws plus what 16 random bits cannot resolve."""
    from fdgs import adamw
    n = 1 << 18
    for x in (1.0009, 1.05, 1.1, 1.9):
        values = torch.full((n,), x, device="cuda")
        for signed in (True, False):
            mean = float(adamw.unpack8(adamw.pack8([values], signed, [adamw.round_key(9, 0, 3)]))[0].double().mean())
            f = (np.float32(x) - 1.0) * 8 % 1
            sigma = 0.125 * math.sqrt(f * (1 - f) / n)
            assert abs(mean - float(np.float32(x))) <= 5 * sigma + 0.125 * 2.0 ** -16, (x, signed, mean)


def test_second_moment_follows_a_falling_gradient():
    """With beta2 = 0.999 a moment cut to the nearest code would stay where it is; the drawn cut follows.  v falls as
    0.999^k; after 2000 steps without gradient the mean over 2^16 elements is 0.135 of the start.  A step that moves v by
    d between points s apart has a variance of at most s d <= (v / 8) (0.001 v), so the variance relative to the mean
    squared, r, grows by at most 1.25e-4 (1 + r) a step, to e^0.25 - 1 = 0.284: five deviations of the mean of 65536 are
    1.04 percent.  16 random bits are off by 2^-16 of s a step, the float32 products by 2 u a step."""
    from fdgs import adamw
    n, k = 1 << 16, 2000
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    m = adamw.Moment8.zeros_like(p, True)
    v, = adamw.pack8([torch.full((n,), 0.37, device="cuda")], False)
    start = float(adamw.unpack8([v])[0][0])
    for t in range(1, k + 1):
        adamw.adamw_step([p], [g], [m], [v], steps=t, lr=0.0, keys=[adamw.round_key(4, 0, t)])
    mean = float(adamw.unpack8([v])[0].double().mean())
    assert abs(mean / (start * 0.999 ** k) - 1) <= 0.0104 + k * 2.0 ** -16 * 0.125 + 2 * k * U


@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_not_finite_stays_where_it_is(bits):
    """A NaN or infinite gradient makes its own element NaN, and with 8-bit moments its block of 256 from the next step on;
    every other element keeps the bits it would have had."""
    from fdgs import adamw
    n = 1024
    gen = torch.Generator().manual_seed(6)
    g = torch.randn(n, generator=gen).cuda()
    bad = g.clone()
    bad[300], bad[301] = float("nan"), float("inf")

    def run(grad):
        p = torch.ones(n, device="cuda")
        m = adamw.Moment8.zeros_like(p, True) if bits == 8 else torch.zeros(n, device="cuda")
        v = adamw.Moment8.zeros_like(p, False) if bits == 8 else torch.zeros(n, device="cuda")
        for t in (1, 2):
            adamw.adamw_step([p], [grad if t == 1 else g], [m], [v], steps=t, lr=0.1, keys=[t] if bits == 8 else None)
        return p.cpu(), [x.cpu() for x in (adamw.unpack8([m, v]) if bits == 8 else (m, v))]
    pa, sa = run(g)
    pb, sb = run(bad)
    hit = torch.zeros(n, dtype=torch.bool)
    hit[256:512 if bits == 8 else 256] = True
    hit[300] = hit[301] = True
    assert torch.equal(pa[~hit], pb[~hit]) and pb[hit].isnan().all()
    for a, b in zip(sa, sb):
        assert torch.equal(a[~hit], b[~hit])
    assert sb[0][hit].isnan().all() if bits == 8 else not sb[0][hit].isfinite().any()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30, 1e-15])
def test_moments_below_the_normal_numbers(bits, eps):
    """Gradients whose squares are below the smallest normal float32 (and, in the first block, ordinary ones beside them): the
    update is the formula's, with what v's evenly spaced numbers there leave of it (2^-148 for each of four roundings)."""
    from fdgs import adamw
    rng = np.random.default_rng(3)
    n = 1024
    g = (10.0 ** rng.uniform(-22, -19, n) * np.where(rng.random(n) < 0.5, -1, 1)).astype(np.float32)
    g[:100] = rng.standard_normal(100)
    p, m, v = (torch.zeros(n, device="cuda") for _ in range(3))
    if bits == 8:
        m, v = adamw.Moment8.zeros_like(p, True), adamw.Moment8.zeros_like(p, False)
    adamw.adamw_step([p], [torch.from_numpy(g).cuda()], [m], [v], steps=1, lr=1e-3, eps=eps, keys=[1] if bits == 8 else None)
    zero = np.zeros(n)
    w64, m64, v64 = ac.adamw64(zero, g, zero, zero, 1, 1e-3, 0.01, 0.9, 0.999, eps)
    off = 4 * 2.0 ** -148
    lo, hi = (1e-3 * np.abs(g) / (np.sqrt(np.maximum(v64 + s * off, 0.0) / (1 - 0.999)) + eps * (1 - s * U) - s * 2.0 ** -149)
              for s in (1, -1))
    hi = np.where((hi > 0) & (v64 > off), hi, np.inf)       # v itself may be rounded to nothing
    got = np.abs(p.cpu().numpy().astype(np.float64))
    rel = 15.3 * U
    ok = got >= lo * (1 - rel) - 2.0 ** -149
    ok &= (got <= hi * (1 + rel)) | ~np.isfinite(got)
    assert ok.all() and np.isfinite(got[v64 > 2 * off]).all(), int((~ok).sum())
    assert (np.sign(p.cpu().numpy())[v64 > 2 * off] == -np.sign(g)[v64 > 2 * off]).all()


def test_bfloat16_weights_gather_small_updates():
    """1000 steps of 1e-5 on weights of 1, where bfloat16's step is 2^-7: the parameter follows the float32 weight."""
    from fdgs import adamw
    n = 513
    p = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    low = torch.zeros(n, device="cuda", dtype=torch.int16)
    g = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for t in range(1, 1001):
        adamw.adamw_step([p], [g], [m], [v], steps=t, lr=1e-5, weight_decay=0.0, residuals=[low])
    w = ((p.view(torch.int16).to(torch.int32) << 16) + low.to(torch.int32)).view(torch.float32).cpu().double()
    # a step moves by 1e-5 and rounds the weight, which lies between a half and one, by u / 2; the moments gather 3 u a
    # step for ten steps and 4 u a step for a thousand, half of which the root keeps: 2050 u of each update; eps 1e-8 of it
    assert (w - (1 - 1e-2)).abs().max() <= 1000 * (0.5 * U + 1e-5 * (2050 * U + 1e-8))
    assert torch.equal(p.float().cpu(), torch.full((n,), 0.98828125))       # 253.44 / 256, to the nearest


def test_bfloat16_parameter_written_from_outside_is_the_new_weight():
    from fdgs import adamw
    p = torch.ones(300, device="cuda", dtype=torch.bfloat16)
    low = torch.full((300,), 123, device="cuda", dtype=torch.int16)
    p.fill_(-2.5)
    adamw.adamw_step([p], [torch.zeros_like(p)], [torch.zeros(300, device="cuda")], [torch.zeros(300, device="cuda")],
                     steps=1, lr=1e-3, weight_decay=0.0, residuals=[low])
    assert (p.float() + 2.5).abs().max() == 0 and (low == 123).all()


def test_same_inputs_same_bits_on_any_stream():
    from fdgs import adamw
    data = _inputs([70001, 257, 4096], 2)

    def run(stream):
        ps, gs = [torch.from_numpy(d[0]).cuda() for d in data], [torch.from_numpy(d[1]).cuda() for d in data]
        ms, vs = ([f(torch.from_numpy(d[0]).cuda()) for d in data] for f in
                  (lambda x: adamw.Moment8.zeros_like(x, True), lambda x: adamw.Moment8.zeros_like(x, False)))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for t in (1, 2, 3):
                adamw.adamw_step(ps, gs, ms, vs, steps=t, lr=1e-2, keys=[t, t + 10, t + 20])
        torch.cuda.synchronize()
        return ps + [x.codes for x in ms + vs] + [x.exponents for x in ms + vs]
    for a, b in zip(run(torch.cuda.current_stream()), run(torch.cuda.Stream())):
        assert torch.equal(a, b)


def test_capture_is_refused_and_leaves_the_state_alone():
    from fdgs import adamw
    p, g = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    m, v = torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            adamw.adamw_step([p], [g], [m], [v], steps=1, lr=1e-3)
        q = p + 1
    graph.replay()
    torch.cuda.synchronize()
    assert (q == 2).all() and (p == 1).all() and (m == 0).all()


@pytest.mark.parametrize("count", [40, 41, 80, 81, 171, 400])
def test_more_tensors_than_one_launch_takes(count):
    """Lists at the limits of a launch's arguments, and of the table in device memory that longer ones go through."""
    from fdgs import adamw
    rng = np.random.default_rng(0)
    sizes = [int(n) for n in rng.integers(0, 700, count)]
    data = _inputs(sizes, 5)
    ps, gs, ms, vs = ([torch.from_numpy(d[k]).cuda() for d in data] for k in range(4))
    adamw.adamw_step(ps, gs, ms, vs, steps=3, lr=1e-3, weight_decay=0.0)
    for d, p, m in zip(data, ps, ms):
        w64, m64, v64 = ac.adamw64(*d, 3, 1e-3, 0.0, 0.9, 0.999, 1e-8)
        tol = 3.03 * U * (0.9 * np.abs(d[2]) + 0.1 * np.abs(d[1])) + 2.0 ** -149
        _within(m.cpu().numpy(), m64, tol, "m")
        denom = np.sqrt(v64 / (1 - 0.999 ** 3)) + 1e-8
        scale = 1e-3 / (1 - 0.9 ** 3) / denom
        _within(p.cpu().numpy(), w64, 12.2 * U * np.abs(m64) * scale + 1.01 * tol * scale + 4.04 * U * np.abs(d[0]) + 2.0 ** -149, "w")
    packed = adamw.pack8(ms, True)                               # and their conversions, there and back
    for m, x in zip(ms, adamw.unpack8(packed)):
        assert np.array_equal(x.cpu().numpy(), ac.decode(*ac.encode(m.cpu().numpy(), 0x8000, True), True))


def _small(bits, bf16, n=3):
    """Arguments of a step over n tensors that holds good."""
    from fdgs.adamw import Moment8
    kind = torch.bfloat16 if bf16 else torch.float32
    p, g = ([torch.ones(300 + i, dtype=kind, device="cuda") for i in range(n)] for _ in range(2))
    m, v = ([Moment8.zeros_like(x, signed) if bits == 8 else torch.zeros(x.shape, device="cuda") for x in p] for signed in (True, False))
    low = [torch.zeros(x.shape, dtype=torch.int16, device="cuda") for x in p]
    return dict(params=p, grads=g, exp_avgs=m, exp_avg_sqs=v, steps=1, lr=0.1, residuals=low if bf16 else None,
                keys=list(range(n)) if bits == 8 else None)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bf16", [False, True])
def test_step_refuses_and_changes_nothing(bits, bf16):
    from fdgs.adamw import Moment8, adamw_step
    dev, other = "cuda", torch.float32 if bf16 else torch.bfloat16
    kind = torch.bfloat16 if bf16 else torch.float32
    z = lambda n, t=kind: torch.zeros(n, dtype=t, device=dev)  # noqa: E731
    both = z(2 * 302 - 1)                                # two tensors that share an element
    cases = [("same length", dict(grads=lambda a: a[:2])), ("same length", dict(exp_avgs=lambda a: a + a[:1])),
             ("one type", dict(params=lambda a: [*a[:2], z(302, other)])), ("one type", dict(grads=lambda a: [*a[:2], z(302, other)])),
             ("contiguous", dict(params=lambda a: [*a[:2], z((302, 2))[:, 0]])), ("its size", dict(grads=lambda a: [*a[:2], z(301)])),
             ("one device", dict(grads=lambda a: [*a[:2], torch.zeros(302, dtype=kind)])),
             ("count from 1", dict(steps=lambda a: 0)), ("count from 1", dict(steps=lambda a: [1, 1, -3])),
             ("one value", dict(lr=lambda a: [0.1, 0.1])), ("one value", dict(steps=lambda a: [1])),
             ("twice", dict(params=lambda a: [a[0], a[1], a[0][:300]], grads=lambda a: [a[0], a[1], a[0]],
                            exp_avgs=lambda a: [a[0], a[1], a[0]], exp_avg_sqs=lambda a: [a[0], a[1], a[0]],
                            **({"residuals": lambda a: [a[0], a[1], a[0]]} if bf16 else {}))),
             ("overlap", dict(params=lambda a: [a[0], both[:301], both[300:602]]))]
    if bf16:
        cases += [("residual", dict(residuals=lambda a: None)), ("residual", dict(residuals=lambda a: a[:2])),
                  ("residual", dict(residuals=lambda a: [*a[:2], z(302, torch.int32)])),
                  ("overlap", dict(residuals=lambda a: [a[0], a[2][:301], a[2]]))]
    if bits == 8:
        cases += [("keys", dict(keys=lambda a: None)), ("keys", dict(keys=lambda a: a[:2])), ("do not mix", dict(exp_avgs=lambda a: [*a[:2], z(302, torch.float32)])),
                  ("the second is not", dict(exp_avgs=lambda a: [x._replace(signed=False) for x in a])),
                  ("one exponent per", dict(exp_avg_sqs=lambda a: [*a[:2], a[2]._replace(exponents=z(1, torch.uint8))])),
                  ("uint8", dict(exp_avg_sqs=lambda a: [*a[:2], a[2]._replace(codes=z(302, torch.int8))])),
                  ("overlap", dict(exp_avgs=lambda a: [x._replace(exponents=a[0].exponents) for x in a]))]
    else:
        cases += [("float32 tensors", dict(exp_avgs=lambda a: [*a[:2], z(302, torch.float16)])),
                  ("Moment8", dict(exp_avgs=lambda a: [*a[:2], Moment8.zeros_like(a[2], True)])),
                  ("overlap", dict(exp_avg_sqs=lambda a: [a[0], a[2][:301], a[2]]))]
    for match, change in cases:
        args = _small(bits, bf16)
        args.update({k: f(args[k]) for k, f in change.items()})
        before = [x.clone() for x in args["params"]]
        with pytest.raises((ValueError, TypeError), match=match):
            adamw_step(**args)
        assert all(torch.equal(x, y) for x, y in zip(before, args["params"])), match
    with pytest.raises(ValueError, match="not torch"):
        adamw_step([z(4, torch.float64)], [z(4, torch.float64)], [z(4)], [z(4)], steps=1, lr=0.1)
    args = _small(bits, bf16)
    adamw_step(**args)                                   # as they stand they are a step
    assert all((x != 1).all() for x in args["params"])


def test_conversions_refuse_overlapping_results():
    from fdgs.adamw import Moment8, pack8, unpack8
    ms = pack8([torch.ones(300, device="cuda"), torch.ones(300, device="cuda")], False)
    out = torch.zeros(599, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        unpack8(ms, out=[out[:300], out[299:]])
    with pytest.raises(ValueError, match="one type"):
        unpack8(ms, out=[out[:300], torch.zeros(300, dtype=torch.bfloat16, device="cuda")])
    with pytest.raises(ValueError, match="for each"):
        unpack8(ms, out=[out[:300]])
    with pytest.raises(ValueError, match="one code per"):
        unpack8(ms, out=[out[:300], out[300:]])
    assert (out == 0).all()
    assert unpack8([]) == [] and pack8([], True) == []
    with pytest.raises(ValueError, match="float32"):
        pack8([torch.ones(4, device="cuda", dtype=torch.bfloat16)], True)
    with pytest.raises(ValueError, match="one value"):
        pack8([torch.ones(4, device="cuda")], True, keys=[1, 2])
    assert isinstance(ms[0], Moment8)


@pytest.mark.parametrize("count", [3, 200])
def test_captured_conversions(count):
    """Values to codes and back in a graph (its records in the launch's arguments, or in a table that the graph fills again at
    every replay), replayed with new values and with eager conversions of other lists in between."""
    from fdgs.adamw import pack8, unpack8
    gen = torch.Generator().manual_seed(count)
    sizes = [int(n) for n in torch.randint(0, 900, (count,), generator=gen)]
    x = [torch.zeros(n, device="cuda") for n in sizes]
    signed = [i % 2 == 0 for i in range(count)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ms = pack8(x, signed)
        back = unpack8(ms)
    for k in range(3):
        new = [torch.randn(n, generator=gen).abs() * 10.0 ** (k - 1) for n in sizes]
        for a, b in zip(x, new):
            a.copy_(b)
        graph.replay()
        other = unpack8(pack8([v.cuda() + 1 for v in new], signed))      # eager, from a table of its own
        want = unpack8(pack8(x, signed))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(back, want)), k
        for v, m, s, b in zip(new, ms, signed, back):
            codes, exps = ac.encode(v.numpy(), 0x8000, s)
            assert np.array_equal(m.codes.cpu().numpy(), codes) and np.array_equal(m.exponents.cpu().numpy(), exps)
        del other


def test_long_lists_without_a_workspace():
    """Through the C ABI, without the device memory that one launch over all tensors needs: as many launches as it takes, and the
    same bits."""
    import ctypes as C
    from fdgs import _lib, _records
    from fdgs.adamw import Moment8, adamw_step, pack8, unpack8
    gen = torch.Generator().manual_seed(0)
    sizes = [int(n) for n in torch.randint(0, 600, (201,), generator=gen)]
    p = [torch.randn(n, generator=gen).cuda() for n in sizes]
    g = [torch.randn(n, generator=gen).cuda() for n in sizes]
    q = [x.clone() for x in p]
    state = [[Moment8.zeros_like(x, s) for x in p] for s in (True, False, True, False)]
    adamw_step(p, g, state[0], state[1], steps=2, lr=1e-2, keys=list(range(201)))
    rows = (_records.AdamWTensor * 201)(*[_records.AdamWTensor(
        param=a.data_ptr(), grad=b.data_ptr(), exp_avg=m.codes.data_ptr(), exp_avg_sq=v.codes.data_ptr(),
        exp_avg_exponents=m.exponents.data_ptr(), exp_avg_sq_exponents=v.exponents.data_ptr(), numel=a.numel(), step=2, lr=1e-2,
        weight_decay=1e-2, round_key=i) for i, (a, b, m, v) in enumerate(zip(q, g, state[2], state[3]))])
    args = _records.AdamWArgs(num_tensors=201, param_type=0, state_bits=8, beta1=0.9, beta2=0.999, eps=1e-8,
                              tensors=C.cast(rows, C.c_char_p))
    _lib.call("fdgs_adamw_step", args)
    for a, b in zip(p + [x for s in state[:2] for m in s for x in m[:2]], q + [x for s in state[2:] for m in s for x in m[:2]]):
        assert torch.equal(a, b)
    moments = state[0] + state[1]
    out = [torch.full(m.codes.shape, -1.0, device="cuda") for m in moments]
    rows = (_records.Moment8Tensor * 402)(*[_records.Moment8Tensor(
        codes=m.codes.data_ptr(), exponents=m.exponents.data_ptr(), value=o.data_ptr(), numel=o.numel(), is_signed=m.signed)
        for m, o in zip(moments, out)])
    args = _records.Moment8Args(num_tensors=402, value_type=0, tensors=C.cast(rows, C.c_char_p))
    _lib.call("fdgs_moment8_unpack", args)
    for a, b in zip(out, unpack8(moments)):
        assert torch.equal(a, b)
    assert len(pack8(out, [m.signed for m in moments])) == 402


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [512, 300])
def test_bfloat16_parameters_set_to_zero_or_infinity(n, bits):
    """A parameter that is masked or reset while its residual stays is the new weight: no pair of a zero or an infinity and a residual
    that cannot belong to it is read as a NaN, and every other pair as pattern plus residual.  Blocks of 256 and what is left."""
    from fdgs.adamw import Moment8, adamw_step
    word = torch.tensor([0x0000, 0x8000, 0x7F80, 0xFF80, 0x3F80], dtype=torch.int32)
    low = torch.tensor([-0x8000, -5, -1, 0, 1, 123, 0x7FFF], dtype=torch.int32)
    hi, lo = (x.reshape(-1).repeat(-(-n // 35))[:n] for x in torch.broadcast_tensors(word[:, None], low[None]))
    p, res = hi.to(torch.int16).cuda().view(torch.bfloat16), lo.to(torch.int16).cuda()
    m, v = (Moment8.zeros_like(p, s) if bits == 8 else torch.zeros(n, device="cuda") for s in (True, False))
    adamw_step([p], [torch.zeros_like(p)], [m], [v], steps=1, lr=1e-3, weight_decay=0.0, residuals=[res], keys=[1] if bits == 8 else None)
    size = hi & 0x7FFF
    gone = ((size == 0) & (lo < 0)) | ((size == 0x7F80) & (lo > 0))
    want = (hi << 16) + torch.where(gone, torch.zeros_like(lo), lo)
    got = (p.view(torch.int16).to(torch.int32) << 16) + res.to(torch.int32)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("eps", [1e-8, 1e-15])
@pytest.mark.parametrize("bits", [32, 8])
def test_update_is_the_formula_rounded_once_an_operation(bits, eps):
    """float32 parameters move by the bits that the formula gives in float32 with every operation rounded to the nearest, whatever
    form the moments have."""
    from fdgs import adamw
    f, b1, b2, lr, wd, t = np.float32, 0.9, 0.999, 3e-3, 0.1, 7
    (w, g, m0, v0), = _inputs([70001], 11)
    p, gd = torch.from_numpy(w).cuda(), torch.from_numpy(g).cuda()
    if bits == 8:
        cm, cv = ac.encode(m0, 0x8000, True), ac.encode(v0, 0x8000, False)
        m0, v0 = ac.decode(*cm, True), ac.decode(*cv, False)
        m, v = (adamw.Moment8(*(torch.from_numpy(x).cuda() for x in c), s) for c, s in ((cm, True), (cv, False)))
    else:
        m, v = torch.from_numpy(m0).cuda(), torch.from_numpy(v0).cuda()
    adamw.adamw_step([p], [gd], [m], [v], steps=t, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, keys=[5] if bits == 8 else None)
    m1, v1 = ac.adamw32(g, m0, v0, b1, b2)
    denom = np.sqrt(v1) * f(1.0 / math.sqrt(1.0 - b2 ** t)) + f(eps)
    want = w * f(1.0 - lr * wd) - (m1 * f(lr / (1.0 - b1 ** t))) / denom
    assert want.dtype == f and np.array_equal(p.cpu().numpy().view(np.int32), want.view(np.int32))


def test_views_that_are_still_to_be_negated():
    """A gradient or a value that lies in memory with the other sign is read as what it is; what is written must lie as it reads."""
    from fdgs.adamw import adamw_step, pack8, unpack8
    z = torch.randn(6, 1, dtype=torch.complex64, device="cuda")
    for neg in (z.conj().imag, torch._neg_view(z.imag.contiguous()), torch._neg_view(torch.randn(6, 9, device="cuda"))[:, :4]):
        assert neg.is_neg()
        moved = []
        for g in (neg, neg.resolve_neg().contiguous()):
            p, m, v = (torch.zeros(g.shape, device="cuda") for _ in range(3))
            adamw_step([p], [g], [m], [v], steps=1, lr=0.1)
            moved.append((p, m, v))
            moved[-1] += (unpack8(pack8([g], True))[0],)
        assert all(torch.equal(a, b) for a, b in zip(*moved)) and (moved[0][1] != 0).all()
    x, y = torch._neg_view(torch.ones(8, device="cuda")), [torch.ones(8, device="cuda") for _ in range(3)]
    for k, match in ((0, "contiguous"), (2, "contiguous"), (3, "contiguous")):
        args = [[t] for t in (y[0], y[0].clone(), y[1], y[2])]
        args[k] = [x]
        with pytest.raises(ValueError, match=match):
            adamw_step(*args, steps=1, lr=0.1)
    with pytest.raises(ValueError, match="contiguous"):
        unpack8(pack8([y[0]], True), out=[x])
    assert (x == -1).all() and all((t == 1).all() for t in y)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bf16", [False, True])
def test_tensors_of_another_shape_are_refused(bits, bf16):
    """As many elements in another order are not the parameter's; flat ones are."""
    from fdgs.adamw import Moment8, adamw_step, unpack8
    kind = torch.bfloat16 if bf16 else torch.float32

    def args(shapes):
        p, g, m, v, low = shapes
        make = (lambda s, signed: Moment8.zeros_like(torch.empty(s, device="cuda"), signed)) if bits == 8 else \
            (lambda s, signed: torch.zeros(s, device="cuda"))
        return dict(params=[torch.ones(p, dtype=kind, device="cuda")], grads=[torch.ones(g, dtype=kind, device="cuda")],
                    exp_avgs=[make(m, True)], exp_avg_sqs=[make(v, False)], steps=1, lr=0.1, keys=[3] if bits == 8 else None,
                    residuals=[torch.zeros(low, dtype=torch.int16, device="cuda")] if bf16 else None)
    right, other, flat = (30, 40), (40, 30), (1200,)
    for k in range(5 if bf16 else 4):
        for shape in (other, (30, 40, 1), (1, 30, 40)):
            bad = args([shape if j == k else right for j in range(5)])
            with pytest.raises(ValueError, match="shape"):
                adamw_step(**bad)
            assert (bad["params"][0] == 1).all()
    with pytest.raises(ValueError, match="shape"):
        adamw_step(**args([right, flat, right, right, right]))           # a flat gradient of a matrix neither
    ends = []
    for shapes in ([right] * 5, [right, right, flat, flat, flat], [flat, flat, right, right, right]):
        a = args(shapes)
        adamw_step(**a)
        ends.append(a["params"][0].reshape(-1))
    assert torch.equal(ends[0], ends[1]) and torch.equal(ends[0], ends[2]) and (ends[0] != 1).all()
    if bits == 8:
        m = Moment8.zeros_like(torch.empty(right, device="cuda"), True)
        with pytest.raises(ValueError, match="shape"):
            unpack8([m], out=[torch.ones(other, device="cuda")])
        assert (unpack8([m], out=[torch.ones(flat, device="cuda")])[0] == 0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bf16", [False, True])
def test_reads_that_overlap_writes_are_refused(bits, bf16):
    """A gradient inside what the step writes, whole or by one element, in one piece or in rows; not rows beside it."""
    from fdgs.adamw import Moment8, adamw_step
    kind = torch.bfloat16 if bf16 else torch.float32
    n = 1203

    def step(p, grads):
        make = (lambda x, s: Moment8.zeros_like(x, s)) if bits == 8 else (lambda x, s: torch.zeros(x.shape, device="cuda"))
        args = dict(params=p, grads=grads, exp_avgs=[make(x, True) for x in p], exp_avg_sqs=[make(x, False) for x in p], steps=1, lr=0.1,
                    residuals=[torch.zeros(x.shape, dtype=torch.int16, device="cuda") for x in p] if bf16 else None,
                    keys=list(range(len(p))) if bits == 8 else None)
        return args
    both = torch.ones(4 * n, dtype=kind, device="cuda")
    other = [torch.ones(77, dtype=kind, device="cuda"), torch.ones(77, dtype=kind, device="cuda")]
    p = both[n:2 * n]
    for g in (p, both[:n + 1][-n:], both[2 * n - 1:3 * n - 1], both[n + 5:2 * n + 5]):
        for order in (slice(None), slice(None, None, -1)):
            args = step([other[0], p][order], [other[1], g][order])
            with pytest.raises(ValueError, match="overlap"):
                adamw_step(**args)
    for k in ("exp_avgs", "exp_avg_sqs") + (("residuals",) if bf16 else ()):     # the gradient lies in another tensor of the step
        args = step([p], [both[:n]])
        t = args[k][0]
        pieces = t[:2] if isinstance(t, tuple) else (t,)
        for x in pieces:
            raw = torch.empty(0, dtype=kind, device="cuda").set_(x.untyped_storage(), 0, (1,), (1,))
            args["params"].append(torch.ones(1, dtype=kind, device="cuda"))
            args["grads"].append(raw)
            for name in ("exp_avgs", "exp_avg_sqs", "residuals", "keys"):
                if args[name] is not None:
                    more = step([args["params"][-1]], [raw])
                    args[name].append(more[name][0])
            with pytest.raises(ValueError, match="overlap"):
                adamw_step(**args)
            for name in ("params", "grads", "exp_avgs", "exp_avg_sqs", "residuals", "keys"):
                if args[name] is not None:
                    args[name].pop()
    # rows of a wider array: a written piece in their gaps is beside them, one that reaches into a row is not
    wide = torch.ones(100, 16, dtype=kind, device="cuda")
    sliced = torch.ones(100, 6, dtype=kind, device="cuda")
    for row in (0, 50, 99):
        for lo, hi, fine in ((6, 16, True), (5, 16, False), (0, 6, False), (2, 3, False), (7, 8, True)):
            piece = wide[row, lo:hi]
            args = step([sliced, piece], [wide[:, :6], torch.ones_like(piece)])
            if fine:
                adamw_step(**args)
                assert (piece != 1).all() and (wide[:, :6] == 1).all()
                piece.fill_(1)
            else:
                with pytest.raises(ValueError, match="overlap"):
                    adamw_step(**args)
    flat = wide.view(-1)
    for at, fine in ((6 + 50 * 16, True), (5 + 50 * 16, False), (7 + 50 * 16, False), (6 + 99 * 16, True)):      # over a row's end
        piece = flat[at:at + 10]
        args = step([sliced, piece], [wide[:, :6], torch.ones_like(piece)])
        if fine:
            adamw_step(**args)
            piece.fill_(1)
        else:
            with pytest.raises(ValueError, match="overlap"):
                adamw_step(**args)
    assert (wide == 1).all() and (both == 1).all()


def test_conversions_refuse_results_in_their_codes():
    from fdgs.adamw import Moment8, pack8, unpack8
    raw = torch.zeros(6000, dtype=torch.uint8, device="cuda")
    values = raw.view(torch.float32)
    ones, = pack8([torch.ones(300, device="cuda")], True)
    for codes_at, exps_at, out_at, fine in ((0, 3000, 75, True), (0, 3000, 74, False), (1203, 3000, 0, True), (1199, 3000, 0, False),
                                            (0, 1199, 0, False), (1200, 1500, 0, True), (3000, 602, 150, False), (3000, 598, 150, True)):
        m = Moment8(raw[codes_at:codes_at + 300], raw[exps_at:exps_at + 2], True)
        out = values[out_at:out_at + 300]
        raw.zero_()
        m.codes.copy_(ones.codes)
        m.exponents.copy_(ones.exponents)
        if fine:
            assert (unpack8([m, m], out=[out, torch.empty(300, device="cuda")])[0] == 1).all()       # one moment twice may be read
        else:
            with pytest.raises(ValueError, match="overlap"):
                unpack8([ones, m], out=[torch.empty(300, device="cuda"), out])


def test_a_read_out_is_seen_by_saved_graphs():
    """A graph that has saved the tensor raises in its backward pass once unpack8 has written it."""
    from fdgs.adamw import pack8, unpack8
    ms = pack8([torch.ones(8, device="cuda")], False)
    out, w = torch.full((8,), 3.0, device="cuda"), torch.ones(8, device="cuda", requires_grad=True)
    loss = (w * out).sum()
    unpack8(ms, out=[out])
    assert (out == 1).all()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                             # tensors without a version
        assert (unpack8(pack8([torch.ones(8, device="cuda")], False))[0] == 1).all()


def test_indexes_past_32_bits():
    """A tensor of 2^32 + 1004 elements with 8-bit moments and a gradient in rows: blocks at both ends and on either side of the numbers
    that 31 and 32 bits hold have the format's codes (whose random numbers depend on all of the index) and the formula's weights,
    everything else stays; then the moments' conversions.  66 GB."""
    from fdgs.adamw import Moment8, adamw_step, pack8, unpack8
    f, b1, b2, lr, eps, t, key = np.float32, 0.9, 0.999, 1e-2, 1e-8, 3, 12345
    rows = 1431656100
    n = 3 * rows
    assert n == (1 << 32) + 1004
    windows = [(at, min(at + 512, n)) for at in (0, (1 << 31) - 256, (1 << 32) - 256, (1 << 32) + 768)]     # the last one's block is not whole
    wide = torch.zeros(rows, 4, device="cuda")
    rng = np.random.default_rng(0)
    grads = []
    for lo, hi in windows:                                   # written through their rows: column 3 lies between
        x = rng.standard_normal(hi - lo).astype(f)
        i = torch.arange(lo, hi, device="cuda")
        wide.view(-1)[torch.div(i, 3, rounding_mode="floor") * 4 + i % 3] = torch.from_numpy(x).cuda()
        grads.append(x)
    p = torch.ones(rows, 3, device="cuda")
    m, v = Moment8.zeros_like(p, True), Moment8.zeros_like(p, False)
    adamw_step([p], [wide[:, :3]], [m], [v], steps=t, lr=lr, eps=eps, weight_decay=0.0, keys=[key])
    del wide
    count = 0
    for (lo, hi), x in zip(windows, grads):
        zero = np.zeros(hi - lo, f)
        m1, v1 = ac.adamw32(x, zero, zero, b1, b2)
        h = ac.hash32(np.arange(lo, hi), key)
        for got, want in ((m, ac.encode(m1, h >> 16, True)), (v, ac.encode(v1, h & 0xFFFF, False))):
            assert np.array_equal(got.codes.view(-1)[lo:hi].cpu().numpy(), want[0])
            assert np.array_equal(got.exponents[lo // 256:-(-hi // 256)].cpu().numpy(), want[1])
        count += int((ac.encode(v1, h & 0xFFFF, False)[0] != 0).sum())
        denom = np.sqrt(v1) * f(1.0 / math.sqrt(1.0 - b2 ** t)) + f(eps)
        want = np.ones_like(x) - (m1 * f(lr / (1.0 - b1 ** t))) / denom
        assert np.array_equal(p.view(-1)[lo:hi].cpu().numpy().view(np.int32), want.view(np.int32))
    chunks = lambda x: x.view(-1).split(1 << 28)             # noqa: E731
    assert sum(int(c.count_nonzero()) for c in chunks(v.codes)) == count
    assert sum(int((c != 1).sum()) for c in chunks(p)) <= count
    del p
    x, = unpack8([m])
    for lo, hi in windows:
        part = Moment8(m.codes.view(-1)[lo:hi], m.exponents[lo // 256:-(-hi // 256)], True)
        assert torch.equal(x.view(-1)[lo:hi], unpack8([part])[0])
    assert sum(int(c.count_nonzero()) for c in chunks(x)) == sum(int((c & 127).count_nonzero()) for c in chunks(m.codes))
    x.mul_(1.03)                                             # off the grid: the random numbers count
    again, = pack8([x], True, [key])
    for lo, hi in windows:
        codes, exps = ac.encode(x.view(-1)[lo:hi].cpu().numpy(), ac.hash32(np.arange(lo, hi), key) >> 16, True)
        assert np.array_equal(again.codes.view(-1)[lo:hi].cpu().numpy(), codes)
        assert np.array_equal(again.exponents[lo // 256:-(-hi // 256)].cpu().numpy(), exps)


@pytest.mark.parametrize("signed", [True, False])
def test_the_largest_code_of_a_block(signed):
    """It stands for the power of two above the block's largest value: infinity where float32 has no such power."""
    from fdgs.adamw import pack8, unpack8
    top = np.float32(2.0 - 2.0 ** -23)
    for e in (-126, 0, 126, 127):
        x = torch.full((300,), float(np.ldexp(top, e)), device="cuda")
        got, = unpack8(pack8([x], signed))
        assert (got == 2.0 ** (e + 1)).all() if e < 127 else got.isinf().all()
        x[:256] = float(np.ldexp(np.float32(1.875), e))          # on the grid
        got, = unpack8(pack8([x], signed, [7]))
        assert torch.equal(got[:256], x[:256])

"""The fused block norm on the GPU against the 64-bit oracle.

Tolerances: an output of type t is off by at most half a step of t (finfo(t).eps / 2 of the value) for its one rounding, plus what
fp32 arithmetic in front of it may lose.  That is K * 2^-24 of the sizes of the terms it is summed from, which the oracle gives:
K counts the additions a term passes through -- at most 16 in a lane, 10 across lanes and 8 across waves in each of up to four
sums that follow one another, a handful of products and the square root, under 256 -- and for sums over rows the rows of a
lane, 128 row groups and 32 partial sums more: under 512 at the sizes here."""
import itertools

import pytest
import torch

from oracle import checkpoint8 as orc

pytestmark = pytest.mark.gpu
K, K_ROWS = 256, 512


@pytest.fixture()
def F():
    from superresolution_amd import functional
    return functional


def _near(got, want, size, k, what):
    got = got.cpu()
    assert got.shape == want.shape, what
    u = torch.finfo(got.dtype).eps / 2
    tol = (1 + u) * k * 2.0 ** -24 * size + u * want.abs() + 1e-38
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (what, float((off / tol).max()))


def _inputs(shape, dtype, kind, gate, post, pre, bias, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    d = {"x": (2 * n(*shape)).to(dtype), "h": ((n(*shape) * torch.exp(0.5 * n(c)) + 0.5 * n(c)) * size).to(dtype),
         "dr": n(*shape).to(dtype), "dn": n(*shape).to(dtype), "post": None, "pre": None, "gate": None}
    if post:
        d["post"] = (1 + 0.3 * n(c), n(c) if bias else None)
    if pre:
        d["pre"] = (1 + 0.3 * n(c), n(c) if bias else None)
    else:
        d["dn"] = None
    if gate:
        d["gate"] = {"channel": lambda: n(c), "sample": lambda: n(shape[0], c), "map": lambda: n(*shape).to(dtype), "map32": lambda: n(*shape)}[gate]()
    return d


def _dev(v):
    return None if v is None else tuple(_dev(t) for t in v) if isinstance(v, tuple) else v.cuda()


def _check(F, d, kind, act, scale, saved8=False):
    learned = isinstance(scale, torch.Tensor)
    how = dict(post=_dev(d["post"]), gate=_dev(d["gate"]), scale=_dev(scale) if learned else scale, pre=_dev(d["pre"]), kind=kind, gate_act=act)
    if d["x"] is not None:
        r, n = F.norm_residual(_dev(d["x"]), _dev(d["h"]), **how)
        want, size = orc.norm_residual(d["x"], d["h"], d["post"], d["gate"], scale, d["pre"], kind, act)
        for got, w, s, what in zip((r, n), want, size, "rn"):
            assert (got is None) == (w is None)
            if w is not None:
                _near(got, w, s, K, what)
        d = {**d, "r": r.cpu()}
    h, rr = _dev(d["h"]), _dev(d["r"])
    if saved8:
        h, rr = F.checkpoint8_pack(h), F.checkpoint8_pack(rr)
        d["h"], d["r"] = F.checkpoint8_restore(h).cpu(), F.checkpoint8_restore(rr).cpu()
    got = F.norm_residual_bwd(h, rr, _dev(d["dr"]), _dev(d["dn"]), **how)._asdict()
    want, size = orc.norm_residual_bwd(d["h"], d["r"], d["dr"], d["dn"], d["post"], d["gate"], scale, d["pre"], kind, act, learned)
    assert {k for k, v in got.items() if v is not None} == set(want)
    for name, w in want.items():
        _near(got[name], w, size[name], K if name in ("dx", "dh") else K_ROWS, name)
    return got


WIDTHS = [1, 2, 3, 8, 10, 16, 17, 32, 33, 48, 64, 99, 128, 200, 256, 257, 512, 513, 1000, 1024, 1025, 2047, 2048, 2056, 4095, 4096, 4104, 8191, 8192]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("c", WIDTHS)
def test_every_width(F, c, dtype):
    for i, (kind, rows) in enumerate([("layer", (2, 3)), ("rms", (1, 1)), ("layer", (3, 50)), ("rms", (5, 7))]):
        d = _inputs(rows + (c,), dtype, kind, ["sample", "channel", "map", None][i], True, True, i % 2 == 0, c + i)
        _check(F, d, kind, ["sigmoid", "none"][i % 2], 0.2 if i % 2 else torch.tensor(0.7))


CASES = list(itertools.product(["layer", "rms"], [None, "channel", "sample", "map", "map32"], ["none", "sigmoid"], [True, False], [True, False]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind,gate,act,post,pre", CASES)
def test_every_combination(F, kind, gate, act, post, pre, dtype):
    for i, c in enumerate((64, 45)):
        d = _inputs((3, 5, 9, c), dtype, kind, gate, post, pre, i == 0, 7 * c)
        _check(F, d, kind, act, torch.tensor(0.3) if i == 0 else -1.5, saved8=i == 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("c", [6, 48, 64, 160, 1000, 4100])
def test_saved_maps_as_checkpoints(F, c, dtype):
    d = _inputs((4, 33, c), dtype, "layer", "sample", True, True, True, c)
    _check(F, d, "layer", "sigmoid", torch.tensor(0.4), saved8=True)
    # one of the two alone: equal to the restored map's gradients, bit for bit
    h, r = F.checkpoint8_pack(d["h"].cuda()), F.checkpoint8_pack(d["x"].cuda())
    how = dict(post=_dev(d["post"]), pre=_dev(d["pre"]))
    rest = [F.checkpoint8_restore(t) for t in (h, r)]
    want = F.norm_residual_bwd(*rest, d["dr"].cuda(), d["dn"].cuda(), **how)
    for a, b in ((h, r), (h, rest[1]), (rest[0], r)):
        for x, y in zip(F.norm_residual_bwd(a, b, d["dr"].cuda(), d["dn"].cuda(), **how), want):
            assert (x is None and y is None) or torch.equal(x, y)


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 1000, 70001])
def test_numbers_of_rows(F, rows):
    d = _inputs((1, rows, 24), torch.float32, "layer", "channel", True, True, True, rows)
    _check(F, d, "layer", "none", torch.tensor(0.5))


@pytest.mark.parametrize("samples,rows", [(1, 5000), (2, 2500), (300, 2), (2000, 3), (5, 1), (7, 333)])
def test_gates_by_sample(F, samples, rows):
    for dtype in (torch.bfloat16, torch.float32):
        d = _inputs((samples, rows, 40), dtype, "rms", "sample", True, True, False, rows)
        _check(F, d, "rms", "sigmoid", 0.2)


def test_only_the_norm_in_front(F):
    for dtype, c in ((torch.bfloat16, 64), (torch.float32, 37)):
        d = _inputs((4, 21, c), dtype, "layer", None, False, True, True, c)
        d["h"] = None
        x = d["x"].cuda()
        r, _ = F.norm_residual(x, pre=_dev(d["pre"]))
        assert r is x
        _check(F, d, "layer", "none", 1.0)
        d["dr"] = None        # no gradient of the sum itself
        d["x"], d["r"] = None, d["x"]
        _check(F, d, "layer", "none", 1.0)


def test_rows_that_are_constant_zero_or_not_finite(F):
    """A constant row normalises to its bias; a row with NaN or infinity spoils itself and no other."""
    c = 64
    g = torch.Generator().manual_seed(3)
    x, h = torch.randn(12, c, generator=g), torch.randn(12, c, generator=g)
    h[0], h[1], x[2], h[2] = 0.0, 3.0, 0.0, 0.0
    w, b = torch.randn(c, generator=g), torch.randn(c, generator=g)
    clean = F.norm_residual(x.cuda(), h.cuda(), post=_dev((w, b)), pre=_dev((w, b)))
    (r, n), (rs, ns) = orc.norm_residual(x, h, (w, b), None, 1.0, (w, b), "layer", "none")
    _near(clean[0], r, rs, K, "r")
    _near(clean[1], n, ns, K, "n")
    assert torch.equal(clean[0][0].cpu(), x[0] + b)
    bad = h.clone()
    bad[4, 7], bad[5, 0], x2 = float("nan"), float("inf"), x.clone()
    x2[6, 63] = -float("inf")
    got = F.norm_residual(x2.cuda(), bad.cuda(), post=_dev((w, b)), pre=_dev((w, b)))
    fine = [i for i in range(12) if i not in (4, 5, 6)]
    for a, e in zip(got, clean):
        assert torch.equal(a[fine], e[fine])
    assert bool(torch.isnan(got[1][4:7]).all()) and bool(torch.isnan(got[0][4:6]).all())
    dr = torch.randn(12, c, generator=g).cuda()
    clean = F.norm_residual_bwd(h.cuda(), x.cuda(), dr, dr, post=_dev((w, b)), pre=_dev((w, b)))
    got = F.norm_residual_bwd(bad.cuda(), x2.cuda(), dr, dr, post=_dev((w, b)), pre=_dev((w, b)))
    for a, e in zip(got[:2], clean[:2]):
        assert torch.equal(a[fine], e[fine])


@pytest.mark.parametrize("c", [64, 37, 5, 131])
def test_an_infinity_leaves_the_rest_of_an_rms_row_at_zero(F, c):
    """x / inf = 0 and inf / inf = NaN, at every place of the row and of its last vector."""
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.ones(c, c, dtype=dtype)
        x.fill_diagonal_(float("inf"))
        w = torch.ones(c).cuda()
        _, n = F.norm_residual(x.cuda(), pre=(w, None), kind="rms")
        eye = torch.eye(c, dtype=torch.bool)
        assert bool(torch.isnan(n.cpu()[eye]).all()) and bool((n.cpu()[~eye] == 0).all())


def test_without_a_branch_the_sum_is_the_map_that_was_given(F):
    x = torch.randn(64, 33, device="cuda").t()                          # not contiguous: the norm reads a copy
    w = torch.rand(64, device="cuda")
    r, n = F.norm_residual(x, pre=(w, None))
    assert r is x and torch.equal(n, F.norm_residual(x.contiguous(), pre=(w, None))[1])


def test_a_large_mean_costs_no_digits(F):
    """Rows of 1000 +- 1: the spread is what counts."""
    d = _inputs((2, 9, 256), torch.float32, "layer", None, True, True, True, 5)
    d["h"] = d["h"] + 1000.0
    r, _ = F.norm_residual(torch.zeros(2, 9, 256).cuda(), d["h"].cuda(), post=_dev(d["post"]))
    (want, _), _ = orc.norm_residual(torch.zeros(2, 9, 256), d["h"], d["post"], None, 1.0, None, "layer", "none")
    # the inputs' own differences from the mean are exact to 2^-24 * 1000; rstd about 1, |w| and |b| under 5
    assert float((r.cpu().double() - want).abs().max()) < 32 * 1000 * 2.0 ** -24 * 5


def test_maps_at_odd_addresses_strided_ones_and_bytes_around_the_outputs(F):
    from superresolution_amd._lib import NormResidualArgs, check, lib
    g = torch.Generator().manual_seed(9)
    for dtype, dt, c in ((torch.bfloat16, 0, 37), (torch.float32, 1, 37), (torch.bfloat16, 0, 64)):
        rows = 13
        flat = [torch.randn(rows * c + 3, generator=g).to(dtype).cuda() for _ in range(2)]
        x, h = (t[3:].view(rows, c) for t in flat)
        w = torch.randn(c, generator=g).cuda()
        want = F.norm_residual(x.clone(), h.clone(), post=(w, None), pre=(w, None), kind="rms")
        for got in (F.norm_residual(x, h, post=(w, None), pre=(w, None), kind="rms"),
                    F.norm_residual(x.t().contiguous().t(), h, post=(w, None), pre=(w, None), kind="rms")):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        outs = [torch.full((rows * c + 35,), 5.0, dtype=dtype, device="cuda") for _ in range(2)]
        a = NormResidualArgs(x=x.data_ptr(), h=h.data_ptr(), post_weight=w.data_ptr(), pre_weight=w.data_ptr(), r=outs[0][3:].data_ptr(), n=outs[1][3:].data_ptr(),
                             rows=rows, c=c, dtype=dt, kind=1, post=1, pre=1, scale=1.0, eps=1e-6)
        check(lib.srhip_norm_residual_fwd(a, torch.cuda.current_stream().cuda_stream))
        for o, e in zip(outs, want):
            assert torch.equal(o[3:-32].view(rows, c), e) and bool((o[:3] == 5).all()) and bool((o[-32:] == 5).all())


def test_empty_maps_and_refusals(F):
    w = torch.ones(8, device="cuda")
    e = torch.empty(0, 4, 8, device="cuda")
    r, n = F.norm_residual(e, e, post=(w, w), pre=(w, None))
    assert r.shape == n.shape == e.shape
    g = F.norm_residual_bwd(e, e, e, e, post=(w, w), pre=(w, None), gate=torch.ones(8, device="cuda"), scale=torch.ones((), device="cuda"))
    assert g.dx.shape == e.shape and all(float(t.abs().sum()) == 0 for t in (g.dpost_weight, g.dpost_bias, g.dgate, g.dscale, g.dpre_weight))
    x = torch.zeros(2, 3, 8, device="cuda")
    for bad in (dict(pre=w), dict(pre=(w[:4], None)), dict(pre=(None, w)), dict(gate=torch.ones(3, 8, device="cuda")), dict(gate=torch.ones(2, 3, 8).cuda().bfloat16()),
                dict(kind="batch"), dict(gate_act="tanh"), dict(scale=torch.ones(2, device="cuda")), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            F.norm_residual(x, x, **{"pre": (w, None), **bad})
    with pytest.raises(TypeError):
        F.norm_residual(x, x.bfloat16())
    with pytest.raises(TypeError):
        F.norm_residual(x, x, gate=w.bfloat16())
    with pytest.raises(ValueError):
        F.norm_residual(x, x[:1])
    with pytest.raises(ValueError):
        F.norm_residual(x)
    with pytest.raises(ValueError):
        F.norm_residual(x, gate=w, pre=(w, None))
    with pytest.raises(ValueError):
        F.norm_residual(torch.zeros(1, 8193, device="cuda"), torch.zeros(1, 8193, device="cuda"))
    with pytest.raises(ValueError):
        F.norm_residual_bwd(x, x, x, None, pre=(w, None))
    with pytest.raises(ValueError):
        F.norm_residual_bwd(None, x, x, x, pre=(w, None), gate=w)
    with pytest.raises(ValueError):
        F.norm_residual_bwd(x[:1], x, x, x, pre=(w, None))
    ck = F.checkpoint8_pack(x.bfloat16())
    with pytest.raises(ValueError):
        F.norm_residual_bwd(ck, x, x, x, pre=(w, None))   # a bf16 map's checkpoint beside fp32 gradients


def test_results_repeat_and_streams_do_not_disturb_each_other(F):
    d = _inputs((2, 3000, 64), torch.bfloat16, "layer", "sample", True, True, True, 11)
    how = dict(post=_dev(d["post"]), gate=_dev(d["gate"]), scale=torch.tensor(0.3).cuda(), pre=_dev(d["pre"]), gate_act="sigmoid")
    h, r, dr, dn = (d[k].cuda() for k in ("h", "x", "dr", "dn"))
    want = F.norm_residual_bwd(h, r, dr, dn, **how)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] = F.norm_residual_bwd(h, r, dr, dn, **how)
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_first_call_of_a_width_inside_a_capture(F):
    """What a kernel asks of the runtime on its first call is answered while a stream is being captured, too."""
    x, h = (torch.randn(9, 5, 372, generator=torch.Generator().manual_seed(s)).cuda() for s in (1, 2))
    w = torch.rand(372, generator=torch.Generator().manual_seed(3)).cuda()
    how = dict(post=(w, None), pre=(w, w), kind="rms")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, n = F.norm_residual(x, h, **how)
        g = F.norm_residual_bwd(h, r, x, h, **how)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = F.norm_residual(x, h, **how)
        wg = F.norm_residual_bwd(h, want[0], x, h, **how)
        assert torch.equal(r, want[0]) and torch.equal(n, want[1])
        assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(g, wg))


def test_offsets_beyond_32_bits(F):
    """2^31 elements and more: the last rows of a map equal the same rows on their own, forward, backward, packed, restored."""
    rows, c, tail = (1 << 25) + 12345, 64, 4097
    x = torch.empty((rows, c), dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(5))
    assert x.numel() > 1 << 31
    w, b = torch.rand(c, device="cuda") + 0.5, torch.rand(c, device="cuda")
    how = dict(post=(w, b), gate=b, gate_act="sigmoid", scale=0.3, pre=(w, None))
    t = x[-tail:]
    r, n = F.norm_residual(x, x, **how)
    rt, nt = F.norm_residual(t, t, **how)
    assert torch.equal(r[-tail:], rt) and torch.equal(n[-tail:], nt)
    del n
    ck = F.checkpoint8_pack(x)
    ct = F.checkpoint8_pack(t)
    assert torch.equal(ck.codes[-tail:].view(torch.uint8), ct.codes.view(torch.uint8)) and torch.equal(ck.scales[-tail:], ct.scales)
    y = F.checkpoint8_restore(ck)
    assert torch.equal(y[-tail:], F.checkpoint8_restore(ct))
    del y
    m = F.relu_mask(x, ck)
    assert torch.equal(m[-tail:], F.relu_mask(t, ct))
    del m
    g = F.norm_residual_bwd(ck, r, x, x, **how)
    gt = F.norm_residual_bwd(ct, rt, t, t, **how)
    assert torch.equal(g.dx[-tail:], gt.dx) and torch.equal(g.dh[-tail:], gt.dh)
    del g, r
    # a pointwise gradient that only the last pixels contribute to
    dz = torch.zeros((rows, 16), dtype=torch.bfloat16, device="cuda")
    dz[-tail:] = t[:, :16]
    dw, _ = F.conv_wgrad((ck,), dz, c, 16, 1)
    want = dz[-tail:].double().t() @ F.checkpoint8_restore(ct).double()
    size = dz[-tail:].double().abs().t() @ F.checkpoint8_restore(ct).double().abs()
    assert bool(((dw[:, :, 0, 0].double() - want).abs() <= tail * 2.0 ** -24 * size).all())


def test_captured_and_replayed(F):
    def work(x, h, dr, dn, gate, scale, w, b):
        how = dict(post=(w, b), gate=gate, scale=scale, pre=(w, b), gate_act="sigmoid")
        r, n = F.norm_residual(x, h, **how)
        return (r, n) + tuple(F.norm_residual_bwd(h, r, dr, dn, **how)) + tuple(F.norm_residual_bwd(F.checkpoint8_pack(h), F.checkpoint8_pack(r), dr, dn, **how))

    def data(seed):
        d = _inputs((2, 700, 48), torch.bfloat16, "layer", "sample", True, True, True, seed)
        return [t.cuda() for t in (d["x"], d["h"], d["dr"], d["dn"], d["gate"], torch.tensor(0.1 * seed), *d["post"])]

    sets = [data(1), data(2)]
    static, graphs, outs = [[t.clone() for t in sets[0]] for _ in range(2)], [], []
    work(*static[0])
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(*static[i]))
        graphs.append(graph)
    for turn in range(3):
        for i in range(2):
            for s, v in zip(static[i], sets[(i + turn) % 2]):
                s.copy_(v)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = work(*sets[(i + turn) % 2])
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want):
                assert (a is None and b is None) or torch.equal(a, b)


def _same_with_infinities(got, want, size, k, what):
    """Infinities and NaN where the definition has them, the rest near to it."""
    got, w = got.cpu().double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(w)), what
    inf = torch.isinf(w)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], w[inf]), what
    fine = torch.isfinite(w)
    u = torch.finfo(torch.bfloat16 if what[1] == torch.bfloat16 else torch.float32).eps / 2
    tol = (1 + u) * k * 2.0 ** -24 * size[fine] + u * w[fine].abs() + 1e-38
    assert bool(((got[fine] - w[fine]).abs() <= tol).all()), what


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate", ["channel", "sample", "map", "map32"])
@pytest.mark.parametrize("kind,post,bias", [("rms", True, False), ("rms", True, True), ("layer", True, True), ("rms", False, False)])
def test_an_infinite_gate_is_an_infinite_term(F, kind, post, bias, gate, dtype):
    """Infinities and NaN among the gates reach their own channels, with the branch's sign: no infinity meets a bias on its own.
    Gradients: the gates' are finite (no gate is in them), the branch's are infinite where the gate is."""
    d = _inputs((3, 7, 40), dtype, kind, gate, post, False, bias, 21)
    for i, v in ((5, float("inf")), (6, -float("inf")), (7, float("nan"))):
        d["gate"][..., i] = v
    r, _ = F.norm_residual(_dev(d["x"]), _dev(d["h"]), post=_dev(d["post"]), gate=_dev(d["gate"]), scale=0.5, kind=kind)
    (want, _), (size, _) = orc.norm_residual(d["x"], d["h"], d["post"], d["gate"], 0.5, None, kind, "none")
    assert bool(torch.isinf(want[..., 5:7]).all())
    _same_with_infinities(r, want, size, K, ("r", dtype))
    g = F.norm_residual_bwd(_dev(d["h"]), None, _dev(d["dr"]), None, post=_dev(d["post"]), gate=_dev(d["gate"]), scale=0.5, kind=kind)
    want, size = orc.norm_residual_bwd(d["h"], None, d["dr"], None, d["post"], d["gate"], 0.5, None, kind, "none", False)
    assert bool(torch.isfinite(want["dgate"]).all())
    dt = dtype if gate == "map" else torch.float32
    _same_with_infinities(g.dgate, want["dgate"], size["dgate"], K_ROWS, ("dgate", dt))
    if not post:
        _same_with_infinities(g.dh, want["dh"], size["dh"], K, ("dh", dtype))


@pytest.mark.parametrize("gate", [None, "channel", "sample", "map"])
@pytest.mark.parametrize("bias", [False, True])
def test_an_infinite_scale_and_infinite_gradients(F, bias, gate):
    """The residual scale at infinity: every term is infinite, with its sign; the gate's gradient too.  An infinite gradient of the sum
    reaches the gate's gradient as an infinity where the norm has no bias."""
    d = _inputs((2, 9, 24), torch.float32, "rms", gate, True, False, bias, 22)
    for scale in (float("inf"), torch.tensor(float("inf"))):
        how = dict(post=_dev(d["post"]), gate=_dev(d["gate"]), scale=_dev(scale) if isinstance(scale, torch.Tensor) else scale, kind="rms")
        r, _ = F.norm_residual(_dev(d["x"]), _dev(d["h"]), **how)
        (want, _), _ = orc.norm_residual(d["x"], d["h"], d["post"], d["gate"], scale, None, "rms", "none")
        assert bool(torch.isinf(want).all()) and torch.equal(r.cpu().double(), want)
        if gate == "map" or (gate and not bias):
            g = F.norm_residual_bwd(_dev(d["h"]), None, _dev(d["dr"]), None, **how)
            want = _p_of(d, "rms") * d["dr"].double()
            want = torch.inf * (want if gate == "map" else want.sum((0, 1)) if gate == "channel" else want.sum(1))
            assert torch.equal(g.dgate.cpu().double(), want)
    if gate in ("channel", "sample") and not bias:
        d["dr"][1, 4, 3] = float("inf")
        g = F.norm_residual_bwd(_dev(d["h"]), None, _dev(d["dr"]), None, post=_dev(d["post"]), gate=_dev(d["gate"]), kind="rms")
        got = (g.dgate if gate == "channel" else g.dgate[1]).cpu()
        assert float(got[3]) == torch.inf * float(_p_of(d, "rms")[1, 4, 3]) and int(torch.isfinite(got).sum()) == 23


def _p_of(d, kind):
    """The branch behind its norm, in 64 bits."""
    w, b = d["post"]
    return orc._norm(d["h"].double(), (w.double(), None if b is None else b.double()), kind, 1e-6)[2]


@pytest.mark.parametrize("c,gates", [(8192, 16397), (4096, 2 * 32763 + 5)])
def test_gates_beyond_one_row_of_the_launch(F, c, gates):
    """Gates times channel blocks beyond 2^22 (2^32 threads): the second and third row of the launch; the first and last gates' gradients equal
    those of the same gates on their own (an item to a gate in both, added in the same order)."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = torch.Generator(device="cuda").manual_seed(9)
    h, dr = (torch.empty((gates, 2, c), dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2))
    gate, w = torch.empty((gates, c), device="cuda").normal_(generator=g), torch.rand(c, device="cuda", generator=g)
    got = F.norm_residual_bwd(h, None, dr, None, post=(w, None), gate=gate, gate_act="sigmoid", kind="rms").dgate
    per = (1 << 22) // (c // 32)
    for lo in (0, per - 300, gates - 600):
        part = slice(lo, lo + 600)
        want = F.norm_residual_bwd(h[part], None, dr[part], None, post=(w, None), gate=gate[part], gate_act="sigmoid", kind="rms").dgate
        assert torch.equal(got[part], want), lo
    off = torch.zeros(gates, device="cuda")
    for lo in range(0, gates, 4096):          # every gate against its sum, in 32 bits
        part = slice(lo, lo + 4096)
        hat = h[part].float()
        p = dr[part].float() * (hat / (hat.square().mean(-1, keepdim=True) + 1e-6).sqrt()) * w
        a = torch.sigmoid(gate[part])
        # the sums' arithmetic, and 1 - a, whose error is that of a: two roundings of at most one unit in the last place
        size = p.abs().sum(1) * (K * a * (1 - a) + 4 * a)
        off[part] = ((got[part] - p.sum(1) * a * (1 - a)).abs() / (size * 2.0 ** -24 + 1e-30)).amax(-1)
    assert float(off.max()) < 2               # once on each side


def test_more_rows_than_a_launch_has_work_groups(F):
    """2^32 rows of one channel and more, forward and backward: the last rows equal those on their own."""
    rows, tail = (1 << 32) + 4099, 5003
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    t = torch.randn(tail, 1, generator=torch.Generator().manual_seed(31)).bfloat16().cuda()
    x = torch.full((rows, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    x[-tail:] = t
    w = torch.full((1,), 1.5, device="cuda")
    how = dict(gate=w, scale=0.5, pre=(w, w), kind="rms")
    r, n = F.norm_residual(x, x, **how)
    rt, nt = F.norm_residual(t, t, **how)
    first = F.norm_residual(x[:8], x[:8], **how)
    assert torch.equal(r[-tail:], rt) and torch.equal(n[-tail:], nt)
    for lo in range(0, rows - tail, 1 << 28):
        part = slice(lo, min(lo + (1 << 28), rows - tail))
        assert bool((r[part] == first[0][0]).all()) and bool((n[part] == first[1][0]).all()), lo
    del n
    g = F.norm_residual_bwd(x, r, x, x, **how)
    gt = F.norm_residual_bwd(t, rt, t, t, **how)
    assert torch.equal(g.dx[-tail:], gt.dx) and torch.equal(g.dh[-tail:], gt.dh)
    del g, r, x
    torch.cuda.empty_cache()


def test_no_round_of_a_few_items(F):
    """How the backward pass cuts rows into items, read from the workspace that it asks for (work-groups x 2c sums, items x (2c + 1)): the
    rounds of items take about the time that the rows would take on all work-groups, for any number of crops and for more gates than
    work-groups.  (An item more than a round holds would double it.)"""
    from superresolution_amd._lib import NormResidualBwdArgs, lib
    c = 64

    def floats(gates, per, **kw):
        a = NormResidualBwdArgs(rows=gates * per, rows_per_gate=per, c=c, gate_mode=1, **kw)
        return lib.srhip_norm_residual_bwd_workspace_bytes(a) // 4

    for kw in (dict(dtype=0), dict(dtype=1), dict(dtype=0, h_scales=1, r_scales=1)):
        most = floats(1, 1 << 24, **kw) // (4 * c + 1)       # work-groups at once: an item each
        assert most >= 256
        for per, many, bound in ((1 << 20, range(1, 33), 1.08), (2048, (most // 2 + 88, most + 1, most * 3 // 2, most * 2 + 1), 1.3)):
            for gates in many:
                got = floats(gates, per, **kw)
                items = got // (4 * c + 1) if got <= most * (4 * c + 1) else (got - most * 2 * c) // (2 * c + 1)
                rounds = -(-items // most)
                assert rounds * most <= bound * items, (kw, gates, items, most)


@pytest.mark.parametrize("c", [10, 16, 24, 31, 32, 45, 64, 99, 128, 200, 255, 256, 401, 512])
def test_two_waves_to_a_simd_at_least(F, c):
    """Rows of up to 512 channels, of either type, from maps and checkpoints, with a gate map (the most registers) and without: two work-groups
    of four waves fit a CU, read from the workspace that the call asks for."""
    from superresolution_amd._lib import NormResidualBwdArgs, lib
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for dtype in (0, 1):
        for ck in (None, 1):
            for gate in (0, 2):
                a = NormResidualBwdArgs(rows=1 << 24, rows_per_gate=1 << 24, c=c, dtype=dtype, gate_mode=gate, h_scales=ck, r_scales=ck)
                groups = lib.srhip_norm_residual_bwd_workspace_bytes(a) // 4 // (4 * c + 1)
                assert groups >= 2 * cus * 0.95, (dtype, ck, gate, groups)


FIRST_CALLS = """
import torch
from superresolution_amd import functional as F
c = {c}
x, h = (torch.randn(9, 5, c, generator=torch.Generator().manual_seed(s)).to({dtype}).cuda() for s in (1, 2))
w = torch.rand(c, generator=torch.Generator().manual_seed(3)).cuda()
how = dict(post=(w, None), pre=(w, w), kind="rms")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    r, n = F.norm_residual(x, h, **how)
    g = F.norm_residual_bwd(h, r, x, h, **how)
for _ in range(3):
    for t in (r, n, g.dx, g.dh, g.dpost_weight):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    want = F.norm_residual(x, h, **how)
    wg = F.norm_residual_bwd(h, want[0], x, h, **how)
    assert torch.equal(r, want[0]) and torch.equal(n, want[1])
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(g, wg))
print("replayed")
"""


@pytest.mark.parametrize("c,dtype", [(1000, "torch.float32"), (2056, "torch.bfloat16")])
def test_first_call_of_a_process_inside_a_capture(c, dtype):
    """A process whose first calls are recorded: what the long rows' kernels, forward and backward, ask of the runtime once is asked while the
    stream is being captured (in this process other tests have asked before)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(c=c, dtype=dtype)], cwd=root, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and "replayed" in run.stdout, (run.returncode, run.stdout, run.stderr[-2000:])

"""8-bit activation checkpoints on the GPU: codes and scales against the 64-bit oracle (equal, not near), what reads them back, the
weight gradient formed from them."""
import pytest
import torch

from oracle import checkpoint8 as orc

pytestmark = pytest.mark.gpu


@pytest.fixture()
def F():
    from superresolution_amd import functional
    return functional


def _values(shape, dtype, seed):
    """Values of many magnitudes, channels of different size, with zeros of both signs, the type's extremes and non-finite ones."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[-1], generator=g)) * torch.exp(6 * torch.randn(shape[:-1] + (1,), generator=g))
    x = torch.where(torch.rand(shape, generator=g) < 0.3, 0.0, x)
    special = torch.tensor([float("inf"), -float("inf"), float("nan"), -0.0, torch.finfo(dtype).max, -torch.finfo(dtype).max, torch.finfo(dtype).tiny,
                            1e-40, -3e-41, 2.0 ** -127, 448.0, 449.0, 464.0, 1.75, 1.7578125])
    at = torch.rand(shape, generator=g)
    pick = special[torch.randint(len(special), shape, generator=g)]
    return torch.where(at < 0.02, pick, x).to(dtype)


def _check_pack(F, x):
    ck = F.checkpoint8_pack(x.cuda())
    codes, scales = orc.encode(x)
    got = ck.codes.view(torch.uint8).cpu()
    nan = (codes & 127) == 127
    assert torch.equal(ck.scales.cpu(), scales)
    assert torch.equal((got & 127) == 127, nan) and torch.equal(got[~nan], codes[~nan])
    y = F.checkpoint8_restore(ck).cpu()
    want = orc.decode(codes, scales)
    assert y.dtype == x.dtype and y.shape == x.shape
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y.double().nan_to_num(), want.nan_to_num())
    return ck


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 8), (2, 9, 10), (4, 31), (7, 32), (6, 33), (2, 3, 5, 48), (3, 64), (1, 17, 70), (2, 4, 96),
                                   (11, 127), (3, 160), (2, 257), (1, 1031), (300, 64)])
def test_codes_scales_and_values_equal_the_oracle(F, shape, dtype):
    _check_pack(F, _values(shape, dtype, sum(shape)))


def test_every_bf16_number_alone_in_its_group(F):
    """All 65536 bit patterns, each the only channel of its row: scale, code and value of every number there is."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)[:, None]
    _check_pack(F, x)


def test_every_bf16_number_beside_a_large_one(F):
    """... and beside a 1.5 * 2^k that sets the scale: rounding, ties, subnormal codes, what must not become 0."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    for k in (-60, 0, 40):
        _check_pack(F, torch.stack([x, torch.full_like(x, 1.5 * 2.0 ** k)], -1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_code_with_every_scale(F, dtype):
    """What a checkpoint can hold, all of it: 256 codes times the scale bytes 10 .. 246, exact."""
    s = torch.arange(10, 247, dtype=torch.uint8)
    codes = torch.arange(256, dtype=torch.uint8).view(1, 8, 32).expand(237, 8, 32).reshape(237, 256).contiguous()
    scales = s[:, None].expand(237, 8).contiguous()
    y = F.checkpoint8_restore(F.Checkpoint8(codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), dtype)).cpu()
    want = orc.decode(codes, scales)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y.double().nan_to_num(), want.nan_to_num())


def test_error_of_a_checkpoint(F):
    """Half a step of 3 mantissa bits (2^-4 of the value), or less than the smallest code where that is larger."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(50, 64, generator=g).cuda()
    ck = F.checkpoint8_pack(x)
    y = F.checkpoint8_restore(ck)
    step = torch.exp2(ck.scales.float() - 127 - 9).repeat_interleave(32, -1)
    assert bool(((y - x).abs() <= torch.maximum(x.abs() / 16, step)).all())


@pytest.mark.parametrize("off", [1, 3, 7])
def test_maps_at_odd_addresses_and_strided_ones(F, off):
    for dtype in (torch.bfloat16, torch.float32):
        flat = _values((9 * 37 + off,), dtype, off)
        x = flat.cuda()[off:].view(9, 37)
        assert x.data_ptr() % 16 != 0
        ck = F.checkpoint8_pack(x)
        codes, scales = orc.encode(flat[off:].view(9, 37))
        nan = (codes & 127) == 127
        assert torch.equal(ck.scales.cpu(), scales) and torch.equal(ck.codes.view(torch.uint8).cpu()[~nan], codes[~nan])
        wide = torch.zeros(37, 2 * 9, dtype=dtype)
        wide[:, ::2] = flat[off:].view(9, 37).t()
        again = F.checkpoint8_pack(wide.cuda()[:, ::2].t())      # neither contiguous nor in order
        assert torch.equal(again.scales, ck.scales) and torch.equal(again.codes.view(torch.uint8), ck.codes.view(torch.uint8))


def test_nothing_is_written_behind_a_map(F):
    """C entry points on the middle of larger buffers: the bytes around the outputs stay as they were."""
    from superresolution_amd._lib import check, lib
    for c, dt, dtype in ((10, 0, torch.bfloat16), (33, 1, torch.float32), (64, 0, torch.bfloat16)):
        rows, groups = 77, (c + 31) // 32
        x = _values((rows, c), dtype, c).cuda()
        codes = torch.full((rows * c + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        scales = torch.full((rows * groups + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        y = torch.full((rows * c + 64,), 3.0, dtype=dtype, device="cuda")
        s = torch.cuda.current_stream().cuda_stream
        check(lib.srhip_checkpoint8_pack(x.data_ptr(), dt, codes.data_ptr() + 32, scales.data_ptr() + 32, rows, c, s))
        check(lib.srhip_checkpoint8_restore(codes.data_ptr() + 32, scales.data_ptr() + 32, y[32:].data_ptr(), dt, rows, c, s))
        for t, v in ((codes, 0xA5), (scales, 0xA5), (y, 3.0)):
            assert bool((t[:32] == v).all()) and bool((t[-32:] == v).all())
        want = F.checkpoint8_restore(F.checkpoint8_pack(x))
        assert torch.equal(y[32:-32].view(rows, c).nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 31), (1, 4, 32), (2, 2, 77), (1, 5, 200)])
def test_sign_bits_of_the_same_pass(F, shape):
    x = _values(shape + (64,), torch.bfloat16, sum(shape))
    ck = F.checkpoint8_pack(x.cuda(), signbits=True)
    plain = F.checkpoint8_pack(x.cuda())
    assert torch.equal(ck.codes.view(torch.uint8), plain.codes.view(torch.uint8)) and torch.equal(ck.scales, plain.scales)
    assert torch.equal(F.signbits_unpack(ck.signbits, shape[2]).cpu(), x > 0)
    # bits of pixels behind the row's last one are clear
    n, h, w = shape
    pad = (-w) % 32
    if pad:
        full = F.signbits_unpack(ck.signbits, w + pad)
        assert not bool(full[:, :, w:].any())


@pytest.mark.parametrize("shape", [(1, 1), (3, 9), (2, 5, 48), (7, 129), (300, 64)])
def test_relu_mask_from_a_checkpoint(F, shape):
    x = _values(shape, torch.bfloat16, 5)
    x = torch.where(torch.isfinite(x), x, 1.0).to(torch.bfloat16)
    dy = torch.randn(shape, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    dy.view(-1)[0] = float("nan")
    ck = F.checkpoint8_pack(x.cuda())
    want = torch.where(x.cuda() > 0, dy, torch.zeros_like(dy))
    got = F.relu_mask(dy, ck)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    assert F.relu_mask(dy, ck, out=dy) is dy and torch.equal(dy.view(torch.int16), want.view(torch.int16))   # in place


def test_relu_mask_of_values_that_are_not_finite(F):
    """NaN is not positive; an infinity is kept as NaN."""
    x = torch.tensor([[float("nan"), float("inf"), -float("inf"), 1.0, -1.0, 0.0, -0.0, 1e-30]], dtype=torch.bfloat16).cuda()
    dy = torch.arange(1, 9, dtype=torch.bfloat16, device="cuda")[None]
    assert F.relu_mask(dy, F.checkpoint8_pack(x)).tolist() == [[0, 0, 0, 4, 0, 0, 0, 8]]


def test_empty_maps_and_refusals(F):
    for shape in ((0, 64), (2, 0, 5)):
        ck = F.checkpoint8_pack(torch.empty(shape, device="cuda"))
        assert ck.shape == torch.Size(shape) and F.checkpoint8_restore(ck).shape == torch.Size(shape)
        assert F.relu_mask(torch.empty(shape, dtype=torch.bfloat16, device="cuda"), ck).numel() == 0
    x = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, device="cuda")
    ck = F.checkpoint8_pack(x)
    with pytest.raises(ValueError):
        F.checkpoint8_pack(torch.empty(3, 0, device="cuda"))
    with pytest.raises(TypeError):
        F.checkpoint8_pack(x.half())
    with pytest.raises(ValueError):
        F.checkpoint8_pack(x.float(), signbits=True)
    with pytest.raises(ValueError):
        F.checkpoint8_pack(x[..., :32], signbits=True)
    with pytest.raises(ValueError):
        F.checkpoint8_restore(ck._replace(scales=ck.scales[..., :1]))
    with pytest.raises(TypeError):
        F.checkpoint8_restore(ck._replace(codes=ck.codes.view(torch.uint8)))
    with pytest.raises(ValueError):
        F.relu_mask(x[:1], ck)
    with pytest.raises(ValueError):
        F.relu_mask(x, ck, out=torch.empty_like(x[:1]))
    dw = torch.empty(64, 64, 3, 3, device="cuda")
    with pytest.raises(ValueError, match="maps and checkpoints"):
        F.conv3x3_wgrad_multi([(ck, 0, 64, 0, x, 0, 64, 0, False), (x, 0, 64, 0, x, 0, 64, 0, False)], dw, None, 64, 64)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        F.conv3x3_wgrad(ck, x, dw, None, 16, 16, x_window=(8, 16), dz_window=(0, 16))
    with pytest.raises(ValueError):
        F.checkpoint8_wgrad(ck, x, 65, 64)
    odd = F.checkpoint8_pack(torch.zeros(1, 2, 2, 24, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="multiples of 16"):
        F.checkpoint8_wgrad(odd, torch.zeros(1, 2, 2, 16, dtype=torch.bfloat16, device="cuda"), 24, 16)


def _layer(n, h, w, cin, cout, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, h, w, cin, generator=g) * torch.exp(torch.randn(cin, generator=g))).relu().bfloat16().cuda()
    dz = (torch.randn(n, h, w, cout, generator=g) * 1e-3).bfloat16().cuda()
    return x, dz


@pytest.mark.parametrize("k", [1, 3])
@pytest.mark.parametrize("ci", [16, 32, 64])
@pytest.mark.parametrize("co", [16, 32, 64])
@pytest.mark.parametrize("size", [(1, 1, 1), (1, 5, 127), (2, 9, 130)])
def test_weight_gradient_equals_that_of_the_restored_map(F, size, ci, co, k):
    """Same products, same order of additions: bit for bit; and against 64 bits."""
    x, dz = _layer(*size, ci, co, ci + co + size[2])
    ck = F.checkpoint8_pack(x)
    dw, db = F.checkpoint8_wgrad(ck, dz, ci, co, k)
    rx = F.checkpoint8_restore(ck)
    want_w, want_b = F.conv_wgrad((rx,), dz, ci, co, k)
    assert torch.equal(dw, want_w) and torch.equal(db, want_b)
    xd, zd = torch.nn.functional.pad(rx.double().cpu(), (0, 0, k // 2, k // 2, k // 2, k // 2)), dz.double().cpu()
    n, h, w = size
    for ky in range(k):
        for kx in range(k):
            a, b = zd.reshape(-1, co), xd[:, ky:ky + h, kx:kx + w].reshape(-1, ci)
            # fp32 sums of n*h*w exact products: an addition's rounding is at most 2^-24 of the terms' sizes so far, and a
            # term passes fewer than n*h*w additions
            bound = n * h * w * 2.0 ** -24 * (a.abs().t() @ b.abs())
            assert bool(((dw[:, :, ky, kx].double().cpu() - a.t() @ b).abs() <= bound).all())
    assert bool(((db.double().cpu() - zd.sum((0, 1, 2))).abs() <= n * h * w * 2.0 ** -24 * zd.abs().sum((0, 1, 2))).all())


@pytest.mark.parametrize("cin,cout,k", [(160, 112, 1), (100, 48, 3), (256, 130, 1), (96, 64, 3)])
def test_weight_gradient_of_wide_layers(F, cin, cout, k):
    x, dz = _layer(2, 17, 33, (cin + 15) // 16 * 16, (cout + 15) // 16 * 16, cin)
    ck = F.checkpoint8_pack(x)
    got, want = F.checkpoint8_wgrad(ck, dz, cin, cout, k), F.conv_wgrad((F.checkpoint8_restore(ck),), dz, cin, cout, k)
    assert got[0].shape == (cout, cin, k, k) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("cin,cout", [(1, 1), (16, 7), (33, 129), (128, 128), (130, 250), (320, 48), (257, 257)])
@pytest.mark.parametrize("size", [(1, 1, 1), (1, 1, 31), (1, 3, 43), (2, 16, 16), (1, 70, 333)])
def test_pointwise_weight_gradients(F, size, cin, cout):
    """Every width and length of the pixel GEMM, from checkpoints and from maps: equal to each other, near to 64 bits; channels
    behind the layer's, filled with NaN here, reach nothing."""
    x, dz = _layer(*size, (cin + 15) // 16 * 16, (cout + 7) // 8 * 8, cin + cout + size[2])
    x[..., cin:], dz[..., cout:] = float("nan"), float("nan")
    ck = F.checkpoint8_pack(x)
    rx = F.checkpoint8_restore(ck)
    dw, db = F.checkpoint8_wgrad(ck, dz, cin, cout, 1)
    dw2, db2 = F.conv_wgrad((rx,), dz, cin, cout, 1)
    assert dw.shape == (cout, cin, 1, 1) and torch.equal(dw, dw2) and torch.equal(db, db2)
    a, b = dz[..., :cout].reshape(-1, cout).double().cpu(), rx[..., :cin].reshape(-1, cin).double().cpu()
    # fp32 sums of exact products: a term passes fewer additions than there are pixels, each rounding by 2^-24 of the sizes so far
    bound = a.shape[0] * 2.0 ** -24
    assert bool(((dw[:, :, 0, 0].double().cpu() - a.t() @ b).abs() <= bound * (a.abs().t() @ b.abs())).all())
    assert bool(((db.double().cpu() - a.sum(0)).abs() <= bound * a.abs().sum(0)).all())


def test_pointwise_weight_gradient_refusals(F):
    x = torch.zeros(1, 4, 4, 24, dtype=torch.bfloat16, device="cuda")
    ck = F.checkpoint8_pack(x)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        F.checkpoint8_wgrad(ck, x, 24, 24, 1)
    with pytest.raises(ValueError):
        F.conv_wgrad((x,), x[:, :2], 24, 24, 1)
    with pytest.raises(ValueError):
        F.conv_wgrad((x,), x, 25, 24, 1)
    with pytest.raises(ValueError):
        F.conv_wgrad((x[:0],), x[:0], 24, 24, 1)
    with pytest.raises(RuntimeError):
        F.conv_wgrad((x,), torch.zeros(1, 4, 4, 10, dtype=torch.bfloat16, device="cuda"), 24, 10, 1)


def test_weight_gradient_of_maps_and_checkpoints_side_by_side(F):
    xa, dz = _layer(1, 20, 70, 32, 64, 1)
    xb, _ = _layer(1, 20, 70, 64, 64, 2)
    ck = F.checkpoint8_pack(xb)
    got, want = F.conv_wgrad((xa, ck), dz, 96, 64, 3), F.conv_wgrad((xa, F.checkpoint8_restore(ck)), dz, 96, 64, 3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_weight_gradient_accumulates_scales_and_fills_a_slice(F):
    x, dz = _layer(2, 12, 40, 64, 32, 3)
    ck = F.checkpoint8_pack(x)
    base = torch.randn(32, 96, 3, 3, generator=torch.Generator().manual_seed(4)).cuda()
    a, b, ba, bb = base.clone(), base.clone(), torch.ones(32, device="cuda"), torch.ones(32, device="cuda")
    F.conv3x3_wgrad(ck, dz, a, ba, 64, 32, ci_off=32, accumulate=True, scale=0.2)
    F.conv3x3_wgrad(F.checkpoint8_restore(ck), dz, b, bb, 64, 32, ci_off=32, accumulate=True, scale=0.2)
    assert torch.equal(a, b) and torch.equal(ba, bb) and torch.equal(a[:, :32], base[:, :32])


def test_on_another_stream_and_two_calls_at_once(F):
    x, dz = _layer(1, 64, 300, 64, 64, 7)
    ref = F.checkpoint8_wgrad(F.checkpoint8_pack(x), dz, 64, 64)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] = F.checkpoint8_wgrad(F.checkpoint8_pack(x), dz, 64, 64)
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], ref[0]) and torch.equal(o[1], ref[1])


def test_captured_weight_gradients_do_not_share_a_workspace(F):
    """Two graphs recorded on one stream, replayed on two at once: from maps and from checkpoints, 3x3 and 1x1."""
    data = [_layer(2, 90, 400, 64, 64, s) for s in (3, 4)]
    cks = [F.checkpoint8_pack(x) for x, _ in data]

    def work(i):
        x, dz = data[i]
        return F.conv_wgrad((x,), dz, 64, 64, 3) + F.conv_wgrad((x,), dz, 64, 64, 1) + F.checkpoint8_wgrad(cks[i], dz, 64, 64, 3) + F.checkpoint8_wgrad(cks[i], dz, 64, 64, 1)

    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            outs.append(work(i))
        graphs.append(g)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


def test_captured_and_replayed(F):
    """Two graphs of the whole run, replayed in turn with eager calls between: every replay equals the eager result."""
    def work(x, dz):
        ck = F.checkpoint8_pack(x, signbits=True)
        return (F.checkpoint8_restore(ck), F.relu_mask(dz, ck), ck.signbits) + F.checkpoint8_wgrad(ck, dz, 64, 64)

    data = [_layer(1, 30, 90, 64, 64, s) for s in (8, 9)]
    static, graphs, outs = [tuple(t.clone() for t in data[0]) for _ in range(2)], [], []
    work(*static[0])
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(*static[i]))
        graphs.append(graph)
    for turn in range(3):
        for i in range(2):
            for s, d in zip(static[i], data[(i + turn) % 2]):
                s.copy_(d)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = work(*data[(i + turn) % 2])
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want):
                assert torch.equal(a, b)


def _room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GB")


@pytest.mark.parametrize("rows,c,dtype", [((1 << 30) // 2 + 77, 64, torch.bfloat16), ((1 << 31) + 4321, 1, torch.bfloat16), ((1 << 31) + 513, 9, torch.bfloat16)])
def test_maps_that_take_more_than_one_launch(F, rows, c, dtype):
    """More rows than a launch holds (2^32 threads, or 2^31 units): values at the start, around where the launches meet and at the end are
    those of the same rows on their own, zeros in between; saved, brought back, as a ReLU mask."""
    _room(190)
    groups = (c + 31) // 32
    lanes = 1 if c <= 8 else 2 if c <= 16 else 4
    meet = min((1 << 32) // lanes, 1 << 31) // groups
    places = [0, meet - 700, rows - 400]
    blocks = [_values((min(1000, rows - p), c), dtype, p % 97).cuda() for p in places]
    x = torch.zeros((rows, c), dtype=dtype, device="cuda")
    for p, b in zip(places, blocks):
        x[p:p + len(b)] = b
    ck = F.checkpoint8_pack(x)
    dy = torch.empty_like(x).fill_(3.0) if x.numel() < 1 << 35 else None
    del x
    want = [F.checkpoint8_pack(b) for b in blocks]

    def same(t, of):
        for p, w in zip(places, want):
            b = of(w)
            n = min([len(b)] + [q - p for q in places if q > p])       # where two overlap the later one stands
            assert torch.equal(t[p:p + n], b[:n]), p
        for lo in range(1000, places[1], 1 << 24):
            assert not bool(t[lo:min(lo + (1 << 24), places[1])].any()), lo

    same(ck.codes.view(torch.uint8), lambda w: w.codes.view(torch.uint8))
    assert torch.equal(ck.scales[-400:], want[-1].scales[-400:])
    y = F.checkpoint8_restore(ck)
    same(y.view(torch.int16), lambda w: F.checkpoint8_restore(w).view(torch.int16))
    if dy is None:
        dy = y      # in place: the map itself where it is positive
        mask = lambda w: F.relu_mask(F.checkpoint8_restore(w), w).view(torch.int16)  # noqa: E731
    else:
        del y
        mask = lambda w: F.relu_mask(torch.full(w.codes.shape, 3.0, dtype=dtype, device="cuda"), w).view(torch.int16)  # noqa: E731
    same(F.relu_mask(dy, ck, out=dy).view(torch.int16), mask)
    del ck, dy
    torch.cuda.empty_cache()

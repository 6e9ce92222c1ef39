"""CPU checks of the 8-bit checkpoints and the fused block norm: the oracle against the e4m3 type and against differences, the
boundary's structs and refusals (C entries are called with arguments that they turn down before any launch)."""
import ctypes

import pytest
import torch

from oracle import checkpoint8 as orc


def test_oracle_codes_are_the_e4m3_numbers():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double()
    got = orc.decode(codes[:, None], torch.full((256, 1), 127, dtype=torch.uint8))[:, 0]
    assert torch.equal(torch.isnan(want), torch.isnan(got))
    assert torch.equal(want.nan_to_num(), got.nan_to_num())


def test_oracle_rounds_like_the_type_and_never_saturates():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 70, generator=g) * torch.exp(torch.randn(64, 1, generator=g) * 8)
    codes, scales = orc.encode(x)
    assert scales.shape == (64, 3)
    s = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)[:, :70]
    want = (x.double() / s).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = (want & 127) != 0
    assert torch.equal(codes[keep], want[keep]) and bool(((codes & 127) == 1)[~keep & (x != 0)].all())
    top = (x.double() / s).abs()
    for lo in (0, 32, 64):
        assert bool((top[:, lo:lo + 32].amax(-1) <= 448).all()) and bool((top[:, lo:lo + 32].amax(-1) > 224).all())


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", [None, "channel", "sample", "map"])
@pytest.mark.parametrize("act", ["none", "sigmoid"])
def test_oracle_gradients_against_differences(kind, gate, act):
    g = torch.Generator().manual_seed(1)
    D, shape, c = torch.float64, (2, 3, 5), 5
    n = lambda *s: torch.randn(s, generator=g, dtype=D)  # noqa: E731
    x, h, dr, dn = n(*shape), n(*shape), n(*shape), n(*shape)
    post, pre = (n(c), n(c)), (n(c), n(c))
    gt = {None: None, "channel": lambda: n(c), "sample": lambda: n(2, c), "map": lambda: n(*shape)}[gate]
    gt = gt() if gt else None
    scale = n(1)[0]

    def value(x, h, pw, pb, qw, qb, s, *gg):
        (r, m), _ = orc.norm_residual(x, h, (pw, pb), gg[0] if gg else None, s, (qw, qb), kind, act)
        return float((r * dr).sum() + (m * dn).sum())

    args = [x, h, post[0], post[1], pre[0], pre[1], scale] + ([gt] if gt is not None else [])
    (r, _), _ = orc.norm_residual(x, h, post, gt, scale, pre, kind, act)
    got, _ = orc.norm_residual_bwd(h, r, dr, dn, post, gt, scale, pre, kind, act, True)
    names = ["dx", "dh", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias", "dscale", "dgate"]
    for i, name in zip(range(len(args)), names):
        v = torch.randn(args[i].shape, generator=g, dtype=D)
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + 1e-5 * v, args[i] - 1e-5 * v
        want = (value(*hi) - value(*lo)) / 2e-5
        # central differences: error of the order step^2 times the third derivative, and 1e-16 / step of rounding
        assert abs(float((got[name] * v).sum()) - want) <= 1e-6 * (1 + abs(want)), name


def test_struct_layouts():
    from superresolution_amd._lib import NormResidualArgs, NormResidualBwdArgs
    assert ctypes.sizeof(NormResidualArgs) == 10 * 8 + 2 * 8 + 8 * 4 + 2 * 4
    assert ctypes.sizeof(NormResidualBwdArgs) == 20 * 8 + 2 * 8 + 8 * 4 + 2 * 4
    assert NormResidualArgs.rows.offset == 80 and NormResidualArgs.c.offset == 96 and NormResidualArgs.scale.offset == 128
    assert NormResidualBwdArgs.workspace.offset == 152 and NormResidualBwdArgs.rows.offset == 160 and NormResidualBwdArgs.eps.offset == 212


P = 1 << 20   # an address that no refused call reads


def _refused(rc, text):
    from superresolution_amd._lib import lib
    assert rc == -1 and text in lib.srhip_last_error().decode(), (rc, lib.srhip_last_error())


def test_c_entries_refuse_before_any_launch():
    from superresolution_amd._lib import NormResidualArgs, NormResidualBwdArgs, WgradJob, lib
    _refused(lib.srhip_checkpoint8_pack(P, 7, P, P, 1, 32, None), "unknown type")
    _refused(lib.srhip_checkpoint8_pack(P, 0, P, P, 1, 0, None), "bad shape")
    _refused(lib.srhip_checkpoint8_pack(P, 0, P, P, -1, 3, None), "bad shape")
    _refused(lib.srhip_checkpoint8_pack(P, 0, None, P, 1, 3, None), "null pointer")
    _refused(lib.srhip_checkpoint8_restore(P, P, None, 0, 1, 3, None), "null pointer")
    _refused(lib.srhip_checkpoint8_pack_signbits(P + 8, P, P, P, 1, 1, 1, None), "multiples of 16")
    _refused(lib.srhip_relu_mask_checkpoint8(P, None, P, 8, None), "null pointer")
    assert lib.srhip_checkpoint8_pack(None, 0, None, None, 0, 3, None) == 0      # no rows: nothing to do
    assert lib.srhip_checkpoint8_restore(None, None, None, 1, 0, 3, None) == 0
    assert lib.srhip_relu_mask_checkpoint8(None, None, None, 0, None) == 0

    job = (WgradJob * 1)(WgradJob(x=P, dz=P, dw=P, db=None, ci_real=16, ci_off=0, co_real=16, x_cstride=16, x_coff=0, dz_cstride=16, dz_coff=0))
    sc = (ctypes.c_void_p * 1)(P)
    _refused(lib.srhip_conv_wgrad_checkpoint8(job, None, 1, P, 1, 1, 1, 16, 16, 16, 3, 0, 1.0, None), "null pointer")
    _refused(lib.srhip_conv_wgrad_checkpoint8(job, sc, 1, P, 1, 1, 1, 16, 16, 16, 5, 0, 1.0, None), "kernel size")
    _refused(lib.srhip_conv_wgrad_checkpoint8(job, (ctypes.c_void_p * 1)(None), 1, P, 1, 1, 1, 16, 16, 16, 3, 0, 1.0, None), "null scales")
    job[0].x_cstride = 24
    _refused(lib.srhip_conv_wgrad_checkpoint8(job, sc, 1, P, 1, 1, 1, 16, 16, 16, 3, 0, 1.0, None), "multiples of 16")
    job[0].x_cstride, job[0].x = 16, P + 8
    _refused(lib.srhip_conv_wgrad_checkpoint8(job, sc, 1, P, 1, 1, 1, 16, 16, 16, 3, 0, 1.0, None), "multiples of 16")

    _refused(lib.srhip_wgrad1x1(P, P, P, P, P, P, 0, 16, 16, 16, 16, None), "empty layer")
    _refused(lib.srhip_wgrad1x1(P, P, None, P, P, P, 8, 16, 16, 16, 16, None), "null pointer")
    _refused(lib.srhip_wgrad1x1(P, P, P, P, P, P, 8, 16, 24, 16, 16, None), "multiples of 16")
    _refused(lib.srhip_wgrad1x1(P, None, P, P, P, P, 8, 16, 16, 17, 16, None), "channels per pixel")
    _refused(lib.srhip_wgrad1x1(P + 2, None, P, P, P, P, 8, 16, 16, 16, 16, None), "multiples of 16 bytes")
    _refused(lib.srhip_wgrad1x1(P, None, P, P, P, None, 1 << 20, 16, 16, 16, 16, None), "null workspace")
    assert lib.srhip_wgrad1x1_workspace_bytes(0, 16, 16) == 0 and lib.srhip_wgrad1x1_workspace_bytes(100, 16, 16) == 0

    a = dict(x=P, h=P, r=P, n=P, pre_weight=P, post_weight=P, rows=4, rows_per_gate=2, c=8, post=1, pre=1, eps=1e-6)
    for change, text in ((dict(c=0), "bad shape"), (dict(c=8193), "bad shape"), (dict(rows=-1), "bad shape"), (dict(dtype=2), "unknown type"),
                         (dict(kind=2), "unknown norm"), (dict(gate_mode=3), "unknown gate"), (dict(h=None, pre=0), "neither"),
                         (dict(h=None), "without a branch"), (dict(eps=-1.0), "eps"), (dict(n=None), "null pointer"),
                         (dict(pre_weight=None), "null pointer"), (dict(gate_mode=1), "null gate"),
                         (dict(gate_mode=1, gate=P, rows_per_gate=3), "not a multiple"), (dict(gate_mode=1, gate=P, rows_per_gate=0), "not a multiple")):
        _refused(lib.srhip_norm_residual_fwd(NormResidualArgs(**{**a, **change}), None), text)
    assert lib.srhip_norm_residual_fwd(NormResidualArgs(**{**a, "rows": 0}), None) == 0
    _refused(lib.srhip_norm_residual_fwd(None, None), "null pointer")

    b = dict(h=P, r=P, dr=P, dn=P, dx=P, dh=P, pre_weight=P, post_weight=P, dpost_weight=P, dpre_weight=P, workspace=P, rows=4, rows_per_gate=2, c=8,
             post=1, pre=1, eps=1e-6)
    for change, text in ((dict(c=8193), "bad shape"), (dict(dtype=9), "unknown type"), (dict(kind=-1), "unknown norm"), (dict(rows=0), "no rows"),
                         (dict(dx=None), "null pointer"), (dict(dn=None), "behind the sum"), (dict(r=None), "behind the sum"),
                         (dict(dh=None), "without a branch"), (dict(dpost_weight=None), "post norm"), (dict(gate_mode=2, gate=P), "null gate"),
                         (dict(h=None), "null branch"), (dict(workspace=None), "null workspace"),
                         (dict(gate_mode=1, gate=P, dgate=P, rows_per_gate=3), "not a multiple"), (dict(dr=None, pre=0), "null pointer")):
        _refused(lib.srhip_norm_residual_bwd(NormResidualBwdArgs(**{**b, **change}), None), text)
    assert lib.srhip_norm_residual_bwd_workspace_bytes(NormResidualBwdArgs(**{**b, "c": 0})) == 0


def test_python_entries_refuse_host_tensors_and_wrong_types():
    from superresolution_amd import functional as F
    x = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="GPU"):
        F.checkpoint8_pack(x)
    with pytest.raises(TypeError):
        F.checkpoint8_pack(x.half())
    ck = F.Checkpoint8(x.to(torch.float8_e4m3fn), torch.zeros(2, 4, 2, dtype=torch.uint8), torch.float32)
    with pytest.raises(ValueError, match="GPU"):
        F.checkpoint8_restore(ck)
    with pytest.raises(ValueError, match="GPU"):
        F.norm_residual(x, x, pre=(torch.ones(64), None))
    with pytest.raises(TypeError):
        F.norm_residual(x.double(), x.double())
    with pytest.raises(ValueError):
        F.norm_residual_bwd(x, x, None, None)
    with pytest.raises(ValueError):
        F.norm_residual_bwd(x, x, x, x)
    with pytest.raises(ValueError):
        F.conv_wgrad((x[None],), x[None], 64, 64, 5)


def test_launches_of_too_many_threads_are_refused_on_the_host():
    from superresolution_amd._lib import lib
    # one pixel to a group of 32: 2^26 groups, 2^32 threads
    _refused(lib.srhip_checkpoint8_pack_signbits(P, P, P, P, 1024, 65536, 1, None), "too large")
    # 2^28 weights: 2^32 threads of the launch that adds the runs (1024 for 64), square or in a row
    _refused(lib.srhip_wgrad1x1(P, None, P, P, P, P, 1 << 20, 1 << 14, 1 << 14, 1 << 14, 1 << 14, None), "too large")
    _refused(lib.srhip_wgrad1x1(P, None, P, P, P, P, 64, 1 << 28, 1 << 28, 1, 8, None), "too large")

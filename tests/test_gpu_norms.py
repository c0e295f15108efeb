"""gated_norm and residual_norm against their 64-bit definitions."""
import pytest
import torch

import rows_util as ru
from rows_util import ALL, IDS

pytestmark = pytest.mark.gpu

LENGTHS = [1, 7, 64, 511, 512, 520, 1000, 1024, 1283, 2048, 2055, 4096, 5000, 8192, 10001, 16384, 16385, 20479, 33000]


def values(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def cuda(t):
    return None if t is None else t.cuda()


def check_gated(x, w, z, groups=1, norm_first=False, eps=1e-5):
    from pto_einsum import gated_norm

    ref, units = ru.gated(x, w, z, eps, groups, norm_first)
    more = dict(groups=groups, norm_first=norm_first, eps=eps)
    y = gated_norm(cuda(x), cuda(w), cuda(z), **more)
    assert y.dtype is x.dtype and y.is_contiguous()
    ru.assert_within(y, ref, ru.gated_bound(ref, units, x.dtype), "y")
    q, s = gated_norm(cuda(x), cuda(w), cuda(z), quantize=True, **more)
    assert q.dtype is torch.int8 and s.shape == x.shape[:-1]
    err = ru.U * units * ref.abs()
    ru.assert_within(q.double() * s.double()[..., None], ref, ru.rows_bound(ref, err, s.cpu()), "rows")
    return y, q, s


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("d", LENGTHS)
def test_gated(d, dtype):
    x, z, w = values((3, d), dtype, d), values((3, d), dtype, d + 1, 2.0), values((d,), dtype, d + 2)
    check_gated(x, w, z)
    check_gated(x, w, z, norm_first=True)
    check_gated(x, None, None)


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("d,groups", [(512, 8), (4096, 8), (1000, 5), (77, 7), (30000, 3), (8192, 8192), (48000, 2), (9, 9),
                                      (33, 11), (40010, 10), (34002, 2),
                                      # groups of whole 512 elements, and a few more
                                      (1024, 2), (1024, 1), (1536, 3), (3584, 7), (4096, 2), (8192, 16), (7168, 7),
                                      (12288, 3), (16384, 32), (16384, 4), (17408, 2), (1040, 2), (2064, 4)])
def test_groups(d, groups, dtype):
    x, z, w = values((2, 3, d), dtype, d), values((2, 3, d), dtype, d + 1), values((d,), dtype, d + 2)
    check_gated(x, w, z, groups=groups)
    check_gated(x, w, z, groups=groups, norm_first=True)


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
def test_gated_slices_and_orders(dtype):
    """x and the gate as slices of a projection, leading axes in other orders."""
    wide = values((4, 5, 1500), dtype, 1)
    x, z, w = wide[..., 3:703], wide[..., 703:1403], values((700,), dtype, 2)
    y, q, s = check_gated(x, w, z)
    from pto_einsum import gated_norm

    g = wide.cuda()
    for xs, zs in ((g[..., 3:703], g[..., 703:1403]),
                   (g[..., 3:703].transpose(0, 1).contiguous().transpose(0, 1), g[..., 703:1403]),
                   (g[..., 3:703], g[..., 703:1403].transpose(1, 2).contiguous().transpose(1, 2))):
        assert torch.equal(gated_norm(xs, w.cuda(), zs), y)
        q2, s2 = gated_norm(xs, w.cuda(), zs, quantize=True)
        assert torch.equal(q2, q) and torch.equal(s2, s)
    # every second channel of the weight
    w2 = torch.stack([w, w + 1], 1).cuda()[:, 0]
    assert torch.equal(gated_norm(x.cuda(), w2, z.cuda()), y)


@pytest.mark.parametrize("eps", [0.0, 1e-12, 0.5])
def test_eps_and_rows_of_zeros(eps):
    x = values((4, 300), torch.float32, 5)
    x[1] = 0
    from pto_einsum import gated_norm

    y = gated_norm(x.cuda(), eps=eps).cpu()
    want = x.double() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + eps)
    keep = [0, 2, 3]
    ru.assert_within(y[keep], want[keep], 40 * ru.U * want[keep].abs(), "rows")
    # 0 / 0 without eps, as the formula has it
    assert torch.isnan(y[1]).all() if eps == 0 else not y[1].any()


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("d", [40, 1500, 20000])
def test_infinities_and_nan_stay_in_their_rows(d, dtype):
    from pto_einsum import gated_norm, residual_norm

    x, z = values((6, d), dtype, 1), values((6, d), dtype, 2)
    clean = gated_norm(x.cuda(), None, z.cuda())
    x[1, d - 1], x[2, 0], z[3, d // 2] = float("nan"), float("inf"), float("nan")
    y = gated_norm(x.cuda(), None, z.cuda())
    q, s = gated_norm(x.cuda(), None, z.cuda(), quantize=True)
    rest = [0, 4, 5]
    assert torch.equal(y[rest], clean[rest])
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.isnan(y[2, 0])
    assert torch.isnan(s[1:4]).all() and not q[1:4].any() and torch.isfinite(s[rest]).all()
    y, r = residual_norm(x.cuda(), z.cuda())
    assert torch.isnan(y[1]).all() and torch.isnan(r[1, d - 1]) and torch.isfinite(r[1, :d - 1]).all()
    assert torch.isfinite(y[rest]).all()


def check_residual(x, res, w, pw, gate, scale=1.0, eps=1e-5):
    from pto_einsum import residual_norm

    y_ref, r_ref, y_err, r_err = ru.residual(x, res, w, pw, gate, scale, eps)
    args = (cuda(x), cuda(res), cuda(w))
    more = dict(post_weight=cuda(pw), gate=cuda(gate), scale=scale, eps=eps)
    y, r = residual_norm(*args, **more)
    assert y.dtype is x.dtype and r.dtype is res.dtype and y.is_contiguous() and r.is_contiguous()
    ru.assert_within(r, r_ref, ru.bound(r_ref, r_err, res.dtype), "r")
    ru.assert_within(y, y_ref, ru.bound(y_ref, y_err, x.dtype), "y")
    (q, s), r2 = residual_norm(*args, quantize=True, **more)
    assert torch.equal(r, r2)
    ru.assert_within(q.double() * s.double()[..., None], y_ref, ru.rows_bound(y_ref, y_err, s.cpu()), "rows")
    return y, r


@pytest.mark.parametrize("wide", [False, True], ids=["same", "float32"])
@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("d", LENGTHS)
def test_residual(d, dtype, wide):
    x, w, pw = values((3, d), dtype, d), values((d,), dtype, d + 1), values((d,), dtype, d + 2)
    res = values((3, d), torch.float32 if wide else dtype, d + 3, 2.0)
    check_residual(x, res, w, pw, values((3, d), dtype, d + 4), 0.7)
    check_residual(x, res, w, None, None)
    check_residual(x, res, None, pw, None, -0.25)


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("d", [48, 1283, 17000])
@pytest.mark.parametrize("shape", ["(d,)", "(1, d)", "(b, 1, d)", "(1, t, d)", "(b, t, d)", "(b, t, 1)", "(b, 1, 1)", "(1,)",
                                   "()", "(t, 1)"])
def test_gates(shape, d, dtype):
    b, t = 3, 4
    x, res, w = values((b, t, d), dtype, 1), values((b, t, d), dtype, 2), values((d,), dtype, 3)
    check_residual(x, res, w, None, values(eval(shape, {}, dict(b=b, t=t, d=d)), dtype, 4))


def test_residual_orders():
    """Leading axes of the operands in different orders; a strided gate."""
    from pto_einsum import residual_norm

    x, res, gate = (values((3, 4, 5, 200), torch.float16, i) for i in range(3))
    y, r = check_residual(x, res, None, None, gate)
    xs = x.cuda().permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    rs = res.cuda().permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)
    gs = gate.cuda().transpose(2, 3).contiguous().transpose(2, 3)
    wide = torch.zeros(3, 4, 5, 400, dtype=torch.float16, device="cuda")
    wide[..., ::2] = gate.cuda()
    for g in (gate.cuda(), gs, wide[..., ::2]):
        y2, r2 = residual_norm(xs, rs, gate=g)
        assert torch.equal(y, y2) and torch.equal(r, r2) and r2.is_contiguous()
    per_row = values((3, 4, 5, 1), torch.float16, 9).cuda()
    sparse = torch.zeros(3, 4, 5, 7, dtype=torch.float16, device="cuda")
    sparse[..., 3:4] = per_row
    assert torch.equal(residual_norm(xs, rs, gate=sparse[..., 3:4])[0], residual_norm(x.cuda(), res.cuda(), gate=per_row)[0])


def test_y_comes_from_the_unrounded_sum():
    """A residual that swallows x in 16 bits: r rounds back to it, y does not."""
    from pto_einsum import residual_norm

    x = torch.full((1, 64), 0.25, dtype=torch.bfloat16)
    res = torch.full((1, 64), 256.0, dtype=torch.bfloat16)
    res[0, ::2] = -256.0
    y, r = residual_norm(x.cuda(), res.cuda(), scale=1.0)
    assert torch.equal(r.cpu(), res)
    (q, s), _ = residual_norm(x.cuda().float(), res.cuda().float(), quantize=True)
    assert float(s) > 1.0 / 127


@pytest.mark.parametrize("shape", [(0, 8), (2, 0, 8), (3, 0)])
def test_empty(shape):
    from pto_einsum import gated_norm, residual_norm

    x = torch.zeros(shape, dtype=torch.float16, device="cuda")
    w = torch.zeros(shape[-1], dtype=torch.float16, device="cuda")
    assert gated_norm(x, w, x).shape == shape
    q, s = gated_norm(x, w, x, quantize=True)
    assert q.shape == shape and s.shape == shape[:-1] and not s.any()
    y, r = residual_norm(x, x, w, gate=x)
    assert y.shape == shape and r.shape == shape


def test_many_rows():
    """More rows than a launch has blocks for, each read in its place."""
    from pto_einsum import gated_norm, residual_norm

    x = torch.randn(4_500_000, 16, device="cuda").half()
    z = torch.randn(4_500_000, 16, device="cuda").half()
    y = gated_norm(x, None, z, groups=2)
    at = torch.tensor([0, 1, 2_097_151, 2_097_152, 4_194_303, 4_194_304, 4_499_999], device="cuda")
    ref, units = ru.gated(x[at].cpu(), None, z[at].cpu(), 1e-5, 2, False)
    ru.assert_within(y[at], ref, ru.gated_bound(ref, units, torch.float16))
    y, r = residual_norm(x, z)
    y_ref, r_ref, y_err, r_err = ru.residual(x[at].cpu(), z[at].cpu(), None, None, None, 1.0, 1e-5)
    ru.assert_within(y[at], y_ref, ru.bound(y_ref, y_err, torch.float16))
    ru.assert_within(r[at], r_ref, ru.bound(r_ref, r_err, torch.float16))

"""Norms of rows whose squares float32 does not hold: values from 1e19 on, and small
ones with an eps as small, against the 64-bit definitions."""
import pytest
import torch

import rows_util as ru

pytestmark = pytest.mark.gpu

WIDE = [torch.bfloat16, torch.float32]
IDS = ["bf16", "f32"]
# (a gate's product and a sum are float32: where the smallest are multiples of 2^-149,
# nothing relative holds of them)
SUMS = [1e-28, 1e-21, 1e-16, 1e18, 2e19, 1e27, 1e37]
SIZES = [2.0 ** -148, 1e-42, 1e-36, *SUMS]
# every width of the kernel, and the one for long rows
LENGTHS = [1, 5, 300, 512, 700, 1500, 3000, 8192, 16384, 20000]


def rows(d, dtype, seed, sizes=SIZES):
    """A row of each size, the first and the last of size 1."""
    g = torch.Generator().manual_seed(seed)
    size = torch.tensor([1.0, *sizes, 1.0], dtype=torch.float64)
    return nonzero((torch.randn(len(size), d, generator=g, dtype=torch.float64) * size[:, None]).to(dtype))


def nonzero(x):
    """x, the first of a row of nothing but zeros (0 / 0 without eps) the smallest bfloat16."""
    x[..., 0] = torch.where((x == 0).all(-1), 2.0 ** -133, x[..., 0])
    return x


def sizable(ref):
    """Rows whose scale in 8 bits is a normal float32."""
    return ref.abs().amax(-1) > 1e-30


def weight(d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.1 * torch.randn(d, generator=g)).to(dtype)


def cuda(t):
    return None if t is None else t.cuda()


def lost(x, w, z, norm_first):
    """What the float32 products of y lose below 2^-126, where a rounding is up to 2^-150
    whatever the value: x times its factor, that times the weight, that times the gate;
    each loss is multiplied by what follows."""
    w = torch.ones(x.shape[-1]) if w is None else w.double().abs()
    g = ru.silu(z.double()).abs() if z is not None and norm_first else torch.ones(x.shape)
    return 2.0 ** -150 * (w * g + g + 1)


def check_gated(x, w, z, groups, norm_first, eps):
    from pto_einsum import gated_norm

    more = dict(groups=groups, norm_first=norm_first, eps=eps)
    ref, units = ru.gated(x, w, z, eps, groups, norm_first)
    y = gated_norm(cuda(x), cuda(w), cuda(z), **more)
    ru.assert_within(y, ref, ru.gated_bound(ref, units, x.dtype) + lost(x, w, z, norm_first), "y")
    q, s = gated_norm(cuda(x), cuda(w), cuda(z), quantize=True, **more)
    at = sizable(ref)
    limit = ru.rows_bound(ref, ru.U * units * ref.abs(), s.cpu())
    ru.assert_within((q.double() * s.double()[..., None])[at.cuda()], ref[at], limit[at], "rows")
    # rows of ordinary size are what they are alone
    for i in (0, len(x) - 1):
        alone = gated_norm(cuda(x[i:i + 1]), cuda(w), cuda(None if z is None else z[i:i + 1]), **more)
        assert torch.equal(alone[0], y[i])


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -140, 1e-5])
@pytest.mark.parametrize("dtype", WIDE, ids=IDS)
@pytest.mark.parametrize("d", LENGTHS)
def test_gated(d, dtype, eps):
    x, w = rows(d, dtype, d), weight(d, dtype, d + 1)
    z = rows(d, dtype, d + 2, [1.0] * len(SIZES))
    check_gated(x, w, None, 1, False, eps)
    check_gated(x, w, z, 1, True, eps)
    x = rows(d, dtype, d, SUMS)
    check_gated(x, w, z[:len(x)], 1, False, eps)


@pytest.mark.parametrize("dtype", WIDE, ids=IDS)
@pytest.mark.parametrize("d,groups", [(1024, 2), (2048, 4), (4096, 2), (4096, 8), (8192, 4), (16384, 32), (1000, 5), (77, 7),
                                      (17408, 2), (40010, 10)])
def test_groups_of_different_sizes(d, groups, dtype):
    """Each group of a row of a size of its own."""
    g = torch.Generator().manual_seed(d)
    x = torch.randn(4, groups, d // groups, generator=g, dtype=torch.float64)
    at = torch.randint(0, len(SUMS), (4, groups), generator=g)
    size = torch.tensor(SUMS, dtype=torch.float64)[at]
    size[0], size[3] = 1.0, 1.0
    x = (x * size[..., None]).flatten(1).to(dtype)
    z = torch.randn(4, d, generator=g).to(dtype)
    for eps in (0.0, 1e-5):
        check_gated(x, weight(d, dtype, 1), z, groups, False, eps)
        check_gated(x, None, z, groups, True, eps)


@pytest.mark.parametrize("dtype", WIDE, ids=IDS)
@pytest.mark.parametrize("d", LENGTHS)
def test_residual(d, dtype):
    from pto_einsum import residual_norm

    x, w, pw = rows(d, dtype, d), weight(d, dtype, d + 1), weight(d, dtype, d + 2)
    xs, res = rows(d, dtype, d, SUMS), rows(d, torch.float32, d + 3, SUMS)
    unit = rows(d, torch.float32, d + 4, [1.0] * len(SIZES))
    gate = weight(d, dtype, d + 5)
    for eps in (0.0, 2.0 ** -140, 1e-5):
        # sums of every size; and a block's output of every size, whose norm brings it to 1
        for x0, r0, post in ((xs, res, None), (xs, res.to(dtype), None), (x, unit, pw), (x, unit.to(dtype), pw)):
            args, more = (cuda(x0), cuda(r0), cuda(w)), dict(post_weight=cuda(post), gate=cuda(gate), scale=0.5, eps=eps)
            y_ref, r_ref, y_err, r_err = ru.residual(x0, r0, w, post, gate, 0.5, eps)
            y, r = residual_norm(*args, **more)
            ru.assert_within(r, r_ref, ru.bound(r_ref, r_err, r0.dtype), "r")
            ru.assert_within(y, y_ref, ru.bound(y_ref, y_err, dtype), "y")
            (q, s), r2 = residual_norm(*args, quantize=True, **more)
            assert torch.equal(r, r2)
            at = sizable(y_ref)
            limit = ru.rows_bound(y_ref, y_err, s.cpu())
            ru.assert_within((q.double() * s.double()[..., None])[at.cuda()], y_ref[at], limit[at], "rows")


@pytest.mark.parametrize("d", [1, 40, 700, 3000, 16384, 20000])
def test_infinities_stay(d):
    """A row with an infinity: NaN there, 0 elsewhere, as the definition has it."""
    from pto_einsum import gated_norm

    x = rows(d, torch.float32, 1)
    x[3, d // 2] = float("-inf")
    y = gated_norm(x.cuda(), eps=0.0).cpu()
    assert torch.isnan(y[3, d // 2]) and int(torch.isnan(y).sum()) == 1
    assert not y[3].nan_to_num(nan=0.0).any()

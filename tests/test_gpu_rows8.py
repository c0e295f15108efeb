"""Rows in 8 bits: values, scales and their padding against the definition."""
import pytest
import torch

from rows_util import ALL, IDS, quantize

pytestmark = pytest.mark.gpu


def run(x):
    from pto_einsum import quantize_q8

    q, s = quantize_q8(x)
    assert q.shape == x.shape and q.dtype is torch.int8 and s.shape == x.shape[:-1] and s.dtype is torch.float32
    return q, s


def assert_same(x, q, s):
    want, scale = quantize(x.cpu())
    assert torch.equal(q.cpu().double(), want)
    assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(scale.float(), nan=-1.0))


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (3, 16), (2, 511), (4, 513), (3, 1000), (2, 1025), (3, 2048), (2, 2055),
                                   (2, 4097), (3, 8192), (2, 8200), (1, 16384), (2, 16385), (1, 40003), (300, 24),
                                   (2, 3, 5, 100)])
def test_values_and_scales(shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=g) * torch.exp(2 * torch.randn((*shape[:-1], 1), generator=g))).to(dtype)
    q, s = run(x.cuda())
    # (the scale of a float64 quotient rounded again is the float32 quotient:
    # 53 bits are more than twice 24 and 2)
    assert_same(x, q, s)


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
def test_ties_go_to_even(dtype):
    """Largest values of every mantissa and their halves, quarters and thirds of
    them, whose quotients are halves or next to one."""
    top = (torch.arange(128, 256).float() / 128).to(dtype)
    parts = torch.tensor([0.5, 0.25, 0.125, 1 / 3, 3 / 254, 1 / 254, 5 / 254, 253 / 254, 127 / 254])
    x = torch.cat([top[:, None].float(), top[:, None].float() * parts, -top[:, None].float() * parts], 1).to(dtype)
    assert_same(x, *run(x.cuda()))
    assert_same(x.repeat(1, 60), *run(x.repeat(1, 60).cuda()))


def test_float32_next_to_ties():
    """Values a unit in the last place off (k + 1/2) / 127 of the largest one."""
    g = torch.Generator().manual_seed(7)
    top = 1 + torch.rand(64, 1, generator=g)
    half = (top.double() * (torch.arange(127) + 0.5) / 127).float()
    x = torch.cat([top, half, torch.nextafter(half, torch.tensor(9.0)), torch.nextafter(half, torch.tensor(0.0))], 1)
    assert_same(x, *run(x.cuda()))


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("k", [40, 1100, 5000, 20000])
def test_rows_of_zeros_infinities_and_nan(k, dtype):
    g = torch.Generator().manual_seed(k)
    x = torch.randn(7, k, generator=g).to(dtype)
    x[0] = 0
    x[1, k - 1] = float("inf")
    x[2, 3] = float("-inf")
    x[3, k // 2] = float("nan")
    x[4] = 0
    x[4, k - 2] = -0.0
    q, s = run(x.cuda())
    assert_same(x, q, s)
    assert torch.isnan(s[1:4]).all() and not torch.isnan(s[[0, 4, 5, 6]]).any()


@pytest.mark.parametrize("size", [2.0 ** -149, 2.0 ** -140, 1e-38, 1e-36, 3e-36, 1e30, 3.4e38])
def test_float32_near_both_ends(size):
    g = torch.Generator().manual_seed(3)
    x = (torch.rand(9, 333, generator=g).double() * 2 - 1) * size
    x = x.float()
    q, s = run(x.cuda())
    want, scale = quantize(x)
    assert torch.equal(q.cpu().double(), want)
    # (a scale below float32's normal range is itself rounded to a multiple of 2^-149)
    assert torch.equal(s.cpu(), scale.float())


@pytest.mark.parametrize("k,pitch", [(3, 16), (1003, 1008), (1100, 1152), (5001, 5120), (16300, 16384), (17001, 17024)])
def test_padding_is_zero(k, pitch):
    from pto_einsum import quantize_q8

    x = torch.randn(37, k, device="cuda")
    for _ in range(2):
        q, _ = quantize_q8(x)
        assert q.stride() == (pitch, 1)
        pad = q.as_strided((37, pitch - k), (pitch, 1), k)
        assert not pad.any()
        pad.fill_(77)
        del q, pad          # (what the next rows get)


def test_strides_and_broadcast_rows():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 5, 300, generator=g).to(torch.float16)
    wide = torch.randn(6, 5, 700, generator=g).to(torch.float16)
    wide[..., 11:311] = x
    for view in (wide.cuda()[..., 11:311], x.cuda().transpose(0, 1).contiguous().transpose(0, 1),
                 x.cuda().transpose(1, 2).contiguous().transpose(1, 2)):
        assert_same(x, *run(view))
    row = x[0, 0].cuda().expand(4, 300)
    assert_same(x[0, 0].expand(4, 300), *run(row))


def test_empty():
    for shape in ((0, 5), (3, 0, 7), (4, 0)):
        q, s = run(torch.zeros(shape, device="cuda", dtype=torch.float16))
        assert not s.numel() or torch.equal(s.cpu(), torch.zeros(4))


def test_many_rows():
    """More rows than a launch has blocks for."""
    x = torch.randn(5_000_000, 8, device="cuda").to(torch.bfloat16)
    q, s = run(x)
    at = torch.tensor([0, 1, 4_194_303, 4_194_304, 4_194_305, 4_999_999], device="cuda")
    assert_same(x[at], q[at], s[at])
    top = x.float().abs().amax(-1)
    assert torch.equal(s, top / torch.full_like(top, 127.0))

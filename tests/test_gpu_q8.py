"""matmul_q8 against the exact product: whole sums, then a few float32 roundings."""
import pytest
import torch

import rows_util as ru
from rows_util import ALL, IDS

pytestmark = pytest.mark.gpu


def whole(shape, seed, lo=-127, hi=127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi + 1, shape, generator=g, dtype=torch.int8)


def uniform(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(shape, generator=g) * 1e-2 + 1e-3


def padded(t, fill=0):
    """t in rows every 16 bytes, the bytes between of some value."""
    k = t.shape[-1]
    out = torch.full((*t.shape[:-1], -(-k // 16) * 16), fill, dtype=torch.int8, device="cuda")
    out[..., :k] = t.cuda()
    return out[..., :k]


def check(q, w, dtype, bias=None, fill=0):
    from pto_einsum import matmul_q8

    s, ws = uniform(q.shape[:-1], 5), uniform((w.shape[0],), 6)
    ref, size = ru.product(q, s, w, ws, bias)
    b = None if bias is None else bias.cuda()
    y = matmul_q8(padded(q, fill), padded(w, fill), ws.cuda(), scales=s.cuda(), bias=b, dtype=dtype)
    assert y.dtype is dtype and y.is_contiguous()
    ru.assert_within(y, ref, ru.product_bound(ref, size, dtype), f"{tuple(q.shape)} x {tuple(w.shape)}")
    return y


SIZES = [(1, 1, 1), (1, 5, 16), (2, 64, 64), (3, 17, 100), (1, 1000, 4096), (5, 129, 65), (16, 256, 2048), (17, 255, 127),
         (33, 513, 1000), (64, 1024, 512), (65, 66, 129), (100, 300, 700), (128, 128, 128), (200, 96, 5000),
         (257, 1001, 2500), (500, 2000, 192), (1024, 1024, 64), (1, 50000, 48), (3000, 7, 33),
         # weight tiles of the kernel for few rows: one, two and four, whole and not
         (7, 5000, 130), (16, 9000, 256), (20, 8200, 200), (30, 16500, 64), (64, 8200, 300), (60, 17000, 128), (64, 1000, 6000),
         # the other kernel's tiles, slabs odd and even, with and without a tail
         (70, 30000, 64), (2000, 1300, 65), (2100, 2200, 129), (4000, 300, 1000), (1000, 20000, 320), (9000, 2100, 200),
         (2048, 4096, 1024), (3001, 4100, 777), (6000, 3100, 90)]


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(m, n, k, dtype):
    check(whole((m, k), m + k), whole((n, k), n + k), dtype, fill=93)


@pytest.mark.parametrize("m,n,k", [(2, 40, 300), (70, 130, 80), (600, 900, 700)])
@pytest.mark.parametrize("dtype", ALL, ids=IDS)
def test_bias(m, n, k, dtype):
    g = torch.Generator().manual_seed(n)
    bias = torch.randn(n, generator=g) * 3
    check(whole((m, k), 1), whole((n, k), 2), dtype, bias)
    check(whole((m, k), 1), whole((n, k), 2), dtype, bias.to(dtype))


@pytest.mark.parametrize("m", [1, 16, 50, 300])
def test_largest_sums(m):
    """-128 throughout, to the last bit of 32: 128 * 128 * 131071 < 2^31."""
    k = 131071
    q = torch.full((m, k), -128, dtype=torch.int8)
    w = torch.full((20, k), -128, dtype=torch.int8)
    w[1] = 127
    w[2, 1::2] = 127
    check(q, w, torch.float32)


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 300, 1000), (4, 64, 33), (20, 500, 2048), (150, 200, 4096), (700, 900, 1283)])
def test_values_in(m, n, k, dtype):
    """Rows that the call takes to 8 bits itself."""
    from pto_einsum import matmul_q8, quantize_q8

    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, k, generator=g).to(dtype)
    w, ws = whole((n, k), 8), uniform((n,), 9)
    q, s = ru.quantize(x)
    ref, size = ru.product(q, s, w, ws, None)
    y = matmul_q8(x.cuda(), padded(w), ws.cuda())
    assert y.dtype is dtype
    ru.assert_within(y, ref, ru.product_bound(ref, size, dtype))
    for out in ALL:
        y2 = matmul_q8(x.cuda(), padded(w), ws.cuda(), dtype=out)
        qs, ss = quantize_q8(x.cuda())
        assert torch.equal(y2, matmul_q8(qs, padded(w), ws.cuda(), scales=ss, dtype=out))
    assert torch.equal(y, matmul_q8(x.cuda(), padded(w), ws.cuda(), dtype=dtype))


@pytest.mark.parametrize("m", [1, 9, 80, 400])
def test_layouts(m):
    """Contiguous odd rows, bases off 16 bytes, transposed and strided operands,
    storage that ends with the last row."""
    from pto_einsum import matmul_q8

    k, n = 203, 150
    q, w = whole((m, k), 1), whole((n, k), 2)
    s, ws = uniform((m,), 3).cuda(), uniform((n,), 4).cuda()
    want = matmul_q8(padded(q), padded(w), ws, scales=s)

    def layouts(t):
        t = t.cuda()
        yield t
        yield t.t().contiguous().t()
        off = torch.zeros(t.numel() + 5, dtype=torch.int8, device="cuda")
        off[5:] = t.flatten()
        yield off[5:].view(t.shape)
        every = torch.zeros(t.shape[0], 2 * k, dtype=torch.int8, device="cuda")
        every[:, ::2] = t
        yield every[:, ::2]
        tight = torch.zeros((t.shape[0] - 1) * 208 + k, dtype=torch.int8, device="cuda")
        view = tight.as_strided(t.shape, (208, 1))
        view.copy_(t)
        yield view
        apart = torch.full((t.shape[0], 400), 55, dtype=torch.int8, device="cuda")
        apart[:, 16:16 + k] = t
        yield apart[:, 16:16 + k]
        shifted = torch.full((t.shape[0], 400), 55, dtype=torch.int8, device="cuda")
        shifted[:, 3:3 + k] = t
        yield shifted[:, 3:3 + k]

    for a in layouts(q):
        assert torch.equal(matmul_q8(a, padded(w), ws, scales=s), want)
    for b in layouts(w):
        assert torch.equal(matmul_q8(padded(q), b, ws, scales=s), want)
    every = torch.stack([ws, ws], 1)[:, 0]
    assert torch.equal(matmul_q8(padded(q), padded(w), every, scales=torch.stack([s, s], 1)[:, 0]), want)


def test_leading_axes_and_float_strides():
    from pto_einsum import matmul_q8, quantize_q8

    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 4, 5, 100, generator=g).cuda().half()
    w, ws = padded(whole((60, 100), 1)), uniform((60,), 2).cuda()
    want = matmul_q8(x.reshape(60, 100), w, ws).reshape(3, 4, 5, 60)
    assert torch.equal(matmul_q8(x, w, ws), want)
    assert torch.equal(matmul_q8(x.transpose(0, 1), w, ws), want.transpose(0, 1))
    wide = torch.zeros(3, 4, 5, 333, dtype=torch.float16, device="cuda")
    wide[..., 7:107] = x
    assert torch.equal(matmul_q8(wide[..., 7:107], w, ws), want)
    q, s = quantize_q8(x)
    assert torch.equal(matmul_q8(q, w, ws, scales=s, dtype=torch.float16), want)
    assert torch.equal(matmul_q8(q.transpose(0, 2), w, ws, scales=s.transpose(0, 2), dtype=torch.float16),
                       want.transpose(0, 2))
    one = x[0, 0, 0]
    assert torch.equal(matmul_q8(one, w, ws), want[0, 0, 0])
    assert torch.equal(matmul_q8(one.expand(7, 100), w, ws), want[0, 0, 0].expand(7, 60))


@pytest.mark.parametrize("dtype", ALL, ids=IDS)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 7), (1, 128), (1, 130), (1, 2500), (1, 16384), (1, 16385), (2, 8192), (3, 5001),
                                 (4, 4096), (5, 4096), (7, 300), (16, 1024), (16, 1025), (16, 257), (16, 5), (9, 129)])
def test_few_rows_in_one_launch(m, k, dtype):
    """Rows that the product's own blocks take to 8 bits, and those one element past
    it: what quantize_q8 and the product of its rows give, bit for bit, halves,
    zeros and NaN among them, at any address."""
    from pto_einsum import matmul_q8, quantize_q8

    g = torch.Generator().manual_seed(k)
    wide = torch.randn(m, k + 3, generator=g).to(dtype)
    x = wide.cuda()[:, 1:k + 1]
    x[m // 2, k // 2] = 2 * x[m // 2].abs().max()
    if m > 3:
        x[0] = 0
        x[1, k - 1] = float("nan")
        x[2, 0] = float("-inf")
    for n in (33, 5000, 9000, 17000):
        w, ws = padded(whole((n, k), 8), 93), uniform((n,), 9).cuda()
        bias = uniform((n,), 4).cuda()
        q, s = quantize_q8(x)
        want = matmul_q8(q, w, ws, scales=s, bias=bias, dtype=dtype)
        got = matmul_q8(x, w, ws, bias=bias)
        assert torch.equal(torch.nan_to_num(got, nan=-3.0), torch.nan_to_num(want, nan=-3.0))
        if m > 3:
            assert torch.isnan(got[1:3]).all() and torch.isfinite(got[3:]).all()


def test_rows_with_nan_scales():
    """A row that held an infinity gives NaN throughout, and no other row does."""
    from pto_einsum import matmul_q8

    x = torch.randn(5, 300).cuda()
    x[2, 7] = float("inf")
    y = matmul_q8(x, padded(whole((40, 300), 1)), uniform((40,), 2).cuda())
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4]]).all()


def test_empty():
    from pto_einsum import matmul_q8

    ws, bias = uniform((6,), 1).cuda(), uniform((6,), 2).cuda()
    for shape in ((0, 32), (2, 0, 32)):
        y = matmul_q8(torch.zeros(shape, device="cuda"), padded(whole((6, 32), 1)), ws)
        assert y.shape == (*shape[:-1], 6)
    w0 = torch.zeros(6, 0, dtype=torch.int8, device="cuda")
    x0 = torch.zeros(4, 0, device="cuda")
    assert not matmul_q8(x0, w0, ws).any()
    assert torch.equal(matmul_q8(x0, w0, ws, bias=bias), bias.expand(4, 6))
    s0 = torch.ones(4, device="cuda")
    assert not matmul_q8(x0.to(torch.int8), w0, ws, scales=s0).any()
    assert matmul_q8(torch.zeros(4, 32, device="cuda"), torch.zeros(0, 32, dtype=torch.int8, device="cuda"), ws[:0]).shape == (4, 0)


@pytest.mark.parametrize("kernel", range(1, 9))
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (40, 70, 64), (129, 257, 65), (300, 520, 1000), (513, 300, 4096), (257, 513, 191),
                                   (70, 1000, 6001), (256, 256, 128)])
def test_every_kernel(m, n, k, kernel):
    """The kernels that sizes choose among answer alike, in each type."""
    import ctypes

    from pto_einsum import abi, launch

    q, w = padded(whole((m, k), m), 93), padded(whole((n, k), n), 93)
    s, ws = uniform((m,), 5), uniform((n,), 6)
    g = torch.Generator().manual_seed(3)
    bias = torch.randn(n, generator=g)
    ref, size = ru.product(q.cpu(), s, w.cpu(), ws, bias)
    sg, wg, bg = s.cuda(), ws.cuda(), bias.cuda()
    lib = abi.bind()
    for dtype, code in ((torch.float32, launch.DT_F32), (torch.float16, launch.DT_F16), (torch.bfloat16, launch.DT_BF16)):
        # rows of y past the last stay as they were
        out = torch.full((m + 3, n), -7.0, dtype=dtype, device="cuda")
        d = abi.Q8Desc(launch.DT_I8, code, launch.DT_F32, kernel, m, n, k, q.stride(0), w.stride(0), m * q.stride(0),
                       n * w.stride(0))
        rc = lib.pe_matmul_q8(ctypes.byref(d), q.data_ptr(), sg.data_ptr(), w.data_ptr(), wg.data_ptr(), bg.data_ptr(),
                              out.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        ru.assert_within(out[:m], ref, ru.product_bound(ref, size, dtype), f"kernel {kernel}")
        assert (out[m:] == -7.0).all()

"""scale and eps from call to call: each call has its own, and plans are kept by layouts."""
import threading

import pytest
import torch

import rows_util as ru

pytestmark = pytest.mark.gpu


def test_numbers_of_each_call():
    from pto_einsum import gated_norm, residual_norm, ssm

    g = torch.Generator().manual_seed(1)
    x, res = torch.randn(3, 200, generator=g), torch.randn(3, 200, generator=g)
    a, b = x.cuda(), res.cuda()
    residual_norm(a, b), gated_norm(a)
    before = len(ssm._plans)
    for i in list(range(300)) + [5, 5, 299, 0]:
        scale, eps = 0.01 * i - 1, 1e-6 * (i + 1)
        y_ref, r_ref, y_err, r_err = ru.residual(x, res, None, None, None, scale, eps)
        y, r = residual_norm(a, b, scale=scale, eps=eps)
        ru.assert_within(r, r_ref, ru.bound(r_ref, r_err, torch.float32), "r")
        ru.assert_within(y, y_ref, ru.bound(y_ref, y_err, torch.float32), "y")
        eps = 0.5 * i
        ref, units = ru.gated(x, None, None, eps, 1, False)
        ru.assert_within(gated_norm(a, eps=eps), ref, ru.gated_bound(ref, units, torch.float32), "gated")
    assert len(ssm._plans) == before


def test_numbers_of_threads_at_once():
    from pto_einsum import residual_norm

    g = torch.Generator().manual_seed(2)
    a, b = torch.randn(50, 300, generator=g).cuda(), torch.randn(50, 300, generator=g).cuda()
    scales = [[0.25 * (t + 1) + 4 * i for i in range(60)] for t in range(4)]
    want = {s: residual_norm(a, b, scale=s)[1].clone() for line in scales for s in line}
    torch.cuda.synchronize()
    bad = []

    def work(line):
        with torch.cuda.stream(torch.cuda.Stream()):
            for s in line * 3:
                r = residual_norm(a, b, scale=s)[1]
                torch.cuda.current_stream().synchronize()
                if not torch.equal(r, want[s]):
                    bad.append(s)

    threads = [threading.Thread(target=work, args=(line,)) for line in scales]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad

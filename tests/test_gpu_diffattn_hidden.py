"""What no query sees may hold anything and gets no gradient."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_diffattn import BF16, F32, check_all, make, no_wait_ran_out, ops, run_all  # noqa: E402,F401

pytestmark = pytest.mark.gpu

SHAPES = [(2, 20, 45, 2, 1, 16), (2, 1, 90, 2, 1, 16), (2, 3, 777, 8, 2, 40), (2, 80, 200, 4, 2, 32), (1, 200, 1000, 2, 2, 64),
          (2, 130, 300, 2, 1, 24), (2, 100, 200, 2, 2, 33)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", SHAPES)
def test_keys_after_the_last_query(ops, n, tq, tk, h, hkv, dh, dtype):
    """causal="start" over more keys than queries: the keys from tq on."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, dtype, 13)
    k[:, tq:], v[:, tq:] = math.nan, math.inf
    check_all(ops, q, k, v, lam, dout, causal="start")
    klen = torch.tensor([tk - 1, max(1, tq // 2)][:n], dtype=torch.int32, device="cuda")
    check_all(ops, q, k, v, lam, dout, causal="start", klen=klen)
    _, _, _, _, dk, dv, _ = run_all(ops, q, k, v, lam, dout, causal="start")
    assert not bool(dk[:, tq:].any()) and not bool(dv[:, tq:].any())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", SHAPES)
def test_gradient_of_hidden_keys_where_a_query_is_not_a_number(ops, n, tq, tk, h, hkv, dh, dtype):
    """NaN in a query or in its output's gradient reaches the keys that lengths and masks leave, and no other."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, dtype, 14)
    klen = torch.tensor([tk, tk // 2 + 1][:n], dtype=torch.int32, device="cuda")
    kmask = torch.rand(n, tk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) < 0.7
    kmask[:, 0] = True
    hidden = (torch.arange(tk, device="cuda")[None] >= klen[:, None]) | ~kmask
    for x in (q, dout):
        keep = x[0, tq // 2].clone()
        x[0, tq // 2] = math.nan
        for how in (dict(klen=klen, kmask=kmask), dict(klen=klen)):
            gone = hidden if "kmask" in how else torch.arange(tk, device="cuda")[None] >= klen[:, None]
            _, _, _, dq, dk, dv, _ = run_all(ops, q, k, v, lam, dout, **how)
            assert bool(torch.isnan(dk[0][~gone[0]]).all()) and bool(torch.isnan(dv[0][~gone[0]]).all())
            assert not bool(dk[gone].any()) and not bool(dv[gone].any())
            rest = torch.arange(tq, device="cuda") != tq // 2
            assert bool(torch.isfinite(dq[0, rest]).all()) and bool(torch.isnan(dq[0, tq // 2]).all())
            if n > 1:
                assert bool(torch.isfinite(dk[1]).all()) and bool(torch.isfinite(dv[1]).all())
        x[0, tq // 2] = keep

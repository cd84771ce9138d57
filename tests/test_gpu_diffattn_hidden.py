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

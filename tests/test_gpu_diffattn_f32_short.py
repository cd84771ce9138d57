"""f32 calls that stay on the warp-level matrix products keep f32's precision.

A score is a chain of dh / 8 <= 8 products, each of which cuts off up to 2^-23 of
the sum, half of that on the average: 8 * 2^-24 = 4.8e-7.  An output passes one
such sum after the scores' exponentials (5e-7), a gradient two (1e-6)."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_diffattn import F32, make, no_wait_ran_out, ops, reference, rel, run_all  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", [(16, 48, 48, 4, 4, 64), (64, 60, 60, 4, 4, 64), (8, 50, 50, 4, 2, 33),
                                              (128, 64, 64, 4, 4, 32), (64, 30, 60, 4, 4, 16)])
def test_short_sequences(ops, n, tq, tk, h, hkv, dh):
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, F32, 5)
    want = reference(q, k, v, lam, dout, dh ** -0.5)
    o, o2, _, dq, dk, dv, _ = run_all(ops, q, k, v, lam, dout)
    assert rel(o, want[0]) < 5e-7 and rel(o2, want[1]) < 5e-7
    for x, y in zip((dq, dk, dv), want[2:5]):
        assert rel(x, y) < 1e-6


@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", [(4, 1, 5000, 8, 2, 64), (2, 3, 2000, 4, 4, 64), (8, 1, 777, 4, 4, 32)])
def test_tokens_over_a_cache(ops, n, tq, tk, h, hkv, dh):
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, F32, 6)
    want = reference(q, k, v, lam, dout, dh ** -0.5)[0]
    assert rel(ops.diffattn_forward(q, k, v, lam), want) < 5e-7

"""What a query sees decides its result: NaN and infinities that are visible come
out as NaN, in every kernel that a call's size may choose, and what no query
sees may hold anything."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_diffattn import BF16, F32, TOL, check_all, make, no_wait_ran_out, ops, rel, run_all  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# one of each way through the kernels: short calls, tokens over a cache (whole and in parts), many tiles, few rows
# whose keys are split, halves of more than 32 columns, odd widths
ROUTES = [
    (2, 20, 45, 2, 1, 16),
    (2, 1, 90, 2, 1, 16),
    (2, 1, 3000, 4, 1, 64),
    (2, 3, 777, 8, 2, 40),
    (2, 200, 300, 4, 2, 32),
    (2, 256, 190, 2, 2, 64),
    (2, 130, 3000, 2, 1, 24),
    (2, 100, 200, 2, 2, 33),
]


def finite(*ts):
    return all(bool(torch.isfinite(t).all()) for t in ts)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", ROUTES)
def test_query_that_is_not_a_number(ops, n, tq, tk, h, hkv, dh, half, bad, dtype):
    """One element of one query: its map, output and gradients are NaN, those of the others are what they were."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, dtype, 7)
    clean = run_all(ops, q, k, v, lam, dout)
    at = (1, tq // 2, h - 1)
    q[at][half * dh + dh // 2] = bad
    o, o2, lse, dq, dk, dv, dlam = run_all(ops, q, k, v, lam, dout)
    assert bool(torch.isnan(o[at]).all()) and bool(torch.isnan(dq[at][half * dh:(half + 1) * dh]).all())
    assert bool(torch.isnan(o2[at]).all()) if half else finite(o2[at])
    assert bool(torch.isnan(lse[1, h - 1, half, tq // 2])) and finite(lse[1, h - 1, 1 - half, tq // 2])
    # dlam sums P_2 dP over the head's rows
    assert bool(torch.isnan(dlam[h - 1])) if half else finite(dlam)
    assert finite(dlam[:h - 1])
    assert bool(torch.isnan(dk[1, :, hkv - 1, half * dh:(half + 1) * dh]).all()) and bool(torch.isnan(dv[1, :, hkv - 1]).all())
    rest = torch.ones(n, tq, h, dtype=torch.bool, device="cuda")
    rest[at] = False
    for got, want in ((o, clean[0]), (o2, clean[1]), (dq, clean[3])):
        if bool(rest.any()):
            assert rel(got[rest], want[rest].double()) < 2 * TOL[dtype]
    assert finite(dk[0], dv[0], lse[0])
    # without the saved tensors the same
    assert torch.equal(torch.isnan(ops.diffattn_forward(q, k, v, lam)), torch.isnan(o))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", ROUTES)
def test_key_that_is_not_a_number(ops, n, tq, tk, h, hkv, dh, half, dtype):
    """One element of a visible key: every query of its group that sees it is NaN; a query that does not is not."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, dtype, 8)
    last = tk - 1
    k[1, last, 0, half * dh] = math.nan
    grp = h // hkv
    # the last query alone sees the last key
    o, o2, lse, dq, _, _, dlam = run_all(ops, q, k, v, lam, dout, causal="end")
    assert bool(torch.isnan(o[1, -1, :grp]).all()) and bool(torch.isnan(lse[1, :grp, half, -1]).all())
    assert finite(o[0], o[1, :-1], o[1, -1, grp:], dq[0])
    assert not bool(torch.isnan(lse[0]).any()) and not bool(torch.isnan(lse[1, :, :, :-1]).any())
    assert finite(o2[1, -1]) if half == 0 else bool(torch.isnan(o2[1, -1, :grp]).all())
    assert finite(dlam) if half == 0 else bool(torch.isnan(dlam[:grp]).all())
    # all do
    o, o2, lse, dq, _, _, dlam = run_all(ops, q, k, v, lam, dout)
    assert bool(torch.isnan(o[1, :, :grp]).all()) and bool(torch.isnan(lse[1, :grp, half]).all())
    assert bool(torch.isnan(dq[1, :, :grp, half * dh:(half + 1) * dh]).all())
    assert finite(o[0], o[1, :, grp:], lse[0], dq[0])


@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", ROUTES)
def test_scores_of_minus_infinity_alone(ops, n, tq, tk, h, hkv, dh):
    """Finite queries and keys whose scores in one map all overflow to -inf: that map is 0, the other what it was.
    (bf16 only: f32 operands are multiplied in parts of either sign, whose overflow is inf - inf.)"""
    q, k, v, lam, _ = make(n, tq, tk, h, hkv, dh, BF16, 9)
    for half in (0, 1):
        q2, k2 = q.clone(), k.clone()
        cols = slice(half * dh, (half + 1) * dh)
        q2[..., cols], k2[..., cols] = 1e25, -1e25
        o, o2, lse = ops.diffattn_forward(q2, k2, v, lam, save=True)
        grp = h // hkv
        other = slice((1 - half) * dh, (2 - half) * dh)
        s = torch.einsum("nihc,njhc->nhij", q[..., other].double(), k[..., other].double().repeat_interleave(grp, 2))
        p = torch.einsum("nhij,njhc->nihc", torch.softmax(s * dh ** -0.5, -1), v.double().repeat_interleave(grp, 2))
        assert rel(o, p if half else -lam.double()[:, None] * p) < TOL[BF16]
        assert not bool(o2.any()) if half else rel(o2, p) < TOL[BF16]
        assert bool((lse[:, :, half] == math.inf).all()) and finite(lse[:, :, 1 - half])

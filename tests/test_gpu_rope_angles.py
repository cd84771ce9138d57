"""Rotary angles at far positions and high frequencies, against integer arithmetic, and the largest row counts."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# 1 / (2 pi) to 200 bits, from pi to 70 digits
_PI = 31415926535897932384626433832795028841971693993751058209749445923078164
_INV_TURN = (10 ** 70 << 199) // _PI


def turns(pos, freq):
    """pos * freq / (2 pi) less its whole turns, exact to 2^-90: freq's 24 bits times an integer, in integers."""
    m, e = math.frexp(freq)
    whole = pos * int(m * (1 << 24)) * _INV_TURN  # at 2^(200 + 24 - e)
    one = 1 << (224 - e)
    return (whole % one) / one


@pytest.mark.parametrize("low,high", [(0, 4096), (-(1 << 20), 1 << 20), (-(1 << 31), (1 << 31) - 1)])
@pytest.mark.parametrize("inter", [False, True])
def test_angles_are_exact(low, high, inter):
    """Every product of a position and a frequency, from 2^-20 to 2^10 radians a step: cos and sin to the same 2^-21 of
    the pair's length as at small angles."""
    from rustnn_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(3)
    rows, count = 48, 31
    freq = torch.exp2(torch.linspace(-20, 10, count, device="cuda")) * 1.3333334
    pos = torch.randint(low, high, (rows, 1), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    pos[0], pos[1] = low, high - 1
    x = torch.zeros(rows, 1, 2 * count, device="cuda")
    first = x[..., 0::2] if inter else x[..., :count]
    first.fill_(1.0)
    y = ops.rope(x, pos, freq, (count,), interleaved=inter)
    a = torch.tensor([[turns(p, f) for f in freq.tolist()] for p in pos[:, 0].tolist()], dtype=torch.float64,
                     device="cuda") * (2 * math.pi)
    c, s = (y[:, 0, 0::2], y[:, 0, 1::2]) if inter else (y[:, 0, :count], y[:, 0, count:])
    assert float((c.double() - torch.cos(a)).abs().max()) < 2.0 ** -21
    assert float((s.double() - torch.sin(a)).abs().max()) < 2.0 ** -21


def test_most_rows():
    """2^31 - 1 rows of two columns: the launch counts its blocks without passing int."""
    from rustnn_b200 import ops

    rows = (1 << 31) - 1
    pos = torch.zeros(rows, 1, device="cuda", dtype=torch.int32)
    pos[-1] = 1
    x = torch.ones(rows, 1, 2, device="cuda", dtype=torch.bfloat16)
    y = ops.rope(x, pos, torch.ones(1, device="cuda"), (1,), out=x)
    assert y is x and bool((y[:4] == 1).all())
    want = torch.tensor([math.cos(1) - math.sin(1), math.cos(1) + math.sin(1)], device="cuda").bfloat16()
    assert torch.equal(y[-1, 0], want)
    torch.cuda.synchronize()
    del x, y, pos
    torch.cuda.empty_cache()

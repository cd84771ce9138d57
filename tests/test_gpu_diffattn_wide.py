"""Shapes whose kernels had no test of their own: f32 halves of 33 to 64 columns
over tiles with masks, lengths and addresses that allow no wide loads, and a
bf16 call of several waves of blocks against the formula."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_diffattn import BF16, F32, TOL, check_all, make, no_wait_ran_out, ops, reference, rel  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", [(2, 200, 300, 2, 1, 64), (3, 130, 257, 2, 2, 40), (2, 128, 200, 2, 1, 33),
                                              (1, 100, 1000, 4, 2, 47), (2, 64, 130, 2, 2, 64)])
def test_f32_wide_halves_over_tiles(ops, n, tq, tk, h, hkv, dh, causal, shift):
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, F32, 33)

    def moved(x):  # the same values at an address that allows no wide loads
        return torch.zeros(x.numel() + shift, device="cuda")[shift:].view(x.shape).copy_(x)

    q, k, v, dout = (moved(x) for x in (q, k, v, dout))
    check_all(ops, q, k, v, lam, dout, causal=causal)
    klen = torch.tensor([tk - 3, 0, 64][:n], dtype=torch.int32, device="cuda")
    kmask = torch.rand(n, tk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) < 0.7
    for mask, length in ((kmask, klen), (kmask, None), (None, klen)):
        hidden = torch.zeros(n, tk, dtype=torch.bool, device="cuda")
        if mask is not None:
            hidden |= ~mask
        if length is not None:
            hidden |= torch.arange(tk, device="cuda")[None] >= length[:, None]
        k2, v2 = moved(k), moved(v)
        k2.masked_fill_(hidden[:, :, None, None], math.nan)
        v2.masked_fill_(hidden[:, :, None, None], math.inf)
        check_all(ops, q, k2, v2, lam, dout, causal=causal, klen=length, kmask=mask)


def test_several_waves_of_blocks(ops):
    """640 blocks of 128 queries, each head's rows against the formula in 64 bits."""
    q, k, v, lam, dout = make(2, 2500, 2500, 16, 8, 64, BF16, 12)
    o, o2, _ = ops.diffattn_forward(q, k, v, lam, causal="start", save=True)
    for b in range(2):
        for e in range(16):
            at = (slice(b, b + 1), slice(None), slice(e, e + 1))
            kv = (slice(b, b + 1), slice(None), slice(e // 2, e // 2 + 1))
            want = reference(q[at], k[kv], v[kv], lam[e:e + 1], dout[at], 64 ** -0.5, "start")
            assert rel(o[at], want[0]) < TOL[BF16] and rel(o2[at], want[1]) < TOL[BF16]
            # early rows see few keys and late ones many; none is lost among the others
            row = (o[at].double() - want[0]).norm(dim=-1) / want[0].norm(dim=-1)
            assert float(row.max()) < 2.0 ** -6

"""Gradients in bf16 row by row, where single keys hold nearly all of a row or
keys and values have much in common, against the formulas in 64 bits.

Bound of a row of dq, map m (f_1 = 1, f_2 = -lam; u = 2^-8 the rounding of
bf16): dq_m = scale f_m sum_j dS_j k_j, so
  (a) each dS_j is rounded once:  scale |f| u sum_j |dS_j| |k_j|,
  (b) D may be off by 1/64 of the norm of the row's dS (a bit over, since the
      kernel measures that norm with the D it has):
      scale |f| 2^-6 (1 + 2^-5) |dS| |sum_j P_j k_j|,
  (c) scores of up to 2^5 in base 2, rounded about six times in f32, move P by
      2^-17 of itself, and dP - D by twice that of |do| max |v|:
      scale |f| 2^-15 |do| max_j |v_j| sum_j P_j |k_j|,
  (d) the result is rounded: u |dq|.
Rows of dk: (a) and (c) summed over the queries, and (d); the keys' kernel has D
from f32 sums, which (c) covers."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_diffattn import BF16, make, no_wait_ran_out, ops, run_all, visible  # noqa: E402,F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def check_rows(ops, q, k, v, lam, dout, scale, **how):
    n, tq, h, w = q.shape
    tk, hkv, dh = k.shape[1], k.shape[2], w // 2
    grp = h // hkv
    see = visible(n, tq, tk, how.get("causal"), how.get("klen"), how.get("kmask"))[:, None]
    gone = ~see.any(2)[:, 0]
    _, _, _, dq, dk, _, _ = run_all(ops, q, k, v, lam, dout, scale=scale, **how)
    Q, G = q.double().transpose(1, 2), dout.double().transpose(1, 2)
    K, V = (x.double().masked_fill(gone[:, :, None, None], 0.0).repeat_interleave(grp, 2).transpose(1, 2) for x in (k, v))
    dP = G @ V.transpose(-1, -2)
    size = G.norm(dim=-1)[..., None] * V.norm(dim=-1).amax(-1)[..., None, None]  # |do| max |v|, [n, h, tq, 1]
    for m in range(2):
        c = slice(m * dh, (m + 1) * dh)
        f = torch.ones(1, h, 1, 1, dtype=torch.float64, device="cuda") if m == 0 else -lam.double().view(1, h, 1, 1)
        s = (Q[..., c] @ K[..., c].transpose(-1, -2) * scale).masked_fill(~see, -torch.inf)
        P = torch.softmax(s.masked_fill(~see.any(-1, keepdim=True), 0.0), -1) * see
        dS = P * (dP - (P * dP).sum(-1, keepdim=True))
        kn, qn = K[..., c].norm(dim=-1), Q[..., c].norm(dim=-1)
        want = scale * f * (dS @ K[..., c])
        bound = scale * f.abs() * (U * (dS.abs() @ kn[..., None]) + 2.0 ** -15 * size * (P @ kn[..., None])
                                   + 2.0 ** -6 * (1 + 2.0 ** -5) * dS.norm(dim=-1, keepdim=True)
                                   * (P @ K[..., c]).norm(dim=-1, keepdim=True))
        bound = abs(bound) + U * want.norm(dim=-1, keepdim=True) + 1e-30
        err = (dq.double().transpose(1, 2)[..., c] - want).norm(dim=-1, keepdim=True)
        assert float((err / bound).max()) <= 1.0, ("dq", m, float((err / bound).max()))
        fold = lambda x: x.view(n, hkv, grp, *x.shape[2:]).sum(2)  # noqa: E731
        want = fold(scale * f * (dS.transpose(-1, -2) @ Q[..., c]))
        bound = fold(abs(scale) * f.abs() * (U * dS.abs() + 2.0 ** -15 * size * P).transpose(-1, -2) @ qn[..., None])
        bound = bound + U * want.norm(dim=-1, keepdim=True) + 1e-30
        err = (dk.double().transpose(1, 2)[..., c] - want).norm(dim=-1, keepdim=True)
        assert float((err / bound).max()) <= 1.0, ("dk", m, float((err / bound).max()))


SHAPES = [(2, 409, 409, 3, 3, 56), (1, 1024, 1024, 2, 2, 32), (2, 300, 700, 4, 2, 64), (3, 100, 210, 2, 1, 8), (1, 40, 2000, 4, 1, 64),
          (2, 300, 300, 2, 1, 33), (2, 60, 190, 2, 2, 16)]


@pytest.mark.parametrize("scale", [0.3, 0.6, 1.0, -0.6])
@pytest.mark.parametrize("causal", [None, "end"])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", SHAPES)
def test_sharp_rows(ops, n, tq, tk, h, hkv, dh, causal, scale):
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, BF16, 12)
    check_rows(ops, q, k, v, lam, dout, scale, causal=causal)


@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", SHAPES)
def test_sharp_rows_of_masked_keys(ops, n, tq, tk, h, hkv, dh):
    """Few and many keys left by masks and lengths, what is hidden not a number."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, BF16, 15)
    kmask = torch.rand(n, tk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) < 0.5
    kmask[0, tk // 3] = True
    klen = torch.tensor([tk, tk // 2 + 3, 70][:n], dtype=torch.int32, device="cuda")
    for mask, length in ((kmask, None), (None, klen), (kmask, klen)):
        hide = torch.zeros(n, tk, dtype=torch.bool, device="cuda")
        if mask is not None:
            hide |= ~mask
        if length is not None:
            hide |= torch.arange(tk, device="cuda")[None] >= length[:, None]
        k2, v2 = (x.masked_fill(hide[:, :, None, None], torch.nan) for x in (k, v))
        for scale in (0.2, 0.8):
            check_rows(ops, q, k2, v2, lam, dout, scale, kmask=mask, klen=length)
            check_rows(ops, q, k2, v2, lam, dout, scale, kmask=mask, klen=length, causal="start")


@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", SHAPES)
def test_keys_and_values_with_much_in_common(ops, n, tq, tk, h, hkv, dh):
    """sum dS k leaves out what all keys share, and dP - D what all values share."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, BF16, 16)
    check_rows(ops, q, (k.float() + 3).bfloat16(), (v.float() + 4).bfloat16(), lam, dout, dh ** -0.5 / 4)


def test_one_visible_key_of_many(ops):
    """A lone key has P = 1 and dS = 0: what is left of dq and dk, row by row, is the rounding of P dP - D in f32, far
    below what a D of rounded outputs would leave."""
    for n, tq, tk, h, hkv, dh in SHAPES:
        q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, BF16, 17)
        kmask = torch.zeros(n, tk, dtype=torch.bool, device="cuda")
        at = 2 * tk // 3
        kmask[:, at] = True
        _, _, _, dq, dk, _, _ = run_all(ops, q, k, v, lam, dout, kmask=kmask)
        size = dout.double().norm(dim=-1) * v[:, at].double().norm(dim=-1).repeat_interleave(h // hkv, 1)[:, None]
        kn = k[:, at].double().norm(dim=-1).repeat_interleave(h // hkv, 1)[:, None]
        # P within 2^-18 of 1 (scores below 2^4), dP of up to 128 products summed in f32: 2^-17 of |do| |v| together
        assert bool((dq.double().norm(dim=-1) <= 2.0 ** -17 * dh ** -0.5 * size * kn + 1e-30).all()), (n, tq, tk)
        qn = q.double().norm(dim=-1)
        bound = (2.0 ** -17 * dh ** -0.5 * size * qn).view(n, tq, hkv, h // hkv).sum((1, 3))
        assert bool((dk[:, at].double().norm(dim=-1) <= bound + 1e-30).all()), (n, tq, tk)

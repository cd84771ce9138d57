"""GPU parity of differential attention, forward and backward, against the
definition in 64 bits (autograd of the plain formula), on the inputs as the
kernels get them.

Bounds (relative Frobenius per output).  f32: scores come from split-TF32
products (2^-22) of magnitude up to about 8 in base 2, so a map entry is off by
at most about 2^-20; subtracting the maps at most triples that: 1e-5.  bf16:
rounding to 8 bits leaves a relative error of at most 2^-8, 2^-8 / sqrt(3) =
2.3e-3 in the mean square; the combined map and the output are each rounded
once, 3.2e-3 together; the gradients read D from saved outputs that were
rounded once more: 5e-3.  dlam is summed in
f32 either way: 4e-6 of the sum of the magnitudes of its terms."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 5e-3}
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from rustnn_b200 import ops as _ops

    return _ops


@pytest.fixture(autouse=True)
def no_wait_ran_out(ops):
    yield
    ops.default_context(0).synchronize()  # raises what a kernel has recorded


def visible(n, tq, tk, causal, klen, kmask):
    i, j = torch.arange(tq, device="cuda")[:, None], torch.arange(tk, device="cuda")[None]
    length = (klen.long().clamp(0, tk) if klen is not None else torch.full((n,), tk, device="cuda"))[:, None, None]
    see = (j < length).expand(n, tq, tk)
    if causal == "start":
        see = see & (j <= i)
    elif causal == "end":
        see = see & (j <= i + length - tq)
    if kmask is not None:
        see = see & kmask.bool()[:, None]
    return see


def reference(q, k, v, lam, dout, scale, causal=None, klen=None, kmask=None):
    """o, P_2 v, dq, dk, dv, dlam and the magnitude of dlam's terms, in 64 bits."""
    n, tq, h, w = q.shape
    tk, hkv, dh = k.shape[1], k.shape[2], q.shape[3] // 2
    see = visible(n, tq, tk, causal, klen, kmask)[:, None]
    hidden = torch.zeros(n, tk, dtype=torch.bool, device="cuda") if tk == 0 else ~see.any(2)[:, 0]
    # what no query sees may hold anything
    k = k.double().masked_fill(hidden[:, :, None, None], 0.0)
    v = v.double().masked_fill(hidden[:, :, None, None], 0.0)
    q, lam = q.double().requires_grad_(), lam.double().requires_grad_()
    k, v = k.requires_grad_(), v.requires_grad_()
    rep = h // hkv
    kk, vv = k.repeat_interleave(rep, 2).transpose(1, 2), v.repeat_interleave(rep, 2).transpose(1, 2)
    qq = q.transpose(1, 2)
    some = see.any(-1, keepdim=True) if tk else torch.zeros(n, 1, tq, 1, dtype=torch.bool, device="cuda")
    bias = torch.zeros(see.shape, dtype=torch.float64, device="cuda").masked_fill(~see & some, -math.inf)
    maps = [torch.softmax(qq[..., c] @ kk[..., c].transpose(-1, -2) * scale + bias, -1) * some
            for c in (slice(0, dh), slice(dh, w))]
    o2 = maps[1] @ vv
    o = maps[0] @ vv - lam.view(1, h, 1, 1) * o2
    grads = torch.autograd.grad(o, (q, k, v, lam), dout.double().transpose(1, 2), allow_unused=True)
    grads = [torch.zeros_like(t) if g is None else g for g, t in zip(grads, (q, k, v, lam))]
    dp = dout.double().transpose(1, 2) @ vv.transpose(-1, -2)
    size = (maps[1] * dp.abs()).sum((0, 2, 3)).detach()
    return [x.detach() for x in (o.transpose(1, 2), o2.transpose(1, 2), *grads, size)]


def make(n, tq, tk, h, hkv, dh, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, device="cuda", generator=g).to(dtype)

    lam = 0.2 + 0.6 * torch.rand(h, device="cuda", generator=g)
    return r(n, tq, h, 2 * dh), r(n, tk, hkv, 2 * dh), r(n, tk, hkv, 2 * dh), lam, r(n, tq, h, 2 * dh)


def rel(got, want):
    d, s = float((got.double() - want).norm()), float(want.norm())
    return d / s if s > 0 else d


def run_all(ops, q, k, v, lam, dout, **how):
    o, o2, lse = ops.diffattn_forward(q, k, v, lam, save=True, **how)
    dlam = torch.zeros_like(lam)
    dq, dk, dv = ops.diffattn_backward(dout, q, k, v, lam, o, o2, lse, dlam, **how)
    return o, o2, lse, dq, dk, dv, dlam


def check_all(ops, q, k, v, lam, dout, **how):
    scale = how.get("scale") or (q.shape[-1] // 2) ** -0.5
    want = reference(q, k, v, lam, dout, scale, how.get("causal"), how.get("klen"), how.get("kmask"))
    o, o2, lse, dq, dk, dv, dlam = run_all(ops, q, k, v, lam, dout, **how)
    # without the saved tensors the result is the same
    assert torch.equal(ops.diffattn_forward(q, k, v, lam, **how), o)
    tol = TOL[q.dtype]
    for name, got, ref in zip(("o", "o2", "dq", "dk", "dv"), (o, o2, dq, dk, dv), want):
        assert got.dtype == q.dtype
        assert rel(got, ref) < tol, (name, rel(got, ref))
    assert bool(((dlam.double() - want[5]).abs() <= 4e-6 * want[6] + 1e-30).all())
    return o, lse


SHAPES = [
    # n, tq, tk, h, hkv, dh: one token up to several tiles, around the tile sizes, odd widths, shared key heads
    (1, 1, 1, 1, 1, 8),
    (2, 1, 5, 2, 1, 16),
    (3, 7, 3, 2, 2, 4),
    (2, 16, 16, 4, 2, 8),
    (1, 31, 33, 1, 1, 32),
    (2, 64, 64, 4, 4, 32),
    (2, 65, 63, 3, 1, 24),
    (1, 128, 129, 2, 2, 64),
    (2, 100, 257, 6, 2, 40),
    (1, 300, 300, 2, 1, 64),
    (2, 50, 70, 2, 2, 1),
    (2, 50, 70, 2, 2, 5),
    (1, 77, 90, 3, 3, 33),
    (1, 33, 1000, 8, 2, 64),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", SHAPES)
def test_parity(ops, n, tq, tk, h, hkv, dh, causal, dtype):
    check_all(ops, *make(n, tq, tk, h, hkv, dh, dtype, tq + tk + dh), causal=causal)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("tq,tk", [(80, 200), (129, 129), (300, 90), (3, 500)])
def test_lengths_and_masks_with_anything_hidden(ops, tq, tk, causal, dtype):
    """Lengths from 0 to beyond tk, key masks that hide a whole sequence, and
    NaN, infinities and the type's lowest value in every hidden key and value:
    rows that see nothing are 0 with no gradient."""
    n, h, hkv, dh = 6, 4, 2, 32
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, dtype, 11)
    klen = torch.tensor([0, 1, tk // 2, tk, tk - 1, tk + 7], dtype=torch.int32, device="cuda")
    kmask = torch.rand(n, tk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.7
    kmask[3] = False
    kmask[1, 0] = True
    see = visible(n, tq, tk, causal, klen, kmask)
    hidden = ~((torch.arange(tk, device="cuda")[None] < klen[:, None]) & kmask)
    for i, bad in enumerate((math.nan, math.inf, -math.inf, torch.finfo(dtype).min)):
        at = hidden & (torch.arange(tk, device="cuda")[None] % 4 == i)
        k.masked_fill_(at[:, :, None, None], bad)
        v.masked_fill_(at[:, :, None, None], bad)
    how = dict(causal=causal, klen=klen, kmask=kmask)
    o, lse = check_all(ops, q, k, v, lam, dout, **how)
    none = ~see.any(-1)
    assert bool((o[none] == 0).all())
    assert bool(torch.isposinf(lse.permute(0, 3, 1, 2)[none]).all())
    assert bool(torch.isfinite(lse.permute(0, 3, 1, 2)[~none]).all())
    _, _, _, dq, dk, dv, _ = run_all(ops, q, k, v, lam, dout, **how)
    assert bool((dq[none] == 0).all())
    assert bool((dk[hidden] == 0).all()) and bool((dv[hidden] == 0).all())
    # the same by a byte mask with the length written into it
    both = ((torch.arange(tk, device="cuda")[None] < klen[:, None]) & kmask).to(torch.uint8) * 3
    if causal != "end":
        assert torch.equal(ops.diffattn_forward(q, k, v, lam, causal=causal, kmask=both), o)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("tq,tk,h,hkv,dh", [(700, 700, 2, 1, 40), (130, 1000, 2, 2, 64), (300, 700, 1, 1, 16)])
def test_ragged_lengths_over_many_tiles(ops, tq, tk, h, hkv, dh, causal, dtype):
    """Lengths that end anywhere in any of many key tiles; what lies beyond them is NaN or infinite."""
    lens = [0, 1, 63, 64, 65, 127, 130, 300, 449, 511, 577, 640, 699, tk]
    q, k, v, lam, dout = make(len(lens), tq, tk, h, hkv, dh, dtype, 17)
    klen = torch.tensor(lens, dtype=torch.int32, device="cuda")
    hidden = torch.arange(tk, device="cuda")[None] >= klen[:, None]
    k.masked_fill_(hidden[:, :, None, None], math.nan)
    v.masked_fill_(hidden[:, :, None, None], math.inf)
    check_all(ops, q, k, v, lam, dout, causal=causal, klen=klen)
    # and each sequence by itself, whose rows outweigh none
    want = reference(q, k, v, lam, dout, dh ** -0.5, causal, klen)
    got = run_all(ops, q, k, v, lam, dout, causal=causal, klen=klen)
    for b in range(len(lens)):
        for x, y in zip((got[0], got[3], got[4], got[5]), (want[0], want[2], want[3], want[4])):
            assert rel(x[b], y[b]) < 2 * TOL[dtype] or lens[b] <= 1, (lens[b], rel(x[b], y[b]))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_single_key_has_no_score_gradient(ops, dtype):
    """One visible key: the maps are 1, o = (1 - lam) v, dq and dk are exactly 0."""
    q, k, v, lam, dout = make(3, 5, 9, 2, 2, 16, dtype, 4)
    klen = torch.ones(3, dtype=torch.int32, device="cuda")
    _, _, _, dq, dk, _, _ = run_all(ops, q, k, v, lam, dout, klen=klen)
    assert bool((dq == 0).all()) and bool((dk == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", [(2, 1, 4097, 4, 1, 64), (1, 1, 20000, 2, 2, 32), (3, 2, 3001, 8, 1, 64),
                                              (1, 5, 9000, 3, 1, 16), (2, 16, 2500, 1, 1, 40), (1, 40, 7000, 2, 2, 64)])
def test_few_rows_over_a_long_cache(ops, n, tq, tk, h, hkv, dh, dtype):
    """New tokens against a cache: the keys are split over blocks and joined."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, dtype, tk)
    check_all(ops, q, k, v, lam, dout, causal="end")
    klen = torch.randint(1, tk, (n,), dtype=torch.int32, device="cuda",
                         generator=torch.Generator(device="cuda").manual_seed(2))
    klen[0] = 3
    check_all(ops, q, k, v, lam, dout, causal="end", klen=klen)


@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", [(1, 70, 3000, 2, 1, 40), (3, 20, 1500, 2, 2, 64), (2, 200, 5001, 4, 2, 16),
                                              (1, 129, 1025, 3, 1, 32)])
def test_new_rows_over_a_long_cache(ops, n, tq, tk, h, hkv, dh, causal):
    """A run of new tokens against a cache: rows fill tiles but not the device, so the keys are split over blocks.
    What lies beyond the lengths is NaN; some parts, and the rows of one sequence, have no keys."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, BF16, tk)
    check_all(ops, q, k, v, lam, dout, causal=causal)
    for first in (tk - 1, tk // 2 + 1, 130, 64, 1, 0):
        klen = torch.tensor([first, tk, 65][:n], dtype=torch.int32, device="cuda")
        hidden = torch.arange(tk, device="cuda")[None] >= klen[:, None]
        k2, v2 = k.clone(), v.clone()
        k2.masked_fill_(hidden[:, :, None, None], math.nan)
        v2.masked_fill_(hidden[:, :, None, None], -math.inf)
        o, lse = check_all(ops, q, k2, v2, lam, dout, causal=causal, klen=klen)
        if first == 0:
            assert bool((o[0] == 0).all()) and bool((lse[0] == math.inf).all())
        # any alignment of the output's rows
        at = torch.full((n, tq, h * 2 * dh + 3), 7.0, device="cuda", dtype=BF16)
        out = at[..., 1:1 + h * 2 * dh].unflatten(-1, (h, 2 * dh))
        assert torch.equal(ops.diffattn_forward(q, k2, v2, lam, causal=causal, klen=klen, out=out), o)
        assert bool((at[..., 0] == 7).all()) and bool((at[..., -2:] == 7).all())


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("n,tq,tk,h,hkv,dh", [(2, 128, 128, 2, 2, 32), (3, 130, 257, 2, 1, 32), (2, 70, 1000, 2, 2, 7),
                                              (1, 33, 2000, 4, 1, 20), (2, 500, 65, 2, 2, 12)])
def test_f32_over_tiles(ops, n, tq, tk, h, hkv, dh, causal, shift):
    """f32 calls of several tiles: any width and alignment, lengths and masked keys with anything in them, rows packed
    across heads, keys split over blocks."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, F32, 31)

    def moved(x):  # the same values at an address that allows no wide loads
        return torch.zeros(x.numel() + shift, device="cuda")[shift:].view(x.shape).copy_(x)

    q, k, v, dout = (moved(x) for x in (q, k, v, dout))
    check_all(ops, q, k, v, lam, dout, causal=causal)
    klen = torch.tensor([tk - 3, 0, 64][:n], dtype=torch.int32, device="cuda")
    kmask = torch.rand(n, tk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) < 0.7
    hidden = (torch.arange(tk, device="cuda")[None] >= klen[:, None]) | ~kmask
    k.masked_fill_(hidden[:, :, None, None], math.nan)
    v.masked_fill_(hidden[:, :, None, None], math.inf)
    check_all(ops, q, k, v, lam, dout, causal=causal, klen=klen, kmask=kmask)


def test_f32_keeps_its_precision(ops):
    """Products of three bf16 planes leave 2^-24: far below what a product of fewer parts would."""
    q, k, v, lam, dout = make(2, 256, 300, 2, 2, 32, F32, 3)
    want = reference(q, k, v, lam, dout, 32 ** -0.5)
    got = run_all(ops, q, k, v, lam, dout)
    # 300 terms added in f32: 2^-24 sqrt(300) / 2 = 5e-7; gradients pass two such sums
    assert rel(got[0], want[0]) < 5e-7 and rel(got[1], want[1]) < 5e-7
    for x, y in zip(got[3:6], want[2:5]):
        assert rel(x, y) < 1e-6


@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("tq,tk,h,hkv,dh", [(300, 700, 2, 1, 40), (130, 1000, 2, 2, 64), (700, 700, 2, 2, 32),
                                            (70, 90, 2, 1, 24), (200, 200, 2, 2, 5)])
def test_masked_keys_over_many_tiles(ops, tq, tk, h, hkv, dh, causal):
    """bf16 with key masks: some keys, whole tiles, all but three keys, all but one, or all of them hidden, and NaN or
    infinite; with lengths besides."""
    n = 6
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, BF16, 23)
    g = torch.Generator(device="cuda").manual_seed(6)
    kmask = torch.rand(n, tk, device="cuda", generator=g) < 0.7
    kmask[1, :67] = False
    kmask[2] = False
    kmask[2, [1, tk // 2, tk - 60]] = True
    kmask[3] = False
    kmask[4] = False
    kmask[4, tk // 3] = True
    klen = torch.tensor([tk, tk - 5, tk, tk, tk, tk // 2 + 3], dtype=torch.int32, device="cuda")
    hidden = (torch.arange(tk, device="cuda")[None] >= klen[:, None]) | ~kmask
    k.masked_fill_(hidden[:, :, None, None], math.nan)
    v.masked_fill_(hidden[:, :, None, None], math.inf)
    o, lse = check_all(ops, q, k, v, lam, dout, causal=causal, klen=klen, kmask=kmask)
    assert bool((o[3] == 0).all()) and bool((lse[3] == math.inf).all())
    want = reference(q, k, v, lam, dout, dh ** -0.5, causal, klen, kmask)
    got = run_all(ops, q, k, v, lam, dout, causal=causal, klen=klen, kmask=kmask)
    for b in (0, 1, 2, 5):  # each sequence by itself, whose rows outweigh none
        for x, y in zip((got[0], got[3], got[4], got[5]), (want[0], want[2], want[3], want[4])):
            assert rel(x[b], y[b]) < 2 * TOL[BF16], (b, rel(x[b], y[b]))
    # one key: dq and dk are 0 but for what two roundings of P dP - D leave
    for x, y in ((got[3], dout), (got[4], dout)):
        assert float(x[4].double().norm()) < 1e-5 * float(y[4].double().norm()) * float(q[4].double().norm())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tq,tk,h,hkv,dh", [(1, 3000, 4, 1, 64), (2, 700, 2, 2, 32), (3, 1111, 8, 2, 40), (1, 90, 2, 1, 16),
                                            (1, 500, 2, 1, 5)])
def test_few_rows_over_a_masked_cache(ops, tq, tk, h, hkv, dh, dtype):
    """New tokens against a cache of which keys are masked (left-padded prompts, dropped entries) and hold anything."""
    n = 5
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, dh, dtype, 3)
    g = torch.Generator(device="cuda").manual_seed(6)
    kmask = torch.rand(n, tk, device="cuda", generator=g) < 0.7
    kmask[1] = torch.arange(tk, device="cuda") >= tk // 2 + 3  # left padding
    kmask[2] = False
    kmask[2, [0, tk // 2]] = True
    kmask[3] = False
    klen = torch.tensor([tk, tk - 1, tk, tk, tk // 2 + 1], dtype=torch.int32, device="cuda")
    hidden = (torch.arange(tk, device="cuda")[None] >= klen[:, None]) | ~kmask
    k.masked_fill_(hidden[:, :, None, None], math.nan)
    v.masked_fill_(hidden[:, :, None, None], math.inf)
    want = reference(q, k, v, lam, dout, dh ** -0.5, "end", klen, kmask)[0]
    o = ops.diffattn_forward(q, k, v, lam, causal="end", klen=klen, kmask=kmask)
    assert bool((o[3] == 0).all())
    for b in (0, 1, 2, 4):
        assert rel(o[b], want[b]) < TOL[dtype], (b, rel(o[b], want[b]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("n,tq,tk,h,hkv", [(2, 200, 200, 2, 2), (3, 70, 500, 4, 2), (1, 513, 65, 2, 1), (4, 130, 3000, 2, 2)])
def test_narrowest_heads(ops, n, tq, tk, h, hkv, causal, dtype):
    """Halves of eight columns over tiles, with lengths and masked keys that hold anything."""
    q, k, v, lam, dout = make(n, tq, tk, h, hkv, 8, dtype, 41)
    check_all(ops, q, k, v, lam, dout, causal=causal)
    klen = torch.tensor([tk - 3, 1, tk // 2, 0][:n], dtype=torch.int32, device="cuda")
    kmask = torch.rand(n, tk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) < 0.7
    for m in (None, kmask):
        hidden = torch.arange(tk, device="cuda")[None] >= klen[:, None]
        hidden = hidden if m is None else hidden | ~m
        k2, v2 = k.masked_fill(hidden[:, :, None, None], math.nan), v.masked_fill(hidden[:, :, None, None], math.inf)
        check_all(ops, q, k2, v2, lam, dout, causal=causal, klen=klen, kmask=m)


@pytest.mark.parametrize("tq,tk,h,hkv,dh", [(409, 409, 3, 3, 56), (100, 210, 4, 2, 32), (1, 223, 8, 2, 64), (2, 3000, 4, 1, 64),
                                            (273, 273, 2, 2, 64), (130, 3000, 2, 2, 48), (300, 300, 2, 1, 5)])
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.6])
def test_sharp_maps(ops, tq, tk, h, hkv, dh, scale):
    """A few keys hold most of a row, and the maps' sums grow apart from tile to tile: the bf16 output keeps its
    precision, masked or not."""
    q, k, v, lam, dout = make(3, tq, tk, h, hkv, dh, BF16, 12)
    kmask = torch.rand(3, tk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) < 0.3
    kmask[2] &= torch.arange(tk, device="cuda") > tk // 2
    for m in (None, kmask):
        want = reference(q, k, v, lam, dout, scale, None, None, m)
        o, o2, _ = ops.diffattn_forward(q, k, v, lam, scale=scale, kmask=m, save=True)
        for b in range(3):
            assert rel(o[b], want[0][b]) < TOL[BF16] and rel(o2[b], want[1][b]) < TOL[BF16]


def test_nearly_equal_maps_over_a_long_cache(ops):
    """What is left of the difference keeps the type's precision when the keys are split too."""
    q, k, v, _, dout = make(1, 130, 3000, 2, 2, 32, BF16, 9)
    q[..., 32:], k[..., 32:] = q[..., :32], k[..., :32]
    lam = torch.full((2,), 0.75, device="cuda")
    want = reference(q, k, v, lam, dout, 32 ** -0.5)[0]
    assert rel(ops.diffattn_forward(q, k, v, lam), want) < 2.0 ** -8


def test_large_scores(ops):
    """Scores far apart, and maps whose sums differ by many orders: no overflow, no loss to the running ratio."""
    q, k, v, lam, dout = make(2, 70, 300, 2, 2, 32, F32, 8)
    check_all(ops, q, k, v, lam, dout, scale=2.0)
    up = torch.linspace(-1, 1, 300, device="cuda")[None, :, None, None]
    k2 = k.clone()
    k2[..., 32:] = q[:, :1, :, 32:] * up * 3  # the second map moves to the late keys
    check_all(ops, q, k2, v, lam, dout)
    check_all(ops, q, k, v, lam, dout, scale=-0.2)
    for value in (0.0, -0.5, 1.5):
        check_all(ops, q, k, v, torch.full_like(lam, value), dout)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_maps_in_common_are_rounded_together(ops, dtype):
    """Nearly equal maps: what is left of the difference keeps the type's precision."""
    q, k, v, _, dout = make(2, 130, 200, 2, 2, 32, dtype, 9)
    q[..., 32:], k[..., 32:] = q[..., :32], k[..., :32]
    lam = torch.full((2,), 0.75, device="cuda")
    want = reference(q, k, v, lam, dout, 32 ** -0.5)[0]
    # o = P v / 4: off by the map's and the output's rounding alone in bf16; f32 subtracts terms 4 times o
    assert rel(ops.diffattn_forward(q, k, v, lam), want) < (2.0 ** -8 if dtype == BF16 else 1e-5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_fused_projection_views(ops, dtype, shift):
    """q, k, v and their gradients as parts of one buffer, at any alignment, and heads outermost."""
    n, t, h, dh = 2, 90, 3, 32
    g = torch.Generator(device="cuda").manual_seed(0)
    base = torch.randn(n * t * 3 * h * 2 * dh + shift, device="cuda", generator=g).to(dtype)
    qkv = base[shift:].view(n, t, 3, h, 2 * dh)
    q, k, v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
    lam = torch.rand(h, device="cuda", generator=g)
    dout = torch.randn(n, h, t, 2 * dh, device="cuda", generator=g).to(dtype).transpose(1, 2)
    want = reference(q, k, v, lam, dout, dh ** -0.5, "start")
    out = torch.empty(n, h, t, 2 * dh, device="cuda", dtype=dtype).transpose(1, 2)
    o, o2, lse = ops.diffattn_forward(q, k, v, lam, causal="start", save=True, out=out)
    assert o is out and rel(o, want[0]) < TOL[dtype]
    dbase = torch.full_like(base, 7.0)
    dqkv = dbase[shift:].view(n, t, 3, h, 2 * dh)
    dlam = torch.ones(h, device="cuda")
    got = ops.diffattn_backward(dout, q, k, v, lam, o, o2, lse, dlam, causal="start", dq=dqkv[:, :, 0],
                                dk=dqkv[:, :, 1], dv=dqkv[:, :, 2])
    for x, y in zip(got, want[2:5]):
        assert rel(x, y) < TOL[dtype]
    assert bool((dbase[:shift] == 7).all())
    # dlam accumulates: 1 was there
    assert bool(((dlam.double() - 1 - want[5]).abs() <= 4e-6 * want[6] + 1e-6).all())


def test_broadcast_keys(ops):
    """One memory for all sequences: k and v expanded (stride 0); the gradient comes per sequence."""
    q, k, v, lam, dout = make(3, 40, 50, 2, 2, 16, F32, 2)
    k, v = k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)
    check_all(ops, q, k, v, lam, dout)


def test_offsets_past_32_bits(ops):
    """A cache whose rows lie more than 2^31 elements from its first."""
    n, tq, tk, h, dh = 1, 1, 70, 1, 32
    stride = 1 << 26
    kb = torch.empty(tk * stride, device="cuda", dtype=BF16)
    q, k, v, lam, dout = make(n, tq, tk, h, h, dh, BF16, 3)
    kv = kb.as_strided((n, tk, h, 2 * dh), (0, stride, 0, 1))
    vv = kb[64:].as_strided((n, tk, h, 2 * dh), (0, stride, 0, 1))
    kv.copy_(k)
    vv.copy_(v)
    want = reference(q, k, v, lam, dout, dh ** -0.5)
    assert rel(ops.diffattn_forward(q, kv, vv, lam), want[0]) < TOL[BF16]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_deterministic(ops, dtype):
    args = make(2, 200, 333, 4, 2, 64, dtype, 6)
    first = run_all(ops, *args, causal="end")
    for _ in range(3):
        for a, b in zip(first, run_all(ops, *args, causal="end")):
            assert torch.equal(a, b)
    q, k, v, lam, _ = make(1, 1, 9000, 4, 1, 64, dtype, 6)
    assert torch.equal(ops.diffattn_forward(q, k, v, lam), ops.diffattn_forward(q, k, v, lam))


def test_side_stream(ops):
    args = make(2, 100, 100, 2, 2, 32, F32, 1)
    want = run_all(ops, *args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_all(ops, *args)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_nothing_to_do(ops):
    """No sequence, no query, no key."""
    for n, tq, tk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, lam, dout = make(n, tq, tk, 2, 1, 8, F32)
        o, o2, lse, dq, dk, dv, dlam = run_all(ops, q, k, v, lam, dout)
        assert o.shape == q.shape and not bool(o.any()) and not bool(dq.any())
        assert not bool(dk.any()) and not bool(dv.any()) and not bool(dlam.any())


@pytest.mark.parametrize("which", ["q", "k", "v", "lam"])
def test_gradient_against_differences(ops, which):
    """Directional derivative of sum(o * dout): central differences of the f32
    forward pass with step 1e-2 have a truncation error near 1e-4 and a rounding
    error near 1e-5 of the terms summed; 5e-3 as the framework's other checks."""
    q, k, v, lam, dout = make(2, 20, 45, 2, 1, 16, F32, 21)
    how = dict(causal="end", klen=torch.tensor([45, 30], dtype=torch.int32, device="cuda"))
    _, _, _, dq, dk, dv, dlam = run_all(ops, q, k, v, lam, dout, **how)
    grad = {"q": dq, "k": dk, "v": dv, "lam": dlam}[which].double()
    args = {"q": q, "k": k, "v": v, "lam": lam}
    # along the gradient itself the derivative is its norm
    step = grad / grad.norm()

    def loss(e):
        moved = dict(args)
        moved[which] = (args[which].double() + e * step).float()
        return float((ops.diffattn_forward(**moved, **how).double() * dout.double()).sum())

    num = (loss(1e-2) - loss(-1e-2)) / 2e-2
    assert abs(num - float(grad.norm())) / float(grad.norm()) < 5e-3


def test_refusals(ops):
    q, k, v, lam, dout = make(2, 8, 9, 4, 2, 16, F32)
    f = ops.diffattn_forward
    o, o2, lse = f(q, k, v, lam, save=True)
    dlam = torch.zeros_like(lam)
    wide = make(1, 2, 2, 1, 1, 65, F32)
    i32 = dict(dtype=torch.int32, device="cuda")
    bad = [
        lambda: f(q.half(), k.half(), v.half(), lam),
        lambda: f(q, k.bfloat16(), v, lam),
        lambda: f(q[0], k[0], v[0], lam),
        lambda: f(q, k[:1], v[:1], lam),
        lambda: f(q, k, v[:, :8], lam),
        lambda: f(q[:, :, :3], k, v, lam[:3]),  # 3 heads over 2
        lambda: f(q[..., :31], k[..., :31], v[..., :31], lam),
        lambda: f(q.transpose(2, 3), k, v, lam),
        lambda: f(q, k, v, lam[:2]),
        lambda: f(q, k, v, lam.bfloat16()),
        lambda: f(q, k, v, lam.cpu()),
        lambda: f(q, k, v, lam, causal="both"),
        lambda: f(q, k, v, lam, klen=torch.zeros(3, **i32)),
        lambda: f(q, k, v, lam, klen=torch.zeros(2, device="cuda")),
        lambda: f(q, k, v, lam, kmask=torch.ones(2, 8, dtype=torch.bool, device="cuda")),
        lambda: f(q, k, v, lam, kmask=torch.ones(2, 9, device="cuda")),
        lambda: f(q, k, v, lam, out=torch.empty_like(q)[:1].expand(2, -1, -1, -1)),
        lambda: f(*wide[:4]),  # more than 64 columns a half
        lambda: ops.diffattn_backward(dout[:1], q, k, v, lam, o, o2, lse, dlam),
        lambda: ops.diffattn_backward(dout, q, k, v, lam, o, o2[:, :4], lse, dlam),
        lambda: ops.diffattn_backward(dout, q, k, v, lam, o, o2, lse[:1], dlam),
        lambda: ops.diffattn_backward(dout, q, k, v, lam, o, o2, lse, dlam[:1]),
        lambda: ops.diffattn_backward(dout, q, k, v, lam, o, o2, lse, dlam, dk=torch.empty_like(q)),
        lambda: ops.diffattn_backward(dout, q, k, v, lam, o, o2, lse, dlam,
                                      dk=torch.empty_like(k)[:1].expand(2, -1, -1, -1)),
    ]
    for i, g in enumerate(bad):
        with pytest.raises(ops.RnnError):
            g()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(ops.RnnError, match="UNSUPPORTED"):
        f(*wide[:4])


@pytest.mark.parametrize("causal", [None, "start"])
@pytest.mark.parametrize("second", [False, True])
def test_scores_that_keep_rising(ops, second, causal):
    """bf16 over several key tiles, each tile's scores far above those before
    it (up to 2^400 in all), in one map or in both: the running references move
    at every tile.  The scores themselves are exact to 2^-15 in f32, so the
    bounds of the type hold for the outputs.  (Not for dq: its sum of dS k cancels
    against the large column of k that all keys of a step have in common.)"""
    n, t, h, dh = 1, 700, 2, 32
    q, k, v, lam, dout = make(n, t, t, h, h, dh, BF16, 31)
    step = (torch.arange(t, device="cuda") // 50).float()[None, :, None]
    for half in ((0, 32) if second else (0,)):
        q[..., half] = 8.0
        k[..., half] = (step * 14).to(BF16)  # 8 * 14 / sqrt(32) = 20 more each 50 keys, 28 in base 2
    want = reference(q, k, v, lam, dout, dh ** -0.5, causal)
    o, o2, lse = ops.diffattn_forward(q, k, v, lam, causal=causal, save=True)
    assert rel(o, want[0]) < TOL[BF16] and rel(o2, want[1]) < TOL[BF16]
    assert bool(torch.isfinite(lse).all())


def test_many_blocks_same_result(ops):
    """More blocks than SMs, long rows, run after run the same bits, and the same as without the fast path's
    conditions (a key mask that hides nothing) up to rounding."""
    q, k, v, lam, _ = make(2, 2500, 2500, 16, 8, 64, BF16, 12)
    first = ops.diffattn_forward(q, k, v, lam, causal="start", save=True)
    for _ in range(8):
        for a, b in zip(first, ops.diffattn_forward(q, k, v, lam, causal="start", save=True)):
            assert torch.equal(a, b)
    mask = torch.ones(2, 2500, dtype=torch.bool, device="cuda")
    other = ops.diffattn_forward(q, k, v, lam, causal="start", kmask=mask, save=True)
    row = (first[0].double() - other[0].double()).norm(dim=-1) / other[0].double().norm(dim=-1)
    assert float(row.max()) < 2.0 ** -6  # two results, each within 2^-7 of every row
    assert rel(first[2], other[2].double()) < 1e-6

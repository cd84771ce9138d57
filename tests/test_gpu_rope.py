"""GPU parity of the multi-axis rotary positions against the definition in 64
bits: each pair as a complex number times exp(i * pos * inv_freq).

Bounds.  f32: cos and sin are off by at most about 2^-22 (2 ulp of sincospif
on an argument rounded once) and the rotation adds two roundings, so an
element is off by less than 4 * 2^-23 of its pair's length.  bf16: the same
and one rounding to 8 significant bits, half of 2^-7 of the element."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rustnn_b200 import ops as _ops

    return _ops


def pair_columns(pairs, inter):
    total = sum(pairs)
    p = torch.arange(total, device="cuda")
    return (2 * p, 2 * p + 1) if inter else (p, p + total)


def reference(x, pos, freq, pairs, inter, back):
    """(output, length of each element's pair) in 64 bits."""
    x = x.double()
    axis = torch.tensor([a for a, c in enumerate(pairs) for _ in range(c)], dtype=torch.long, device=x.device)
    angle = pos.double()[:, axis] * freq.double() * (-1.0 if back else 1.0)
    i, j = pair_columns(pairs, inter)
    z = torch.complex(x[..., i], x[..., j]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    y, size = x.clone(), x.abs()
    y[..., i], y[..., j] = z.real, z.imag
    size[..., i] = size[..., j] = z.abs()
    return y, size


def check(got, x, pos, freq, pairs, inter, back):
    want, size = reference(x, pos, freq, pairs, inter, back)
    tol = size * 2.0 ** -21
    if got.dtype == torch.bfloat16:
        tol = tol + want.abs() * 2.0 ** -8
    assert bool(((got.double() - want).abs() <= tol).all())


def make(rows, heads, dh, pairs, dtype, seed=0, high=4096):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, heads, dh, device="cuda", generator=g).to(dtype)
    pos = torch.randint(-high, high, (rows, len(pairs)), device="cuda", generator=g, dtype=torch.int32)
    freq = torch.tensor([100.0 ** (-k / max(1, c)) for c in pairs for k in range(c)], dtype=torch.float32, device="cuda")
    return x, pos, freq


SHAPES = [
    # rows, heads, dh, pairs: one token, odd rows and widths, every vector width, unrotated columns, no pair at all
    (1, 1, 2, (1,)),
    (1, 24, 64, (32,)),
    (7, 3, 64, (8, 12, 12)),
    (130, 5, 48, (10, 11)),
    (33, 2, 20, (3, 3, 2, 1)),
    (1000, 16, 32, (8, 8)),
    (257, 1, 7, (2, 1)),
    (64, 4, 96, (16, 16, 16)),
    (5, 2, 6, (0, 3)),
    (3, 2, 8, (0,)),
    (20000, 4, 64, (16, 16)),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rows,heads,dh,pairs", SHAPES)
def test_rope_parity(ops, rows, heads, dh, pairs, inter, dtype):
    x, pos, freq = make(rows, heads, dh, pairs, dtype, rows + dh)
    check(ops.rope(x, pos, freq, pairs, interleaved=inter), x, pos, freq, pairs, inter, False)
    check(ops.rope_backward(x, pos, freq, pairs, interleaved=inter), x, pos, freq, pairs, inter, True)


def test_rope_far_positions(ops):
    """The angle stays exact at the largest coordinates."""
    pairs = (16, 16)
    x, pos, freq = make(64, 2, 64, pairs, torch.float32, 5, high=2**31 - 1)
    check(ops.rope(x, pos, freq, pairs), x, pos, freq, pairs, False, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_strided_views_and_in_place(ops, dtype, shift, inter):
    """q and k of a fused projection, at any alignment, in place; other columns untouched."""
    rows, heads, dh, pairs = 50, 6, 32, (8, 4)
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(rows * 3 * heads * dh + shift, device="cuda", generator=g).to(dtype)
    view = base[shift:].view(rows, 3 * heads, dh)
    keep = base.clone()
    x = view[:, : 2 * heads]
    _, pos, freq = make(rows, 1, dh, pairs, dtype)
    want_in = x.clone()
    assert ops.rope(x, pos, freq, pairs, interleaved=inter, out=x) is x
    check(x, want_in, pos, freq, pairs, inter, False)
    assert torch.equal(view[:, 2 * heads:], keep[shift:].view(rows, 3 * heads, dh)[:, 2 * heads:])
    # heads outermost: [heads, rows, dh] seen as [rows, heads, dh]
    y = want_in.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(heads * 2, rows, dh, device="cuda", dtype=dtype).transpose(0, 1)
    check(ops.rope(y, pos, freq, pairs, interleaved=inter, out=out), want_in, pos, freq, pairs, inter, False)


def test_rope_offsets_past_32_bits(ops):
    """Rows more than 2^31 elements apart."""
    stride = (1 << 31) + 64
    base = torch.empty(2 * stride, device="cuda", dtype=torch.bfloat16)
    x = base.as_strided((2, 2, 32), (stride, 32, 1))
    pairs = (16,)
    fresh, pos, freq = make(2, 2, 32, pairs, torch.bfloat16)
    x.copy_(fresh)
    check(ops.rope(x, pos, freq, pairs), fresh, pos, freq, pairs, False, False)


def test_rope_empty_and_side_stream(ops):
    x, pos, freq = make(0, 3, 16, (8,), torch.float32)
    assert ops.rope(x, pos, freq, (8,)).shape == (0, 3, 16)
    x, pos, freq = make(100, 3, 16, (8,), torch.float32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.rope(x, pos, freq, (8,))
    s.synchronize()
    check(y, x, pos, freq, (8,), False, False)


def test_rope_backward_undoes_forward(ops):
    """The rotation is orthogonal: <R x, g> = <x, R^T g>, in f64 to f32 rounding."""
    pairs = (10, 6)
    x, pos, freq = make(40, 3, 40, pairs, torch.float32, 1)
    g = torch.randn_like(x)
    a = (ops.rope(x, pos, freq, pairs).double() * g.double()).sum()
    b = (x.double() * ops.rope_backward(g, pos, freq, pairs).double()).sum()
    # 4800 products of order 1, each off by at most 2^-21
    assert abs(float(a - b)) < 4800 * 2.0 ** -20


def test_rope_refusals(ops):
    x, pos, freq = make(4, 2, 16, (8,), torch.float32)
    bad = [
        lambda: ops.rope(x.double(), pos, freq, (8,)),
        lambda: ops.rope(x[0], pos, freq, (8,)),
        lambda: ops.rope(x.transpose(1, 2), pos, freq, (8,)),
        lambda: ops.rope(x, pos.long(), freq, (8,)),
        lambda: ops.rope(x, pos[:3], freq, (8,)),
        lambda: ops.rope(x, pos, freq[:7], (8,)),
        lambda: ops.rope(x, pos, torch.ones(9, device="cuda"), (9,)),  # does not fit 16 columns
        lambda: ops.rope(x, pos, torch.ones(7, device="cuda"), (8, -1)),
        lambda: ops.rope(x, torch.zeros(4, 5, dtype=torch.int32, device="cuda"), torch.ones(5, device="cuda"), (1,) * 5),
        lambda: ops.rope(x, pos, freq, (8,), out=torch.empty(4, 2, 15, device="cuda")),
        lambda: ops.rope(x, pos, freq, (8,), out=torch.empty(4, 2, 16, device="cuda", dtype=torch.bfloat16)),
        lambda: ops.rope(x, pos, freq, (8,), out=torch.empty(1, 2, 16, device="cuda").expand(4, 2, 16)),
        lambda: ops.rope(x, pos.cpu(), freq, (8,)),
    ]
    for f in bad:
        with pytest.raises(ops.RnnError):
            f()



"""The attention layer over video tokens (rustnn_b200/diff.py): gradients of a
whole layer against differences, ragged clips, tokens answered one at a time
against the whole clip, and a short training run."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def diff():
    from rustnn_b200 import diff as _diff

    return _diff


def clip_inputs(diff, layer, n, frames, side, seed=0):
    t = frames * side * side
    x = diff.clips(n, frames, side, layer.c, seed).contiguous()
    return x, t, diff.grid_positions(frames, side, side).repeat(n, 1)


@pytest.mark.parametrize("name", ["x", "wqkv", "lam", "hn_g", "wo"])
def test_gradient_against_differences(diff, name):
    """Along the gradient, central differences with a step of 1e-2: 5e-3 as the framework's other checks."""
    layer = diff.DiffLayer(h=2, dh=16, pairs=(2, 3, 3))
    x, t, pos = clip_inputs(diff, layer, 2, 2, 4)
    r = torch.randn(x.numel(), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    klen = torch.tensor([t, t - 5], dtype=torch.int32, device="cuda")
    layer.forward(x.view(-1), 2, t, pos, klen)
    dx = layer.backward(r)
    grad = (dx if name == "x" else layer.grads[name]).double().clone()
    step = grad / grad.norm()
    base = (x.view(-1) if name == "x" else layer.params[name]).clone()

    def loss(e):
        moved = (base.double() + e * step.view(base.shape)).float()
        if name == "x":
            y = layer.forward(moved, 2, t, pos, klen)
        else:
            layer.params[name].copy_(moved)
            y = layer.forward(x.view(-1), 2, t, pos, klen)
            layer.params[name].copy_(base)
        return float((y.double() * r.double()).sum())

    num = (loss(1e-2) - loss(-1e-2)) / 2e-2
    assert abs(num - float(grad.norm())) / float(grad.norm()) < 5e-3


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 5e-2)])
def test_one_token_at_a_time(diff, dtype, tol):
    """Tokens answered against the cache, one or several at a time, give the clip's rows: to the framework's 1e-4
    in f32; in bf16 to two roundings of values of order 1 scaled up by the head norm."""
    layer = diff.DiffLayer(h=2, dh=32, pairs=(4, 6, 6), dtype=dtype)
    n = 3
    x, t, pos = clip_inputs(diff, layer, n, 3, 5)
    whole = layer.forward(x.view(-1), n, t, pos).view(n, t, layer.c)
    cache, i = diff.Cache(layer, n, t), 0
    one = pos[:t]
    while i < t:
        m = min(t - i, 1 if i % 3 else 4)
        y = layer.extend(x[:, i:i + m].reshape(-1).contiguous(), n, m, one[i:i + m].repeat(n, 1), cache)
        assert float((y.view(n, m, layer.c) - whole[:, i:i + m]).abs().max()) < tol * float(whole.abs().max())
        i += m
    with pytest.raises(diff.RnnError):
        layer.extend(x[:, :1].reshape(-1).contiguous(), n, 1, one[:1].repeat(n, 1), cache)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_lowers_the_loss(diff, dtype):
    from rustnn_b200 import ops

    layer = diff.DiffLayer(h=2, dh=32, pairs=(4, 6, 6), dtype=dtype)
    losses = []
    for i in range(30):
        x, t, pos = clip_inputs(diff, layer, 4, 2, 8, i)
        target = torch.cat([x[:, 1:], x[:, :1] * 0], 1).contiguous().view(-1)
        y = layer.forward(x.view(-1), 4, t, pos)
        dy = torch.zeros_like(y)
        losses.append(float(ops.hint_mse(y, target, 4 * t, layer.c, 1.0, dy)))
        layer.backward(dy)
        layer.step()
    assert losses[-1] < 0.7 * losses[0], losses


def test_layer_refuses_what_does_not_fit(diff):
    with pytest.raises(diff.RnnError):
        diff.DiffLayer(h=2, dh=16, pairs=(4, 4, 4))

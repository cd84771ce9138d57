"""Sizes next to what the kernels' 32-bit row counts hold: refused before any launch."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_up_to_the_end_of_int(dtype):
    """2^30 - 1 queries of two heads on one key head: 2^31 - 2 rows, whose last block would end past 2^31."""
    from rustnn_b200 import ops

    tq = (1 << 30) - 1
    q = torch.zeros(1, 1, 1, 2, device="cuda", dtype=dtype).expand(1, tq, 2, 2)
    k = torch.zeros(1, 1, 1, 2, device="cuda", dtype=dtype)
    lam = torch.zeros(2, device="cuda")
    with pytest.raises(ops.RnnError, match="too large"):
        ops.diffattn_forward(q, k, k, lam)


def test_keys_past_int():
    """2^32 + 3 keys (one, expanded) are not taken for three."""
    from rustnn_b200 import ops

    q = torch.randn(1, 2, 1, 8, device="cuda")
    k = torch.randn(1, 1, 1, 8, device="cuda").expand(1, (1 << 32) + 3, 1, 8)
    with pytest.raises(ops.RnnError, match="along an axis"):
        ops.diffattn_forward(q, k, k, torch.zeros(1, device="cuda"))


def test_rope_rows_past_int():
    """2^32 + 3 rows are not taken for three."""
    from rustnn_b200 import ops

    rows = (1 << 32) + 3
    x = torch.ones(1, 1, 2, device="cuda", dtype=torch.bfloat16).expand(rows, 1, 2)
    pos = torch.empty(rows, 1, device="cuda", dtype=torch.int32)
    out = torch.empty(rows, 1, 2, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ops.RnnError, match="along an axis"):
        ops.rope(x, pos, torch.ones(1, device="cuda"), (1,), out=out)
    del pos, out
    torch.cuda.empty_cache()

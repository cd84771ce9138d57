"""CPU-side checks of the rotary and differential attention entries: calls
with bad arguments are refused on the host before any CUDA call."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    import os

    from rustnn_b200 import _lib

    if not os.path.exists(_lib.LIB_PATH):
        from rustnn_b200 import build

        build.build()
    return _lib.lib()


def test_null_context_is_refused(lib):
    from rustnn_b200._lib import DiffAttn

    assert lib.rnn_rope_dev(None, 0, None, 0, 0, 0, 1, 2, None, 1, None, None, 0, 0, None, 0, 0) == -1
    assert b"context" in lib.rnn_last_error()
    d = DiffAttn()
    assert lib.rnn_diffattn_fwd_dev(None, C.byref(d), *[None] * 7) == -1
    assert lib.rnn_diffattn_bwd_dev(None, C.byref(d), None, *[None] * 12) == -1
    assert b"context" in lib.rnn_last_error()


def test_description_layout_matches_header():
    """The ctypes, C and Rust declarations of rnn_diffattn list the same fields in the same order."""
    import os
    import re

    from rustnn_b200._lib import DiffAttn

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "rnn_b200.h")).read(), flags=re.S)
    body = re.search(r"typedef struct rnn_diffattn \{(.*?)\} rnn_diffattn;", text, flags=re.S).group(1)
    names = [re.sub(r"[^a-z0-9_]", "", part.split()[-1]) for line in body.split(";") if line.strip()
             for part in line.split(",")]
    assert names == [f[0] for f in DiffAttn._fields_]
    rust = open(os.path.join(root, "rust", "rnn-b200-sys", "src", "lib.rs")).read()
    body = re.search(r"pub struct RnnDiffAttn \{(.*?)\n\}", rust, flags=re.S).group(1)
    assert re.findall(r"pub ([a-z0-9_]+):", body) == names
    assert C.sizeof(DiffAttn) == 10 * 4 + 12 * 8 + 3 * 8


@pytest.mark.parametrize("name", ["rope", "rope_backward"])
def test_rope_refuses_cpu_tensors(name):
    import torch

    from rustnn_b200 import ops

    with pytest.raises(ops.RnnError):
        getattr(ops, name)(torch.zeros(2, 1, 4), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2), (2,))


def test_diffattn_refuses_cpu_tensors():
    import torch

    from rustnn_b200 import ops

    x = torch.zeros(1, 2, 1, 8)
    with pytest.raises(ops.RnnError):
        ops.diffattn_forward(x, x, x, torch.zeros(1))

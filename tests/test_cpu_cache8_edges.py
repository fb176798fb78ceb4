"""The 8-bit cache's host side at its edges, without a GPU: what a launch would be given."""
from dataclasses import replace

import pytest
import torch

from rbitnet_b200.kernels.ops import CudaOps
from test_cpu_cache8 import _NoLibrary, bare_ops, meta_of, view_of


class _Recorder(_NoLibrary):
    """Takes note of what would be launched."""
    def __init__(self):
        self.calls = []

    def call(self, name, *a, **kw):
        self.calls.append((name, a))


@pytest.mark.parametrize("kind", ["16 bits", "8 bits"])
@pytest.mark.parametrize("tokens", [1, 3, 100])
def test_queries_that_begin_between_16_bytes_are_copied(monkeypatch, kind, tokens):
    """The attention kernels load queries 16 bytes at a time, whichever of them takes the step."""
    ops, H, D = bare_ops(), 8, 128
    ops.lib, ops.prefill_on_tcgen05, ops.decode_on_tma = _Recorder(), True, True
    for name in ("_stream", "_raw_stream"):
        monkeypatch.setattr(CudaOps, name, lambda self: 0)
    monkeypatch.setattr(CudaOps, "_check", lambda self, t, dtype, what: None)
    monkeypatch.setattr(CudaOps, "_check_cache8", lambda self, view, what: 64)
    view = view_of()
    if kind == "16 bits":
        view = replace(view, k=view.k.to(torch.bfloat16), v=view.v.to(torch.bfloat16), scales=())
    base = torch.zeros(tokens * H * D + 8, dtype=torch.bfloat16)
    for off in range(8):
        ops.lib.calls.clear()
        q = base[off:off + tokens * H * D].view(tokens, H, D)
        ops.attention(q, meta_of(tokens), view, H, 1.0, None)
        name, args = next(c for c in ops.lib.calls if c[0].startswith("rb_attention") and not c[0].endswith("_plan"))
        at = args[1] if isinstance(args[1], int) else args[1].value or 0
        assert at % 16 == 0, (name, off)
        assert (at == q.data_ptr()) == (q.data_ptr() % 16 == 0)

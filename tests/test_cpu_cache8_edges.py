"""The 8-bit cache's host side at its edges, without a GPU: what a launch would be given."""
from dataclasses import replace

import pytest
import torch

from rbitnet_b200.engine.step import SeqChunk, build_meta
from rbitnet_b200.kernels.lib import KernelError
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


@pytest.mark.parametrize("seqs", [[(0, 0, 0), (1, 0, 100)], [(0, 3, 0), (1, 60, 40)], [(1, 5, 90), (0, 128, 0)], [(0, 0, 0)], []])
def test_a_step_may_hold_sequences_without_tokens(monkeypatch, seqs):
    """They bring no rows and no pages; a step of them alone launches nothing."""
    import numpy as np
    ops, H, D, at, chunks = bare_ops(), 64, 128, 0, []
    ops.lib, ops.prefill_on_tcgen05, ops.decode_on_tma = _Recorder(), True, True
    for name in ("_stream", "_raw_stream"):
        monkeypatch.setattr(CudaOps, name, lambda self: 0)
    monkeypatch.setattr(CudaOps, "_check", lambda self, t, dtype, what: None)
    monkeypatch.setattr(CudaOps, "_check_cache8", lambda self, view, what: 64)
    for slot, start, n in seqs:
        chunks.append(SeqChunk(slot, start, n, at))
        at += n
    meta = build_meta(chunks, np.zeros(at, dtype=np.int32), np.zeros(0, dtype=np.int32), "cpu")
    out = ops.attention(torch.zeros(at, H, D, dtype=torch.bfloat16), meta, view_of(), H, 1.0, None)
    assert out.shape == (at, H * D) and bool(ops.lib.calls) == (at > 0)
    if at:
        plan, table, step = next(v for k, v in meta.extra.items() if k[0] == "unpacked")
        assert [c.n_new for c in step.seqs] == [n for _, _, n in seqs if n] and table.shape[0] == 1
        assert plan.count == 2 and set(step.tok_slot.tolist()) == {0}


@pytest.mark.parametrize("kind", ["16 bits", "8 bits"])
@pytest.mark.parametrize("tokens", [1, 3, 100])
def test_options_are_not_left_behind_where_a_call_fails(monkeypatch, kind, tokens):
    """A sink, a cap and first keys are set for the launch that follows: whatever fails before it, they are not."""
    ops, H, D = bare_ops(), 8, 128
    ops.prefill_on_tcgen05, ops.decode_on_tma = True, True
    for name in ("_stream", "_raw_stream"):
        monkeypatch.setattr(CudaOps, name, lambda self: 0)
    monkeypatch.setattr(CudaOps, "_check", lambda self, t, dtype, what: None)
    monkeypatch.setattr(CudaOps, "_check_cache8", lambda self, view, what: 64)
    view = view_of()
    if kind == "16 bits":
        view = replace(view, k=view.k.to(torch.bfloat16), v=view.v.to(torch.bfloat16), scales=())
    real, fails = torch.empty, [0]

    def empty(*a, **kw):                         # the nth tensor cannot be had
        fails[0] -= 1
        if fails[0] < 0:
            raise torch.OutOfMemoryError("none left")
        return real(*a, **kw)
    monkeypatch.setattr(torch, "empty", empty)
    for n in range(5):
        ops.lib, fails[0] = _Recorder(), n
        ops.lib.raw = lambda name: lambda *a: 0 if name.endswith("_on_chip") else 2
        try:
            ops.attention(torch.zeros(tokens, H, D, dtype=torch.bfloat16), meta_of(tokens), view, H, 1.0, None, sinks=torch.zeros(H), softcap=3.0)
        except torch.OutOfMemoryError:
            pass
        names = [name for name, _ in ops.lib.calls]
        for i, name in enumerate(names):
            assert name != "rb_attention_next" or names[i + 1:][:1] and names[i + 1].startswith("rb_attention"), names
    assert "rb_attention_next" in names


@pytest.mark.parametrize("kind", ["16 bits", "8 bits"])
@pytest.mark.parametrize("tokens", [1, 3, 100])
def test_sinks_of_other_heads_are_refused(monkeypatch, kind, tokens):
    """(A kernel reads one for every head of the queries.)"""
    ops, H, D = bare_ops(), 8, 128
    ops.lib, ops.prefill_on_tcgen05, ops.decode_on_tma = _Recorder(), True, True
    for name in ("_stream", "_raw_stream"):
        monkeypatch.setattr(CudaOps, name, lambda self: 0)
    monkeypatch.setattr(CudaOps, "_check", lambda self, t, dtype, what: None)
    monkeypatch.setattr(CudaOps, "_check_cache8", lambda self, view, what: 64)
    view = view_of()
    if kind == "16 bits":
        view = replace(view, k=view.k.to(torch.bfloat16), v=view.v.to(torch.bfloat16), scales=())
    for shape in ((H - 1,), (H + 1,), (2, H), ()):
        with pytest.raises(KernelError, match="sinks"):
            ops.attention(torch.zeros(tokens, H, D, dtype=torch.bfloat16), meta_of(tokens), view, H, 1.0, None, sinks=torch.zeros(shape))
        assert "rb_attention_next" not in [name for name, _ in ops.lib.calls]
    ops.attention(torch.zeros(tokens, H, D, dtype=torch.bfloat16), meta_of(tokens), view, H, 1.0, None, sinks=torch.zeros(H))


def test_frequencies_that_are_too_few_or_elsewhere_are_refused(monkeypatch):
    """(A kernel reads one for every pair that it turns.)"""
    ops, H, D = bare_ops(), 4, 128
    ops.lib = _Recorder()
    monkeypatch.setattr(CudaOps, "_raw_stream", lambda self: 0)
    monkeypatch.setattr(CudaOps, "_check_cache8", lambda self, view, what: 64)
    rows = torch.zeros(3, (H + 4) * D, dtype=torch.bfloat16)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    good = torch.zeros(64)
    for bad in (good[:63], good.double(), torch.zeros(128)[::2], good.to("meta")):
        with pytest.raises(KernelError, match="frequencies"):
            ops.rotate_append(rows, (bad, False, D), meta_of(3), view_of(), H)
    assert ops.lib.calls == []
    for fine in ((good, False, D), (good[:32], True, 64), None):
        ops._zf = good
        ops.rotate_append(rows, fine, meta_of(3), view_of(), H)
    assert [name for name, _ in ops.lib.calls] == ["rb_append8"] * 3


def test_tensors_on_different_devices_are_refused(monkeypatch):
    ops, H, D = bare_ops(), 8, 128
    ops.lib = _Recorder()
    for name in ("_stream", "_raw_stream"):
        monkeypatch.setattr(CudaOps, name, lambda self: 0)
    monkeypatch.setattr(CudaOps, "_check_cache8", lambda self, view, what: 64)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    view = view_of()
    with pytest.raises(KernelError, match="meta"):
        ops.attention(torch.zeros(3, H, D, dtype=torch.bfloat16, device="meta"), meta_of(3), view, H, 1.0, None)
    with pytest.raises(KernelError, match="meta"):
        ops.rotate_append(torch.zeros(3, (H + 4) * D, dtype=torch.bfloat16, device="meta"), None, meta_of(3), view, H)
    args = [torch.zeros(3, 10), torch.tensor([0, 2, 3], dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2), torch.zeros(3, 2)]
    for i in range(len(args)):
        with pytest.raises(KernelError, match="meta"):
            ops.verify_drafts(*[t.to("meta") if j == i else t for j, t in enumerate(args)], 1)
    with pytest.raises(KernelError, match="meta"):
        ops.verify_drafts(*args, 1, draft_probs=torch.zeros(3, 10, device="meta"))
    assert ops.lib.calls == []
    ops.lib.raw = lambda name: lambda *a: 64
    ops.verify_drafts(*args, 1)
    assert [name for name, _ in ops.lib.calls] == ["rb_verify"]

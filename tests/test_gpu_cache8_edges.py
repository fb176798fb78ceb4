"""The 8-bit cache's kernels at their edges, against plain 64-bit torch or against themselves; tolerances as in test_gpu_cache8."""
import pytest
import torch

from rbitnet_b200.cache import CacheLayerView
from test_gpu_cache8 import BF16, make_meta, make_view, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rbitnet_b200.kernels.ops import CudaOps
    return CudaOps(BF16)


@pytest.mark.parametrize("H,Kh,D,seqs,window", [
    (8, 2, 128, [(0, 100, 90), (1, 3, 70)], 0),                # bfloat16 pages, the prefill kernel
    (16, 1, 64, [(0, 100, 5), (1, 3, 8)], 70),
    (4, 2, 80, [(0, 100, 20), (1, 3, 1)], 0),                  # other head sizes
    (8, 2, 128, [(0, 100, 5), (1, 3, 2)], 0),                  # codes as they are
    (8, 2, 128, [(0, 100, 1), (1, 3, 1)], 0),
])
@pytest.mark.parametrize("bits", [8, 16])
def test_queries_that_begin_anywhere(ops, H, Kh, D, seqs, window, bits):
    """A part of a wider tensor is attended as a tensor of its own is, to the bit."""
    view, _ = make_view(12, Kh, 64, D, 2, 3, seed=1)
    if bits == 16:
        k, v = (torch.randn(12, Kh, 64, D, generator=torch.Generator().manual_seed(s)).to(BF16).cuda() for s in (1, 2))
        view = CacheLayerView(k, v, view.page_table, 3, 64, Kh, D, True, 0, (k, v))
    T = sum(n for _, _, n in seqs)
    base = rows_of([(0, 0, 1)], T * H * D + 8, seed=3).cuda().view(-1)
    for off in (1, 4, 7):
        q = base[off:off + T * H * D].view(T, H, D)
        want = ops.attention(q.clone(), make_meta(seqs), view, H, D ** -0.5, window)
        assert torch.equal(ops.attention(q, make_meta(seqs), view, H, D ** -0.5, window), want), off

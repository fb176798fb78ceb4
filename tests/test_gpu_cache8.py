"""The cache held in 8 bits and the check of drafted tokens, kernel by kernel, against plain 64-bit torch (plain_cache8).

Tolerances.  A code is off by at most half a step of e4m3: 2^-4 of the value, 2^-10 of the scale near zero; keys are turned
in float32 first (a few 2^-24 of the pair's size).  A bfloat16 result is off by 2^-8 of itself; the weights of a softmax
are rounded to 16 bits at most as bfloat16 (2^-8 of a weight) in the products, so that a sum of weight * value is off by that
part of the sum of weight * |value|; scores and sums are float32 (2^-14 of the same covers scores up to 64 and sums of
thousands of terms)."""
import math

import pytest
import torch

import plain_cache8 as plain
from rbitnet_b200.cache import CacheLayerView
from rbitnet_b200.engine.step import SeqChunk, build_meta

pytestmark = pytest.mark.gpu

BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from rbitnet_b200.kernels.ops import CudaOps
    return CudaOps(BF16)


def make_view(n_pages, Kh, page, D, n_slots, max_pages, seed=0, writes=True):
    """A view with random codes and scales, pages dealt in random order; and its copy on the CPU."""
    g = torch.Generator().manual_seed(seed)
    block = plain.block_of(page)
    codes = [plain.to_e4m3(torch.randn(n_pages, Kh, page, D, generator=g) * 100).to(E4M3) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-9, -5, (n_pages, Kh, page // block), generator=g).float()) for _ in range(2)]
    assert n_slots * max_pages <= n_pages
    table = torch.randperm(n_pages, generator=g)[:n_slots * max_pages].to(torch.int32).view(n_slots, max_pages)
    return both_views(codes, scales, table, page, writes)


def both_views(codes, scales, table, page, writes=True):
    Kh, D = codes[0].shape[1], codes[0].shape[3]
    made = []
    for dev in ("cuda", "cpu"):
        k, v, ks, vs, t = (x.to(dev).clone() for x in (*codes, *scales, table))
        made.append(CacheLayerView(k, v, t, table.shape[1], page, Kh, D, writes, 0, (k, v), (ks, vs)))
    return made


def make_meta(seqs):
    """seqs: (slot, first position, new tokens)."""
    import numpy as np
    chunks, at = [], 0
    for slot, start, n in seqs:
        chunks.append(SeqChunk(slot, start, n, at))
        at += n
    return build_meta(chunks, np.zeros(at, dtype=np.int32), np.zeros(0, dtype=np.int32), torch.device("cuda"))


def rows_of(seqs, width, seed=1, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(sum(n for _, _, n in seqs), width, generator=g) * size).to(BF16)


def frequencies(rot_dim):
    return 1.0 / 10000.0 ** (torch.arange(0, max(rot_dim, 2), 2, dtype=F32) / max(rot_dim, 2))


def same_codes(got, want, where=None):
    a, b = got.cpu().view(torch.uint8), want.view(torch.uint8)
    return torch.equal(a, b) if where is None else torch.equal(a[where], b[where])


APPENDS = [
    # heads, kv heads, head size, page, rotated values, interleaved, (slot, first position, new tokens) of every sequence
    (8, 2, 128, 64, 128, False, [(0, 0, 1), (2, 63, 1), (1, 64, 1), (3, 130, 1)]),
    (8, 2, 128, 64, 128, False, [(0, 0, 64), (2, 60, 9), (1, 127, 2), (3, 5, 200)]),
    (4, 4, 64, 64, 64, True, [(1, 0, 1)]),
    (4, 1, 64, 128, 32, False, [(1, 70, 70), (0, 0, 129)]),
    (3, 3, 80, 16, 80, False, [(1, 3, 40), (0, 15, 2)]),
    (6, 2, 10, 8, 4, True, [(1, 3, 17), (0, 0, 1)]),
    (16, 1, 512, 64, 512, False, [(0, 10, 70)]),
    (7, 7, 2, 1, 2, False, [(0, 0, 3), (1, 2, 1)]),
    (32, 8, 128, 64, 128, False, [(0, 0, 700), (1, 100, 333)]),
]


@pytest.mark.parametrize("H,Kh,D,page,rot,inter,seqs", APPENDS)
def test_append(ops, H, Kh, D, page, rot, inter, seqs):
    most = max(s + n for _, s, n in seqs)
    max_pages = -(-most // page)
    view, cpu = make_view(4 * max_pages + 2, Kh, page, D, 4, max_pages, seed=H + D)
    before = [t.clone() for t in (view.k, view.v)]
    freq = frequencies(rot)
    x = rows_of(seqs, (H + 2 * Kh) * D, size=2.0)
    meta = make_meta(seqs)
    q = ops.rotate_append(x.cuda(), (freq.cuda(), inter, rot), meta, view, H)
    rows = x.to(F64).view(-1, H + 2 * Kh, D)
    at = 0
    touched = torch.zeros(view.k.shape[0], page, dtype=torch.bool)
    for slot, start, n in seqs:
        pos = torch.arange(start, start + n)
        r = rows[at:at + n]
        t = plain.turned(r[:, :H + Kh], pos, freq, rot, inter)
        size = r[:, :H].abs().amax(-1, keepdim=True)
        assert torch.all((q[at:at + n].cpu().to(F64) - t[:, :H]).abs() <= 2.0 ** -8 * t[:, :H].abs() + 2.0 ** -21 * size)
        plain.append(cpu, slot, start, t[:, H:], r[:, H + Kh:])
        block = plain.block_of(page)
        for p in range(start - start % block, start + n):
            touched[int(cpu.page_table[slot, p // page]), p % page] = True
        at += n
    # the scales; the values, which no rotation has touched, to the bit; what no new position shares a block with, as it was
    assert torch.equal(view.scales[0].cpu(), cpu.scales[0]) and torch.equal(view.scales[1].cpu(), cpu.scales[1])
    assert same_codes(view.v, cpu.v)
    for now, was in ((view.k, before[0]), (view.v, before[1])):
        keep = ~touched[:, None, :, None].expand(now.shape)
        assert same_codes(now, was.cpu(), keep)
    # the keys: a code apart where the two rotations round to different sides
    at = 0
    for slot, start, n in seqs:
        t = plain.turned(rows[at:at + n, H:H + Kh], torch.arange(start, start + n), freq, rot, inter)
        got = plain.values(CacheLayerView(view.k.cpu(), None, cpu.page_table, max_pages, page, Kh, D, True, 0, (), (cpu.scales[0],)),
                           slot, start + n, 0)[:, start:].transpose(0, 1)
        unit = torch.stack([cpu.scales[0][int(cpu.page_table[slot, p // page]), :, p % page // plain.block_of(page)]
                            for p in range(start, start + n)]).to(F64)[..., None]
        assert torch.all((got - t).abs() <= (1 + 2.0 ** -10) * torch.maximum(2.0 ** -4 * t.abs(), 2.0 ** -10 * unit) + 2.0 ** -20)
        at += n


def test_a_scale_grows_with_a_block_and_begins_afresh(ops):
    """Single tokens of growing and shrinking size through two blocks: the codes are those of the plain form at every step."""
    H, Kh, D, page = 2, 2, 64, 64
    view, cpu = make_view(4, Kh, page, D, 1, 2, seed=5)
    g = torch.Generator().manual_seed(9)
    for pos in range(0, 70):
        size = 2.0 ** ((pos * 7) % 23 - 11)
        x = (torch.randn(1, 3 * H * D, generator=g) * size).to(BF16)
        ops.rotate_append(x.cuda(), None, make_meta([(0, pos, 1)]), view, H)
        r = x.to(F64).view(1, 3 * H, D)
        plain.append(cpu, 0, pos, r[:, H:2 * H], r[:, 2 * H:])
        assert torch.equal(view.scales[0].cpu(), cpu.scales[0]) and torch.equal(view.scales[1].cpu(), cpu.scales[1]), pos
        assert same_codes(view.k, cpu.k) and same_codes(view.v, cpu.v), pos


def test_append_again_changes_nothing(ops):
    H, Kh, D = 4, 2, 128
    view, _ = make_view(9, Kh, 64, D, 2, 3, seed=6)
    seqs = [(0, 20, 100), (1, 63, 2)]
    x, meta = rows_of(seqs, (H + 2 * Kh) * D, size=30.0).cuda(), make_meta(seqs)
    rotary = (frequencies(D).cuda(), False, D)
    ops.rotate_append(x, rotary, meta, view, H)
    kept = [t.clone() for t in (view.k.view(torch.uint8), view.v.view(torch.uint8), *view.scales)]
    ops.rotate_append(x, rotary, meta, view, H)
    assert all(torch.equal(a, b) for a, b in zip(kept, (view.k.view(torch.uint8), view.v.view(torch.uint8), *view.scales)))


def test_values_that_are_not_finite_and_the_ends_of_the_range(ops):
    H, D = 1, 64
    view, cpu = make_view(2, 1, 64, D, 1, 1, seed=7)
    x = torch.randn(4, 3 * D, generator=torch.Generator().manual_seed(3)).to(BF16)
    x[1, D + 3], x[1, 2 * D + 5] = math.nan, math.nan
    x[2, 2 * D + 1] = 1e-30
    x[3] = 0
    ops.rotate_append(x.cuda(), None, make_meta([(0, 0, 4)]), view, H)
    r = x.to(F64).view(4, 3, D)
    plain.append(cpu, 0, 0, r[:, 1:2], r[:, 2:])
    assert torch.equal(view.scales[0].cpu(), cpu.scales[0]) and torch.equal(view.scales[1].cpu(), cpu.scales[1])
    for got, want in ((view.k, cpu.k), (view.v, cpu.v)):
        a, b = got[int(cpu.page_table[0, 0]), 0, :4].float().cpu(), want[int(cpu.page_table[0, 0]), 0, :4].float()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])
    # an infinity takes the largest scale, and is stored as the largest value; all zeros take the smallest one
    x = torch.zeros(1, 3 * D).to(BF16)
    x[0, 2 * D] = -math.inf
    ops.rotate_append(x.cuda(), None, make_meta([(0, 0, 1)]), view, H)
    page = int(cpu.page_table[0, 0])
    assert float(view.scales[0][page, 0, 0]) == 2.0 ** -60 and float(view.scales[1][page, 0, 0]) == 2.0 ** 119
    assert float(view.v[page, 0, 0, 0]) == -448.0 and not view.v[page, 0, 0, 1:].float().any()


@pytest.mark.parametrize("page,D", [(64, 128), (128, 64), (16, 80), (8, 10)])
def test_values_read_back(ops, page, D):
    Kh = 3
    view, cpu = make_view(20, Kh, page, D, 2, 8, seed=8)
    ranges = [(1, page // 2, 3 * page - 1), (0, 0, 1), (1, 4 * page, 8 * page)]
    plan = ops.cache_ranges(view, ranges)
    k, v = ops.cache_values(view, plan)
    assert k.dtype == BF16 and plan.count == 3 + 1 + 4 and plan.first_item == [0, 3, 4]
    for stream, got in ((0, k), (1, v)):
        for (slot, first, end), at in zip(ranges, plan.first_item):
            lo = first - first % page
            want = plain.values(cpu, slot, end, stream)[:, lo:]
            n = -(-end // page) - lo // page
            have = got[at:at + n].transpose(0, 1).reshape(Kh, n * page, D).cpu().to(F64)
            assert torch.equal(have[:, :end - lo], want) and not have[:, end - lo:].any()


ATTENDS = [
    # heads, kv heads, head size, page, (slot, first position, new tokens), window, sinks, cap, first keys that stay visible
    (8, 2, 128, 64, [(0, 0, 1), (2, 63, 1), (1, 64, 1), (3, 200, 1)], 0, False, 0.0, 0),
    (4, 4, 64, 64, [(0, 500, 1)], 0, False, 0.0, 0),
    (8, 1, 128, 128, [(0, 300, 1), (1, 5, 1)], 100, True, 0.0, 0),
    (16, 1, 64, 64, [(0, 300, 1), (1, 5, 1)], 70, False, 30.0, 10),
    (12, 2, 128, 64, [(0, 300, 5), (1, 0, 3), (2, 62, 4)], 0, True, 20.0, 0),
    (24, 8, 64, 64, [(0, 300, 2), (1, 130, 8)], 65, False, 0.0, 70),
    (28, 4, 128, 64, [(0, 10, 130), (1, 0, 77)], 0, False, 0.0, 0),
    (4, 2, 80, 16, [(0, 30, 1), (1, 0, 1)], 0, False, 0.0, 0),
    (4, 2, 80, 16, [(0, 30, 20), (1, 0, 7)], 9, True, 0.0, 3),
    (3, 3, 10, 8, [(0, 30, 3)], 0, False, 5.0, 0),
    (64, 2, 128, 64, [(0, 100, 1), (1, 3, 1)], 0, False, 0.0, 0),
    (40, 1, 64, 64, [(0, 100, 2)], 0, True, 0.0, 0),
    (32, 8, 128, 64, [(0, 1900, 1)], 0, False, 0.0, 0),
]


@pytest.mark.parametrize("H,Kh,D,page,seqs,window,sinks,cap,keep", ATTENDS)
def test_attention(ops, H, Kh, D, page, seqs, window, sinks, cap, keep):
    max_pages = -(-max(s + n for _, s, n in seqs) // page)
    view, cpu = make_view(4 * max_pages + 2, Kh, page, D, 4, max_pages, seed=H * D)
    q = rows_of(seqs, H * D, seed=2).view(-1, H, D)
    sink = torch.linspace(-2.0, 3.0, H) if sinks else None
    got = ops.attention(q.cuda(), make_meta(seqs), view, H, D ** -0.5, window, sinks=None if sink is None else sink.cuda(), softcap=cap,
                        keep_first=keep).cpu().to(F64)
    at = 0
    for slot, start, n in seqs:
        want, size = plain.attend(cpu, slot, start, q[at:at + n], D ** -0.5, window, sink, cap, keep)
        off = (got[at:at + n] - want).abs()
        assert torch.all(off <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size + 1e-30), float((off / (size + 1e-30)).max())
        at += n


def drafts_case(B, most, V, certain, seed, ragged=True):
    g = torch.Generator().manual_seed(seed)
    rows = [1 + (most if not ragged else int(torch.randint(0, most + 1, (1,), generator=g))) for _ in range(B)]
    first = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    R = int(first[-1])
    logits = torch.randn(R, V, generator=g) * 3
    drafts = torch.where(torch.rand(R, generator=g) < 0.7, logits.argmax(1), torch.randint(V, (R,), generator=g)).to(torch.int32)
    probs = None if certain else torch.softmax(logits + torch.randn(R, V, generator=g), dim=1)
    temperature = 0.5 + torch.rand(B, generator=g)
    temperature[::3] = 0.0
    return logits, first, drafts, temperature, torch.rand(R, 2, generator=g), most, probs


def verified(ops, logits, first, drafts, temperature, uniforms, most, probs):
    a, t = ops.verify_drafts(logits.cuda(), first.cuda(), drafts.cuda(), temperature.cuda(), uniforms.cuda(), most,
                             draft_probs=None if probs is None else probs.cuda())
    return a.tolist(), t.tolist()


@pytest.mark.parametrize("B,most,V,certain", [(1, 4, 1000, True), (5, 3, 5000, False), (9, 1, 1, True), (4, 0, 77, False), (7, 8, 4096, False),
                                              (3, 5, 32000, True), (2, 2, 128256, False), (70, 2, 33, False)])
def test_verify(ops, B, most, V, certain):
    for seed in range(3):
        case = drafts_case(B, most, V, certain, seed)
        assert verified(ops, *case) == plain.verify(*case)


def test_verify_at_the_edges(ops):
    """Rows of -inf and NaN, infinite logits, drafts that are no tokens, equal logits, drafters whose probabilities leave nothing."""
    V, inf = 300, math.inf
    logits = torch.randn(9, V, generator=torch.Generator().manual_seed(1))
    logits[0] = -inf
    logits[1] = math.nan
    logits[2, 7] = inf
    logits[2, 9] = inf
    logits[3] = 0.5
    logits[4, 100:] = -inf
    logits[5, ::2] = math.nan
    first = torch.arange(0, 10, 1, dtype=torch.int32)
    for temperature in (0.0, 0.7, 1e-30, 1e30, -1.0):
        for u in (0.0, 0.25, 1.0 - 2.0 ** -24):
            t = torch.full((9,), temperature)
            case = (logits, first, torch.zeros(9, dtype=torch.int32), t, torch.full((9, 2), u), 0, None)
            assert verified(ops, *case) == plain.verify(*case), (temperature, u)
            pairs = torch.tensor([0, 2, 4, 6, 8, 9], dtype=torch.int32)
            for d in (-1, 0, 7, 99, V, V + 5):
                drafts = torch.full((9,), d, dtype=torch.int32)
                for probs in (None, torch.softmax(logits.nan_to_num(0.0, 1.0, -1.0), dim=1), torch.full((9, V), 1.0)):
                    case = (logits, pairs, drafts, t[:5].clone(), torch.full((9, 2), u), 1, probs)
                    assert verified(ops, *case) == plain.verify(*case), (temperature, u, d)
    # a sequence without rows
    a, t = verified(ops, logits, torch.tensor([0, 0, 2], dtype=torch.int32), torch.zeros(9, dtype=torch.int32), torch.zeros(2),
                    torch.zeros(9, 2), 3, None)
    assert a[0] == 0 and t[0] == [-1, -1, -1, -1]

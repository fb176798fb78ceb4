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
from helpers import bf16_rtol
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
    (4, 2, 256, 64, 256, False, [(0, 10, 70), (1, 5, 1)]),
    (4, 2, 256, 64, 256, True, [(0, 3, 1), (2, 70, 1)]),
    (8, 1, 96, 64, 96, False, [(0, 61, 5), (2, 0, 3)]),
    (20, 1, 64, 64, 64, True, [(0, 61, 5), (2, 0, 3)]),
    (12, 12, 64, 64, 64, False, [(0, 7, 1)]),
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


@pytest.mark.parametrize("H,Kh,D,page,rot,inter,seqs", [
    (4, 4, 128, 64, 128, False, [(0, 9000, 1500), (1, 9998, 3)]),                    # whole tiles
    (8, 8, 64, 64, 64, True, [(0, 9000, 1500)]),
    (2, 2, 256, 64, 256, False, [(0, 9000, 500)]),
    (16, 16, 128, 64, 128, False, [(s, 8000 + 77 * s, 1) for s in range(8)]),        # a token a sequence
    (16, 16, 128, 64, 128, True, [(s, 8000 + 77 * s, 3) for s in range(8)]),
    (4, 4, 80, 16, 40, False, [(0, 9000, 500)]),                                     # any sizes
    (4, 4, 10, 8, 10, True, [(0, 900, 700)]),
])
def test_the_codes_of_keys_are_those_of_the_exact_rotation(ops, H, Kh, D, page, rot, inter, seqs):
    """To the bit: a number that lies as near a border between two codes as float32 sines are off is turned in float64."""
    max_pages = -(-max(s + n for _, s, n in seqs) // page)
    slots = 1 + max(s for s, _, _ in seqs)
    view, cpu = make_view(slots * max_pages, Kh, page, D, slots, max_pages, seed=3 * D)
    freq = frequencies(rot)
    x = rows_of(seqs, (H + 2 * Kh) * D, seed=21, size=3.0)
    ops.rotate_append(x.cuda(), (freq.cuda(), inter, rot), make_meta(seqs), view, H)
    rows, at = x.to(F64).view(-1, H + 2 * Kh, D), 0
    for slot, start, n in seqs:
        r = rows[at:at + n]
        plain.append(cpu, slot, start, plain.turned(r[:, H:H + Kh], torch.arange(start, start + n), freq, rot, inter), r[:, H + Kh:])
        at += n
    assert torch.equal(view.scales[0].cpu(), cpu.scales[0]) and torch.equal(view.scales[1].cpu(), cpu.scales[1])
    assert same_codes(view.k, cpu.k) and same_codes(view.v, cpu.v)


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


@pytest.mark.parametrize("new", [1, 3, 90])
def test_one_step_over_caches_of_different_pages(ops, new):
    """What a step keeps for its layers goes by the pages' size and the table's, so that layers of another cache get their own."""
    H, Kh, D = 4, 2, 64
    seqs = [(0, 130, new), (2, 40, new)]
    meta = make_meta(seqs)
    q = rows_of(seqs, H * D, seed=4).view(-1, H, D)
    for i, (page, spare, slots) in enumerate([(64, 0, 4), (16, 0, 4), (64, 3, 3), (128, 0, 4), (64, 0, 4)]):
        max_pages = -(-(130 + new) // page) + spare
        view, cpu = make_view(slots * max_pages, Kh, page, D, slots, max_pages, seed=50 + i)
        got = ops.attention(q.cuda(), meta, view, H, D ** -0.5, 0).cpu().to(F64)
        at = 0
        for slot, start, n in seqs:
            want, size = plain.attend(cpu, slot, start, q[at:at + n], D ** -0.5)
            off = (got[at:at + n] - want).abs()
            assert torch.all(off <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size + 1e-30), (i, float((off / (size + 1e-30)).max()))
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
                                              (3, 5, 32000, True), (2, 2, 128256, False), (70, 2, 33, False), (4, 40, 60, True)])
def test_verify(ops, B, most, V, certain):
    for seed in range(3):
        case = drafts_case(B, most, V, certain, seed)
        assert verified(ops, *case) == plain.verify(*case)
    # everything is accepted but the last few
    case[2].copy_(torch.where(torch.arange(len(case[2])) % 37 < 36, case[0].argmax(1).to(torch.int32), case[2]))
    case[3].zero_()
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


# ---- used as a program uses them
def test_a_step_on_another_stream_with_strided_rows(ops):
    """Rows that are a part of wider ones, a stream of the caller's own, the result read there."""
    H, Kh, D = 8, 2, 128
    view, cpu = make_view(9, Kh, 64, D, 2, 3, seed=11)
    seqs = [(0, 100, 1), (1, 63, 1)]
    wide = rows_of(seqs, (H + 2 * Kh) * D + 64, seed=4)
    x = wide[:, 64:]
    meta, freq = make_meta(seqs), frequencies(D)
    on_gpu, side = wide.cuda()[:, 64:], torch.cuda.Stream()
    rotary = (freq.cuda(), False, D)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        q = ops.rotate_append(on_gpu, rotary, meta, view, H)
        out = ops.attention(q, meta, view, H, D ** -0.5, None)
    side.synchronize()
    r = x.to(F64).view(2, -1, D)
    for i, (slot, start, n) in enumerate(seqs):
        t = plain.turned(r[i:i + 1, :H + Kh], torch.tensor([start]), freq, D, False)
        plain.append(cpu, slot, start, t[:, H:], r[i:i + 1, H + Kh:])
    assert same_codes(view.v, cpu.v)
    cpu.k.copy_(view.k.cpu())                   # (a code apart at most: compared in test_append)
    for i, (slot, start, n) in enumerate(seqs):
        want, size = plain.attend(cpu, slot, start, q[i:i + 1].cpu(), D ** -0.5)
        assert torch.all((out[i:i + 1].cpu().to(F64) - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size)


@pytest.mark.parametrize("H,Kh,D", [(8, 2, 128), (8, 8, 64), (4, 2, 80)])
def test_a_captured_step_replayed_at_other_positions(ops, H, Kh, D):
    """Append and attention of single tokens recorded once: the replays work on the positions, slots and rows that lie in the buffers
    then, also where two graphs alternate, and give what the calls themselves give, to the bit."""
    a, _ = make_view(40, Kh, 64, D, 4, 10, seed=12)
    b, _ = make_view(40, Kh, 64, D, 4, 10, seed=12)
    rotary = (frequencies(D).cuda(), True, D)
    x = torch.zeros(3, (H + 2 * Kh) * D, dtype=BF16, device="cuda")
    metas, graphs, outs = [], [], []
    side = torch.cuda.Stream()
    for g in range(2):
        meta = make_meta([(0, 0, 1), (1, 0, 1), (2, 0, 1)])
        meta.max_context = 640
        body = lambda meta=meta: ops.attention(ops.rotate_append(x, rotary, meta, a, H), meta, a, H, D ** -0.5, 100 if g else None)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            body()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(body())
        metas.append(meta)
        graphs.append(graph)
    for t in (a.k, a.v):
        t.view(torch.uint8).copy_((b.k if t is a.k else b.v).view(torch.uint8))
    for s, t in zip(a.scales, b.scales):
        s.copy_(t)
    gen = torch.Generator().manual_seed(5)
    for i in range(8):
        pos = [64 * i + 5, 63 + i, 600 + i]
        metas[i % 2].tok_pos.copy_(torch.tensor(pos, dtype=torch.int32))
        metas[i % 2].tok_slot.copy_(torch.tensor([3, 1, i % 2 * 2], dtype=torch.int32))
        x.copy_((torch.randn(x.shape, generator=gen) * 2.0 ** (i - 3)).to(BF16))
        graphs[i % 2].replay()
        eager = make_meta([(3, pos[0], 1), (1, pos[1], 1), (i % 2 * 2, pos[2], 1)])
        eager.max_context = 640
        want = ops.attention(ops.rotate_append(x, rotary, eager, b, H), eager, b, H, D ** -0.5, 100 if i % 2 else None)
        assert torch.equal(outs[i % 2], want), i
        assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.scales[1], b.scales[1])


def test_rows_that_do_not_begin_on_16_bytes(ops):
    H, Kh, D = 4, 2, 64
    seqs = [(0, 40, 30), (1, 0, 1)]
    view, cpu = make_view(7, Kh, 64, D, 2, 2, seed=13)
    other, _ = make_view(7, Kh, 64, D, 2, 2, seed=13)
    wide = rows_of(seqs, (H + 2 * Kh) * D + 8, seed=5).cuda()
    rotary = (frequencies(D).cuda(), False, D)
    q = ops.rotate_append(wide[:, 1:-7], rotary, make_meta(seqs), view, H)
    want = ops.rotate_append(wide[:, 1:-7].contiguous(), rotary, make_meta(seqs), other, H)
    # (two kernels: products and sums of float32 pairs, 2^-22 of the row's size apart, may round to different sides in bfloat16)
    assert torch.all((q.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -20 * want.float().abs().max())
    assert same_codes(view.v, other.v.cpu()) and torch.equal(view.scales[1], other.scales[1])
    # queries that begin elsewhere
    one = [(0, 60, 1)]
    base = rows_of(one, H * D + 8, seed=6).cuda()
    x = base.view(-1)[1:1 + H * D].view(1, H, D)
    a = ops.attention(x, make_meta(one), view, H, 0.1, None)
    b = ops.attention(x.clone(), make_meta(one), view, H, 0.1, None)
    assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.float().abs().max())


def test_masked_places_may_hold_anything(ops):
    """NaN codes behind a sequence's end and before its window, pages that were given back (-1 places), scales that are NaN there."""
    H, Kh, D, page = 8, 2, 128, 64
    for seqs, window, keep in (([(0, 130, 1)], 0, 0), ([(0, 250, 1)], 60, 0), ([(0, 250, 4)], 60, 10), ([(0, 250, 1)], 100, 5)):
        view, cpu = make_view(12, Kh, page, D, 2, 5, seed=14)
        start, n = seqs[0][1], seqs[0][2]
        first = max(0, start - window + 1) if window else 0
        for pool in (view.k, view.v, cpu.k, cpu.v):
            codes = pool.view(torch.uint8)
            for pos in list(range(start + n, 5 * page)) + [p for p in range(first) if p >= keep]:
                codes[int(cpu.page_table[0, pos // page]), :, pos % page] = 0x7f
        for i in range(5):                       # whole pages that no row sees
            if window and (i + 1) * page <= first and i * page >= keep:
                view.page_table[0, i] = -1
        q = rows_of(seqs, H * D, seed=7).view(-1, H, D)
        got = ops.attention(q.cuda(), make_meta(seqs), view, H, D ** -0.5, window, keep_first=keep).cpu().to(F64)
        # (a row may see a window's older keys that the later rows do not: only what no row sees holds NaN)
        want, size = plain.attend(cpu, 0, start, q, D ** -0.5, window, None, 0.0, keep)
        assert torch.isfinite(got).all()
        assert torch.all((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size)


def test_blocks_of_very_different_size(ops):
    """Scales from 2^-60 to 2^100 side by side: the sums stay finite and right where large values have no weight, and where they have."""
    H, Kh, D, page = 4, 1, 128, 64
    view, cpu = make_view(8, Kh, page, D, 1, 8, seed=15)
    for i, e in enumerate((0, 100, -60, 3, 90, -40, 1, -7)):
        for v in (view, cpu):
            v.scales[1][int(cpu.page_table[0, i])] = 2.0 ** e
    for v in (view, cpu):
        v.scales[0].fill_(2.0 ** -9)
    q = rows_of([(0, 511, 1)], H * D, seed=8).view(1, H, D)
    got = ops.attention(q.cuda(), make_meta([(0, 511, 1)]), view, H, D ** -0.5, None).cpu().to(F64)
    want, size = plain.attend(cpu, 0, 511, q, D ** -0.5)
    assert torch.all((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size)
    # only the small blocks are seen
    got = ops.attention(q.cuda(), make_meta([(0, 511, 1)]), view, H, D ** -0.5, 100).cpu().to(F64)
    want, size = plain.attend(cpu, 0, 511, q, D ** -0.5, 100)
    assert torch.all((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size)


def test_many_sequences_of_unequal_lengths(ops):
    """More pairs than blocks: all tiles are dealt out, pairs are shared by blocks and joined again; steps of one and of several tokens."""
    for H, Kh, D, new in ((32, 8, 128, 1), (16, 16, 64, 1), (8, 2, 128, 5), (7, 1, 64, 4)):
        B, max_pages = 40, 24
        view, cpu = make_view(B * max_pages, Kh, 64, D, B, max_pages, seed=H)
        seqs = [(B - 1 - i, (i * 37 * (1 + i % 5)) % (24 * 64 - new), 1 + i % new) for i in range(B)]
        q = rows_of(seqs, H * D, seed=9).view(-1, H, D)
        got = ops.attention(q.cuda(), make_meta(seqs), view, H, D ** -0.5, None).cpu().to(F64)
        at = 0
        for slot, start, n in seqs:
            want, size = plain.attend(cpu, slot, start, q[at:at + n], D ** -0.5)
            assert torch.all((got[at:at + n] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size), (H, slot)
            at += n


def test_many_short_pairs(ops):
    """Pairs that are one warp's work each: one tile, a few, windows with sinks and first keys that stay; one and two eights of rows; more
    pairs than run at once."""
    for H, Kh, D, new, most, window, sinks, cap, keep in ((16, 16, 128, 1, 60, 0, False, 0.0, 0), (32, 8, 64, 1, 250, 0, True, 0.0, 0),
                                                          (8, 8, 128, 1, 1100, 150, True, 20.0, 70), (16, 8, 64, 5, 200, 0, False, 0.0, 0),
                                                          (32, 8, 128, 4, 300, 90, True, 0.0, 10), (12, 6, 128, 2, 64, 0, False, 5.0, 0)):
        B, max_pages = 100 if most < 500 else 60, -(-(most + new) // 64)
        view, cpu = make_view(B * max_pages, Kh, 64, D, B, max_pages, seed=H + D)
        seqs = [(B - 1 - i, (i * 37 * (1 + i % 5)) % (most + 1 - new), 1 + i % new) for i in range(B)]
        q = rows_of(seqs, H * D, seed=9).view(-1, H, D)
        sink = torch.linspace(-2.0, 3.0, H) if sinks else None
        meta = make_meta(seqs)
        got = ops.attention(q.cuda(), meta, view, H, D ** -0.5, window, sinks=None if sink is None else sink.cuda(), softcap=cap,
                            keep_first=keep).cpu().to(F64)
        assert [v[5] for k, v in meta.extra.items() if k[0] == "attention8"][0] < 0
        at = 0
        for slot, start, n in seqs:
            want, size = plain.attend(cpu, slot, start, q[at:at + n], D ** -0.5, window, sink, cap, keep)
            assert torch.all((got[at:at + n] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size), (H, slot)
            at += n


def test_prompts_through_bfloat16_pages_and_through_codes_are_the_same_attention(ops):
    """The rule between the two is one of speed: rows of a few tokens either way."""
    H, Kh, D = 8, 2, 128
    seqs = [(0, 100, 7), (1, 0, 7), (2, 300, 2)]
    view, _ = make_view(30, Kh, 64, D, 3, 6, seed=16)
    q = rows_of(seqs, H * D, seed=10).view(-1, H, D).cuda()
    a = ops.attention(q, make_meta(seqs), view, H, D ** -0.5, None)
    kept, ops.cache8_rows = ops.cache8_rows, 0
    try:
        b = ops.attention(q, make_meta(seqs), view, H, D ** -0.5, None)
    finally:
        ops.cache8_rows = kept
    assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -6 * float(b.float().abs().max())


def test_verify_of_rows_that_are_part_of_wider_ones_and_of_long_vocabularies(ops):
    case = list(drafts_case(3, 2, 5003, False, 5))
    wide, wide_p = torch.randn(case[0].shape[0], 6001), torch.rand(case[0].shape[0], 5500)
    wide[:, 3:5006], wide_p[:, 1:5004] = case[0], case[6]
    a, t = ops.verify_drafts(wide.cuda()[:, 3:5006], case[1].cuda(), case[2].cuda(), case[3].cuda(), case[4].cuda(), 2,
                             draft_probs=wide_p.cuda()[:, 1:5004])
    assert (a.tolist(), t.tolist()) == plain.verify(*case)
    case = drafts_case(2, 2, 300001, False, 6)
    assert verified(ops, *case) == plain.verify(*case)
    # a draft on the very border of acceptance: float32 sums leave it open
    z = torch.randn(2, 40000, generator=torch.Generator().manual_seed(2)) * 2
    p = torch.softmax(z[0].double(), 0)
    top = int(p.argmax())
    for d in (-3, -1, 0, 1, 3):
        u = torch.full((2, 2), float(p[top]) * (1 + d * 2.0 ** -22))
        case = (z, torch.tensor([0, 2], dtype=torch.int32), torch.tensor([top, 0], dtype=torch.int32), torch.ones(1), u, 1, None)
        assert verified(ops, *case) == plain.verify(*case), d


def test_verify_captured_twice_and_replayed_in_turn(ops):
    cases = [drafts_case(4, 3, 3000, True, s, ragged=False) for s in (1, 2)]
    held = [[t.cuda() for t in c[:5]] for c in cases]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for h in held:
        ops.verify_drafts(*h, 3)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.verify_drafts(*h, 3))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c, (a, t) in zip(cases, outs):
            assert (a.tolist(), t.tolist()) == plain.verify(*c)


# ---- the engine
def test_a_run_of_them_together():
    """A model whose heads the fast kernels take: prompts, drafted steps, decode steps (captured), over a cache of 8 bits.  Logits are
    near the bfloat16 cache's (a tenth of the largest: what codes of four digits move, see the CPU tests); the tokens that drafted steps
    give are the arg-max of the logits that plain steps over the same cache give, but for near ties."""
    from rbitnet_b200 import Engine, StepEntry
    cfg = dict(architectures=["LlamaForCausalLM"], num_hidden_layers=2, hidden_size=512, num_attention_heads=8, num_key_value_heads=2,
               head_dim=64, intermediate_size=1024, vocab_size=1000, rope_theta=10000.0, rms_norm_eps=1e-5, max_position_embeddings=1024,
               tie_word_embeddings=False, hidden_act="silu")
    kw = dict(seed=5, dtype="bfloat16", max_tokens=8192, max_batch=8)
    full, half = Engine.from_random(cfg, **kw), Engine.from_random(cfg, cache_dtype="float8_e4m3", **kw)
    assert half.cache.bytes() < 0.52 * full.cache.bytes() and "cache=" in half.model_summary()
    g = torch.Generator().manual_seed(1)
    ps = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (300, 64, 63, 1, 130)]
    rows = []
    for eng in (full, half):
        slots = [eng.new_sequence() for _ in ps]
        out = [eng.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, ps)])]
        for i in range(70):
            out.append(eng.step([StepEntry(s, [(7 * i + j) % 1000], [0]) for j, s in enumerate(slots)], captured=i % 2 == 0))
        out.append(eng.step([StepEntry(s, [3, 4, 5 + j, 6], [0, 3]) for j, s in enumerate(slots)]))
        rows.append(torch.cat(out))
        for s in slots:
            eng.end_sequence(s)
        eng.ops.check_errors()
    size = float(rows[0].abs().max())
    assert 0 < float((rows[0] - rows[1]).abs().max()) <= 0.1 * size
    again = [p + p[-40:] for p in ps]
    plainly = half.generate(again, max_tokens=40, temperature=0.0, stop_ids=[])
    drafted = half.generate(again, max_tokens=40, temperature=0.0, stop_ids=[], draft_tokens=4)
    assert half.last_stats["drafted_tokens"] > 0 and half.last_stats["steps"] <= 40
    for p, a, b in zip(again, plainly, drafted):
        assert len(b.tokens) == 40
        if a.tokens == b.tokens:
            continue
        at = next(i for i in range(40) if a.tokens[i] != b.tokens[i])
        slot = half.new_sequence()
        z = half.step([StepEntry(slot, p + a.tokens[:at], [len(p) + at - 1])])[0]
        half.end_sequence(slot)
        # a near tie: two logits, each off by the band of two layers in bfloat16 (helpers.bf16_rtol: 1.7 % of the largest)
        assert abs(float(z[a.tokens[at]] - z[b.tokens[at]])) <= 2 * bf16_rtol(2) * float(z.abs().max()), at
    sampled = half.generate(again, max_tokens=20, temperature=0.8, seed=3, stop_ids=[], draft_tokens=4)
    assert [len(r.tokens) for r in sampled] == [20] * len(ps)
    assert [r.tokens for r in half.generate(again, max_tokens=20, temperature=0.8, seed=3, stop_ids=[], draft_tokens=4)] == [r.tokens for r in sampled]


def test_the_checked_build_sees_addresses_outside_the_8_bit_cache():
    """In a process of its own with RBITNET_CHECKED: a slot and a position outside are recorded, not read or written."""
    import os
    import subprocess
    import sys
    code = '''
import torch, sys
sys.path[:0] = ["tests"]
from test_gpu_cache8 import make_view, make_meta, rows_of, BF16
from rbitnet_b200.kernels.ops import CudaOps
from rbitnet_b200.kernels.lib import KernelError
ops = CudaOps(BF16)
view, _ = make_view(4, 2, 64, 128, 2, 2)
for bad in (lambda m: ops.rotate_append(rows_of([(0, 0, 1)], 8 * 128).cuda(), None, m, view, 4),
            lambda m: ops.attention(rows_of([(0, 0, 1)], 4 * 128).view(1, 4, 128).cuda(), m, view, 4, 0.1, None)):
    meta = make_meta([(0, 64 * 2, 1)])
    bad(meta)
    torch.cuda.synchronize()
    try:
        ops.check_errors()
        print("not seen")
    except KernelError as e:
        assert "checked build" in str(e), e
        print("seen")
'''
    env = dict(os.environ, RBITNET_CHECKED="1")
    out = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), env=env,
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and out.stdout.split() == ["seen", "seen"], out.stdout + out.stderr


@pytest.mark.parametrize("H,Kh,D,B,start,n,window,keep", [(8, 2, 128, 1, 130, 4, 0, 0), (8, 2, 128, 1, 250, 5, 60, 10), (16, 4, 64, 1, 61, 7, 0, 0),
                                                          (8, 8, 128, 100, 61, 5, 0, 0), (8, 2, 64, 60, 700, 8, 0, 0)])
def test_a_later_token_of_the_step_may_hold_nan(ops, H, Kh, D, B, start, n, window, keep):
    """NaN among values that only some of a step's tokens see: a drafted token's, and a window's oldest; just the sums of the rows that see
    them are NaN (one sequence: a cluster's parts; many: a warp a pair, or tiles dealt out)."""
    page = 64
    max_pages = -(-(start + n) // page)
    view, cpu = make_view(B * max_pages, Kh, page, D, B, max_pages, seed=D + n)
    places = [(start + 2, 0, 5), (start + n - 1, Kh - 1, D - 1)] + ([(start - window + 2, Kh - 1, 7)] if window else [])
    for slot in range(B):
        for pos, kvh, d in places:
            for v in (view, cpu):
                v.v.view(torch.uint8)[int(cpu.page_table[slot, pos // page]), kvh, pos % page, d] = 0x7f
                v.k.view(torch.uint8)[int(cpu.page_table[slot, (start + 3) // page]), 0, (start + 3) % page, 1] = 0xff
    seqs = [(slot, start, n) for slot in range(B)]
    q = rows_of(seqs, H * D, seed=7).view(-1, H, D)
    got = ops.attention(q.cuda(), make_meta(seqs), view, H, D ** -0.5, window, keep_first=keep).cpu().to(F64).view(B, n, H * D)
    some = 0
    for slot in (0, B // 2, B - 1):
        for i in range(n):
            row = q[slot * n + i][None]
            want, size = plain.attend(cpu, slot, start + i, row, D ** -0.5, window, None, 0.0, keep)
            nan = want[0].isnan()
            some += int(nan.sum())
            assert torch.equal(got[slot, i].isnan(), nan), (slot, i)
            fine = ~nan
            assert torch.all((got[slot, i] - want[0]).abs()[fine] <= (2.0 ** -8 * want[0].abs() + (2.0 ** -8 + 2.0 ** -14) * size[0])[fine])
            assert i > 1 or not nan[5]
    assert some

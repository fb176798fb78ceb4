"""The 8-bit cache's kernels at their edges, against plain 64-bit torch or against themselves; tolerances as in test_gpu_cache8."""
import math

import pytest
import torch

import plain_cache8 as plain
from rbitnet_b200.cache import CacheLayerView
from test_gpu_cache8 import BF16, F64, both_views, frequencies, make_meta, make_view, rows_of, same_codes

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


def uneven_view(B, Kh, D, tiles, seed, step=8, far=40):
    """A view whose tiles' values are of very different scales (2^-far .. 2^far, `step` apart), and whose keys weigh them against it: a
    query with 5 as its first value (score scale 0.2) gives a tile of scale 2^e about 2^-e of the weight, so that all tiles count."""
    view, cpu = make_view(B * tiles, Kh, 64, D, B, tiles, seed=seed)
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(-far // step, far // step + 1, (B * tiles, Kh, 1), generator=g) * step
    codes = (torch.randn(B * tiles, Kh, 64, D, generator=g) * 4).to(torch.float8_e4m3fn)
    codes[..., 0] = (-e.expand(-1, -1, 64) * (math.log(2.0) / 0.125)).to(torch.float8_e4m3fn)
    for v in (view, cpu):
        v.k.view(torch.uint8).copy_(codes.view(torch.uint8))
        v.scales[0].fill_(0.125)
        v.scales[1].copy_(torch.exp2(e.float()))
    return view, cpu


def attended_as_plain(ops, view, cpu, seqs, q, scale, window=0, sink=None, cap=0.0, keep=0, cut=None):
    """The attention of a step beside the plain form's.  ``cut``: "cluster", "dealt" or "alone", the way that the step has to go."""
    H, meta = q.shape[1], make_meta(seqs)
    got = ops.attention(q.cuda(), meta, view, H, scale, window, sinks=None if sink is None else sink.cuda(), softcap=cap, keep_first=keep)
    if cut is not None:
        parts = [v[5] for k, v in meta.extra.items() if k[0] == "attention8"][0]
        assert cut == ("cluster" if parts > 0 else "dealt" if parts == 0 else "alone"), parts
    got, at = got.cpu().to(F64), 0
    for slot, start, n in seqs:
        want, size = plain.attend(cpu, slot, start, q[at:at + n], scale, window, sink, cap, keep)
        off = (got[at:at + n] - want).abs()
        assert torch.all(off <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size), (slot, float((off / size).max()))
        at += n


CUTS = [
    # heads, kv heads, head size, sequences, positions at most, new tokens at most, the way that such a step goes
    (4, 1, 128, 1, 8000, 1, "cluster"), (8, 2, 64, 2, 5000, 1, "cluster"), (16, 1, 128, 2, 6000, 1, "cluster"), (20, 1, 64, 1, 4096, 1, "cluster"),
    (4, 1, 128, 2, 6000, 5, "cluster"), (32, 1, 128, 1, 3000, 2, "cluster"),
    (8, 4, 128, 60, 1500, 1, "dealt"), (16, 4, 64, 100, 1500, 1, "dealt"), (16, 4, 128, 60, 1500, 2, "dealt"), (8, 4, 64, 100, 1500, 4, "dealt"),
    (16, 4, 128, 60, 1500, 4, "dealt"), (16, 4, 64, 60, 1500, 4, "dealt"), (16, 4, 128, 60, 1500, 5, "dealt"), (16, 4, 64, 60, 1500, 6, "dealt"),
    (16, 4, 128, 60, 1500, 8, "dealt"), (16, 4, 64, 60, 1500, 8, "dealt"), (16, 4, 128, 60, 1500, 16, "dealt"), (24, 1, 128, 200, 600, 1, "dealt"),
    (8, 8, 128, 100, 180, 1, "alone"), (16, 8, 64, 100, 180, 5, "alone"), (24, 8, 128, 100, 120, 3, "alone"),
]


def a_step(B, most, new):
    return [(B - 1 - i, (i * 97 * (1 + i % 5)) % (most + 1 - new) if i else most - new, 1 + (i + new - 1) % new) for i in range(B)]


@pytest.mark.parametrize("H,Kh,D,B,most,new,cut", CUTS)
def test_weights_and_scales_of_very_different_size(ops, H, Kh, D, B, most, new, cut):
    """What counts in a sum is a weight times its values' scale: small weights of large values, and all of them where a sink holds most
    of the weight, are kept as they are where weights and scales are near one another."""
    view, cpu = uneven_view(B, Kh, D, -(-most // 64), seed=H + D + new)
    seqs = a_step(B, most, new)
    q = rows_of(seqs, H * D, seed=5).view(-1, H, D)
    q[..., 0] = 5.0
    attended_as_plain(ops, view, cpu, seqs, q, 0.2, cut=cut)
    sink = torch.linspace(-3.0, 40.0, H)                     # (weights of 2^-58 x 2^-40 and some more: float32 numbers)
    attended_as_plain(ops, view, cpu, seqs, q, 0.2, sink=sink, cut=cut)


@pytest.mark.parametrize("H,Kh,D,B,most,new,cut", CUTS)
def test_a_first_token_that_takes_the_weight_and_holds_nothing(ops, H, Kh, D, B, most, new, cut):
    """Position 0 weighs e^14 times as much as others, and its values are zeros: the result is the others', each at 2^-20 of the largest weight
    (e^14 = 2^20.2: rounded to float16 around a largest of 2^7 .. 2^15 that is 2^-13.2 or more, of steps of 2^-24: 2^-11.8 of a weight)."""
    view, cpu = make_view(B * -(-most // 64), Kh, 64, D, B, -(-most // 64), seed=D + new)
    g = torch.Generator().manual_seed(1)
    codes = (torch.randn(view.k.shape, generator=g) * 4).to(torch.float8_e4m3fn)
    codes[..., 0] = 0
    codes = codes.view(torch.uint8)
    for slot in range(B):
        page = int(cpu.page_table[slot, 0])
        codes[page, :, 0] = 0
        codes[page, :, 0, 0] = int(torch.tensor(112.0).to(torch.float8_e4m3fn).view(torch.uint8))         # 14 / 0.125
        for v in (view, cpu):
            v.v.view(torch.uint8)[page, :, 0] = 0
    for v in (view, cpu):
        v.k.view(torch.uint8).copy_(codes)
        v.scales[0].fill_(0.125)
        v.scales[1].fill_(0.125)
    seqs = [(s, max(p, 1), n) for s, p, n in a_step(B, most, new)]
    q = rows_of(seqs, H * D, seed=6).view(-1, H, D) * 0.25
    q[..., 0] = 5.0
    attended_as_plain(ops, view, cpu, seqs, q, 0.2, cut=cut)


def pairs_at_a_border(freq, positions, count):
    """(position, x0, x1): bfloat16 pairs whose turn by position * freq has its larger value within 2^-23.5 of itself of 448 * 2^-8 and not
    within 2^-36 (what float64 may be off), and the other below nine tenths of it."""
    border, found = 448.0 * 2.0 ** -8, []
    x0 = (torch.arange(128, 256).to(F64)[None] * torch.exp2(torch.arange(-11.0, -5.0).to(F64))[:, None]).view(-1)
    x0 = torch.cat([x0, -x0])
    for pos in positions:
        angle = torch.tensor(float(pos), dtype=F64) * float(freq)
        c, s = float(angle.cos()), float(angle.sin())
        if min(abs(c), abs(s)) < 0.05:
            continue
        for sign in (1.0, -1.0):
            x1 = ((x0 * c - sign * border) / s).to(BF16).to(F64)
            y, other = x0 * c - x1 * s, x0 * s + x1 * c
            off = (y.abs() / border - 1).abs()
            for i in ((off < 2.0 ** -23.5) & (off > 2.0 ** -36) & (other.abs() < 0.9 * border)).nonzero()[:, 0].tolist():
                found.append((pos, float(x0[i]), float(x1[i])))
        if len(found) >= count:
            break
    return found[:count]


@pytest.mark.parametrize("D,rot,inter,new", [(128, 128, False, 1), (64, 64, True, 1), (128, 128, True, 2), (64, 64, False, 2), (256, 256, False, 2),
                                             (128, 32, False, 1), (10, 10, True, 2)])
def test_the_scale_of_keys_is_that_of_the_exact_rotation(ops, D, rot, inter, new):
    """Keys whose largest value lies nearer to a border of scales than float32 sines are exact, on either side of it."""
    Kh, B = 2, 96
    freq = frequencies(rot)
    which = rot // 2 - 1 if rot < 16 else 3                    # the pair that turns
    at = (2 * which, 2 * which + 1) if inter else (which, which + rot // 2)
    found = pairs_at_a_border(float(freq[which]), (p for p in range(1, 400000, 3) if p % 64), B)
    assert len(found) == B
    page, codes = 64, torch.zeros(B, Kh, 64, D).to(torch.float8_e4m3fn)
    scales = torch.full((B, Kh, 1), 2.0 ** -60)
    table = torch.arange(B, dtype=torch.int32)[:, None].expand(B, 1 + max(p for p, _, _ in found) // page).contiguous()
    view, cpu = both_views([codes, codes], [scales, scales], table, page)
    seqs = [(i, p + 1 - new, new) for i, (p, _, _) in enumerate(found)]
    x = torch.zeros(B, new, 3 * Kh, D)
    for i, (_, a, b) in enumerate(found):
        x[i, -1, Kh, at[0]], x[i, -1, Kh, at[1]] = a, b        # (and the other kv head's the other way)
        x[i, -1, Kh + 1, at[0]], x[i, -1, Kh + 1, at[1]] = -a, -b
    x = x.to(BF16).view(B * new, 3 * Kh * D)
    ops.rotate_append(x.cuda(), (freq.cuda(), inter, rot), make_meta(seqs), view, Kh)
    rows = x.to(F64).view(B, new, 3 * Kh, D)
    for i, start, _ in seqs:
        t = plain.turned(rows[i][:, Kh:2 * Kh], torch.arange(start, start + new), freq, rot, inter)
        plain.append(cpu, i, start, t, rows[i][:, 2 * Kh:])
    assert set(cpu.scales[0].view(-1).tolist()) == {2.0 ** -8, 2.0 ** -7}
    assert torch.equal(view.scales[0].cpu(), cpu.scales[0]) and same_codes(view.k, cpu.k)


@pytest.mark.parametrize("new", [1, 4, 100])
def test_sequences_without_tokens_in_a_step(ops, new):
    """They change nothing for the others: a few rows, and many."""
    H, Kh, D = 8, 2, 128
    rotary = (frequencies(D).cuda(), False, D)
    x = rows_of([(0, 0, 2 * new)], (H + 2 * Kh) * D, seed=2).cuda()
    results = []
    for seqs in ([(0, 60, new), (2, 3, new)], [(1, 0, 0), (0, 60, new), (3, 64, 0), (2, 3, new)]):
        view, _ = make_view(12, Kh, 64, D, 4, 3, seed=4)
        meta = make_meta(seqs)
        q = ops.rotate_append(x, rotary, meta, view, H)
        results.append((q, ops.attention(q, meta, view, H, 0.1, None), view.k.view(torch.uint8), view.v.view(torch.uint8), *view.scales))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    meta = make_meta([(1, 0, 0), (0, 70, 0)])
    q = ops.rotate_append(x[:0], rotary, meta, view, H)
    assert ops.attention(q, meta, view, H, 0.1, None).shape == (0, H * D)


# ---- every way that a step is cut, with everything that a row may be asked for: eights of rows 1 to 4, both head sizes
OPTIONS = [
    # heads, kv heads, head size, sequences, positions at most, new tokens at most, window, sinks, cap, first keys that stay, the way it goes
    (16, 4, 128, 60, 1500, 2, 0, True, 0.0, 0, "dealt"), (16, 4, 128, 60, 1500, 4, 700, False, 0.0, 100, "dealt"),
    (16, 4, 128, 60, 1500, 5, 0, True, 15.0, 0, "dealt"), (16, 4, 128, 60, 1500, 6, 650, True, 0.0, 0, "dealt"),
    (16, 4, 128, 60, 1500, 8, 900, True, 20.0, 70, "dealt"), (16, 4, 128, 60, 1500, 16, 0, False, 0.0, 0, "dealt"),
    (16, 4, 64, 60, 1500, 4, 0, True, 0.0, 0, "dealt"), (16, 4, 64, 60, 1500, 6, 700, False, 10.0, 3, "dealt"),
    (16, 4, 64, 60, 1500, 8, 800, True, 0.0, 65, "dealt"), (24, 1, 128, 200, 600, 1, 300, True, 0.0, 64, "dealt"),
    (28, 1, 64, 250, 600, 2, 0, True, 5.0, 0, "dealt"), (8, 4, 128, 60, 1500, 1, 900, True, 12.0, 100, "dealt"),
    (16, 2, 128, 3, 5000, 2, 0, True, 0.0, 0, "cluster"), (16, 2, 64, 3, 5000, 3, 3000, True, 9.0, 100, "cluster"),
    (16, 2, 128, 3, 5000, 4, 2500, False, 0.0, 10, "cluster"), (8, 2, 128, 3, 4000, 1, 2000, True, 0.0, 100, "cluster"),
    (16, 8, 128, 100, 180, 3, 100, True, 8.0, 5, "alone"), (16, 8, 64, 100, 180, 8, 70, True, 0.0, 66, "alone"),
]


@pytest.mark.parametrize("H,Kh,D,B,most,new,window,sinks,cap,keep,cut", OPTIONS)
def test_options_however_a_step_is_cut(ops, H, Kh, D, B, most, new, window, sinks, cap, keep, cut):
    tiles = -(-most // 64)
    view, cpu = make_view(B * tiles, Kh, 64, D, B, tiles, seed=H + D + new)
    seqs = a_step(B, most, new)
    q = rows_of(seqs, H * D, seed=8).view(-1, H, D)
    attended_as_plain(ops, view, cpu, seqs, q, D ** -0.5, window, torch.linspace(-2.0, 3.0, H) if sinks else None, cap, keep, cut)


@pytest.mark.parametrize("H,Kh,D,B,most,new,window,sinks,cap,keep,cut", [o for o in OPTIONS if o[5] > 1])
def test_nan_that_later_tokens_see_however_a_step_is_cut(ops, H, Kh, D, B, most, new, window, sinks, cap, keep, cut):
    """NaN among the values of a step's later tokens and of a window's oldest: in the sums of the rows that see them, and in no other's."""
    tiles = -(-most // 64)
    view, cpu = make_view(B * tiles, Kh, 64, D, B, tiles, seed=H + D + new)
    seqs = a_step(B, most, new)
    for slot, start, n in seqs:
        places = [(start + n - 1, 0, D - 1), (start + n // 2, Kh - 1, 5)]
        if window and start + 1 - window >= keep:
            places.append((start + 1 - window, Kh - 1, 7))     # the first token's oldest key, which the second does not see
        for pos, kvh, d in places:
            for v in (view, cpu):
                v.v.view(torch.uint8)[int(cpu.page_table[slot, pos // 64]), kvh, pos % 64, d] = 0x7f
    q = rows_of(seqs, H * D, seed=8).view(-1, H, D)
    meta, sink = make_meta(seqs), torch.linspace(-2.0, 3.0, H) if sinks else None
    got = ops.attention(q.cuda(), meta, view, H, D ** -0.5, window, sinks=None if sink is None else sink.cuda(), softcap=cap, keep_first=keep)
    parts = [v[5] for k, v in meta.extra.items() if k[0] == "attention8"][0]
    assert cut == ("cluster" if parts > 0 else "dealt" if parts == 0 else "alone")
    got, at = got.cpu().to(F64), 0
    for slot, start, n in seqs:
        for i in range(n):
            # (a row at a time: the plain form multiplies what one of its rows sees with all rows' weights)
            want, size = plain.attend(cpu, slot, start + i, q[at + i:at + i + 1], D ** -0.5, window, sink, cap, keep)
            nan = want[0].isnan()
            assert torch.equal(got[at + i].isnan(), nan), (slot, i)
            off = (got[at + i] - want[0]).abs()[~nan]
            assert torch.all(off <= (2.0 ** -8 * want[0].abs() + (2.0 ** -8 + 2.0 ** -14) * size[0])[~nan]), (slot, i)
        at += n


@pytest.mark.parametrize("page,D,seqs,window", [
    (128, 128, [(0, 200, 1), (1, 30, 1)], 0), (128, 64, [(0, 600, 1), (1, 30, 1)], 64), (256, 128, [(0, 300, 4), (1, 130, 2)], 100),
    (128, 128, [(0, 150, 40), (1, 260, 60)], 0), (128, 80, [(0, 200, 1), (1, 30, 1)], 0), (256, 80, [(0, 300, 3), (1, 130, 20)], 90),
])
def test_scales_of_blocks_that_no_row_sees_may_be_nan(ops, page, D, seqs, window):
    """Behind a sequence's end, and before its window (where steps of many rows read whole pages, only pages before the window)."""
    H, Kh, max_pages = 8, 2, -(-700 // page)
    view, cpu = make_view(2 * max_pages, Kh, page, D, 2, max_pages, seed=page + D)
    whole = max(n for _, _, n in seqs) * H // Kh > 64 or D == 80 and max(n for _, _, n in seqs) > 1
    for slot, start, n in seqs:
        first = max(0, start - window + 1) if window else 0
        first -= first % (page if whole else 64)
        for block in range(max_pages * page // 64):
            if block * 64 >= start + n or block * 64 + 64 <= first:
                p, b = int(cpu.page_table[slot, block * 64 // page]), block % (page // 64)
                for v in (view, cpu):
                    for s in v.scales:
                        s[p, :, b] = math.nan
    q = rows_of(seqs, H * D, seed=9).view(-1, H, D)
    got, at = ops.attention(q.cuda(), make_meta(seqs), view, H, D ** -0.5, window).cpu().to(F64), 0
    for s in cpu.scales:
        s.nan_to_num_(0.0)                       # (the plain form multiplies them with weights of zero)
    for slot, start, n in seqs:
        want, size = plain.attend(cpu, slot, start, q[at:at + n], D ** -0.5, window)
        assert torch.all((got[at:at + n] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size), slot
        at += n


@pytest.mark.parametrize("H,Kh,D,B,most,new,cut", CUTS + [(4, 2, 80, 2, 100, 1, None)])
def test_sinks_that_are_no_numbers(ops, H, Kh, D, B, most, new, cut):
    """Minus infinity is no sink at all; NaN makes its head's rows NaN, and no other's."""
    tiles = -(-most // 64)
    view, cpu = make_view(B * tiles, Kh, 64, D, B, tiles, seed=D)
    seqs = a_step(B, most, new)
    q = rows_of(seqs, H * D, seed=8).view(-1, H, D)
    meta = make_meta(seqs)
    sink = torch.linspace(-1.0, 1.0, H)
    sink[1] = -math.inf
    bare = torch.linspace(-1.0, 1.0, H)
    bare[1] = -1e30
    attend = lambda s: ops.attention(q.cuda(), meta, view, H, D ** -0.5, None, sinks=s.cuda()).view(-1, H, D)
    want = attend(bare)
    assert torch.equal(attend(sink), want) and torch.isfinite(want).all()
    sink[2] = math.nan
    got = attend(sink)
    assert got[:, 2].isnan().all()
    rest = [h for h in range(H) if h != 2]
    assert torch.equal(got[:, rest], want[:, rest])

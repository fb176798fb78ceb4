"""The cache held in 8 bits and drafted steps without a GPU: the plain forms against themselves, the host's part, the refusals."""
import math
from dataclasses import replace

import pytest
import torch

import plain_cache8 as plain
from ops_cache8 import TorchOps8
from tiny import TINY_A, TINY_B, prompts
from rbitnet_b200 import Engine, StepEntry
from rbitnet_b200.cache import CacheLayerView, SequenceCache
from rbitnet_b200.config import config_from_dict
from rbitnet_b200.engine.generate import Lookup
from rbitnet_b200.engine.step import SeqChunk, build_meta
from rbitnet_b200.kernels.lib import KernelError
from rbitnet_b200.kernels.ops import CudaOps
from rbitnet_b200.parts.base import CacheNeed

E4M3 = torch.float8_e4m3fn


def engine(config, dtype="float32", seed=3, **kw):
    return Engine.from_random(config, seed=seed, dtype=dtype, ops=TorchOps8({"float32": torch.float32, "bfloat16": torch.bfloat16}[dtype]), **kw)


# ---- the plain form itself
def test_plain_codes_are_e4m3():
    """Against the type's own conversion, over its range and its smallest steps; ties go to the even code."""
    x = torch.cat([torch.linspace(-448, 448, 4001), torch.linspace(-0.05, 0.05, 4001), torch.exp2(torch.linspace(-12, 8.5, 999))]).double()
    assert torch.equal(plain.to_e4m3(x), x.to(torch.float32).to(E4M3).double())
    assert plain.to_e4m3(torch.tensor([17.0, 19.0, 1.0625, 3 * 2.0 ** -10, 500.0, math.nan]).double()).tolist()[:5] == [16.0, 20.0, 1.0, 2.0 ** -8, 448.0]


def test_plain_scale_is_the_least_power_of_two_that_holds_the_value():
    for amax in (0.0, 1e-30, 1.0, 447.9, 448.0, 448.1, 896.0, 3e38, math.inf):
        s = plain.scale_for(amax)
        assert math.log2(s) == round(math.log2(s)) and 2.0 ** -60 <= s <= 2.0 ** 119
        assert amax <= 448 * s or s == 2.0 ** 119
        assert s == 2.0 ** -60 or amax > 448 * s / 2


def test_a_key_s_distance_to_what_is_stored():
    """Half a step of e4m3: 2^-4 of the value, 2^-10 of the scale near zero; in a block whose scale grew, twice that near zero."""
    view = CacheLayerView(torch.zeros(1, 1, 64, 32).to(E4M3), torch.zeros(1, 1, 64, 32).to(E4M3), torch.zeros(1, 1, dtype=torch.int32), 1, 64,
                          1, 32, True, 0, (), (torch.zeros(1, 1, 1), torch.zeros(1, 1, 1)))
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(64, 1, 32, generator=g).double() * torch.exp2(torch.linspace(-6, 6, 64))[:, None, None]
    for pos in range(64):
        plain.append(view, 0, pos, rows[pos:pos + 1], rows[pos:pos + 1])
    got = plain.values(view, 0, 64, 0)[0]
    scale = float(view.scales[0][0, 0, 0])
    assert scale == plain.scale_for(float(rows.abs().max()))
    assert torch.all((got - rows[:, 0]).abs() <= torch.maximum(2.0 ** -4 * rows[:, 0].abs(), torch.tensor(2.0 ** -9 * scale)))


def test_plain_verify_keeps_the_target_s_distribution():
    """Whatever the drafter's probabilities: the first token of a step is distributed as the target's row, within five deviations."""
    V, n = 6, 4000
    g = torch.Generator().manual_seed(1)
    z = torch.randn(2, V, generator=g)
    p = torch.softmax(z[0].double() / 0.8, 0)
    for probs in (None, torch.softmax(torch.randn(2, V, generator=g), dim=1)):
        seen = torch.zeros(V)
        for i in range(n):
            u = torch.rand(2, 2, generator=g)
            d = int(torch.multinomial(probs[0], 1, generator=g)) if probs is not None else 2
            _, tokens = plain.verify(z, [0, 2], [d, -1], [0.8], u, 1, probs)
            seen[tokens[0][0]] += 1
        assert torch.all((seen / n - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n))


# ---- drafts from the sequence itself
def test_lookup_takes_what_followed_the_longest_run():
    look = Lookup([1, 2, 3, 4, 9, 2, 3])
    assert look.propose(4) == [4, 9, 2, 3] and look.propose(2) == [4, 9] and look.propose(0) == []
    look.extend([5, 3])                      # the last one alone: behind the latest 3 before it
    assert look.propose(3) == [5, 3]
    assert Lookup([7]).propose(3) == [] and Lookup([1, 2, 3]).propose(3) == []
    assert Lookup([5, 5]).propose(3) == [5] and Lookup([5, 5, 5]).propose(3) == [5]


@pytest.mark.parametrize("config", [TINY_A, TINY_B])
@pytest.mark.parametrize("most", [1, 3, 7])
def test_greedy_tokens_are_the_same_with_drafts(config, most):
    ps = [p * 3 for p in prompts([4, 7, 1], config["vocab_size"], 5)] + [[5], list(range(20))]
    want = engine(config, max_tokens=2048).generate(ps, max_tokens=14, temperature=0.0, stop_ids=[])
    eng = engine(config, max_tokens=2048)
    seen = []
    got = eng.generate(ps, max_tokens=14, temperature=0.0, stop_ids=[], draft_tokens=most, on_token=lambda r, t: seen.append((r, t)))
    assert [(r.tokens, r.finish_reason) for r in got] == [(r.tokens, r.finish_reason) for r in want]
    assert [[t for r, t in seen if r == i] for i in range(len(ps))] == [r.tokens for r in got]
    assert eng.last_stats["drafted_tokens"] > 0 and eng.live_sequences() == []
    # a stop token in the midst of accepted drafts, and the cache's end
    stop = want[0].tokens[6]
    a = engine(config, max_tokens=2048).generate(ps, max_tokens=14, temperature=0.0, stop_ids=[stop])
    b = engine(config, max_tokens=2048).generate(ps, max_tokens=14, temperature=0.0, stop_ids=[stop], draft_tokens=most)
    assert [(r.tokens, r.finish_reason) for r in a] == [(r.tokens, r.finish_reason) for r in b]
    a = engine(config, max_tokens=2048, max_seq=24).generate(ps, max_tokens=40, temperature=0.0, stop_ids=[])
    b = engine(config, max_tokens=2048, max_seq=24).generate(ps, max_tokens=40, temperature=0.0, stop_ids=[], draft_tokens=most)
    assert [(r.tokens, r.finish_reason) for r in a] == [(r.tokens, r.finish_reason) for r in b]


def test_drafted_requests_at_their_edges():
    eng = engine(TINY_A, max_tokens=512)
    out = eng.generate([[], [1, 2]], max_tokens=0, draft_tokens=2)
    assert [r.finish_reason for r in out] == ["empty", "length"]
    out = eng.generate([[], [1, 2, 1, 2]], max_tokens=1, draft_tokens=2, temperature=0.9)
    assert out[0].finish_reason == "empty" and len(out[1].tokens) == 1
    assert len(eng.generate([[3, 4] * 6], max_tokens=9, temperature=1.0, seed=4, stop_ids=[], draft_tokens=4)[0].tokens) == 9
    with pytest.raises(ValueError, match="negative"):
        eng.generate([[1]], draft_tokens=-1)
    # more requests than fit at once
    eng = engine(TINY_A, max_tokens=3 * 64, max_batch=2)
    ps = [[i, i + 1, i, i + 1] for i in range(5)]
    want = engine(TINY_A, max_tokens=2048).generate(ps, max_tokens=6, temperature=0.0, stop_ids=[])
    assert [r.tokens for r in eng.generate(ps, max_tokens=6, temperature=0.0, stop_ids=[], draft_tokens=3)] == [r.tokens for r in want]


def test_a_step_that_does_not_move_on():
    """The positions behind a sequence's length are written over: two rows, one of them kept, then the rest again."""
    eng = engine(TINY_B, max_tokens=512)
    a, b = eng.new_sequence(), eng.new_sequence()
    ps = prompts([70], TINY_B["vocab_size"], 2)[0]
    eng.step([StepEntry(a, ps[:60]), StepEntry(b, ps[:60])])
    eng.stepper.step([StepEntry(a, [ps[60], 1, 2, 3, 4, 5], [0])], advance=False)
    assert eng.cache.length(a) == 60
    eng.cache.advance(a, 1)
    eng.step([StepEntry(b, [ps[60]], [0])])
    x, y = eng.step([StepEntry(a, ps[61:], [8]), StepEntry(b, ps[61:], [8])])
    # (the row at position 60 comes from a batch of six rows here and of one there: float32 sums of up to 256 terms in another order,
    # 256 * 2^-24 = 1.5e-5 of their size apart)
    assert float((x - y).abs().max()) <= 1e-5 + 2e-5 * float(y.abs().max())


# ---- the cache
def test_pools_scales_and_bytes():
    cache = SequenceCache({0: CacheNeed(2, 32), 1: CacheNeed(2, 32)}, {}, {}, 256, 256, E4M3, "cpu", page_size=128)
    view = cache.view(1)
    assert view.k.dtype == E4M3 and view.k.shape == (2, 2, 128, 32)
    assert [tuple(s.shape) for s in view.scales] == [(2, 2, 2)] * 2 and view.scales[0].dtype == torch.float32
    assert cache.bytes() == 2 * 2 * 2 * 2 * (128 * 32 + 2 * 4)
    assert cache.groups[0].bytes_per_position() == 2 * 2 * 2 * 32 + 1      # and 2 layers x 4 scales of 4 bytes a 64 positions: a half
    assert SequenceCache({0: CacheNeed(2, 32)}, {}, {}, 256, 256, torch.bfloat16, "cpu").view(0).scales == ()
    with pytest.raises(ValueError, match="pages"):
        SequenceCache({0: CacheNeed(2, 32)}, {}, {}, 256, 256, E4M3, "cpu", page_size=96)


@pytest.mark.parametrize("config,page", [(TINY_A, 64), (TINY_B, 16)])
def test_an_engine_with_8_bits_is_near_the_one_without(config, page):
    """Logits within the part that rounding keys and values to 2^-4 of themselves moves (a tenth of the largest logit is far above what
    it does here and far below what a wrong page, scale or position would do), whatever the steps are cut into."""
    ps = prompts([70, 90], config["vocab_size"], 6)
    full = engine(config, "bfloat16", max_tokens=1024, page_size=page)
    half = engine(config, "bfloat16", max_tokens=1024, page_size=page, cache_dtype="float8_e4m3")
    assert half.cache.bytes() < 0.6 * full.cache.bytes()
    out = []
    for eng, cuts in ((full, (90,)), (half, (90,)), (half, (17, 60, 61, 62, 90))):
        slots, last, rows = [eng.new_sequence() for _ in ps], 0, None
        for cut in cuts:
            entries = [StepEntry(s, p[last:cut], [len(p[last:cut]) - 1]) for s, p in zip(slots, ps) if p[last:cut]]
            rows = eng.step(entries)
            last = cut
        out.append(rows[-1].float())
        for s in slots:
            eng.end_sequence(s)
    size = float(out[0].abs().max())
    assert 0 < float((out[1] - out[0]).abs().max()) <= 0.1 * size
    assert float((out[2] - out[1]).abs().max()) <= 0.1 * size


def test_the_command_line(tmp_path, capsys):
    """generate with a cache of 8 bits and drafts: the engine's own results."""
    import json
    from rbitnet_b200 import write_random_model
    from rbitnet_b200.cli import main
    write_random_model(tmp_path / "m", config_from_dict(TINY_B), seed=7)
    argv = ["generate", "--model", str(tmp_path / "m"), "--cache-dtype", "float8_e4m3", "--cache-tokens", "512", "--draft-tokens", "3",
            "--prompt-ids", "1 5 9 1 5 9 1", "--max-tokens", "8", "--temperature", "0"]
    assert main(argv, ops=TorchOps8(torch.bfloat16)) == 0
    got = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    eng = Engine.load_path(tmp_path / "m", dtype="bfloat16", ops=TorchOps8(torch.bfloat16), max_tokens=512, cache_dtype="float8_e4m3")
    want = eng.generate([[1, 5, 9, 1, 5, 9, 1]], max_tokens=8, temperature=0.0, draft_tokens=3)[0]
    assert got == {"tokens": want.tokens, "finish_reason": want.finish_reason, "prompt_tokens": 7}


# ---- refusals
def test_what_is_refused():
    with pytest.raises(ValueError, match="bfloat16 mode"):
        engine(TINY_A, "float32", max_tokens=256, cache_dtype="float8_e4m3")
    with pytest.raises(ValueError, match="cache_dtype"):
        engine(TINY_A, "bfloat16", max_tokens=256, cache_dtype="int8")
    with pytest.raises(ValueError, match="pages"):
        engine(TINY_A, "bfloat16", max_tokens=256, cache_dtype="float8_e4m3", page_size=80)
    from gozotar_tiny import CONFIGS, make_tensors
    name = sorted(CONFIGS)[0]
    with pytest.raises(ValueError, match="compute dtype only"):
        Engine(config_from_dict(CONFIGS[name]), dict(make_tensors(CONFIGS[name], seed=3)), dtype="bfloat16", ops=TorchOps8(torch.bfloat16),
               max_tokens=512, max_seq=128, cache_dtype="float8_e4m3")
    eng = Engine(config_from_dict(CONFIGS[name]), dict(make_tensors(CONFIGS[name], seed=3)), dtype="float32", ops=TorchOps8(torch.float32),
                 max_tokens=512, max_seq=128)
    with pytest.raises(ValueError, match="step back"):
        eng.generate([[1, 2]], draft_tokens=2)


class _NoLibrary:
    """Stands for the kernel library where nothing may be launched."""
    def raw(self, name):
        return lambda *a: 1

    def call(self, name, *a, **kw):
        raise AssertionError(f"{name} was called")


def bare_ops(dtype=torch.bfloat16):
    ops = object.__new__(CudaOps)
    ops.dtype, ops.lib, ops.device, ops.cache8_rows = dtype, _NoLibrary(), torch.device("cpu"), 64
    return ops


def view_of(page=64, D=128, Kh=2, code=E4M3, scale=torch.float32, blocks=1):
    k, v = (torch.zeros(4, Kh, page, D).to(code) for _ in range(2))
    return CacheLayerView(k, v, torch.zeros(2, 2, dtype=torch.int32), 2, page, Kh, D, True, 0, (k, v),
                          tuple(torch.zeros(4, Kh, blocks, dtype=scale) for _ in range(2)))


def meta_of(n):
    import numpy as np
    return build_meta([SeqChunk(0, 0, n, 0)], np.zeros(n, dtype=np.int32), np.zeros(0, dtype=np.int32), "cpu")


def test_kernel_calls_that_are_refused_before_anything_is_launched():
    """(Tensors on the CPU are refused like those of a wrong type or shape.)"""
    rows = torch.zeros(3, 8 * 128, dtype=torch.bfloat16)
    for ops, view, match in ((bare_ops(), view_of(), "CUDA device"), (bare_ops(torch.float32), view_of(), "bfloat16 mode"),
                             (bare_ops(), view_of(page=96), "multiple of 64"), (bare_ops(), view_of(page=128, blocks=1), "scales"),
                             (bare_ops(), view_of(code=torch.bfloat16), "float8"), (bare_ops(), view_of(scale=torch.float64), "float32 scales")):
        with pytest.raises(KernelError, match=match):
            ops.rotate_append(rows, None, meta_of(3), view, 4)
        with pytest.raises(KernelError, match=match):
            ops.attention(rows.view(3, 8, 128), meta_of(3), view, 8, 1.0, None)
    with pytest.raises(KernelError, match="compute dtype"):
        bare_ops().cache_values(CacheLayerView(None, None, None, 1, 64, 1, 8, True, 0), None)
    for bad in ((2, 0, 1), (-1, 0, 1), (0, 3, 3), (0, -1, 2), (0, 0, 129)):
        with pytest.raises(KernelError, match="cache_ranges"):
            bare_ops().cache_ranges(view_of(), [bad])
    z, i, f = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2)
    for args in ((z, i, i, torch.zeros(2), f, 1), (z.double(), i, i, torch.zeros(2), f, 1), (z[0], i, i, torch.zeros(2), f, 1)):
        with pytest.raises(KernelError, match="verify_drafts"):
            bare_ops().verify_drafts(*args)


def test_ranges_of_a_cache_of_other_sizes_are_refused():
    """(Their slots and pages would be looked up outside the other cache's table.)"""
    ops = bare_ops()
    made = ops.cache_ranges(view_of(), [(1, 0, 128)])
    for other in (view_of(page=32), replace(view_of(), max_pages=1, page_table=torch.zeros(2, 1, dtype=torch.int32)),
                  replace(view_of(), page_table=torch.zeros(1, 2, dtype=torch.int32))):
        with pytest.raises(KernelError, match="ranges of"):
            ops.cache_values(other, made)
    with pytest.raises(KernelError, match="CUDA device"):
        ops.cache_values(view_of(), made)


def test_the_command_line_refuses_drafts_for_text(tmp_path):
    from rbitnet_b200.cli import main
    with pytest.raises(SystemExit, match="draft-tokens"):
        main(["generate", "--model", str(tmp_path), "--draft-tokens", "2", "--prompt", "text"])

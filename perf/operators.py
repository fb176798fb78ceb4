"""The operators of a serving step over a cache held in 8 bits: what is measured, and their plain forms.

append   rows of the q/k/v product are turned by their positions; the keys and values enter a paged cache as 8-bit floating
         point codes (e4m3) with one power-of-two scale per block of 64 positions and kv head
attend   the queries of the step's new tokens over that cache: one token a sequence, a few drafted ones, whole prompts
verify   drafted tokens against the target's logits: accepted or not from given random numbers, then one token of the model's own

The plain forms are elementary torch operations in float32 (angles, and all of ``verify``, in 64 bits); ``exact`` restates the
definitions a sequence at a time in 64 bits.
"""
import math

import torch

own = False

PAGE = 64                   # positions of a page; a block of one scale is a page here
BASE = 500000.0             # the rotation's base
LOWEST, HIGHEST = -60, 119  # exponents that a scale may have

#: (query heads, kv heads, head size): the grouped heads of bench.py's default model, of its two other shapes, and odd groups
HEADS = [(32, 8, 128), (32, 4, 64), (32, 32, 128), (28, 4, 128), (24, 8, 64), (16, 16, 64), (16, 1, 128)]


def _case(op, seqs, new, context, heads, **more):
    return {"op": op, "seqs": seqs, "new": new, "context": context, "heads": heads[0], "kv": heads[1], "dim": heads[2], "ragged": False,
            "window": 0, **more}


def listed():
    grouped, small, single = HEADS[0], HEADS[1], HEADS[2]
    return [
        # one sequence's decode step: latency counts
        dict(_case("append", 1, 1, 2047, grouped), name="append_1"),
        # a full decode batch, every sequence at a length of its own
        dict(_case("append", 64, 1, 4000, grouped, ragged=True), name="append_64"),
        # a step that checks up to five tokens of 16 sequences, small heads
        dict(_case("append", 16, 5, 3000, small, ragged=True), name="append_drafts"),
        # the longest prompt in one step
        dict(_case("append", 1, 8192, 0, grouped), name="append_prompt"),
        # one sequence's decode step
        dict(_case("attend", 1, 1, 2048, grouped), name="attend_1"),
        # long contexts of a full batch: the cache's bytes count
        dict(_case("attend", 64, 1, 8000, grouped, ragged=True), name="attend_64"),
        # heads that share no keys, a window of 1,024 keys
        dict(_case("attend", 24, 1, 4000, single, window=1024), name="attend_window"),
        # a step that checks up to five tokens of 16 sequences
        dict(_case("attend", 16, 5, 6001, grouped, ragged=True), name="attend_drafts"),
        # a prompt over its own keys
        dict(_case("attend", 1, 2048, 0, grouped), name="attend_prompt"),
        # one sequence's four drafted tokens, taken for certain by the drafter
        {"op": "verify", "seqs": 1, "drafts": 4, "vocab": 32000, "ragged": False, "certain": True, "greedy": 0, "name": "verify_1"},
        # a full batch with the drafter's probabilities
        {"op": "verify", "seqs": 64, "drafts": 4, "vocab": 128256, "ragged": False, "certain": False, "greedy": 0, "name": "verify_64"},
        # drafts found in the text, unequally many, every other sequence greedy
        {"op": "verify", "seqs": 17, "drafts": 7, "vocab": 128256, "ragged": True, "certain": True, "greedy": 2, "name": "verify_ragged"},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo .. hi, even in its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "verify"])
    if op == "verify":
        seqs, drafts = _spread(rng, 1, 64), rng.randint(1, 8)
        vocab = min(_spread(rng, 500, 128256), 320 * 128256 // (seqs * (drafts + 1)))
        return {"op": op, "seqs": seqs, "drafts": drafts, "vocab": vocab, "ragged": rng.random() < 0.5, "certain": rng.random() < 0.5,
                "greedy": rng.choice([0, 0, 2, 1])}
    heads = rng.choice(HEADS)
    kind = rng.choice(["single", "single", "drafts", "prompt"])
    ragged = rng.random() < 0.6
    if kind == "prompt":
        if op == "append":
            new, most = _spread(rng, 9, 8192), 8192
        else:
            new, most = _spread(rng, 9, 2048), 2048
        seqs = max(1, min(8, most // new))
        context = rng.choice([0, 0, _spread(rng, 1, 1500)]) if op == "append" or new * seqs <= 1024 else 0
    else:
        new = 1 if kind == "single" else rng.randint(2, 8)
        seqs = _spread(rng, 1, 64)
        context = _spread(rng, 1, 4000 if op == "append" else 8000)
        if op == "attend":                  # the cache of the largest listed case bounds what a drawn one reads and computes
            context = max(1, min(context, 64 * 8000 * 8 * 128 // (seqs * heads[1] * heads[2] * (1 if new == 1 else 2))))
    window = rng.choice([0, 0, 0, _spread(rng, 17, 2048)]) if op == "attend" else 0
    return _case(op, seqs, new, context, heads, ragged=ragged, window=window)


# ------------------------------------------------------------------------------------------- sizes of a case
def _sizes(case):
    """Per sequence (positions held before the step, new tokens)."""
    n, new, context = case["seqs"], case["new"], case["context"]
    part = [((i * 0.6180339887498949) % 1.0) if case["ragged"] and i else 1.0 for i in range(n)]
    held = [int(context * p) for p in part]
    return held, [max(1, int(math.ceil(new * part[n - 1 - i]))) for i in range(n)]


def _rows(case):
    """Rows of logits per sequence: its drafts, and one more."""
    n, most = case["seqs"], case["drafts"]
    return [1 + (most if not case["ragged"] or i == 0 else int((i * 0.6180339887498949) % 1.0 * (most + 1))) for i in range(n)]


def work(case):
    if case["op"] == "verify":
        rows, V = sum(_rows(case)), case["vocab"]
        # every row's logits once; of the draft probabilities one row a sequence, and one number for every draft
        return {"bytes": 4 * rows * V + (0 if case["certain"] else 4 * V * case["seqs"]) + 24 * rows, "flops": 4 * rows * V}
    held, new = _sizes(case)
    H, Kh, D, T = case["heads"], case["kv"], case["dim"], sum(_sizes(case)[1])
    if case["op"] == "append":
        # rows in, turned queries out, codes out and the values they stand for read back (two bytes each)
        return {"bytes": 2 * T * (H + 2 * Kh) * D + 2 * T * H * D + 2 * T * Kh * D * (1 + 2), "flops": 6 * T * (H + Kh) * D}
    w = case["window"]
    seen = sum(min(h + n, w + n - 1) if w else h + n for h, n in zip(held, new))
    pairs = sum(min(h + j + 1, w) if w else h + j + 1 for h, n in zip(held, new) for j in range(n))
    return {"bytes": 2 * seen * Kh * D + 4 * T * H * D, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------------- inputs
def _exponent(amax):
    """The least whole e with amax <= 448 * 2^e, within the bounds of a scale (``amax`` float32 or float64)."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, e, torch.full_like(e, LOWEST)).clamp(LOWEST, HIGHEST)


def _filled(shape, spread, g, dev):
    """Random codes and scales of a pool [pages, kv heads, PAGE, dim]: normal values, some channels large, as a model's keys are."""
    codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty((*shape[:2], 1), dtype=torch.float32, device=dev)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for at in range(0, shape[0], step):
        n = min(step, shape[0] - at)
        v = torch.randn((n, *shape[1:]), generator=g, device=dev) * spread
        s = torch.ldexp(torch.ones((), device=dev), _exponent(v.abs().amax((2, 3))))
        codes[at:at + n] = (v / s[:, :, None, None]).to(torch.float8_e4m3fn)
        scales[at:at + n] = s[:, :, None]
    return codes, scales


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, g, dev)
    held, new = _sizes(case)
    H, Kh, D, n = case["heads"], case["kv"], case["dim"], case["seqs"]
    total = [h + t for h, t in zip(held, new)]
    pages = [-(-t // PAGE) for t in total]
    max_pages = max(pages)
    order = torch.randperm(sum(pages) + 3, generator=g, device=dev).to(torch.int32)          # where a sequence's pages lie
    slots = torch.randperm(n + 1, generator=g, device=dev)[:n].tolist()
    table = torch.zeros((n + 1, max_pages), dtype=torch.int32, device=dev)
    at = 0
    for s, p in zip(slots, pages):
        table[s, :p] = order[at:at + p]
        at += p
    spread = 1.0 + 3.0 * (torch.rand((Kh, 1, D), generator=g, device=dev) > 0.95)
    shape = (sum(pages) + 3, Kh, PAGE, D)
    k, ks = _filled(shape, spread, g, dev)
    v, vs = _filled(shape, 0.5, g, dev)
    T = sum(new)
    state = {"case": case, "k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table, "held": held, "new": new, "slots": slots,
             "pos": torch.cat([torch.arange(h, h + t, device=dev, dtype=torch.int32) for h, t in zip(held, new)]),
             "slot": torch.tensor([s for s, t in zip(slots, new) for _ in range(t)], dtype=torch.int32, device=dev),
             "seq": torch.tensor([i for i, t in enumerate(new) for _ in range(t)], device=dev),
             "nth": torch.cat([torch.arange(t, device=dev) for t in new])}
    if case["op"] == "append":
        state["qkv"] = torch.randn((T, (H + 2 * Kh) * D), generator=g, device=dev).to(torch.bfloat16)
        state["inv_freq"] = (1.0 / BASE ** (torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)).to(torch.float32)
        # the pages that hold the new positions, and how many positions of each are in use
        items = [(s, p, min(PAGE, h + t - p * PAGE)) for s, h, t in zip(slots, held, new) for p in range(h // PAGE, -(-(h + t) // PAGE))]
        item = torch.tensor(items, device=dev)
        state["pages"], state["used"] = table[item[:, 0], item[:, 1]].long(), item[:, 2]
    else:
        state["q"] = torch.randn((T, H, D), generator=g, device=dev).to(torch.bfloat16)
    if own:
        _plan(state)
    return state


def _prepare_verify(case, g, dev):
    rows, V = _rows(case), case["vocab"]
    R, n = sum(rows), case["seqs"]
    first = torch.tensor([0] + rows, device=dev).cumsum(0)
    logits = torch.randn((R, V), generator=g, device=dev) * 3.0
    temperature = 0.6 + 0.6 * torch.rand((n,), generator=g, device=dev)
    if case["greedy"]:
        temperature[::case["greedy"]] = 0.0
    probs = None
    if case["certain"]:
        # the likeliest token, or another one
        drafts = torch.where(torch.rand((R,), generator=g, device=dev) < 0.7, logits.argmax(1),
                             torch.randint(V, (R,), generator=g, device=dev))
    else:
        # the drafter's distribution is near the target's, and its drafts are drawn from it
        probs = torch.softmax((logits + 0.5 * torch.randn((R, V), generator=g, device=dev)) / 0.9, dim=1)
        target = torch.rand((R, 1), generator=g, device=dev, dtype=torch.float64)
        drafts = (probs.double().cumsum(1) < target).sum(1).clamp(max=V - 1)
    return {"case": case, "logits": logits, "first_row": first.to(torch.int32), "drafts": drafts.to(torch.int32), "probs": probs,
            "temperature": temperature, "uniforms": torch.rand((R, 2), generator=g, device=dev), "most": case["drafts"]}


# ------------------------------------------------------------------------------------------- the framework's calls
_OPS = []


def _ops():
    from rbitnet_b200.kernels.ops import CudaOps
    if not _OPS:
        _OPS.append(CudaOps(torch.bfloat16))
    return _OPS[0]


def _plan(state):
    """What a step keeps for all of its layers: where its rows belong, and a layer's view of the cache."""
    import numpy as np
    from rbitnet_b200.cache import CacheLayerView
    from rbitnet_b200.engine.step import SeqChunk, build_meta
    case, at, chunks = state["case"], 0, []
    for s, h, t in zip(state["slots"], state["held"], state["new"]):
        chunks.append(SeqChunk(s, h, t, at))
        at += t
    state["meta"] = build_meta(chunks, np.zeros(at, dtype=np.int32), np.zeros(0, dtype=np.int32), _ops().device)
    state["view"] = CacheLayerView(state["k"], state["v"], state["table"], state["table"].shape[1], PAGE, case["kv"], case["dim"], True, 0,
                                   (state["k"], state["v"]), (state["k_scale"], state["v_scale"]))
    if case["op"] == "append":
        state["ranges"] = _ops().cache_ranges(state["view"], [(c.slot, c.start, c.start + c.n_new) for c in chunks])


def _own(state):
    case, ops = state["case"], _ops()
    if case["op"] == "append":
        q = ops.rotate_append(state["qkv"], (state["inv_freq"], False, case["dim"]), state["meta"], state["view"], case["heads"])
        return (q, *ops.cache_values(state["view"], state["ranges"]))
    if case["op"] == "attend":
        return ops.attention(state["q"], state["meta"], state["view"], case["heads"], case["dim"] ** -0.5, case["window"])
    return ops.verify_drafts(state["logits"], state["first_row"], state["drafts"], state["temperature"], state["uniforms"], state["most"],
                             draft_probs=state["probs"])


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "attend": _attend, "verify": _verify}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------- plain forms
def _append(state):
    case = state["case"]
    H, Kh, D = case["heads"], case["kv"], case["dim"]
    x = state["qkv"].float().view(-1, H + 2 * Kh, D)
    angle = state["pos"].double()[:, None] * state["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[:, :H + Kh, :D // 2], x[:, :H + Kh, D // 2:]
    turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=2)
    page = state["table"][state["slot"].long(), (state["pos"] // PAGE).long()].long()
    at = (state["pos"] % PAGE).long()
    first = torch.full((state["k"].shape[0],), PAGE, device=x.device).scatter_reduce(0, page, at, "amin")    # a page's first new position
    pages, out = state["pages"], []
    before = torch.arange(PAGE, device=x.device)[None, :, None] < first[pages][:, None, None]
    for rows, pool, scale in ((turned[:, H:], state["k"], state["k_scale"]), (x[:, H + Kh:], state["v"], state["v_scale"])):
        codes = pool.view(torch.uint8)
        largest = torch.zeros((pool.shape[0], Kh), device=x.device).scatter_reduce(0, page[:, None].expand(-1, Kh), rows.abs().amax(2), "amax")
        needed = torch.ldexp(torch.ones((), device=x.device), _exponent(largest[pages]))
        old = scale[pages, :, 0]
        now = torch.where((first[pages] == 0)[:, None], needed, torch.maximum(old, needed))
        # what the block holds already, in the scale that it has from here on
        held = (pool[pages].float() * (old / now)[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        codes[pages] = torch.where(before[:, None], held, codes[pages])
        scale[pages, :, 0] = now
        codes[page, :, at] = (rows / scale[page]).to(torch.float8_e4m3fn).view(torch.uint8)
        values = pool[pages].float() * scale[pages][..., None]
        used = torch.arange(PAGE, device=x.device)[None, None, :, None] < state["used"][:, None, None, None]
        out.append(torch.where(used, values, torch.zeros((), device=x.device)).to(torch.bfloat16))
    return turned[:, :H].to(torch.bfloat16), out[0], out[1]


def _attend(state):
    case = state["case"]
    H, Kh, D, n = case["heads"], case["kv"], case["dim"], case["seqs"]
    G, most = H // Kh, max(state["new"])
    pages = state["table"][state["slots"]].long()
    k, v = ((pool[pages].float() * scale[pages][..., None]).transpose(1, 2).reshape(n, Kh, -1, D)
            for pool, scale in ((state["k"], state["k_scale"]), (state["v"], state["v_scale"])))
    q = torch.zeros((n, most, H, D), device=k.device)
    q[state["seq"], state["nth"]] = state["q"].float()
    q = q.view(n, most, Kh, G, D).permute(0, 2, 3, 1, 4).reshape(n, Kh, G * most, D)
    pos = torch.full((n, most), -1, device=k.device, dtype=torch.int32)
    pos[state["seq"], state["nth"]] = state["pos"]
    key = torch.arange(k.shape[2], device=k.device)
    seen = key <= pos[:, :, None]
    if case["window"]:
        seen &= key > pos[:, :, None] - case["window"]
    s = (q @ k.transpose(2, 3) * D ** -0.5).view(n, Kh, G, most, -1)
    s = torch.where(seen[:, None, None], s, torch.full((), -math.inf, device=k.device))
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    o = (e.view(n, Kh, G * most, -1) @ v).view(n, Kh, G, most, D) / e.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4)[state["seq"], state["nth"]].reshape(-1, H * D).to(torch.bfloat16)


def _verify(state):
    z, first, most = state["logits"].double(), state["first_row"].long(), state["most"]
    R, V = z.shape
    dev = z.device
    row = torch.arange(R, device=dev)
    seq = (first[1:, None] <= row).sum(0)
    z = torch.where(torch.isnan(z), -math.inf, z)
    m = z.amax(1, keepdim=True)
    top = z == m
    T = state["temperature"].double()[seq]
    # a token's weight: exp((z - max) / T); the lowest of the largest alone where there is no temperature, or nothing to weigh
    w = torch.where(top, 1.0, torch.exp((z - m) / T[:, None]))
    only = torch.zeros_like(w)
    only[row, top.int().argmax(1)] = 1.0
    w = torch.where((T[:, None] > 0) & (m > -math.inf), w, only)
    total = w.sum(1)
    draft = state["drafts"].long()
    last = row == first[1:][seq] - 1
    inside = ~last & (draft >= 0) & (draft < V)
    at = draft.clamp(0, V - 1)
    taken = state["probs"].double()[row, at] if state["probs"] is not None else torch.ones(R, device=dev, dtype=torch.float64)
    ok = inside & (state["uniforms"][:, 0].double() * taken * total < w[row, at])
    # per sequence: its rows side by side, how many are accepted before the first that is not
    nth = torch.arange(most + 1, device=dev)
    beside = first[:-1, None] + nth
    valid = beside < first[1:, None]
    beside = beside.clamp(max=R - 1)
    accepted = (ok[beside] & valid).cumprod(1).sum(1)
    pick = first[:-1] + accepted
    p = w[pick] / total[pick, None]
    if state["probs"] is not None:
        minus = state["probs"].double()[pick]
    else:
        minus = torch.zeros_like(p)
        minus[torch.arange(len(pick), device=dev), at[pick]] = 1.0
    left = torch.where(inside[pick, None], (p - minus).clamp(min=0.0), p)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, p)
    run_ = left.cumsum(1)
    goal = state["uniforms"][pick, 1].double() * left.sum(1)
    number = torch.arange(V, device=dev)
    token = torch.minimum((run_ <= goal[:, None]).sum(1), torch.where(left > 0, number, 0).amax(1))
    tokens = torch.where(nth < accepted[:, None], draft[beside], torch.where(nth == accepted[:, None], token[:, None], -1))
    return accepted.to(torch.int32), tokens.to(torch.int32)


# ------------------------------------------------------------------------------------------- in 64 bits
def _to_e4m3(x):
    """Float64 values rounded to four binary digits (the nearest, ties to even), steps of 2^-9 near zero, 448 at most."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones((), dtype=torch.float64, device=x.device), (e - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_append(state):
    case = state["case"]
    H, Kh, D = case["heads"], case["kv"], case["dim"]
    freq, qs, ks, vs, at = state["inv_freq"].double(), [], [], [], 0
    for slot, held, new in zip(state["slots"], state["held"], state["new"]):
        x = state["qkv"][at:at + new].double().view(new, H + 2 * Kh, D)
        at += new
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                           torch.arange(held, held + new, device=x.device, dtype=torch.float64)[:, None] * freq)[:, None]
        z = torch.complex(x[:, :H + Kh, :D // 2], x[:, :H + Kh, D // 2:]) * turn
        turned = torch.cat([z.real, z.imag], dim=2)
        qs.append(turned[:, :H])
        for p in range(held // PAGE, -(-(held + new) // PAGE)):
            lo, hi = max(held, p * PAGE), min(held + new, (p + 1) * PAGE)
            page = int(state["table"][slot, p])
            for got, rows, pool, scale in ((ks, turned[lo - held:hi - held, H:], state["k"], state["k_scale"]),
                                           (vs, x[lo - held:hi - held, H + Kh:], state["v"], state["v_scale"])):
                e = _exponent(rows.abs().amax((0, 2)))
                old = scale[page, :, 0].double()
                if lo > p * PAGE:
                    e = torch.maximum(e, torch.log2(old).round().to(e.dtype))
                now = torch.ldexp(torch.ones((), dtype=torch.float64, device=x.device), e)[:, None, None]
                block = torch.zeros((Kh, PAGE, D), dtype=torch.float64, device=x.device)
                block[:, :lo - p * PAGE] = _to_e4m3(pool[page, :, :lo - p * PAGE].double() * old[:, None, None] / now) * now
                block[:, lo - p * PAGE:hi - p * PAGE] = _to_e4m3(rows.transpose(0, 1) / now) * now
                got.append(block)
    return torch.cat(qs), torch.stack(ks), torch.stack(vs)


def _exact_attend(state):
    case = state["case"]
    H, Kh, D, out, at = case["heads"], case["kv"], case["dim"], [], 0
    for slot, held, new in zip(state["slots"], state["held"], state["new"]):
        n = held + new
        pages = state["table"][slot, :-(-n // PAGE)].long()
        k, v = (torch.cat(list(pool[pages].double() * scale[pages, :, :, None].double()), dim=1)[:, :n]
                for pool, scale in ((state["k"], state["k_scale"]), (state["v"], state["v_scale"])))
        for lo in range(0, new, 256):
            q = state["q"][at + lo:at + min(new, lo + 256)].double()
            where = held + lo + torch.arange(len(q), device=q.device)[:, None]
            key = torch.arange(n, device=q.device)
            hidden = (key > where) | (key <= where - case["window"] if case["window"] else key < 0)
            heads = [torch.softmax((q[:, h] @ k[h * Kh // H].T / math.sqrt(D)).masked_fill(hidden, -math.inf), dim=1) @ v[h * Kh // H]
                     for h in range(H)]
            out.append(torch.cat(heads, dim=1))
        at += new
    return torch.cat(out)


def exact(case, seed):
    if case["op"] == "verify":
        return None                        # whole numbers, decided in 64 bits by the plain form itself
    state = prepare(case, seed)
    return _exact_append(state) if case["op"] == "append" else _exact_attend(state)

"""The cache held in 8 bits, and drafts against logits, in plain 64-bit torch: what tests compare the kernels with."""
import math

import torch

F64 = torch.float64


def block_of(page):
    """Positions that share a scale in pages of ``page`` positions."""
    assert page <= 64 or page % 64 == 0
    return min(page, 64)


def scale_for(amax: float) -> float:
    """The least power of two, 2^-60 .. 2^119, with amax <= 448 of it (NaN does not count)."""
    e = -60
    while e < 119 and not amax <= 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """float64 values rounded to e4m3: four binary digits, steps of 2^-9 below 2^-6, ties to even, 448 at most; NaN stays."""
    x = x.to(F64)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20, max=1e300)))
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, e)
    step = torch.exp2(e.clamp(min=-6) - 3)
    return torch.where(x.isnan(), x, (torch.round(x / step) * step).clamp(-448.0, 448.0))


def turned(x, pos, inv_freq, rot_dim, interleaved):
    """x [n, heads, D] float64, the first rot_dim values of a head turned by pos [n] times the frequencies."""
    if rot_dim == 0:
        return x
    angle = pos.to(F64)[:, None] * inv_freq.to(F64)[None, :rot_dim // 2]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    y = x.clone()
    a, b = (slice(0, rot_dim, 2), slice(1, rot_dim, 2)) if interleaved else (slice(0, rot_dim // 2), slice(rot_dim // 2, rot_dim))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def append(view, slot, pos0, k_rows, v_rows):
    """Rows [n, kv heads, D] at positions pos0 .. of a slot, into a view whose tensors lie on the CPU (changed in place)."""
    P, block = view.page_size, block_of(view.page_size)
    n = k_rows.shape[0]
    done = 0
    while done < n:
        pos = pos0 + done
        start = pos - pos % block
        m = min(n - done, start + block - pos)
        page, at = int(view.page_table[slot, pos // P]), start % P
        for pool, scales, rows in ((view.k, view.scales[0], k_rows), (view.v, view.scales[1], v_rows)):
            for h in range(view.n_kv_heads):
                new = rows[done:done + m, h].to(F64)
                fine = new[~new.isnan()].abs()
                need = scale_for(float(fine.max()) if fine.numel() else 0.0)
                old = float(scales[page, h, at // block])
                now = max(old, need) if pos > start else need
                if pos > start and old < now:
                    held = pool[page, h, at:at + pos - start].to(F64)
                    pool[page, h, at:at + pos - start] = to_e4m3(held * (old / now)).to(pool.dtype)
                pool[page, h, at + pos - start:at + pos - start + m] = to_e4m3(new / now).to(pool.dtype)
                scales[page, h, at // block] = now
        done += m


def values(view, slot, length, stream):
    """float64 [kv heads, length, D]: what a slot's first positions hold."""
    P, block = view.page_size, block_of(view.page_size)
    pool, scales = (view.k, view.scales[0]) if stream == 0 else (view.v, view.scales[1])
    out = []
    for pos in range(0, length, P):
        page = int(view.page_table[slot, pos // P])
        s = scales[page].to(F64).repeat_interleave(block, dim=1)
        out.append(pool[page].to(F64) * s[..., None])
    return torch.cat(out, dim=1)[:, :length]


def attend(view, slot, pos0, q, scale, window=0, sinks=None, softcap=0.0, keep_first=0):
    """(outputs, sums of weight * |value|) of rows q [n, H, D] at positions pos0 .. of a slot: both [n, H * D] float64."""
    n, H, D = q.shape
    K, V = values(view, slot, pos0 + n, 0), values(view, slot, pos0 + n, 1)
    key, where = torch.arange(pos0 + n), pos0 + torch.arange(n)[:, None]
    seen = key <= where
    if window:
        seen &= (key > where - window) | (key < keep_first)
    out, size = [], []
    for h in range(H):
        kvh = h // (H // view.n_kv_heads)
        s = q[:, h].to(F64) @ K[kvh].T * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        s = s.masked_fill(~seen, -math.inf)
        m = s.amax(1, keepdim=True)
        if sinks is not None:
            m = m.clamp(min=float(sinks[h]))
        e = torch.exp(s - m)
        total = e.sum(1, keepdim=True)
        if sinks is not None:
            total = total + torch.exp(sinks[h].to(F64) - m)
        v = V[kvh].clone()
        v[~seen.any(0)] = 0.0
        out.append(e @ v / total)
        size.append(e @ v.abs() / total)
    return torch.cat(out, dim=1), torch.cat(size, dim=1)


def verify(logits, first_row, drafts, temperature, uniforms, most, draft_probs=None):
    """(accepted, tokens) as lists, a sequence and a row at a time."""
    V = logits.shape[1]
    accepted, tokens = [], []
    for b in range(len(first_row) - 1):
        got, rows = [], range(int(first_row[b]), int(first_row[b + 1]))
        n = 0
        for r in rows:
            z = logits[r].to(F64)
            z = torch.where(z.isnan(), -math.inf, z)
            m, T = float(z.max()), float(temperature[b])
            greedy = not (T > 0 and m > -math.inf)
            # probabilities times their sum: nothing is divided, so that equal logits are equal steps exactly
            if greedy:
                w = torch.zeros(V, dtype=F64)
                w[int((z == m).nonzero()[0])] = 1.0
            else:
                w = torch.where(z == m, 1.0, torch.exp((z - m) / T))
            d = int(drafts[r])
            judged = r != rows[-1] and 0 <= d < V
            q = torch.zeros(V, dtype=F64)
            if judged:
                if draft_probs is not None:
                    q = draft_probs[r].to(F64)
                else:
                    q[d] = 1.0
                if float(uniforms[r, 0]) * float(q[d]) * float(w.sum()) < float(w[d]):
                    got.append(d)
                    n += 1
                    continue
            left = (w - q * w.sum()).clamp(min=0.0)
            if float(left.sum()) == 0.0:
                left = w
            run = left.cumsum(0)
            over = (run > float(uniforms[r, 1]) * float(left.sum())).nonzero()
            got.append(int(over[0]) if len(over) else int((left > 0).nonzero()[-1]))
            break
        accepted.append(n)
        tokens.append(got + [-1] * (most + 1 - len(got)))
    return accepted, tokens

"""The stand-in for the kernel layer (torch_ops) with a cache held in 8 bits and the check of drafts, for tests on the CPU."""
import torch

import plain_cache8 as plain
from torch_ops import TorchOps


class TorchOps8(TorchOps):
    def rotate_append(self, qkv, rotary, meta, view, n_heads):
        if not view.scales:
            return super().rotate_append(qkv, rotary, meta, view, n_heads)
        D, Kh, T = view.head_dim, view.n_kv_heads, qkv.shape[0]
        x = qkv.to(plain.F64).view(T, -1, D)
        inv, interleaved, rot = rotary
        t = plain.turned(x[:, :n_heads + Kh], meta.tok_pos, inv, rot, interleaved)
        for c in meta.seqs if view.writes else ():
            rows = slice(c.offset, c.offset + c.n_new)
            plain.append(view, c.slot, c.start, t[rows, n_heads:], x[rows, n_heads + Kh:])
        return t[:, :n_heads].to(self.dtype)

    def attention(self, q, meta, view, n_heads, scale, window, sinks=None, softcap=0.0, keep_first=0):
        if not view.scales:
            return super().attention(q, meta, view, n_heads, scale, window, sinks, softcap, keep_first)
        return torch.cat([plain.attend(view, c.slot, c.start, q[c.offset:c.offset + c.n_new], scale, window or 0, sinks, softcap, keep_first)[0]
                          for c in meta.seqs]).to(self.dtype)

    def verify_drafts(self, logits, first_row, drafts, temperature, uniforms, most, draft_probs=None):
        a, t = plain.verify(logits, first_row.tolist(), drafts.tolist(), temperature.tolist(), uniforms, most, draft_probs)
        return torch.tensor(a, dtype=torch.int32), torch.tensor(t, dtype=torch.int32)

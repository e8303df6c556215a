"""The decoder-block operators in 64 bits, element by element from their
definitions, for the tests of the kernels and of their argument checks."""

import math

import torch

F32_INV127 = torch.tensor(1.0 / 127.0, dtype=torch.float32).double()


def norm(v, kind, weight=None, bias=None, eps=1e-6):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    out = (v - mean) / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        out = out * weight.double()
    return out if bias is None else out + bias.double()


def f32(t):
    return t.float().double()


class Cache:
    """The cache as codes and scales on the host, token by token."""

    def __init__(self, pages, heads, dim, block):
        self.block = block
        self.codes = torch.zeros(pages, heads, 2, block, dim, dtype=torch.float64)
        self.scales = torch.zeros(pages, heads, 2, dtype=torch.float64)

    def write(self, k, v, table, lengths, starts):
        for b, length in enumerate(lengths):
            n = starts[b + 1] - starts[b]
            first = length - n
            for ordinal in range(max(0, first) // self.block,
                                 (length + self.block - 1) // self.block):
                lo = max(0, first, ordinal * self.block)
                hi = min(length, (ordinal + 1) * self.block)
                if lo >= hi:
                    continue
                page = int(table[b][ordinal])
                at = lo - ordinal * self.block
                for side, x in enumerate((k, v)):
                    rows = x[starts[b] + lo - first:starts[b] + hi - first].double()
                    for h in range(rows.shape[1]):
                        part = rows[:, h]
                        finite = part[torch.isfinite(part)].abs()
                        amax = float(finite.max()) if finite.numel() else 0.0
                        want = f32(torch.tensor(max(amax, 2.0 ** -80)).double() * F32_INV127)
                        old = self.scales[page, h, side] if at else torch.zeros(()).double()
                        scale = torch.maximum(old, want)
                        inverse = f32(1.0 / scale)
                        if at and scale > old:
                            held = self.codes[page, h, side, :at]
                            held.copy_(torch.round(f32(f32(held * old) * inverse)))
                        fresh = torch.round(f32(part * inverse)).clamp(-127, 127)
                        self.codes[page, h, side, at:at + hi - lo] = torch.where(
                            torch.isnan(part), torch.zeros_like(part), fresh)
                        self.scales[page, h, side] = scale

    def value_scales(self, table_row, length):
        """[length, heads]: the value scale of each token's block."""
        pages = [int(p) for p in table_row[:(length + self.block - 1) // self.block]]
        return self.scales[pages, :, 1].repeat_interleave(self.block, 0)[:length]

    def values(self, table_row, length, side):
        """[length, heads, dim] of one sequence."""
        pages = [int(p) for p in table_row[:(length + self.block - 1) // self.block]]
        v = self.codes[pages, :, side] * self.scales[pages, :, side][..., None, None]
        return v.permute(0, 2, 1, 3).reshape(-1, *v.permute(0, 2, 1, 3).shape[2:])[:length]


def attend(q, k, v, offset, scale, causal, window, value_scales=None):
    """One sequence: q [n, heads, dim], k and v [length, kv_heads, dim]; returns
    (out, lse, sum of |weight * v|, largest sum of |scale * q * k|, largest
    weight * value scale times the number of keys)."""
    n, heads, dim = q.shape
    group = heads // k.shape[1] if k.shape[1] else 1
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    size = torch.zeros(n, heads, dim, dtype=torch.float64)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros(n, heads, dtype=torch.float64)
    peak = torch.zeros(n, heads, dtype=torch.float64)
    for i in range(n):
        p = offset + i
        keys = [j for j in range(k.shape[0])
                if (not causal or j <= p) and (not window or j > p - window)]
        if not keys:
            continue
        for h in range(heads):
            s = k[keys, h // group] @ q[i, h].double() * scale
            lse[i, h] = torch.logsumexp(s, 0)
            w = torch.exp(s - lse[i, h])
            out[i, h] = w @ v[keys, h // group]
            size[i, h] = w @ v[keys, h // group].abs()
            reach[i, h] = (k[keys, h // group].abs() @ q[i, h].double().abs()).max() * abs(scale)
            if value_scales is not None:
                peak[i, h] = (w * value_scales[keys, h // group]).max() * len(keys)
    return out, lse, size, reach, peak

"""Cases of the decoder-block operators: the norms around a block, the 8-bit
key/value cache (written and read back) and attention over that cache.

``run`` makes one pass: with ``own`` false in plain elementary torch
operations in 32 bits, with ``own`` true through ``cim22_b200``'s entry
points. ``exact`` computes the same outputs from the definitions in 64 bits.

Definitions.
  block norm   h = residual_scale * residual + act(gate) * post(x),  y = pre(h)
               with post / pre an RMS or layer norm over the last axis.
  cache        int8 codes [pages, kv_heads, 2 (K, V), block, head_dim] and one
               f32 scale per (page, kv head, K or V). Sequence b holds
               lengths[b] tokens, token p in page table[b, p // block]. A write
               of n_b tokens fills the last n_b positions: per block and head
               amax = the largest finite |new value|, s = max(old scale (none
               for a block whose first token is written), max(amax, 2^-80) *
               f32(1/127)); where the scale grew the block's earlier codes q
               become rint(f32(q * s_old) * f32(1 / s)); new codes are
               rint(x * f32(1 / s)), within +-127. A code stands for q * s.
  attention    softmax(scale * q k^T) v over the values the codes stand for;
               query i of n_b sits at position lengths[b] - n_b + i, sees
               positions up to its own (causal) and the last `window` of them
               (window > 0); a query that sees nothing gives zeros.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_INV127 = torch.tensor(1.0 / 127.0, dtype=torch.float32).item()


# ---------------------------------------------------------------------------
# Cases.


def listed():
    return [
        # One token of a decoder at batch 1: launch latency decides.
        dict(name="norm_one_token", op="norm", dtype="f32", rows=1, dim=4096, post="rms",
             pre="rms", gate="channel", act="none", residual_scale=1.0),
        # A batch of rows between two Linear stacks of width 4096.
        dict(name="norm_stack_512", op="norm", dtype="f32", rows=512, dim=4096, post="layer",
             pre="layer", gate="group", act="tanh", residual_scale=0.5),
        # An odd width, rows that start off a vector boundary.
        dict(name="norm_odd_width", op="norm", dtype="f16", rows=3001, dim=1001, post="none",
             pre="layer", gate="full", act="sigmoid", residual_scale=1.0),
        # A long prompt's residual stream.
        dict(name="norm_prompt", op="norm", dtype="bf16", rows=32768, dim=4096, post="rms",
             pre="rms", gate="row", act="sigmoid", residual_scale=0.8),
        # One new token for each of a batch of sequences.
        dict(name="cache_one_token", op="cache", dtype="f32", batch=64, new=1, context=2000,
             kv_heads=8, dim=128, block=64, shape_seed=1),
        # Prompts of many lengths written at once.
        dict(name="cache_prompts", op="cache", dtype="bf16", batch=13, new=8192, context=200,
             kv_heads=8, dim=128, block=64, shape_seed=2),
        # A single user with a short context, in the layers' f32.
        dict(name="decode_short", op="attend", dtype="f32", batch=1, new=1, context=500,
             q_heads=32, kv_heads=8, dim=128, block=64, causal=True, window=0, lse=False,
             ragged=False, shape_seed=3),
        # A serving batch of uneven lengths (one slot is empty).
        dict(name="decode_batch", op="attend", dtype="bf16", batch=64, new=1, context=8191,
             q_heads=32, kv_heads=8, dim=128, block=64, causal=True, window=0, lse=False,
             ragged=True, shape_seed=4),
        # One very long context: the axis has to be split.
        dict(name="decode_long", op="attend", dtype="f16", batch=1, new=1, context=200000,
             q_heads=32, kv_heads=4, dim=128, block=32, causal=True, window=0, lse=True,
             ragged=False, shape_seed=5),
        # Uneven prompts in f32, as CIM layers give their queries.
        dict(name="prompt_f32", op="attend", dtype="f32", batch=5, new=1500, context=300,
             q_heads=16, kv_heads=4, dim=80, block=16, causal=True, window=0, lse=True,
             ragged=True, shape_seed=6),
        # A long prompt.
        dict(name="prompt_long", op="attend", dtype="bf16", batch=1, new=8192, context=0,
             q_heads=32, kv_heads=8, dim=128, block=64, causal=True, window=0, lse=False,
             ragged=False, shape_seed=7),
        # A chunk of a prompt against a long context through a window.
        dict(name="chunk_window", op="attend", dtype="f16", batch=3, new=1024, context=15000,
             q_heads=24, kv_heads=8, dim=64, block=128, causal=True, window=4096, lse=False,
             ragged=True, shape_seed=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "cache", "attend", "attend"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        dim = rng.choice([_log(rng, 16, 8192), 8 * _log(rng, 8, 1024)])
        rows = _log(rng, 1, max(2, min(60000, 100000000 // dim)))
        post = rng.choice(["none", "rms", "layer"])
        return dict(op=op, dtype=dtype, rows=rows, dim=dim, post=post,
                    pre=rng.choice(["rms", "layer"]),
                    gate=rng.choice(["none", "channel", "row", "group", "full"]),
                    act=rng.choice(["none", "sigmoid", "tanh"]),
                    residual_scale=rng.choice([1.0, 0.5, 1.25]))
    dim = rng.choice([16, 48, 64, 80, 96, 128, 128])
    block = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    seed = rng.randrange(1 << 30)
    if op == "cache":
        new = rng.choice([1, _log(rng, 2, 4000)])
        batch = _log(rng, 1, max(1, min(64, 60000 // new)))
        return dict(op=op, dtype=dtype, batch=batch, new=new, context=_log(rng, 1, 3000),
                    kv_heads=kv_heads, dim=dim, block=block, shape_seed=seed)
    group = rng.choice([1, 2, 3, 4, 6, 8])
    new = rng.choice([1, 1, _log(rng, 2, 30), _log(rng, 30, 3000)])
    context = _log(rng, 1, 30000 if new < 30 else 6000)
    cost = (new + 16) * (context + new) * kv_heads * group
    batch = _log(rng, 1, max(1, min(48, int(1.2e9 // cost), 1500000 // (context + new))))
    return dict(op=op, dtype=dtype, batch=batch, new=new, context=context,
                q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, block=block,
                causal=rng.random() < 0.8, window=rng.choice([0, 0, _log(rng, 1, 4000)]),
                lse=rng.random() < 0.5, ragged=rng.random() < 0.7, shape_seed=seed)


def _sizes(case):
    """New tokens and lengths (after the write) of each sequence."""
    rng = random.Random(case["shape_seed"])
    ragged = case.get("ragged", True)
    new, lengths = [], []
    for b in range(case["batch"]):
        n = case["new"]
        if ragged and n > 1:
            n = rng.randint(max(1, n // 8), n)
        c = rng.randint(case["context"] // 8, case["context"]) if ragged else case["context"]
        if b == 0:
            n, c = case["new"], case["context"]
        new.append(n)
        lengths.append(c + n)
    if ragged and case["batch"] > 8:
        # An empty slot of a fixed batch: its one row (if any) sees nothing.
        lengths[case["batch"] // 2] = 0
        if case["new"] > 1:
            new[case["batch"] // 2] = 0
    return new, lengths


# ---------------------------------------------------------------------------
# Inputs.


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev).mul_(scale).to(dtype)

    dtype = _TYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        s = dict(case=case, x=normal(rows, dim, dtype=dtype, scale=2.0),
                 residual=normal(rows, dim, dtype=dtype, scale=3.0), gate_rows=0)
        for which in ("post", "pre"):
            s[which + "_w"] = normal(dim, scale=0.2).add_(1.0)
            s[which + "_b"] = normal(dim, scale=0.1)
        if case["gate"] == "channel":
            s["gate"] = normal(dim)
        elif case["gate"] == "row":
            s["gate"] = normal(rows, 1, dtype=dtype)
        elif case["gate"] == "group":
            groups = next(q for q in (8, 4, 2, 1) if rows % q == 0)
            s["gate"] = normal(groups, dim, dtype=dtype)
        elif case["gate"] == "full":
            s["gate"] = normal(rows, dim, dtype=dtype)
        else:
            s["gate"] = None
        return s

    new, lengths = _sizes(case)
    block, heads, dim = case["block"], case["kv_heads"], case["dim"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    used = [(n + block - 1) // block for n in lengths]
    width = max(1, max(used))
    total = sum(used) + 3
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    # The cache as earlier writes left it: codes of normally distributed
    # values, a scale for each block and head.
    codes = torch.empty(total, heads, 2, block, dim, dtype=torch.int8, device=dev)
    scales = torch.empty(total, heads, 2, device=dev)
    step = max(1, (1 << 28) // (heads * 2 * block * dim))
    for lo in range(0, total, step):
        n = min(step, total - lo)
        v = normal(n, heads, 2, block, dim)
        amax = v.abs().amax(dim=(3, 4))
        codes[lo:lo + n] = (v * (127.0 / amax)[..., None, None]).round_().to(torch.int8)
        spread = normal(n, heads, 2, scale=0.3).exp_()
        scales[lo:lo + n] = amax * _INV127 * spread
    s = dict(case=case, codes=codes, scales=scales, table=table,
             lengths=torch.tensor(lengths, dtype=torch.int32, device=dev),
             starts=None if case["new"] == 1 else torch.tensor(starts, dtype=torch.int32,
                                                               device=dev),
             most=case["new"], longest=max(lengths), tokens=starts[-1])
    # Where each packed row belongs (a plain program's index plan).
    seq = [b for b, n in enumerate(new) for _ in range(n)]
    s["row_seq"] = torch.tensor(seq, device=dev)
    s["row_at"] = torch.tensor([i for n in new for i in range(n)], device=dev)
    s["row_pos"] = torch.tensor([lengths[b] - n + i for b, n in enumerate(new)
                                 for i in range(n)], device=dev)
    if case["op"] == "cache":
        # Keys and values as slices of one projection's rows.
        kv = normal(s["tokens"], 2, heads, dim, dtype=dtype, scale=1.2)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
        # Every block that the write touches is read back whole.
        first = [max(0, lengths[b] - n) // block for b, n in enumerate(new)]
        back = [max(0, lengths[b] - f * block) if new[b] else 0 for b, f in enumerate(first)]
        at = [0]
        for n in back:
            at.append(at[-1] + n)
        s["back_starts"] = torch.tensor(at, dtype=torch.int32, device=dev)
        s["back_tokens"], s["back_most"] = at[-1], max(back)
        s["back_seq"] = torch.tensor([b for b, n in enumerate(back) for _ in range(n)],
                                     device=dev)
        s["back_pos"] = torch.tensor([lengths[b] - n + i for b, n in enumerate(back)
                                      for i in range(n)], device=dev)
        pairs = [(b, f + t) for b, f in enumerate(first)
                 for t in range((lengths[b] + block - 1) // block - f if new[b] else 0)]
        s["touch_seq"] = torch.tensor([p[0] for p in pairs], device=dev)
        s["touch_page"] = torch.tensor([p[1] for p in pairs], device=dev)
    else:
        qkv = normal(s["tokens"], case["q_heads"] + 2 * heads, dim, dtype=dtype)
        s["q"] = qkv[:, :case["q_heads"]]
    return s


# ---------------------------------------------------------------------------
# One pass.


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "norm":
        return _norm_plain(state, case)
    if case["op"] == "cache":
        return _cache_plain(state, case)
    return _attend_plain(state, case)


def _own(s, case):
    if "kept" not in s:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "mlir-cim22_b200"))
        from cim22_b200 import cim_ops, kv_cache

        dev = torch.device("cuda", torch.cuda.current_device())
        if case["op"] == "norm":
            post = None if case["post"] == "none" else cim_ops.Norm(
                case["post"], s["post_w"], s["post_b"] if case["post"] == "layer" else None)
            pre = cim_ops.Norm(case["pre"], s["pre_w"],
                               s["pre_b"] if case["pre"] == "layer" else None)
            s["kept"] = (cim_ops, post, pre)
        else:
            s["kept"] = (kv_cache.Int8KVCache.over(s["codes"], s["scales"]),
                         cim_ops.Workspace(dev), cim_ops.StatusWord(dev))
    if case["op"] == "norm":
        cim_ops, post, pre = s["kept"]
        return cim_ops.block_norm(s["x"], s["residual"], post=post, pre=pre, gate=s["gate"],
                                  gate_activation=case["act"],
                                  residual_scale=case["residual_scale"])
    cache, workspace, status = s["kept"]
    if case["op"] == "cache":
        cache.write(s["k"], s["v"], s["table"], s["lengths"], s["starts"], most=s["most"],
                    status=status)
        return cache.read(s["table"], s["lengths"], s["back_starts"], tokens=s["back_tokens"],
                          most=s["back_most"], dtype=s["k"].dtype, status=status)
    return cache.attend(s["q"], s["table"], s["lengths"], s["starts"], causal=case["causal"],
                        window=case["window"], return_lse=case["lse"], most=s["most"],
                        longest=s["longest"], workspace=workspace, status=status)


def _norm_f32(x, kind, weight, bias, eps=1e-6):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    return y + bias if kind == "layer" else y


def _norm_plain(s, case):
    dtype = s["x"].dtype
    h = _norm_f32(s["x"].float(), case["post"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        gate = s["gate"].float()
        if case["act"] == "sigmoid":
            gate = 1.0 / (1.0 + torch.exp(-gate))
        elif case["act"] == "tanh":
            gate = torch.tanh(gate)
        if case["gate"] == "group":
            gate = gate.repeat_interleave(case["rows"] // gate.shape[0], dim=0)
        h = h * gate
    h = s["residual"].float() * case["residual_scale"] + h
    y = _norm_f32(h, case["pre"], s["pre_w"], s["pre_b"])
    return h.to(dtype), y.to(dtype)


def _cache_plain(s, case):
    block = case["block"]
    lengths = s["lengths"].long()
    b, p = s["touch_seq"], s["touch_page"]
    start = s["starts"][:-1].long() if s["starts"] is not None else torch.arange(
        case["batch"], device=lengths.device)
    count = (s["starts"][1:] - s["starts"][:-1]).long() if s["starts"] is not None else (
        torch.ones_like(lengths))
    pages = s["table"].long()[b, p]
    pos = p[:, None] * block + torch.arange(block, device=p.device)  # [touched, block]
    begin = (lengths - count).clamp(min=0)[b][:, None]
    fresh = (pos >= begin) & (pos < lengths[b][:, None])
    row = (start[b][:, None] + pos - (lengths - count)[b][:, None]).clamp(0, s["tokens"] - 1)
    kv = torch.stack((s["k"], s["v"]), dim=2).float()  # [tokens, heads, 2, dim]
    x = kv[row].permute(0, 2, 3, 1, 4)  # [touched, heads, 2, block, dim]
    fresh = fresh[:, None, None, :, None]
    amax = torch.where(fresh, x.abs(), 0.0).amax(dim=(3, 4))
    held = (begin[:, 0] > p * block)[:, None, None]  # the block holds earlier tokens
    old = torch.where(held, s["scales"][pages], 0.0)
    scale = torch.maximum(old, amax.clamp(min=2.0 ** -80) * _INV127)
    inverse = (1.0 / scale)[..., None, None]
    q = s["codes"][pages].float()
    moved = torch.round(q * old[..., None, None] * inverse)
    q = torch.where((scale > old)[..., None, None] & held[..., None, None], moved, q)
    q = torch.where(fresh, torch.round(x * inverse).clamp(-127, 127), q)
    s["codes"][pages] = q.to(torch.int8)
    s["scales"][pages] = scale
    # Read back.
    page = s["table"].long()[s["back_seq"], s["back_pos"] // block]
    at = s["back_pos"] % block
    values = s["codes"][page, :, :, at].float() * s["scales"][page][..., None]
    return values[:, :, 0].to(s["k"].dtype), values[:, :, 1].to(s["v"].dtype)


def _attend_plain(s, case):
    batch, hq, hk, dim, block = (case[k] for k in ("batch", "q_heads", "kv_heads", "dim",
                                                   "block"))
    group, most, width = hq // hk, s["most"], s["table"].shape[1]
    pages = s["table"].long().clamp(min=0)
    q = torch.zeros(batch, most, hq, dim, device=pages.device)
    q[s["row_seq"], s["row_at"]] = s["q"].float()
    q = q.view(batch, most, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(
        batch, hk, group * most, dim)
    held = s["codes"][pages]  # [batch, width, heads, 2, block, dim]
    scales = s["scales"][pages][..., None, None]
    k = (held[:, :, :, 0].float() * scales[:, :, :, 0]).permute(0, 2, 1, 3, 4).reshape(
        batch, hk, width * block, dim)
    scores = q @ k.transpose(-1, -2) * (1.0 / math.sqrt(dim))
    del k
    key = torch.arange(width * block, device=pages.device)[None, None, :]
    lengths = s["lengths"].long()
    rows = torch.zeros(batch, most, dtype=torch.long, device=pages.device)
    rows[s["row_seq"], s["row_at"]] = s["row_pos"]
    sees = (key < lengths[:, None, None]).expand(batch, most, -1)
    if case["causal"]:
        sees = sees & (key <= rows[..., None])
    if case["window"]:
        sees = sees & (key > rows[..., None] - case["window"])
    sees = sees[:, None, None]
    scores = scores.view(batch, hk, group, most, -1)
    scores = torch.where(sees, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    v = (held[:, :, :, 1].float() * scales[:, :, :, 1]).permute(0, 2, 1, 3, 4).reshape(
        batch, hk, width * block, dim)
    out = p.view(batch, hk, group * most, -1) @ v
    out = out.view(batch, hk, group, most, dim) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, hq, dim)
    out = out[s["row_seq"], s["row_at"]].to(s["q"].dtype)
    if not case["lse"]:
        return out
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(batch, most, hq)
    return out, lse[s["row_seq"], s["row_at"]]


# ---------------------------------------------------------------------------
# What a pass cannot do without.


def _seen(case):
    """(query, key) pairs over all heads, and the cached tokens that some query sees."""
    new, lengths = _sizes(case)
    pairs = keys = 0
    for n, length in zip(new, lengths):
        window = case["window"] or length
        first = length - n
        if length == 0:
            continue
        if case["causal"]:
            # Query at position p sees min(p + 1, window) keys.
            short = max(0, min(n, window - first))  # queries whose window is not full
            pairs += short * first + short * (short + 1) // 2 + (n - short) * window
        else:
            pairs += sum(length - max(0, p - window + 1) for p in range(first, length))
        keys += length - max(0, first - window + 1)
    return pairs, keys


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        gate = {"none": 0, "channel": case["dim"], "row": case["rows"],
                "group": 8 * case["dim"], "full": n}[case["gate"]]
        return {"bytes": 4 * n * size + 4 * case["dim"] * 4 + gate * size, "flops": 14 * n}
    new, lengths = _sizes(case)
    heads, dim, block = case["kv_heads"], case["dim"], case["block"]
    if case["op"] == "cache":
        written = sum(min(n, length) for n, length in zip(new, lengths))
        back = sum(length - max(0, length - n) // block * block
                   for n, length in zip(new, lengths) if n and length)
        values = 2 * heads * dim
        # New values in, codes out; the touched blocks' codes in, values out.
        return {"bytes": values * (written * (size + 1) + back * (1 + size)),
                "flops": values * (3 * written + back)}
    pairs, keys = _seen(case)
    rows = sum(new)
    return {"bytes": keys * heads * (2 * dim + 8 / block) + 2 * rows * case["q_heads"] * dim * size,
            "flops": 4 * pairs * case["q_heads"] * dim}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _norm_exact(s, case)
    if case["op"] == "cache":
        return _cache_exact(s, case)
    return _attend_exact(s, case)


def _norm_exact(s, case):
    def norm(v, kind, w, b):
        if kind == "none":
            return v
        mean = v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else 0.0
        power = ((v - mean) ** 2).sum(-1, keepdim=True) / v.shape[-1]
        out = (v - mean) * (power + 1e-6) ** -0.5 * w.double()
        return out + b.double() if kind == "layer" else out

    hs, ys = [], []
    gate = s["gate"]
    step = max(1, (1 << 26) // case["dim"])
    for lo in range(0, case["rows"], step):
        hi = min(case["rows"], lo + step)
        h = norm(s["x"][lo:hi].double(), case["post"], s["post_w"], s["post_b"])
        if gate is not None:
            if case["gate"] == "channel":
                g = gate.double()[None]
            else:
                each = case["rows"] // gate.shape[0]
                g = gate[torch.arange(lo, hi, device=gate.device) // each].double()
            g = {"none": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["act"]](g)
            h = g * h
        h = h + case["residual_scale"] * s["residual"][lo:hi].double()
        hs.append(h)
        ys.append(norm(h, case["pre"], s["pre_w"], s["pre_b"]))
    return torch.cat(hs), torch.cat(ys)


def _cache_exact(s, case):
    def f32(t):
        return t.float().double()

    new, lengths = _sizes(case)
    block = case["block"]
    inv127 = torch.tensor(_INV127, dtype=torch.float64)
    table = s["table"].tolist()
    outs = [[], []]
    row = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        if n and length:
            first = length - n
            page0, page1 = first // block, (length - 1) // block
            ids = torch.tensor(table[b][page0:page1 + 1], device=s["codes"].device)
            for side, x in enumerate((s["k"], s["v"])):
                x = x[row:row + n].double().transpose(0, 1)  # [heads, n, dim]
                q = s["codes"][ids, :, side].double()  # [pages, heads, block, dim]
                scale = s["scales"][ids, :, side].double()
                parts = []
                for i in range(len(ids)):
                    lo = max(first, (page0 + i) * block)
                    hi = min(length, (page0 + i + 1) * block)
                    part = x[:, lo - first:hi - first]
                    at, end = lo - (page0 + i) * block, hi - (page0 + i) * block
                    want = f32(part.abs().amax(dim=(1, 2)).clamp(min=2.0 ** -80) * inv127)
                    t = torch.maximum(scale[i], want) if at else want
                    inv = f32(1.0 / t)[:, None, None]
                    held = q[i, :, :at]
                    again = torch.round(f32(f32(held * scale[i][:, None, None]) * inv))
                    held = torch.where((t > scale[i])[:, None, None], again, held)
                    fresh = torch.round(f32(part * inv)).clamp(-127, 127)
                    block_values = torch.cat((held, fresh), dim=1)[:, :end]
                    parts.append(block_values * t[:, None, None])
                outs[side].append(torch.cat(parts, dim=1).transpose(0, 1))
        row += n
    return torch.cat(outs[0]), torch.cat(outs[1])


def _attend_exact(s, case):
    if _seen(case)[0] * case["q_heads"] * case["dim"] > 3e11:
        return None
    new, lengths = _sizes(case)
    hq, hk, dim, block = (case[k] for k in ("q_heads", "kv_heads", "dim", "block"))
    group = hq // hk
    out = torch.zeros(s["tokens"], hq, dim, dtype=torch.float64, device=s["codes"].device)
    lse = torch.full((s["tokens"], hq), -math.inf, dtype=torch.float64, device=out.device)
    row = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        if n and length:
            ids = s["table"][b, :(length + block - 1) // block].long()
            for h in range(hk):
                kv = s["codes"][ids, h].double() * s["scales"][ids, h].double()[..., None, None]
                k = kv[:, 0].reshape(-1, dim)[:length]
                v = kv[:, 1].reshape(-1, dim)[:length]
                step = max(1, (1 << 28) // (length * group))
                for lo in range(0, n, step):
                    hi = min(n, lo + step)
                    q = s["q"][row + lo:row + hi, h * group:(h + 1) * group].double()
                    w = torch.einsum("tgd,kd->tgk", q, k) / dim ** 0.5
                    p = torch.arange(length - n + lo, length - n + hi, device=w.device)
                    j = torch.arange(length, device=w.device)
                    hide = torch.zeros(hi - lo, length, dtype=torch.bool, device=w.device)
                    if case["causal"]:
                        hide |= j[None] > p[:, None]
                    if case["window"]:
                        hide |= j[None] <= p[:, None] - case["window"]
                    w.masked_fill_(hide[:, None], -math.inf)
                    z = torch.logsumexp(w, -1)
                    out[row + lo:row + hi, h * group:(h + 1) * group] = torch.einsum(
                        "tgk,kd->tgd", torch.exp(w - z[..., None]), v)
                    lse[row + lo:row + hi, h * group:(h + 1) * group] = z
        row += n
    return (out, lse) if case["lse"] else out

"""The 8-bit key/value cache and attention over it against their definitions in
64 bits (tests/decoder_reference.py)."""

import copy
import math
import pickle

import pytest
import torch

import decoder_reference as ref
from cim22_b200.cim_ops import CimLayer, Norm, StatusWord, Workspace, block_norm
from cim22_b200.kv_cache import Int8KVCache

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


class Setup:
    """A device cache and its host twin, with a shuffled page table."""

    def __init__(self, lengths, heads, dim, block, seed=0, spare=2, width=None):
        self.g = torch.Generator().manual_seed(seed)
        self.block, self.heads, self.dim = block, heads, dim
        used = [(n + block - 1) // block for n in lengths]
        total = sum(used) + spare
        order = torch.randperm(total, generator=self.g)
        self.table = torch.full((len(lengths), width or max(1, max(used))), -1,
                                dtype=torch.int32)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = order[at:at + u]
            at += u
        self.cache = Int8KVCache(total, heads, dim, block)
        self.host = ref.Cache(total, heads, dim, block)
        # What a page held before it was given to a sequence must not matter.
        self.cache.codes.fill_(93)
        self.cache.scales.fill_(1e30)
        self.lengths = list(lengths)
        self.status = StatusWord(torch.device("cuda", 0))

    def rows(self, n, heads, dtype, scale=1.0):
        return (torch.randn(n, heads, self.dim, generator=self.g) * scale).to(dtype)

    def device(self, lengths, starts=None):
        return (self.table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                None if starts is None else torch.tensor(starts, dtype=torch.int32,
                                                         device="cuda"))

    def write(self, new, lengths, dtype=torch.float32, scale=1.0, **kw):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        k, v = (self.rows(starts[-1], self.heads, dtype, scale) for _ in range(2))
        self.host.write(k, v, self.table, lengths, starts)
        table, at, first = self.device(lengths, starts)
        self.cache.write(k.cuda(), v.cuda(), table, at, first, status=self.status, **kw)
        return k, v

    def fill(self, dtype=torch.float32, scale=1.0):
        """Writes every sequence whole."""
        self.write(self.lengths, self.lengths, dtype, scale)

    def check_read(self, dtype=torch.float32):
        starts = [0]
        for n in self.lengths:
            starts.append(starts[-1] + n)
        table, at, first = self.device(self.lengths, starts)
        got = self.cache.read(table, at, first, tokens=starts[-1], dtype=dtype,
                              status=self.status)
        self.status.raise_if_set()
        for side in range(2):
            want = torch.cat([self.host.values(self.table[b], n, side)
                              for b, n in enumerate(self.lengths)])
            # Codes and scales are defined to the bit, and so are values.
            assert torch.equal(got[side].cpu(), want.float().to(dtype))

    def check_attend(self, new, dtype, causal=True, window=0, group=2, scale=None, starts="rows",
                     q=None, **kw):
        heads = self.heads * group
        total = sum(new)
        q = self.rows(total, heads, dtype) if q is None else q
        first = [0]
        for n in new:
            first.append(first[-1] + n)
        table, at, dev_starts = self.device(self.lengths, first if starts == "rows" else None)
        # Rows behind the last sequence choose the kernel: as given, more than
        # the decode kernel takes, and enough that the keys are not split.
        runs = []
        for least in (0, 7200, 38000) if starts == "rows" else (0,):
            pad = max(0, least // (heads * len(new)) + 1 - total) if least else 0
            more = torch.cat([q, torch.full((pad, heads, self.dim), math.nan, dtype=dtype)])
            out, lse = self.cache.attend(more.cuda(), table, at, dev_starts, causal=causal,
                                         window=window, scale=scale, return_lse=True,
                                         status=self.status, **kw)
            self.status.raise_if_set()
            runs.append((out[:total], lse[:total]))
        parts = 2 if dtype == torch.float32 else 1
        step = 2.0 ** -22  # one product or sum of the tensor cores, truncation allowed for
        # A probability is off by half a step of f16 (one part) or of its two
        # parts' 22 bits; weights and their sum both carry it.
        p_err = torch.finfo(torch.float16).eps / 2 if parts == 1 else step
        # Far below the largest, a probability (times its block's value scale)
        # is off by half a step of f16's subnormals, 2^-25, where the largest is
        # at least 2^6 (one part) or 2^13; it multiplies a code of at most 127.
        floor = 127 * 2.0 ** (-31 if parts == 1 else -38)
        for b, n in enumerate(new):
            keys = self.lengths[b]
            k, v = (self.host.values(self.table[b], keys, side) for side in range(2))
            s = self.dim ** -0.5 if scale is None else scale
            want, want_lse, size, reach, peak = ref.attend(
                q[first[b]:first[b + 1]], k, v, keys - n, s, causal, window,
                self.host.value_scales(self.table[b], keys))
            # Score error: the contraction's steps, the queries' parts and the
            # exponent's own rounding (arguments below 128).
            delta = (parts * (self.dim / 16) + 6) * step * reach + 130 * 2.0 ** -24
            steps = (keys / 16 + 70) * step
            tol = torch.finfo(dtype).eps / 2 * want.abs() + size * (
                2 * p_err + 2 * delta + steps)[..., None] + floor * peak[..., None]
            if dtype == torch.float16:
                tol = tol + 2.0 ** -25
            seen = torch.isfinite(want_lse)
            lse_tol = delta + steps + 2.0 ** -23 * want_lse.abs()
            for run, (out, lse) in enumerate(runs):
                got = out[first[b]:first[b + 1]].double().cpu()
                got_lse = lse[first[b]:first[b + 1]].double().cpu()
                off = (got - want).abs()
                assert bool((off <= tol).all()), (
                    run, b, float((off / tol.clamp(min=1e-300)).max()))
                assert torch.equal(seen, torch.isfinite(got_lse))
                assert bool((got_lse[~seen] == -math.inf).all())
                assert bool(((got_lse - want_lse).abs() <= lse_tol)[seen].all())
        return runs[0][0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block,dim,heads", [(16, 16, 1), (32, 80, 3), (64, 128, 2), (128, 48, 2)])
def test_write_and_read_back(dtype, block, dim, heads):
    s = Setup([1, block - 1, block, block + 1, 3 * block + 5, 0, 2], heads, dim, block)
    s.fill(dtype)
    s.check_read(dtype)
    s.check_read()


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_token_by_token_equals_the_definition(block, dtype):
    """Scales grow and earlier codes are rounded again as tokens arrive."""
    s = Setup([block + 3, 0, 2 * block], 2, 32, block)
    for t in range(2 * block):
        lengths = [min(t + 1, s.lengths[0]), 0, t + 1]
        new = [1 if t < s.lengths[0] else 0, 0, 1]
        s.write(new, lengths, dtype, scale=1.0 + t % 7)
    s.check_read()


def test_decode_rows_without_starts_and_an_empty_slot():
    s = Setup([5, 0, 40], 1, 16, 16)
    s.write([4, 0, 39], [4, 0, 39])
    k, v = s.rows(3, 1, torch.float32), s.rows(3, 1, torch.float32)
    s.host.write(k, v, s.table, s.lengths, [0, 1, 2, 3])
    table, at, _ = s.device(s.lengths)
    before = s.cache.codes.clone()
    s.cache.write(k.cuda(), v.cuda(), table, at, status=s.status)
    changed = (s.cache.codes != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {int(s.table[0, 0]), int(s.table[2, 2])}
    s.check_read()


def test_chunked_prompt_writes_join():
    s = Setup([150, 70], 2, 64, 32)
    s.write([40, 70], [40, 70], torch.bfloat16)
    s.write([61, 0], [101, 70], torch.bfloat16)
    s.write([49, 0], [150, 70], torch.bfloat16)
    s.check_read(torch.bfloat16)


def test_values_of_all_sizes_and_not_finite():
    s = Setup([64], 1, 16, 16)
    k = torch.zeros(64, 1, 16)
    k[0:16] = torch.linspace(-3e38, 3e38, 256).view(16, 1, 16)  # the largest
    k[16:32] = torch.linspace(-1e-38, 1e-38, 256).view(16, 1, 16)  # below the floor
    k[40, 0, 3], k[41, 0, 4], k[42, 0, 5], k[43] = math.nan, math.inf, -math.inf, 2.5
    v = torch.zeros(64, 1, 16)  # all zero: codes zero
    s.host.write(k, v, s.table, [64], [0, 64])
    table, at, first = s.device([64], [0, 64])
    s.cache.write(k.cuda(), v.cuda(), table, at, first, status=s.status)
    with pytest.raises(RuntimeError, match="does not support NaN or infinity"):
        s.status.raise_if_set()
    s.status.reset()
    s.check_read()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_a_fused_projection(dtype):
    """Strided views, rows off a 16-byte boundary too."""
    s = Setup([37, 20], 2, 32, 16)
    for base, pad, more in ((0, 0, 0), (3, 1, 0), (0, 0, 4000), (3, 1, 4000)):
        flat = torch.randn(57 * (6 * 32 + pad) + 8, generator=s.g).to(dtype)
        fused = flat.as_strided((57, 6, 32), (6 * 32 + pad, 32, 1), base)
        k, v = fused[:, 2:4], fused[:, 4:6]
        s.host.write(k, v, s.table, s.lengths, [0, 37, 57])
        dev = flat.cuda().as_strided((57, 6, 32), (6 * 32 + pad, 32, 1), base)
        table, at, first = s.device(s.lengths, [0, 37, 57])
        s.cache.write(dev[:, 2:4], dev[:, 4:6], table, at, first, status=s.status)
        s.check_read(dtype)
        q = dev[:, 0:2]
        if more: # rows behind the last sequence: the prompt kernel
            q = torch.empty(base + (57 + more) * (6 * 32 + pad), dtype=dtype, device="cuda"
                            ).as_strided((57 + more, 2, 32), (6 * 32 + pad, 32, 1), base)
            q[:57] = dev[:, 0:2]
        want = s.cache.attend(q.contiguous(), table, at, first, status=s.status)
        got = s.cache.attend(q, table, at, first, status=s.status)
        assert torch.equal(got[:57], want[:57])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,block", [(16, 16), (64, 32), (80, 16), (128, 64), (112, 128)])
def test_decode(dtype, dim, block):
    s = Setup([1, 2, 15, 16, 17, 0, 63, 64, 200], 2, dim, block)
    s.fill()
    s.check_attend([1] * 9, dtype, group=4, starts=None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [1, 3, 8])
def test_chunks_and_prompts(dtype, group):
    s = Setup([5, 33, 130, 260, 0], 1, 64, 32)
    s.fill()
    s.check_attend([5, 2, 130, 17, 0], dtype, group=group)
    s.check_attend([1, 33, 64, 129, 0], dtype, group=group)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [1, 5, 16, 100])
def test_windows(causal, window):
    s = Setup([7, 90, 300], 1, 128, 16)
    s.fill()
    s.check_attend([7, 30, 140], torch.bfloat16, causal=causal, window=window)
    s.check_attend([1, 1, 1], torch.float32, causal=causal, window=window, starts=None)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_queries_than_tokens_leaves_empty_rows(dtype):
    s = Setup([3, 0, 20], 2, 32, 16)
    s.fill()
    out = s.check_attend([5, 4, 20], dtype)
    assert bool((out[:2] == 0).all()) and bool((out[5:9] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_long_axis_is_split_and_joined(dtype):
    s = Setup([3000], 1, 64, 64)
    s.fill()
    s.check_attend([1], dtype, group=2, starts=None)
    s.check_attend([1], dtype, group=2, starts=None, longest=64)
    s.check_attend([1], dtype, group=2, starts=None, window=700)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [48, 128])
def test_a_chunk_against_a_long_context(dtype, dim):
    """Many tiles of keys for each of a CTA's two query streams (f32 takes its
    sums out of the accumulators between them), one part and several."""
    s = Setup([2900], 1, dim, 32)
    s.fill()
    s.check_attend([40], dtype, group=2, longest=1024)
    s.check_attend([40], dtype, group=2)
    s.check_attend([150], dtype, group=2, longest=1024, window=1500)


@pytest.mark.parametrize("dtype", TYPES)
def test_chunks_of_many_sequences(dtype):
    """One tile of at most 128 query rows for both streams of a CTA."""
    s = Setup([700, 704, 513, 130, 700, 0, 64, 129], 16, 32, 32)
    s.fill()
    s.check_attend([40, 33, 40, 40, 1, 0, 40, 17], dtype, group=1, most=40)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_large_score_late_in_the_context(dtype):
    """References are set again in the middle of the keys, for some rows only."""
    s = Setup([700], 1, 64, 64)
    k, v = s.rows(700, 1, torch.float32), s.rows(700, 1, torch.float32)
    k[300] *= 12
    k[600] *= 40
    s.host.write(k, v, s.table, [700], [0, 700])
    table, at, first = s.device([700], [0, 700])
    s.cache.write(k.cuda(), v.cuda(), table, at, first, status=s.status)
    s.check_attend([1], dtype, group=8, starts=None)
    s.check_attend([90], dtype, group=2)


@pytest.mark.parametrize("dtype", TYPES)
def test_an_empty_cache(dtype):
    cache = Int8KVCache(0, 1, 32, 16)
    status = StatusWord(torch.device("cuda", 0))
    table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    at = torch.zeros(2, dtype=torch.int32, device="cuda")
    for n in (1, 40, 3000):
        first = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
        q = torch.ones(2 * n, 2, 32, dtype=dtype, device="cuda")
        out, lse = cache.attend(q, table, at, first, return_lse=True, status=status)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    status.raise_if_set()
    none = cache.attend(q[:0], table[:0], at[:0], status=status)
    assert none.shape == (0, 2, 32)


def test_more_query_tiles_than_one_grid_axis_holds():
    """32,767 kv heads x 3 tiles of 128 rows; a head's results are those it has
    in a cache by itself."""
    g = torch.Generator(device="cuda").manual_seed(3)
    codes = torch.randint(-127, 128, (1, 32767, 2, 16, 16), generator=g, device="cuda",
                          dtype=torch.int8)
    scales = torch.rand(1, 32767, 2, generator=g, device="cuda") * 0.02 + 0.01
    q = torch.randn(257, 1, 16, generator=g, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    at = torch.tensor([16], dtype=torch.int32, device="cuda")
    first = torch.tensor([0, 257], dtype=torch.int32, device="cuda")
    out = Int8KVCache.over(codes, scales).attend(q.expand(257, 32767, 16), table, at, first,
                                                 causal=False)
    more = torch.cat([q, torch.zeros(8000, 1, 16, device="cuda")])  # the same kernel's
    for h in (0, 1, 21844, 21845, 32766):
        one = Int8KVCache.over(codes[:, h:h + 1].contiguous(), scales[:, h:h + 1].contiguous())
        assert torch.equal(out[:, h:h + 1],
                           one.attend(more, table, at, first, causal=False)[:257])


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_that_differ_by_blocks(dtype):
    """Value scales 1e-6 to 1e6 and key scales apart: probabilities carry the
    value scale in their exponent."""
    s = Setup([128], 1, 32, 16)
    k = s.rows(128, 1, torch.float32)
    v = s.rows(128, 1, torch.float32)
    for i in range(8):
        v[16 * i:16 * i + 16] *= 10.0 ** (3 - i if i % 2 else i - 6)
        k[16 * i:16 * i + 16] *= 2.0 ** (i - 4)
    s.host.write(k, v, s.table, [128], [0, 128])
    table, at, first = s.device([128], [0, 128])
    s.cache.write(k.cuda(), v.cuda(), table, at, first, status=s.status)
    s.check_attend([128], dtype, group=1)
    s.check_attend([1], dtype, group=1, starts=None)
    for new in (3, 128):
        s.check_attend([new], dtype, group=1, scale=-0.3)
        s.check_attend([new], dtype, group=1, scale=0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_of_all_sizes(dtype):
    s = Setup([40], 1, 48, 16)
    s.fill()
    q = s.rows(40, 2, dtype)
    q[0] = 0
    q[1] *= 1e-6
    q[2] *= 100
    q[3, 0, 0] = 300
    s.check_attend([40], dtype, q=q)


@pytest.mark.parametrize("rows", [20, 4000])
def test_not_finite_queries_stay_in_their_rows(rows):
    s = Setup([40], 1, 32, 16)
    s.fill()
    q = s.rows(rows, 2, torch.float32)
    clean = q.clone()
    q[3, 0, 5], q[7, 1, 0] = math.nan, math.inf
    table, at, first = s.device([40], [0, 20])
    got = s.cache.attend(q.cuda(), table, at, first, status=s.status)
    want = s.cache.attend(clean.cuda(), table, at, first, status=s.status)
    assert bool(torch.isnan(got[3, 0]).all()) and bool(torch.isnan(got[7, 1]).all())
    keep = torch.ones(20, 2, dtype=torch.bool)
    keep[3, 0] = keep[7, 1] = False
    assert torch.equal(got[:20].cpu()[keep], want[:20].cpu()[keep])


def test_rows_behind_the_last_sequence_are_left():
    s = Setup([20, 9], 1, 16, 16)
    s.fill()
    table, at, first = s.device(s.lengths, [0, 6, 9])
    for rows in (15, 3000):
        q = s.rows(rows, 2, torch.float32).cuda()
        out = torch.full((rows, 2, 16), 5.0, device="cuda")
        s.cache.attend(q, table, at, first, out=out, status=s.status)
        assert bool((out[9:] == 5).all()) and not bool((out[:9] == 5).any())
    k = torch.full((15, 1, 16), 5.0, device="cuda")
    v = k.clone()
    s.cache.read(table, at, first, out=(k, v), status=s.status)
    assert bool((k[9:] == 5).all()) and bool((v[9:] == 5).all())
    s.status.raise_if_set()


def bad_descriptions(s):
    table, at, first = s.device(s.lengths, [0, 6, 9])
    high = table.clone()
    high[0, 0] = s.cache.pages
    low = table.clone()
    low[0, 0] = -5
    long = at.clone()
    long[0] = 16 * table.shape[1] + 1
    negative = at.clone()
    negative[0] = -1
    back = first.clone()
    back[1] = -3
    past = first.clone()
    past[2] = 2001
    return {"page past the cache": (high, at, first), "negative page": (low, at, first),
            "length past the table": (table, long, first), "negative length": (table, negative, first),
            "starts run backwards": (table, at, back), "starts past the rows": (table, at, past)}


@pytest.mark.parametrize("which", ["page past the cache", "negative page", "length past the table",
                                   "negative length", "starts run backwards",
                                   "starts past the rows"])
@pytest.mark.parametrize("rows", [9, 2000])
def test_bad_descriptions_are_reported_not_followed(which, rows):
    s = Setup([12, 9], 1, 16, 16)
    s.fill()
    s.status.raise_if_set()
    table, at, first = bad_descriptions(s)[which]
    q = s.rows(rows, 2, torch.float32).cuda()
    k = s.rows(9, 1, torch.float32).cuda()
    calls = [lambda: s.cache.attend(q, table, at, first, status=s.status),
             lambda: s.cache.read(table, at, first, tokens=9, status=s.status),
             lambda: s.cache.write(k, k, table, at, first, status=s.status)]
    for call in calls:
        s.status.reset()
        call()
        with pytest.raises(RuntimeError, match="page, length or start out of range"):
            s.status.raise_if_set()
    # More rows in a sequence than the host said.
    table, at, first = s.device(s.lengths, [0, 6, 9])
    s.status.reset()
    s.cache.attend(q, table, at, first, most=5, status=s.status)
    with pytest.raises(RuntimeError, match="page, length or start out of range"):
        s.status.raise_if_set()


def test_offsets_past_32_bits():
    """A cache of more than 2^31 codes: its last pages."""
    block, heads, dim = 128, 8, 128
    pages = 2 ** 31 // (heads * 2 * block * dim) + 3
    cache = Int8KVCache(pages, heads, dim, block)
    table = torch.tensor([[pages - 1, 0], [pages - 2, 1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([200, 130], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 200, 330], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(330, heads, dim, generator=g, device="cuda") for _ in range(2))
    cache.write(k, v, table, lengths, starts)
    got = cache.read(table, lengths, starts, tokens=330)
    small = Int8KVCache(4, heads, dim, block)
    near = torch.tensor([[3, 0], [2, 1]], dtype=torch.int32, device="cuda")
    small.write(k, v, near, lengths, starts)
    want = small.read(near, lengths, starts, tokens=330)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = torch.randn(330, 16, dim, generator=g, device="cuda")
    assert torch.equal(cache.attend(q, table, lengths, starts),
                       small.attend(q, near, lengths, starts))


def test_captured_step_takes_new_contents():
    """Write and attention of a decoding step in one graph, replayed as the
    sequences grow; two graphs with one workspace, one after the other."""
    s = Setup([600, 300], 2, 64, 32, width=30)
    s.lengths = [600, 300]
    s.fill()
    table, at, _ = s.device(s.lengths)
    workspace = Workspace(torch.device("cuda", 0))
    q = torch.zeros(2, 4, 64, device="cuda")
    kv = torch.zeros(2, 4, 64, device="cuda")

    def step():
        s.cache.write(kv[:, :2], kv[:, 2:], table, at, status=s.status)
        return s.cache.attend(q, table, at, workspace=workspace, status=s.status)

    # New tokens go to pages of their own: the table has room for 30 pages a row.
    spare = Int8KVCache(s.cache.pages + 40, 2, 64, 32)
    spare.codes[:s.cache.pages] = s.cache.codes
    spare.scales[:s.cache.pages] = s.cache.scales
    old = s.cache.pages
    s.cache = spare
    for b, used in enumerate((19, 10)):
        for i in range(used, 30):
            table[b, i] = old + 11 * b + i - used
    at += 1
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(40):
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        kv.copy_(torch.randn(kv.shape, generator=g, device="cuda"))
        at += 1
        graph, out = graphs[i % 2]
        graph.replay()
        want = s.cache.attend(q, table, at, status=s.status)
        assert torch.equal(out, want)
    s.status.raise_if_set()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("longest", [300, 40000])
def test_captured_prompt_takes_new_contents(dtype, longest):
    s = Setup([300, 90], 2, 128, 64, width=700)
    s.fill()
    table, at, first = s.device(s.lengths, [0, 70, 120])
    workspace = Workspace(torch.device("cuda", 0))
    q = s.rows(120, 4, dtype).cuda()

    def step():
        return s.cache.attend(q, table, at, first, most=70, longest=longest,
                              workspace=workspace, status=s.status)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in (300, 250, 71):
        q.copy_(s.rows(120, 4, dtype))
        at[0] = n
        graph.replay()
        assert torch.equal(out, s.cache.attend(q, table, at, first, most=70, longest=longest,
                                               status=s.status))
    s.status.raise_if_set()


def test_results_repeat_and_do_not_hang_on_streams():
    s = Setup([900, 40, 300], 2, 128, 64)
    s.fill()
    q = s.rows(1240, 8, torch.bfloat16).cuda()
    table, at, first = s.device(s.lengths, [0, 900, 940, 1240])
    want = s.cache.attend(q, table, at, first, status=s.status)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append(s.cache.attend(q, table, at, first, status=s.status))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("call", [
    lambda s, q, k, t, n, st: s.cache.attend(q.double(), t, n, st),
    lambda s, q, k, t, n, st: s.cache.attend(q[..., :8], t, n, st),
    lambda s, q, k, t, n, st: s.cache.attend(q[:, :1].repeat(1, 3, 1), t, n, st),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n, st, window=-1),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n, st, scale=math.inf),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n, st, longest=-1),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n, st, most=-1),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n),
    lambda s, q, k, t, n, st: s.cache.attend(q, t.long(), n, st),
    lambda s, q, k, t, n, st: s.cache.attend(q, t.t(), n, st),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n.cpu(), st),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n, st[:2]),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n, st, out=q.half()),
    lambda s, q, k, t, n, st: s.cache.attend(q.cpu(), t, n, st),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n, st, out=q),
    lambda s, q, k, t, n, st: s.cache.attend(q, t, n, st,
                                             workspace=Workspace(torch.device("cpu"))),
    lambda s, q, k, t, n, st: s.cache.write(k, k.half(), t, n, st),
    lambda s, q, k, t, n, st: s.cache.write(k, k[:8], t, n, st),
    lambda s, q, k, t, n, st: s.cache.write(q, q, t, n, st),
    lambda s, q, k, t, n, st: s.cache.read(t, n, st),
    lambda s, q, k, t, n, st: s.cache.read(t, n, st, tokens=9, dtype=torch.int8),
    lambda s, q, k, t, n, st: Int8KVCache(4, 2, 24),
    lambda s, q, k, t, n, st: Int8KVCache(4, 2, 144),
    lambda s, q, k, t, n, st: Int8KVCache(4, 2, 64, 48),
    lambda s, q, k, t, n, st: Int8KVCache(4, 0, 64),
    lambda s, q, k, t, n, st: Int8KVCache.over(s.cache.codes[:, :, :1], s.cache.scales),
    lambda s, q, k, t, n, st: Int8KVCache.over(s.cache.codes.float(), s.cache.scales),
    lambda s, q, k, t, n, st: Int8KVCache.over(s.cache.codes, s.cache.scales.half()),
    lambda s, q, k, t, n, st: Int8KVCache.over(s.cache.codes, s.cache.scales[:1]),
])
def test_refusals(call):
    s = Setup([20, 9], 2, 16, 16)
    q, k = s.rows(9, 4, torch.float32).cuda(), s.rows(9, 2, torch.float32).cuda()
    table, at, first = s.device(s.lengths, [0, 6, 9])
    with pytest.raises((TypeError, ValueError)):
        call(s, q, k, table, at, first)


def test_a_decoder_block_of_cim_layers():
    """Norm, CIM projections, cache, attention and the gated residual as one
    block, prompt then single tokens, against the same block in 64 bits around
    the same CIM layers."""
    dev = torch.device("cuda", 0)
    g = torch.Generator().manual_seed(0)
    width, heads, kv_heads, dim, block = 96, 4, 2, 32, 16
    wq = (torch.randn((heads + 2 * kv_heads) * dim, width, generator=g) * 0.1).numpy()
    wo = (torch.randn(width, heads * dim, generator=g) * 0.1).numpy()
    qkv_layer, out_layer = CimLayer(wq, device=dev), CimLayer(wo, device=dev)
    pre, post = (Norm("rms", 1 + 0.1 * torch.randn(width, generator=g).to(dev)) for _ in range(2))
    gate = torch.randn(width, generator=g).to(dev)
    cache, host = Int8KVCache(8, kv_heads, dim, block), ref.Cache(8, kv_heads, dim, block)
    table = torch.arange(8, dtype=torch.int32).view(2, 4).to(dev)
    status, workspace = StatusWord(dev), Workspace(dev)
    lengths = [0, 0]
    for new in ([21, 9], [1, 1], [1, 1], [4, 2]):
        total = sum(new)
        starts = [0, new[0], total]
        lengths = [n + a for n, a in zip(lengths, new)]
        x = torch.randn(total, width, generator=g).to(dev)
        at = torch.tensor(lengths, dtype=torch.int32, device=dev)
        first = torch.tensor(starts, dtype=torch.int32, device=dev)
        _, y = block_norm(x, pre=pre)
        qkv = qkv_layer.linear_bf16(y, status=status).view(total, -1, dim)
        q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
        cache.write(k, v, table, at, first, status=status)
        o = cache.attend(q, table, at, first, workspace=workspace, status=status)
        f = out_layer.linear_bf16(o.view(total, -1), status=status)
        h, y2 = block_norm(f, x, post=post, pre=pre, gate=gate, gate_activation="sigmoid")
        status.raise_if_set()

        # Each stage against 64 bits on its own inputs: the f32 stages differ
        # from it by roundings of 2^-24 of their terms (at most a few hundred).
        near = dict(rtol=2.0 ** -16, atol=2.0 ** -16)
        assert torch.allclose(y.double(), ref.norm(x.double(), "rms", pre.weight), **near)
        host.write(k.cpu(), v.cpu(), table.cpu(), lengths, starts)
        for b in range(2):
            held = [host.values(table.cpu()[b], lengths[b], side) for side in range(2)]
            want = ref.attend(q[starts[b]:starts[b + 1]].cpu(), *held, lengths[b] - new[b],
                              dim ** -0.5, True, 0)[0]
            assert torch.allclose(o[starts[b]:starts[b + 1]].cpu().double(), want, **near)
        stream = x.double() + torch.sigmoid(gate.double()) * ref.norm(f.double(), "rms", post.weight)
        assert torch.allclose(h.double(), stream, **near)
        assert torch.allclose(y2.double(), ref.norm(stream, "rms", pre.weight), **near)


def test_copies_of_a_cache_are_caches_of_their_own():
    s = Setup([20, 9], 2, 16, 16)
    s.fill()
    table, at, first = s.device(s.lengths, [0, 20, 29])
    want = s.cache.read(table, at, first, tokens=29)
    for other in (copy.deepcopy(s.cache), pickle.loads(pickle.dumps(s.cache))):
        codes, scales = s.cache.codes.clone(), s.cache.scales.clone()
        got = other.read(table, at, first, tokens=29)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        k = s.rows(29, 2, torch.float32).cuda()
        other.write(k, k, table, at, first)
        assert torch.equal(s.cache.codes, codes) and torch.equal(s.cache.scales, scales)
        assert not torch.equal(other.codes, codes)
    same = copy.copy(s.cache)
    assert same.codes is s.cache.codes and same.scales is s.cache.scales


def test_a_status_word_on_the_host_is_refused():
    s = Setup([20, 9], 2, 16, 16)
    q, k = s.rows(9, 4, torch.float32).cuda(), s.rows(9, 2, torch.float32).cuda()
    table, at, first = s.device(s.lengths, [0, 6, 9])
    host = StatusWord(torch.device("cpu"))
    for call in (lambda: s.cache.attend(q, table, at, first, status=host),
                 lambda: s.cache.read(table, at, first, tokens=9, status=host),
                 lambda: s.cache.write(k, k, table, at, first, status=host)):
        with pytest.raises(ValueError, match="status"):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 3, 2 ** 31 - 1])
def test_windows_of_any_width_with_rows_before_the_start(dtype, causal, window):
    """Positions down to -8 less the window do not fit 32 bits."""
    s = Setup([2, 16, 0, 60], 2, 32, 16)
    s.fill()
    s.check_attend([5, 24, 4, 60], dtype, causal=causal, window=window)


def check_far_scales(s, q, length, causal, paddings, bounds):
    """As check_attend, but a block's log2 of its scale is below 128 and off by up
    to an ulp, 2^-17, as is the exponent that it goes into; so is the logarithm
    of the sum of weights over scales in lse."""
    new, heads, dtype = q.shape[0], q.shape[1], q.dtype
    table, at, first = s.device([length], [0, new])
    held = [s.host.values(s.table[0], length, side) for side in range(2)]
    want, want_lse, size, reach, peak = ref.attend(
        q, *held, length - new, s.dim ** -0.5, causal, 0,
        s.host.value_scales(s.table[0], length))
    parts = 2 if dtype == torch.float32 else 1
    step = 2.0 ** -22
    p_err = torch.finfo(torch.float16).eps / 2 if parts == 1 else step
    delta = (parts * (s.dim / 16) + 6) * step * reach + 2 * 2.0 ** -17
    steps = (length / 16 + 70) * step
    tol = torch.finfo(dtype).eps / 2 * want.abs() + size * (
        2 * p_err + 2 * delta + steps)[..., None] + (
        127 * 2.0 ** (-31 if parts == 1 else -38)) * peak[..., None]
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    lse_tol = delta + steps + 2 * 2.0 ** -17
    for rows in paddings:
        more = torch.cat([q, torch.full((rows - new, heads, s.dim), math.nan, dtype=dtype)])
        for longest in bounds:
            out, lse = s.cache.attend(more.cuda(), table, at, first, causal=causal,
                                      longest=longest, return_lse=True, status=s.status)
            s.status.raise_if_set()
            off = (out[:new].double().cpu() - want).abs()
            assert bool((off <= tol).all()), (
                rows, longest, float((off / tol.clamp(min=1e-300)).max()))
            lse_off = (lse[:new].double().cpu() - want_lse).abs()
            assert bool((lse_off <= lse_tol).all()), (rows, longest, float(lse_off.max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["small first", "large first", "mixed"])
@pytest.mark.parametrize("new", [1, 40])
def test_value_scales_further_apart_than_exponents_reach(dtype, order, new):
    """Blocks of zeros (the least scale, 2^-87) beside values near 1e30 (65,000
    for f16): every key's weight counts, whatever its block's scale."""
    n, large = 1120, 6e4 if dtype == torch.float16 else 1e30
    s = Setup([n], 1, 32, 16)
    k, v = s.rows(n, 1, torch.float32), s.rows(n, 1, torch.float32).clamp(-1, 1)
    sizes = torch.tensor({"small first": [0, 0, 1e-20, 1, 0, large, 0],
                          "large first": [large, 0, 0, 1, 1e-20, 0, 0],
                          "mixed": [0, large, 0, 0, large, 1e-20, 0]}[order])
    if order == "mixed":
        sizes = sizes.repeat(10)  # every block of another size
    v *= sizes.repeat_interleave(n // len(sizes))[:, None, None]
    s.host.write(k, v, s.table, [n], [0, n])
    table, at, first = s.device([n], [0, n])
    s.cache.write(k.cuda(), v.cuda(), table, at, first, status=s.status)
    q = s.rows(new, 2, dtype)
    for causal, length in ((True, n), (False, n), (True, n // 7 * 2)):
        check_far_scales(s, q, length, causal, (new, 7200, 38000), (64, n))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", [3, 580])
def test_one_block_of_large_values_in_a_long_context(dtype, where):
    """More pages than a CTA of the prompt kernel has threads to look at them."""
    n = 600 * 16
    s = Setup([n], 1, 16, 16)
    k, v = s.rows(n, 1, torch.float32) * 0.5, torch.zeros(n, 1, 16)
    v[16 * where:16 * where + 16] = 1e30
    s.host.write(k, v, s.table, [n], [0, n])
    table, at, first = s.device([n], [0, n])
    s.cache.write(k.cuda(), v.cuda(), table, at, first, status=s.status)
    check_far_scales(s, s.rows(40, 1, dtype), n, True, (40, 38000), (64, n))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 4000, 38000])
@pytest.mark.parametrize("causal", [True, False])
def test_a_not_finite_query_that_sees_nothing_gives_zeros(dtype, rows, causal):
    """Rows before the start, in one tile with rows that see keys."""
    s = Setup([3], 2, 32, 16)
    s.fill()
    table, at, first = s.device([3], [0, 5])
    q = torch.zeros(rows, 4, 32, dtype=dtype)
    q[:5] = s.rows(5, 4, dtype)
    clean = q.clone()
    q[0], q[1, :, 3], q[3, 1, 2] = math.nan, math.inf, -math.inf
    kw = dict(return_lse=True, causal=causal, window=0 if causal else 2, status=s.status)
    out, lse = s.cache.attend(q.cuda(), table, at, first, **kw)
    want, want_lse = s.cache.attend(clean.cuda(), table, at, first, **kw)
    s.status.raise_if_set()
    blind = 2 if causal else 0  # without a causal mask every row sees what follows it
    assert bool((out[:blind] == 0).all()) and bool((lse[:blind] == -math.inf).all())
    assert bool(torch.isnan(out[3, 1]).all()) and bool(torch.isnan(lse[3, 1]))
    assert torch.equal(out[2], want[2]) and torch.equal(out[4], want[4])
    assert torch.equal(lse[2], want_lse[2]) and torch.equal(lse[4], want_lse[4])
    if not causal:
        assert bool(torch.isnan(out[:2]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,longest", [(9, 20), (3000, 20), (3000, 100000)])
def test_no_rows_to_a_sequence(dtype, rows, longest):
    """A bound of no rows: nothing to do where there are none, an index error
    where there are some."""
    s = Setup([20, 9], 1, 16, 16, width=7000)
    s.fill()
    q = s.rows(rows, 2, dtype).cuda()
    k = s.rows(rows, 1, dtype).cuda()
    out = torch.full_like(q, 5.0)
    pair = torch.full_like(k, 5.0), torch.full_like(k, 5.0)
    for starts, error in (([0, 0, 0], False), ([0, 6, 9], True)):
        table, at, first = s.device(s.lengths, starts)
        codes = s.cache.codes.clone()
        for call in (lambda: s.cache.attend(q, table, at, first, most=0, longest=longest, out=out,
                                            status=s.status),
                     lambda: s.cache.read(table, at, first, most=0, out=pair, status=s.status),
                     lambda: s.cache.write(k, k, table, at, first, most=0, status=s.status)):
            call()
            if error:
                with pytest.raises(RuntimeError, match="page, length or start out of range"):
                    s.status.raise_if_set()
                s.status.reset()
            s.status.raise_if_set()
        assert all(bool((t == 5).all()) for t in (out, *pair))
        assert torch.equal(s.cache.codes, codes)


@pytest.mark.parametrize("most", [31, 1000, 2 ** 31 - 1])
def test_a_bound_of_rows_past_those_there_are(most):
    s = Setup([20, 31], 1, 16, 16)
    s.fill()
    table, at, first = s.device(s.lengths, [0, 20, 51])
    q, k = s.rows(51, 4, torch.float32).cuda(), s.rows(51, 1, torch.float32).cuda()
    want = s.cache.attend(q, table, at, first, most=31, status=s.status)
    assert torch.allclose(s.cache.attend(q, table, at, first, most=most, status=s.status), want,
                          rtol=2.0 ** -18, atol=2.0 ** -18)
    s.cache.write(k, k, table, at, first, most=most, status=s.status)
    got = s.cache.read(table, at, first, tokens=51, most=most, status=s.status)
    assert torch.equal(got[0], got[1])
    s.status.raise_if_set()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim,block", [(1, 16, 16), (3, 80, 32)])
def test_rows_before_the_start_read_as_zeros(dtype, heads, dim, block):
    s = Setup([5, 0, 70, 3, 2 * block], heads, dim, block)
    s.fill()
    new = [9, 40, 70, 1, 3 * block + 1]
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    table, at, starts = s.device(s.lengths, first)
    k, v = (torch.full((first[-1] + 6, heads, dim), 5.0, dtype=dtype, device="cuda")
            for _ in range(2))
    s.cache.read(table, at, starts, out=(k, v), status=s.status)
    s.status.raise_if_set()
    for side, got in enumerate((k, v)):
        for b, n in enumerate(new):
            want = torch.zeros(max(0, n - s.lengths[b]), heads, dim, dtype=dtype)
            held = s.host.values(s.table[b], s.lengths[b], side)[-n:].float().to(dtype)
            assert torch.equal(got[first[b]:first[b + 1]].cpu(), torch.cat([want, held]))
        assert bool((got[first[-1]:] == 5).all())
    # An empty slot of a fixed batch.
    k, v = (torch.full((5, heads, dim), 5.0, dtype=dtype, device="cuda") for _ in range(2))
    s.cache.read(table, at, out=(k, v), status=s.status)
    assert bool((k[1] == 0).all()) and bool((v[1] == 0).all())
    assert not bool((k == 5).all(-1).any())


@pytest.mark.parametrize("dim", [48, 128])
def test_a_low_bound_of_lengths_costs_no_accuracy(dim):
    """f32 prompts take their sums out of the accumulators by what the table can
    hold: with one part of the key axis either way, the bits are the same."""
    s = Setup([2900], 1, dim, 32)
    s.fill()
    table, at, first = s.device([2900], [0, 40])
    q = torch.zeros(38000, 2, dim)
    q[:40] = s.rows(40, 2, torch.float32)
    q = q.cuda()
    want, want_lse = s.cache.attend(q, table, at, first, return_lse=True, status=s.status)
    for longest in (0, 64, 512, 2900, 10 ** 6):
        out, lse = s.cache.attend(q, table, at, first, return_lse=True, longest=longest,
                                  status=s.status)
        assert torch.equal(out[:40], want[:40]) and torch.equal(lse[:40], want_lse[:40])
    s.status.raise_if_set()


def test_a_workspace_stays_on_its_device():
    """A device without an index is the one that was current at the start."""
    workspace = Workspace(torch.device("cuda"))
    assert workspace.device == torch.device("cuda", torch.cuda.current_device())
    assert workspace.get(1 << 20).device == workspace.device


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new", [1, 64])
def test_a_key_of_all_the_weight_loses_nothing(dtype, new):
    """Its probability is a power of two when the reference is set by it, so that
    rounding it to f16 costs nothing: the output is the value, rounded once
    (2^-16 for its exponent, below 512 and so off by up to 2^-16, twice)."""
    s = Setup([64], 1, 64, 16)
    k, v = s.rows(64, 1, torch.float32), s.rows(64, 1, torch.float32)
    s.host.write(k, v, s.table, [64], [0, 64])
    table, at, first = s.device([64], [0, new])
    s.cache.write(k.cuda(), v.cuda(), *s.device([64], [0, 64]), status=s.status)
    want = s.host.values(s.table[0], 64, 1)[-new:]
    for padding in (new, 15000, 40000):
        q = torch.zeros(padding, 1, 64, dtype=dtype)
        q[:new] = (20 * k[-new:]).to(dtype)  # 100 or more above every other key
        out = s.cache.attend(q.cuda(), table, at, first, causal=False, status=s.status)
        off = (out[:new].cpu().double() - want).abs()
        tol = (torch.finfo(dtype).eps / 2 + 2 * 2.0 ** -16) * want.abs() + 2.0 ** -25
        assert bool((off <= tol).all()), (padding, float((off / tol).max()))
    s.status.raise_if_set()

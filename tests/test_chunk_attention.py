"""Chunk attention over a paged KV cache against the 64-bit definition.

The reference reads the same cache (the values its codes stand for), so the
only errors are those of the operator's own roundings; the bound per output
element is derived in ``oracle.kv_quant_ref.attention_bound``.
"""
import math

import pytest
import torch

import inputs as I
from oracle import kv_quant_ref as Q

D = 128
TYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


@pytest.fixture(scope="module")
def dev():
    d = torch.device("cuda:0")
    torch.cuda.set_device(d)
    from dllmserve_b200 import _native

    _native.lib()
    return d


def _ops():
    from dllmserve_b200 import ops

    return ops


def _cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32)


class Case:
    """Inputs of one launch on the CPU, with caches whose unused rows are NaN."""

    def __init__(self, seed, fmt, hq, hkv, nq, nc, nf, tables, page=16, spread=True):
        g = I.gen(seed)
        self.fmt, self.hq, self.hkv, self.page = fmt, hq, hkv, page
        self.nq, self.nc, self.nf = nq, nc, nf
        self.q = I.normal(g, (sum(nq) + 2, hq, D)).to(torch.bfloat16)  # two rows of no sequence
        self.k = I.normal(g, (sum(nf), hkv, D)).to(torch.bfloat16) if nf else None
        self.v = I.normal(g, (sum(nf), hkv, D)).to(torch.bfloat16) if nf else None
        of = [-(-n // page) for n in nc]
        pages = sum(of) + 2
        order = torch.randperm(pages, generator=g)
        self.tables = torch.full((len(nc), max(1, max(of) + 1)), -1, dtype=torch.int32)
        lists, at = [], 0
        for b, n in enumerate(of):
            mine = order[at:at + n]
            at += n
            self.tables[b, :n] = mine.int()
            every = (mine[:, None] * page + torch.arange(page)).flatten()[:nc[b]]
            if not tables and b % 2:  # scattered rows
                every = every[torch.randperm(nc[b], generator=g)]
            lists.append(every)
        self.use_tables = tables
        self.slots = torch.cat(lists).int()
        self.lists = lists
        rows = [I.normal(g, (pages * page, hkv, D)) for _ in range(2)]
        if spread:  # heads and tokens of different sizes
            rows = [x * torch.exp2(torch.randint(-3, 3, (pages * page, hkv, 1), generator=g).float()) for x in rows]
        used = torch.zeros(pages * page, dtype=torch.bool)
        used[self.slots.long()] = True
        self.values, self.caches, self.exps = [], [], []
        for x in rows:
            x = x.to(torch.bfloat16)
            if fmt == "bf16":
                x[~used] = float("nan")
                self.values.append(x.double())
                self.caches.append(x.view(pages, page, hkv, D))
                self.exps.append(None)
            else:
                codes, e = Q.quantise(x, fmt)
                self.values.append(Q.values(codes, e))
                c = codes.float().to(TYPES[fmt])
                byte = (e + 127).to(torch.uint8)
                c.view(torch.uint8)[~used] = 0x7f
                byte[~used] = 255
                self.caches.append(c.view(pages, page, hkv, D))
                self.exps.append(byte.view(pages, page, hkv))

    def args(self, dev):
        to = lambda t: None if t is None else t.to(dev)  # noqa: E731
        kw = {"k_exp": to(self.exps[0]), "v_exp": to(self.exps[1])}
        if self.use_tables:
            kw |= {"block_tables": to(self.tables), "context_lens": torch.tensor(self.nc, dtype=torch.int32, device=dev)}
        else:
            kw |= {"slots": to(self.slots), "cu_seqlens_slots": _cu(self.nc).to(dev)}
        if self.k is not None:
            kw |= {"k": to(self.k), "v": to(self.v), "cu_seqlens_k": _cu(self.nf).to(dev), "max_seqlen_k": max(self.nf)}
        return (to(self.q), to(self.caches[0]), to(self.caches[1]), _cu(self.nq).to(dev), max(self.nq)), kw

    def check(self, out, causal, scale=D ** -0.5, seqs=None):
        out = out.cpu().double()
        start, fresh = 0, 0
        for b, n in enumerate(self.nq):
            keys, vals = (x[self.lists[b].long()] for x in self.values)
            if self.k is not None:
                keys = torch.cat([keys, self.k[fresh:fresh + self.nf[b]].double()])
                vals = torch.cat([vals, self.v[fresh:fresh + self.nf[b]].double()])
                fresh += self.nf[b]
            got = out[start:start + n]
            start += n
            if seqs is not None and b not in seqs:
                continue
            o, mag, big = Q.chunk_attention(self.q[start - n:start], keys, vals, scale, causal)
            off = (got - o).abs()
            floor = None if self.fmt == "bf16" else Q.small_probability_floor(vals, self.hq)
            bound = Q.attention_bound(o, mag, big, floor)
            assert torch.isfinite(got).all(), f"sequence {b}"
            worst = (off / bound).max().item() if off.numel() else 0.0
            assert worst <= 1.0, f"sequence {b}: {worst:.2f} of the bound, off by {off.max():.3e}"


SHAPES = [
    # hq, hkv, query rows, cached rows, fresh rows (None: the cached rows hold the chunk's own)
    (4, 4, [1], [1], None),
    (4, 4, [1, 1, 1], [16, 17, 0], [1, 1, 1]),
    (28, 4, [1, 1, 1, 1], [96, 5, 33, 130], None),
    (7, 1, [1, 1], [300, 31], [1, 1]),
    (8, 2, [3, 1, 5], [40, 64, 7], None),
    (8, 8, [32, 32], [45, 152], [32, 32]),
    (28, 4, [32, 7, 1], [50, 0, 111], [32, 7, 1]),
    (2, 2, [70, 1, 33], [0, 200, 19], [70, 1, 33]),
    (6, 2, [130, 12], [150, 300], None),
    (3, 1, [9, 4], [5, 2], None),     # more query rows than keys: the first rows see none
    (2, 1, [4, 0, 3], [10, 20, 0], [2, 5, 0]),  # fresh rows fewer or more than the chunk's, an empty chunk
]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("causal,tables", [(True, True), (False, False), (True, False)])
def test_small(dev, fmt, shape, causal, tables):
    hq, hkv, nq, nc, nf = SHAPES[shape]
    c = Case(100 + shape, fmt, hq, hkv, nq, nc, nf, tables)
    args, kw = c.args(dev)
    out = torch.full(c.q.shape, 5.0, dtype=torch.bfloat16, device=dev)
    got = _ops().chunk_attention(*args, causal=causal, out=out, **kw)
    assert got is out
    c.check(out, causal)
    assert (out[sum(nq):] == 5).all()  # rows behind the last sequence are left as they were
    assert _ops().read_device_status(dev) == 0


LONG = [
    # hq, hkv, query rows, cached rows, fresh rows, sequences checked against 64 bits
    (28, 4, [1, 1, 1], [9000, 130, 4097], None, [0, 1, 2]),
    (4, 4, [1, 1], [20000, 3], [1, 1], [0, 1]),
    (8, 8, [32, 32], [2500, 1200], [32, 32], [1]),
    (28, 4, [33, 20], [700, 1500], [33, 20], [0]),
    (4, 2, [200], [600], [200], [0]),
    (4, 2, [260, 3], [700, 400], None, [0, 1]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("shape", range(len(LONG)))
@pytest.mark.parametrize("causal,tables", [(True, True), (False, False)])
def test_long(dev, fmt, shape, causal, tables):
    hq, hkv, nq, nc, nf, seqs = LONG[shape]
    c = Case(300 + shape, "bf16" if fmt == "bf16" else fmt, hq, hkv, nq, nc, nf, tables, page=256, spread=shape % 2 == 0)
    args, kw = c.args(dev)
    out = _ops().chunk_attention(*args, causal=causal, max_context=max(nc), **kw)
    c.check(out, causal, seqs=seqs)
    again = _ops().chunk_attention(*args, causal=causal, max_context=max(nc), **kw)
    assert torch.equal(again[:sum(nq)], out[:sum(nq)])  # the same bits every time
    # a loose bound of the context changes the split of the work, not the result's accuracy
    c.check(_ops().chunk_attention(*args, causal=causal, **kw), causal, seqs=seqs[:1])
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("tables", [True, False])
@pytest.mark.parametrize("most", [60, 34])
def test_many_units(dev, fmt, tables, most):
    """More row tiles than the GPU has SMs, of unequal lengths, so that a CTA
    takes several one after another. Some sequences are held to the 64-bit
    bound; where a launch of one sequence cuts its rows into the same units
    (at most 34 x 3 packed rows: one tile), its bits are the batch's."""
    g = I.gen(17)
    n = 90
    nq = torch.randint(0, most, (n,), generator=g).tolist()
    nc = torch.randint(0, 500, (n,), generator=g).tolist()
    nc[3], nc[40], nq[7], nq[40] = 0, 0, 0, 33
    seqs = [3, 7, 11, 40] + list(range(0, n, 8))
    nf = [x if i % 3 else min(x, 17) for i, x in enumerate(nq)]
    c = Case(18, fmt, 12, 4, nq, nc, nf, tables, page=128, spread=False)
    args, kw = c.args(dev)
    ops = _ops()
    for causal in (False, True):
        out = ops.chunk_attention(*args, causal=causal, max_context=512, **kw)
        c.check(out, causal, seqs=seqs)
        for _ in range(3):  # launches back to back
            again = ops.chunk_attention(*args, causal=causal, max_context=512, **kw)
        assert torch.equal(again[:sum(nq)], out[:sum(nq)])
        cu, cuk, cus = (_cu(x).tolist() for x in (nq, nf, nc))
        for b in range(0, n, 4):
            if nq[b] == 0 or most > 34:
                continue
            one = dict(kw)
            one |= {"k": kw["k"][cuk[b]:cuk[b + 1]], "v": kw["v"][cuk[b]:cuk[b + 1]], "cu_seqlens_k": _cu([nf[b]]).to(dev)}
            if tables:
                one |= {"block_tables": kw["block_tables"][b:b + 1], "context_lens": kw["context_lens"][b:b + 1]}
            else:
                one |= {"slots": kw["slots"][cus[b]:cus[b + 1]], "cu_seqlens_slots": _cu([nc[b]]).to(dev)}
            if nf[b] == 0 and nc[b] == 0:
                assert (out[cu[b]:cu[b + 1]] == 0).all()
                continue
            alone = ops.chunk_attention(args[0][cu[b]:cu[b + 1]], *args[1:3], _cu([nq[b]]).to(dev), max(nq),
                                        causal=causal, max_context=512, **one)
            assert torch.equal(alone, out[cu[b]:cu[b + 1]]), b
    assert ops.read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("heads,tables", [((4, 4), True), ((12, 4), False), ((10, 2), True)])
def test_long_chunks_of_many_sequences(dev, fmt, heads, tables):
    """Enough rows that a work unit takes two row tiles (and a quantised cache
    is expanded first), of unequal lengths; 3 and 5 heads per KV head do not
    divide a tile's 128 rows."""
    hq, hkv = heads
    g = I.gen(23)
    n = 40 if hkv == 4 else 80
    nq = torch.randint(1, 280, (n,), generator=g).tolist()
    nc = torch.randint(0, 420, (n,), generator=g).tolist()
    nq[5], nq[6], nc[6], nc[9] = 257, 0, 0, 0
    nf = nq if hkv == 4 else [0] * n
    if hkv == 2:
        nc = [a + b if i % 5 else a for i, (a, b) in enumerate(zip(nc, nq))]
    c = Case(24, fmt, hq, hkv, nq, nc, nf if hkv == 4 else None, tables, page=128, spread=hq == 4)
    args, kw = c.args(dev)
    for causal in (True, False):
        out = torch.full(c.q.shape, 5.0, dtype=torch.bfloat16, device=dev)
        _ops().chunk_attention(*args, causal=causal, out=out, **kw)
        c.check(out, causal, seqs=[5, 6, 9, 10] if hq == 4 else [9, 13])
        assert (out[sum(nq):] == 5).all()
        for _ in range(2):
            again = _ops().chunk_attention(*args, causal=causal, **kw)
        assert torch.equal(again[:sum(nq)], out[:sum(nq)])
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("heads,nq,causal", [((16, 16), [1000, 1100], True), ((48, 16), [340, 345], False)])
def test_two_row_tiles_per_unit(dev, fmt, heads, nq, causal):
    """Sizes at which a work unit takes two row tiles (the second one partial,
    or missing at a sequence's end), the last sequence's slots scattered."""
    c = Case(25, fmt, *heads, nq, [200, 37], nq, False, page=128)
    args, kw = c.args(dev)
    out = torch.full(c.q.shape, 5.0, dtype=torch.bfloat16, device=dev)
    _ops().chunk_attention(*args, causal=causal, out=out, **kw)
    c.check(out, causal, seqs=[1])
    assert (out[sum(nq):] == 5).all()
    again = _ops().chunk_attention(*args, causal=causal, **kw)
    assert torch.equal(again[:sum(nq)], out[:sum(nq)])
    # the first sequence alone, one tile per unit: both forms are within the bound of each other's roundings
    one = dict(kw)
    one |= {"k": kw["k"][:nq[0]], "v": kw["v"][:nq[0]], "cu_seqlens_k": _cu(nq[:1]).to(dev), "max_seqlen_k": nq[0],
            "slots": kw["slots"][:200], "cu_seqlens_slots": _cu([200]).to(dev)}
    alone = _ops().chunk_attention(args[0][:nq[0]], *args[1:3], _cu(nq[:1]).to(dev), nq[0], causal=causal, **one)
    # two results of bf16 roundings each: of the output (2^-8) and of every probability (2^-8 sum p |v|)
    big = max(float(c.values[1][c.lists[0].long()].abs().max()), float(c.v[:nq[0]].abs().max()))
    assert (alone.float() - out[:nq[0]].float()).abs().max() <= 4 * 2.0 ** -8 * big
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_fresh_only(dev, fmt):
    """No cache at all: causal attention among the chunk's own rows."""
    c = Case(7, "bf16", 6, 2, [33, 1, 140], [0, 0, 0], [33, 1, 140], True)
    args, kw = c.args(dev)
    for name in ("block_tables", "context_lens", "k_exp", "v_exp"):
        kw.pop(name)
    for causal in (True, False):
        c.check(_ops().chunk_attention(args[0], None, None, *args[3:], causal=causal, **kw), causal)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 7, 48, 512])
def test_page_sizes(dev, page):
    c = Case(11 + page, "int8", 4, 2, [2, 1], [101, 64], [2, 1], True, page=page)
    args, kw = c.args(dev)
    c.check(_ops().chunk_attention(*args, **kw), True)
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
def test_strides_and_scale(dev, fmt):
    """Rows of a fused projection, table rows wider than the table, a slice of
    the output buffer, and a scale of the caller's."""
    c = Case(21, fmt, 8, 2, [17, 1, 40], [60, 3, 29], [17, 1, 40], True)
    args, kw = c.args(dev)
    n, pad = c.q.shape[0], 8
    qkv = torch.full((n, 12 * D + pad), 3.0, dtype=torch.bfloat16, device=dev)
    q = qkv[:, :8 * D].view(n, 8, D)
    q.copy_(args[0])
    m = c.k.shape[0]
    k, v = qkv[:m, 8 * D:10 * D].view(m, 2, D), qkv[:m, 10 * D:12 * D].view(m, 2, D)
    k.copy_(kw["k"])
    v.copy_(kw["v"])
    wide = torch.full((3, c.tables.shape[1] + 5), 1 << 30, dtype=torch.int32, device=dev)
    wide[:, :c.tables.shape[1]] = kw["block_tables"]
    buf = torch.full((n, 10 * D), 4.0, dtype=torch.bfloat16, device=dev)
    out = buf[:, D:9 * D].view(n, 8, D)
    kw |= {"k": k, "v": v, "block_tables": wide[:, :c.tables.shape[1]], "out": out}
    _ops().chunk_attention(q, *args[1:], 0.25, causal=True, **kw)
    c.check(out, True, scale=0.25)
    assert (buf[:, :D] == 4).all() and (buf[:, 9 * D:] == 4).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
def test_large_scores(dev, fmt):
    """Scores far apart (differences of hundreds): the running maximum moves by
    a lot and most probabilities vanish."""
    c = Case(31, fmt, 4, 2, [3, 40], [333, 70], [3, 40], False)
    c.q = (c.q.float() * 30).to(torch.bfloat16)
    args, kw = c.args(dev)
    for causal in (True, False):
        c.check(_ops().chunk_attention(*args, causal=causal, **kw), causal)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("step", [1, 6, 30])
def test_value_sizes_far_apart(dev, fmt, step):
    """Value rows whose exponents rise, fall and jump along the sequence by up
    to 2^90, with weight on the small ones: the unit of the outputs moves, and
    chunks whose values lie far below it take the wider operands."""
    for seed, order in ((91, 1), (92, -1), (93, 0)):
        c = Case(seed, fmt, 4, 2, [2, 1, 33], [300, 410, 200], [2, 1, 33], True)
        for b, at in enumerate(c.lists):
            n = len(at)
            e = (torch.arange(n) * 3 // n) * step * (order or 1)
            if order == 0:  # jumps from key to key
                e = torch.randint(0, 3, (n,), generator=I.gen(seed + b)) * step
            byte = c.exps[1].view(-1, 2)[at].int() + e.int()[:, None]
            assert byte.min() >= 27 and byte.max() <= 240
            c.exps[1].view(-1, 2)[at] = byte.to(torch.uint8)
            c.values[1][at] *= torch.exp2(e.double())[:, None, None]
        args, kw = c.args(dev)
        c.check(_ops().chunk_attention(*args, causal=True, **kw), True)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("nq,page", [([1, 2], 16), ([20, 33], 16), ([20, 33], 128)])
def test_bad_pages_and_lengths(dev, fmt, nq, page):
    """Pages outside the cache read as zero rows and are flagged; lengths past
    their bounds are cut and flagged. Nothing outside the buffers is touched."""
    ops = _ops()
    n = sum(nq)
    nc = [2 * page + 8, page + 30]
    c = Case(41, fmt, 4, 4, nq, nc, None, True, page=page)
    args, kw = c.args(dev)
    for bad in (10 ** 6, -3, 2 ** 31 - 1):
        tables = kw["block_tables"].clone()
        at = int(tables[0, 1])
        tables[0, 1] = bad
        out = ops.chunk_attention(*args, **{**kw, "block_tables": tables})
        assert ops.read_device_status(dev) == 1
        saved = [x.clone() for x in c.values]
        for x in c.values:
            x[at * page:at * page + page] = 0
        c.check(out, True)
        c.values = saved
    # a context longer than its table row
    ctx = torch.tensor([nc[0], 10 ** 6], dtype=torch.int32, device=dev)
    out = ops.chunk_attention(*args, **{**kw, "context_lens": ctx})
    assert ops.read_device_status(dev) in (1, 3)
    c.check(out, True, seqs=[0])
    ctx = torch.tensor([nc[0], -5], dtype=torch.int32, device=dev)
    out = ops.chunk_attention(*args, **{**kw, "context_lens": ctx})
    assert ops.read_device_status(dev) == 3
    assert (out[nq[0]:n] == 0).all()
    # a chunk longer than max_seqlen_q: the rows past it are not computed
    out = torch.full_like(args[0], 5.0)
    ops.chunk_attention(*args[:4], nq[0], out=out, **kw)
    assert ops.read_device_status(dev) == 3
    assert (out[2 * nq[0]:] == 5).all()
    # slots outside the cache
    c = Case(42, fmt, 4, 4, nq, nc, None, False, page=page)
    args, kw = c.args(dev)
    slots = kw["slots"].clone()
    slots[3], slots[nc[0] + 10] = 10 ** 8, -1
    out = ops.chunk_attention(*args, **{**kw, "slots": slots})
    assert ops.read_device_status(dev) == 1
    for x in c.values:
        x[c.slots[3].long()] = 0
        x[c.slots[nc[0] + 10].long()] = 0
    c.check(out, True)


@pytest.mark.gpu
def test_streams_and_graph(dev):
    """Two streams at once, and a captured launch replayed on new contents."""
    ops = _ops()
    cases = [Case(51, "e4m3", 28, 4, [1, 1], [5000, 800], [1, 1], True, page=256),
             Case(52, "int8", 8, 8, [1, 1], [4000, 1900], None, True, page=256)]
    made = [c.args(dev) for c in cases]
    streams = [torch.cuda.Stream(dev) for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.chunk_attention(*made[i][0], **made[i][1]))
    torch.cuda.synchronize()
    for i, c in enumerate(cases):
        c.check(outs[i][0], True)
        for o in outs[i][1:]:
            assert torch.equal(o[:2], outs[i][0][:2])
    args, kw = made[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.chunk_attention(*args, **kw)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[:2], outs[0][0][:2])
    cases[0].q = -cases[0].q
    args[0].copy_(cases[0].q)
    cases[0].nc = [4000, 0]
    cases[0].lists = [x[:n] for x, n in zip(cases[0].lists, cases[0].nc)]
    kw["context_lens"].copy_(torch.tensor(cases[0].nc, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    cases[0].check(out, True)


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """A cache of more than 2^31 elements, used at its far end."""
    hkv, page = 32, 256
    pages = 2200
    cache = torch.zeros(pages, page, hkv, D, dtype=torch.float8_e4m3fn, device=dev)
    vcache = torch.zeros_like(cache)
    ke = torch.full((pages, page, hkv), 127, dtype=torch.uint8, device=dev)
    c = Case(61, "e4m3", 32, 32, [1, 1], [300, 80], None, True, page=page)
    n = c.caches[0].shape[0]
    cache[-n:].view(torch.uint8).copy_(c.caches[0].to(dev).view(torch.uint8))
    vcache[-n:].view(torch.uint8).copy_(c.caches[1].to(dev).view(torch.uint8))
    ve = ke.clone()
    ke[-n:], ve[-n:] = c.exps[0].to(dev), c.exps[1].to(dev)
    args, kw = c.args(dev)
    tables = torch.where(kw["block_tables"] >= 0, kw["block_tables"] + (pages - n), kw["block_tables"])
    out = _ops().chunk_attention(args[0], cache, vcache, *args[3:], block_tables=tables.int(),
                                 context_lens=kw["context_lens"], k_exp=ke, v_exp=ve)
    c.check(out, True)
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
def test_store_then_attend(dev):
    """The operators as they are used together: prefill in two chunks, then
    decode steps, over a quantised cache, each step storing its rows first."""
    ops = _ops()
    for fmt in ("e4m3", "int8"):
        g = I.gen(71)
        hq, hkv, page = 14, 2, 16
        lens = [37, 90]
        pages = 12
        kc = torch.zeros(pages, page, hkv, D, dtype=torch.uint8, device=dev).view(TYPES[fmt])
        vc = torch.zeros_like(kc)
        ke = torch.zeros(pages, page, hkv, dtype=torch.uint8, device=dev)
        ve = torch.zeros_like(ke)
        tables = torch.randperm(pages, generator=g)[:12].view(2, 6).int()
        total = [0, 0]
        seen = [[torch.zeros(0, hkv, D, dtype=torch.float64)] * 2 for _ in lens]
        for step in ([20, 64], [17, 26], [1, 1], [1, 1]):
            n = sum(step)
            q, k, v = (I.normal(g, (n, h, D)).to(torch.bfloat16) for h in (hq, hkv, hkv))
            pos = [torch.arange(total[b], total[b] + step[b]) for b in range(2)]
            slots = torch.cat([tables[b][p // page].long() * page + p % page for b, p in enumerate(pos)]).int()
            ops.store_kvcache_quant(k.to(dev), v.to(dev), kc, vc, ke, ve, slots.to(dev))
            total = [t + s for t, s in zip(total, step)]
            out = ops.chunk_attention(q.to(dev), kc, vc, _cu(step).to(dev), max(step), block_tables=tables.to(dev),
                                      context_lens=torch.tensor(total, dtype=torch.int32, device=dev), k_exp=ke, v_exp=ve)
            at = 0
            for b, s in enumerate(step):
                rows = slice(at, at + s)
                at += s
                seen[b] = [torch.cat([old, Q.values(*Q.quantise(x[rows], fmt))]) for old, x in zip(seen[b], (k, v))]
                o, mag, big = Q.chunk_attention(q[rows], *seen[b], D ** -0.5, True)
                bound = Q.attention_bound(o, mag, big, Q.small_probability_floor(seen[b][1], hq))
                assert ((out[rows].cpu().double() - o).abs() <= bound).all()
        assert ops.read_device_status(dev) == 0


def test_refusals():
    """Bad arguments are refused before any device work."""
    from dllmserve_b200 import _native, ops

    lib = _native.lib()

    def call(**kw):
        a = dict(q=64, qs=512, k=0, ks=0, v=0, vs=0, kc=64, vc=64, ke=64, ve=64, slots_n=64, bt=64, bts=4, ctx=64, sl=0,
                 cus=0, ts=0, o=64, os=512, cuq=64, cuk=0, tq=1, tk=0, ws=0, wb=0, err=0, stream=0, fmt=1, mb=4, bs=16,
                 mc=64, B=1, mq=1, mf=0, hq=4, hkv=4, hd=128, ca=1, sc=0.1)
        a.update(kw)
        return lib.dllm_attn_chunk_fwd(_native.CHUNK_ARGS.pack(*a.values()))

    E = _native
    assert call(hd=64) == E.DLLM_ERR_UNSUPPORTED
    assert call(fmt=3) == E.DLLM_ERR_UNSUPPORTED
    assert call(hq=6) == E.DLLM_ERR_UNSUPPORTED
    assert call(hq=4 * 129, qs=4 * 129 * 128) == E.DLLM_ERR_UNSUPPORTED
    assert lib.dllm_attn_chunk_fwd(None) == E.DLLM_ERR_INVALID_ARG
    assert _native.CHUNK_ARGS.size == 27 * 8 + 12 * 4
    assert call(B=-1) == E.DLLM_ERR_INVALID_ARG
    assert call(sc=0.0) == E.DLLM_ERR_INVALID_ARG
    assert call(sc=math.nan) == E.DLLM_ERR_INVALID_ARG
    assert call(sl=64, cus=64) == E.DLLM_ERR_INVALID_ARG       # tables and a slot list
    assert call(ctx=0) == E.DLLM_ERR_INVALID_ARG
    assert call(bs=0) == E.DLLM_ERR_INVALID_ARG
    assert call(bts=3) == E.DLLM_ERR_INVALID_ARG
    assert call(bt=0, sl=64) == E.DLLM_ERR_INVALID_ARG      # slots without offsets
    assert call(kc=0) == E.DLLM_ERR_INVALID_ARG
    assert call(ke=0) == E.DLLM_ERR_INVALID_ARG
    assert call(kc=72) == E.DLLM_ERR_ALIGNMENT
    assert call(k=64) == E.DLLM_ERR_INVALID_ARG                # k without v
    assert call(cuq=0, mq=2, wb=1 << 40, ws=64) == E.DLLM_ERR_INVALID_ARG  # without offsets: one row per sequence
    assert "max_seqlen_q" in lib.dllm_last_error().decode()
    assert call(slots_n=0) == E.DLLM_ERR_INVALID_ARG
    assert call(ctx=0, cus=0) == E.DLLM_ERR_INVALID_ARG
    assert call(ctx=64, cus=64) == E.DLLM_ERR_INVALID_ARG
    assert call(mc=2 ** 29 + 1, mf=2 ** 29) == E.DLLM_ERR_TOO_LARGE
    assert call(q=72) == E.DLLM_ERR_ALIGNMENT
    assert call(qs=516) == E.DLLM_ERR_ALIGNMENT
    assert call(os=500) == E.DLLM_ERR_INVALID_ARG
    assert call(slots_n=2 ** 31) == E.DLLM_ERR_TOO_LARGE
    assert call(mc=2 ** 30 + 1) == E.DLLM_ERR_TOO_LARGE
    assert call(B=0) == E.DLLM_OK
    assert call(mc=100000, mb=10000, bts=10000) == E.DLLM_ERR_INVALID_ARG  # no workspace for the splits
    assert "workspace" in lib.dllm_last_error().decode()
    ws = lib.dllm_attn_chunk_workspace
    assert ws(1, 1, 4, 4, 1, 100000, 0) > 0
    assert ws(1, 64, 32, 32, 1, 64, 0) == 0
    assert ws(9, 1, 4, 4, 1, 64, 0) == -1
    kernels = lib.dllm_attn_chunk_launches
    assert kernels(1, 1, 4, 4, 1, 100000, 0) == 2                # splits and their merge
    assert kernels(1, 64, 32, 32, 1, 64, 0) == 1
    assert kernels(1, 1, 4, 4, 1024, 100000, 0) == 3             # the expanded copy, splits, merge
    assert kernels(9, 1, 4, 4, 1, 64, 0) == -1
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(ValueError, match="no keys"):
        ops.chunk_attention(q, None, None, cu, 1)
    with pytest.raises(ValueError, match="go together"):
        ops.chunk_attention(q, None, None, cu, 1, k=q)
    with pytest.raises(ValueError, match="CUDA"):
        ops.chunk_attention(q, None, None, cu, 1, k=q, v=q, cu_seqlens_k=cu)


@pytest.mark.gpu
def test_refusals_on_device_tensors(dev):
    ops = _ops()
    c = Case(81, "int8", 4, 2, [1, 2], [20, 9], [1, 2], True)
    args, kw = c.args(dev)
    q, kc, vc, cu, mq = args

    def refused(*a, **k):
        with pytest.raises(ValueError):
            ops.chunk_attention(*(a or args), **{**kw, **k})

    refused(q.float(), kc, vc, cu, mq)
    refused(q, kc, vc.view(torch.uint8), cu, mq)
    refused(q, kc[:, :, :1], vc, cu, mq)
    refused(q, kc, vc[:1], cu, mq)
    refused(q, kc, vc, cu.long(), mq)
    refused(k_exp=None)
    refused(v_exp=kw["v_exp"].int())
    refused(block_tables=kw["block_tables"].long())
    refused(block_tables=kw["block_tables"][:1])
    refused(block_tables=kw["block_tables"].t().contiguous().t())
    refused(context_lens=None)
    refused(slots=c.slots.to(dev))
    refused(k=kw["k"][:, :1])
    refused(cu_seqlens_k=kw["cu_seqlens_k"][:2])
    refused(out=torch.empty_like(q[:1]))
    refused(softmax_scale=0.0)
    y = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=dev)
    with pytest.raises(NotImplementedError):
        ops.chunk_attention(y, None, None, cu, 2, k=y, v=y, cu_seqlens_k=cu)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
def test_one_row_per_sequence_and_summed_lengths(dev, fmt):
    """cu_seqlens_q None: row b is sequence b's; lengths as running sums. Both
    give the bits of the arrays they stand for."""
    ops = _ops()
    c = Case(82, fmt, 12, 4, [1] * 5, [70, 0, 300, 16, 31], None, True)
    args, kw = c.args(dev)
    q = args[0][:5]
    want = ops.chunk_attention(q, *args[1:], **kw)
    c.check(want, True)
    assert torch.equal(ops.chunk_attention(q, *args[1:3], None, 1, **kw), want)
    sums = {k: v for k, v in kw.items() if k != "context_lens"} | {"cu_seqlens_slots": _cu(c.nc).to(dev)}
    assert torch.equal(ops.chunk_attention(q, *args[1:], **sums), want)
    assert torch.equal(ops.chunk_attention(q, *args[1:3], None, 1, **sums), want)
    assert ops.read_device_status(dev) == 0
    with pytest.raises(ValueError, match="max_seqlen_q"):
        ops.chunk_attention(q, *args[1:3], None, 2, **kw)
    with pytest.raises(ValueError, match="either"):
        ops.chunk_attention(q, *args[1:3], None, 1, **kw, cu_seqlens_slots=sums["cu_seqlens_slots"])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nq", [2, 40])
def test_nothing_to_read(dev, fmt, nq):
    """Fresh rows, slot list or table of length zero: the other keys, or zero rows."""
    ops = _ops()
    c = Case(83, fmt, 8, 2, [nq, nq], [50, 9], [nq, nq], False)
    args, kw = c.args(dev)
    zero = torch.zeros(3, dtype=torch.int32, device=dev)
    none = {"k": kw["k"][:0], "v": kw["v"][:0], "cu_seqlens_k": zero}
    full, c.nf, c.k = c.k, [0, 0], None
    out = ops.chunk_attention(*args, causal=False, **{**kw, **none})
    c.check(out, False)
    c.k, c.nf = full, [nq, nq]
    out = ops.chunk_attention(*args, causal=False, **{**kw, "slots": kw["slots"][:0], "cu_seqlens_slots": zero})
    c.lists = [x[:0] for x in c.lists]
    c.check(out, False)
    table = torch.zeros(2, 0, dtype=torch.int32, device=dev)
    rest = {k: kw[k] for k in ("k_exp", "v_exp")}
    for keys in ({**kw, **none, "slots": kw["slots"][:0], "cu_seqlens_slots": zero},
                 {**rest, "block_tables": table, "context_lens": zero[:2]}):
        out = torch.full(c.q.shape, 5.0, dtype=torch.bfloat16, device=dev)
        ops.chunk_attention(*args, causal=False, out=out, **keys)
        assert (out[:2 * nq] == 0).all() and (out[2 * nq:] == 5).all()
    empty = torch.zeros(3, 8, D, dtype=torch.bfloat16, device=dev)[:0]
    assert ops.chunk_attention(empty, *args[1:3], zero, 1, **kw).shape == empty.shape
    assert ops.read_device_status(dev) == 0


@pytest.mark.gpu
def test_layouts_of_a_single_row_or_head(dev):
    """A length-one dimension may have any stride."""
    ops = _ops()
    c = Case(84, "int8", 6, 1, [1], [40], [1], True)
    args, kw = c.args(dev)
    q = args[0][:1].clone().as_strided((1, 6, D), (D, D, 1))
    k, v = (x.clone().as_strided((1, 1, D), (3, 5, 1)) for x in (kw["k"], kw["v"]))
    want = ops.chunk_attention(args[0][:1], *args[1:], **kw)
    c.check(want, True)
    assert torch.equal(ops.chunk_attention(q, *args[1:], **{**kw, "k": k, "v": v}), want)
    more = torch.randn(1, 5, D, generator=I.gen(3)).to(torch.bfloat16).to(dev).transpose(0, 1)  # [5, 1, D], stride 5 D
    assert more.stride(1) == 5 * D
    kc, ke = kw["k_exp"].clone().zero_(), kw["k_exp"]
    slots = torch.arange(5, dtype=torch.int32, device=dev)
    caches = [torch.zeros_like(args[1]) for _ in range(4)]
    ops.store_kvcache_quant(more, more, *caches[:2], kc, ke.clone(), slots)
    ke2, ve2 = torch.zeros_like(ke), torch.zeros_like(ke)
    ops.store_kvcache_quant(more.contiguous(), more.contiguous(), *caches[2:], ke2, ve2, slots)
    assert torch.equal(caches[0].flatten()[:5 * D], caches[2].flatten()[:5 * D])
    assert torch.equal(kc.flatten()[:5], ke2.flatten()[:5])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("nq", [1, 20, 60])
def test_sizes_at_the_ends_of_the_range(dev, fmt, nq):
    """Cached values of 2^-88 with fresh ones of 2^20 and 2^100 (the outputs'
    unit), and keys of 2^115 against queries of 2^-115 (the scores)."""
    for dv, df, dk in ((-88, 20, 0), (-88, 100, 0), (0, 100, 0), (100, -90, 0), (0, 0, 115)):
        c = Case(85, fmt, 4, 2, [nq, 1], [200, 33], [nq, 1], False)
        up = lambda t, e: (t.double() * 2.0 ** e).to(torch.bfloat16)  # noqa: E731
        c.v = up(c.v, df)
        c.q, c.k = up(c.q, -dk), up(c.k, dk)
        for i, e in ((0, dk), (1, dv)):
            used = c.slots.long()
            byte = c.exps[i].view(-1, 2)[used].int() + e
            assert byte.min() >= 27 and byte.max() <= 246
            c.exps[i].view(-1, 2)[used] = byte.to(torch.uint8)
            c.values[i][used] *= 2.0 ** e
        args, kw = c.args(dev)
        for causal in (True, False):
            c.check(_ops().chunk_attention(*args, causal=causal, **kw), causal)


# hq, hkv, query rows, cached rows, fresh rows, kernels of a launch over bf16 and over quantised caches
FORMS = [
    (4, 4, [1, 3], [40, 9], [1, 3], 1, 1),                  # few rows, one split
    (28, 4, [2, 1], [1100, 40], None, 1, 1),                # splits merged by their cluster
    (4, 2, [8, 3], [9000, 70], [8, 3], 2, 2),               # splits merged by a second kernel
    (4, 4, [32, 20], [60, 5], [32, 20], 1, 1),              # 32 rows
    (3, 1, [50, 4], [30, 2], None, 1, 1),                   # one row tile per unit; more rows than keys
    (4, 2, [40, 70], [1500, 20], [40, 70], 2, 2),           # its splits
    (16, 16, [1000, 1100], [130, 20], [1000, 1100], 1, 2),  # two row tiles per unit; rows expanded once
]


def _form(seed, fmt, shape):
    hq, hkv, nq, nc, nf, *kernels = FORMS[shape]
    c = Case(seed + shape, fmt, hq, hkv, nq, nc, nf, shape % 2 == 0, page=32, spread=False)
    args, kw = c.args("cuda:0")
    kw["max_context"] = max(nc)
    ops = _ops()
    before = ops.LAUNCHES[0]
    out = ops.chunk_attention(*args, causal=True, **kw)
    assert ops.LAUNCHES[0] - before == kernels[fmt != "bf16"]
    return c, args, kw, out


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("shape", range(len(FORMS)))
def test_nan_queries(dev, fmt, shape):
    """A query row with a NaN is NaN, unless it sees no key; the others do not change."""
    c, args, kw, want = _form(600, fmt, shape)
    n = sum(c.nq)
    want = want[:n].clone()
    bad = torch.zeros(n, c.hq, dtype=torch.bool)
    bad[torch.arange(0, n, 3), torch.arange(0, n, 3) % c.hq] = True
    bad[n - 1] = True
    q = args[0].clone()
    q[:n, :, 5][bad.to(dev)] = math.nan
    got = _ops().chunk_attention(q, *args[1:], causal=True, **kw)[:n]
    length = [a + (0 if c.nf is None else b) for a, b in zip(c.nc, c.nf or c.nc)]
    sees = torch.cat([torch.arange(m) + (k - m + 1) > 0 for m, k in zip(c.nq, length)])
    hit = (bad & sees[:, None]).to(dev)
    assert hit.any() and torch.isnan(got[hit]).all()
    got, want = got.float().masked_fill(hit[..., None], 0), want.float().masked_fill(hit[..., None], 0)
    if max(c.nq) * (c.hq // c.hkv) <= (16 if fmt == "bf16" else 32):  # the kernel for few rows
        assert torch.equal(got, want)
    else:
        # (the 128-row kernel rescales the rows of a warp together, so the bits may differ: both results
        # are within (2^-8 + e) sum p |v| + 2^-8 |o|, e <= 2^-11, of the definition)
        big = max([float(c.values[1][x.long()].abs().max()) for x in c.lists] + ([] if c.v is None else [float(c.v.abs().max())]))
        assert (got - want).abs().max() <= 4.3 * 2.0 ** -8 * big
    assert (got[~sees.to(dev)] == 0).all()
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("shape", range(len(FORMS)))
def test_nan_keys(dev, fmt, shape):
    """Every key of a KV head is NaN: so is every row that sees one, in that head alone."""
    c, args, kw, want = _form(600, fmt, shape)
    n, group = sum(c.nq), c.hq // c.hkv
    want = want[:n].clone()
    kc = args[1].clone()
    if fmt == "bf16":
        kc[:, :, 0] = math.nan
    else:
        kw["k_exp"][:, :, 0] = 255
    if c.k is not None:
        kw["k"][:, 0] = math.nan
    got = _ops().chunk_attention(args[0], kc, *args[2:], causal=True, **kw)[:n]
    length = [a + (0 if c.nf is None else b) for a, b in zip(c.nc, c.nf or c.nc)]
    sees = torch.cat([torch.arange(m) + (k - m + 1) > 0 for m, k in zip(c.nq, length)]).to(dev)
    assert torch.isnan(got[sees][:, :group]).all()
    assert torch.equal(got[:, group:], want[:, group:])
    assert (got[~sees] == 0).all()
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", range(len(FORMS)))
def test_scores_of_minus_infinity(dev, shape):
    """Rows whose scores are all -inf have no softmax: NaN, as the definition gives."""
    c, args, kw, want = _form(600, "bf16", shape)
    n, group = sum(c.nq), c.hq // c.hkv
    want = want[:n].clone()
    args[0][:, :group] = args[0][:, :group].abs() + 1
    args[1][:, :, 0] = -math.inf
    if c.k is not None:
        kw["k"][:, 0] = -math.inf
    got = _ops().chunk_attention(*args, causal=True, **kw)[:n]
    length = [a + (0 if c.nf is None else b) for a, b in zip(c.nc, c.nf or c.nc)]
    sees = torch.cat([torch.arange(m) + (k - m + 1) > 0 for m, k in zip(c.nq, length)]).to(dev)
    assert torch.isnan(got[sees][:, :group]).all()
    assert torch.equal(got[:, group:], want[:, group:])
    assert (got[~sees] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("nq", [1, 8, 16, 40])
@pytest.mark.parametrize("dk", [-90, 100])
def test_queries_at_the_end_of_the_range(dev, fmt, nq, dk):
    """Every other row has an element of 2^108 where its head's keys are zero,
    with a scale of 2^10: the scores are ordinary (keys of 2^-90), or those of
    the rows between are and the large rows' are zero (keys of 2^100)."""
    c = Case(86, fmt, 4, 2, [nq, 2], [200, 33], [nq, 2], False, spread=False)
    up = lambda t, e: (t.double() * 2.0 ** e).to(torch.bfloat16)  # noqa: E731
    used = c.slots.long()
    if fmt == "bf16":
        rows = c.caches[0].view(-1, 2, D)
        rows[used] = up(rows[used], dk)
        c.values[0][used] = rows[used].double()
    else:
        byte = c.exps[0].view(-1, 2)[used].int() + dk
        assert byte.min() >= 27 and byte.max() <= 246
        c.exps[0].view(-1, 2)[used] = byte.to(torch.uint8)
        c.values[0][used] *= 2.0 ** dk
    c.caches[0].view(-1, 2, D).view(torch.int8 if fmt != "bf16" else torch.bfloat16)[used, :, :1] = 0
    c.values[0][used, :, 0] = 0
    c.k = up(c.k, dk)
    c.k[:, :, 0] = 0
    c.q = up(torch.round(c.q.float() * 4) / 4, -dk - 13)  # (multiples of 2^-33 of the largest: exact in f16)
    if dk > 0:
        c.q[::2] = 0
    c.q[::2, :, 0] = 2.0 ** 108
    args, kw = c.args(dev)
    for causal in (True, False):
        c.check(_ops().chunk_attention(*args, 1024.0, causal=causal, **kw), causal, scale=1024.0)
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("tables", [True, False])
def test_expanded_rows_and_splits(dev, fmt, tables):
    """Rows of a quantised cache expanded once, with keys split between units:
    the partial results lie behind the expanded copy in one workspace."""
    nq, nc = [130, 160], [1500, 1300]
    c = Case(87, fmt, 14, 2, nq, nc, None if tables else nq, tables, page=64, spread=False)
    args, kw = c.args(dev)
    from dllmserve_b200 import _native

    sizes = (_native.KV_E4M3 if fmt == "e4m3" else _native.KV_INT8, 2, 14, 2, max(nq), max(nc), 0 if tables else max(nq))
    assert _native.lib().dllm_attn_chunk_launches(*sizes) == 3  # the expansion, the units, the merge
    for causal in (True, False):
        out = torch.full(c.q.shape, 5.0, dtype=torch.bfloat16, device=dev)
        _ops().chunk_attention(*args, causal=causal, max_context=max(nc), out=out, **kw)
        c.check(out, causal)
        assert (out[sum(nq):] == 5).all()
        again = _ops().chunk_attention(*args, causal=causal, max_context=max(nc), **kw)
        assert torch.equal(again[:sum(nq)], out[:sum(nq)])
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("nq", [[1, 3], [8, 5], [32, 20], [33, 1, 140]])
def test_fresh_rows_over_an_empty_quantised_cache(dev, fmt, nq):
    """Contexts of length zero in every kernel that reads codes: the fresh rows alone."""
    c = Case(88, fmt, 6, 6, nq, [0] * len(nq), nq, True)
    args, kw = c.args(dev)
    for causal in (True, False):
        c.check(_ops().chunk_attention(*args, causal=causal, **kw), causal)
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("nq", [[1], [8], [32], [100], [600, 600]])
def test_nan_value_of_small_weight(dev, fmt, nq):
    """A visible value that is NaN makes the row NaN, however far its score lies below the largest."""
    c = Case(89, fmt, 16, 16, nq, [128] * len(nq), None, True, page=128, spread=False)
    c.q = c.q.abs() + 1
    at = c.slots.long()
    if fmt == "bf16":
        keys = c.caches[0].view(-1, 16, D)
        keys[at] = keys[at].abs()
        keys[at[::128][:, None] + torch.arange(64)] = -32.0  # scores of -360 and less against at least 0
        c.caches[1].view(-1, 16, D)[at[3::128], 5] = math.nan
    else:
        codes = c.caches[0].view(-1, 16, D)
        codes[at] = codes[at].float().abs().to(codes.dtype)
        low = at[::128][:, None] + torch.arange(64)
        codes[low] = torch.tensor(-1.0).to(codes.dtype)
        c.exps[0].view(-1, 16)[low] = 127 + 5
        c.exps[1].view(-1, 16)[at[3::128], 5] = 255
    args, kw = c.args(dev)
    out = _ops().chunk_attention(*args, causal=False, **kw)[:sum(nq)]
    assert torch.isnan(out[:, 5]).all()
    assert torch.isfinite(out[:, :5]).all() and torch.isfinite(out[:, 6:]).all()

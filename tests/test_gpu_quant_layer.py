"""The Attention layer's regular (causal) path, and both of its paths over a
quantised cache, driven the way the model runner drives them."""
import pytest
import torch

import inputs as I
from oracle import kv_quant_ref as Q

pytestmark = pytest.mark.gpu

D = 128
TYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


@pytest.fixture(scope="module")
def dev():
    d = torch.device("cuda:0")
    torch.cuda.set_device(d)
    return d


def _cu(lens, dev):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=dev)


def _layer(fmt, hq, hk, pages, page, dev, causal):
    from dllmserve_b200.layers.attention import Attention

    layer = Attention(hq, D, D ** -0.5, hk, causal=causal)
    layer.k_cache = torch.zeros(pages, page, hk, D, dtype=torch.uint8 if fmt != "bf16" else torch.bfloat16,
                                device=dev).view(TYPES[fmt])
    layer.v_cache = torch.zeros_like(layer.k_cache)
    if fmt != "bf16":
        layer.k_exp = torch.zeros(pages, page, hk, dtype=torch.uint8, device=dev)
        layer.v_exp = torch.zeros_like(layer.k_exp)
    return layer


def _stands_for(x, fmt):
    return x.double() if fmt == "bf16" else Q.values(*Q.quantise(x, fmt))


def _check(out, q, keys, vals, fmt, what):
    o, mag, big = Q.chunk_attention(q, keys, vals, D ** -0.5, True)
    floor = None if fmt == "bf16" else Q.small_probability_floor(vals, q.shape[1])
    off = (out.cpu().double() - o).abs()
    bound = Q.attention_bound(o, mag, big, floor)
    assert (off <= bound).all(), f"{what}: {(off / bound).max():.2f} of the bound"


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
def test_causal_prefill_chunk_and_decode(dev, fmt):
    """A fresh prefill, a second chunk over block tables, then decode steps."""
    from dllmserve_b200 import ops
    from dllmserve_b200.utils.context import reset_context, set_context

    g = I.gen(5)
    hq, hk, page, pages = 8, 2, 256, 6
    layer = _layer(fmt, hq, hk, pages, page, dev, causal=True)
    tables = torch.tensor([[4, 1], [0, 5]], dtype=torch.int32)
    total = [0, 0]
    seen = [[torch.zeros(0, hk, D, dtype=torch.float64)] * 2 for _ in total]
    for step, kind in (([200, 37], "prefill"), ([90, 130], "chunk"), ([1, 1], "decode"), ([1, 1], "decode")):
        n = sum(step)
        q, k, v = (I.normal(g, (n, h, D)).to(torch.bfloat16) for h in (hq, hk, hk))
        slots = torch.cat([tables[b][torch.arange(total[b], total[b] + s) // page] * page
                           + torch.arange(total[b], total[b] + s) % page for b, s in enumerate(step)]).int().to(dev)
        total = [t + s for t, s in zip(total, step)]
        if kind == "decode":
            set_context(False, slot_mapping=slots, context_lens=torch.tensor(total, dtype=torch.int32, device=dev),
                        block_tables=tables.to(dev))
        else:
            set_context(True, cu_seqlens_q=_cu(step, dev), cu_seqlens_k=_cu(total, dev), max_seqlen_q=max(step),
                        max_seqlen_k=max(total), slot_mapping=slots,
                        block_tables=tables.to(dev) if kind == "chunk" else None)
        out = layer(*(t.to(dev).reshape(n, -1) for t in (q, k, v)))
        again = layer(*(t.to(dev).reshape(n, -1) for t in (q, k, v)))  # the next layer of the same step
        reset_context()
        assert torch.equal(out, again)
        out = out.view(n, hq, D)
        at = 0
        for b, s in enumerate(step):
            rows = slice(at, at + s)
            at += s
            stored = [_stands_for(x[rows], fmt) for x in (k, v)]
            seen[b] = [torch.cat([old, new]) for old, new in zip(seen[b], stored)]
            keys, vals = seen[b]
            if kind == "prefill":  # its own rows, not the cache's
                keys, vals = k[rows].double(), v[rows].double()
            _check(out[rows], q[rows], keys, vals, fmt, (fmt, kind, b))
    assert ops.read_device_status(dev) == 0


class Seq:
    def __init__(self, prompt, gen, state):
        self.num_prompt_tokens, self.num_tokens, self.sparse_state = prompt, prompt + gen, state


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("head_select", [True, False])
@pytest.mark.parametrize("heads", [(4, 4), (14, 2), (6, 3)])
def test_diffusion_block(dev, fmt, head_select, heads):
    """A compute-cache step and a reuse step. The selection and the first
    step's output are those of a bf16 cache, bit for bit; the stored rows are
    what quantising the bf16 cache's rows gives; the reuse step attends to
    those rows and the block's own."""
    from dllmserve_b200 import ops
    from dllmserve_b200.sparse.state import PerRequestSparseState, SparseConfig
    from dllmserve_b200.utils.context import reset_context, set_context

    hq, hk = heads
    g = I.gen(31 + hq)
    cfg = SparseConfig(enabled=True, retention_ratio=0.5, head_select=head_select)
    seqs = [Seq(100, 32, PerRequestSparseState(0, cfg, dev)), Seq(300, 64, PerRequestSparseState(1, cfg, dev)),
            Seq(40, 24, None)]
    pages, page = 4, 256
    plain, quant = _layer("bf16", hq, hk, pages, page, dev, False), _layer(fmt, hq, hk, pages, page, dev, False)
    for layer in (plain, quant):
        layer.record_selection = True
    keep = [50, 166]  # int((L - 32) * 0.5)
    slots = [torch.arange(keep[0], dtype=torch.int32) + 512, torch.randperm(256, generator=g)[:keep[1]].int()]
    mapping = [slots[0].to(dev), slots[1].to(dev), []]
    for step in (1, 2):
        for s in seqs[:2]:
            s.sparse_state.cache_state = step
        rows = [32, 32, 64] if step == 2 else [132, 364, 64]
        n = sum(rows)
        q, k, v = (I.normal(g, (n, h, D)).to(torch.bfloat16) for h in (hq, hk, hk))
        outs = []
        for layer in (plain, quant):
            set_context(True, is_diffusion=True, seqs=seqs, slot_mapping=mapping)
            outs.append(layer(*(t.to(dev).reshape(n, -1) for t in (q, k, v))))
            reset_context()
        if step == 1:
            assert torch.equal(outs[0], outs[1])
            assert torch.equal(plain.last_selection[head_select], quant.last_selection[head_select])
            want = {}
            for name in ("k", "v"):
                rows_bf16 = getattr(plain, name + "_cache").view(-1, hk, D).cpu()
                codes, exps = Q.quantise(rows_bf16, fmt)
                got = getattr(quant, name + "_cache").view(-1, hk, D).cpu().float().double()
                byte = getattr(quant, name + "_exp").view(-1, hk).cpu().long()
                at = torch.cat(slots).long()
                assert torch.equal(got[at], codes[at]) and torch.equal(byte[at], exps[at] + 127)
                rest = torch.ones(pages * page, dtype=torch.bool)
                rest[at] = False
                assert (byte[rest] == 0).all() and (got[rest] == 0).all()
                want[name] = Q.values(codes, exps)
        else:
            out = outs[1].view(n, hq, D).cpu().double()
            start = 0
            for b, r in enumerate(rows):
                keys, vals = k[start:start + r].double(), v[start:start + r].double()
                if b < 2:
                    keys = torch.cat([want["k"][slots[b].long()], keys])
                    vals = torch.cat([want["v"][slots[b].long()], vals])
                o, mag, big = Q.chunk_attention(q[start:start + r], keys, vals, D ** -0.5, False)
                bound = Q.attention_bound(o, mag, big, Q.small_probability_floor(vals, hq))
                assert ((out[start:start + r] - o).abs() <= bound).all(), b
                start += r
    assert ops.read_device_status(dev) == 0


def test_selection_into_a_quantised_cache_edges(dev):
    """Negative slots are skipped, slots past the cache flagged, a NaN marks its row."""
    from dllmserve_b200 import ops

    g = I.gen(77)
    H, L = 2, 64
    q, k, v = (I.normal(g, (L, H, D)).to(torch.bfloat16).to(dev) for _ in range(3))
    v[3, 1, 7] = float("nan")
    desc = torch.tensor([[0, L, 32, 32, 32, 0, 0, 1]], dtype=torch.int32, device=dev)  # keep all 32 candidates
    slots = torch.arange(32, dtype=torch.int32, device=dev)
    slots[4], slots[9] = -1, 64
    for head_select in (True, False):
        for fmt in ("e4m3", "int8"):
            layer = _layer(fmt, H, H, 1, 64, dev, False)
            top = torch.empty(32 * (H if head_select else 1), dtype=torch.int64, device=dev)
            ops.select_kv_store(q, k, v, desc, 32, head_select, layer.k_cache, layer.v_cache, slots, top,
                                k_exp=layer.k_exp, v_exp=layer.v_exp)
            assert ops.read_device_status(dev) in (1, 5)
            idx = top.cpu().view(-1, 32)
            byte = layer.v_exp.view(64, H).cpu()
            for h in range(H):
                order = idx[h if head_select else 0]
                for j in range(32):
                    if j in (4, 9):
                        assert byte[j, h] == 0
                    else:
                        assert (byte[j, h] == 255) == (int(order[j]) == 3 and h == 1)
            assert (byte[32:] == 0).all()
    with pytest.raises(ValueError, match="k_exp"):
        ops.select_kv_store(q, k, v, desc, 32, True, layer.k_cache, layer.v_cache, slots)
    with pytest.raises(ValueError):
        ops.select_kv_store(q, k, v, desc, 32, True, layer.k_cache, layer.v_cache.view(torch.uint8), slots,
                            k_exp=layer.k_exp, v_exp=layer.v_exp)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("chunk", [True, False])
@pytest.mark.parametrize("warm", [True, False])
def test_captured_step_follows_its_buffers(dev, fmt, chunk, warm):
    """A step captured into a graph, replayed after its lengths, tables, slots
    and rows were changed in place, gives what an eager step on them gives;
    ``warm``: the same context ran eagerly first. An eager step on the captured
    context afterwards gives it too."""
    from dllmserve_b200 import ops
    from dllmserve_b200.utils.context import get_context, reset_context, set_context, use_context

    g = I.gen(9)
    hq, hk, page, pages = 8, 2, 16, 12
    layers = [_layer(fmt, hq, hk, pages, page, dev, causal=True) for _ in range(2)]
    rows = [[5, 3], [2, 6]] if chunk else [[1, 1], [1, 1]]
    total = [[37, 20], [50, 44]]
    tables = torch.randperm(pages, generator=g).view(2, 6).int()
    data = []
    for step, tot in zip(rows, total):
        slots = torch.cat([tables[b][torch.arange(t - s, t) // page] * page + torch.arange(t - s, t) % page
                           for b, (s, t) in enumerate(zip(step, tot))]).int()
        x = [I.normal(g, (sum(step), h * D)).to(torch.bfloat16).to(dev) for h in (hq, hk, hk)]
        data.append((x, slots.to(dev), _cu(step, dev), _cu(tot, dev), torch.tensor(tot, dtype=torch.int32, device=dev)))
    fill = [I.normal(g, (pages * page, hk, D)).to(torch.bfloat16).to(dev) for _ in range(2)]
    every = torch.arange(pages * page, dtype=torch.int32, device=dev)
    for layer in layers:
        if fmt == "bf16":
            layer.k_cache.view(-1, hk, D).copy_(fill[0])
            layer.v_cache.view(-1, hk, D).copy_(fill[1])
        else:
            ops.store_kvcache_quant(*fill, layer.k_cache, layer.v_cache, layer.k_exp, layer.v_exp, every)

    def enter(slots, cu_q, cu_k, ctx):
        if chunk:
            set_context(True, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=8, max_seqlen_k=64, slot_mapping=slots,
                        block_tables=tables.to(dev))
        else:
            set_context(False, slot_mapping=slots, context_lens=ctx, block_tables=tables.to(dev))

    want = []
    for x, *meta in data:
        enter(*meta)
        want.append(layers[0](*x))
        reset_context()
    x, *meta = [[t.clone() for t in data[0][0]]] + [t.clone() for t in data[0][1:]]
    enter(*meta)
    ctx = get_context()
    if warm:
        assert torch.equal(layers[1](*x), want[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layers[1](*x)
    graph.replay()
    assert torch.equal(out, want[0])
    for have, new in zip(x + meta, data[1][0] + list(data[1][1:])):
        have.copy_(new)
    graph.replay()
    assert torch.equal(out, want[1])
    reset_context()
    use_context(ctx)
    assert torch.equal(layers[1](*x), want[1])
    reset_context()
    assert ops.read_device_status(dev) == 0


def test_decode_without_a_cache_is_refused(dev):
    from dllmserve_b200.layers.attention import Attention
    from dllmserve_b200.utils.context import reset_context, set_context

    layer = Attention(4, D, D ** -0.5, 4)
    x = torch.zeros(1, 4 * D, dtype=torch.bfloat16, device=dev)
    one = torch.ones(1, dtype=torch.int32, device=dev)
    for tables in (None, torch.zeros(1, 1, dtype=torch.int32, device=dev)):
        set_context(False, slot_mapping=one, context_lens=one, block_tables=tables)
        with pytest.raises(ValueError):
            layer(x, x, x)
        reset_context()

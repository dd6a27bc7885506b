"""Quantised KV cache: store / load against the 64-bit definition, exactly.

Codes and exponent bytes have one right value each (x * 2^-e is exact, so the
code is the rounding of an exact number), so every comparison is for equality.
"""
import ctypes

import pytest
import torch

import inputs as I
from oracle import kv_quant_ref as Q

FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


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


def _cache(pages, page, hkv, D, fmt, dev, fill=0):
    k = torch.full((pages, page, hkv, D), fill, dtype=torch.uint8, device=dev).view(FORMATS[fmt])
    e = torch.full((pages, page, hkv), fill, dtype=torch.uint8, device=dev)
    return k, k.clone(), e, e.clone()


def _rows(g, n, hkv, D):
    """Rows of very different sizes: normal values times 2^-40 .. 2^40, zero
    rows, rows whose maximum sits just above or at a power-of-two multiple of
    the format's largest value, and odd multiples of half steps (ties)."""
    x = I.normal(g, (n, hkv, D))
    x *= torch.exp2(torch.randint(-40, 41, (n, hkv, 1), generator=g).float())
    x = x.to(torch.bfloat16)
    flat = x.view(-1, D)
    m = flat.shape[0]
    for i in range(0, m, 7):
        flat[i] = 0
    for i in range(1, m, 7):
        flat[i, 0] = (448.0, 450.0, 127.0, 127.5, 7.0, 896.0)[(i // 7) % 6]
        flat[i, 1:] = torch.randint(-255, 256, (D - 1,), generator=g).float() / 2 * min(1.0, float(flat[i, 0]) / 128)
    return x


def _check_slots(fmt, cache, exp, x, slots, hkv, D, canary):
    codes, exps = Q.quantise(x, fmt)
    got = cache.cpu().view(-1, hkv, D).float().double()
    bytes_ = exp.cpu().view(-1, hkv).long()
    live = slots >= 0
    at = slots[live].long()
    assert torch.equal(got[at], codes[live])
    assert torch.equal(bytes_[at], exps[live] + 127)
    rest = torch.ones(got.shape[0], dtype=torch.bool)
    rest[at] = False
    raw = cache.cpu().view(torch.uint8).view(-1, hkv, D)
    assert (raw[rest] == canary).all() and (bytes_[rest] == canary).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("n,hkv,D", [(1, 4, 128), (7, 1, 128), (65, 32, 128), (300, 3, 128), (33, 4, 64), (19, 5, 256)])
def test_store_and_load(dev, fmt, n, hkv, D):
    g = I.gen(n * 1000 + hkv)
    page = 16
    pages = n // page + 3
    k, v = _rows(g, n, hkv, D), _rows(g, n, hkv, D)
    slots = torch.randperm(pages * page, generator=g)[:n].to(torch.int32)
    slots[5::11] = -1
    kc, vc, ke, ve = _cache(pages, page, hkv, D, fmt, dev, fill=7)
    _ops().store_kvcache_quant(k.to(dev), v.to(dev), kc, vc, ke, ve, slots.to(dev))
    _check_slots(fmt, kc, ke, k, slots, hkv, D, 7)
    _check_slots(fmt, vc, ve, v, slots, hkv, D, 7)
    ko = torch.full((n, hkv, D), float("nan"), dtype=torch.bfloat16, device=dev)
    vo = ko.clone()
    _ops().load_kvcache_quant(ko, vo, kc, vc, ke, ve, slots.to(dev))
    for x, got in ((k, ko), (v, vo)):
        want = Q.values(*Q.quantise(x, fmt))
        want[slots < 0] = 0
        assert torch.equal(got.cpu().double(), want)
        # half a step: 2^-4 of the value (e4m3, above its subnormals), half the unit (int8)
        unit = torch.exp2(Q.quantise(x, fmt)[1].double()).unsqueeze(-1)
        x64 = x.double().masked_fill((slots < 0).view(-1, 1, 1), 0)
        half = (x64.abs() * 2.0 ** -4).clamp(min=0) + unit * 2.0 ** -10 if fmt == "e4m3" else unit / 2
        assert ((want - x64).abs() <= half).all()
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("pad", [8, 16])  # rows on 16-byte and on 32-byte boundaries
def test_strided_rows(dev, fmt, pad):
    g = I.gen(3 + pad)
    n, hq, hkv, D = 45, 3, 2, 128
    width = (hq + 2 * hkv) * D + pad
    qkv = I.normal(g, (n, width)).to(torch.bfloat16).to(dev)
    k = qkv[:, hq * D:(hq + hkv) * D].view(n, hkv, D)
    v = qkv[:, (hq + hkv) * D:(hq + 2 * hkv) * D].view(n, hkv, D)
    slots = torch.randperm(64, generator=g)[:n].to(torch.int32)
    kc, vc, ke, ve = _cache(4, 16, hkv, D, fmt, dev)
    _ops().store_kvcache_quant(k, v, kc, vc, ke, ve, slots.to(dev))
    _check_slots(fmt, kc, ke, k.cpu(), slots, hkv, D, 0)
    _check_slots(fmt, vc, ve, v.cpu(), slots, hkv, D, 0)
    out = torch.full((n, width), 9.0, dtype=torch.bfloat16, device=dev)
    ko = out[:, hq * D:(hq + hkv) * D].view(n, hkv, D)
    vo = out[:, (hq + hkv) * D:(hq + 2 * hkv) * D].view(n, hkv, D)
    _ops().load_kvcache_quant(ko, vo, kc, vc, ke, ve, slots.to(dev))
    assert torch.equal(ko.cpu().double(), Q.values(*Q.quantise(k.cpu(), fmt)))
    assert torch.equal(vo.cpu().double(), Q.values(*Q.quantise(v.cpu(), fmt)))
    assert (out[:, :hq * D] == 9).all() and (out[:, (hq + 2 * hkv) * D:] == 9).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_extreme_values(dev, fmt):
    """Largest and smallest bf16 numbers, infinities and NaN."""
    top = float(torch.finfo(torch.bfloat16).max)
    rows = [[top, -top, 1.0], [2.0 ** -133, -(2.0 ** -126)], [2.0 ** -95, 2.0 ** -99, 2.0 ** -108],
            [float("inf"), 3.0, -1.5], [float("-inf")], [float("nan"), 2.0], [3.0e38, 1.0e38]]
    x = torch.zeros(len(rows), 1, 128)
    for i, r in enumerate(rows):
        x[i, 0, :len(r)] = torch.tensor(r)
    x = x.to(torch.bfloat16)
    slots = torch.arange(len(rows), dtype=torch.int32, device=dev)
    kc, vc, ke, ve = _cache(1, 16, 1, 128, fmt, dev)
    ones = torch.ones_like(x)
    _ops().store_kvcache_quant(x.to(dev), ones.to(dev), kc, vc, ke, ve, slots)
    assert _ops().read_device_status(dev) == 5
    codes, exps = Q.quantise(x, fmt)
    keep = [0, 1, 2, 3, 4, 6]  # row 5 holds a NaN: all of it reads as NaN
    got = kc.cpu().view(-1, 1, 128)[:len(rows)].float().double()
    assert torch.equal(got[keep], codes[keep])
    assert torch.isfinite(got).all()
    assert torch.equal(ke.cpu().view(-1, 1)[keep].long(), exps[keep] + 127)
    assert int(ke.cpu().view(-1)[5]) == 255
    ko, vo = torch.zeros_like(x, device=dev), torch.zeros_like(x, device=dev)
    _ops().load_kvcache_quant(ko, vo, kc, vc, ke, ve, slots)
    want = Q.values(codes, exps)
    assert torch.equal(ko.cpu()[keep].double(), want[keep])
    assert torch.isfinite(ko.cpu()[keep].float()).all() and torch.isnan(ko.cpu()[5].float()).all()
    # finite rows do not set the status word
    _ops().store_kvcache_quant(ones.to(dev), ones.to(dev), kc, vc, ke, ve, slots)
    assert _ops().read_device_status(dev) == 0


@pytest.mark.gpu
def test_slot_edge_cases(dev):
    ops = _ops()
    kc, vc, ke, ve = _cache(1, 16, 2, 128, "int8", dev)
    x = torch.ones(3, 2, 128, dtype=torch.bfloat16, device=dev)
    slots = torch.tensor([-1, 5, 16], dtype=torch.int32, device=dev)
    ops.store_kvcache_quant(x, x, kc, vc, ke, ve, slots)
    assert ops.read_device_status(dev) == 1
    assert kc.cpu().view(16, -1).any(1).nonzero().flatten().tolist() == [5]
    ko = torch.full_like(x, 3.0)
    vo = ko.clone()
    ops.load_kvcache_quant(ko, vo, kc, vc, ke, ve, slots)
    assert ops.read_device_status(dev) == 1
    assert (ko[0] == 0).all() and (ko[1] == 1).all() and (ko[2] == 0).all()
    # a slot never written reads as zeros
    ops.load_kvcache_quant(ko, vo, kc, vc, ke, ve, torch.tensor([0, 1, 2], dtype=torch.int32, device=dev))
    assert (ko == 0).all() and (vo == 0).all()
    ops.store_kvcache_quant(x[:0], x[:0], kc, vc, ke, ve, slots[:0])  # nothing to do
    assert ops.read_device_status(dev) == 0


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """Slots whose codes lie more than 2^31 bytes into the cache."""
    hkv, D, page = 32, 128, 256
    pages = 2300  # 2.4 GB of codes
    kc = torch.zeros(pages, page, hkv, D, dtype=torch.int8, device=dev)
    vc = torch.zeros_like(kc)
    ke = torch.zeros(pages, page, hkv, dtype=torch.uint8, device=dev)
    ve = torch.zeros_like(ke)
    g = I.gen(77)
    x = I.normal(g, (3, hkv, D)).to(torch.bfloat16)
    slots = torch.tensor([pages * page - 1, 0, 2 ** 31 // (hkv * D) + 5], dtype=torch.int32)
    _ops().store_kvcache_quant(x.to(dev), x.to(dev), kc, vc, ke, ve, slots.to(dev))
    assert int((ke.view(-1, hkv) != 0).all(1).sum()) == 3
    ko, vo = torch.empty_like(x, device=dev), torch.empty_like(x, device=dev)
    _ops().load_kvcache_quant(ko, vo, kc, vc, ke, ve, slots.to(dev))
    want = Q.values(*Q.quantise(x, "int8"))
    assert torch.equal(ko.cpu().double(), want) and torch.equal(vo.cpu().double(), want)
    assert torch.equal(kc.view(-1, hkv, D)[slots.long().to(dev)].cpu().double(), Q.quantise(x, "int8")[0])
    assert _ops().read_device_status(dev) == 0


def test_exponent_rule():
    """The oracle's rule at the borders (the kernel is compared with it)."""
    assert Q.exponent(torch.tensor([448.0]), "e4m3") == 0 and Q.exponent(torch.tensor([450.0]), "e4m3") == 1
    assert Q.exponent(torch.tensor([127.0]), "int8") == 0 and Q.exponent(torch.tensor([127.5]), "int8") == 1
    assert Q.exponent(torch.tensor([0.0, -0.0]), "int8") == -100
    y = torch.tensor([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 1000.0, -0.3])
    assert Q.round_code(y, "e4m3").tolist() == y.clamp(-448, 448).to(torch.float8_e4m3fn).double().tolist()


def test_refusals():
    """Bad arguments are refused before any device work."""
    from dllmserve_b200 import _native, ops

    lib = _native.lib()
    f = lib.dllm_store_kvcache_quant

    def call(fn, key=64, ks=256, val=64, vs=256, kc=64, vc=64, ke=64, ve=64, sl=64, n=4, h=2, D=128, fmt=1, slots=8):
        return fn(key, ks, val, vs, kc, vc, ke, ve, sl, n, h, D, fmt, slots, None, None)

    for fn in (lib.dllm_store_kvcache_quant, lib.dllm_load_kvcache_quant):
        assert call(fn, n=0) == _native.DLLM_OK
        assert call(fn, fmt=0) == _native.DLLM_ERR_UNSUPPORTED
        assert call(fn, fmt=3) == _native.DLLM_ERR_UNSUPPORTED
        assert call(fn, D=96) == _native.DLLM_ERR_UNSUPPORTED
        assert call(fn, n=-1) == _native.DLLM_ERR_INVALID_ARG
        assert call(fn, h=0) == _native.DLLM_ERR_INVALID_ARG
        assert call(fn, ke=None) == _native.DLLM_ERR_INVALID_ARG
        assert call(fn, ks=255) == _native.DLLM_ERR_INVALID_ARG
        assert call(fn, ks=260) == _native.DLLM_ERR_ALIGNMENT
        assert call(fn, key=72) == _native.DLLM_ERR_ALIGNMENT
        assert call(fn, kc=40) == _native.DLLM_ERR_ALIGNMENT
        assert call(fn, n=2 ** 40) == _native.DLLM_ERR_TOO_LARGE
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    c = torch.zeros(1, 16, 2, 128, dtype=torch.int8)
    e = torch.zeros(1, 16, 2, dtype=torch.uint8)
    s = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.store_kvcache_quant(x, x, c, c, e, e, s)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.store_kvcache_quant(x.float(), x.float(), c, c, e, e, s)
    with pytest.raises(ValueError, match="shape"):
        ops.load_kvcache_quant(x, x[:1], c, c, e, e, s)
    with pytest.raises(ValueError, match="heads"):
        ops.load_kvcache_quant(x.transpose(0, 1).contiguous().transpose(0, 1), x, c, c, e, e, s)
    assert f is not None and isinstance(ctypes.c_int(0), ctypes.c_int)


@pytest.mark.gpu
def test_refusals_on_device_tensors(dev):
    ops = _ops()
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=dev)
    c = torch.zeros(1, 16, 2, 128, dtype=torch.int8, device=dev)
    e = torch.zeros(1, 16, 2, dtype=torch.uint8, device=dev)
    s = torch.zeros(2, dtype=torch.int32, device=dev)
    bad = [
        (x, x, c.view(torch.uint8), c, e, e, s), (x, x, c, c.view(torch.float8_e4m3fn), e, e, s),
        (x, x, c[:, :, :1], c, e, e, s), (x, x, c, c, e[:, :8], e, s), (x, x, c, c, e.int(), e, s),
        (x, x, c, c, e, e, s.long()), (x, x, c, c, e, e, s[:1]),
        (x, x, c, torch.zeros(2, 16, 2, 128, dtype=torch.int8, device=dev), e,
         torch.zeros(2, 16, 2, dtype=torch.uint8, device=dev), s),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            ops.store_kvcache_quant(*args)
    y = torch.zeros(2, 2, 96, dtype=torch.bfloat16, device=dev)
    with pytest.raises(NotImplementedError):
        ops.store_kvcache_quant(y, y, c.new_zeros(1, 16, 2, 96), c.new_zeros(1, 16, 2, 96), e, e, s)


def test_selection_refusals():
    from dllmserve_b200 import _native

    fn = _native.lib().dllm_select_kv_store_quant

    def call(fmt=1, ke=64, ve=64, n=1, klen=32, hd=128, h=2):
        return fn(64, 256, 64, 256, 64, 256, 64, n, klen, h, 2, hd, 1, 64, 64, ke, ve, fmt, 64, 64, None, None, None)

    assert call(fmt=0) == _native.DLLM_ERR_UNSUPPORTED
    assert call(ke=None) == _native.DLLM_ERR_INVALID_ARG
    assert call(hd=64) == _native.DLLM_ERR_UNSUPPORTED
    assert call(h=3) == _native.DLLM_ERR_UNSUPPORTED
    assert call(klen=20000) == _native.DLLM_ERR_TOO_LARGE
    assert call(n=0, ke=None) == _native.DLLM_OK

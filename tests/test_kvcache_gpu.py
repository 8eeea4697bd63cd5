"""GPU: the paged key/value cache (ngram_amd.kvcache): codes and scales against the definition restated in 32 bits (the
same IEEE operations: they are equal), the values against float64, strides, head sizes that are not whole loads or pages,
slots out of range, rows of zeros, NaN and infinities, addresses past 2^32 bytes, and the refusals.

Tolerance of the values against x in 64 bits: int8 rounds to half a step a / 127, of which the 32-bit products move it by at
most 127.5 * 3 * 2^-24 of a step more; e4m3 rounds to 2^-4 of the value, or half of 2^-9 in codes."""

import pytest
import torch

from ngram_amd.kvcache import KVCache, padded

pytestmark = pytest.mark.gpu

TOP = {"int8": 127.0, "fp8": 448.0}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _quantise(x, codes):
    x = x.float()
    a = x.abs().amax(-1)
    top = torch.full_like(a, TOP[codes])  # a tensor: dividing by or into a number is a product with a reciprocal
    y = x * torch.where(a > 0, top / a, 0.0)[..., None]
    return (y.round() if codes == "int8" else y.to(torch.float8_e4m3fn).float()), a / top


def _held(cache, slots):
    """codes and scales of slots: [n, heads, row], [n, heads]"""
    page, row = slots // cache.page, slots % cache.page
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        bits = c.view(torch.uint8 if c.element_size() == 1 else torch.int16)
        out.append((bits[page, :, row].view(c.dtype), None if s is None else s[page, :, row]))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("n,heads,dim,page", [(1, 1, 1, 16), (7, 3, 64, 16), (50, 8, 128, 64), (33, 5, 80, 32),
                                              (40, 2, 192, 128), (21, 1, 250, 16), (2000, 4, 96, 256)])
def test_write_and_read(gpu, dtype, codes, n, heads, dim, page):
    g = torch.Generator().manual_seed(n + dim)
    k, v = ((torch.randn((n, heads, dim), generator=g) * 3).to(dtype).cuda() for _ in range(2))
    pages = n // page + 4
    cache = KVCache.empty(pages, page, heads, dim, codes)
    slots = torch.randperm(pages * page, generator=g)[:n].cuda()
    cache.write(k, v, slots)
    for x, (c, s) in zip((k, v), _held(cache, slots)):
        want, scale = _quantise(x, codes)
        assert torch.equal(c.float()[..., :dim], want) and torch.equal(s, scale)
        assert not c.float()[..., dim:].any() and c.shape[-1] == padded(dim)
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots.cpu()] = False
    for c, s in _held(cache, rest.nonzero()[:, 0].cuda()):
        assert not c.float().any() and not s.any()  # nothing else was written
    for want_type in (torch.float32, torch.bfloat16, torch.float16):
        for x, got, (c, s) in zip((k, v), cache.read(slots, want_type), _held(cache, slots)):
            assert got.dtype == want_type and torch.equal(got, (c.float()[..., :dim] * s[..., None]).to(want_type))
            if want_type == torch.float32:
                a = x.double().abs().amax(-1, keepdim=True)
                step = a / 127 * (0.5 + 127.5 * 3 * 2.0**-24)
                near = step if codes == "int8" else torch.maximum(x.double().abs() * 2.0**-4, a / 448 * 2.0**-10) * 1.0001
                assert ((got.double() - x.double()).abs() <= near).all()


@pytest.mark.parametrize("codes", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 100, 256])
def test_sixteen_bits_hold_the_values(gpu, codes, dim):
    k, v = (torch.randn((90, 3, dim)).to(DT[codes]).cuda() for _ in range(2))
    k[5, 1, 3] = float("inf")
    cache = KVCache.empty(9, 16, 3, dim, codes)
    slots = torch.randperm(9 * 16)[:90].cuda()
    cache.write(k, v, slots)
    rk, rv = cache.read(slots, DT[codes])
    assert torch.equal(rk, k) and torch.equal(rv, v)


def test_strides(gpu):
    """Keys and values as views of one projection's output, at an offset that no wide load is aligned to, and transposed."""
    n, heads, dim = 60, 4, 72
    cache = KVCache.empty(5, 16, heads, dim, "int8")
    qkv = torch.randn((n, 3 * heads * dim + 1), dtype=torch.float32).bfloat16().cuda()
    slots = torch.arange(10, 10 + n).cuda()
    for k, v in ((qkv[:, 1:1 + heads * dim].view(n, heads, dim), qkv[:, -heads * dim:].view(n, heads, dim)),
                 (qkv[:, :heads * dim].view(n, dim, heads).transpose(1, 2), qkv[:, 1:1 + heads * dim].view(n, heads, dim)),
                 (qkv[:1, :heads * dim].view(1, heads, dim).expand(n, heads, dim),) * 2):
        cache.write(k, v, slots)
        for x, (c, s) in zip((k, v), _held(cache, slots)):
            want, scale = _quantise(x.contiguous(), "int8")
            assert torch.equal(c.float()[..., :dim], want) and torch.equal(s, scale)


def test_slots_out_of_range(gpu):
    cache = KVCache.empty(4, 16, 2, 64, "fp8")
    k, v = (torch.randn((8, 2, 64)).cuda() for _ in range(2))
    slots = torch.tensor([-1, 3, 64, 1 << 40, -(1 << 62), 63, 0, 5]).cuda()
    cache.write(k, v, slots)
    ok = (slots >= 0) & (slots < 64)
    got = cache.read(slots, torch.float32)[0]
    assert not got[~ok].any() and (got[ok] != 0).any(-1).all()
    assert int((cache.k_scale != 0).sum()) == 2 * int(ok.sum())


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_zeros_and_values_that_are_not_finite(gpu, codes):
    x = torch.randn((7, 2, 96))
    x[1] = 0
    x[2, 0, 5], x[3, 1, 95], x[4, 0, 0] = float("nan"), float("inf"), -float("inf")
    x[5] = 1e-44  # its inverse is past the largest float
    x[6, 0, 3] = 3e38
    cache = KVCache.empty(1, 16, 2, 96, codes)
    at = torch.arange(7).cuda()
    cache.write(x.cuda(), x.cuda(), at)
    (c, s), _ = _held(cache, at)
    bad = ~torch.isfinite(x).all(-1)
    assert torch.equal(torch.isnan(s).cpu(), bad) and not c.float()[bad.cuda()].any()
    assert not s[1].any() and not s[5].any() and not c.float()[1].any() and not c.float()[5].any()
    got = cache.read(at, torch.float32)[0].cpu()
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()


def test_addresses_past_32_bits(gpu):
    """A cache of over 2^32 bytes a side: its last and first slots, and one past 2^31 rows' worth of bytes."""
    pages = (1 << 32) // (2 * 4096 * 64) + 3  # 64-byte rows of int8, two heads, pages of 4096
    k = torch.empty((pages, 2, 4096, 64), dtype=torch.int8, device="cuda")
    s = torch.empty((pages, 2, 4096), dtype=torch.float32, device="cuda")
    cache = KVCache(k, k, s, s, dim=64)
    total = pages * 4096
    slots = torch.tensor([0, total // 2 + 17, total - 1]).cuda()
    x = torch.randn((3, 2, 64)).cuda()
    cache.write(x, x, slots)
    got = cache.read(slots, torch.float32)[0]
    want, scale = _quantise(x, "int8")
    assert torch.equal(got, want * scale[..., None])


def test_slots_of_positions(gpu):
    cache = KVCache.empty(20, 16, 1, 64, "int8")
    table = torch.tensor([[3, 19, -1, 25], [0, 1, 2, 4]], dtype=torch.int32).cuda()
    start = torch.tensor([10, 62], dtype=torch.int32).cuda()
    got = cache.slots(table, start, 30).cpu()
    for b in range(2):
        for i in range(30):
            p = int(start[b]) + i
            g = int(table[b, p // 16]) if p < 64 else -1
            assert got[b, i] == (g * 16 + p % 16 if 0 <= g < 20 else -1), (b, i)
    assert cache.slots(table, start, 0).shape == (2, 0)
    assert torch.equal(cache.slots(table.repeat(1, 2)[:, :4], start, 30).cpu(), got)  # rows with a stride
    assert (cache.slots(table, torch.tensor([-5, -1], dtype=torch.int32).cuda(), 3).cpu()[:, 0] == -1).all()


def test_nothing_to_write(gpu):
    cache = KVCache.empty(1, 16, 2, 64, "int8")
    none = torch.zeros((0, 2, 64)).cuda()
    cache.write(none, none, torch.zeros(0, dtype=torch.int64).cuda())
    assert cache.read(torch.zeros(0, dtype=torch.int64).cuda())[0].shape == (0, 2, 64)
    assert not cache.k.any()


def test_refusals(gpu):
    e = KVCache.empty
    for args in ((1, 16, 1, 64, "int4"), (1, 8, 1, 64), (1, 48, 1, 64), (1, 8192, 1, 64), (0, 16, 1, 64), (1, 16, 0, 64),
                 (1, 16, 1, 0), (1, 16, 1, 257)):
        with pytest.raises(ValueError):
            e(*args)
    c = e(2, 16, 2, 64, "int8")
    for args in ((c.k, c.v), (c.k, c.v, c.k_scale), (c.k, c.v[:1], c.k_scale, c.v_scale), (c.k, c.v, c.k_scale[:1], c.v_scale),
                 (c.k.cpu(), c.v.cpu(), c.k_scale.cpu(), c.v_scale.cpu()), (c.k.float(), c.v.float()),
                 (c.k, c.v, c.k_scale.double(), c.v_scale.double()), (c.k.transpose(0, 2), c.v.transpose(0, 2))):
        with pytest.raises(ValueError):
            KVCache(*args)
    with pytest.raises(ValueError):
        KVCache(c.k, c.v, c.k_scale, c.v_scale, dim=65)
    b = e(2, 16, 2, 64, "bf16")
    with pytest.raises(ValueError):
        KVCache(b.k, b.v, c.k_scale, c.v_scale)
    x, at = torch.randn(3, 2, 64).cuda(), torch.arange(3).cuda()
    for k, v, s in ((x, x.half(), at), (x[:2], x, at), (x, x, at[:2]), (x, x, at.int()), (x, x, at.cpu()),
                    (x.double(), x.double(), at), (x[..., :63], x[..., :63], at), (x.cpu(), x.cpu(), at)):
        with pytest.raises(ValueError):
            c.write(k, v, s)
    with pytest.raises(ValueError):
        b.write(x, x, at)
    with pytest.raises(ValueError):
        c.read(at, torch.int8)
    with pytest.raises(ValueError):
        c.slots(torch.zeros((1, 2)).cuda(), torch.zeros(1, dtype=torch.int32).cuda(), 1)
    with pytest.raises(ValueError):
        c.slots(torch.zeros((1, 2), dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda(), 1)


def test_gradients_are_refused(gpu):
    """Writing quantises and has no backward pass: keys or values that require gradients raise instead of losing them."""
    import torch.autograd.forward_ad as fw

    c = KVCache.empty(2, 16, 2, 64, "int8")
    x, at = torch.randn(3, 2, 64).cuda(), torch.arange(3).cuda()
    y = x.clone().requires_grad_(True)
    for k, v in ((y, x), (x, y)):
        with pytest.raises(RuntimeError, match="gradient"):
            c.write(k, v, at)
    with fw.dual_level(), pytest.raises(RuntimeError, match="gradient"):
        c.write(fw.make_dual(x, x), x, at)
    assert not c.k.any()
    with torch.no_grad():
        c.write(y, y, at)
    assert c.k.any()
    b = KVCache.empty(2, 16, 2, 64, "bf16")
    with pytest.raises(ValueError):
        KVCache(b.k.clone().requires_grad_(True), b.v)  # the cache is no leaf to train


def test_the_tensors_are_not_replaced(gpu):
    """The cache's tensors are its own for good: assigning others raises. One whose memory is exchanged in place is used
    where it lies now."""
    c = KVCache.empty(2, 16, 2, 64, "int8")
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    x, at = torch.randn(3, 2, 64).cuda(), torch.arange(3).cuda()
    before = [t.data for t in (c.k, c.v, c.k_scale, c.v_scale)]  # the old memory stays alive
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        t.data = torch.zeros_like(t)
    c.write(x, x, at)
    assert not any(t.float().any() for t in before)
    want, scale = _quantise(x, "int8")
    assert torch.equal(c.read(at, torch.float32)[1], want * scale[..., None])


def test_counts_past_32_bits_are_refused(gpu):
    c = KVCache.empty(2, 16, 2, 64, "int8")
    table, start = torch.zeros((1, 2), dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    for count in (1 << 31, (1 << 32) + 1):
        with pytest.raises(ValueError):
            c.slots(table, start, count)

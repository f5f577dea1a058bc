"""Parity of the paged 8-bit KV cache operators with the plain 64-bit restatement in
oracle/kv_cache.py.

Store, copies and table operations are compared exactly: scales are powers of two, so every
division by one is exact and the codes' rounding is the only one.  Attention is compared within a
bound derived per output from its own terms.  With u the unit roundoff of the output type, e_s the
error of a score and e_p that of a probability's rounding before the product with V,
  |error| <= (u + e_p + 2 e_s + 2^-16) * sum_j p_j |v_j|,
where e_s = 2^-23 * D * scale * max_j sum_d |q_d k_jd| (D fp32 additions of products that are each
rounded once, with queries rounded to within 2^-24 of their largest element where the kernel holds
them in fp16), e_p = 2^-11 for 16-bit queries (probabilities in fp16) and 0 for fp32 queries, and
2^-16 covers the hardware base-2 exponential and the fp32 sums over up to 2^7 rescaled blocks."""

import math

import pytest
import torch

import oracle.kv_cache as OK

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ntops_b200 import kv_cache as kc

DEV = "cuda"
E4M3, I8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROUNDOFF = {BF16: 2.0**-8, F16: 2.0**-11, F32: 2.0**-24}


def _values(codes):
    """Codes on any device -> fp64 values on the CPU."""
    return codes.cpu().double() if codes.dtype == I8 else codes.cpu().float().double()


def _random_cache(layers, pages, heads, page, d, code, scale_lo=-8, scale_hi=-4):
    shape = (layers, pages, heads, page, d)
    top = OK.QMAX[code]

    def codes():
        x = (torch.randn(shape) * (top / 3)).clamp(-top, top)
        return (x.round() if code == I8 else x).to(code).to(DEV)

    def scales():
        return torch.exp2(torch.randint(scale_lo, scale_hi, shape[:3]).float()).to(DEV)

    return kc.PagedKVCache(codes(), codes(), scales(), scales())


def _table(lengths, page, pages, extra=0):
    """Random distinct pages for each row's tokens, -1 after them."""
    m = max(-(-n // page) for n in lengths) + extra
    perm = torch.randperm(pages).tolist()
    rows = [[perm.pop() if i < -(-n // page) else -1 for i in range(m)] for n in lengths]
    return torch.tensor(rows, dtype=torch.int32).view(len(lengths), m)


def _check_attention(got, q, cache, layer, table, lengths, scale, causal, start=None):
    c = cache.layer(layer)
    want, (mag, dots) = OK.attention(q.cpu(), _values(c.key), _values(c.value), c.key_scale.cpu().double(),
                                     c.value_scale.cpu().double(), table, lengths, scale, causal, start)
    e_s = 2.0**-23 * q.shape[-1] * dots.unsqueeze(-1)
    e_p = 0.0 if q.dtype == F32 else 2.0**-11
    tol = (ROUNDOFF[q.dtype] + e_p + 2 * e_s + 2.0**-16) * mag + 1e-30
    err = (got.cpu().double() - want).abs()
    assert got.dtype == q.dtype and got.shape == q.shape
    worst = (err / tol).max()
    assert (err <= tol).all(), f"error up to {worst:.3g} of its bound"


# b, lengths, sq, hq, hkv, d, page, code, dtype
ATTEND = [
    ([1], 1, 4, 1, 128, 16, E4M3, BF16),
    ([17, 0, 1, 64], 1, 8, 2, 128, 16, E4M3, BF16),
    ([300, 1025, 129, 128, 127], 1, 32, 8, 128, 64, E4M3, F16),
    ([4000], 1, 8, 8, 64, 32, I8, BF16),
    ([777, 2], 4, 8, 2, 64, 16, I8, F16),
    ([530, 3], 5, 12, 4, 128, 32, E4M3, BF16),
    ([1000], 1, 16, 1, 128, 128, I8, F16),
    ([260], 2, 16, 2, 128, 16, E4M3, BF16),
    ([100, 333], 1, 6, 2, 96, 16, E4M3, BF16),
    ([65], 3, 4, 4, 80, 8, I8, F16),
    ([70, 5], 1, 4, 2, 256, 16, E4M3, BF16),
    ([33, 200], 1, 4, 2, 33, 5, I8, BF16),
    ([150, 40], 1, 8, 2, 128, 16, E4M3, F32),
    ([150, 40], 7, 4, 2, 64, 16, I8, F32),
    ([400, 390], 33, 8, 2, 128, 16, E4M3, BF16),
    ([300, 70], 70, 4, 1, 64, 64, I8, F16),
    ([260], 130, 8, 8, 128, 32, E4M3, F16),
    ([129, 640], 65, 16, 2, 128, 128, I8, BF16),
    ([500, 49], 1, 8, 2, 128, 48, E4M3, BF16),  # pages of 16-token groups that are no power of two
    ([500, 49], 24, 4, 2, 64, 48, I8, F16),
    ([385, 97], 40, 8, 2, 128, 48, E4M3, BF16),
    ([700, 257], 1, 4, 2, 64, 256, I8, BF16),
    ([700, 257], 45, 4, 2, 128, 256, E4M3, F16),
    ([333, 20], 8, 8, 2, 128, 16, I8, BF16),    # 32 rows: the most of the few-row kernel
    ([333, 20], 33, 2, 2, 128, 16, I8, BF16),   # one more
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,sq,hq,hkv,d,page,code,dtype", ATTEND)
def test_attention(lengths, sq, hq, hkv, d, page, code, dtype, causal):
    pages = sum(-(-n // page) for n in lengths) + 3
    cache = _random_cache(2, pages, hkv, page, d, code)
    table = _table(lengths, page, pages, extra=1)
    q = torch.randn(len(lengths), sq, hq, d).to(dtype).transpose(1, 2)
    n = torch.tensor(lengths, dtype=torch.int32)
    scale = 1 / math.sqrt(d)
    got = kc.attention(q.to(DEV), cache.layer(1), table.to(DEV), n.to(DEV), is_causal=causal)
    assert got.stride() == q.stride()
    _check_attention(got, q, cache, 1, table, n, scale, causal)


@pytest.mark.parametrize("b,sq,group,d,code,dtype", [
    # fewer segments than multiprocessors: keys are cut
    (3, 33, 1, 128, E4M3, BF16), (3, 32, 4, 128, I8, F16), (3, 129, 1, 64, E4M3, F16), (3, 96, 4, 128, E4M3, BF16),
    (3, 64, 2, 64, I8, BF16),
    # and more
    (20, 33, 1, 128, E4M3, BF16), (20, 17, 2, 64, I8, F16), (10, 257, 1, 128, I8, BF16),
])
def test_attention_last_rows_share_the_keys(b, sq, group, d, code, dtype):
    """Up to 128 rows, alone or after whole tiles of 256: odd and even numbers of key blocks, values'
    scales that grow from page to page, rows with none or one of the blocks."""
    page, hkv = 32, 8
    lengths = [(1000, 0, 257, 128, 1, 640, 129)[i % 7] for i in range(b)]
    cache = _random_cache(1, sum(-(-n // page) for n in lengths) + 1, hkv, page, d, code, scale_lo=-9, scale_hi=-3)
    table = _table(lengths, page, cache.key.shape[1])
    q = torch.randn(b, hkv * group, sq, d).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32)
    got = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV), is_causal=b == 3)
    _check_attention(got, q, cache, 0, table, n, 1 / math.sqrt(d), b == 3)


@pytest.mark.parametrize("dtype,d,sq", [(BF16, 128, 1), (F16, 64, 3), (F32, 64, 2), (BF16, 128, 40)])
def test_attention_rows_that_see_nothing(dtype, d, sq):
    """Empty rows, rows of holes only, and queries before the first key give zeros."""
    page, hkv, hq = 16, 2, 4
    cache = _random_cache(1, 12, hkv, page, d, E4M3)
    table = torch.tensor([[0, 1, 2], [-1, -1, -1], [3, -1, 4], [5, 1000, 6], [7, 8, 9]], dtype=torch.int32)
    n = torch.tensor([0, 40, 41, 48, 30], dtype=torch.int32)
    start = torch.tensor([0, 39, 45, 47, -2], dtype=torch.int32)
    q = torch.randn(5, hq, sq, d).to(dtype)
    got = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV), scale=0.2, start=start.to(DEV))
    _check_attention(got, q, cache, 0, table, n, 0.2, True, start)
    assert (got[:2] == 0).all() and (got[4, :, :2] == 0).all()
    assert torch.isfinite(got.float()).all()


@pytest.mark.parametrize("dtype,d,sq", [(BF16, 128, 1), (F16, 64, 3), (F32, 64, 2), (BF16, 128, 40)])
def test_attention_ignores_what_lies_past_the_length(dtype, d, sq):
    """NaN codes after a row's last token and NaN scales of pages it does not use change nothing."""
    page, hkv = 32, 2
    cache = _random_cache(1, 9, hkv, page, d, E4M3)
    table = torch.tensor([[4, 2, 7], [1, 5, -1]], dtype=torch.int32)
    n = torch.tensor([75, 33], dtype=torch.int32)
    q = torch.randn(2, 4, sq, d).to(dtype)
    want = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV))
    for t in (cache.key, cache.value):
        raw = t.view(torch.uint8)
        raw[0, 7, :, 75 - 64:] = 0x7F
        raw[0, 5, :, 1:] = 0xFF
        raw[0, [0, 3, 6, 8]] = 0x7F
    for s in (cache.key_scale, cache.value_scale):
        s[0, [0, 3, 6, 8]] = float("nan")
    got = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV))
    assert torch.equal(got, want)
    # a NaN among the tokens that are seen does show
    cache.value.view(torch.uint8)[0, 4, 0, 3, 5] = 0x7F
    got = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV))
    assert torch.isnan(got[0, :2, :, 5]).all() and torch.isfinite(got[0, 2:].float()).all()


@pytest.mark.parametrize("sq", [1, 20])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_attention_scales(scale, sq):
    cache = _random_cache(1, 8, 2, 16, 64, I8, -20, 0)
    table = _table([100], 16, 8)
    n = torch.tensor([100], dtype=torch.int32)
    q = (torch.randn(1, 4, sq, 64) * 1e-3).to(BF16)
    q[0, 1] *= 1e6
    q[0, 2] *= 1e-30
    got = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV), scale=scale)
    _check_attention(got, q, cache, 0, table, n, scale, True)


def test_attention_value_scales_far_apart():
    """Pages whose value scales differ by 2^60, in both orders, with scores that prefer either."""
    cache = _random_cache(1, 8, 1, 16, 64, E4M3)
    cache.value_scale.copy_(torch.exp2(torch.tensor([0., 60, 3, -50, 40, -90, 1, 5])).view(1, 8, 1))
    table = torch.tensor([[5, 3, 2, 1, 0], [1, 4, 5, 3, 2]], dtype=torch.int32)
    n = torch.tensor([80, 79], dtype=torch.int32)
    q = torch.randn(2, 4, 1, 64).to(F32)
    for dtype in (F32, BF16):
        qd = q.to(dtype)
        got = kc.attention(qd.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV))
        _check_attention(got, qd, cache, 0, table, n, 0.125, True)


@pytest.mark.parametrize("sq", [1, 4, 24])
def test_attention_layouts(sq):
    """Token-major pages, strided queries, tables and lengths, and a cache that is a view."""
    pages, page, hkv, d = 10, 16, 2, 128
    base = _random_cache(2, pages, hkv, page, d, E4M3)
    flat = [t.transpose(2, 3).contiguous() for t in (base.key.view(torch.uint8), base.value.view(torch.uint8))]
    wide = [torch.zeros(2, pages, page, hkv, d + 16, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for w, f in zip(wide, flat):
        w[..., :d] = f
    scales = [torch.stack((s, s), -1)[..., 0] for s in (base.key_scale, base.value_scale)]
    lengths = [97, 33]
    table = _table(lengths, page, pages)
    n = torch.tensor(lengths, dtype=torch.int32)
    q = torch.randn(2, sq, 8, d).to(BF16)
    want = kc.attention(q.transpose(1, 2).contiguous().to(DEV), base.layer(1), table.to(DEV), n.to(DEV))
    t2 = torch.stack((table, table), -1).to(DEV)[..., 1]
    n2 = torch.stack((n, n), -1).to(DEV)[:, 0]
    qw = torch.zeros(2, sq, 8, 2 * d, dtype=BF16, device=DEV)
    qw[..., :d] = q.to(DEV)
    for views in (flat, [w[..., :d] for w in wide]):
        k, v = (x.view(E4M3).transpose(2, 3) for x in views)
        got = kc.attention(qw[..., :d].transpose(1, 2), kc.PagedKVCache(k, v, *scales).layer(1), t2, n2)
        assert torch.equal(got, want)
    # an odd start address and an odd row length take no vector loads
    qo = torch.zeros(2 * sq * 8 * (d + 1) + 1, dtype=BF16, device=DEV)[1:].view(2, sq, 8, d + 1)
    qo[..., :d] = q.to(DEV)
    got = kc.attention(qo[..., :d].transpose(1, 2), base.layer(1), table.to(DEV), n.to(DEV))
    _check_attention(got, q.transpose(1, 2), base, 1, table, n, 1 / math.sqrt(d), True)


def test_attention_offsets_past_32_bits():
    """Pages whose byte offset passes 2^31."""
    pages, page, hkv, d = 70000, 32, 8, 128
    k, v = (torch.zeros((1, pages, hkv, page, d), dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((1, pages, hkv), 2.0**-6, device=DEV) for _ in range(2))
    ids = [69999, 2, 65536, 66001]
    for t in (k, v):
        t[0, ids] = torch.randint(-127, 128, (4, hkv, page, d), dtype=torch.int8).to(DEV)
    table = torch.tensor([ids[:3], [ids[3], -1, -1]], dtype=torch.int32)
    small = torch.tensor([[0, 1, 2], [3, -1, -1]], dtype=torch.int32)
    n = torch.tensor([90, 7], dtype=torch.int32)
    cache = kc.PagedKVCache(k, v, ks, vs)
    sub = kc.PagedKVCache(k[:, ids].contiguous(), v[:, ids].contiguous(), ks[:, ids].contiguous(), vs[:, ids].contiguous())
    for sq in (1, 40):
        q = torch.randn(2, 16, sq, d).to(BF16)
        got = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV))
        _check_attention(got, q, sub, 0, small, n, 1 / math.sqrt(d), True)
    new = torch.randn(2, hkv, 3, d, device=DEV).to(BF16)
    start = n.to(DEV)
    kc.store(cache.layer(0), new, new, table.to(DEV), start)
    kc.store(sub.layer(0), new, new, small.to(DEV), start)
    assert torch.equal(k[:, ids], sub.key) and torch.equal(v[:, ids], sub.value)
    one = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)  # noqa: E731
    kc.copy_pages(cache, one(69999), one(69998))
    assert torch.equal(k[:, 69998], k[:, 69999])


def test_attention_many_rows():
    """More batch rows than one launch takes, and a table far wider than the lengths."""
    b, page = 4100, 16
    cache = _random_cache(1, 50, 1, page, 64, E4M3)
    table = torch.randint(0, 50, (b, 700), dtype=torch.int32)
    n = torch.randint(0, 60, (b,), dtype=torch.int32)
    q = torch.randn(b, 2, 1, 64).to(BF16)
    got = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV))
    pick = torch.tensor([0, 1, 2, 77, 2047, 2048, 4094, 4095, 4096, 4097, 4099])
    _check_attention(got[pick.to(DEV)], q[pick], cache, 0, table[pick], n[pick], 0.125, True)


@pytest.mark.parametrize("sq", [1, 24])
def test_attention_long_uneven_rows(sq):
    """One long row among short ones: segments are cut and joined."""
    lengths = [5000, 1, 0, 33, 2047]
    page, hkv, d = 64, 2, 128
    pages = sum(-(-x // page) for x in lengths)
    cache = _random_cache(1, pages, hkv, page, d, I8)
    table = _table(lengths, page, pages)
    n = torch.tensor(lengths, dtype=torch.int32)
    q = torch.randn(5, 4, sq, d).to(F16)
    got = kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV))
    _check_attention(got, q, cache, 0, table, n, 1 / math.sqrt(d), True)
    assert torch.equal(got, kc.attention(q.to(DEV), cache.layer(0), table.to(DEV), n.to(DEV)))


def test_no_wait_gave_up():
    """The kernels' bounded waits (the copy ring, the tensor-core pipeline) end in time: a device error
    word would say otherwise."""
    from ntops_b200 import _lib

    cache = _random_cache(1, 130, 2, 64, 128, E4M3)
    table = _table([4000, 4100], 64, 130)
    n = torch.tensor([4000, 4100], dtype=torch.int32, device=DEV)
    for sq in (1, 8, 40, 300):
        q = torch.randn(2, 8, sq, 128, device=DEV).to(BF16)
        first = kc.attention(q, cache.layer(0), table.to(DEV), n)
        for _ in range(20):
            assert torch.equal(kc.attention(q, cache.layer(0), table.to(DEV), n), first)
    assert _lib.load().ntb_check_device_error(None) == 0


def test_attention_of_nothing():
    cache = _random_cache(1, 4, 2, 16, 64, E4M3)
    n = torch.zeros(0, dtype=torch.int32, device=DEV)
    t = torch.zeros((0, 3), dtype=torch.int32, device=DEV)
    assert kc.attention(torch.zeros(0, 4, 1, 64, dtype=BF16, device=DEV), cache.layer(0), t, n).shape == (0, 4, 1, 64)
    n, t = torch.tensor([5], dtype=torch.int32, device=DEV), torch.zeros((1, 3), dtype=torch.int32, device=DEV)
    assert kc.attention(torch.zeros(1, 4, 0, 64, dtype=BF16, device=DEV), cache.layer(0), t, n).numel() == 0
    got = kc.attention(torch.ones(1, 4, 1, 64, dtype=BF16, device=DEV), cache.layer(0), t[:, :0], n)
    assert (got == 0).all()


# --------------------------------------------------------------------------------- store ----
STORE = [
    # b, s, start, heads, d, page, code, dtype
    (1, 1, [0], 1, 128, 16, E4M3, BF16),
    (3, 1, [15, 16, 17], 2, 128, 16, E4M3, F16),
    (2, 40, [5, 0], 2, 64, 16, I8, BF16),
    (2, 200, [1, 63], 1, 128, 64, E4M3, BF16),
    (2, 300, [130, 7], 2, 128, 128, I8, F32),
    (1, 33, [3], 3, 96, 32, E4M3, F32),
    (2, 20, [2, 9], 2, 33, 5, I8, F16),
    (1, 300, [10], 1, 256, 256, E4M3, BF16),
]


def _store_both(cache, key, value, table, start, counts=None):
    ks, vs = cache.key_scale[1].cpu().double(), cache.value_scale[1].cpu().double()
    kv, vv = _values(cache.key[1]), _values(cache.value[1])
    other = [t[0].clone().view(torch.uint8) for t in (cache.key, cache.value)]
    kc.store(cache.layer(1), key, value, table.to(DEV), start.to(DEV), None if counts is None else counts.to(DEV))
    for codes, scales, new in ((kv, ks, key), (vv, vs, value)):
        OK.store(codes, scales, new.cpu(), table, start, counts, cache.key.dtype)
    assert torch.equal(cache.key_scale[1].cpu().double(), ks)
    assert torch.equal(cache.value_scale[1].cpu().double(), vs)
    for got, want in ((cache.key[1], kv), (cache.value[1], vv)):
        torch.testing.assert_close(_values(got), want, rtol=0, atol=0, equal_nan=True)
    for t, was in zip((cache.key, cache.value), other):
        assert torch.equal(t[0].view(torch.uint8), was)  # the other layer


@pytest.mark.parametrize("b,s,start,heads,d,page,code,dtype", STORE)
def test_store(b, s, start, heads, d, page, code, dtype):
    ends = [x + s for x in start]
    pages = sum(-(-x // page) for x in ends) + 2
    cache = _random_cache(2, pages, heads, page, d, code, -8, -5)
    table = _table(ends, page, pages, extra=1)
    # token sizes spread over 2^8, so some pages' scales grow and some do not
    size = torch.exp2(torch.randint(-4, 4, (b, s, 1, 1)).float())
    key, value = ((torch.randn(b, s, heads, d) * size).to(dtype).transpose(1, 2).to(DEV) for _ in range(2))
    start = torch.tensor(start, dtype=torch.int32)
    _store_both(cache, key, value, table, start)
    # storing the same tokens again changes nothing
    was = [t.clone() for t in (cache.key.view(torch.uint8), cache.value.view(torch.uint8), cache.key_scale)]
    kc.store(cache.layer(1), key, value, table.to(DEV), start.to(DEV))
    assert torch.equal(was[0], cache.key.view(torch.uint8)) and torch.equal(was[1], cache.value.view(torch.uint8))
    assert torch.equal(was[2], cache.key_scale)


@pytest.mark.parametrize("code", [E4M3, I8])
def test_store_token_by_token(code):
    """A page filled one token at a time, each larger than the last, then smaller ones."""
    cache = _random_cache(2, 3, 2, 16, 64, code)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    for i in range(20):
        size = 2.0 ** (i if i < 10 else 20 - i)
        k, v = ((torch.randn(1, 2, 1, 64) * size).to(BF16).to(DEV) for _ in range(2))
        _store_both(cache, k, v, table, torch.tensor([i], dtype=torch.int32))


@pytest.mark.parametrize("code", [E4M3, I8])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_store_special_values(code, dtype):
    """Zeros, infinities, NaN, subnormals, the largest values, exact powers of two and ties."""
    cache = _random_cache(2, 12, 1, 16, 64, code)
    x = torch.zeros(10, 1, 16, 64)
    x[1, 0, 3, 5], x[1, 0, 3, 6] = float("inf"), 2.0
    x[2, 0, 3, 5], x[2, 0, 4, 6] = float("nan"), -3.0
    x[3] = 1e-39
    x[4, 0, 0, 0] = torch.finfo(BF16).max
    x[5] = torch.arange(1024).view(1, 16, 64) / 2.0
    x[6, 0, 0] = 448.0
    x[7, 0, 0] = 127.0 * 2.0**-20
    x[8, 0, 0, :3] = torch.tensor([449.0, 127.5, float("-inf")])
    x[9] = torch.linspace(-1.0, 1.0, 1024).view(1, 16, 64) * 2.0**-60
    x = x.to(dtype)
    table = torch.arange(10, dtype=torch.int32).view(10, 1)
    start = torch.zeros(10, dtype=torch.int32)
    _store_both(cache, x.to(DEV), x.flip(0).contiguous().to(DEV), table, start)


def test_store_drops_what_has_no_place():
    """Holes, ids out of range, tokens past the table, counts and padding rows."""
    cache = _random_cache(2, 9, 2, 16, 64, E4M3)
    table = torch.tensor([[0, -1, 1], [2, 77, 3], [4, 5, 6], [7, 8, -5]], dtype=torch.int32)
    start = torch.tensor([10, 0, 40, -1], dtype=torch.int32)
    counts = torch.tensor([30, 48, 30, 30], dtype=torch.int32)
    key, value = (torch.randn(4, 2, 40, 64, device=DEV).to(F16) for _ in range(2))
    _store_both(cache, key, value, table, start)
    _store_both(cache, value, key, table, start, torch.tensor([3, 0, -2, 9], dtype=torch.int32))
    _store_both(cache, key, value, table, start, counts)


def test_store_layouts():
    """Odd input strides (no vector loads) and token-major pages give the same codes."""
    pages, page, h, d = 8, 16, 2, 64
    a = _random_cache(1, pages, h, page, d, E4M3)
    b = kc.PagedKVCache(*(t.view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3).view(E4M3)
                          for t in (a.key, a.value)), a.key_scale.clone(), a.value_scale.clone())
    x = torch.randn(2, 30, h, d, device=DEV).to(BF16)
    odd = torch.zeros(2 * 30 * h * (d + 1) + 1, dtype=BF16, device=DEV)[1:].view(2, 30, h, d + 1)
    odd[..., :d] = x
    inner = torch.stack((x, x), -1)[..., 0]
    table = torch.tensor([[3, 1, 0, 5], [2, 4, 6, 7]], dtype=torch.int32, device=DEV)
    start = torch.tensor([[9, 0], [20, 0]], dtype=torch.int32, device=DEV)[:, 0]
    kc.store(a.layer(0), x.transpose(1, 2), x.transpose(1, 2), table, start)
    kc.store(b.layer(0), odd[..., :d].transpose(1, 2), inner.transpose(1, 2), table, start)
    assert torch.equal(a.key.view(torch.uint8), b.key.view(torch.uint8))
    assert torch.equal(a.value.view(torch.uint8), b.value.view(torch.uint8))
    assert torch.equal(a.key_scale, b.key_scale) and torch.equal(a.value_scale, b.value_scale)


def test_store_then_attend_on_another_stream():
    """Calls follow the current stream: a chain of steps on a side stream gives the same result."""
    def steps():
        cache = kc.PagedKVCache.allocate(1, 20, 2, 16, 64, I8)
        table = torch.arange(20, dtype=torch.int32, device=DEV).view(2, 10)
        outs = []
        for i in range(0, 120, 40):
            g = torch.Generator(device=DEV).manual_seed(i)
            x = torch.randn(3, 2, 40, 2, 64, generator=g, device=DEV).to(BF16)
            start = torch.full((2,), i, dtype=torch.int32, device=DEV)
            kc.store(cache.layer(0), x[0].transpose(1, 2), x[1].transpose(1, 2), table, start)
            outs.append(kc.attention(x[2][:, -3:].transpose(1, 2), cache.layer(0), table, start + 40))
        return torch.stack(outs)

    want = steps()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = steps()
    s.synchronize()
    assert torch.equal(got, want)


# --------------------------------------------------------------------------------- pages ----
def _page_views(cache):
    return [t.clone() for t in (cache.key.view(torch.uint8), cache.value.view(torch.uint8), cache.key_scale,
                                cache.value_scale)]


def _assert_copied(cache, was, moves):
    now = _page_views(cache)
    for w in was:
        for src, dst in moves:
            w[:, dst] = w[:, src]
    for w, x in zip(was, now):
        assert torch.equal(w, x)


@pytest.mark.parametrize("layers,h,page,d,major", [(1, 1, 16, 64, "head"), (3, 8, 16, 128, "token"), (2, 3, 5, 33, "head"),
                                                   (2, 2, 16, 64, "wide")])
def test_copy_pages(layers, h, page, d, major):
    base = _random_cache(layers, 12, h, page, d, I8)
    if major == "head":
        cache = base
    elif major == "token":
        k, v = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (base.key, base.value))
        cache = kc.PagedKVCache(k, v, base.key_scale, base.value_scale)
    else:
        k, v = (torch.zeros(layers, 12, h, page, d + 7, dtype=I8, device=DEV)[..., :d] for _ in range(2))
        k.copy_(base.key), v.copy_(base.value)
        cache = kc.PagedKVCache(k, v, base.key_scale, base.value_scale)
    was = _page_views(cache)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    kc.copy_pages(cache, i32([3, 0, 3, -1, 5, 2]), i32([7, 11, 1, 4, 12, 2]))
    _assert_copied(cache, was, [(3, 7), (0, 11), (3, 1)])
    kc.copy_pages(cache, i32([]), i32([]))
    _assert_copied(cache, _page_views(cache), [])


def _pool(rows, page, pages, extra=1):
    """Block table, refs with a page pinned by the caller."""
    table = _table(rows, page, pages - 2, extra)
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in table.reshape(-1).tolist():
        if p >= 0:
            refs[p] += 1
    refs[pages - 1] = 1
    return table, refs


@pytest.mark.parametrize("lengths,parents,pages", [
    ([20], [0, 0, 0], 8),
    ([5, 48, 33, 0], [1, 1, 2, 2, 3, 0], 20),
    ([40, 41, 42, 43], [3, 3, 1, 1], 20),
    ([17, 18], [1, 0], 6),
    ([17, 18], [], 6),
    ([30, 31], [0, 7, -1, 1, 1], 9),
    ([16, 32], [0, 0, 1, 1, 1], 6),
    ([20, 21, 22], [0, 0, 1, 1, 2, 2, 2], 9),  # too few free pages
    ([100] * 40, [i // 2 for i in range(80)], 400),
])
def test_reorder(lengths, parents, pages):
    page = 16
    cache = _random_cache(2, pages, 2, page, 64, E4M3)
    table, refs = _pool(lengths, page, pages)
    if len(lengths) > 2:  # the first pages of two rows are one shared page
        if lengths[0] >= page and lengths[1] >= page:
            refs[table[1, 0]] -= 1
            table[1, 0] = table[0, 0]
            refs[table[0, 0]] += 1
    n, par = torch.tensor(lengths, dtype=torch.int32), torch.tensor(parents, dtype=torch.int32)
    was = _page_views(cache)
    got = kc.reorder(cache, table.to(DEV), n.to(DEV), refs.to(DEV), par.to(DEV))
    want = OK.reorder(table, n, refs, par, page)
    for g, w in zip(got[:3], want[:3]):
        assert g.dtype == torch.int32 and torch.equal(g.cpu(), w)
    assert got[3].tolist() == [want[3]]
    _assert_copied(cache, was, want[4])


@pytest.mark.parametrize("lengths,grown,pages", [
    ([0], [1], 3),
    ([5, 16, 33], [6, 17, 90], 20),
    ([0, 0, 10], [100, 40, 11], 9),       # too few free pages
    ([64, 1], [64, 1], 9),
    ([3] * 300, [40] * 300, 1500),
    ([3] * 50, [40] * 50, 5000),
])
def test_extend(lengths, grown, pages):
    page = 16
    cache = _random_cache(1, pages, 1, page, 64, I8)
    table, refs = _pool(lengths, page, pages, extra=max(grown) // page + 1)
    n = torch.tensor(grown, dtype=torch.int32)
    got = kc.extend(cache, table.to(DEV), refs.to(DEV), n.to(DEV))
    want = OK.extend(table, n, refs, page)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert got[2].tolist() == [want[2]]


@pytest.mark.parametrize("lengths,pages", [([40, 3], 9), ([0, 0], 5), ([16] * 100, 103), ([50] * 60, 3000), ([10], 2100)])
def test_compact(lengths, pages):
    page = 16
    cache = _random_cache(2, pages, 2, page, 32, E4M3)
    table, refs = _pool(lengths, page, pages)
    was = _page_views(cache)
    got = kc.compact(cache, table.to(DEV), refs.to(DEV))
    want = OK.compact(table, refs)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert got[2].tolist() == [want[2]]
    _assert_copied(cache, was, want[3])


def test_attention_survives_reorder_and_compact():
    """The tokens a row attends to are the same before and after its pages move."""
    lengths, page, pages = [70, 33, 5], 16, 16
    cache = _random_cache(1, pages, 2, page, 64, E4M3)
    table, refs = _pool(lengths, page, pages)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = torch.randn(3, 4, 1, 64, device=DEV).to(BF16)
    want = kc.attention(q, cache.layer(0), table.to(DEV), n)
    par = torch.tensor([2, 0, 0, 1], dtype=torch.int32, device=DEV)
    t, n2, refs2, missing = kc.reorder(cache, table.to(DEV), n, refs.to(DEV), par)
    assert missing.tolist() == [0]
    t, refs2, used = kc.compact(cache, t, refs2)
    assert int(t.max()) < used.item()
    got = kc.attention(q[par.long()], cache.layer(0), t, n2)
    assert torch.equal(got, want[par.long()])


# ------------------------------------------------------------------------------ refusals ----
def _operands():
    cache = _random_cache(1, 6, 2, 16, 64, E4M3)
    return dict(cache=cache, layer=cache.layer(0), q=torch.zeros(2, 4, 1, 64, dtype=BF16, device=DEV),
                new=torch.zeros(2, 2, 3, 64, dtype=BF16, device=DEV),
                table=torch.zeros(2, 3, dtype=torch.int32, device=DEV), n=torch.ones(2, dtype=torch.int32, device=DEV),
                refs=torch.zeros(6, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("change,match", [
    (dict(q=lambda o: o["q"].double()), "query must be one of"),
    (dict(q=lambda o: o["q"][:, :3]), "multiple"),
    (dict(q=lambda o: o["q"][..., :32]), "head_dim"),
    (dict(q=lambda o: o["q"][0]), "4-D"),
    (dict(q=lambda o: o["q"].cpu()), "CUDA"),
    (dict(q=lambda o: o["q"].transpose(1, 3).contiguous().transpose(1, 3)), "inner stride"),
    (dict(table=lambda o: o["table"].long()), "block_table must be one of"),
    (dict(table=lambda o: o["table"][:1]), "batch"),
    (dict(n=lambda o: o["n"][:1]), "batch"),
    (dict(n=lambda o: o["n"].float()), "lengths must be one of"),
])
def test_attention_refusals(change, match):
    o = _operands()
    o.update({k: f(o) for k, f in change.items()})
    with pytest.raises(RuntimeError, match=match):
        kc.attention(o["q"], o["layer"], o["table"], o["n"])


@pytest.mark.parametrize("change,match", [
    (dict(new=lambda o: o["new"][:, :1]), "heads"),
    (dict(new=lambda o: o["new"][..., :8]), "head_dim"),
    (dict(new=lambda o: o["new"].int()), "key must be one of"),
    (dict(table=lambda o: o["table"][:1]), "batch"),
    (dict(n=lambda o: o["n"][:1]), "batch"),
])
def test_store_refusals(change, match):
    o = _operands()
    o.update({k: f(o) for k, f in change.items()})
    with pytest.raises(RuntimeError, match=match):
        kc.store(o["layer"], o["new"], o["new"], o["table"], o["n"])


def test_other_refusals():
    o = _operands()
    with pytest.raises(RuntimeError, match="shape"):
        kc.store(o["layer"], o["new"], o["new"][:, :, :2], o["table"], o["n"])
    with pytest.raises(RuntimeError, match="dtype"):
        kc.store(o["layer"], o["new"], o["new"].float(), o["table"], o["n"])
    with pytest.raises(TypeError, match="layer"):
        kc.attention(o["q"], o["cache"], o["table"], o["n"])
    with pytest.raises(RuntimeError, match="refs has 5"):
        kc.compact(o["cache"], o["table"], o["refs"][:5])
    with pytest.raises(RuntimeError, match="differ"):
        kc.copy_pages(o["cache"], o["n"], o["n"][:1])
    with pytest.raises(RuntimeError, match="batch"):
        kc.reorder(o["cache"], o["table"], o["n"][:1], o["refs"], o["n"])
    c = o["cache"]
    with pytest.raises(RuntimeError, match="float8_e4m3fn or int8"):
        kc.PagedKVCache(c.key, c.value.view(torch.int8), c.key_scale, c.value_scale)
    with pytest.raises(RuntimeError, match="float32"):
        kc.PagedKVCache(c.key, c.value, c.key_scale.half(), c.value_scale)
    with pytest.raises(RuntimeError, match="layers, pages, kv_heads"):
        kc.PagedKVCache(c.key, c.value, c.key_scale[:, :3], c.value_scale)
    wide = torch.zeros(1, 6, 2, 16, 300, dtype=torch.int8, device=DEV)
    big = kc.PagedKVCache(wide, wide.clone(), c.key_scale, c.value_scale)
    with pytest.raises(RuntimeError, match="above 256"):
        kc.attention(torch.zeros(2, 4, 1, 300, dtype=BF16, device=DEV), big.layer(0), o["table"], o["n"])

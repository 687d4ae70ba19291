"""Attention over 8-bit pages whose exponents are far apart, keys and queries of zeros, and what a row sees of others' tokens,
against the definition in 64 bits.

Tolerances are those of the attention's other tests, except that what is small is measured by what the row itself sees: with
u = 2^-11 (probabilities in fp16), r the output's half step, w the softmax, A = sum_j w_j |v_j|, T = max_j w_j max_d |v_jd|:
  r |o| + smallest subnormal / 2     the output's rounding
  u A                                the rounding of every p_j
  2 d A                              scores off by d = (hd + 8) 2^-24 max_j sum_i |q_i k_ij| scale, and 2^-16 for the addition of an
                                     exponent (|z + e| 2^-24 with |e| < 2^7 and |z| < 2^7 where p_j counts); keys without weight
                                     (below 2^-200) stay without it, and a lone key has a probability of one whatever its score
  (n / 16 + 64) 2^-23 A              fp32 sums of n keys
  n 2^-20 T                          probabilities below fp16's normal range: off by 2^-34 of the largest at most, times a value that is at
                                     most 2^14 times that of the largest (2^12 of exponents and 2^2 of codes, where exponents are
                                     left to the values; elsewhere they are part of the probabilities)
"""
import math

import pytest
import torch

from oracle import paged_oracle as O
from test_gpu_paged import _cache, _host, _pages, _table

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
FORMS = [(torch.float16, E4M3), (torch.bfloat16, E4M3), (torch.float16, torch.int8), (torch.bfloat16, torch.int8)]
IDS = ["f16-e4m3", "bf16-e4m3", "f16-i8", "bf16-i8"]


def _check(host, table, q, p, out, window=0, sinks=0):
    """Rows q [n, heads, hd] of one sequence, at positions p .., against ``out``."""
    n, heads, hd = q.shape
    scale = 1.0 / math.sqrt(hd)
    keys, there = O.positions(host[0], host[2], table, p + n, False)
    values, _ = O.positions(host[1], host[3], table, p + n, True)
    i, j = p + torch.arange(n)[:, None], torch.arange(p + n)[None]
    see = (j <= i) & there
    if window:
        see &= (j > i - window) | (j < sinks)
    keys[~see.any(0)] = values[~see.any(0)] = 0.0
    group = heads // keys.shape[1]
    k, v = (x.repeat_interleave(group, 1).transpose(0, 1) for x in (keys, values))   # [heads, positions, hd]
    x = q.double().transpose(0, 1)
    z = (x @ k.mT * scale).masked_fill(~see, -math.inf)
    w = torch.nan_to_num(torch.softmax(z, -1))
    want, weight, most = w @ v, w @ v.abs(), (w * v.abs().amax(-1).unsqueeze(1)).amax(-1, keepdim=True)
    counts = w > 2.0 ** -200
    size = (x.abs() @ k.abs().mT * scale * counts).amax(-1, keepdim=True) * (counts.sum(-1, keepdim=True) > 1)
    d = (hd + 8) * 2.0 ** -24 * size + 2.0 ** -16
    f = torch.finfo(q.dtype)
    tol = f.eps / 2 * (want.abs() + f.smallest_normal) + (2.0 ** -11 + 2 * d + ((p + n) / 16 + 64) * 2.0 ** -23) * weight \
        + (p + n) * 2.0 ** -20 * most
    off = (out.double().transpose(0, 1) - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[0].tolist(), float((off / tol).nan_to_num(math.inf).max()))


def _stored(form, dtype, k, v, page=16):
    """A cache with one sequence's keys and values [positions, kv_heads, hd], and its table."""
    n, kvh, hd = k.shape
    blocks = -(-n // page)
    cache = _cache(_pages(form, blocks + 1, kvh, page, hd, 3))
    table = _table(1, [blocks], blocks + 1, 4)
    cache.append(cache.batch([n], [0], table.to(DEV)), k.to(dtype).to(DEV), v.to(dtype).to(DEV))
    return cache, table


def _attend(cache, table, q, p, **kw):
    return cache.attend(cache.batch([len(q)], [p], table.to(DEV)), q.to(DEV), **kw).cpu()


@pytest.mark.parametrize("new", [1, 5, 70, 150])
@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_queries_and_keys_of_zeros(dtype, form, new):
    """A row that likes no key better than another has the mean of the values it sees."""
    g = torch.Generator().manual_seed(1)
    p = 37
    cache, table = _stored(form, dtype, torch.zeros(p + new, 1, 64), torch.randn(p + new, 1, 64, generator=g))
    host = _host(cache)
    assert bool((host[2].view(-1) == -126).any())
    q = torch.randn(new, 2, 64, generator=g)
    for size in (0.0, 2.0 ** -20, 2.0 ** -24) + ((2.0 ** -60, 2.0 ** -100) if dtype == torch.bfloat16 else ()):
        rows = (q * size).to(dtype)
        _check(host, table[0], rows, p, _attend(cache, table, rows, p))


@pytest.mark.parametrize("new", [3, 150])
@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_rows_whose_first_pages_are_nowhere(dtype, form, new):
    g = torch.Generator().manual_seed(2)
    cache, table = _stored(form, dtype, torch.randn(250, 1, 64, generator=g), torch.randn(250, 1, 64, generator=g))
    table[0, :6] = -1
    p = 92
    for size in (0.0, 2.0 ** -24, 1.0):
        q = (torch.randn(new, 2, 64, generator=g) * size).to(dtype)
        out = _attend(cache, table, q, p)
        assert bool((out[:min(new, 4)] == 0).all())
        _check(_host(cache), table[0], q, p, out)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("new,p", [(1, 60), (5, 60), (40, 60), (150, 60), (2, 3000), (130, 3000)])
@pytest.mark.parametrize("dtype,form", [(torch.float16,) * 2, (torch.bfloat16,) * 2] + FORMS, ids=["f16", "bf16"] + IDS)
def test_scores_of_any_size(dtype, form, new, p, sign):
    """Products up to the largest that two numbers of the type have, every one of them exact: the row has the mean of the
    values whose score is the largest, positive or negative."""
    n, hd = p + new, 64
    k = torch.zeros(n, 1, hd)
    at = torch.arange(n)
    k[at, 0, at % 4] = (1.0 if sign < 0 else 1.0 - 2.0 * (at // 4 % 2).float()) * 2.0 ** (15 if dtype == torch.float16 else 60)
    v = torch.randn(n, 1, hd, generator=torch.Generator().manual_seed(9))
    q = torch.zeros(new, 2, hd)
    q[:, :, :4] = sign * torch.tensor([1.0, 2.0, 3.0, 5.0]) * 2.0 ** (13 if dtype == torch.float16 else 40)
    best = k[:, 0, 3] > 0 if sign > 0 else k[:, 0, 0] > 0
    if form == dtype:
        cache, table = _cache(_pages(form, -(-n // 16), 1, 16, hd, 3)), torch.arange(-(-n // 16), dtype=torch.int32)[None]
        cache.append(cache.batch([n], [0], table.to(DEV)), k.to(dtype).to(DEV), v.to(dtype).to(DEV))
    else:
        cache, table = _stored(form, dtype, k, v)
    out = _attend(cache, table, q.to(dtype), p).double()
    host = _host(cache)
    values, _ = O.positions(host[1], host[3], table[0], n, True)
    u = 2.0 ** -8 if form == torch.bfloat16 else 2.0 ** -11
    for i in range(new):
        seen = values[:p + i + 1][best[:p + i + 1], 0]
        want, weight = seen.mean(0), seen.abs().mean(0)
        tol = torch.finfo(dtype).eps / 2 * want.abs() + (u + (n / 16 + 64) * 2.0 ** -23) * weight
        assert bool(((out[i] - want).abs() <= tol).all()), i


def _with_infinities(dtype, form, new, p, sign, at, key, value):
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(p + new, 1, 64, generator=g) for _ in range(2))
    if key:
        k[at, 0, 7] = math.inf
    if value:
        v[at, 0, 9] = -math.inf
    q = torch.randn(new, 2, 64, generator=g)
    q[:, :, 7] = sign * 2.0 ** (-9 if dtype == torch.bfloat16 else -4)
    cache, table = _stored(form, dtype, k, v)
    q = q.to(dtype)
    _check(_host(cache), table[0], q, p, _attend(cache, table, q, p))


@pytest.mark.parametrize("where", ["last", "first"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("new", [1, 5, 40, 150])
@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_a_key_that_overflowed(dtype, form, new, sign, where):
    """It is held as the largest that codes can stand for, in few rows and in portions.  Queries that are small and positive in its place look at nothing
    else, negative ones not at it; rows in front of it do not see it."""
    _with_infinities(dtype, form, new, 60, sign, 60 + new - 1 if where == "last" else 33, True, False)


@pytest.mark.parametrize("where", ["last", "first"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("key", [False, True], ids=["seen", "weighed"])
@pytest.mark.parametrize("new", [1, 5, 40, 150])
@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_a_value_that_overflowed(dtype, form, new, key, sign, where):
    """With an ordinary key, and with one that gives it all the weight or none: where it has none, or is not seen, it takes
    nothing from the others."""
    _with_infinities(dtype, form, new, 60, sign, 60 + new - 1 if where == "last" else 33, key, True)


FEW = [(2, 64, 16, [1, 3], 90, 0, 0), (2, 64, 32, [20, 7], 31, 0, 0), (2, 80, 32, [5], 64, 0, 0), (4, 96, 64, [16], 130, 0, 0),
       (4, 128, 16, [10, 1], 200, 40, 5), (2, 192, 32, [3], 3, 0, 0), (2, 256, 64, [9], 50, 33, 0), (2, 128, 64, [1], 3000, 0, 0),
       (16, 64, 128, [2], 2500, 1500, 10)]
MANY = [(4, 64, 16, [150], 100, 0, 0), (2, 80, 32, [70], 31, 0, 0), (2, 96, 64, [129, 5], 64, 0, 0), (4, 128, 16, [100, 1], 200, 40, 5),
        (2, 192, 32, [90], 3, 0, 0), (2, 256, 64, [64, 2], 50, 33, 0), (2, 128, 64, [140], 3000, 0, 0),
        (2, 64, 128, [130], 2500, 1500, 10), (1, 128, 128, [300], 0, 0, 0)]


@pytest.mark.parametrize("case", FEW + MANY, ids=lambda c: "h%d-d%d-p%d-n%d-at%d-w%d" % (c[:3] + (c[3][0],) + c[4:6]))
@pytest.mark.parametrize("spread", [5, 10, 60])
@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_exponents_of_any_size(dtype, form, spread, case):
    """Exponents of neighbouring positions up to 2^120 apart: keys (with queries that bring the largest scores to a few units)
    and values, over tiles, splits, windows and heads that share keys."""
    heads, hd, page, new, p, window, sinks = case
    if dtype == torch.float16 and spread > 10:
        spread = 14       # (values and queries are within fp16's range)
    blocks = [-(-(p + n) // page) for n in new]
    host = _pages(form, sum(blocks), 1, page, hd, 6)
    g = torch.Generator().manual_seed(7)
    host[2] = torch.randint(-spread, spread + 1, host[2].shape, generator=g).to(torch.int8)
    host[3] = torch.randint(-spread, spread + 1, host[3].shape, generator=g).to(torch.int8) - 9
    if spread == 10:      # far apart in one place only
        host[2].clamp_(-5, 5)
        host[3].clamp_(-14, -4)
        host[3][:, 0, 11] = -30
    table = _table(len(new), blocks, sum(blocks), 8)
    cache = _cache(host)
    top = float(host[2].max())
    q = (torch.randn(sum(new), heads, hd, generator=g) * 2.0 ** (-top - 4)).to(dtype)
    out = cache.attend(cache.batch(new, [p] * len(new), table.to(DEV)), q.to(DEV), window=window, sinks=sinks).cpu()
    row = 0
    for s, n in enumerate(new):
        _check(host, table[s], q[row:row + n], p, out[row:row + n], window, sinks)
        row += n


@pytest.mark.parametrize("wide", [False, True], ids=["near", "far"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("new", [5, 40, 150])
def test_a_nan_code_reaches_the_rows_that_see_it(dtype, new, wide):
    """e4m3's NaN among values at a position that some rows of a tile see and others do not; then among keys."""
    p, page = 60, 16
    host = _pages(E4M3, 16, 1, page, 64, 17)
    if wide:
        host[3][:, 0, ::5] = -90
    table = _table(1, [14], 16, 18)
    q = torch.randn(new, 2, 64, generator=torch.Generator().manual_seed(19)).to(dtype)
    place = lambda j: (int(table[0, j // page]), 0, j % page)  # noqa: E731
    for j, d, code in ((p + 1, 5, 0x7f), (p + 4, 9, 0xff)):
        a, h, o = place(j)
        host[1].view(torch.uint8)[a, h, d, o] = code
    out = _attend(_cache(host), table, q, p).float()
    for i in range(new):
        assert bool(torch.isnan(out[i, :, 5]).all()) == (i >= 1), i
        assert bool(torch.isnan(out[i, :, 9]).all()) == (i >= 4), i
        rest = [d for d in range(64) if d not in (5, 9)]
        assert bool(torch.isfinite(out[i][:, rest]).all()), i
    host = _pages(E4M3, 16, 1, page, 64, 17)
    if wide:
        host[2][:, 0, ::5] = -90
    a, h, o = place(p + 3)
    host[0].view(torch.uint8)[a, h, o, 7] = 0x7f
    out = _attend(_cache(host), table, q, p)
    assert bool(torch.isnan(out[3:]).all()) and bool(torch.isfinite(out[:3]).all())

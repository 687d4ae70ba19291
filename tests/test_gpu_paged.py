"""The paged cache and its attention against oracle/paged_oracle.py (plain loops in 64 bits).

Tolerances.  Stored codes, exponents and values read back are exact: a scale is a power of two, so that the code is the one
rounding.  An output o = sum_j p_j v_j / sum_j p_j may be off by, with u the half step of the probabilities' format
(fp16 2^-11, bf16 2^-8; 8-bit pages use fp16), r that of the output and A = sum_j p_j |v_j| / sum_j p_j:
  r |o|                       the output's rounding
  u A                         the rounding of every p_j (their sum is not rounded)
  2 d A                       scores off by d (absolute): each p_j is off by a factor exp(+-d), their sum too;
                              d = (hd + 8) 2^-24 max_j sum_i |q_i k_ij| scale for the fp32 product, its scaling and
                              the subtraction of the maximum (at most 2 max_j |z_j| <= that sum, 3 roundings)
  (n / 16 + 64) 2^-23 A       fp32 sums of n keys by tiles, exp2 (2 ulp), waves and splits
  n 2^-24 max |v|             probabilities below the normal range: 2^-25 / 2^10 of the maximum in fp16, which is at
                              least 1 / 32 of the sum's reference: less than 2^-24
"""
import math

import pytest
import torch

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def _pages(dtype, pages, kvh, page, hd, seed, junk=False):
    """(k_pages, v_pages, k_exp, v_exp) on the CPU; junk: NaN and infinities, as unwritten memory may hold."""
    g = torch.Generator().manual_seed(seed)
    shapes = (pages, kvh, page, hd), (pages, kvh, hd, page)
    if dtype in (E4M3, torch.int8):
        kv = [torch.randint(0, 256, s, generator=g).to(torch.uint8).view(dtype) if junk else
              (torch.randn(s, generator=g) * O.TOP[dtype] / 4).clamp(-O.TOP[dtype], O.TOP[dtype]).round().to(dtype)
              for s in shapes]
        lo, hi = (-128, 128) if junk else ((-9, -6) if dtype == E4M3 else (-7, -4))
        return kv + [torch.randint(lo, hi, (pages, kvh, page), generator=g).to(torch.int8) for _ in range(2)]
    if junk:
        bits = [torch.randint(-2 ** 15, 2 ** 15, s, generator=g).to(torch.int16) for s in shapes]
        for b in bits:
            b.view(-1)[::3] = torch.tensor(float("nan"), dtype=dtype).view(torch.int16)
        return [b.view(dtype) for b in bits] + [None, None]
    return [torch.randn(s, generator=g).to(dtype) for s in shapes] + [None, None]


def _cache(t):
    from metaseq_amd import PagedCache

    return PagedCache(*(None if x is None else x.to(DEV) for x in t))


def _host(cache):
    return [None if t is None else t.cpu() for t in (cache.k_pages, cache.v_pages, cache.k_exp, cache.v_exp)]


def _table(seqs, blocks, pages, seed):
    g = torch.Generator().manual_seed(seed)
    need = sum(blocks)
    assert need <= pages
    order = torch.randperm(pages, generator=g)[:need].tolist()
    t = torch.full((seqs, max(max(blocks), 1)), -1, dtype=torch.int32)
    at = 0
    for i, b in enumerate(blocks):
        t[i, :b] = torch.tensor(order[at:at + b], dtype=torch.int32)
        at += b
    return t


def _bits(t):
    return t.contiguous().view(torch.uint8)


FORMS = [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float16, E4M3),
         (torch.bfloat16, E4M3), (torch.float16, torch.int8), (torch.bfloat16, torch.int8)]
IDS = ["f16", "bf16", "f16-e4m3", "bf16-e4m3", "f16-i8", "bf16-i8"]


def _stored(x, form):
    """(codes as the page holds them, exponents) of rows x."""
    if form in (torch.float16, torch.bfloat16):
        return x, None
    c, e = O.quantise(x, form)
    if form == E4M3:
        c = c.float().to(E4M3)
    return c.to(form) if form == torch.int8 else c, e.to(torch.int8)


@pytest.mark.parametrize("tokens", [1, 24], ids=["one", "many"])
@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_every_value_is_stored_as_defined(dtype, form, tokens):
    """All 65536 bit patterns of the dtype, in rows of like magnitudes and of mixed ones: infinities, NaN, subnormals and
    zeros among them; one token of many sequences, and many of few."""
    every = torch.arange(-2 ** 15, 2 ** 15).to(torch.int16)
    mixed = every[torch.randperm(2 ** 16, generator=torch.Generator().manual_seed(3))]
    zeros = torch.zeros(2048, dtype=torch.int16)
    x = torch.cat([every, mixed, zeros]).view(dtype).view(-1, 1, 64)
    seqs = -(-len(x) // tokens)
    new = [min(tokens, len(x) - i * tokens) for i in range(seqs)]
    blocks = [-(-(5 + n) // 16) for n in new]
    table = _table(seqs, blocks, sum(blocks), 1)
    cache = _cache(_pages(form, sum(blocks), 1, 16, 64, 2))
    batch = cache.batch(new, [5] * seqs, table.to(DEV))
    v = x.flip(0).contiguous()
    cache.append(batch, x.to(DEV), v.to(DEV))
    got = _host(cache)
    for rows, at, ex, transposed in ((x, 0, 2, False), (v, 1, 3, True)):
        want, e = _stored(rows, form)
        pages = _bits(got[at]).view(got[at].shape[:3] + (-1,)) if form != torch.float16 and form != torch.bfloat16 else got[at].view(torch.int16)
        pages = pages.transpose(2, 3) if transposed else pages
        seq = torch.repeat_interleave(torch.arange(seqs), torch.tensor(new))
        pos = 5 + torch.cat([torch.arange(n) for n in new])
        pg = table[seq, pos // 16].long()
        have = pages[pg, :, pos % 16]
        ref = want.view(torch.int16) if e is None else _bits(want).view(want.shape)
        if form == E4M3:  # one NaN is as good as another
            nan = (ref & 0x7f) == 0x7f
            assert torch.equal((have & 0x7f) == 0x7f, nan)
            assert torch.equal(have[~nan], ref[~nan])
        else:
            assert torch.equal(have, ref)
        if e is not None:
            assert torch.equal(got[ex][pg, :, pos % 16], e)


CASES = [
    # heads (kv), hd, page, new, positions
    (3, 64, 16, [1, 1, 1, 1], [0, 15, 16, 47]),
    (5, 80, 32, [1, 0, 7, 33], [31, 4, 30, 0]),
    (1, 96, 64, [64, 65, 1], [0, 63, 200]),
    (2, 128, 128, [130, 3], [127, 0]),
    (4, 192, 16, [17, 40], [3, 0]),
    (2, 256, 256, [1, 300, 9], [255, 1, 0]),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "h%d-d%d-p%d" % c[:3])
@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_positions_are_stored_read_and_left_alone(dtype, form, case):
    """Rows of a fused projection; nothing but their positions changes; sequences that sit out, entries that name no
    page, positions behind the table and rows behind the last sequence."""
    kvh, hd, page, new, pos = case
    seqs = len(new)
    blocks = [-(-(p + n) // page) for n, p in zip(new, pos)]
    table = _table(seqs, blocks, sum(blocks) + 2, 4)
    before = _pages(form, sum(blocks) + 2, kvh, page, hd, 5)
    cache = _cache(before)
    g = torch.Generator().manual_seed(6)
    rows = torch.randn(sum(new), (1 + 2 * kvh) * hd, generator=g) * torch.exp2(torch.randn(sum(new), 1, generator=g) * 4)
    rows = rows.to(dtype)
    k, v = (rows[:, a * hd:(a + kvh) * hd].unflatten(1, (kvh, hd)) for a in (1, 1 + kvh))
    gone = seqs - 1                       # sits the call out
    bad = next((i for i in range(seqs - 1) if new[i]), None)   # its last page is nowhere
    use, where = list(pos), table.clone()
    use[gone] = -1
    if bad is not None:
        where[bad, blocks[bad] - 1] = [-1, sum(blocks) + 2, 2 ** 31 - 1][seqs % 3]
    dev = rows.to(DEV)
    dk, dv = (dev[:, a * hd:(a + kvh) * hd].unflatten(1, (kvh, hd)) for a in (1, 1 + kvh))
    batch = cache.batch(new, torch.tensor(use, dtype=torch.int32, device=DEV), where.to(DEV))
    out = [torch.full((sum(new), kvh, hd), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    cache.append(batch, dk, dv)
    assert cache.read(batch, out=out) is out
    want = [None if t is None else t.clone() for t in before]
    raw = [t.view(torch.uint8) if t.dtype in (E4M3, torch.int8) else t for t in want[:2]]
    back = [torch.full((sum(new), kvh, hd), 7.0, dtype=torch.float64) for _ in range(2)]
    (kc, ke), (vc, ve) = _stored(k, form), _stored(v, form)
    r = 0
    for s in range(seqs):
        for i in range(new[s]):
            p = pos[s] + i
            if s != gone:
                at = int(where[s, p // page])
                there = 0 <= at < sum(blocks) + 2
                for x, c, e, j in ((k, kc, ke, 0), (v, vc, ve, 1)):
                    val = c[r].double() if e is None else c[r].double() * 2.0 ** e[r].double().unsqueeze(-1)
                    back[j][r] = val if there else 0.0
                    if there:
                        to = raw[j][at, :, p % page] if j == 0 else raw[j][at, :, :, p % page]
                        to.copy_(c[r].view(torch.uint8) if c.dtype in (E4M3, torch.int8) else c[r])
                        if e is not None:
                            want[2 + j][at, :, p % page] = e[r]
            r += 1
    for name, have, ref in zip(("k", "v", "k_exp", "v_exp"), _host(cache), want):
        assert have is None or torch.equal(_bits(have), _bits(ref)), name
    for have, ref in zip(out, back):
        assert torch.equal(have.cpu().double(), ref.to(dtype).double())


def test_a_batch_may_end_before_its_rows():
    """Rows behind the last sequence belong to none."""
    from metaseq_amd import _capi
    import ctypes

    cache = _cache(_pages(torch.float16, 4, 2, 16, 64, 7))
    table = _table(2, [1, 1], 4, 8).to(DEV)
    batch = cache.batch([2, 3], [0, 4], table)
    q, k, v = (torch.randn(9, 2, 64, device=DEV).half() for _ in range(3))
    before = _host(cache)
    c = _capi.PagedBatchC.from_buffer_copy(batch.c)
    c.M = 9
    batch.c, batch.rows, batch.by_ref = c, 9, ctypes.byref(c)
    cache.append(batch, k, v)
    changed = [(a != b).any(-1).any(1) for a, b in zip(_host(cache)[:1], before[:1])][0]
    assert int(changed.sum()) == 5
    out = torch.full_like(q, 3.0)
    cache.attend(batch, q, out=out)
    assert bool((out[5:] == 3.0).all()) and not bool((out[:5] == 3.0).any())
    got = cache.read(batch, out=(torch.full_like(q, 3.0), torch.full_like(q, 3.0)))
    assert torch.equal(got[0][:5], k[:5]) and torch.equal(got[1][:5], v[:5])
    assert bool((got[0][5:] == 3.0).all())


def _check_attention(cache, host, new, pos, table, q, out, window=0, sinks=0, scale=None, seqs=None):
    dtype, hd = q.dtype, q.shape[-1]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    u = 2.0 ** -8 if host[0].dtype == torch.bfloat16 else 2.0 ** -11
    r = torch.finfo(dtype).eps / 2
    row = 0
    for s, (n, p) in enumerate(zip(new, pos)):
        if n and p >= 0 and (seqs is None or s in seqs):
            keys, there = O.positions(host[0], host[2], table[s], p + n, False)
            values, _ = O.positions(host[1], host[3], table[s], p + n, True)
            keys[~there] = values[~there] = 0.0
            want, weight, size = O.attend(q[row:row + n], keys, values, there, p, scale, window, sinks)
            keyn = min(p + n, window + sinks + n) if window else p + n
            d = (hd + 8) * 2.0 ** -24 * size
            tol = r * want.abs() + (u + 2 * d + (keyn / 16 + 64) * 2.0 ** -23) * weight + keyn * 2.0 ** -24 * values.abs().max()
            off = (out[row:row + n].double() - want).abs()
            assert bool((off <= tol).all()), (s, n, p, float((off / tol.clamp(min=1e-30)).max()))
        row += n


ATTENTION = [
    # heads, kv heads, hd, page, new, positions, window, sinks
    (2, 2, 64, 16, [1, 1, 1, 1, 1], [0, 1, 15, 16, 333], 0, 0),
    (12, 12, 64, 64, [1, 1], [57, 700], 0, 0),
    (4, 1, 80, 32, [1, 2, 3], [31, 100, 0], 0, 0),
    (5, 5, 96, 128, [1, 4], [1000, 127], 0, 0),
    (8, 2, 128, 16, [1, 1, 2], [0, 511, 70], 0, 0),
    (16, 1, 128, 64, [1, 5], [90, 200], 0, 0),
    (32, 2, 64, 16, [3, 1], [40, 77], 0, 0),
    (6, 2, 192, 256, [1, 9], [300, 20], 0, 0),
    (4, 2, 256, 32, [1, 17], [70, 64], 0, 0),
    # windows: inside a tile, across tiles, of one, longer than everything; first positions in and out of it
    (2, 2, 64, 16, [1, 1, 1], [3, 100, 500], 7, 0),
    (4, 2, 128, 32, [1, 3, 2], [200, 333, 0], 64, 4),
    (2, 1, 64, 16, [1, 1, 40], [400, 20, 100], 33, 65),
    (4, 4, 80, 64, [2, 1], [150, 149], 1, 1),
    (2, 2, 128, 128, [1, 2], [90, 10], 5000, 3),
    # portions
    (2, 2, 64, 16, [130, 65, 1, 0, 17], [0, 33, 7, 5, 100], 0, 0),
    (4, 2, 128, 64, [200, 31], [77, 0], 0, 0),
    (3, 1, 96, 32, [100, 129], [0, 40], 50, 10),
    (2, 1, 256, 64, [70, 150], [100, 3], 0, 0),
    (3, 3, 192, 16, [90], [50], 20, 0),
    (2, 2, 80, 32, [128, 257], [0, 64], 0, 0),
    # rows on both sides of 32 and of 64, which different kernels take, in one batch
    (4, 2, 64, 16, [16, 17, 32, 33, 3], [0, 50, 7, 100, 20], 0, 0),
    (3, 1, 128, 32, [21, 22, 11, 10], [100, 0, 33, 200], 40, 5),
    (5, 5, 96, 64, [64, 65, 32, 33], [5, 0, 90, 2], 0, 0),
    (4, 4, 256, 128, [33, 48], [120, 300], 0, 0),
    # many blocks of eight heads behind as many keys
    (8, 8, 64, 64, [1030], [1100], 0, 0),
]


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "%d-%d-d%d-p%d-n%d-w%d-s%d" % (c[:4] + (max(c[4]),) + c[6:]))
@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_attention(dtype, form, case):
    """Everything that no row sees - unwritten rests of pages, other pages, positions behind the last one - holds NaN,
    infinities and exponents of any size."""
    heads, kvh, hd, page, new, pos, window, sinks = case
    seqs = len(new)
    blocks = [-(-(p + n) // page) for n, p in zip(new, pos)]
    pages = sum(blocks) + 2
    table = _table(seqs, blocks, pages, 11)
    good, host = _pages(form, pages, kvh, page, hd, 12), _pages(form, pages, kvh, page, hd, 13, junk=True)
    clean = [None if x is None else torch.zeros_like(x) for x in good]
    for s in range(seqs):
        for j in range(pos[s] + new[s]):
            at, o = int(table[s, j // page]), j % page
            if not new[s] or (window and j <= pos[s] - window and j >= sinks):
                continue
            for to in (host, clean):
                for i, (x, of) in enumerate(zip(to, good)):
                    if x is not None:
                        x, of = (y.view(torch.uint8) if y.dtype == E4M3 else y for y in (x, of))
                        where = (at, slice(None), slice(None), o) if i == 1 else (at, slice(None), o)
                        x[where] = of[where]
    cache = _cache(host)
    q = torch.randn(sum(new), heads, hd, generator=torch.Generator().manual_seed(14)).to(dtype)
    batch = cache.batch(new, pos, table.to(DEV))
    out = cache.attend(batch, q.to(DEV), window=window, sinks=sinks).cpu()
    _check_attention(cache, clean, new, pos, table, q, out, window, sinks)


@pytest.mark.parametrize("dtype,form", FORMS, ids=IDS)
def test_rows_without_a_key_are_zeros_and_missing_pages_are_not_seen(dtype, form):
    new, pos, page = [1, 3, 2, 1], [20, 30, 5, 3], 16
    table = torch.tensor([[0, -1, 2 ** 31 - 1], [-5, 3, 4], [7, 9, 9], [2, 5, 9]], dtype=torch.int32)
    host = _pages(form, 6, 2, page, 64, 15)
    cache = _cache(host)
    q = torch.randn(7, 4, 64, generator=torch.Generator().manual_seed(16)).to(dtype)
    out = cache.attend(cache.batch(new, pos, table.to(DEV)), q.to(DEV)).cpu()
    _check_attention(cache, host, new, pos, table, q, out)
    assert bool((out[4:6] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("new", [[5], [40], [150]], ids=str)
def test_what_is_not_finite_reaches_the_rows_that_see_it(dtype, new):
    """Values that are infinite or NaN at positions that some rows of a tile see and others do not; a key that is NaN."""
    host = _pages(dtype, 16, 1, 16, 64, 17)
    table = _table(1, [14], 16, 18)
    p = 60
    at = lambda j: (int(table[0, j // 16]), 0, slice(None), j % 16)  # noqa: E731
    host[1][at(p + 2)][3], host[1][at(p + 1)][5], host[1][at(p + 4)][9] = float("inf"), float("-inf"), float("nan")
    cache = _cache(host)
    q = torch.randn(new[0], 2, 64, generator=torch.Generator().manual_seed(19)).to(dtype)
    out = cache.attend(cache.batch(new, [p], table.to(DEV)), q.to(DEV)).cpu().float()
    for i in range(new[0]):
        assert bool((out[i, :, 3] == float("inf")).all()) == (i >= 2), i
        assert bool((out[i, :, 5] == float("-inf")).all()) == (i >= 1), i
        assert bool(torch.isnan(out[i, :, 9]).all()) == (i >= 4), i
        rest = [d for d in range(64) if d not in (3, 5, 9)]
        assert bool(torch.isfinite(out[i][:, rest]).all()), i
    host = _pages(dtype, 16, 1, 16, 64, 17)
    host[0][int(table[0, (p + 3) // 16]), 0, (p + 3) % 16, 7] = float("nan")
    cache = _cache(host)
    out = cache.attend(cache.batch(new, [p], table.to(DEV)), q.to(DEV)).cpu()
    assert bool(torch.isnan(out[3:]).all()) and bool(torch.isfinite(out[:3]).all())


@pytest.mark.parametrize("form", [torch.float16, E4M3, torch.int8], ids=["f16", "e4m3", "i8"])
@pytest.mark.parametrize("new,pos,window", [(1, 9000, 0), (3, 5000, 0), (1, 9000, 2500), (300, 2000, 0), (50, 4000, 0), (20, 3000, 1500)])
def test_long_histories(form, new, pos, window):
    """Keys split over workgroups; values and keys of very different sizes, zeros among them."""
    host = _pages(form, 160, 1, 64, 128, 20)
    g = torch.Generator().manual_seed(21)
    if form == torch.float16:
        for t in host[:2]:
            t *= torch.exp2(torch.randint(-8, 4, (160, 1, 1, 1), generator=g).float()).half()
    else:
        host[2] += torch.randint(-8, 4, (160, 1, 64), generator=g).to(torch.int8)
        host[3] += torch.randint(-8, 4, (160, 1, 64), generator=g).to(torch.int8)
        v, k = host[1].view(torch.uint8), host[0].view(torch.uint8)
        v[::7], k[::9] = 0, 0
        host[3][::7], host[2][::9] = -126, -126
    table = _table(1, [-(-(pos + new) // 64)], 160, 22)
    cache = _cache(host)
    q = torch.randn(new, 4, 128, generator=g).half()
    out = cache.attend(cache.batch([new], [pos], table.to(DEV)), q.to(DEV), window=window, sinks=4).cpu()
    if new > 100:  # a few rows, one by one
        keys, there = O.positions(host[0], host[2], table[0], pos + new, False)
        values, _ = O.positions(host[1], host[3], table[0], pos + new, True)
        for i in (0, 1, 150, 299):
            want, weight, size = O.attend(q[i:i + 1], keys[:pos + i + 1], values[:pos + i + 1], there, pos + i, 128 ** -0.5)
            d = 136 * 2.0 ** -24 * size
            tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2 * d + (pos / 16 + 64) * 2.0 ** -23) * weight + pos * 2.0 ** -24 * values.abs().max()
            assert bool(((out[i:i + 1].double() - want).abs() <= tol).all()), i
    else:
        _check_attention(cache, host, [new], [pos], table, q, out, window, 4)


def test_a_whole_run_of_steps_matches_one_attention_of_all():
    """Portions and single tokens stored and attended one after the other, in pages whose order is mixed, against the
    attention of the same tokens in one piece; with a window whose pages behind are nowhere any more.  The two differ by twice
    what one may be off (above, with 2^-13 for what is fp32); A is the attention over the values' magnitudes."""
    from metaseq_amd import PagedCache

    g = torch.Generator().manual_seed(30)
    n, heads, kvh, hd, page, window, sinks = 200, 4, 2, 128, 16, 40, 5
    qkv = torch.randn(n, (heads + 2 * kvh) * hd, generator=g).half().to(DEV)
    split = lambda x: (x[:, :heads * hd].unflatten(1, (heads, hd)), x[:, heads * hd:(heads + kvh) * hd].unflatten(1, (kvh, hd)),  # noqa: E731
                       x[:, (heads + kvh) * hd:].unflatten(1, (kvh, hd)))
    for form in (torch.float16, E4M3, torch.int8):
        whole, steps, sizes = (PagedCache.empty(20, kvh, hd, page=page, dtype=form) for _ in range(3))
        table = torch.randperm(20, generator=g)[:13].to(torch.int32).view(1, 13).to(DEV)
        q, k, v = split(qkv)
        b = whole.batch([n], [0], table)
        whole.append(b, k, v)
        sizes.append(b, k, v.abs())
        for w, s in ((0, 0), (window, sinks)):
            want, weight = (c.attend(b, q, window=w, sinks=s).double() for c in (whole, sizes))
            got, at = [], 0
            mine = table.clone()
            for m in (70, 1, 1, 30, 5, 64, 1, 28):
                pq, pk, pv = split(qkv[at:at + m])
                part = steps.batch([m], [at], mine)
                steps.append(part, pk, pv)
                got.append(steps.attend(part, pq, window=w, sinks=s))
                at += m
                if w:  # pages that neither the window nor the first positions reach any more
                    mine = mine.clone()
                    for j in range(1, 13):
                        if (j + 1) * page <= at - w:
                            mine[0, j] = -1
            assert at == n
            tol = 2 * (2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * 1.01 * weight)
            assert bool(((torch.cat(got).double() - want).abs() <= tol).all())


def test_captured_steps_follow_positions_and_tables():
    """append and attend in a graph, replayed while positions advance and a table changes, with eager work between the
    replays; two graphs at once."""
    from metaseq_amd import PagedCache

    g = torch.Generator().manual_seed(31)
    B, heads, kvh, hd, page = 3, 8, 2, 128, 16
    for form in (torch.bfloat16, E4M3):
        cache = PagedCache.empty(40, kvh, hd, page=page, dtype=form)
        table = torch.randperm(40, generator=g)[:36].to(torch.int32).view(3, 12).to(DEV)
        pos = torch.tensor([0, 17, 100], dtype=torch.int32, device=DEV)
        first = cache.batch([120] * 3, [0] * 3, table)
        fill = torch.randn(360, 2 * kvh, hd, generator=g).bfloat16().to(DEV)
        cache.append(first, fill[:, :kvh], fill[:, kvh:])
        rows = torch.zeros(B, heads + 2 * kvh, hd, dtype=torch.bfloat16, device=DEV)
        q, k, v = rows[:, :heads], rows[:, heads:heads + kvh], rows[:, heads + kvh:]
        batch = cache.batch([1] * B, pos, table)
        outs, graphs = [], []
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cache.append(batch, k, v)
            cache.attend(batch, q)
        torch.cuda.current_stream().wait_stream(side)
        for w in (0, 20):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                cache.append(batch, k, v)
                outs.append(cache.attend(batch, q, window=w, sinks=2))
            graphs.append(graph)
        for step in range(6):
            rows.copy_(torch.randn(rows.shape, generator=g).bfloat16())
            if step == 3:
                pos[1] = -1                      # one sequence sits out from here on
            for graph, out, w in zip(graphs, outs, (0, 20)):
                out.fill_(5.0)
                graph.replay()
                torch.cuda.synchronize()
                want = cache.attend(batch, q, window=w, sinks=2, out=torch.full_like(out, 5.0))
                assert torch.equal(out, want), (step, w)
                assert bool((out[1] == 5.0).all()) == (step >= 3)
            pos += torch.tensor([1, 1 if step < 3 else 0, 1], dtype=torch.int32, device=DEV)


def test_streams_strides_and_outputs_in_place():
    """On another stream than the default one; operands that need a copy; an output with rows apart."""
    cache = _cache(_pages(torch.float16, 8, 2, 32, 64, 40))
    table = _table(2, [3, 2], 8, 41).to(DEV)
    batch = cache.batch([2, 1], [70, 40], table)
    g = torch.Generator().manual_seed(42)
    q, k, v = (torch.randn(3, h, 64, generator=g).half().to(DEV) for h in (4, 2, 2))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache.append(batch, k, v)
        one = cache.attend(batch, q)
    side.synchronize()
    odd = torch.empty(3, 4, 65, dtype=torch.float16, device=DEV)[:, :, 1:]
    odd.copy_(q)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(3, 9 * 64, dtype=torch.float16, device=DEV)
    to = wide[:, 128:384].unflatten(1, (4, 64))
    assert torch.equal(cache.attend(batch, odd), one) and torch.equal(cache.attend(batch, swapped), one)
    assert cache.attend(batch, q, out=to) is to and torch.equal(to, one)
    assert bool((wide[:, :128] == 0).all()) and bool((wide[:, 384:] == 0).all())
    with pytest.raises(ValueError):
        cache.attend(batch, q, out=odd)


def test_pages_beyond_4_gb():
    """Offsets that pass 32 bits: the last pages of a pool of 5 GB of keys."""
    from metaseq_amd import PagedCache

    pages = 5 * 2 ** 30 // (256 * 8 * 128 * 2) + 1
    cache = PagedCache.empty(pages, 8, 128, page=256)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    g = torch.Generator().manual_seed(50)
    x = torch.randn(600, 24, 128, generator=g).half()
    b = cache.batch([600], [0], table.to(DEV))
    d = x.to(DEV)
    cache.append(b, d[:, 8:16], d[:, 16:])
    k, v = cache.read(b)
    assert torch.equal(k.cpu(), x[:, 8:16]) and torch.equal(v.cpu(), x[:, 16:])
    out = cache.attend(cache.batch([1], [599], table.to(DEV)), d[599:, :8]).cpu()
    want, weight, _ = O.attend(x[599:, :8], x[:, 8:16].double(), x[:, 16:].double(), torch.ones(600, dtype=torch.bool), 599, 128 ** -0.5)
    assert bool(((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * weight).all())


@pytest.mark.parametrize("rows", [1, 17, 70])
def test_packed_outputs(rows):
    """The activation layout of the packed products, through the C ABI."""
    import ctypes

    from metaseq_amd import _capi

    cache = _cache(_pages(torch.float16, 2 * rows, 2, 16, 64, 60))
    table = _table(rows, [2] * rows, 2 * rows, 61).to(DEV)
    batch = cache.batch([1] * rows, [(7 * i) % 32 for i in range(rows)], table)
    q = torch.randn(rows, 4, 64, generator=torch.Generator().manual_seed(62)).half().to(DEV)
    want = cache.attend(batch, q).view(rows, 256)
    mb = -(-rows // 16) if rows <= 64 else 8
    out = torch.zeros(mb * 16 * 256, dtype=torch.float16, device=DEV)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    a = _capi.PagedAttentionArgs(4, q.data_ptr(), 256, out.data_ptr(), 0, mb, 0, 0, 0.125, ws.data_ptr(), ws.numel())
    rc = cache._lib.msa_paged_attention(cache._of(torch.float16), batch.by_ref, ctypes.byref(a), _capi.stream_ptr())
    assert rc == 0, cache._lib.msa_last_error()
    got = out.view(8, mb, 4, 16, 8).permute(1, 3, 0, 2, 4).reshape(mb * 16, 256)
    assert torch.equal(got[:rows], want)


def test_batches_without_rows():
    cache = _cache(_pages(torch.float16, 2, 2, 16, 64, 70))
    before = _host(cache)
    for seqs in (0, 3):
        b = cache.batch([0] * seqs, [0] * seqs, torch.zeros(seqs, 1, dtype=torch.int32, device=DEV))
        e = torch.empty(0, 2, 64, dtype=torch.float16, device=DEV)
        cache.append(b, e, e)
        assert cache.attend(b, e).shape == (0, 2, 64) and cache.read(b)[0].shape == (0, 2, 64)
    assert torch.equal(_host(cache)[0], before[0]) and torch.equal(_host(cache)[1], before[1])


@pytest.mark.parametrize("new", [1, 60])
def test_windows_of_any_size(new):
    """From those that hold nothing but the row's own position to the largest number."""
    cache = _cache(_pages(torch.bfloat16, 40, 1, 16, 64, 71))
    table = _table(1, [40], 40, 72).to(DEV)
    b = cache.batch([new], [570], table)
    q = torch.randn(new, 2, 64, generator=torch.Generator().manual_seed(73)).bfloat16().to(DEV)
    want = cache.attend(b, q)
    for window in (570 + new, 640, 641, 2 ** 30, 2 ** 31 - 1):
        for sinks in (0, 2 ** 31 - 1):
            assert torch.equal(cache.attend(b, q, window=window, sinks=sinks), want), window
    own = cache.attend(b, q, window=1)
    v = cache.read(b)[1].expand(new, 2, 64) if new == 1 else cache.read(b)[1].expand(-1, 2, -1)
    assert torch.equal(own, v)
    assert torch.equal(cache.attend(b, q, window=1, sinks=2 ** 31 - 1), want)


@pytest.mark.parametrize("new", [[1, 2], [20, 70]], ids=str)
@pytest.mark.parametrize("form", [torch.float16, torch.int8], ids=["f16", "i8"])
def test_positions_behind_every_table(form, new):
    """Up to the largest that 32 bits hold: nothing is stored, zeros are read, and rows see what one at the table's last
    position sees."""
    before = _pages(form, 4, 2, 16, 64, 40)
    cache = _cache(before)
    table = torch.arange(4, dtype=torch.int32).view(2, 2)
    pos = torch.tensor([2 ** 31 - 1 - new[0], 2 ** 31 - 1 - new[1] // 2], dtype=torch.int32)
    batch = cache.batch(new, pos.to(DEV), table.to(DEV))
    k, v, q = (torch.randn(sum(new), 2, 64, generator=torch.Generator().manual_seed(41)).half() for _ in range(3))
    cache.append(batch, k.to(DEV), v.to(DEV))
    assert all(a is None or torch.equal(_bits(a), _bits(b)) for a, b in zip(_host(cache), before))
    out = cache.read(batch, out=tuple(torch.full((sum(new), 2, 64), 5.0, device=DEV).half() for _ in range(2)))
    assert not bool(out[0].any()) and not bool(out[1].any())
    rows = table.repeat_interleave(torch.tensor(new), 0)
    for window, sinks in ((0, 0), (9, 3), (40, 0)):
        got = cache.attend(batch, q.to(DEV), window=window, sinks=sinks).cpu()
        _check_attention(cache, before, [1] * sum(new), [31] * sum(new), rows, q, got, window, sinks)


def test_what_does_not_belong_together_is_refused():
    cache = _cache(_pages(torch.float16, 4, 2, 16, 64, 42))
    batch = cache.batch([1], [0], torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    q = torch.zeros(1, 2, 64, dtype=torch.float16, device=DEV)
    for window, sinks in ((-1, 0), (0, -1), (2 ** 31, 0), (2 ** 32 + 1, 0), (1, 2 ** 32)):
        with pytest.raises(ValueError, match="window and sinks"):
            cache.attend(batch, q, window=window, sinks=sinks)
    cache.attend(batch, q, window=2 ** 31 - 1, sinks=2 ** 31 - 1)
    batch.table = torch.zeros(1, 1, dtype=torch.int32)   # (as a batch made for pages elsewhere)
    for call in (lambda: cache.append(batch, q, q), lambda: cache.read(batch), lambda: cache.attend(batch, q)):
        with pytest.raises(ValueError, match="the batch is on"):
            call()


@pytest.mark.parametrize("form", [torch.float16, E4M3, torch.int8], ids=["f16", "e4m3", "i8"])
def test_a_call_of_many_rows_stores_and_reads_what_small_ones_do(form):
    """More than 64 MB of rows, which go past the caches: pages and rows to the last bit those of calls of one sequence."""
    seqs, n, heads, hd, page = 9, 510, 32, 128, 64
    g = torch.Generator(device=DEV).manual_seed(50)
    k, v = (torch.randn(seqs * n, heads, hd, generator=g, device=DEV).half() for _ in range(2))
    table = torch.randperm(seqs * 8, generator=g, device=DEV).int().view(seqs, 8)
    got = []
    for each in (seqs, 1):
        cache = _cache(_pages(form, seqs * 8, heads, page, hd, 51))
        rows = []
        for s in range(0, seqs, each):
            batch = cache.batch([n] * each, [0 if i % 2 else 2 for i in range(s, s + each)], table[s:s + each])
            part = slice(s * n, (s + each) * n)
            cache.append(batch, k[part], v[part])
            rows.append(cache.read(batch))
        got.append(_host(cache) + [torch.cat([r[i] for r in rows]).cpu() for i in range(2)])
    for a, b in zip(*got):
        assert a is None or torch.equal(_bits(a), _bits(b))

"""Batches that mix single tokens, drafts and portions over split histories.  Oracle and tolerances: those of the attention's other
tests."""
import pytest
import torch

from test_gpu_paged import DEV, E4M3, _cache, _check_attention, _host, _pages, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,pos", [([150, 1, 1, 2], [20, 3000, 0, 1700]), ([1, 200, 3], [2900, 1500, 900]),
                                     ([1] * 9 + [70], [300 * i for i in range(9)] + [2000])], ids=["portion", "split", "many"])
@pytest.mark.parametrize("form", [torch.float16, E4M3, torch.int8], ids=["f16", "e4m3", "i8"])
def test_single_tokens_beside_a_portion(form, new, pos):
    """The sums of a sequence's splits lie where only its own are read, and every row has the result that it has alone."""
    heads, kvh, hd, page = 4, 2, 64, 64
    blocks = [-(-(p + n) // page) for n, p in zip(new, pos)]
    table = _table(len(new), blocks, sum(blocks), 1)
    cache = _cache(_pages(form, sum(blocks), kvh, page, hd, 2))
    q = torch.randn(sum(new), heads, hd, generator=torch.Generator().manual_seed(3)).half()
    for window, sinks in ((0, 0), (1000, 5)):
        batch = cache.batch(new, pos, table.to(DEV))
        out = cache.attend(batch, q.to(DEV), window=window, sinks=sinks).cpu()
        assert max(batch.workspaces.values()) > 0
        _check_attention(cache, _host(cache), new, pos, table, q, out, window, sinks)


def test_what_requires_gradients_is_refused_while_they_are_recorded():
    cache = _cache(_pages(torch.float16, 2, 2, 16, 64, 4))
    batch = cache.batch([1], [0], torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    x = torch.randn(1, 2, 64, device=DEV).half()
    with_grad = x.clone().requires_grad_()
    for call in (lambda: cache.append(batch, with_grad, x), lambda: cache.append(batch, x, with_grad), lambda: cache.attend(batch, with_grad)):
        with pytest.raises(RuntimeError, match="no gradients"):
            call()
        with torch.no_grad():
            call()
    assert torch.equal(cache.attend(batch, x), with_grad.detach())


@pytest.mark.parametrize("new,pos", [([1] * 5, [3000, 0, 16, 700, 4000]), ([9, 1], [2000, 40]), ([200, 3], [1500, 10])], ids=str)
@pytest.mark.parametrize("form", [torch.float16, E4M3, torch.int8], ids=["f16", "e4m3", "i8"])
def test_a_call_repeats_itself_to_the_last_bit(form, new, pos):
    blocks = [-(-(p + n) // 16) for n, p in zip(new, pos)]
    cache = _cache(_pages(form, sum(blocks), 2, 16, 64, 5))
    batch = cache.batch(new, pos, _table(len(new), blocks, sum(blocks), 6).to(DEV))
    q = torch.randn(sum(new), 4, 64, generator=torch.Generator().manual_seed(7)).half().to(DEV)
    first = cache.attend(batch, q)
    for _ in range(3):
        assert torch.equal(cache.attend(batch, q), first)

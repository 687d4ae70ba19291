"""Decode steps of OPT decoders over pools that are smaller than their slots' capacity.  Oracle and tolerances: those of the decoder's
other tests over pages."""
import pytest
import torch

from metaseq_amd import random_prompts
from test_gpu_paged_decoder import _close, _model

pytestmark = pytest.mark.gpu


def _decode(d, cfg, cache, tokens):
    """One step; ``tokens``: per slot the last token, or None for a pad.  Logits."""
    last = torch.tensor([cfg.padding_idx if t is None else t for t in tokens], device="cuda")
    logits = torch.zeros(len(tokens), cfg.vocab_size, dtype=torch.float16, device="cuda")
    d.decode_slots(cache, last, tok_out=torch.zeros_like(last), score_out=torch.zeros(len(tokens), device="cuda"), logits_out=logits)
    return logits


@pytest.mark.parametrize("form", [torch.float16, torch.int8], ids=["f16", "i8"])
def test_a_paused_slot_leaves_the_pool_to_the_others(form):
    cfg, sd, model = _model()
    d = model.decoder
    cache = d.new_paged_cache(3, 96, pages=1 + 6 + 6, page=16, dtype=form)
    ids = [random_prompts(cfg, 1, n, seed=n)[0].tolist() for n in (9, 20, 30)]
    d.prefill_slots(cache, [0, 1, 2], [torch.tensor(t, device="cuda") for t in ids])
    g = torch.Generator().manual_seed(1)
    for step in range(60):     # (the prompts are 10, 21 and 31 tokens long)
        toks = [None] + torch.randint(4, cfg.vocab_size, (2,), generator=g).tolist()
        logits = _decode(d, cfg, cache, toks)
        for s in (1, 2):
            ids[s].append(toks[s])
    for s in (1, 2):
        _close(logits[s:s + 1], cfg, sd, torch.tensor(ids[s]), form, [len(ids[s]) - 1])
    assert cache.lens.tolist() == [len(t) for t in ids]
    # the one that was paused goes on where it was
    ids[0].append(77)
    logits = _decode(d, cfg, cache, [77, None, None])
    _close(logits[:1], cfg, sd, torch.tensor(ids[0]), form, [len(ids[0]) - 1])
    assert cache.lens.tolist() == [len(t) for t in ids]


def test_decode_steps_in_a_window_go_on_in_a_small_pool():
    cfg, sd, model = _model()
    d = model.decoder
    cache = d.new_paged_cache(2, 250, pages=2 * 5, page=16, window=40, sinks=5)
    ids = [random_prompts(cfg, 1, n, seed=n)[0].tolist() for n in (30, 12)]
    d.prefill_slots(cache, [0, 1], [torch.tensor(t, device="cuda") for t in ids])
    g = torch.Generator().manual_seed(2)
    for step in range(200):
        toks = torch.randint(4, cfg.vocab_size, (2,), generator=g).tolist()
        if step % 7 == 3:
            toks[step % 2] = None
        logits = _decode(d, cfg, cache, toks)
        for s in (0, 1):
            if toks[s] is not None:
                ids[s].append(toks[s])
                if step % 40 > 36:
                    _close(logits[s:s + 1], cfg, sd, torch.tensor(ids[s]), torch.float16, [len(ids[s]) - 1], 40, 5)
    assert cache.lens.tolist() == [len(t) for t in ids]
    for s in (0, 1):
        d.release_slot(cache, s)
    assert sorted(cache.free) == list(range(10))


@pytest.mark.parametrize("slots", [129, 200, 256])
def test_int8_weights_take_many_slots_in_chunks(slots):
    """No product of a step has more than 128 rows (the int8 product of more is many times slower); every slot has its result."""
    cfg, _, model = _model(heads=2)
    d = model.decoder
    d.quantize_int8_()
    cache = d.new_paged_cache(slots, 48, page=16)
    ids = [random_prompts(cfg, 1, 3 + s % 20, seed=s)[0].tolist() for s in range(slots)]
    for s in range(0, slots, 50):
        d.prefill_slots(cache, list(range(s, min(s + 50, slots))), [torch.tensor(t, device="cuda") for t in ids[s:s + 50]])
    sd = d.dequantized_state_dict()
    sd = {k if k.startswith("decoder.") else "decoder." + k: v for k, v in sd.items()}
    rows = []
    linear = d._linear
    d._linear = lambda lib, stream, x, lin, M, *a, **k: (rows.append(M), linear(lib, stream, x, lin, M, *a, **k))[1]
    g = torch.Generator().manual_seed(3)
    for step in range(3):
        toks = torch.randint(4, cfg.vocab_size, (slots,), generator=g).tolist()
        toks[step * 40 + 7] = None
        logits = _decode(d, cfg, cache, toks)
        for s, t in enumerate(toks):
            ids[s] += [] if t is None else [t]
        for s in (0, 63, 64, 99, 100, 127, 128, slots - 1):
            if toks[s] is not None:
                _close(logits[s:s + 1], cfg, sd, torch.tensor(ids[s]), torch.float16, [len(ids[s]) - 1])
    assert rows and max(rows) <= 128
    assert cache.lens.tolist() == [len(t) for t in ids]


def test_wanted_places_belong_to_entries():
    """As many as entries; any iterables; nothing has run when they are refused."""
    cfg, sd, model = _model()
    d = model.decoder
    cache = d.new_paged_cache(3, 40, page=16)
    entries = [(0, [5, 6, 7]), (2, [8, 9])]
    for want in ([[2]], [[2], [1], [0]], []):
        with pytest.raises(ValueError, match="wanted places for"):
            d.extend(cache, entries, want=want)
    assert cache.host_lens == [-1] * 3 and len(cache.free) == 9
    with pytest.raises(ValueError, match="not a paged cache"):
        d.extend(d.new_slot_cache(2, 40), entries)
    got = d.extend(cache, iter(entries), want=(iter(w) for w in ([2, 0], (1,))))
    assert got.shape == (3, cfg.vocab_size)
    _close(got[:2], cfg, sd, torch.tensor([5, 6, 7]), torch.float16, [2, 0])
    _close(got[2:], cfg, sd, torch.tensor([8, 9]), torch.float16, [1])


def test_bad_pages_are_refused_before_the_first_request():
    from metaseq_amd import Dictionary, GeneratorInterface
    from metaseq_amd.service import ContinuousBatcher

    cfg, _, model = _model()
    api = GeneratorInterface(model, Dictionary(cfg.vocab_size))
    for page in (0, -16, 24, 512):
        with pytest.raises(ValueError, match="positions"):
            model.decoder.new_paged_cache(2, 100, page=page)
        with pytest.raises(ValueError, match="positions"):
            ContinuousBatcher(api, slots=4, capacity=64, cache_args=dict(page=page))
    with pytest.raises(ValueError, match="no argument pgae"):
        ContinuousBatcher(api, slots=4, capacity=64, cache_args=dict(pgae=16))

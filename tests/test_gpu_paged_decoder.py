"""OPT decoders over a paged cache: ``extend`` (prompts, portions and single tokens in any mix), the slot interface and
continuous batching, against a plain OPT forward in 64 bits that can keep its keys and values as 8-bit pages do.

Tolerances: those of the contiguous path against its oracle (tests of the decoder: largest 2e-2, mean 2e-3 on logits
of such models), which rounds at more places than this one.  In 8 bits a key or value that fp16 arithmetic moves
across a rounding border changes by one step, at most twice the half step that the format itself may be off by, and few do:
their effect is bounded by twice that of the format, the distance between the 64-bit results with and without it."""
import math

import pytest
import torch

from metaseq_amd import (Dictionary, GeneratorInterface, OPTConfig, TransformerLanguageModel, random_prompts,
                         random_state_dict)
from oracle import paged_oracle

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _model(hd=64, layers=2, heads=4, vocab=512, max_pos=300, seed=5):
    cfg = OPTConfig(layers, heads * hd, heads, vocab_size=vocab, max_target_positions=max_pos)
    sd = random_state_dict(cfg, seed=seed)
    return cfg, sd, TransformerLanguageModel.build_model(cfg, sd, device="cuda:0")


def _plain(cfg, sd, ids, form=None, window=0, sinks=0):
    """Logits [n, V] of one sequence, in 64 bits; ``form``: keys and values as such pages hold them."""
    w = {k.replace("decoder.", "", 1): v.double().cpu() for k, v in sd.items()}
    D, H, hd, n = cfg.decoder_embed_dim, cfg.decoder_attention_heads, cfg.head_dim, len(ids)

    def norm(x, name):
        return torch.nn.functional.layer_norm(x, (D,), w[name + ".weight"], w[name + ".bias"], 1e-5)

    def held(x):
        x = x.view(n, H, hd)
        if form in (None, torch.float16):
            return x
        c, e = paged_oracle.quantise(x.half(), form)
        return c * 2.0 ** e.double().unsqueeze(-1)

    x = w["embed_tokens.weight"][ids] + w["embed_positions.weight"][cfg.padding_idx + 1 + torch.arange(n)]
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    hidden = j > i
    if window:
        hidden = hidden | ((j <= i - window) & (j >= sinks))
    for layer in range(cfg.decoder_layers):
        p = "layers.%d." % layer
        h = norm(x, p + "self_attn_layer_norm")
        k, v, q = (h @ w[p + "self_attn.qkv_proj.weight"].T + w[p + "self_attn.qkv_proj.bias"]).split(D, 1)
        k, v, q = held(k), held(v), q.view(n, H, hd)
        z = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)
        o = torch.einsum("hij,jhd->ihd", torch.softmax(z.masked_fill(hidden, -math.inf), -1), v).reshape(n, D)
        x = x + o @ w[p + "self_attn.out_proj.weight"].T + w[p + "self_attn.out_proj.bias"]
        h = torch.relu(norm(x, p + "final_layer_norm") @ w[p + "fc1.weight"].T + w[p + "fc1.bias"])
        x = x + h @ w[p + "fc2.weight"].T + w[p + "fc2.bias"]
    return norm(x, "layer_norm") @ w["embed_tokens.weight"].T


def _close(got, cfg, sd, ids, form, at, window=0, sinks=0):
    want = _plain(cfg, sd, ids, form, window, sinks)[at]
    d = (got.double().cpu() - want).abs()
    own = (0.0, 0.0)
    if form != torch.float16:
        e = (want - _plain(cfg, sd, ids, None, window, sinks)[at]).abs()
        own = (float(e.max()), float(e.mean()))
    assert float(d.max()) <= 2e-2 + 2 * own[0] and float(d.mean()) <= 2e-3 + 2 * own[1], (float(d.max()), float(d.mean()), own)


@pytest.mark.parametrize("form", [torch.float16, E4M3, torch.int8], ids=["f16", "e4m3", "i8"])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64)])
def test_extend_in_any_portions(form, hd, page):
    cfg, sd, model = _model(hd)
    d = model.decoder
    cache = d.new_paged_cache(3, 250, page=page, dtype=form)
    ids = [t[0] for t in (random_prompts(cfg, 1, n, seed=n) for n in (230, 140, 9))]
    dev = [t.cuda() for t in ids]
    at = [0, 0, 0]
    # a long portion beside single tokens, short ones, one of all slots, a last one of one slot
    for counts in ((140, 1, 0), (1, 1, 5), (1, 70, 1), (30, 1, 1), (57, 66, 0), (1, 1, 2)):
        entries = [(s, dev[s][at[s]:at[s] + n]) for s, n in enumerate(counts) if n]
        got = d.extend(cache, entries, want=[[len(t) - 1, 0] for _, t in entries])
        row = 0
        for s, t in entries:
            places = [at[s] + len(t) - 1, at[s]]
            _close(got[row:row + 2], cfg, sd, ids[s][:at[s] + len(t)], form, places)
            at[s] += len(t)
            row += 2
    assert at == [230, 140, 9] and cache.host_lens == at and cache.lens.tolist() == at


@pytest.mark.parametrize("form", [torch.float16, torch.int8], ids=["f16", "i8"])
@pytest.mark.parametrize("slots", [3, 70, 150])
def test_the_slot_interface(form, slots):
    """Prefill, copies that share pages, decode steps with empty slots and pads between, release, and extend again."""
    cfg, sd, model = _model()
    d = model.decoder
    cache = d.new_paged_cache(slots, 100, page=16, dtype=form)
    pages = len(cache.free)
    a, b = (random_prompts(cfg, 1, n, seed=n)[0] for n in (37, 20))
    lg = d.prefill_slots(cache, [0, 2], [a.cuda(), b.cuda()])
    _close(lg[0], cfg, sd, a, form, slice(None))
    d.copy_slot(cache, 0, 1, length=len(a))
    assert len(cache.free) == pages - 3 - 2            # the copy holds the same pages
    ids = {0: a.tolist(), 1: a.tolist(), 2: b.tolist()}
    step = {0: [11, 12, 13, 14], 1: [21, 22, 23, 24], 2: [31, None, 33, 34]}   # None: a pad
    V = cfg.vocab_size
    tok, score = torch.zeros(slots, dtype=torch.long, device="cuda"), torch.zeros(slots, device="cuda")
    for i in range(4):
        last = torch.full((slots,), cfg.padding_idx, dtype=torch.long)
        for s in (0, 1, 2):
            if step[s][i] is not None:
                last[s] = step[s][i]
                ids[s].append(step[s][i])
        logits = torch.zeros(slots, V, dtype=torch.float16, device="cuda")
        d.decode_slots(cache, last.cuda(), tok_out=tok, score_out=score, logits_out=logits)
        for s in (0, 1, 2):
            if step[s][i] is not None:
                _close(logits[s:s + 1], cfg, sd, torch.tensor(ids[s]), form, [len(ids[s]) - 1])
                assert int(tok[s]) == int(logits[s].argmax())
    assert cache.lens.tolist()[:3] == [len(ids[s]) for s in (0, 1, 2)]
    d.release_slot(cache, 1)
    got = d.extend(cache, [(2, [41, 42]), (0, [51])], want_all=True)
    _close(got[:2], cfg, sd, torch.tensor(ids[2] + [41, 42]), form, [len(ids[2]), len(ids[2]) + 1])
    _close(got[2:], cfg, sd, torch.tensor(ids[0] + [51]), form, [len(ids[0])])
    for s in (0, 2):
        d.release_slot(cache, s)
    assert sorted(cache.free) == list(range(pages)) and cache.lens.tolist() == [-1] * slots


def test_a_window_gives_pages_back():
    cfg, sd, model = _model()
    d = model.decoder
    cache = d.new_paged_cache(2, 250, pages=9, page=16, window=40, sinks=5)   # fewer than the slots could fill
    ids = random_prompts(cfg, 1, 240, seed=7)[0]
    for at in range(0, 240, 30):
        got = d.extend(cache, [(1, ids[at:at + 30].cuda())], want=[[29]])
        _close(got, cfg, sd, ids[:at + 30], torch.float16, [at + 29], 40, 5)
        assert int((cache.host_table[1] >= 0).sum()) <= 1 + 4
    with pytest.raises(ValueError, match="pages are needed"):
        d.extend(cache, [(0, ids[:100].cuda())])
    assert cache.host_lens[0] == -1


def test_portions_longer_than_a_pass_and_wanted_places_in_any_order():
    cfg, sd, model = _model()
    d = model.decoder
    ids = [random_prompts(cfg, 1, n, seed=n)[0] for n in (100, 61)]
    whole = d.new_paged_cache(2, 150, page=32)
    want = [[99, 3, 50, 3], [60, 0]]
    a = d.extend(whole, [(0, ids[0].cuda()), (1, ids[1].cuda())], want=want)
    cut = d.new_paged_cache(2, 150, page=32)
    d.PORTION = 47
    b = d.extend(cut, [(0, ids[0].cuda()), (1, ids[1].cuda())], want=want)
    del d.PORTION
    assert a.shape == b.shape == (6, cfg.vocab_size)
    assert torch.equal(b[1], b[3])
    for got in (a, b):
        _close(got[:4], cfg, sd, ids[0], torch.float16, want[0])
        _close(got[4:], cfg, sd, ids[1], torch.float16, want[1])


def test_refusals():
    cfg, sd, model = _model()
    d = model.decoder
    with pytest.raises(ValueError):
        d.new_paged_cache(300, 100)
    with pytest.raises(ValueError):
        d.new_paged_cache(2, 1000)
    with pytest.raises(ValueError):
        d.new_paged_cache(2, 100, page=24)
    with pytest.raises(ValueError):
        d.new_paged_cache(2, 100, dtype=torch.bfloat16)
    cache = d.new_paged_cache(2, 40, page=16)
    with pytest.raises(ValueError, match="named twice"):
        d.extend(cache, [(0, [5]), (0, [6])])
    with pytest.raises(ValueError, match="more than 40"):
        d.extend(cache, [(0, list(range(4, 45)))])
    with pytest.raises(ValueError, match="outside"):
        d.extend(cache, [(2, [5])])
    with pytest.raises(ValueError, match="wanted place"):
        d.extend(cache, [(0, [5, 6])], want=[[2]])
    assert cache.host_lens == [-1, -1] and len(cache.free) == 6


@pytest.mark.parametrize("form", [torch.float16, torch.int8], ids=["f16", "i8"])
def test_continuous_batching_over_pages(form):
    """Requests through the engine: their tokens are the arg-max of the plain forward over what came before, or within
    the tolerance of it."""
    from metaseq_amd.service import ContinuousBatcher

    cfg, sd, model = _model()
    api = GeneratorInterface(model, Dictionary(cfg.vocab_size))
    engine = ContinuousBatcher(api, slots=4, capacity=64, prefill_batch=2, cache_args=dict(page=16, dtype=form))
    prompts = [random_prompts(cfg, 1, n, seed=n)[0].tolist()[1:] for n in (5, 17, 30, 9, 22)]
    replies = [engine.submit(p, max_tokens=10, min_tokens=10) for p in prompts]
    for _ in range(200):
        if not engine.step() and all(not r.empty() for r in replies):
            break
    for p, r in zip(prompts, replies):
        toks = [int(t) for t in r.get_nowait()[1][0]["tokens"]]
        assert len(toks) >= 9        # (the tenth is the end of the sequence, which a record leaves out)
        ids = torch.tensor([cfg.eos_idx] + p + toks)
        want = _plain(cfg, sd, ids, form)
        own = 0.0 if form == torch.float16 else float((want - _plain(cfg, sd, ids)).abs().max())
        want[:, [cfg.padding_idx, cfg.eos_idx]] = -math.inf
        for i, tok in enumerate(toks):
            z = want[len(p) + i]
            assert float(z.max() - z[tok]) <= 2 * (2e-2 + 2 * own), (i, tok)
    assert all(n == -1 for n in engine.cache.host_lens) and sorted(engine.cache.free) == list(range(16))


def test_an_engine_is_refused_pages_that_a_step_could_run_out_of():
    from metaseq_amd.service import ContinuousBatcher

    cfg, _, model = _model()
    api = GeneratorInterface(model, Dictionary(cfg.vocab_size))
    with pytest.raises(ValueError, match="15 pages"):
        ContinuousBatcher(api, slots=4, capacity=64, cache_args=dict(page=16, pages=15))
    ContinuousBatcher(api, slots=4, capacity=64, cache_args=dict(page=16, pages=16))

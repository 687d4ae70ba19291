"""The paged cache's boundary without a GPU: the header and its binding, what is refused, and workspaces."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from metaseq_amd import PagedCache, _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "metaseq_paged.h")
ONE = 4096  # a pointer that is never followed


def _cache(**kw):
    c = _capi.PagedCacheC(_capi.MSA_F16, _capi.MSA_PAGES_SAME, 4, 128, 64, 100, ONE, ONE, None, None)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def _batch(**kw):
    b = _capi.PagedBatchC(8, 8, 1, 1, 1000, 16, 16, ONE, ONE, ONE)
    for name, value in kw.items():
        setattr(b, name, value)
    return b


def _args(**kw):
    a = _capi.PagedAttentionArgs(8, ONE, 1024, ONE, 1024, 0, 0, 0, 0.1, ONE, 1 << 40)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def test_the_binding_matches_the_header(tmp_path):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    decls = {m.group(1): len(m.group(2).split(",")) for m in
             re.finditer(r"\b(msa_\w+)\s*\(([^;{]*?)\)\s*;", text, flags=re.S)}
    assert decls == {n: len(a) for n, a in _capi.PAGED_SIGNATURES.items()}
    lib = _capi.load()
    structs = {"msa_paged_cache": _capi.PagedCacheC, "msa_paged_batch": _capi.PagedBatchC,
               "msa_paged_attention_args": _capi.PagedAttentionArgs}
    code = '#include <stdio.h>\n#include "%s"\nint main(void) {\n' % HEADER
    for name, s in structs.items():
        code += '  printf("%%zu", sizeof(%s));\n' % name
        for field, _ in s._fields_:
            code += '  printf(" %%zu", offsetof(%s, %s));\n' % (name, field)
        code += '  printf("\\n");\n'
    (tmp_path / "a.c").write_text(code + "  return 0;\n}\n")
    subprocess.run(["gcc", "-o", str(tmp_path / "a"), str(tmp_path / "a.c")], check=True)
    lines = subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, s in zip(lines, structs.values()):
        assert [int(x) for x in line.split()] == [ctypes.sizeof(s)] + [getattr(s, f).offset for f, _ in s._fields_]
    assert all(hasattr(lib, n) for n in decls)


BAD_CACHES = [dict(dtype=_capi.MSA_F32), dict(dtype=7), dict(format=3), dict(format=-1), dict(hd=72), dict(hd=32), dict(hd=0),
              dict(page=8), dict(page=48), dict(page=512), dict(page=0), dict(kv_heads=0), dict(pages=0), dict(k_pages=None),
              dict(v_pages=None), dict(k_pages=4100), dict(format=1), dict(format=2, k_exp=ONE),
              dict(format=2, k_exp=ONE, v_exp=4097)]
BAD_BATCHES = [dict(M=-1), dict(M=1 << 24), dict(max_count=1 << 24), dict(nseq=-1), dict(max_count=-1), dict(key_bound=-1), dict(min_count=-1), dict(min_count=2), dict(blocks=0), dict(table_stride=15),
               dict(blocks=(1 << 24) + 1, table_stride=1 << 25), dict(nseq=(1 << 20) + 1), dict(seq_start=None), dict(seq_pos=None),
               dict(table=None)]
BAD_ARGS = [dict(heads=0), dict(heads=6), dict(heads=-4), dict(q=None), dict(out=None), dict(q=4100), dict(out=4104),
            dict(ldq=1016), dict(ldq=1028), dict(ldo=1000), dict(ldo=1025), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
            dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(out_mb=2), dict(out_mb=-1)]


@pytest.mark.parametrize("bad", BAD_CACHES + BAD_BATCHES, ids=str)
def test_bad_caches_and_batches_are_refused(bad):
    lib = _capi.load()
    fields = [f for f, _ in _capi.PagedCacheC._fields_]
    here = all(k in fields for k in bad)
    c, b = (_cache(**bad), _batch()) if here else (_cache(), _batch(**bad))
    for rc in (lib.msa_paged_append(ctypes.byref(c), ctypes.byref(b), ONE, 512, ONE, 512, None),
               lib.msa_paged_read(ctypes.byref(c), ctypes.byref(b), ONE, 512, ONE, 512, None),
               lib.msa_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), ctypes.byref(_args())),
               lib.msa_paged_attention(ctypes.byref(c), ctypes.byref(b), ctypes.byref(_args()), None)):
        assert rc == -1 and lib.msa_last_error()


@pytest.mark.parametrize("bad", BAD_ARGS, ids=str)
def test_bad_attention_arguments_are_refused(bad):
    lib = _capi.load()
    assert lib.msa_paged_attention(ctypes.byref(_cache()), ctypes.byref(_batch()), ctypes.byref(_args(**bad)), None) == -1


@pytest.mark.parametrize("k,ldk,v,ldv", [(None, 512, ONE, 512), (ONE, 512, None, 512), (ONE, 504, ONE, 512), (ONE, 512, ONE, 516),
                                         (4100, 512, ONE, 512), (ONE, 512, 4098, 512)])
def test_bad_rows_are_refused(k, ldk, v, ldv):
    lib = _capi.load()
    for fn in (lib.msa_paged_append, lib.msa_paged_read):
        assert fn(ctypes.byref(_cache()), ctypes.byref(_batch()), k, ldk, v, ldv, None) == -1


def test_nothing_to_do_needs_no_gpu():
    lib = _capi.load()
    for b in (_batch(M=0), _batch(nseq=0), _batch(max_count=0, min_count=0)):
        assert lib.msa_paged_append(ctypes.byref(_cache()), ctypes.byref(b), None, 512, None, 512, None) == 0
        assert lib.msa_paged_read(ctypes.byref(_cache()), ctypes.byref(b), ONE, 512, ONE, 512, None) == 0
        assert lib.msa_paged_attention(ctypes.byref(_cache()), ctypes.byref(b), ctypes.byref(_args()), None) == 0
        assert lib.msa_paged_attention_workspace_bytes(ctypes.byref(_cache()), ctypes.byref(b), ctypes.byref(_args())) == 0


def test_a_workspace_that_is_too_small_is_refused():
    lib = _capi.load()
    b = _batch(M=1, nseq=1, key_bound=100000, blocks=2000, table_stride=2000)
    a = _args()
    need = lib.msa_paged_attention_workspace_bytes(ctypes.byref(_cache()), ctypes.byref(b), ctypes.byref(a))
    assert need > 0
    a.workspace_bytes = need - 1
    assert lib.msa_paged_attention(ctypes.byref(_cache()), ctypes.byref(b), ctypes.byref(a), None) == -1
    assert b"workspace" in lib.msa_last_error()
    a.workspace, a.workspace_bytes = None, need
    assert lib.msa_paged_attention(ctypes.byref(_cache()), ctypes.byref(b), ctypes.byref(a), None) == -1


def test_python_refuses_what_it_can_see():
    t = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype)  # noqa: E731
    with pytest.raises(ValueError, match="page"):
        PagedCache(t(3, 2, 24, 64), t(3, 2, 64, 24))
    with pytest.raises(ValueError, match="heads"):
        PagedCache(t(3, 2, 16, 72), t(3, 2, 72, 16))
    with pytest.raises(ValueError, match="v_pages"):
        PagedCache(t(3, 2, 16, 64), t(3, 2, 16, 64))
    with pytest.raises(ValueError, match="exponents"):
        PagedCache(t(3, 2, 16, 64), t(3, 2, 64, 16), t(3, 2, 16, dtype=torch.int8), t(3, 2, 16, dtype=torch.int8))
    with pytest.raises(ValueError, match="k_exp"):
        PagedCache(t(3, 2, 16, 64, dtype=torch.int8), t(3, 2, 64, 16, dtype=torch.int8))
    with pytest.raises(ValueError, match="not torch.float32"):
        PagedCache(t(3, 2, 16, 64, dtype=torch.float32), t(3, 2, 64, 16, dtype=torch.float32))
    with pytest.raises(ValueError, match="contiguous"):
        PagedCache(t(3, 16, 2, 64).transpose(1, 2), t(3, 2, 64, 16))
    with pytest.raises(RuntimeError, match="GPU"):
        PagedCache(t(3, 2, 16, 64), t(3, 2, 64, 16))


@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 128), (12, 12, 64), (8, 1, 256)])
@pytest.mark.parametrize("form", [_capi.MSA_PAGES_SAME, _capi.MSA_PAGES_INT8], ids=["same", "i8"])
@pytest.mark.parametrize("tokens", [300, 8191])
def test_single_tokens_beside_a_portion_need_little_more_than_alone(form, heads, kv_heads, hd, tokens):
    """The sums of split keys have room for the rows whose keys are split - of every sequence as many as the kernel of few rows
    takes, for the host does not say which have fewer - not for every row of the batch."""
    lib = _capi.load()
    c = _cache(format=form, kv_heads=kv_heads, hd=hd, k_exp=ONE, v_exp=ONE)

    def need(new):
        b = _batch(M=sum(new), nseq=len(new), max_count=max(new), min_count=min(new), key_bound=131072, blocks=2048, table_stride=2048)
        n = lib.msa_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), ctypes.byref(_args(heads=heads)))
        assert n >= 0
        return n

    few = max(1, (32 if form == _capi.MSA_PAGES_SAME else 64) * kv_heads // heads)   # tokens that the kernel of few rows takes
    assert need([1]) > 0
    for singles in (1, 7):
        got = need([tokens] + [1] * singles)
        assert got <= max(need([tokens]), (1 + singles) * need([few])) and got <= 64 << 20


@pytest.mark.parametrize("heads", [256, 4096, 32768, 65535])
@pytest.mark.parametrize("max_count", [1 << 23, (1 << 24) - 1])
@pytest.mark.parametrize("splits", [0, 1])
def test_counts_whose_blocks_pass_32_bits_are_refused(heads, max_count, splits):
    """A batch may name more rows for its longest sequence than it has; blocks for all of them must fit a launch."""
    lib = _capi.load()
    c = _cache(kv_heads=1)
    b = _batch(M=200, nseq=1, max_count=max_count, min_count=0, key_bound=100000 * splits, blocks=2000, table_stride=2000)
    a = _args(heads=heads, ldq=heads * 128, ldo=heads * 128)
    assert lib.msa_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), ctypes.byref(a)) >= 0
    if max_count * heads > 128 * ((1 << 24) - 1):
        assert lib.msa_paged_attention(ctypes.byref(c), ctypes.byref(b), ctypes.byref(a), None) == -1
        assert b"too many rows" in lib.msa_last_error()

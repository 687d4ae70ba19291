"""Keys and values of one attention layer in pages, as they are or in 8 bits, and the attention that reads them.

The reference appends to one tensor per layer and re-copies the history at every step
(metaseq/modules/multihead_attention.py:449-479); ``KVCache`` reserves a row of a fixed capacity per sequence.  Here
a sequence's positions lie in pages of 16 to 256 positions that a table names in order, so that sequences of any length
share one pool, several of them may share the pages of a common beginning, and pages that no window sees any more can be given
to others.

Layouts (contiguous): ``k_pages`` [pages, kv_heads, page, head_dim], ``v_pages`` [pages, kv_heads, head_dim, page].
Their dtype is the format: fp16 or bf16 (that of keys, values, queries and outputs), or float8_e4m3fn or int8, whose codes c
stand for c 2^e with one exponent e per position and head, ``k_exp`` and ``v_exp`` (int8 [pages, kv_heads, page]).
"""
import ctypes
import math

import torch

from . import _capi
from .decoder_base import upload

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 80, 96, 128, 192, 256)
_DTYPES = {torch.float16: _capi.MSA_F16, torch.bfloat16: _capi.MSA_BF16}
_FORMATS = {torch.float8_e4m3fn: _capi.MSA_PAGES_E4M3, torch.int8: _capi.MSA_PAGES_INT8}


class PagedBatch:
    """The new tokens of several sequences, one sequence's rows behind the other's (``PagedCache.batch``).

    ``rows``: how many there are.  ``seq_start``, ``seq_pos``, ``table``: what the kernels read (int32, device);
    ``seq_pos`` and ``table`` may be written between calls, on the stream that the calls run on - a captured graph
    follows them - as long as no position reaches ``key_bound``."""

    def __init__(self, c, rows, seq_start, seq_pos, table):
        self.c, self.rows, self.seq_start, self.seq_pos, self.table = c, rows, seq_start, seq_pos, table
        self.by_ref = ctypes.byref(c)
        self.workspaces = {}   # bytes that attention over such heads and pages asks for

    @property
    def key_bound(self):
        return self.c.key_bound


def _no_gradients(*tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("metaseq_amd: the paged cache records no gradients; call it under torch.no_grad()")


class PagedCache:
    """The pages of one layer.  The tensors are used as they are, not copied."""

    def __init__(self, k_pages, v_pages, k_exp=None, v_exp=None):
        if k_pages.dim() != 4:
            raise ValueError("k_pages must be [pages, kv_heads, page, head_dim]")
        pages, kv_heads, page, hd = k_pages.shape
        eight = k_pages.dtype in _FORMATS
        if not eight and k_pages.dtype not in _DTYPES:
            raise ValueError("pages are fp16, bf16, float8_e4m3fn or int8, not %s" % k_pages.dtype)
        if page not in PAGE_SIZES or hd not in HEAD_DIMS:
            raise ValueError("pages of %d positions and heads of %d: pages of %s and heads of %s are supported"
                             % (page, hd, PAGE_SIZES, HEAD_DIMS))
        wanted = [("v_pages", v_pages, (pages, kv_heads, hd, page), k_pages.dtype)]
        if eight:
            wanted += [(n, t, (pages, kv_heads, page), torch.int8) for n, t in (("k_exp", k_exp), ("v_exp", v_exp))]
        elif k_exp is not None or v_exp is not None:
            raise ValueError("16-bit pages have no exponents")
        for name, t, shape, dtype in wanted:
            if t is None or tuple(t.shape) != shape or t.dtype != dtype or t.device != k_pages.device:
                raise ValueError("%s must be %s %s on %s" % (name, dtype, list(shape), k_pages.device))
        for t in (k_pages, v_pages, k_exp, v_exp):
            if t is not None and not t.is_contiguous():
                raise ValueError("pages and exponents must be contiguous")
        if not k_pages.is_cuda:
            raise RuntimeError("metaseq_amd: pages must live on the GPU (no CPU path exists)")
        self.k_pages, self.v_pages, self.k_exp, self.v_exp = k_pages, v_pages, k_exp, v_exp
        self.pages, self.kv_heads, self.page, self.head_dim = pages, kv_heads, page, hd
        self.device = k_pages.device
        self._lib = _capi.load()
        self._scale = 1.0 / math.sqrt(hd)
        self._c = {}
        for dtype, code in _DTYPES.items():
            if eight or dtype == k_pages.dtype:
                c = _capi.PagedCacheC(code, _FORMATS.get(k_pages.dtype, _capi.MSA_PAGES_SAME), kv_heads, hd, page, pages,
                                      *(_capi.ptr(t) for t in (k_pages, v_pages, k_exp, v_exp)))
                self._c[dtype] = (c, ctypes.byref(c))

    @classmethod
    def empty(cls, pages, kv_heads, head_dim, page=64, dtype=torch.float16, device="cuda"):
        """A cache of that many pages of ``dtype`` (float16, bfloat16, float8_e4m3fn or int8)."""
        new = lambda *shape, dtype=dtype: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
        exps = [new(pages, kv_heads, page, dtype=torch.int8) for _ in range(2)] if dtype in _FORMATS else []
        return cls(new(pages, kv_heads, page, head_dim), new(pages, kv_heads, head_dim, page), *exps)

    def bytes(self):
        return sum(t.numel() * t.element_size() for t in (self.k_pages, self.v_pages, self.k_exp, self.v_exp)
                   if t is not None)

    # ------------------------------------------------------------------ batches
    def batch(self, new, positions, table, key_bound=None):
        """``new``: how many tokens each sequence adds (host).  ``positions``: the position of each one's first (host
        list, or int32 device tensor that the calls read when they run; negative: the sequence sits them out).
        ``table``: int32 device tensor [sequences, blocks], the page of each page-full of positions; positions whose
        entry names no page are not stored, read as zeros and seen by no row.  ``key_bound``: no position reaches it
        (default: from ``positions``, or what the table can name)."""
        new = [int(n) for n in new]
        if any(n < 0 for n in new):
            raise ValueError("a negative number of new tokens")
        if table.dim() != 2 or table.dtype != torch.int32 or table.device != self.device or table.shape[0] != len(new) \
                or table.shape[1] < 1 or (table.shape[1] > 1 and table.stride(1) != 1) \
                or (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
            raise ValueError("table must be int32 [%d, blocks] on %s with its rows apart" % (len(new), self.device))
        span = table.shape[1] * self.page
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        if torch.is_tensor(positions):
            if positions.dtype != torch.int32 or tuple(positions.shape) != (len(new),) or positions.device != self.device \
                    or (len(new) > 1 and positions.stride(0) != 1):
                raise ValueError("positions must be int32 [%d] on %s" % (len(new), self.device))
            seq_start, seq_pos, bound = upload(start, torch.int32, self.device), positions, span
        else:
            positions = [int(p) for p in positions]
            if len(positions) != len(new):
                raise ValueError("one position per sequence")
            ends = [p + n for p, n in zip(positions, new) if p >= 0]
            bound = max(ends, default=0)
            if bound > span:
                raise ValueError("position %d lies behind the %d that the table can name" % (bound - 1, span))
            both = upload(start + positions, torch.int32, self.device)
            seq_start, seq_pos = both[:len(start)], both[len(start):]
        if key_bound is not None:
            bound = int(key_bound)
        stride = table.stride(0) if table.shape[0] > 1 else table.shape[1]
        c = _capi.PagedBatchC(start[-1], len(new), max(new, default=0), min((n for n in new if n), default=0),
                              max(0, min(bound, span)), table.shape[1], stride,
                              seq_start.data_ptr(), seq_pos.data_ptr(), table.data_ptr())
        return PagedBatch(c, start[-1], seq_start, seq_pos, table)

    # ------------------------------------------------------------------ calls
    def _of(self, dtype, batch=None):
        if batch is not None and batch.table.device != self.device:
            raise ValueError("the batch is on %s, the pages are on %s" % (batch.table.device, self.device))
        if dtype not in self._c:
            raise ValueError("pages of %s hold no %s" % (self.k_pages.dtype, dtype))
        return self._c[dtype][1]

    def _rows(self, name, t, rows, heads, copy):
        """``t`` as rows of heads, one behind the other, that the kernels can read or write in place: (tensor, address,
        row stride)."""
        if t.shape != (rows, heads, self.head_dim) or t.device != self.device:
            raise ValueError("%s must be [%d, %d, %d] on %s, not %s on %s"
                             % (name, rows, heads, self.head_dim, self.device, list(t.shape), t.device))
        sr, sh, sd = t.stride()
        at, width = t.data_ptr(), heads * self.head_dim
        if sd == 1 and (heads == 1 or sh == self.head_dim) and at % 16 == 0 and (rows < 2 or (sr % 8 == 0 and sr >= width)):
            return t, at, sr if rows > 1 else width
        if not copy:
            raise ValueError("%s must have its heads one behind the other, 16-byte aligned, rows a multiple of 8 apart"
                             % name)
        t = t.contiguous() if not t.is_contiguous() else t.clone()
        return t, t.data_ptr(), width

    def _run(self, fn, *args):
        at = self.device.index
        stream = torch._C._cuda_getCurrentRawStream(at)   # (torch.cuda.current_stream without its object)
        if torch._C._cuda_getDevice() == at:
            rc = fn(*args, stream)
        else:
            with torch.cuda.device(self.device):
                rc = fn(*args, stream)
        if rc:
            _capi.check(rc, self._lib)

    def append(self, batch, k, v):
        """Stores the keys and values ([rows, kv_heads, head_dim], fp16 or bf16, any row stride) of a batch's tokens at
        their positions.  Nothing of this class records gradients: what requires them is refused unless recording is off
        (``torch.no_grad``)."""
        _no_gradients(k, v)
        if k.dtype != v.dtype:
            raise ValueError("keys are %s, values %s" % (k.dtype, v.dtype))
        c = self._of(k.dtype, batch)
        k, k_at, ldk = self._rows("k", k, batch.rows, self.kv_heads, True)
        v, v_at, ldv = self._rows("v", v, batch.rows, self.kv_heads, True)
        self._run(self._lib.msa_paged_append, c, batch.by_ref, k_at, ldk, v_at, ldv)

    def read(self, batch, dtype=None, out=None):
        """Keys and values at the positions of a batch's tokens, ([rows, kv_heads, head_dim],) * 2 of ``dtype`` (8-bit
        pages; default fp16).  ``out``: a pair of tensors to write them to; rows of sequences that sit the call out, and rows
        behind the last sequence's, keep what they hold there."""
        if out is None:
            dtype = dtype or (torch.float16 if self.k_pages.dtype in _FORMATS else self.k_pages.dtype)
            shape = (batch.rows, self.kv_heads, self.head_dim)
            out = tuple(torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        elif out[0].dtype != out[1].dtype or dtype not in (None, out[0].dtype):
            raise ValueError("keys and values come in one dtype")
        c = self._of(out[0].dtype, batch)
        (_, k_at, ldk), (_, v_at, ldv) = (self._rows("out", t, batch.rows, self.kv_heads, False) for t in out)
        self._run(self._lib.msa_paged_read, c, batch.by_ref, k_at, ldk, v_at, ldv)
        return out

    def attend(self, batch, q, *, scale=None, window=0, sinks=0, out=None):
        """Attention of a batch's tokens, whose keys and values are stored already: ``q`` [rows, heads, head_dim], the
        output alike.  A token at position i sees positions j <= i; with ``window`` only those with j > i - window or
        j < ``sinks``.  ``scale``: default head_dim ** -0.5.  Rows of sequences that sit the call out keep what ``out``
        holds (or are undefined)."""
        _no_gradients(q)
        if q.dim() != 3 or q.shape[1] % self.kv_heads or q.shape[1] == 0:
            raise ValueError("q must be [rows, heads, head_dim], heads a multiple of %d" % self.kv_heads)
        if not (0 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31):
            raise ValueError("window and sinks must be 0 .. 2^31 - 1")
        c = self._of(q.dtype, batch)
        heads = q.shape[1]
        q, q_at, ldq = self._rows("q", q, batch.rows, heads, True)
        if out is None:
            out = torch.empty(batch.rows, heads, self.head_dim, dtype=q.dtype, device=self.device)
            out_at, ldo = out.data_ptr(), heads * self.head_dim
        elif out.dtype != q.dtype:
            raise ValueError("out must be %s" % q.dtype)
        else:
            _, out_at, ldo = self._rows("out", out, batch.rows, heads, False)
        a = _capi.PagedAttentionArgs(heads, q_at, ldq, out_at, ldo, 0, window, sinks,
                                     self._scale if scale is None else scale, None, 0)
        ref = ctypes.byref(a)
        what = (self.kv_heads, self.head_dim, self.k_pages.dtype, heads, window, sinks)
        need = batch.workspaces.get(what)
        if need is None:
            need = self._lib.msa_paged_attention_workspace_bytes(c, batch.by_ref, ref)
            if need < 0:
                _capi.check(need, self._lib)
            batch.workspaces[what] = need
        if need:
            # (from torch's allocator, so that two captured graphs never share one)
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        self._run(self._lib.msa_paged_attention, c, batch.by_ref, ref)
        return out


class PagedSlots:
    """The cache of a decoder's slots in pages: one ``PagedCache`` per layer, one table for all of them, and the
    pages that no slot holds (``TransformerDecoder.new_paged_cache``).  It takes the place of a slot ``KVCache``: a
    slot is filled by prefills or ``extend``, advanced by decode steps, copied and released.

    A slot takes pages as it grows.  Copies share the full pages of what they copy (``refs`` counts the holders).
    With ``window``, attention is over the last ``window`` positions and the first ``sinks``, and a page that no
    position to come can see is given back by the next ``extend`` or when pages run out.  ``lens``: positions each slot
    holds (int32 on the device, negative: empty); ``host_lens``: the same on the host, except that decode steps count every
    slot of ``stale`` as having taken part, which only the device knows: a slot may hold pages ahead of its positions
    until ``reclaim`` takes them."""

    has_pads = False
    ragged = True

    def __init__(self, n_layers, slots, capacity, kv_heads, head_dim, pages, page, dtype, window, sinks, device):
        blocks = -(-capacity // page)
        self.batch, self.capacity, self.page, self.device = int(slots), int(capacity), int(page), device
        self.window, self.sinks = int(window), int(sinks)
        if not (0 <= self.window < 2 ** 31 and 0 <= self.sinks < 2 ** 31):
            raise ValueError("window and sinks must be 0 .. 2^31 - 1")
        self.layers = [PagedCache.empty(pages, kv_heads, head_dim, page, dtype, device) for _ in range(n_layers)]
        self.lens = torch.full((self.batch,), -1, dtype=torch.int32, device=device)
        self.host_lens = [-1] * self.batch
        self.table = torch.full((self.batch, blocks), -1, dtype=torch.int32, device=device)
        self.host_table = torch.full((self.batch, blocks), -1, dtype=torch.int32)
        self._blocks = self.host_table.numpy()   # the same memory, whose elements are read ten times as fast
        self.refs = [0] * pages
        self.free = list(range(pages - 1, -1, -1))
        self._passed = [0] * self.batch   # blocks below, behind those of the first positions, have been given back
        self.stale = set()

    def _page(self):
        if not self.free:
            raise ValueError("all %d pages are held" % len(self.refs))
        at = self.free.pop()
        self.refs[at] = 1
        return at

    def _drop(self, at):
        self.refs[at] -= 1
        if self.refs[at] == 0:
            self.free.append(at)

    def _missing(self, wanted):
        """What the positions [pos, pos + n) of every (slot, pos, n) lack: (slot, block) of new pages, and of copies."""
        new = [(s, b) for s, pos, n in wanted for b in range(pos // self.page, -(-(pos + n) // self.page))
               if int(self._blocks[s, b]) < 0]
        # a page that others hold too is not written to: whose next position lies in one gets a copy, but for the last
        copies, left = [], {}
        for s, pos, n in wanted:
            at = int(self._blocks[s, pos // self.page]) if n and pos % self.page else -1
            if at >= 0 and left.setdefault(at, self.refs[at]) > 1:
                left[at] -= 1
                copies.append((s, pos // self.page))
        return new, copies

    def reclaim(self):
        """Takes back the pages behind what each slot holds (waits for the device if decode steps have left that open), and
        those that its window has passed."""
        self.exact_lens(list(self.stale))
        for slot, n in enumerate(self.host_lens):
            for b in range(-(-max(n, 0) // self.page), self._blocks.shape[1]):
                if int(self._blocks[slot, b]) >= 0:
                    self._drop(int(self._blocks[slot, b]))
                    self._blocks[slot, b] = -1
            if n >= 0:
                self.holds(slot, n)

    def reserve(self, wanted, again=None):
        """Pages for the positions [pos, pos + n) of every (slot, pos, n); all of them or, with ValueError, none.  Where they are
        short, after a ``reclaim``, which makes the slots' lengths exact: then for what ``again()`` returns.  Returns what
        pages were reserved for."""
        if any(pos + n > self.capacity for _, pos, n in wanted):
            raise ValueError("a slot would hold more than %d positions" % self.capacity)
        new, copies = self._missing(wanted)
        if len(new) + len(copies) > len(self.free):
            self.reclaim()
            wanted = wanted if again is None else again()
            new, copies = self._missing(wanted)
        if len(new) + len(copies) > len(self.free):
            raise ValueError("%d pages are needed, %d are free" % (len(new) + len(copies), len(self.free)))
        for s, b in new:
            self._blocks[s, b] = self._page()
        for s, b in copies:
            old = int(self._blocks[s, b])
            self._blocks[s, b] = self._page()
            self._copy_page(old, int(self._blocks[s, b]))
            self._drop(old)
        if new or copies:
            self._upload()
        return wanted

    def _copy_page(self, src, dst):
        for layer in self.layers:
            for t in (layer.k_pages, layer.v_pages, layer.k_exp, layer.v_exp):
                if t is not None:
                    t[dst].view(torch.uint8).copy_(t[src].view(torch.uint8))

    def _upload(self):
        # (a copy in pinned memory of its own: the host table changes while the transfer is on its way)
        t = self.host_table.pin_memory() if self.table.is_cuda else self.host_table
        self.table.copy_(t, non_blocking=True)

    def exact_lens(self, slots):
        """Makes ``host_lens`` exact where decode steps may have left one of ``slots`` out (waits for the device)."""
        if not self.stale.isdisjoint(slots):
            lens = self.lens.tolist()
            for s in self.stale:
                self.host_lens[s] = lens[s]
            self.stale.clear()

    def holds(self, slot, n):
        """``slot`` has exactly ``n`` positions from here on; pages behind the window go back."""
        self.host_lens[slot] = n
        self.stale.discard(slot)
        if self.window:
            first = max(-(-self.sinks // self.page), self._passed[slot])
            # blocks below hold positions <= n - window only (a slot that steps took past its capacity has no more blocks)
            past = max(first, min((n - self.window + 1) // self.page, self._blocks.shape[1]))
            for b in range(first, past):
                if int(self._blocks[slot, b]) >= 0:
                    self._drop(int(self._blocks[slot, b]))
                    self._blocks[slot, b] = -1
            self._passed[slot] = past

    def release_row(self, slot):
        for b in range(self._blocks.shape[1]):
            if int(self._blocks[slot, b]) >= 0:
                self._drop(int(self._blocks[slot, b]))
        self.host_table[slot].fill_(-1)
        self.host_lens[slot], self._passed[slot] = -1, 0
        self.stale.discard(slot)

    def copy_row(self, src, dst, n):
        """Slot ``dst`` becomes the first ``n`` positions of slot ``src``: it shares src's pages.  ValueError where src does not
        hold so many, or has given back pages that dst's next position would see."""
        if src == dst:
            return
        if n > self.host_lens[src]:   # (an upper bound of them; exact_lens would wait)
            raise ValueError("slot %d holds no %d positions" % (src, n))
        if any(int(self._blocks[src, b]) < 0 for b in range(-(-n // self.page)) if not self.window
               or b * self.page < self.sinks or min((b + 1) * self.page, n) - 1 > n - self.window):
            raise ValueError("slot %d has given back pages that a copy of %d positions would see" % (src, n))
        self.release_row(dst)
        for b in range(-(-n // self.page)):
            at = int(self._blocks[src, b])
            if at >= 0:
                self.refs[at] += 1
                self._blocks[dst, b] = at
        self.host_lens[dst], self._passed[dst] = n, min(self._passed[src], -(-n // self.page))
        self._upload()

    def bytes(self):
        return sum(layer.bytes() for layer in self.layers)


class PagedRows:
    """One step's rows through a decoder's layers (``PagedSlots``): ``attend(i, ...)`` stores layer i's new keys and values
    and attends them.  Batch, work buffers and arguments are the same for all layers."""

    def __init__(self, lib, slots, batch, heads, head_dim, device):
        self.slots, self.batch, self.heads, self.layer = slots, batch, heads, 0
        D = heads * head_dim
        self.qkv = torch.empty(batch.rows, 3 * D, dtype=torch.float16, device=device)
        self.D = D
        first = slots.layers[0]
        self.args = _capi.PagedAttentionArgs(heads, self.qkv.data_ptr() + 4 * D, 3 * D, None, D, 0, slots.window,
                                             slots.sinks, 1.0 / math.sqrt(head_dim), None, 0)
        need = lib.msa_paged_attention_workspace_bytes(first._of(torch.float16), batch.by_ref, ctypes.byref(self.args))
        if need < 0:
            _capi.check(need, lib)
        self.workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
        self.args.workspace, self.args.workspace_bytes = self.workspace.data_ptr(), need

    def attend(self, lib, stream, out, out_mb):
        """Layer ``self.layer``: ``self.qkv`` holds the rows' keys, values and queries; ``out`` row-major, or packed
        with ``out_mb`` row blocks."""
        c, k = self.slots.layers[self.layer]._of(torch.float16), self.qkv.data_ptr()
        _capi.check(lib.msa_paged_append(c, self.batch.by_ref, k, 3 * self.D, k + 2 * self.D, 3 * self.D, stream), lib)
        self.args.out, self.args.out_mb = out.data_ptr(), out_mb
        _capi.check(lib.msa_paged_attention(c, self.batch.by_ref, ctypes.byref(self.args), stream), lib)

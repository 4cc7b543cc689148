"""The paged HCA cache: sequences of unequal length, chunks of new tokens, 8-bit rows.

``HCADecodingCache`` holds a batch of equally long sequences and takes one
token a step. The operators here serve a changing set of sequences from one pool
of pages:

``hca_paged_append``     a chunk's tokens into the cache, quantised as they are written
``hca_paged_attention``  the chunk's queries over it (``ops_hca.py:132-194``)
``paged_read``           cached rows back as numbers
``HCAPagedCache``        the pool, its page tables and the sequences in it

A pool is ``rows [P, page, c]`` (bfloat16, float8_e4m3fn or int8) with, for the
8-bit formats, ``scales [P, page]`` uint8: value = code * 2**(scale - 127), one
power of two per row. ``block_table [n_slots, nbp]`` and ``ring_table [n_slots,
nrp]`` (int32) give the pages of a slot's compressed rows and of its window rows
(position p at ring row ``p % (nrp * page)``), ``state [n_slots, 3, c]`` fp32 the
running softmax sums of its open block. A step names its sequences' ``slots
[S]``, their packed tokens ``cu_seqlens [S + 1]`` and the tokens cached before
them ``ctx_lens [S]``, int32 on the device. Only the sizes given as
Python numbers enter the launches, so that a captured step replays with new
contents of these tensors.

Forward only, as the caches beside it.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops_csa import _HEAD_DIMS, _aligned, _f32, _kernel_size, _pad_last

_FORMATS = {torch.bfloat16: 0, torch.float8_e4m3fn: 1, torch.int8: 2}
_I32 = torch.int32


def _fail(fn, msg):
    raise ValueError(f"{fn}: {msg}")


def _need_ints(fn, name, t, dim, dev):
    if t.dtype is not _I32 or t.dim() != dim or not t.is_contiguous() or t.get_device() != dev:
        _fail(fn, f"{name} must be a contiguous int32 tensor of {dim} dimension(s) on cuda:{dev}, got "
                  f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _explain(fn, rows, scales, block_table, ring_table, slots, cu_seqlens, ctx_lens):
    """Raises for the first thing wrong with a step's tensors."""
    _lib.require_gpu(fn, rows)
    if rows.dtype not in _FORMATS:
        raise TypeError(f"{fn}: rows must be bfloat16, float8_e4m3fn or int8, got {rows.dtype}")
    if rows.dim() != 3 or not rows.is_contiguous():
        _fail(fn, f"rows must be a contiguous [pages, page, c] tensor, got {tuple(rows.shape)}")
    dev = rows.get_device()
    if rows.dtype is not torch.bfloat16 and (
            scales is None or scales.dtype is not torch.uint8 or scales.shape != rows.shape[:2]
            or not scales.is_contiguous() or scales.get_device() != dev):
        _fail(fn, f"8-bit rows need scales, contiguous uint8 {tuple(rows.shape[:2])} on {rows.device}")
    _need_ints(fn, "block_table", block_table, 2, dev)
    if ring_table is not None:
        _need_ints(fn, "ring_table", ring_table, 2, dev)
        if ring_table.shape[0] != block_table.shape[0]:
            _fail(fn, f"ring_table has {ring_table.shape[0]} slots, block_table {block_table.shape[0]}")
    S = slots.shape[0] if slots.dim() else 0
    for name, t, n in (("slots", slots, S), ("cu_seqlens", cu_seqlens, S + 1), ("ctx_lens", ctx_lens, S)):
        if t is not None:
            _need_ints(fn, name, t, 1, dev)
            if t.shape[0] != n:
                _fail(fn, f"{name} has {t.shape[0]} entries for {S} sequences")
    raise AssertionError(fn)


def _step(fn, rows, scales, block_table, ring_table, slots, cu_seqlens, ctx_lens):
    """(format, device index, P, page, c, slots, block pages, ring pages, S) of a step after its
    checks. One expression over attributes of some 50 ns each, which a decode step pays
    per layer and call; what is wrong is looked for only where it fails."""
    i32 = _I32
    dev = rows.get_device()
    fmt = _FORMATS.get(rows.dtype, -1)
    S = -1
    if (fmt >= 0 and dev >= 0 and rows.dim() == 3 and rows.is_contiguous()
            and block_table.dtype is i32 and block_table.dim() == 2 and block_table.get_device() == dev
            and block_table.is_contiguous()
            and slots.dtype is i32 and slots.dim() == 1 and slots.get_device() == dev and slots.is_contiguous()
            and cu_seqlens.dtype is i32 and cu_seqlens.dim() == 1 and cu_seqlens.get_device() == dev
            and cu_seqlens.is_contiguous()):
        P, page, c = rows.shape
        n_slots, nbp = block_table.shape
        nrp = 0
        S, = slots.shape
        if (cu_seqlens.shape[0] != S + 1
                or (ctx_lens is not None and not (
                    ctx_lens.dtype is i32 and ctx_lens.dim() == 1 and ctx_lens.get_device() == dev
                    and ctx_lens.is_contiguous() and ctx_lens.shape[0] == S))
                or (fmt and (scales is None or scales.dtype is not torch.uint8 or scales.get_device() != dev
                             or not scales.is_contiguous() or scales.shape != (P, page)))):
            S = -1
        elif ring_table is not None:
            if (ring_table.dtype is i32 and ring_table.dim() == 2 and ring_table.get_device() == dev
                    and ring_table.is_contiguous()):
                m, nrp = ring_table.shape
                if m != n_slots:
                    S = -1
            else:
                S = -1
    if S < 0:
        _explain(fn, rows, scales, block_table, ring_table, slots, cu_seqlens, ctx_lens)
    return fmt, dev, P, page, c, n_slots, nbp, nrp, S


def _no_grad(fn, *ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise NotImplementedError(f"{fn}: no gradients (call it under torch.no_grad())")


def _rows2d(x):
    """``x`` ``[N, c]`` with 16-byte aligned rows, and their stride."""
    ld, one = x.stride()
    if one != 1 or (ld * x.element_size()) % 16 or x.data_ptr() % 16 or ld < x.shape[1]:
        x = x.detach().clone(memory_format=torch.contiguous_format)
        ld = x.shape[1]
    return x, ld


def _f32_rows(t, dev):
    """fp32, contiguous and 16-byte aligned on device ``dev``: ``t`` itself where it is (a copy
    is made on every call: keep such parameters in fp32)."""
    if t.dtype is torch.float32 and t.get_device() == dev and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return _aligned(_f32(t, torch.device("cuda", dev)))


def _p(t):
    return None if t is None else t.data_ptr()


def hca_paged_append(C, Z, B_pos, rows, scales, state, block_table, ring_table, slots, cu_seqlens,
                     ctx_lens, *, m2, max_len, normalize=True):
    """A chunk of tokens per sequence into the paged cache, in place.

    ``C, Z`` ``[N, c]`` the packed tokens' projections (rows may be strided views),
    ``B_pos [m2, c]``. Written: the compressed row of every block that the chunk
    ends, each token's window row (with a ``ring_table``), both L2-normalised
    (``normalize``) and quantised, and ``state`` where the chunk ends inside a
    block. ``max_len`` is at least the longest chunk and at most the ring's rows; a slot
    may occur once.
    """
    fn = "hca_paged_append"
    fmt, dev, P, page, c, n_slots, nbp, nrp, S = _step(fn, rows, scales, block_table, ring_table, slots,
                                                       cu_seqlens, ctx_lens)
    if C.dim() != 2 or C.shape != Z.shape or C.shape[1] != c or C.dtype is not Z.dtype \
            or C.get_device() != dev or Z.get_device() != dev:
        _lib.require_gpu(fn, C, Z)
        _fail(fn, f"C and Z must be [N, {c}] of one dtype on {rows.device}, got {tuple(C.shape)} {C.dtype} and "
                  f"{tuple(Z.shape)} {Z.dtype}")
    _no_grad(fn, C, Z, B_pos)
    if m2 < 1:
        _fail(fn, f"m2={m2} must be >= 1")
    if B_pos.shape != (m2, c):
        _fail(fn, f"B_pos.shape={tuple(B_pos.shape)} must equal (m2, c)=({m2}, {c})")
    if state.dtype is not torch.float32 or state.shape != (n_slots, 3, c) or not state.is_contiguous() \
            or state.get_device() != dev:
        _fail(fn, f"state must be contiguous float32 [{n_slots}, 3, {c}] on {rows.device}")
    if max_len < 0 or (nrp and max_len > nrp * page):
        _fail(fn, f"max_len={max_len} must be at most the ring's {nrp * page} rows")
    code = _lib.dtype_code(fn, C.dtype)
    C, ldc = _rows2d(C)
    Z, ldz = _rows2d(Z)
    B_pos = _f32_rows(B_pos, dev)
    _lib.call_on(dev, "kch_hca_paged_append", C.data_ptr(), ldc, Z.data_ptr(), ldz, B_pos.data_ptr(),
                 rows.data_ptr(), _p(scales), state.data_ptr(), block_table.data_ptr(), _p(ring_table),
                 slots.data_ptr(), cu_seqlens.data_ptr(), ctx_lens.data_ptr(), S, C.shape[0], c, m2, P, page,
                 nbp, nrp, n_slots, max_len, 1 if normalize else 0, fmt, code)


def hca_paged_attention(q, rows, scales, block_table, ring_table, slots, cu_seqlens, ctx_lens, *, m2,
                        sliding_window, max_len, max_ctx=None, sink_logits=None, scale=1.0,
                        normalize_q=True, out=None):
    """Attention of each sequence's chunk over its cache, which holds the chunk already.

    ``q`` ``[N, nh, c]`` the packed tokens' queries. The query at position p sees the
    compressed rows ``b < (p + 1) // m2`` and the window rows of positions
    ``max(0, p - sliding_window + 1) .. p`` in one softmax with the sink; 0 where it
    sees none. ``max_len`` is at least the longest chunk, ``max_ctx`` at least the largest
    of ``ctx_lens`` (it lays the work out). Returns ``[N, nh, c]`` in ``q.dtype``, or
    writes ``out``. Rows that no sequence answers are zeros, in ``out`` as they were: ahead of
    the first sequence and behind the last, of a longer chunk past ``max_len``, and of a
    sequence that is passed over (a slot outside the table, as a padding entry has it, a negative
    context, rows outside ``q``).
    The products are bf16 with fp32 sums, for fp16 ``q`` fp16: there a row with values past
    fp16's range reads as NaN. For fp32 ``q`` they take three bf16 parts, which keep fp32's accuracy.
    """
    fn = "hca_paged_attention"
    fmt, dev, P, page, c, n_slots, nbp, nrp, S = _step(fn, rows, scales, block_table, ring_table, slots,
                                                       cu_seqlens, ctx_lens)
    N, nh, width = q.shape if q.dim() == 3 else (0, 0, 0)
    if width != c or nh < 1 or q.get_device() != dev:
        _lib.require_gpu(fn, q)
        _fail(fn, f"q must be [N, nh, {c}] on {rows.device}, got {tuple(q.shape)} on {q.device}")
    _no_grad(fn, q, sink_logits)
    code = _lib.dtype_code(fn, q.dtype)
    if m2 < 1:
        _fail(fn, f"m2={m2} must be >= 1")
    if sliding_window < 0:
        _fail(fn, f"sliding_window={sliding_window} must be >= 0 (0 disables the branch)")
    if max_len < 0 or (sliding_window and sliding_window + max_len - 1 > nrp * page):
        _fail(fn, f"sliding_window={sliding_window} and max_len={max_len} need a ring of "
                  f"{sliding_window + max_len - 1} rows, it has {nrp * page}")
    if max_ctx is None:
        max_ctx = nbp * page * m2
    if max_ctx < 0:
        _fail(fn, f"max_ctx={max_ctx} must be >= 0")
    if max_ctx >= 2 ** 31:
        max_ctx = 2 ** 31 - 1
    if sink_logits is not None:
        if sink_logits.shape != (nh,):
            _fail(fn, f"sink_logits.shape={tuple(sink_logits.shape)} must equal (nh,)=({nh},)")
        sink_logits = _f32_rows(sink_logits, dev)
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = _aligned(q.detach())
    tail = 0
    if out is None:
        tail = 1
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != dev \
            or not out.is_contiguous() or out.data_ptr() % 16:
        _fail(fn, f"out must be a contiguous, 16-byte aligned {tuple(q.shape)} {q.dtype} tensor on {rows.device}")
    nbytes = (_lib._lib or _lib.load()).kch_hca_paged_attn_ws_bytes(S, N, nh, c, m2, sliding_window, max_len, max_ctx)
    ws = torch.empty(nbytes, device=rows.device, dtype=torch.uint8) if nbytes else None
    _lib.call_on(dev, "kch_hca_paged_attn", q.data_ptr(), _p(sink_logits), out.data_ptr(), rows.data_ptr(),
                 _p(scales), block_table.data_ptr(), _p(ring_table), slots.data_ptr(), cu_seqlens.data_ptr(),
                 ctx_lens.data_ptr(), S, N, nh, c, m2, sliding_window, P, page, nbp, nrp, n_slots, max_len,
                 max_ctx, scale, 1 if normalize_q else 0, tail, fmt, code, _p(ws), nbytes)
    return out


def paged_read(rows, scales, table, slots, cu_rows, *, total, first=None, dtype=torch.bfloat16, out=None):
    """Rows of a paged cache as numbers, packed: row ``cu_rows[i] + j`` of the result is
    row ``(first[i] + j) % capacity`` of slot ``slots[i]`` in ``table`` (a block or a ring
    table), capacity its pages times their rows. ``total`` is the number of result rows; those
    ahead of the first sequence and behind the last are zeros (in ``out`` as they were)."""
    fn = "paged_read"
    fmt, dev, P, page, c, n_slots, nbp, _, S = _step(fn, rows, scales, table, None, slots, cu_rows, first)
    if total < 0:
        _fail(fn, f"total={total} must be >= 0")
    tail = 0
    if out is None:
        tail = 1
        out = torch.empty(total, c, device=rows.device, dtype=dtype)
    elif out.shape != (total, c) or out.get_device() != dev or not out.is_contiguous() or out.data_ptr() % 16:
        _fail(fn, f"out must be a contiguous, 16-byte aligned [{total}, {c}] tensor on {rows.device}")
    code = _lib.dtype_code(fn, out.dtype)
    _lib.call_on(dev, "kch_paged_read", rows.data_ptr(), _p(scales), table.data_ptr(), slots.data_ptr(),
                 cu_rows.data_ptr(), _p(first), out.data_ptr(), S, total, c, P, page, nbp, n_slots, tail, fmt,
                 code)
    return out


class HCAPagedCache:
    """HCA decode state of a changing set of sequences over one pool of pages.

    ``add()`` opens a sequence and returns its slot, ``append_step`` takes a chunk of
    new tokens of some sequences, ``forward_step`` their queries, ``release`` gives a
    sequence's pages back. ``max_tokens`` bounds a sequence's length, ``max_chunk``
    the tokens a step takes of one. Widths between the kernels' own are held
    zero-padded. A single-threaded object on one stream, as the other caches; its steps'
    counts come from the host, so they cannot be captured into a graph (the operators
    over the same tensors can).
    """

    def __init__(self, n_pages, c, m2, win, *, max_seqs, max_tokens, max_chunk=1, page=64,
                 kv_dtype=torch.float8_e4m3fn, normalize_qk=True, device="cuda"):
        fn = "HCAPagedCache"
        for name, v, least in (("n_pages", n_pages, 1), ("c", c, 1), ("m2", m2, 1), ("win", win, 0),
                               ("max_seqs", max_seqs, 1), ("max_tokens", max_tokens, 1),
                               ("max_chunk", max_chunk, 1)):
            if v < least:
                _fail(fn, f"{name}={v} must be >= {least}")
        if page < 1 or page > 1024 or page & (page - 1):
            _fail(fn, f"page={page} must be a power of two up to 1024")
        if kv_dtype not in _FORMATS:
            raise TypeError(f"{fn}: kv_dtype must be bfloat16, float8_e4m3fn or int8, got {kv_dtype}")
        if max_tokens >= 2 ** 31:
            _fail(fn, f"max_tokens={max_tokens} must be below 2**31")
        self.c, self.m2, self.win, self.page = c, m2, win, page
        self.width = _kernel_size(fn, "c", c, _HEAD_DIMS)
        self.max_tokens, self.max_chunk = max_tokens, max_chunk
        self.normalize_qk = normalize_qk
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None and torch.cuda.is_available():
            self.device = torch.device("cuda", torch.cuda.current_device())
        nbp = -(-max(1, max_tokens // m2) // page)
        nrp = -(-(win + max_chunk - 1) // page) if win else 0
        kw = {"device": self.device}
        self.rows = torch.zeros(n_pages, page, self.width, dtype=torch.uint8 if kv_dtype != torch.bfloat16
                                else kv_dtype, **kw)
        if kv_dtype != torch.bfloat16:
            self.rows = self.rows.view(kv_dtype)
        self.scales = None if kv_dtype == torch.bfloat16 else \
            torch.full((n_pages, page), 127, dtype=torch.uint8, **kw)
        self.state = torch.zeros(max_seqs, 3, self.width, dtype=torch.float32, **kw)
        self.block_table = torch.full((max_seqs, nbp), -1, dtype=_I32, **kw)
        self.ring_table = torch.full((max_seqs, nrp), -1, dtype=_I32, **kw) if win else None
        self._free_pages = list(range(n_pages - 1, -1, -1))
        self._free_slots = list(range(max_seqs - 1, -1, -1))
        self._len = {}     # slot -> tokens cached
        self._pages = {}   # slot -> (ring pages, block pages)
        self._last = None  # the step that forward_step answers

    @property
    def n_free_pages(self) -> int:
        return len(self._free_pages)

    def n_tokens(self, slot) -> int:
        return self._len[self._slot("n_tokens", slot)]

    def n_blocks(self, slot) -> int:
        return self.n_tokens(slot) // self.m2

    def _slot(self, fn, slot):
        if slot not in self._len:
            _fail(f"HCAPagedCache.{fn}", f"slot {slot!r} holds no sequence")
        return slot

    def _eager(self, fn):
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"HCAPagedCache.{fn}: a graph would replay this step's counts; capture the operators "
                               f"hca_paged_append, hca_paged_attention and paged_read instead")

    def _upload(self, *lists):
        """int32 lists on the device, in one copy."""
        flat = [v for x in lists for v in x]
        t = torch.tensor(flat, dtype=_I32, pin_memory=True).to(self.device, non_blocking=True)
        return t.split([len(x) for x in lists])

    def _take(self, fn, n):
        if n > len(self._free_pages):
            raise RuntimeError(f"HCAPagedCache.{fn}: {n} pages needed, {len(self._free_pages)} are free")
        return [self._free_pages.pop() for _ in range(n)]

    def add(self) -> int:
        """Opens a sequence and returns its slot."""
        self._eager("add")
        if not self._free_slots:
            raise RuntimeError("HCAPagedCache.add: every slot holds a sequence")
        ring = self._take("add", 0 if self.ring_table is None else self.ring_table.shape[1])
        slot = self._free_slots.pop()
        if ring:
            self.ring_table[slot] = self._upload(ring)[0]
        self._len[slot], self._pages[slot] = 0, (ring, [])
        return slot

    def release(self, slot) -> None:
        """Ends a sequence: its pages and its slot are free again."""
        self._slot("release", slot)
        ring, blocks = self._pages.pop(slot)
        del self._len[slot]
        self._free_pages += ring + blocks
        self._free_slots.append(slot)
        if self._last is not None and slot in self._last[0]:
            self._last = None

    def append_step(self, slots, C_new, Z_new, B_pos, lens=None):
        """Appends ``lens[i]`` tokens (1 each by default) to sequence ``slots[i]``:
        ``C_new, Z_new`` ``[sum(lens), c]``, packed in that order."""
        fn = "append_step"
        self._eager(fn)
        _no_grad(f"HCAPagedCache.{fn}", C_new, Z_new, B_pos)
        slots = list(slots)
        lens = [1] * len(slots) if lens is None else list(lens)
        if len(lens) != len(slots) or len(set(slots)) != len(slots):
            _fail(f"HCAPagedCache.{fn}", "one length for each slot, and each slot once")
        need = {}
        for s, n in zip(slots, lens):
            self._slot(fn, s)
            if not 0 <= n <= self.max_chunk:
                _fail(f"HCAPagedCache.{fn}", f"a chunk of {n} tokens (max_chunk={self.max_chunk})")
            if self._len[s] + n > self.max_tokens:
                _fail(f"HCAPagedCache.{fn}", f"slot {s} would hold {self._len[s] + n} tokens "
                                             f"(max_tokens={self.max_tokens})")
            k = -(-((self._len[s] + n) // self.m2) // self.page) - len(self._pages[s][1])
            if k > 0:
                need[s] = k
        if C_new.dim() != 2 or C_new.shape != Z_new.shape or C_new.shape != (sum(lens), self.c):
            _fail(f"HCAPagedCache.{fn}", f"C_new and Z_new must be [{sum(lens)}, {self.c}], got "
                                         f"{tuple(C_new.shape)} and {tuple(Z_new.shape)}")
        _lib.require_gpu(f"HCAPagedCache.{fn}", C_new, Z_new)
        _lib.dtype_code(f"HCAPagedCache.{fn}", C_new.dtype)
        if tuple(B_pos.shape) != (self.m2, self.c):
            _fail(f"HCAPagedCache.{fn}", f"B_pos.shape={tuple(B_pos.shape)} must equal "
                                         f"({self.m2}, {self.c})")
        pages = self._take(fn, sum(need.values()))
        at = []
        for s, k in need.items():
            have = self._pages[s][1]
            at += [s * self.block_table.shape[1] + len(have) + i for i in range(k)]
            have += pages[len(at) - k:len(at)]
        ctx = [self._len[s] for s in slots]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        where, what, slots_d, cu_d, ctx_d = self._upload(at, pages, slots, cu, ctx)
        if at:
            self.block_table.view(-1)[where.long()] = what
        with torch.no_grad():
            hca_paged_append(_pad_last(C_new, self.width), _pad_last(Z_new, self.width),
                             _pad_last(B_pos, self.width), self.rows, self.scales, self.state,
                             self.block_table, self.ring_table, slots_d, cu_d, ctx_d, m2=self.m2,
                             max_len=max(lens, default=0), normalize=self.normalize_qk)
        for s, n in zip(slots, lens):
            self._len[s] += n
        self._last = (slots, slots_d, cu_d, ctx_d, cu[-1], max(lens, default=0), max(ctx, default=0))

    def forward_step(self, q, *, scale=None, sink_logits=None, normalize_q=None):
        """``[N, nh, c]`` in ``q.dtype``: the queries of the last ``append_step``'s tokens."""
        fn = "HCAPagedCache.forward_step"
        self._eager("forward_step")
        _no_grad(fn, q, sink_logits)
        if self._last is None:
            _fail(fn, "append_step first")
        _, slots, cu, ctx, n, max_len, max_ctx = self._last
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != self.c:
            _fail(fn, f"q must be [{n}, nh, {self.c}], got {tuple(q.shape)}")
        if scale is None:
            scale = 1.0 if self.normalize_qk else self.c ** -0.5
        with torch.no_grad():
            out = hca_paged_attention(
                _pad_last(q, self.width), self.rows, self.scales, self.block_table, self.ring_table, slots,
                cu, ctx, m2=self.m2, sliding_window=self.win, max_len=max_len, max_ctx=max_ctx,
                sink_logits=sink_logits, scale=scale,
                normalize_q=self.normalize_qk if normalize_q is None else normalize_q)
        return out if self.width == self.c else out[..., :self.c]

    def read_blocks(self, slot, dtype=torch.bfloat16):
        """The compressed rows ``[n_blocks, c]`` of a sequence."""
        self._eager("read_blocks")
        n = self.n_blocks(self._slot("read_blocks", slot))
        s, cu = self._upload([slot], [0, n])
        out = paged_read(self.rows, self.scales, self.block_table, s, cu, total=n, dtype=dtype)
        return out[:, :self.c]

    def read_window(self, slot, dtype=torch.bfloat16):
        """The window rows ``[min(win, tokens), c]`` of a sequence, oldest first."""
        self._eager("read_window")
        t = self.n_tokens(slot)
        n = min(self.win, t)
        if not n:
            return torch.empty(0, self.c, device=self.device, dtype=dtype)
        cap = self.ring_table.shape[1] * self.page
        s, cu, first = self._upload([slot], [0, n], [(t - n) % cap])
        out = paged_read(self.rows, self.scales, self.ring_table, s, cu, total=n, first=first, dtype=dtype)
        return out[:, :self.c]


__all__ = ["HCAPagedCache", "hca_paged_append", "hca_paged_attention", "paged_read"]

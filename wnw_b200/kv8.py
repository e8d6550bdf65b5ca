"""A paged key/value cache held in 8 bits, its append and its decode attention.

The cache holds ragged segments (one per sample and kv head, as the flat
cache's slots) in blocks of 32 tokens.  A full block's keys and values are
codes (e4m3 or int8) with one scale each, in pages that a page table maps; the
tokens of a block that is not full yet stay in the model's type.  A block is
quantised once, when it fills up, so a cache does not depend on whether its
tokens came one by one or together.

``KV8Store.append`` (``wnw_kv8_append``) adds tokens, rotating keys on the way
and, beside them, the same tokens' queries; ``KV8Attention``
(``wnw_kv8_attn``) attends one query token a segment.  Both read lengths on
the device, so a captured launch serves growing sequences.

No reference counterpart: the reference holds its cache in the model's type
(src/common/kv/flat_cache.py:45-54).
"""
from __future__ import annotations

import ctypes as C

import torch

from wnw_b200 import native as N
from wnw_b200.kernels import check_device_error
from wnw_b200.rotary import Apart, dense, distinct, keep_for, launch, made_on, plain, rows, written

BLOCK = N.KV8_BLOCK
_CONTIGUOUS = torch.contiguous_format
_CODES = {"e4m3": N.KV8_E4M3, "int8": N.KV8_INT8}


def check_layout(head_dim, page_rows, code):
    """Refuse what no store holds; returns the blocks of a page."""
    blocks = page_rows // BLOCK
    if page_rows % BLOCK or blocks < 1 or blocks & (blocks - 1) or blocks > 64:
        raise ValueError(f"page_rows {page_rows}: {BLOCK} times a power of two, up to {64 * BLOCK}")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim {head_dim}: 64 or 128")
    if code not in _CODES:
        raise ValueError(f"code {code!r}: one of {sorted(_CODES)}")
    return blocks


def check_group(group):
    if not 1 <= int(group) <= 8:
        raise ValueError(f"group {group}: 1 to 8 query heads a kv head")


class KV8Store:
    """One layer's cache: pool, page table and unfinished blocks.

    ``page_rows`` tokens a page (32 times a power of two, up to 2048),
    ``num_pages`` pages in the pool, ``max_pages`` pages a segment.  Pages are
    handed out by ``reserve`` (or written into ``page_table`` by the caller;
    no two segments may share a page that is still appended to).  Lengths
    belong to the caller: ``append`` and the attention take them.  Appends to
    one store must be ordered (one stream, or events), as must a store's or a
    handle's making and its first use on another stream."""

    def __init__(self, num_segs, head_dim, num_pages, max_pages, page_rows=128, code="e4m3", dtype=torch.bfloat16,
                 device="cuda"):
        blocks = check_layout(head_dim, page_rows, code)
        device = torch.device(device)
        self._init(torch.zeros(num_pages, blocks, 2 * BLOCK * head_dim + N.KV8_PAD, dtype=torch.uint8, device=device),
                   torch.full((num_segs, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(num_segs, 2, BLOCK, head_dim, dtype=dtype, device=device),
                   torch.zeros(num_segs, 2, head_dim, BLOCK, dtype=dtype, device=device), code)
        self._free = list(range(num_pages - 1, -1, -1))
        self._owned = [[] for _ in range(num_segs)]

    @classmethod
    def wrap(cls, pool, page_table, tail_k, tail_v, code="e4m3"):
        """A store over the caller's memory (whose pages the caller manages)."""
        s = cls.__new__(cls)
        s._init(pool, page_table, tail_k, tail_v, code)
        s._free = s._owned = None
        return s

    def _init(self, pool, page_table, tail_k, tail_v, code):
        if code not in _CODES:
            raise ValueError(f"code {code!r}: one of {sorted(_CODES)}")
        if tail_k.dim() != 4 or tail_k.shape[1:3] != (2, BLOCK) or tail_k.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"tail_k {tuple(tail_k.shape)} {tail_k.dtype}: expected [segments, 2, {BLOCK}, D] in "
                             "bf16 or fp16")
        S, _, _, D = tail_k.shape
        if tail_v.shape != (S, 2, D, BLOCK) or tail_v.dtype != tail_k.dtype:
            raise ValueError(f"tail_v {tuple(tail_v.shape)} {tail_v.dtype}: expected {(S, 2, D, BLOCK)} {tail_k.dtype}")
        if D not in (64, 128):
            raise ValueError(f"head_dim {D}: 64 or 128")
        if pool.dim() != 3 or pool.dtype != torch.uint8 or pool.shape[2] != 2 * BLOCK * D + N.KV8_PAD:
            raise ValueError(f"pool {tuple(pool.shape)} {pool.dtype}: expected uint8 "
                             f"[pages, page rows / {BLOCK}, {2 * BLOCK * D + N.KV8_PAD}]")
        if page_table.dim() != 2 or page_table.shape[0] != S or page_table.dtype != torch.int32:
            raise ValueError(f"page_table {tuple(page_table.shape)} {page_table.dtype}: expected int32 [{S}, pages]")
        for t in (pool, page_table, tail_k, tail_v):
            if not t.is_contiguous() or t.device != pool.device:
                raise ValueError("pool, page_table and tails must be contiguous, on one device")
        self.pool, self.page_table, self.tail_k, self.tail_v, self.code = pool, page_table, tail_k, tail_v, code
        self.num_segs, self.head_dim, self.dtype, self.device = S, D, tail_k.dtype, pool.device
        self.page_rows = pool.shape[1] * BLOCK
        self._index = pool.get_device()
        self._appends = {}  # argument blocks by geometry
        self._held = pool, tail_k, tail_v  # what an append writes
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._desc = N.Kv8StoreDesc(N.dtype_code(self.dtype), D, _CODES[code], S, pool.data_ptr(), pool.shape[0],
                                    pool.shape[1], page_table.data_ptr(), page_table.shape[1], tail_k.data_ptr(),
                                    tail_v.data_ptr(), self.err.data_ptr())

    # ------------------------------------------------------------- pages
    def reserve(self, rows):
        """Pages for ``rows`` tokens of every segment (a number, or one per
        segment); raises, changing nothing, when the pool or the table is too
        small.  Host bookkeeping plus one upload where pages were added."""
        if self._free is None:
            raise RuntimeError("the pages of a wrapped store are the caller's")
        need = [int(r) for r in rows] if hasattr(rows, "__iter__") else [int(rows)] * self.num_segs
        if len(need) != self.num_segs:
            raise ValueError(f"{len(need)} row counts for {self.num_segs} segments")
        want = [max(0, -(-r // self.page_rows) - len(own)) for r, own in zip(need, self._owned)]
        if max(len(o) + w for o, w in zip(self._owned, want)) > self.page_table.shape[1]:
            raise ValueError(f"a segment of {max(need)} rows does not fit its {self.page_table.shape[1]} pages of "
                             f"{self.page_rows}")
        if sum(want) > len(self._free):
            raise ValueError(f"{sum(want)} pages wanted, {len(self._free)} free")
        if not any(want):
            return
        at, pages = [], []
        for s, n in enumerate(want):
            for _ in range(n):
                at.append(s * self.page_table.shape[1] + len(self._owned[s]))
                self._owned[s].append(self._free.pop())
                pages.append(self._owned[s][-1])
        where = torch.tensor([at, pages], dtype=torch.int64).to(self.device)
        self.page_table.view(-1)[where[0]] = where[1].to(torch.int32)

    def release(self, segs=None):
        """Give the pages of ``segs`` (all: None) back to the pool."""
        if self._free is None:
            raise RuntimeError("the pages of a wrapped store are the caller's")
        for s in range(self.num_segs) if segs is None else segs:
            self._free.extend(reversed(self._owned[s]))
            self._owned[s] = []
            self.page_table[s].fill_(-1)

    def grown(self, rows):
        """A store with this one's content, and pages for ``rows`` tokens of
        every segment (the unfinished blocks are shared, and the pool where it
        has pages enough: use the new one)."""
        if self._free is None:
            raise RuntimeError("the pages of a wrapped store are the caller's")
        S, width, have = self.num_segs, -(-int(rows) // self.page_rows), self.pool.shape[0]
        more = max(0, sum(max(0, width - len(o)) for o in self._owned) - len(self._free))
        pool = torch.cat([self.pool, self.pool.new_zeros(more, *self.pool.shape[1:])]) if more else self.pool
        table = self.page_table.new_full((S, max(width, self.page_table.shape[1])), -1)
        table[:, :self.page_table.shape[1]] = self.page_table
        s = KV8Store.wrap(pool, table, self.tail_k, self.tail_v, self.code)
        s._free = list(range(have + more - 1, have - 1, -1)) + self._free
        s._owned = [list(o) for o in self._owned]
        s.err, s._desc.err = self.err, self.err.data_ptr()
        s.reserve(rows)
        return s

    # ------------------------------------------------------------ append
    def append(self, k, v, seg_len, *, starts=None, counts=None, max_count=None, q=None, rotary=None, positions=None,
               q_out=None, stream=None):
        """Append tokens behind every segment's ``seg_len`` rows (int32
        [segments], on the device; the caller advances it).

        k, v [B, kv heads, n, D] in the model's type, rows contiguous, other
        dimensions of any stride that is a multiple of 8 elements (0 too: packed
        ragged tokens [total, heads, D] are passed as one expanded batch).
        ``starts`` / ``counts`` (int32 [B], on the device): sample b's tokens
        are starts[b] ... starts[b] + counts[b] of the n, ``max_count`` (host)
        at least the largest count.  ``rotary`` (a ``Rotary``) with
        ``positions`` [axes, B, n] rotates the keys before they are held, and
        ``q`` [B, q heads, n, D] into the returned tensor: ``q_out``, which may
        be q and shares no memory with k and v, or a new one, contiguous.
        Where a sample has no token a new one is zero and a given one is left
        as it is.  Of packed tokens a new one is as large as B times all
        tokens; a given one may be packed too, one expanded batch, where the
        samples' tokens are apart from one another.  Returns None without q.
        ``stream``: launch there, behind what the caller made it wait for.
        Problems on the device (a segment beyond its pages, an index out of
        range) set bits that ``check()`` reads back.  Not differentiable, like
        the attention."""
        # the checks and the argument block depend on shapes, strides, types and
        # the rotation alone: each geometry is looked at once, a call brings its
        # pointers
        key = (k.shape, k.stride(), v.shape, v.stride(), k.dtype, v.dtype, counts is None, max_count, rotary,
               None if q is None else (q.shape, q.stride(), q.dtype),
               None if q_out is None else (q_out.shape, q_out.stride(), q_out.dtype),
               None if positions is None else (positions.shape, positions.stride(), positions.dtype))
        base = self._appends.get(key)
        if base is None:
            base = self._append_args(k, v, counts is not None, max_count, q, rotary, positions, q_out)
            if len(self._appends) >= 64:
                self._appends.clear()
            self._appends[key] = base
        given = q_out is not None
        if given:
            plain(q_out)
            base[2](q_out.data_ptr(), q.data_ptr(), None, k.data_ptr(), None, v.data_ptr())
        index = self._index
        if index < 0 or k.get_device() != index or v.get_device() != index:
            self._check_device(k, v)
        lengths = _lengths(seg_len, self.num_segs, "seg_len", index)
        first = many = pos = q_in = q_to = None
        if counts is not None:
            many = _lengths(counts, k.shape[0], "counts", index)
            if starts is not None:
                first = _lengths(starts, k.shape[0], "starts", index)
        elif starts is not None or (max_count is not None and max_count != k.shape[2]):
            raise ValueError("starts and max_count go with counts")
        if positions is not None:
            if positions.get_device() != index:
                self._check_device(positions)
            pos = positions.data_ptr()
        if q is not None:
            if q.get_device() != index:
                self._check_device(q)
            if q_out is None:
                make = torch.empty_like if counts is None else torch.zeros_like
                q_out = made_on(stream, index, make, q, memory_format=_CONTIGUOUS)
            elif q_out.get_device() != index:
                self._check_device(q_out)
            q_in, q_to = q.data_ptr(), q_out.data_ptr()
        launch(index, stream, _APPEND, "wnw_kv8_append_step", base[1], k.data_ptr(), v.data_ptr(), lengths, first, many,
               pos, q_in, q_to)
        written(self._held if not given else (*self._held, q_out))
        if stream is not None:
            keep_for(stream, k, v, seg_len, starts, counts, positions, q, q_out, *self._tensors())
            if rotary is not None:
                keep_for(stream, rotary._freq64, rotary.axis)
        return q_out

    def _append_args(self, k, v, ragged, max_count, q, rotary, positions, q_out):
        """(argument block without pointers, a reference to it, the check of a
        given output's address) of one append geometry, checked."""
        shape, dtype = k.shape, self.dtype
        if len(shape) != 4 or v.shape != shape or k.dtype != dtype or v.dtype != dtype:
            raise ValueError(f"k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype}: expected "
                             f"[B, kv heads, n, {self.head_dim}] {self.dtype}")
        B, H, n, D = shape
        if B * H != self.num_segs or D != self.head_dim:
            raise ValueError(f"k {tuple(shape)} does not fit {self.num_segs} segments of head_dim {self.head_dim}")
        max_count = n if max_count is None or not ragged else int(max_count)
        max_count = max(-1, min(max_count, n + 1))  # (either is refused by the launch; neither wraps around)
        rope, queries = _NO_ROPE, _NO_QUERIES
        if rotary is not None and positions is not None:
            if rotary.rot_dim > D or rotary.device != self.device:
                raise ValueError(f"{rotary.rot_dim} rotated dimensions on {rotary.device} in heads of {D} on "
                                 f"{self.device}")
            rope = rotary.rope(positions, B, n)
        elif rotary is not None or positions is not None:
            raise ValueError("rotary and positions go together")
        if q is not None:
            if rotary is None:
                raise ValueError("q is rotated: rotary and positions are needed")
            qs = q.shape
            if len(qs) != 4 or qs[0] != B or qs[2] != n or qs[3] != D or qs[1] % H or not qs[1] or q.dtype != dtype:
                raise ValueError(f"q {tuple(qs)} {q.dtype} does not go with k {tuple(shape)} {k.dtype}")
            if q_out is None:
                to = (None, *dense(qs))
            elif q_out.shape != qs or q_out.dtype != dtype:
                raise ValueError(f"q_out {tuple(q_out.shape)} {q_out.dtype}: expected {tuple(qs)} {dtype}")
            else:
                to = rows(q_out, "q_out", qs)
                packed = ragged and B > 1 and q_out.stride(0) == 0
                distinct(q_out[:1] if packed else q_out, "q_out")
            queries = (qs[1] // H, *rows(q, "q", qs), *to)
        elif q_out is not None:
            raise ValueError("q_out without q")
        a = N.Kv8AppendArgs(self._desc, B, H, n, max_count, None, None, None, *rows(k, "k", shape),
                            *rows(v, "v", shape), *queries, rope)
        return a, C.byref(a), None if q_out is None else Apart(("q_out", q_out, q), ("k", None, k), ("v", None, v))

    def _tensors(self):
        return self.pool, self.page_table, self.tail_k, self.tail_v, self.err

    def _check_device(self, *tensors):
        index = self._index
        for t in tensors:
            if t.get_device() != index or index < 0:
                raise ValueError(f"a tensor on {t.device}: the store is on {self.device} and needs a CUDA device")

    # ---------------------------------------------------------- inspection
    def codes(self):
        """(keys, values): the pool's codes as numbers (float8_e4m3fn or int8),
        [pages, blocks, D / 64, 32, 64] and [pages, blocks, D, 32]; views."""
        t = torch.float8_e4m3fn if self.code == "e4m3" else torch.int8
        c = self.pool[..., :2 * BLOCK * self.head_dim].view(t)
        h = BLOCK * self.head_dim
        return (c[..., :h].unflatten(-1, (self.head_dim // 64, BLOCK, 64)),
                c[..., h:].unflatten(-1, (self.head_dim, BLOCK)))

    def scales(self):
        """[pages, blocks, 2] fp32 (keys, values); a view."""
        h = 2 * BLOCK * self.head_dim
        return self.pool[..., h:h + 8].view(torch.float32)

    def dequantize(self, seg, rows):
        """The first ``rows`` tokens of a segment as they read back: (keys,
        values) fp32 [rows, D] (torch operations, for inspection)."""
        nb, left = divmod(int(rows), BLOCK)
        per = self.page_rows // BLOCK
        j = torch.arange(nb, device=self.device)
        page = self.page_table[seg].long()[j // per]
        k, v = self.codes()
        k, v, s = k[page, j % per], v[page, j % per], self.scales()[page, j % per]
        k = (k.float().transpose(1, 2).flatten(2) * s[:, :1, None]).flatten(0, 1)
        v = (v.float().transpose(1, 2) * s[:, 1:, None]).flatten(0, 1)
        tk, tv = self.tail_k[seg, nb % 2, :left].float(), self.tail_v[seg, nb % 2, :, :left].t().float()
        return torch.cat([k, tk]), torch.cat([v, tv])

    def check(self):
        """Raise if a launch set the device error word (a sync point)."""
        check_device_error(self.err)


class KV8Attention:
    """Decode attention over a ``KV8Store`` for ``group`` query heads a kv head
    (1..8), with its scratch.  Calls through one handle must not run at the
    same time (two streams, or two captured graphs that may be replayed side
    by side, need a handle each: ``KV8Attention(store, ...)`` again); with
    ``scratch_of`` a handle shares another's scratch, for calls that are
    ordered anyway (the layers of a model)."""

    def __init__(self, store, group, scale, scratch_of=None):
        check_group(group)
        self.store, self.group, self.scale = store, int(group), float(scale)
        if store.device.type != "cuda":
            raise ValueError(f"the store is on {store.device}: a CUDA device is needed")
        if scratch_of is not None:
            o = scratch_of.store
            if (o.device, o.head_dim, scratch_of.group) != (store.device, store.head_dim, self.group) \
                    or o.num_segs < store.num_segs:
                raise ValueError("scratch of another device, head_dim, group or of fewer segments")
            self._finish(scratch_of.partials, scratch_of.counters)
            return
        n = C.c_int64()
        with torch.cuda.device(store.device):
            N.call("wnw_kv8_attn_scratch", store.head_dim, self.group, C.byref(n))
        self._finish(torch.empty(n.value, dtype=torch.float32, device=store.device),
                     torch.zeros(store.num_segs, N.KV8_COUNTER_STRIDE, dtype=torch.int32, device=store.device))

    def _finish(self, partials, counters):
        store = self.store
        self.partials, self.counters = partials, counters
        self.shape = (store.num_segs, self.group, store.head_dim)
        # what no call changes; each gives its own pointers beside it
        self._base = N.Kv8AttnArgs(store._desc, self.group, None, None, None, None, self.scale,
                                   self.partials.data_ptr(), self.partials.numel(), self.counters.data_ptr(), -1)
        self._args = C.byref(self._base)
        self._bytes = store.num_segs * self.group * store.head_dim * store.tail_k.element_size()
        self._lse_like = torch.empty(self.shape[:2], dtype=torch.float32, device=store.device)

    def __call__(self, q, seg_len, *, out=None, return_lse=False, fresh=None, stream=None):
        """Attend q [segments, group, D] (the model's type, contiguous) over
        each segment's seg_len (int32 [segments], device) rows: as many as
        were appended, or fewer by whole blocks (a block that is full is no
        longer held in 16 bits, so no length may end inside one); returns
        ``out`` like q, and with ``return_lse`` the natural log-sum-exp
        [segments, group] in fp32.  A segment without rows gives zeros and -inf.

        ``fresh`` (optional) says what the kernel directly before this call
        on its stream may still be doing: appending at most that many tokens
        to each segment, and not touching lengths or page table.  The call
        then streams the older blocks while that kernel finishes.  Leave it
        out wherever anything else may precede the call."""
        s, shape = self.store, self.shape
        if q.shape != shape or q.dtype is not s.dtype or not q.is_contiguous() or q.get_device() != s._index:
            raise ValueError(f"q {tuple(q.shape)} {q.dtype} on {q.device}: expected contiguous {shape} {s.dtype} on "
                             f"{s.device}")
        lengths = _lengths(seg_len, s.num_segs, "seg_len", s._index)
        if fresh is None:
            fresh = -1
        elif not 0 <= fresh < 1 << 31:
            raise ValueError(f"fresh {fresh}: a number of tokens")
        given = out
        if out is None:
            out = made_on(stream, s._index, torch.empty_like, q)
        elif out.shape != shape or out.dtype is not s.dtype or not out.is_contiguous() \
                or out.get_device() != s._index:
            raise ValueError(f"out {tuple(out.shape)} {out.dtype}: expected contiguous {shape} {s.dtype}")
        else:
            plain(out)
            if 0 < abs(out.data_ptr() - q.data_ptr()) < self._bytes:
                raise ValueError("out: shares memory with other rows of q")
        lse = made_on(stream, s._index, torch.empty_like, self._lse_like) if return_lse else None
        launch(s._index, stream, _ATTEND, "wnw_kv8_attn_step", self._args, q.data_ptr(), lengths, out.data_ptr(),
               lse.data_ptr() if return_lse else None, fresh)
        if given is not None:
            written((given,))
        if stream is not None:
            keep_for(stream, q, seg_len, out, lse, self.partials, self.counters, *s._tensors())
        return (out, lse) if return_lse else out


_NO_ROPE = N.Rope()
_NO_QUERIES = (0,) + (None, 0, 0, 0) * 2


_APPEND, _ATTEND = N.lib.wnw_kv8_append_step, N.lib.wnw_kv8_attn_step


def _lengths(t, n, name, index):
    """Address of int32 [n] on device ``index``, checked."""
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} {tuple(t.shape)} {t.dtype}: expected contiguous int32 [{n}]")
    if t.get_device() != index:
        raise ValueError(f"{name} on {t.device}: the store is on CUDA device {index}")
    return t.data_ptr()

"""A key/value cache in pages for several sequences, and the operators of decoding over it (include/qmm.h):

* ``PagedKVCache.append``     -- RoPE of a step's rows and their append            (qmm_kv_append)
* ``PagedKVCache.attention``  -- attention of tokens, runs or drafted trees        (qmm_kv_attention)
* ``PagedKVCache.fork``       -- sequences continued, shared, cut, freed; reserves (qmm_kv_fork)
* ``PagedKVCache.accept``     -- the accepted rows of a drafted tree               (qmm_kv_accept)
* ``PagedKVCache.compact``    -- the pool packed to its lowest pages               (qmm_kv_compact)
* ``beam_select``, ``reorder_rows`` -- a beam search's selection                   (qmm_beam_select, qmm_reorder_rows)

A beam step: fork (reserve=1), per layer append and attention, accept of one row, beam_select, and fork again with
its parents. A speculative step: fork (reserve=nodes), per layer append with depths and attention with masks,
accept with the paths that the verifier kept. Nothing is read back to the host, so a step can be captured.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence, Tuple

import torch

from .qmm import _DENSE, QMM_ERR_INVALID, QMM_OK, QmmError, _call, _device_of, _ptr, _raw_stream, last_error, lib


class _Cache(ctypes.Structure):  # qmm_kv_cache
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("table", ctypes.c_void_p), ("lens", ctypes.c_void_p),
                ("refs", ctypes.c_void_p), ("pages", ctypes.c_int64), ("dtype", ctypes.c_int), ("layers", ctypes.c_int),
                ("kv_heads", ctypes.c_int), ("page_size", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("slots", ctypes.c_int), ("max_pages", ctypes.c_int)]


def _bad(message: str) -> QmmError:
    return QmmError(QMM_ERR_INVALID, message)


def _ints(t: torch.Tensor, shape: Tuple[int, ...], dev: torch.device, what: str) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.device != dev or t.shape != shape or not t.is_contiguous():
        raise _bad(f"{what} must be contiguous int32 {list(shape)} on {dev}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t


def _within(v: int, low: int, high: int, what: str) -> int:
    """v, which a C int would cut off without a word."""
    if not low <= v <= high:
        raise _bad(f"{what} {v} ({low} .. {high})")
    return v


def _kept(sizes: dict, key, size: int) -> int:
    """A workspace size kept under its arguments (a thousand of them)."""
    if len(sizes) >= 1024:
        sizes.clear()
    sizes[key] = size
    return size


def _packed(t: torch.Tensor) -> bool:
    """Whether t's rows (along the first dimension) are contiguous and do not overlap."""
    if t.is_contiguous():
        return True
    n = 1
    for size, stride in zip(t.shape[:0:-1], t.stride()[:0:-1]):
        if stride != n and size != 1:
            return False
        n *= size
    return t.shape[0] <= 1 or t.stride(0) >= n


# The current device's index, which torch.cuda.current_device looks up behind a check of its own.
_device_now = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _run(dev: torch.device, fn, *args) -> None:
    index = dev.index
    status = fn(*args, _raw_stream(index)) if _device_now() == index else _call(dev, fn, *args)
    if status != QMM_OK:
        raise QmmError(status, last_error())


def tree_masks(parents: Sequence[Sequence[int]], words: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Masks and depths (on the host) of drafted trees for PagedKVCache.attention and .append: parents[s][j] is the
    node above node j of sequence s, before it in the list, or -1 for the sequence's text. A node sees itself and
    the nodes above it. masks: int64 [rows, words] (bit i % 64 of word i / 64: row i), depths: int32 [rows]."""
    most = max((len(seq) for seq in parents), default=0)
    words = max(1, -(-most // 64)) if words is None else words
    if words * 64 < most:
        raise _bad(f"trees of {most} nodes need {-(-most // 64)} mask words")
    masks: List[int] = []
    depths: List[int] = []
    for seq in parents:
        m: List[int] = []
        d: List[int] = []
        for j, p in enumerate(seq):
            if not -1 <= p < j:
                raise _bad(f"node {j}'s parent {p} is not before it")
            m.append((m[p] if p >= 0 else 0) | 1 << j)
            d.append(d[p] + 1 if p >= 0 else 0)
        masks += m
        depths += d
    low = (1 << 64) - 1
    bits = [[(v >> 64 * w & low) - ((v >> 64 * w & 1 << 63) << 1) for w in range(words)] for v in masks]
    return torch.tensor(bits, dtype=torch.int64).reshape(-1, words), torch.tensor(depths, dtype=torch.int32)


class PagedKVCache:
    """Keys and values of several sequences in pages that they may share, on one GPU.

    k, v: [layers, pages, kv_heads, page_size, head_dim] (float32, float16 or bfloat16); table: int32 [slots,
    max_pages] of page ids (-1: none); lens: int32 [slots]; refs: int32 [pages], how many table entries name each
    page. All are the caller's tensors, contiguous; ``empty`` makes them. page_size: a power of two, 16..1024;
    head_dim 64, 128 or 256.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor):
        dev = _device_of(k)
        if k.dim() != 5 or k.dtype not in _DENSE or not k.is_contiguous():
            raise _bad(f"k must be contiguous [layers, pages, kv_heads, page_size, head_dim] in float32, float16 or "
                       f"bfloat16, got {k.dtype} {list(k.shape)}")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != dev or not v.is_contiguous():
            raise _bad(f"v must be like k, got {v.dtype} {list(v.shape)} on {v.device}")
        if table.dim() != 2:
            raise _bad(f"table must be [slots, max_pages], got {list(table.shape)}")
        slots, max_pages = table.shape
        layers, pages, kv_heads, page_size, head_dim = k.shape
        _ints(table, (slots, max_pages), dev, "table")
        _ints(lens, (slots,), dev, "lens")
        _ints(refs, (pages,), dev, "refs")
        self._tensors, self.device = (k, v, table, lens, refs), dev
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = layers, pages, kv_heads, page_size, head_dim
        self.slots, self.max_pages, self._starts = slots, max_pages, (slots + 1,)
        self._c = _Cache(k.data_ptr(), v.data_ptr(), table.data_ptr(), lens.data_ptr(), refs.data_ptr(), pages,
                         _DENSE[k.dtype], layers, kv_heads, page_size, head_dim, slots, max_pages)
        self._p = ctypes.addressof(self._c)
        self._sizes: dict = {}  # workspace sizes of attention calls by their host arguments
        self._fork_ws = int(lib().qmm_kv_fork_workspace_size(self._p))
        if self._fork_ws == 0:
            raise _bad("paged cache: " + last_error())
        self._compact_ws = int(lib().qmm_kv_compact_workspace_size(self._p))

    # (fixed: the library has their addresses)
    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    table = property(lambda self: self._tensors[2])
    lens = property(lambda self: self._tensors[3])
    refs = property(lambda self: self._tensors[4])

    @classmethod
    def empty(cls, layers: int, pages: int, kv_heads: int, page_size: int, head_dim: int, slots: int, max_pages: int,
              dtype: torch.dtype = torch.float32, device: Optional[torch.device] = None) -> "PagedKVCache":
        """A cache whose slots are empty and whose pages are free."""
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        shape = (layers, pages, kv_heads, page_size, head_dim)
        zeros = dict(dtype=torch.int32, device=dev)
        return cls(torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev),
                   torch.full((slots, max_pages), -1, **zeros), torch.zeros(slots, **zeros), torch.zeros(pages, **zeros))

    # -- a step's rows ----------------------------------------------------
    def _rows(self, x: torch.Tensor, heads: Optional[int], what: str) -> Tuple[torch.Tensor, int]:
        """x as rows [rows, heads, head_dim] whose heads are contiguous, and the row stride."""
        # (the usual case first: a token's calls are as long as their checks)
        shape = x.shape
        if len(shape) == 3 and shape[2] == self.head_dim and (heads is None or shape[1] == heads) and \
                x.device == self.device and x.dtype in _DENSE and x.is_contiguous():
            return x, shape[1] * shape[2]
        if x.device != self.device or x.dtype not in _DENSE:
            raise _bad(f"{what} must be float32, float16 or bfloat16 on {self.device}, got {x.dtype} on {x.device}")
        dim = self.head_dim
        if x.dim() == 2 and x.shape[1] % dim == 0:
            x = x.unflatten(1, (-1, dim))
        if x.dim() != 3 or x.shape[2] != dim or (heads is not None and x.shape[1] != heads):
            raise _bad(f"{what} must be [rows, {heads or 'heads'}, {dim}], got {list(x.shape)}")
        if x.stride(2) != 1 or (x.shape[1] > 1 and x.stride(1) != dim) or (x.shape[0] > 1 and x.stride(0) < x.shape[1] * dim):
            x = x.contiguous()
        return x, x.stride(0) if x.shape[0] > 1 else x.shape[1] * dim

    def _out(self, out: Optional[torch.Tensor], q: torch.Tensor) -> Tuple[torch.Tensor, int]:
        """Rows for a result like q (`out`, or new ones), and their stride."""
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)
            return out, q.shape[1] * q.shape[2]
        o, ld = self._rows(out, q.shape[1], "out")
        if o.data_ptr() != out.data_ptr() or out.dtype != q.dtype or o.shape != q.shape:
            raise _bad(f"out must be rows like q, got {list(out.shape)} {out.dtype}")
        return out, ld

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
               q: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None, depths: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Rotates a step's rows and appends their keys and values to the layer, into pages that are the slot's alone
        (see ``fork``'s reserve); returns the rotated q (`out`, which may be q, or a new tensor). k, v: [rows, kv_heads,
        head_dim], q: [rows, heads, head_dim], one type. Sequence s has rows starts[s] .. starts[s + 1] - 1 (int32
        [slots + 1]) at cache positions lens[s], lens[s] + 1, ...; row j is rotated at lens[s] + depths[row] (default:
        + j) by cos / sin (float32 [positions, head_dim]; None: not rotated). Rows of no sequence and rows at positions
        past the tables are not written: a padded batch brings its own `out`. lens stays as it is: see ``accept``."""
        dev = self.device
        if not 0 <= layer < self.layers:
            raise _bad(f"layer {layer} of {self.layers}")
        k, ldk = self._rows(k, self.kv_heads, "k")
        v, ldv = self._rows(v, self.kv_heads, "v")
        rows = k.shape[0]
        if v.shape[0] != rows or v.dtype != k.dtype:
            raise _bad(f"k and v must be rows of one type, got {list(k.shape)} {k.dtype}, {list(v.shape)} {v.dtype}")
        _ints(starts, self._starts, dev, "starts")
        if depths is not None:
            _ints(depths, (rows,), dev, "depths")
        positions = 0
        if (cos is None) != (sin is None):
            raise _bad("cos and sin go together")
        if cos is not None:
            positions = cos.shape[0]
            shape = (positions, self.head_dim)
            for t in (cos, sin):
                if t.shape != shape or t.dtype is not torch.float32 or t.device != dev or not t.is_contiguous():
                    raise _bad(f"cos and sin must be contiguous float32 [positions, {self.head_dim}] on {dev}")
        ldq = ldo = heads = 0
        if q is not None:
            q, ldq = self._rows(q, None, "q")
            heads = q.shape[1]
            if q.shape[0] != rows or q.dtype != k.dtype:
                raise _bad(f"q must be rows like k, got {list(q.shape)} {q.dtype}")
            out, ldo = self._out(out, q)
        elif out is not None:
            raise _bad("an output without q")
        _run(dev, lib().qmm_kv_append, self._p, layer, _ptr(q), k.data_ptr(), v.data_ptr(), _DENSE[k.dtype], rows, ldq,
             ldk, ldv, starts.data_ptr(), _ptr(depths), _ptr(cos), _ptr(sin), positions, _ptr(out), ldo, heads)
        return out

    def attention(self, layer: int, q: torch.Tensor, starts: torch.Tensor, masks: Optional[torch.Tensor] = None,
                  max_rows: Optional[int] = None, max_len: Optional[int] = None, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(q . K^T * scale) . V of a step's rows (rotated, their keys and values appended) over their own
        sequences: row j of sequence s sees the positions below lens[s], and lens[s] + i where bit i of its mask is
        set (int64 [rows, words], see tree_masks; None: i <= j). q: [rows, heads, head_dim]; the result is of its
        shape and type, a row that sees nothing is zeros (rows of no sequence are not written: a padded batch brings
        its own `out`, which may be q). max_rows bounds a sequence's rows (at most 64 * words with masks; rows past it are
        not written; default: all, or as many as the masks have bits, and rows past those are zeros in a new result),
        max_len is about the longest lens + rows (default: the table's). scale: head_dim ** -0.5."""
        dev = self.device
        if not 0 <= layer < self.layers:
            raise _bad(f"layer {layer} of {self.layers}")
        q, ldq = self._rows(q, None, "q")
        rows, heads = q.shape[0], q.shape[1]
        _ints(starts, self._starts, dev, "starts")
        ldm = 0
        if masks is not None:
            if masks.dtype != torch.int64 or masks.device != dev or masks.dim() != 2 or masks.shape[0] != rows or \
                    not masks.is_contiguous():
                raise _bad(f"masks must be contiguous int64 [{rows}, words] on {dev}, got {masks.dtype} "
                           f"{list(masks.shape)} on {masks.device}")
            ldm = masks.shape[1]
        given = max_rows
        max_rows = max(1, rows) if given is None else min(given, max(1, rows))
        most = self.max_pages * self.page_size
        max_len = most if max_len is None else min(max_len, most)
        if max_rows < 1 or max_len < 1:
            raise _bad(f"max_rows {max_rows}, max_len {max_len}")
        if masks is not None and max_rows > 64 * ldm:
            if given is not None or ldm == 0:
                raise _bad(f"masks of {ldm} words for {max_rows} rows a sequence")
            max_rows = 64 * ldm
            if out is None:  # (rows past the masks' bits are left out)
                out = torch.zeros(q.shape, dtype=q.dtype, device=dev)
        out, ldo = self._out(out, q)
        L = lib()
        key = (rows, max_rows, max_len, heads)
        nws = self._sizes.get(key)
        if nws is None:
            nws = _kept(self._sizes, key, int(L.qmm_kv_attention_workspace_size(self._p, *key)))
        ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
        _run(dev, L.qmm_kv_attention, self._p, layer, q.data_ptr(), _DENSE[q.dtype], rows, ldq, starts.data_ptr(),
             _ptr(masks), ldm, max_rows, max_len, heads, self.head_dim ** -0.5 if scale is None else scale,
             out.data_ptr(), ldo, _ptr(ws), nws)
        return out

    # -- sequences and pages -------------------------------------------------
    def fork(self, parents: torch.Tensor, keep: Optional[torch.Tensor] = None, reserve: int = 0, out=None,
             shortage: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Slot i goes on with what slot parents[i] holds (int32 [slots]; -1: the slot is emptied), cut to keep[i]
        positions (int32 [slots], negative: uncut), with pages for `reserve` further ones. Pages are shared; a
        part-filled page that is about to be written by several slots is copied for all but the lowest, or for all
        where another one holds it for good. The new lists replace table, lens and refs, or go to out = (table, lens,
        refs). Returns shortage (int32 [1]): 0, or how many pages were missing; then nothing has changed."""
        dev = self.device
        _within(reserve, 0, self.max_pages * self.page_size, "reserve")
        _ints(parents, (self.slots,), dev, "parents")
        if keep is not None:
            _ints(keep, (self.slots,), dev, "keep")
        table, lens, refs = (self.table, self.lens, self.refs) if out is None else out
        if out is not None:
            _ints(table, (self.slots, self.max_pages), dev, "out's table")
            _ints(lens, (self.slots,), dev, "out's lens")
            _ints(refs, (self.pages,), dev, "out's refs")
        if shortage is None:
            shortage = parents.new_empty(1)
        else:
            _ints(shortage, (1,), dev, "shortage")
        ws = torch.empty(self._fork_ws, dtype=torch.uint8, device=dev)
        _run(dev, lib().qmm_kv_fork, self._p, parents.data_ptr(), _ptr(keep), reserve, table.data_ptr(), lens.data_ptr(),
             refs.data_ptr(), shortage.data_ptr(), ws.data_ptr(), self._fork_ws)
        return shortage

    def accept(self, path: Optional[torch.Tensor], counts: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The first counts[s] entries of path[s] (int32 [slots, entries], increasing numbers of a step's rows) are
        accepted: their keys and values move to positions lens[s], lens[s] + 1, ... of every layer, and lens[s] (or
        out[s]) becomes lens[s] + counts[s]. path None: the first counts[s] rows, which are in place."""
        dev = self.device
        _ints(counts, (self.slots,), dev, "counts")
        if path is not None:
            if path.dim() != 2 or path.shape[1] < 1:
                raise _bad(f"path must be [slots, entries], got {list(path.shape)}")
            _ints(path, (self.slots, path.shape[1]), dev, "path")
        out = self.lens if out is None else _ints(out, (self.slots,), dev, "out")
        _run(dev, lib().qmm_kv_accept, self._p, _ptr(path), 0 if path is None else path.shape[1], counts.data_ptr(),
             out.data_ptr())
        return out

    def compact(self, out=None) -> torch.Tensor:
        """Moves the pages in use to the lowest ids: afterwards pages from the returned number (int32 [1]) on are free
        and hold nothing. table and refs follow, or go to out = (table, refs). A page that refs counts but no table row
        names moves too: hold pages by the row of a slot."""
        dev = self.device
        table, refs = (self.table, self.refs) if out is None else out
        if out is not None:
            _ints(table, (self.slots, self.max_pages), dev, "out's table")
            _ints(refs, (self.pages,), dev, "out's refs")
        used = self.refs.new_empty(1)
        ws = torch.empty(self._compact_ws, dtype=torch.uint8, device=dev)
        _run(dev, lib().qmm_kv_compact, self._p, table.data_ptr(), refs.data_ptr(), used.data_ptr(), ws.data_ptr(),
             self._compact_ws)
        return used


_beam_ws: dict = {}  # workspace sizes by their arguments


def beam_select(logits: torch.Tensor, scores: torch.Tensor, beams: int, count: int,
                finished: Optional[torch.Tensor] = None, eos: int = -1):
    """The `count` best continuations of every search of `beams` beams: logits [batch * beams, vocab] (float32,
    float16 or bfloat16), scores float32 [batch * beams] (sums of log probabilities). Returns (tokens, parents, scores,
    finished) of [batch, count], best first, ties to the lower beam and token; a parent is a row of the logits.
    A beam whose `finished` (int32 [batch * beams]) is not 0 goes on with `eos` at its own score. Where there are
    fewer continuations, token and parent are -1 and the score is -inf. Scores are ordered in 64 bits."""
    dev = _device_of(logits)
    if logits.dim() != 2 or logits.dtype not in _DENSE:
        raise _bad(f"logits must be [batch * beams, vocab] in float32, float16 or bfloat16, got {logits.dtype} "
                   f"{list(logits.shape)}")
    rows, vocab = logits.shape
    if beams < 1 or rows % beams:
        raise _bad(f"{rows} rows of logits are not whole searches of {beams} beams")
    if scores.dtype is not torch.float32 or scores.shape != (rows,) or scores.device != dev or not scores.is_contiguous():
        raise _bad(f"scores must be contiguous float32 [{rows}] on {dev}, got {scores.dtype} {list(scores.shape)} on "
                   f"{scores.device}")
    if finished is not None:
        _ints(finished, (rows,), dev, "finished")
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    batch = rows // beams
    _within(count, 1, 128, "count")
    _within(eos, -1, vocab - 1, "eos")
    L = lib()
    key = (batch, beams, vocab, count)
    nws = _beam_ws.get(key)
    if nws is None:
        nws = int(L.qmm_beam_select_workspace_size(*key))
        if nws == 0:
            raise _bad("beam_select: " + last_error())
        _kept(_beam_ws, key, nws)
    # (the four results are one allocation: four take longer than a launch)
    block = torch.empty((4, batch, count), dtype=torch.int32, device=dev)
    tokens, parents, done, out = block.unbind()
    out = out.view(torch.float32)
    first, step = block.data_ptr(), 4 * batch * count
    ws = torch.empty(nws, dtype=torch.uint8, device=dev)
    _run(dev, L.qmm_beam_select, logits.data_ptr(), _DENSE[logits.dtype], logits.stride(0) if rows > 1 else vocab, batch,
         beams, vocab, scores.data_ptr(), _ptr(finished), eos, count, first, first + step, first + 3 * step,
         first + 2 * step, ws.data_ptr(), nws)
    return tokens, parents, out, done


def reorder_rows(src: torch.Tensor, index: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[i] = src[index[i]] along the first dimension (int32 indices): the beams' texts, or any state of one row a
    beam, after a selection. Rows of an index outside src (-1) stay as `out` has them (zeros without `out`)."""
    dev = _device_of(src)
    if src.dim() < 1:
        raise _bad("reorder_rows takes rows")
    if index.dim() != 1:
        raise _bad(f"index must be [rows], got {list(index.shape)}")
    rows, inner = index.shape[0], src.shape[1:]
    _ints(index, (rows,), dev, "index")
    if not _packed(src):
        src = src.contiguous()
    if out is None:
        out = torch.zeros((rows, *inner), dtype=src.dtype, device=dev)
    elif out.dim() < 1 or out.shape[0] != rows or out.shape[1:] != inner or out.dtype != src.dtype or \
            out.device != dev or not _packed(out):
        raise _bad(f"out must be {src.dtype} [{rows}, ...] with rows like src's on {dev}, got {out.dtype} "
                   f"{list(out.shape)} on {out.device}")
    n, size = src.shape[0], src.element_size()
    nbytes = inner.numel() * size
    if rows and n and nbytes:
        _run(dev, lib().qmm_reorder_rows, src.data_ptr(), n, src.stride(0) * size if n > 1 else nbytes, out.data_ptr(),
             out.stride(0) * size if rows > 1 else nbytes, nbytes, index.data_ptr(), rows)
    return out

"""Many sequences at once: a paged 8-bit cache of keys and values, the attention of a step's new
tokens over it, and the draw of the next tokens.

The reference reads and decodes one sequence over a cache of fixed capacity (transformer.rs:166-219)
and predicts its most likely token (lm.rs:147-166); these have no counterpart there. Activations are
float32 device tensors, the arrays that describe a step int32 ones.
"""

import contextlib
import ctypes
import math
import operator

from . import _lib
from ._lib import Error, FgBatch, FgPrefixes, FgSampling, ShapeError, check, lib, stream_handle

PAGE = 64  # tokens of a page: FG_CACHE_PAGE

# A step makes these calls once a layer, and what they compute often takes less time than the call: of a
# write's 7 us on the host the launch is 4. So torch is a name of the module from the first use on, addresses
# go as whole numbers, and tensors of the plain layout are checked by their shape and contiguity alone.
torch = None


def _load():
    global torch
    if torch is None:
        import torch as module
        torch = module


class _Here:
    """A context that changes nothing (contextlib.nullcontext costs a call twice as much)."""

    def __enter__(self):
        pass

    def __exit__(self, *error):
        pass


_here = _Here()


@contextlib.contextmanager
def _on(device, stream):
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


def _place(device, stream):
    """The tensors' device current, and with `stream` that stream too (what a call allocates is then its
    own). A stream of another device is refused: torch would make that device current."""
    if stream is not None and stream.device != device:
        raise ShapeError(f"a stream of {stream.device}, the tensors are on {device}")
    if stream is None and device.index == torch._C._cuda_getDevice():
        return _here
    return _on(device, stream)


def _stream(device):
    """The current stream of `device`, which is current."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _at(t):
    return None if t is None else t.data_ptr()


def _scratch(size, device):
    """Device memory of a call from torch's allocator, which hands it out again in the stream's order
    (a graph that is captured keeps what it uses), for about a fifth of what the library's pool costs."""
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _check_ints(name, t, shape):
    if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
        raise ShapeError(f"{name}: a contiguous int32 device tensor")
    if shape is not None and list(t.shape) != shape:
        raise ShapeError(f"{name} of shape {list(t.shape)}, {shape} expected")


def _check_heads(name, t, heads, head_dim, device, written):
    """[rows, heads, head_dim] float32 whose rows are runs of heads * head_dim values. Returns how far apart rows are (asking
    a tensor for it costs twice what its contiguity does)."""
    if t.dtype is not torch.float32 or t.device != device:
        raise ShapeError(f"{name}: a float32 tensor on {device}")
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim:
        raise ShapeError(f"{name} of shape {list(shape)}, [rows, {heads}, {head_dim}] expected")
    if t.is_contiguous():
        return heads * head_dim
    row, head, value = t.stride()
    if shape[0] == 0:
        return row
    if value != 1 or (heads > 1 and head != head_dim):
        raise ShapeError(f"{name}: a row's heads lie one after the other")
    if written and shape[0] > 1 and row < heads * head_dim:
        raise ShapeError(f"{name}: its rows overlap")
    return row


class Batch:
    """The new tokens of a step's sequences (fg_batch), as int32 device tensors that the kernels read:
    a captured graph's replay reads what they hold then.

    `row_starts` [sequences + 1]: sequence s has the rows row_starts[s] .. row_starts[s + 1] - 1 of the
    operands as new tokens (rows that no sequence holds are left alone); `lengths` [sequences]: its
    tokens, the new ones included; `pages` [sequences, max_pages]: the page of its tokens 64 p on at p.
    """

    def __init__(self, row_starts, lengths, pages):
        _load()
        if pages.dim() != 2:
            raise ShapeError("pages: [sequences, max_pages]")
        sequences = pages.shape[0]
        _check_ints("row_starts", row_starts, [sequences + 1])
        _check_ints("lengths", lengths, [sequences])
        _check_ints("pages", pages, None)
        if not row_starts.device == lengths.device == pages.device:
            raise ShapeError("a batch's tensors are on one device")
        self.row_starts, self.lengths, self.pages = row_starts, lengths, pages

    @property
    def sequences(self):
        return self.lengths.shape[0]

    def _ffi(self, rows):
        p = self.pages
        sequences, max_pages = p.shape
        return FgBatch(sequences, rows, max_pages, self.row_starts.data_ptr(), self.lengths.data_ptr(), p.data_ptr())


class Prefixes:
    """Runs of a batch's sequences that begin with the same pages (fg_prefixes), as int32 device tensors that the
    kernels read: `starts` [groups + 1], group g is the sequences starts[g] .. starts[g + 1] - 1, and `pages` [groups],
    how many pages the tables of all of them begin with. Sequences that no group holds share nothing."""

    def __init__(self, starts, pages):
        _load()
        if pages.dim() != 1:
            raise ShapeError("pages: [groups]")
        _check_ints("starts", starts, [pages.shape[0] + 1])
        _check_ints("pages", pages, None)
        if starts.device != pages.device:
            raise ShapeError("the prefixes' tensors are on one device")
        self.starts, self.pages = starts, pages

    @property
    def groups(self):
        return self.pages.shape[0]

    def _ffi(self):
        return FgPrefixes(self.pages.shape[0], self.starts.data_ptr(), self.pages.data_ptr())


def _rotated_out(x, rows, head_dim, device, out):
    """`out` for `rows` rows `x` [rows, heads, head_dim] turned (made here where None: rows that no sequence holds are
    then 0), both checked; the heads, and how far apart the rows of both are."""
    shape = x.shape
    if len(shape) != 3 or shape[0] != rows:
        raise ShapeError(f"rows to turn of shape {list(shape)}, [{rows}, heads, {head_dim}] expected")
    heads = shape[1]
    stride = out_stride = _check_heads("rows to turn", x, heads, head_dim, device, out is x)
    if out is None:
        out = torch.zeros(shape, dtype=torch.float32, device=device)
        out_stride = heads * head_dim
    elif out is not x:
        out_stride = _check_heads("out", out, heads, head_dim, device, True)
        if out.shape[0] != rows:
            raise ShapeError(f"{rows} rows to turn and {out.shape[0]} of out")
    return out, heads, stride, out_stride


class Rotary:
    """Rotary positions (fg_rotary): the first `dims` values of a head in pairs, pair i turned at position p by
    p * f_i radians, f_i = base ** (-2 i / dims); with `layout` "halves" value i's partner is i + dims / 2, with
    "pairs" 2 i's is 2 i + 1. Cosines and sines are computed in 64 bits at any position.

    For contexts longer than a model was trained on, `stretch` divides the frequencies; with `trained`, the
    tokens it was trained on, only those that turn fewer than `slow` times over them are divided whole, those
    that turn more than `fast` times not at all, and between the two the share of the undivided frequency
    rises evenly with the turns. `magnitude` multiplies the turned values. `frequencies` (dims / 2 numbers,
    radians a token) takes the place of all of these but the magnitude."""

    LAYOUTS = {"halves": 0, "pairs": 1}

    def __init__(self, dims, base=10000.0, layout="halves", stretch=1.0, trained=None, slow=1.0, fast=32.0, magnitude=1.0,
                 frequencies=None, device=None, stream=None):
        _load()
        if layout not in self.LAYOUTS:
            raise ValueError(f'layout {layout!r}: "halves" or "pairs"')
        if dims < 2 or dims % 2:
            raise ShapeError(f"{dims} values to turn: an even number expected")
        if frequencies is None:
            frequencies = self._frequencies(dims, base, stretch, trained, slow, fast)
        self.frequencies = [float(f) for f in frequencies]
        if len(self.frequencies) != dims // 2:
            raise ShapeError(f"{len(self.frequencies)} frequencies for {dims} values")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ShapeError("rotary positions are on a GPU")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.dims, self.layout, self.magnitude, self.device = dims, layout, float(magnitude), device
        handle = ctypes.c_void_p()
        with _place(device, stream):
            check(lib().fg_rotary_create((ctypes.c_double * (dims // 2))(*self.frequencies), dims, self.LAYOUTS[layout], self.magnitude,
                                         stream_handle(), ctypes.byref(handle)))
        self.handle = handle

    @staticmethod
    def _frequencies(dims, base, stretch, trained, slow, fast):
        if not base > 0 or not stretch > 0:
            raise ValueError("a base and a stretch above 0")
        if trained is not None and (not trained > 0 or not fast > slow):
            raise ValueError("trained tokens above 0, and more turns for `fast` than for `slow`")
        out = []
        for i in range(dims // 2):
            f = float(base) ** (-2.0 * i / dims)
            share = 0.0
            if trained is not None:
                share = min(max((trained * f / (2 * math.pi) - slow) / (fast - slow), 0.0), 1.0)
            out.append(f * (share + (1.0 - share) / stretch))
        return out

    def __del__(self):
        h = getattr(self, "handle", None)
        if h is not None and _lib is not None and _lib._lib is not None:  # (None as the interpreter ends)
            _lib._lib.fg_rotary_free(h)
            self.handle = None

    def rotate(self, batch, x, out=None, stream=None):
        """The batch's new rows of `x` [rows, heads, head_dim] turned by their positions, into `out`, which may be
        `x` and otherwise does not overlap it. Rows of `out` that no sequence holds are left as they are (0 in an `out` made here)."""
        if x.dim() != 3 or batch.pages.device != self.device:
            raise ShapeError(f"rows [rows, heads, head_dim] and a batch on {self.device}")
        rows, _, head_dim = x.shape
        with _place(self.device, stream):
            out, heads, stride, out_stride = _rotated_out(x, rows, head_dim, self.device, out)
            check(lib().fg_rotary_rotate(self.handle, ctypes.byref(batch._ffi(rows)), x.data_ptr(), stride, heads, head_dim,
                                         out.data_ptr(), out_stride, _stream(self.device)))
        return out


class PagedCache:
    """The keys and values of one layer's attention over many sequences (fg_cache): `pages` pages of
    PAGE tokens for `kv_heads` heads of `head_dim` values (whole quads, at most 256), each token's
    key and value of a head as int8 levels and one float32 scale."""

    def __init__(self, pages, kv_heads, head_dim, device=None, stream=None):
        _load()
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ShapeError("a cache is on a GPU")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.pages, self.kv_heads, self.head_dim, self.device = pages, kv_heads, head_dim, device
        handle = ctypes.c_void_p()
        with _place(device, stream):
            check(lib().fg_cache_create(pages, kv_heads, head_dim, stream_handle(), ctypes.byref(handle)))
        self.handle = handle

    def __del__(self):
        h = getattr(self, "handle", None)
        if h is not None and _lib is not None and _lib._lib is not None:  # (None as the interpreter ends)
            _lib._lib.fg_cache_free(h)
            self.handle = None

    def _rows(self, batch, keys, values, written):
        if batch.pages.device != self.device:
            raise ShapeError(f"the batch is on {batch.pages.device}, the cache on {self.device}")
        key_stride = _check_heads("keys", keys, self.kv_heads, self.head_dim, self.device, written)
        value_stride = _check_heads("values", values, self.kv_heads, self.head_dim, self.device, written)
        rows = keys.shape[0]
        if rows != values.shape[0]:
            raise ShapeError(f"{rows} rows of keys and {values.shape[0]} of values")
        return ctypes.byref(batch._ffi(rows)), key_stride, value_stride

    def write(self, batch, keys, values, stream=None, rotary=None, queries=None, out=None):
        """The new tokens' `keys` and `values` [rows, kv_heads, head_dim] quantized into their pages
        (a page that is written to belongs to one sequence). With `rotary` (Rotary) the keys are turned by
        their positions on the way, and `queries` [rows, heads, head_dim], if given, by the same call into
        `out`, which is returned (`out` as for Rotary.rotate; it overlaps neither `keys` nor `values`)."""
        fg, key_stride, value_stride = self._rows(batch, keys, values, False)
        if rotary is not None:
            return self._write_rotated(fg, keys, key_stride, values, value_stride, stream, rotary, queries, out)
        if queries is not None or out is not None:
            raise ShapeError("queries are turned by `rotary`: none given")
        with _place(self.device, stream):
            check(lib().fg_cache_write(self.handle, fg, keys.data_ptr(), key_stride, values.data_ptr(), value_stride,
                                       _stream(self.device)))

    def _write_rotated(self, fg, keys, key_stride, values, value_stride, stream, rotary, queries, out):
        if rotary.device != self.device:
            raise ShapeError(f"the rotary positions are on {rotary.device}, the cache on {self.device}")
        if queries is None and out is not None:
            raise ShapeError("an `out` without queries")
        heads = query = query_stride = to = to_stride = 0
        with _place(self.device, stream):
            if queries is not None:
                out, heads, query_stride, to_stride = _rotated_out(queries, keys.shape[0], self.head_dim, self.device, out)
                query, to = queries.data_ptr(), out.data_ptr()
            check(lib().fg_cache_write_rotated(self.handle, fg, rotary.handle, keys.data_ptr(), key_stride, values.data_ptr(),
                                               value_stride, query, query_stride, heads, to, to_stride, _stream(self.device)))
        return out

    def read(self, batch, keys, values, stream=None):
        """The same tokens read back into `keys` and `values`: level * scale."""
        fg, key_stride, value_stride = self._rows(batch, keys, values, True)
        with _place(self.device, stream):
            check(lib().fg_cache_read(self.handle, fg, keys.data_ptr(), key_stride, values.data_ptr(), value_stride,
                                      _stream(self.device)))

    def attend(self, batch, queries, out=None, scale=None, window=0, stream=None, prefixes=None):
        """The attention of the new tokens' `queries` [rows, heads, head_dim] (their keys and values
        written before): each token sees its sequence's tokens up to itself, with `window` the last
        `window` of them. `scale` is 1 / sqrt(head_dim) unless given. A token without a key gives 0;
        `out` may be `queries`; rows of it that no sequence holds are left as they are (0 in an `out`
        made here). Keys may reach 1e33 and scores 1e7 in magnitude. With `prefixes` (Prefixes) the pages that a group
        of sequences begins with are worked through once for all of them, if the batch's tables have room for 224 MiB together and
        its sequences few new tokens on average (fg_cache_attend_shared has the rule); if not, each sequence reads its own."""
        if batch.pages.device != self.device:
            raise ShapeError(f"the batch is on {batch.pages.device}, the cache on {self.device}")
        if queries.dim() != 3:
            raise ShapeError("queries: [rows, heads, head_dim]")
        heads = queries.shape[1]
        stride = _check_heads("queries", queries, heads, self.head_dim, self.device, False)
        if window < 0:
            raise ShapeError("a window of at least one token, or 0 for all")
        with _place(self.device, stream):
            if out is None:
                out = torch.zeros(queries.shape, dtype=torch.float32, device=self.device)
            out_stride = _check_heads("out", out, heads, self.head_dim, self.device, True)
            if out.shape[0] != queries.shape[0]:
                raise ShapeError(f"{queries.shape[0]} rows of queries and {out.shape[0]} of out")
            fg, library = ctypes.byref(batch._ffi(queries.shape[0])), lib()
            if prefixes is not None:
                if prefixes.pages.device != self.device:
                    raise ShapeError(f"the prefixes are on {prefixes.pages.device}, the cache on {self.device}")
                shared = ctypes.byref(prefixes._ffi())
                size = library.fg_cache_attend_shared_scratch(self.handle, fg, shared, heads)
                scratch = _scratch(size, self.device)
                check(library.fg_cache_attend_shared(self.handle, fg, shared, queries.data_ptr(), stride, heads,
                                                     1.0 / math.sqrt(self.head_dim) if scale is None else scale, window, out.data_ptr(),
                                                     out_stride, _at(scratch), size, _stream(self.device)))
                return out
            size = library.fg_cache_attend_scratch(self.handle, fg, heads)
            scratch = _scratch(size, self.device)
            check(library.fg_cache_attend(self.handle, fg, queries.data_ptr(), stride, heads,
                                          1.0 / math.sqrt(self.head_dim) if scale is None else scale, window, out.data_ptr(),
                                          out_stride, _at(scratch), size, _stream(self.device)))
        return out


def copy_pages(caches, sources, targets, stream=None):
    """Pages copied in every one of `caches` (fg_cache_copy): sources[i] to targets[i], whole. The ids are int32 device
    tensors [pages], which a captured graph's replay reads as they are then, or lists, which are checked here: no
    target twice, and none that is a source too (a page with itself apart)."""
    _load()
    caches = list(caches)
    if not caches:
        return
    device = caches[0].device
    if any(c.device != device for c in caches):
        raise ShapeError("the caches are on one device")
    if not isinstance(sources, torch.Tensor) and not isinstance(targets, torch.Tensor):
        sources, targets = ([operator.index(p) for p in ids] for ids in (sources, targets))
        moved = [(s, t) for s, t in zip(sources, targets) if s != t]
        kept = {t for s, t in zip(sources, targets) if s == t}
        ends = {t for _, t in moved}
        if len(ends) != len(moved) or ends & {s for s, _ in moved} or ends & kept:
            raise ShapeError("a page is copied to that is named twice")
        limit = min(c.pages for c in caches)
        if any(not 0 <= p < limit for p in sources + targets):
            raise ShapeError(f"pages 0 to {limit - 1}")
        with _place(device, stream):
            sources, targets = (torch.tensor(p, dtype=torch.int32, device=device) for p in (sources, targets))
            return _copy_pages(caches, sources, targets, device)
    for name, t in (("sources", sources), ("targets", targets)):
        if not isinstance(t, torch.Tensor) or t.dim() != 1:
            raise ShapeError(f"{name}: int32 device tensors [pages] both, or lists both")
        _check_ints(name, t, None)
        if t.device != device:
            raise ShapeError(f"{name} are on {t.device}, the caches on {device}")
    with _place(device, stream):
        _copy_pages(caches, sources, targets, device)


def _copy_pages(caches, sources, targets, device):
    if sources.shape != targets.shape:
        raise ShapeError(f"{sources.shape[0]} sources and {targets.shape[0]} targets")
    handles = (ctypes.c_void_p * len(caches))(*[c.handle.value for c in caches])
    check(lib().fg_cache_copy(handles, len(caches), sources.data_ptr(), targets.data_ptr(), sources.shape[0], _stream(device)))


class Pages:
    """Which of a cache's `count` pages are in use, and by how many sequences: the host's side of forks and compactions
    (one for all layers' caches, which hold a token under the same page id)."""

    def __init__(self, count):
        self.count = count
        self._free = list(range(count - 1, -1, -1))  # the last is handed out next: the lowest ids first
        self._users = [0] * count

    @property
    def free_pages(self):
        return len(self._free)

    def users(self, page):
        """How many sequences hold `page`."""
        return self._users[page]

    def take(self, count):
        """`count` pages that no sequence holds."""
        if count < 0 or count > len(self._free):
            raise Error(f"{count} pages asked for, {len(self._free)} of {self.count} are free")
        pages = [self._free.pop() for _ in range(count)]
        for p in pages:
            self._users[p] = 1
        return pages

    def fork(self, pages, length):
        """A second sequence with the `length` tokens that lie in `pages`: its pages, and the copies to make, (sources,
        targets) for copy_pages. Whole pages are shared; one that is partly full, which both go on writing to, is copied."""
        held = -(-length // PAGE)
        pages = list(pages)
        if length < 0 or held > len(pages):
            raise ShapeError(f"{length} tokens in {len(pages)} pages")
        whole = length // PAGE
        pages = self._held(pages[:held])
        if whole < held and not self._free:
            raise Error("a page asked for, none is free")
        for p in pages[:whole]:
            self._users[p] += 1
        copies = self.take(held - whole)
        return pages[:whole] + copies, (pages[whole:], list(copies))

    def free(self, pages):
        """A sequence lets go of its pages."""
        for p in self._held(pages):
            self._users[p] -= 1
            if self._users[p] == 0:
                self._free.append(p)

    def compact(self):
        """The pages in use moved to the lowest ids: {old id: new id} of those that move. Its keys and values are
        copy_pages' sources and targets; every sequence's table takes the new ids. The pages from the number in use on
        are free then, so that a smaller cache could hold the rest."""
        used = self.count - len(self._free)
        low = sorted(p for p in self._free if p < used)
        high = [p for p in range(used, self.count) if self._users[p]]
        moves = dict(zip(high, low))
        for old, new in moves.items():
            self._users[new], self._users[old] = self._users[old], 0
        self._free = list(range(self.count - 1, used - 1, -1))
        return moves

    def _held(self, pages):
        """The ids as a list of whole numbers (a table's row adds, and holds numbers that compare but do not hash alike)."""
        pages = [operator.index(p) for p in pages]
        if len(set(pages)) != len(pages) or any(not 0 <= p < self.count or not self._users[p] for p in pages):
            raise ShapeError("pages that no sequence holds, or one of them twice")
        return pages


def sample(logits, random, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, chances=None, stream=None):
    """The next token of every row of `logits` [rows, vocab] and its chance (fg_sample), drawn by
    `random` [rows] in [0, 1). The settings are device tensors [rows]: float32 `temperature` (0: the
    most likely token), int32 `top_k` (0: no limit), float32 `top_p` (1: no limit) and `min_p` (0: no
    limit), applied in that order. Returns (tokens int32 [rows], chances float32 [rows])."""
    _load()
    if logits.dim() != 2 or logits.dtype != torch.float32 or not logits.is_cuda:
        raise ShapeError("logits: a float32 device tensor [rows, vocab]")
    rows, vocab = logits.shape
    if rows and vocab > 1 and logits.stride(1) != 1:
        raise ShapeError("logits: a row's values lie one after the other")
    device, shape, f32, i32 = logits.device, (rows,), torch.float32, torch.int32
    if random is None:
        raise ShapeError("random: one number a row")
    for name, t, dtype in (("random", random, f32), ("temperature", temperature, f32), ("top_k", top_k, i32), ("top_p", top_p, f32),
                           ("min_p", min_p, f32), ("tokens", tokens, i32), ("chances", chances, f32)):
        if t is not None and (t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous()):
            raise ShapeError(f"{name}: a contiguous {dtype} tensor [{rows}] on {device}")
    with _place(device, stream):
        if tokens is None:
            tokens = torch.empty(rows, dtype=i32, device=device)
        if chances is None:
            chances = torch.empty(rows, dtype=f32, device=device)
        fg, library = FgSampling(random.data_ptr(), _at(temperature), _at(top_k), _at(top_p), _at(min_p)), lib()
        size = library.fg_sample_scratch(rows, vocab)
        scratch = _scratch(size, device)
        check(library.fg_sample(logits.data_ptr(), rows, vocab, logits.stride(0), ctypes.byref(fg), tokens.data_ptr(),
                                chances.data_ptr(), _at(scratch), size, _stream(device)))
    return tokens, chances

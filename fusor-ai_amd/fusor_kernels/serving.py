"""Many sequences at once: a paged 8-bit cache of keys and values, the attention of a step's new
tokens over it, and the draw of the next tokens.

The reference reads and decodes one sequence over a cache of fixed capacity (transformer.rs:166-219)
and predicts its most likely token (lm.rs:147-166); these have no counterpart there. Activations are
float32 device tensors, the arrays that describe a step int32 ones.
"""

import contextlib
import ctypes
import math

from . import _lib
from ._lib import FgBatch, FgSampling, ShapeError, check, lib, stream_handle

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
    """[rows, heads, head_dim] float32 whose rows are runs of heads * head_dim values."""
    if t.dtype is not torch.float32 or t.device != device:
        raise ShapeError(f"{name}: a float32 tensor on {device}")
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim:
        raise ShapeError(f"{name} of shape {list(shape)}, [rows, {heads}, {head_dim}] expected")
    if t.is_contiguous():
        return
    row, head, value = t.stride()
    if shape[0] == 0:
        return
    if value != 1 or (heads > 1 and head != head_dim):
        raise ShapeError(f"{name}: a row's heads lie one after the other")
    if written and shape[0] > 1 and row < heads * head_dim:
        raise ShapeError(f"{name}: its rows overlap")


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
        _check_heads("keys", keys, self.kv_heads, self.head_dim, self.device, written)
        _check_heads("values", values, self.kv_heads, self.head_dim, self.device, written)
        if keys.shape[0] != values.shape[0]:
            raise ShapeError(f"{keys.shape[0]} rows of keys and {values.shape[0]} of values")
        return batch._ffi(keys.shape[0])

    def write(self, batch, keys, values, stream=None):
        """The new tokens' `keys` and `values` [rows, kv_heads, head_dim] quantized into their pages
        (a page that is written to belongs to one sequence)."""
        fg = self._rows(batch, keys, values, False)
        with _place(self.device, stream):
            check(lib().fg_cache_write(self.handle, ctypes.byref(fg), keys.data_ptr(), keys.stride(0), values.data_ptr(),
                                       values.stride(0), _stream(self.device)))

    def read(self, batch, keys, values, stream=None):
        """The same tokens read back into `keys` and `values`: level * scale."""
        fg = self._rows(batch, keys, values, True)
        with _place(self.device, stream):
            check(lib().fg_cache_read(self.handle, ctypes.byref(fg), keys.data_ptr(), keys.stride(0), values.data_ptr(),
                                      values.stride(0), _stream(self.device)))

    def attend(self, batch, queries, out=None, scale=None, window=0, stream=None):
        """The attention of the new tokens' `queries` [rows, heads, head_dim] (their keys and values
        written before): each token sees its sequence's tokens up to itself, with `window` the last
        `window` of them. `scale` is 1 / sqrt(head_dim) unless given. A token without a key gives 0;
        `out` may be `queries`; rows of it that no sequence holds are left as they are (0 in an `out`
        made here). Keys may reach 1e33 and scores 1e7 in magnitude."""
        if batch.pages.device != self.device:
            raise ShapeError(f"the batch is on {batch.pages.device}, the cache on {self.device}")
        if queries.dim() != 3:
            raise ShapeError("queries: [rows, heads, head_dim]")
        heads = queries.shape[1]
        _check_heads("queries", queries, heads, self.head_dim, self.device, False)
        if window < 0:
            raise ShapeError("a window of at least one token, or 0 for all")
        with _place(self.device, stream):
            if out is None:
                out = torch.zeros(queries.shape, dtype=torch.float32, device=self.device)
            _check_heads("out", out, heads, self.head_dim, self.device, True)
            if out.shape[0] != queries.shape[0]:
                raise ShapeError(f"{queries.shape[0]} rows of queries and {out.shape[0]} of out")
            fg, library = ctypes.byref(batch._ffi(queries.shape[0])), lib()
            size = library.fg_cache_attend_scratch(self.handle, fg, heads)
            scratch = _scratch(size, self.device)
            check(library.fg_cache_attend(self.handle, fg, queries.data_ptr(), queries.stride(0), heads,
                                          1.0 / math.sqrt(self.head_dim) if scale is None else scale, window, out.data_ptr(),
                                          out.stride(0), _at(scratch), size, _stream(self.device)))
        return out


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

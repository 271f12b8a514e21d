"""Operators a decoder needs around its attention when it is served, over the C-ABI of include/ft_serving.h.

`Rotary` turns Q and K by their positions, `PagedCache` holds K and V in pages (append, copy, keep the accepted drafted
tokens), `PagePool` says which sequence holds which page (fork, truncate, compact), `PromptAttention` is the attention over
packed prompts of different lengths and `TreeAttention` that of new or drafted tokens over the cache.  torch supplies device
memory and streams only; the reference has no counterpart to any of them.
"""
import ctypes
import struct
import threading
from typing import List, Optional, Sequence, Tuple

import torch

from . import _abi

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}  # FT_SRC_BF16, FT_SRC_F16
_SCALINGS = {None: 0, "none": 0, "linear": 1, "base": 2, "by_parts": 3}


class FtRows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong), ("heads", ctypes.c_int)]


class FtRotaryOptions(ctypes.Structure):
    _fields_ = [("head_dim", ctypes.c_int), ("rotary_dim", ctypes.c_int), ("interleaved", ctypes.c_int), ("scaling", ctypes.c_int)] + [
        (name, ctypes.c_double) for name in ("base", "factor", "original_length", "low", "high", "magnitude")]


class FtKvCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] + [
        (name, ctypes.c_longlong) for name in ("layer_stride", "page_stride", "token_stride", "head_stride")] + [
        (name, ctypes.c_int) for name in ("layers", "pages", "page_size", "kv_heads", "head_dim", "dtype")]


class FtPromptAttentionArgs(ctypes.Structure):
    _fields_ = [(name, FtRows) for name in ("q", "k", "v", "out")] + [
        (name, ctypes.c_void_p) for name in ("lse", "q_offsets", "k_offsets")] + [
        (name, ctypes.c_int) for name in ("batch", "query_tokens", "key_tokens", "head_dim", "dtype", "causal")] + [("scale", ctypes.c_float)]


class FtTreeAttentionArgs(ctypes.Structure):
    _fields_ = [(name, FtRows) for name in ("q", "out")] + [
        (name, ctypes.c_void_p) for name in ("lse", "q_offsets", "page_table", "lengths", "mask")] + [
        (name, ctypes.c_int) for name in ("mask_words", "mask_stride", "batch", "query_tokens", "table_pages", "table_stride", "layer")] + [
        ("scale", ctypes.c_float)]


# The same structures for the calls below, packed in one step: field by field they take longer than a small kernel runs.
_ROWS = "Pqqi4x"
_PACK_ROWS = struct.Struct(_ROWS).pack
_PACK_PROMPT = struct.Struct(_ROWS * 4 + "PPPiiiiiif0P").pack
_PACK_TREE = struct.Struct(_ROWS * 2 + "PPPPPiiiiiiif0P").pack

# Looked up once: attribute chains cost as much as some of the calls.  (A torch without CUDA has none of them.)
_get_device, _raw_stream, _raw_alloc, _raw_delete = (
    getattr(torch._C, name, None) for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream", "_cuda_cudaCachingAllocator_raw_alloc",
                                               "_cuda_cudaCachingAllocator_raw_delete"))

_bound = False
_binding = threading.Lock()
_calls = {}  # the entry points that run on a device, with structures given as packed bytes


def _lib():
    """The library with the types of this module's entry points.  The first use may come from several threads at once."""
    global _bound, _calls
    lib = _abi.load()
    if not _bound:
        with _binding:
            if not _bound:
                _calls = _bind(lib)
                _bound = True
    return lib


def _bind(lib) -> dict:
    vp, ci, rows, cache = ctypes.c_void_p, ctypes.c_int, ctypes.POINTER(FtRows), ctypes.POINTER(FtKvCache)
    ints = ctypes.POINTER(ci)
    lib.ft_rotary_options_default.argtypes = [ctypes.POINTER(FtRotaryOptions), ci]
    lib.ft_rotary_options_default.restype = None
    lib.ft_rotary_frequencies.argtypes = [ctypes.POINTER(FtRotaryOptions), ctypes.POINTER(ctypes.c_double)]
    lib.ft_rotary_prepare.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(FtRotaryOptions), vp]
    lib.ft_rotary_destroy.argtypes = [vp]
    lib.ft_rotary_run.argtypes = [vp, rows, rows, rows, rows, vp, ci, ci, ci, vp]
    lib.ft_kv_cache_append.argtypes = [cache, ci, rows, rows, vp, ci, vp, vp, rows, rows, vp]
    lib.ft_kv_cache_copy_pages.argtypes = [cache, vp, vp, ci, vp]
    lib.ft_kv_cache_accept.argtypes = [cache, vp, ci, ci, vp, vp, vp, vp, ci, vp, vp]
    lib.ft_page_pool_create.argtypes = [ctypes.POINTER(vp), ci, ci]
    for name in ("destroy", "free_pages"):
        getattr(lib, f"ft_page_pool_{name}").argtypes = [vp]
    lib.ft_page_pool_new_sequence.argtypes = [vp, ints]
    lib.ft_page_pool_fork.argtypes = [vp, ci, ints]
    lib.ft_page_pool_free.argtypes = [vp, ci]
    lib.ft_page_pool_extend.argtypes = [vp, ci, ci, ints, ints]
    lib.ft_page_pool_truncate.argtypes = [vp, ci, ci]
    lib.ft_page_pool_length.argtypes = [vp, ci]
    lib.ft_page_pool_pages.argtypes = [vp, ci, ints, ci]
    lib.ft_page_pool_compact.argtypes = [vp, ints, ints, ci, ints]
    lib.ft_attention_workspace.argtypes = []
    lib.ft_attention_workspace.restype = ctypes.c_size_t
    lib.ft_prompt_attention_run.argtypes = [ctypes.POINTER(FtPromptAttentionArgs), vp, ctypes.c_size_t, vp, vp]
    lib.ft_tree_attention_run.argtypes = [cache, ctypes.POINTER(FtTreeAttentionArgs), vp, ctypes.c_size_t, vp, vp]
    lib.ft_tree_mask.argtypes = [ints, ci, ctypes.POINTER(ctypes.c_uint32), ci]
    size, calls = ctypes.c_size_t, {}
    for name, types in (("ft_rotary_run", [vp] * 6 + [ci] * 3 + [vp]), ("ft_kv_cache_append", [vp, ci, vp, vp, vp, ci] + [vp] * 5),
                        ("ft_kv_cache_copy_pages", [vp, vp, vp, ci, vp]),
                        ("ft_kv_cache_accept", [vp, vp, ci, ci, vp, vp, vp, vp, ci, vp, vp]),
                        ("ft_prompt_attention_run", [vp, vp, size, vp, vp]), ("ft_tree_attention_run", [vp, vp, vp, size, vp, vp])):
        call = lib[name]
        call.argtypes = types
        calls[name] = call
    return calls  # seen by others only now, when all have their types


def _call(name: str, device: torch.device, *args):
    """One of _calls on the device of its tensors, which is nearly always the current one already."""
    if _get_device() == device.index:
        code = _calls[name](*args)
    else:
        with torch.cuda.device(device):
            code = _calls[name](*args)
    if code:
        _abi.check(code)


def _stream(device: torch.device, stream: Optional[torch.cuda.Stream]) -> int:
    if stream is None:
        return _raw_stream(device.index)
    if stream.device != device:
        raise ValueError(f"the stream belongs to {stream.device}, the tensors to {device}")
    return stream.cuda_stream


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device, heads: int, head_dim: int, tokens: int) -> Tuple[int, int, int, int]:
    """The fields of an ft_rows: [tokens, heads, head_dim] of the operator's type, head_dim contiguous; the C side checks
    alignment and strides."""
    stride = t.stride()
    if t.dtype is not dtype or t.get_device() != device.index or t.shape != (tokens, heads, head_dim) or stride[2] != 1:
        raise ValueError(f"{name} must be a [{tokens}, {heads}, {head_dim}] {dtype} tensor on {device} with a contiguous last dimension "
                         f"(got {list(t.shape)}, {t.dtype} on {t.device}, strides {list(stride)})")
    return t.data_ptr(), stride[0], stride[1], heads


def _vector(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device, size: Optional[int] = None) -> int:
    if t.dtype is not dtype or t.get_device() != device.index or t.dim() != 1 or not t.is_contiguous() or (size is not None and len(t) != size):
        raise ValueError(f"{name} must be a contiguous one-dimensional {dtype} tensor on {device}" + (f" of {size} elements" if size is not None else ""))
    return t.data_ptr()


def _matrix(t: torch.Tensor, name: str, device: torch.device, rows: int) -> Tuple[int, int, int]:
    """(address, columns, elements from row to row)"""
    shape, stride = t.shape, t.stride()
    if t.dtype is not torch.int32 or t.get_device() != device.index or len(shape) != 2 or shape[0] != rows or shape[1] == 0 or stride[1] != 1:
        raise ValueError(f"{name} must be a [{rows}, columns] int32 tensor on {device} with contiguous rows")
    return t.data_ptr(), shape[1], max(stride[0], shape[1]) if rows == 1 else stride[0]


def _check_dtype(dtype: torch.dtype) -> int:
    if dtype not in _DTYPES:
        raise ValueError(f"the element type must be torch.bfloat16 or torch.float16 (got {dtype})")
    return _DTYPES[dtype]


class Rotary:
    """Rotary positions of one model: pairs (i, i + rotary_dim/2), or (2i, 2i + 1) when interleaved, of the first
    rotary_dim elements of a head.  scaling: None, "linear" (frequencies / factor), "base" (the base grows with the factor)
    or "by_parts" (only frequencies that turn less than `high` times within original_length are divided, all of those below `low`)."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False,
                 scaling: Optional[str] = None, factor: float = 1.0, original_length: float = 0.0, low: float = 1.0, high: float = 4.0,
                 magnitude: float = 1.0, device="cuda"):
        self.lib = _lib()
        if scaling not in _SCALINGS:
            raise ValueError(f"scaling must be one of {list(_SCALINGS)} (got {scaling!r})")
        self.options = FtRotaryOptions()
        self.lib.ft_rotary_options_default(ctypes.byref(self.options), head_dim)
        o = self.options
        o.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        o.interleaved, o.scaling = int(interleaved), _SCALINGS[scaling]
        o.base, o.factor, o.original_length, o.low, o.high, o.magnitude = base, factor, original_length, low, high, magnitude
        self.head_dim = head_dim
        self.handle = ctypes.c_void_p()
        self.frequencies()  # refuses bad options before a device is touched
        self.device = torch.empty(0, device=device).device
        with torch.cuda.device(self.device):
            _abi.check(self.lib.ft_rotary_prepare(ctypes.byref(self.handle), ctypes.byref(o), _stream(self.device, None)))

    def frequencies(self) -> List[float]:
        """Radians per position of every pair."""
        out = (ctypes.c_double * max(1, self.options.rotary_dim // 2))()
        _abi.check(self.lib.ft_rotary_frequencies(ctypes.byref(self.options), out))
        return list(out)

    def run(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, q_out: torch.Tensor, k_out: Optional[torch.Tensor] = None,
            inverse: bool = False, stream: Optional[torch.cuda.Stream] = None):
        """q [tokens, heads, head_dim], k [tokens, key heads, head_dim] or None, positions int64 [tokens].  An output may be
        its input.  inverse: turn back; with the output gradients as q and k this is the gradient."""
        dtype, device, tokens = q.dtype, q.device, q.shape[0]
        code = _check_dtype(dtype)
        if device != self.device or q.dim() != 3:
            raise ValueError(f"q must be a [tokens, heads, {self.head_dim}] tensor on {self.device}")
        if (k is None) != (k_out is None):
            raise ValueError("k and k_out come together")
        heads = q.shape[1]
        rq = _PACK_ROWS(*_rows(q, "q", dtype, device, heads, self.head_dim, tokens))
        ro = _PACK_ROWS(*_rows(q_out, "q_out", dtype, device, heads, self.head_dim, tokens))
        rk = rko = None
        if k is not None:
            if k.dim() != 3:
                raise ValueError(f"k must be a [{tokens}, heads, {self.head_dim}] tensor")
            heads = k.shape[1]
            rk = _PACK_ROWS(*_rows(k, "k", dtype, device, heads, self.head_dim, tokens))
            rko = _PACK_ROWS(*_rows(k_out, "k_out", dtype, device, heads, self.head_dim, tokens))
        at = _vector(positions, "positions", torch.int64, device, tokens)
        if tokens == 0:
            return
        _call("ft_rotary_run", device, self.handle, rq, ro, rk, rko, at, tokens, code, int(inverse), _stream(device, stream))

    def close(self):
        if getattr(self, "handle", None) is not None and self.handle.value:
            self.lib.ft_rotary_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedCache:
    """K and V of all layers in pages: two tensors [layers, pages, page_size, key heads, head_dim] of the caller's (a page
    may also be laid out by head: a permuted view of [layers, pages, key heads, page_size, head_dim])."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.stride() != v.stride() or not k.is_cuda or k.stride(4) != 1:
            raise ValueError("K and V must be CUDA tensors [layers, pages, page_size, key heads, head_dim] alike in shape, type, device and strides, "
                             "with a contiguous last dimension")
        self.lib = _lib()
        self.k, self.v = k, v
        self.dtype, self.device = k.dtype, k.device
        self.layers, self.pages, self.page_size, self.kv_heads, self.head_dim = k.shape
        s = k.stride()
        self.view = FtKvCache(k.data_ptr(), v.data_ptr(), s[0], s[1], s[2], s[3], *k.shape, _check_dtype(k.dtype))
        _abi.check(self.lib.ft_kv_cache_copy_pages(ctypes.byref(self.view), None, None, 0, None))  # refuses a layout that the kernels cannot take
        self.address = ctypes.addressof(self.view)

    @classmethod
    def empty(cls, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        shape = (layers, pages, page_size, kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, rotary: Optional[Rotary] = None,
               positions: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None):
        """Writes k and v [tokens, key heads, head_dim] to slots (int64: page * page_size + place; negative: not written;
        all different).  With `rotary`, K is rotated at `positions` on the way and q, if given, into q_out."""
        tokens = k.shape[0]
        dtype, device, head_dim = self.dtype, self.device, self.head_dim
        rk = _PACK_ROWS(*_rows(k, "k", dtype, device, self.kv_heads, head_dim, tokens))
        rv = _PACK_ROWS(*_rows(v, "v", dtype, device, self.kv_heads, head_dim, tokens))
        to = _vector(slots, "slots", torch.int64, device, tokens)
        handle = at = rq = ro = None
        if (q is None) != (q_out is None) or (rotary is None) != (positions is None) or (q is not None and rotary is None):
            raise ValueError("q and q_out come together, rotary and positions too, and q only with rotary")
        if rotary is not None:
            if rotary.device != device or rotary.head_dim != head_dim:
                raise ValueError(f"the rotary positions must be on {device} for heads of {head_dim}")
            if not rotary.handle.value:
                raise ValueError("the rotary positions are closed")  # to the library that would be an append without them
            handle, at = rotary.handle, _vector(positions, "positions", torch.int64, device, tokens)
        if q is not None:
            if q.dim() != 3:
                raise ValueError("q must be [tokens, heads, head_dim]")
            heads = q.shape[1]
            rq = _PACK_ROWS(*_rows(q, "q", dtype, device, heads, head_dim, tokens))
            ro = _PACK_ROWS(*_rows(q_out, "q_out", dtype, device, heads, head_dim, tokens))
        if tokens == 0:
            return
        _call("ft_kv_cache_append", device, self.address, layer, rk, rv, to, tokens, handle, at, rq, ro, _stream(device, stream))

    def copy_pages(self, sources: torch.Tensor, targets: torch.Tensor, stream: Optional[torch.cuda.Stream] = None):
        """Copies page sources[i] to page targets[i] (int32) in every layer; no target may be a source or another target."""
        count = sources.shape[0]
        a, b = _vector(sources, "sources", torch.int32, self.device), _vector(targets, "targets", torch.int32, self.device, count)
        _call("ft_kv_cache_copy_pages", self.device, self.address, a, b, count, _stream(self.device, stream))

    def accept(self, page_table: torch.Tensor, lengths: torch.Tensor, drafted_offsets: torch.Tensor, accepted: torch.Tensor,
               accepted_offsets: torch.Tensor, new_lengths: torch.Tensor, stream: Optional[torch.cuda.Stream] = None):
        """Keeps the accepted ones of the drafted tokens at the end of each sequence: moves drafted token
        accepted[accepted_offsets[b] + i] (ascending) to the i-th place behind the tokens that were there before them, in every
        layer, and writes the lengths that result.  All int32; page_table [batch, pages]."""
        batch = lengths.shape[0]
        table, columns, stride = _matrix(page_table, "page_table", self.device, batch)
        held = _vector(lengths, "lengths", torch.int32, self.device)
        offsets = _vector(drafted_offsets, "drafted_offsets", torch.int32, self.device, batch + 1)
        nodes = _vector(accepted, "accepted", torch.int32, self.device)
        ends = _vector(accepted_offsets, "accepted_offsets", torch.int32, self.device, batch + 1)
        out = _vector(new_lengths, "new_lengths", torch.int32, self.device, batch)
        if batch == 0:
            return
        # an empty tensor has no address, but then nothing is read there
        _call("ft_kv_cache_accept", self.device, self.address, table, columns, stride, held, offsets, nodes or out, ends, batch, out,
              _stream(self.device, stream))


class PagePool:
    """Which sequence holds which page of a cache.  Forked sequences share pages until one of them writes to a page that it
    shares; `extend` and `compact` move contents with the cache's copy_pages on `stream`.  All of it is host work: a captured
    step leaves it out, and takes the tables, lengths and slots that it gives from buffers filled before each replay."""

    def __init__(self, pages: int, page_size: int, cache: Optional[PagedCache] = None):
        if cache is not None and (cache.pages < pages or cache.page_size != page_size):
            raise ValueError(f"the cache has {cache.pages} pages of {cache.page_size} tokens")
        self.lib = _lib()
        self.pages, self.page_size, self.cache = pages, page_size, cache
        self.handle = ctypes.c_void_p()
        _abi.check(self.lib.ft_page_pool_create(ctypes.byref(self.handle), pages, page_size))

    @staticmethod
    def _value(code: int) -> int:
        if code < 0:
            _abi.check(code)
        return code

    def free_pages(self) -> int:
        return self._value(self.lib.ft_page_pool_free_pages(self.handle))

    def new_sequence(self) -> int:
        out = ctypes.c_int()
        _abi.check(self.lib.ft_page_pool_new_sequence(self.handle, ctypes.byref(out)))
        return out.value

    def fork(self, sequence: int) -> int:
        out = ctypes.c_int()
        _abi.check(self.lib.ft_page_pool_fork(self.handle, sequence, ctypes.byref(out)))
        return out.value

    def free(self, sequence: int):
        _abi.check(self.lib.ft_page_pool_free(self.handle, sequence))

    def truncate(self, sequence: int, length: int):
        _abi.check(self.lib.ft_page_pool_truncate(self.handle, sequence, length))

    def length(self, sequence: int) -> int:
        return self._value(self.lib.ft_page_pool_length(self.handle, sequence))

    def page_list(self, sequence: int) -> List[int]:
        out = (ctypes.c_int * self.pages)()
        return list(out[:self._value(self.lib.ft_page_pool_pages(self.handle, sequence, out, self.pages))])

    def _check_stream(self, stream: Optional[torch.cuda.Stream]):
        """Refuses what the copies could not be made on, before anything changes."""
        if self.cache is None:
            return
        if stream is not None:
            _stream(self.cache.device, stream)
        with torch.cuda.stream(stream) if stream is not None else torch.cuda.device(self.cache.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the page pool works on the host: a captured step leaves it out")

    def _move(self, pairs: List[Tuple[int, int]], stream: Optional[torch.cuda.Stream]):
        if pairs and self.cache is not None:
            with torch.cuda.stream(stream) if stream is not None else torch.cuda.device(self.cache.device):
                both = torch.tensor(pairs, dtype=torch.int32).t().contiguous().to(self.cache.device)
                self.cache.copy_pages(both[0], both[1])

    def extend(self, sequences: Sequence[int], counts: Sequence[int], stream: Optional[torch.cuda.Stream] = None) -> List[Tuple[int, int]]:
        """Makes room for counts[i] more tokens behind sequences[i]; returns the (source, target) pages that were copied because
        a sequence was about to write to a page it shared.  Raises where the pages do not suffice; sequences before that one keep
        their room."""
        if len(sequences) != len(counts):
            raise ValueError("one count for each sequence")
        self._check_stream(stream)
        pairs = []
        try:
            for sequence, count in zip(sequences, counts):
                a, b = ctypes.c_int(), ctypes.c_int()
                _abi.check(self.lib.ft_page_pool_extend(self.handle, sequence, count, ctypes.byref(a), ctypes.byref(b)))
                if a.value >= 0:
                    pairs.append((a.value, b.value))
        finally:
            self._move(pairs, stream)
        return pairs

    def compact(self, stream: Optional[torch.cuda.Stream] = None) -> List[Tuple[int, int]]:
        """Moves the used pages to the front of the cache; page tables made before are no longer right."""
        self._check_stream(stream)
        a, b, n = (ctypes.c_int * self.pages)(), (ctypes.c_int * self.pages)(), ctypes.c_int()
        _abi.check(self.lib.ft_page_pool_compact(self.handle, a, b, self.pages, ctypes.byref(n)))
        pairs = list(zip(a[:n.value], b[:n.value]))
        self._move(pairs, stream)
        return pairs

    def slots(self, sequence: int, first: int, count: int) -> List[int]:
        """Slots of the places [first, first + count) of a sequence, for `PagedCache.append`."""
        if first < 0 or count < 0 or first + count > self.length(sequence):
            raise ValueError(f"sequence {sequence} holds {self.length(sequence)} tokens")
        pages = self.page_list(sequence)
        return [pages[i // self.page_size] * self.page_size + i % self.page_size for i in range(first, first + count)]

    def table(self, sequences: Sequence[int], device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
        """(page table [sequences, pages] with -1 behind a sequence's last page, lengths), both int32 on the device."""
        lists = [self.page_list(s) for s in sequences]
        width = max([1] + [len(p) for p in lists])
        table = torch.tensor([p + [-1] * (width - len(p)) for p in lists], dtype=torch.int32).reshape(len(lists), width)
        return table.to(device), torch.tensor([self.length(s) for s in sequences], dtype=torch.int32).to(device)

    def close(self):
        if getattr(self, "handle", None) is not None and self.handle.value:
            self.lib.ft_page_pool_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class _Attention:
    """What both attention operators hold: the status word that a wait which gives up writes to."""

    def _begin(self, device):
        self.lib = _lib()
        self.device = torch.empty(0, device=device).device
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.status_at = self.status.data_ptr()
        with torch.cuda.device(self.device):
            self.workspace_bytes = self.lib.ft_attention_workspace()
            # the status word is zero before any other stream can run a kernel that writes to it
            torch.cuda.current_stream().synchronize()

    def _launch(self, name: str, device: torch.device, stream: int, *args):
        """The call with a workspace of its own from torch's allocator, which belongs to `stream`: given back at once, it is used
        again by what follows on that stream only.  (A tensor for it takes a microsecond longer.)"""
        if _get_device() != device.index:
            with torch.cuda.device(device):
                return self._launch(name, device, stream, *args)
        workspace = _raw_alloc(self.workspace_bytes, stream)
        try:
            code = _calls[name](*args, workspace, self.workspace_bytes, self.status_at, stream)
        finally:
            _raw_delete(workspace)
        if code:
            _abi.check(code)

    def report(self):
        """Waits for the device and raises if the output of an earlier run is not valid: a device-side wait gave up, or packed
        prompts made more tiles than can be numbered.  What was reported once does not count against later runs."""
        torch.cuda.synchronize(self.device)
        code = int(self.status.item())
        if code != _abi.FT_OK:
            self.status.zero_()
            torch.cuda.synchronize(self.device)  # before any stream runs a kernel that writes to it
            why = "an earlier run had too many tiles and wrote nothing" if code == _abi.FT_ERR_INVALID else (
                "a device-side wait expired; the output of an earlier run is not valid")
            raise _abi.FtGemmError(code, why)


class PromptAttention(_Attention):
    """softmax(scale * Q K^T) V over packed prompts: sequence b has the tokens offsets[b] .. offsets[b+1] of q
    [tokens, heads, head_dim] and of k, v [tokens, key heads, head_dim]; query head h reads key head
    h // (heads // key heads).  causal: the last query sees every key of its sequence."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, causal: bool = True, scale: float = 0.0,
                 device="cuda"):
        self.code, self.causal, self.scale = _check_dtype(dtype), int(causal), scale
        self.heads, self.kv_heads, self.head_dim, self.dtype = heads, kv_heads, head_dim, dtype
        self._begin(device)

    def run(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, offsets: torch.Tensor,
            key_offsets: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
        """offsets, key_offsets (None: the same): int32 [sequences + 1]; lse: float32 [tokens, heads] or None.  Rows of out
        behind the last sequence are left as they are."""
        dtype, device, heads, kv_heads, head_dim, tokens, keys = self.dtype, self.device, self.heads, self.kv_heads, self.head_dim, len(q), len(k)
        rows = _rows(q, "q", dtype, device, heads, head_dim, tokens) + _rows(k, "k", dtype, device, kv_heads, head_dim, keys) + _rows(
            v, "v", dtype, device, kv_heads, head_dim, keys) + _rows(out, "out", dtype, device, heads, head_dim, tokens)
        batch = len(offsets) - 1
        at = _vector(offsets, "offsets", torch.int32, device)
        if key_offsets is None and keys != tokens:
            raise ValueError("key_offsets are needed where q and k differ in tokens")
        key_at = 0 if key_offsets is None else _vector(key_offsets, "key_offsets", torch.int32, device, batch + 1)
        lse_at = 0 if lse is None else _lse(lse, device, tokens, heads)
        if batch <= 0 or tokens == 0:
            return
        args = _PACK_PROMPT(*rows, lse_at, at, key_at, batch, tokens, keys, head_dim, self.code, self.causal, self.scale)
        self._launch("ft_prompt_attention_run", device, _stream(device, stream), args)


class TreeAttention(_Attention):
    """Attention of new tokens over a `PagedCache`: one token of each sequence (decoding), a chain of them (a piece of a
    prompt over its cached start), or a tree of drafted tokens given by a mask."""

    def __init__(self, heads: int, cache: PagedCache, scale: float = 0.0):
        self.cache, self.heads = cache, heads
        self.scale = scale
        self._begin(cache.device)

    def run(self, q: torch.Tensor, layer: int, offsets: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, out: torch.Tensor,
            mask: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
        """Sequence b holds lengths[b] tokens in the pages of page_table[b]; the queries of its last offsets[b+1] - offsets[b]
        ones are q[offsets[b]:offsets[b+1]].  They see every token before them, and of themselves what the mask says: int32 words
        [tokens, words], bit j of a row is set where the row sees new token j of its sequence; None: each sees up to itself."""
        cache, device, heads, tokens = self.cache, self.device, self.heads, len(q)
        rows = _rows(q, "q", cache.dtype, device, heads, cache.head_dim, tokens) + _rows(out, "out", cache.dtype, device, heads, cache.head_dim, tokens)
        batch = len(offsets) - 1
        at = _vector(offsets, "offsets", torch.int32, device)
        table, columns, table_stride = _matrix(page_table, "page_table", device, batch)
        held = _vector(lengths, "lengths", torch.int32, device, batch)
        mask_at, words, mask_stride = (0, 0, 0) if mask is None else _matrix(mask, "mask", device, tokens)
        lse_at = 0 if lse is None else _lse(lse, device, tokens, heads)
        if batch <= 0 or tokens == 0:
            return
        args = _PACK_TREE(*rows, lse_at, at, table, held, mask_at, words, mask_stride, batch, tokens, columns, table_stride, layer, self.scale)
        self._launch("ft_tree_attention_run", device, _stream(device, stream), cache.address, args)


def _lse(lse: torch.Tensor, device: torch.device, tokens: int, heads: int) -> int:
    if lse.dtype != torch.float32 or lse.device != device or lse.shape != (tokens, heads) or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 [{tokens}, {heads}] tensor on {device}")
    return lse.data_ptr()


def tree_mask(parents: Sequence[int], words: Optional[int] = None) -> torch.Tensor:
    """Mask rows (int32, on the CPU) of a tree of drafted tokens: parents[i] < i, or negative for a root; bit j of row i
    is set where j is i or an ancestor of i."""
    nodes = len(parents)
    words = max(1, -(-nodes // 32)) if words is None else words
    out = torch.zeros((nodes, words), dtype=torch.int32)
    _abi.check(_lib().ft_tree_mask((ctypes.c_int * max(1, nodes))(*parents), nodes,
                                   ctypes.cast(out.data_ptr(), ctypes.POINTER(ctypes.c_uint32)), words))
    return out

"""Serving with alpha-entmax attention: a paged key/value cache held in 4 bits.

``QuantizedKVCache`` owns the pool.  ``write`` quantises new tokens' keys and
values into it, ``attention`` attends to a sequence's cached keys in place
(the exact alpha-entmax threshold, like ``splash_attention(...,
tau_mode="exact")``), and ``read`` gives the cached values back, e.g. for a
chunk of a prompt that goes through ``splash_attention``.  The format and the
C entry points are in ``include/adasplash.h`` (asa_cache); the reference has
no cache.

Positions, pages and lengths stay on the GPU: no call synchronises, and every
call can be captured into a graph.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib, ops

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_QUERIES = 64     # query tokens per sequence of one attention call
GROUP = 32           # channels that share a scale and an offset


def _i32(t, shape, device, name: str) -> torch.Tensor:
    """An integer argument as contiguous int32 on `device`; values outside
    int32 become its bounds (no page, or a length past every page)."""
    if (type(t) is torch.Tensor and t.dtype is torch.int32 and t.shape == shape
            and t.device == device and t.is_contiguous()):
        return t  # the common case: one comparison each
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise TypeError(f"{name} must be an integer tensor, got {t.dtype}")
    if t.dim() != len(shape) or any(a is not None and a != b for a, b in zip(shape, t.shape)):
        want = ", ".join("*" if a is None else str(a) for a in shape)
        raise ValueError(f"{name} must have shape [{want}], got {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError("All tensors must be on same device")
    if t.dtype != torch.int32:
        if t.dtype == torch.int64:
            t = t.clamp(-(2 ** 31), 2 ** 31 - 1)
        t = t.to(torch.int32)
    return t.contiguous()


def _table(t, rows, device) -> torch.Tensor:
    """A page table [rows, P] (rows None: any)."""
    if (type(t) is torch.Tensor and t.dtype is torch.int32 and t.dim() == 2 and t.device == device
            and (rows is None or t.size(0) == rows) and t.size(1) and t.is_contiguous()):
        return t
    t = _i32(t, (rows, None), device, "page_table")
    if t.size(1) < 1:
        raise ValueError(f"page_table must have a column, got shape {tuple(t.shape)}")
    return t


def _operand(t: torch.Tensor) -> tuple:
    """A [B, H, N, d] operand and the strides to pass for it (None: contiguous):
    the tensor where it lies, unless the channels are not next to each other
    or every stride is 0 (the C ABI's mark for a contiguous tensor)."""
    if t.is_contiguous():
        return t, None
    if (t.size(-1) > 1 and t.stride(-1) != 1) or not any(ops.strides_of(t)):
        return t.contiguous(), None
    return t, ops.strides_of(t)


def _stream(dev: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _on_device(dev: torch.device, fn, *args):
    if torch.cuda.current_device() == dev.index:
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _no_grad(*ts) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise RuntimeError("the 4-bit cache has no gradients; call it under torch.no_grad() or "
                           "with detached tensors")


class QuantizedKVCache:
    """A pool of pages of 4-bit keys and values.

    Args:
      num_pages: pages of the pool.
      kv_heads: key/value heads.
      head_dim: 1..128.
      page_size: tokens of a page, 16, 32, 64, 128 or 256.
      device: the GPU that holds it.

    A row (a token's key or value of one head) takes 20 bytes per 32 channels:
    4-bit codes, and a bfloat16 scale and offset (asa_cache in adasplash.h).
    ``page_table`` [B, P] integers throughout: position t of sequence b is row
    ``t % page_size`` of page ``page_table[b, t // page_size]``.  An entry that
    is not a page of the pool (e.g. -1) holds nothing: its positions are not
    written, read as zeros and are seen by no query.
    """

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 device="cuda"):
        c = self._describe(num_pages, kv_heads, head_dim, page_size)
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("Tensors must be on CUDA device")
        shape, G = (c.pages, c.kv_heads, c.page_size), -(-c.head_dim // GROUP)
        codes = dict(size=shape + (16 * G,), dtype=torch.uint8, device=dev)
        params = dict(size=shape + (G, 2), dtype=torch.bfloat16, device=dev)
        self._hold(c, *(torch.zeros(**a) for a in (codes, params, codes, params)))

    @staticmethod
    def _describe(pages, kv_heads, head_dim, page_size) -> _lib.Cache:
        pages, kv_heads, head_dim, page_size = (int(x) for x in (pages, kv_heads, head_dim,
                                                                 page_size))
        if pages < 1 or kv_heads < 1:
            raise ValueError(f"num_pages ({pages}) and kv_heads ({kv_heads}) must be at least 1")
        if head_dim > ops.MAX_HEAD_DIM:
            raise ops.HeadDimError("Head dimension too large; increase D_MAX")
        if head_dim < 1:
            raise ValueError("head dimension must be at least 1")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        return _lib.Cache(pages, kv_heads, page_size, head_dim)

    def _hold(self, c: _lib.Cache, k_codes, k_params, v_codes, v_params) -> None:
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        c.k_codes, c.v_codes = k_codes.data_ptr(), v_codes.data_ptr()
        c.k_params, c.v_params = k_params.data_ptr(), v_params.data_ptr()
        self._c = c
        self.num_pages, self.kv_heads = c.pages, c.kv_heads
        self.page_size, self.head_dim = c.page_size, c.head_dim
        self.device = k_codes.device
        self._ref = ctypes.byref(c)
        self._workspaces = {}  # bytes by call shape

    @classmethod
    def from_tensors(cls, k_codes, k_params, v_codes, v_params, head_dim: int) -> "QuantizedKVCache":
        """A cache over existing pool tensors (e.g. loaded from a file), which
        it uses in place: codes uint8 [pages, kv_heads, page_size, 16 G] and
        params bfloat16 [pages, kv_heads, page_size, G, 2], G = ceil(head_dim
        / 32)."""
        for name, t in (("k_codes", k_codes), ("k_params", k_params), ("v_codes", v_codes),
                        ("v_params", v_params)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a tensor")
            if not t.is_cuda:
                raise RuntimeError("Tensors must be on CUDA device")
            if t.device != k_codes.device:
                raise RuntimeError("All tensors must be on same device")
            want = torch.uint8 if name.endswith("codes") else torch.bfloat16
            if t.dtype != want:
                raise TypeError(f"{name} must be {want}, got {t.dtype}")
        if k_codes.dim() != 4:
            raise ValueError(f"k_codes must be 4-D, got shape {tuple(k_codes.shape)}")
        c = cls._describe(k_codes.size(0), k_codes.size(1), head_dim, k_codes.size(2))
        G = -(-c.head_dim // GROUP)
        shape = tuple(k_codes.shape[:3])
        for name, t, tail in (("k_codes", k_codes, (16 * G,)), ("v_codes", v_codes, (16 * G,)),
                              ("k_params", k_params, (G, 2)), ("v_params", v_params, (G, 2))):
            if tuple(t.shape) != shape + tail:
                raise ValueError(f"{name} must have shape {shape + tail}, got {tuple(t.shape)}")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be contiguous and 16-byte aligned")
        self = cls.__new__(cls)
        self._hold(c, k_codes, k_params, v_codes, v_params)
        return self

    def nbytes(self) -> int:
        """Bytes of the pool."""
        return 2 * (self.k_codes.numel() + 2 * self.k_params.numel())

    def __repr__(self) -> str:
        return (f"QuantizedKVCache(num_pages={self.num_pages}, kv_heads={self.kv_heads}, "
                f"head_dim={self.head_dim}, page_size={self.page_size}, device='{self.device}')")

    def tensors(self) -> tuple:
        """(k_codes, k_params, v_codes, v_params), as from_tensors takes them."""
        return self.k_codes, self.k_params, self.v_codes, self.v_params

    def write(self, K, V, page_table, start, counts=None) -> None:
        """Quantise tokens into the cache: token i < counts[b] (None: every
        token) of sequence b, K[b, :, i] and V[b, :, i], goes to position
        start[b] + i.

        K, V: [B, kv_heads, n, head_dim] of one type (float32, bfloat16 or
        float16), with any strides (read in place where the channels are next
        to each other).  start, counts: [B] integers.  Every other row stays
        as it is.  Two tokens of one call must not share a row (which of the
        two rows' bytes stay is not defined): sequences that share pages write
        to them in different calls.  check_write tells."""
        if torch.compiler.is_compiling():
            from . import library
            return library.cache_write(self, K, V, page_table, start, counts)
        write_tokens(self, K, V, page_table, start, counts)

    def check_write(self, page_table, start, n: int, counts=None) -> None:
        """Debug check (synchronises): raises ValueError if a write of n
        tokens per sequence with these arguments had a token without a row,
        or two tokens with the same one."""
        dev = self.device
        table = _table(page_table, None, dev).long()
        B, P = table.shape
        start = _i32(start, (B,), dev, "start").long()
        i = torch.arange(int(n), device=dev)
        live = torch.ones((B, int(n)), dtype=torch.bool, device=dev)
        if counts is not None:
            live = i < _i32(counts, (B,), dev, "counts")[:, None]
        at = start[:, None] + i
        col = at // self.page_size
        page = table.gather(1, col.clamp(0, P - 1))
        fine = (at >= 0) & (col < P) & (page >= 0) & (page < self.num_pages)
        if bool((live & ~fine).any()):
            raise ValueError("a token has no row: its position is negative or past the page "
                             "table, or its entry is not a page of the cache")
        rows = (page * self.page_size + at % self.page_size)[live]
        if rows.unique().numel() != rows.numel():
            raise ValueError("two tokens go to the same row")

    def read(self, page_table, lengths, n: int | None = None, dtype=torch.bfloat16, start=None):
        """The cached keys and values (K, V), [B, kv_heads, n, head_dim], of
        positions start[b] + i, i < n (start None: 0; n None: every position
        of the page table); zeros at positions at or past lengths[b]."""
        if torch.compiler.is_compiling():
            from . import library
            return library.cache_read(self, page_table, lengths, n, dtype, start)
        return read_tokens(self, page_table, lengths, n, dtype, start)

    def attention(self, Q, page_table, lengths, Q_idx=None, alpha: float = 1.5,
                  sm_scale: float | None = None, max_length: int | None = None) -> torch.Tensor:
        """``cache_attention(Q, self, ...)``."""
        return cache_attention(Q, self, page_table, lengths, Q_idx, alpha, sm_scale, max_length)


def check_tokens(cache, K, V) -> None:
    if (type(K) is torch.Tensor and type(V) is torch.Tensor and K.dtype in ops.INPUT_DTYPES
            and V.dtype is K.dtype and K.dim() == 4 and V.shape == K.shape and K.numel()
            and K.size(1) == cache.kv_heads and K.size(3) == cache.head_dim
            and K.is_cuda and K.device == cache.device and V.device == cache.device
            and not (K.requires_grad or V.requires_grad)):
        return
    for name, t in (("K", K), ("V", V)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D [B, H, N, d], got shape {tuple(t.shape)}")
    if K.dtype not in ops.INPUT_DTYPES:
        raise TypeError(f"unsupported dtype {K.dtype}; use torch.float32, torch.bfloat16 "
                        "or torch.float16")
    if V.dtype != K.dtype:
        raise TypeError("K and V must have the same dtype")
    if V.shape != K.shape:
        raise ValueError(f"V shape {tuple(V.shape)} must equal K shape {tuple(K.shape)}")
    B, H, n, d = K.shape
    if H != cache.kv_heads or d != cache.head_dim:
        raise ValueError(f"K shape {tuple(K.shape)} does not match the cache's {cache.kv_heads} "
                         f"heads of {cache.head_dim}")
    if B < 1 or n < 1:
        raise ValueError("no tokens to write")
    if not K.is_cuda:
        raise RuntimeError("Tensors must be on CUDA device")
    if K.device != cache.device or V.device != cache.device:
        raise RuntimeError("All tensors must be on same device")
    _no_grad(K, V)


def write_tokens(cache, K, V, page_table, start, counts=None) -> None:
    """QuantizedKVCache.write without the torch.compile dispatch."""
    check_tokens(cache, K, V)
    dev = cache.device
    B, _, n, _ = K.shape
    table = _table(page_table, B, dev)
    start = _i32(start, (B,), dev, "start")
    counts = None if counts is None else _i32(counts, (B,), dev, "counts")
    K, ks = _operand(K)
    V, vs = _operand(V)
    t = _lib.CacheTokens(B, n, ops._DTYPES[K.dtype], table.size(1), table.data_ptr(), start.data_ptr())
    if ks:
        t.k_strides[:] = ks
    if vs:
        t.v_strides[:] = vs
    _lib.check(_on_device(dev, _lib.load().asa_cache_write, cache._ref, ctypes.byref(t),
                          None if counts is None else counts.data_ptr(), K.data_ptr(),
                          V.data_ptr(), _stream(dev)))


def read_tokens(cache, page_table, lengths, n=None, dtype=torch.bfloat16, start=None):
    """QuantizedKVCache.read without the torch.compile dispatch."""
    if dtype not in ops.INPUT_DTYPES:
        raise TypeError(f"unsupported dtype {dtype}; use torch.float32, torch.bfloat16 "
                        "or torch.float16")
    dev = cache.device
    table = _table(page_table, None, dev)
    B = table.size(0)
    n = table.size(1) * cache.page_size if n is None else int(n)
    if B < 1 or n < 1:
        raise ValueError("no tokens to read")
    lengths = _i32(lengths, (B,), dev, "lengths")
    start = None if start is None else _i32(start, (B,), dev, "start")
    K = torch.empty((B, cache.kv_heads, n, cache.head_dim), dtype=dtype, device=dev)
    V = torch.empty_like(K)
    t = _lib.CacheTokens(B, n, ops._DTYPES[dtype], table.size(1), table.data_ptr(),
                         None if start is None else start.data_ptr())
    _lib.check(_on_device(dev, _lib.load().asa_cache_read, cache._ref, ctypes.byref(t),
                          lengths.data_ptr(), K.data_ptr(), V.data_ptr(), _stream(dev)))
    return K, V


def check_query(cache, Q, max_length=None) -> None:
    if (type(Q) is torch.Tensor and type(cache) is QuantizedKVCache and max_length is None
            and Q.dtype in ops.INPUT_DTYPES and Q.dim() == 4 and Q.numel()
            and Q.size(3) == cache.head_dim and Q.size(1) % cache.kv_heads == 0
            and Q.size(2) <= MAX_QUERIES and Q.is_cuda and Q.device == cache.device and not Q.requires_grad):
        return
    if not isinstance(cache, QuantizedKVCache):
        raise TypeError("cache must be a QuantizedKVCache")
    if not isinstance(Q, torch.Tensor):
        raise TypeError("Q must be a tensor")
    if Q.dim() != 4:
        raise ValueError(f"Q must be 4-D [B, H, N, d], got shape {tuple(Q.shape)}")
    if Q.dtype not in ops.INPUT_DTYPES:
        raise TypeError(f"unsupported dtype {Q.dtype}; use torch.float32, torch.bfloat16 "
                        "or torch.float16")
    B, H, NQ, d = Q.shape
    if d != cache.head_dim:
        raise ValueError(f"Q head dim {d} does not match the cache's {cache.head_dim}")
    if B < 1 or NQ < 1 or H < 1:
        raise ValueError("empty attention problem")
    if H % cache.kv_heads:
        raise ValueError(f"{H} query heads are not a multiple of the cache's {cache.kv_heads}")
    if NQ > MAX_QUERIES:
        raise ValueError(f"{NQ} query tokens per sequence, at most {MAX_QUERIES}; for a longer "
                         "chunk read the cache back and call splash_attention")
    if max_length is not None and int(max_length) < 1:
        raise ValueError(f"max_length must be at least 1, got {max_length}")
    if not Q.is_cuda:
        raise RuntimeError("Tensors must be on CUDA device")
    if Q.device != cache.device:
        raise RuntimeError("All tensors must be on same device")
    _no_grad(Q)


def attend(cache, Q, page_table, lengths, Q_idx, alpha: float, sm_scale: float,
           max_length=None) -> torch.Tensor:
    """cache_attention without the torch.compile dispatch."""
    check_query(cache, Q, max_length)
    lib, dev = _lib.load(), cache.device
    B, H, NQ, d = Q.shape
    table = _table(page_table, B, dev)
    lengths = _i32(lengths, (B,), dev, "lengths")
    Q_idx = None if Q_idx is None else _i32(Q_idx, (B, NQ), dev, "Q_idx")
    Q, qs = _operand(Q)
    out = torch.empty_like(Q, memory_format=torch.contiguous_format)
    P = table.size(1)
    most = 0 if max_length is None else min(int(max_length), 2 ** 31 - 1)
    dtype = ops._DTYPES[Q.dtype]
    a = _lib.CacheQuery(B, H, NQ, dtype, P, most, alpha, sm_scale, table.data_ptr(),
                        lengths.data_ptr(), None if Q_idx is None else Q_idx.data_ptr())
    if qs:
        a.q_strides[:] = qs
    ref = ctypes.byref(a)
    key = (B, H, NQ, dtype, P, most)
    need = cache._workspaces.get(key)
    if need is None:
        if len(cache._workspaces) >= 1024:
            cache._workspaces.clear()
        z = ctypes.c_size_t()
        _lib.check(_on_device(dev, lib.asa_cache_attention_workspace, cache._ref, ref,
                              ctypes.byref(z)))
        need = cache._workspaces[key] = z.value
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.check(_on_device(dev, lib.asa_cache_attention, cache._ref, ref, Q.data_ptr(),
                          out.data_ptr(), None if ws is None else ws.data_ptr(), _stream(dev)))
    return out


def cache_attention(Q, cache: QuantizedKVCache, page_table, lengths, Q_idx=None, alpha: float = 1.5,
                    sm_scale: float | None = None, max_length: int | None = None) -> torch.Tensor:
    """alpha-entmax attention of a few query tokens per sequence over a 4-bit
    cache: what ``splash_attention(..., tau_mode="exact")`` gives on the
    cached values, without reading them back.

    Q: [B, H, NQ, d], H a multiple of the cache's kv_heads (query head j reads
    key head j // (H // kv_heads)), 1 <= NQ <= 64; float32, bfloat16 or
    float16, any strides.
    page_table: [B, P]; lengths: [B] cached tokens (the query tokens' own keys
    among them, if they are to be seen).
    Q_idx: [B, NQ] positions of the query tokens (None: the last NQ of each
    sequence); query i of sequence b sees the keys at positions <= Q_idx[b, i]
    and below lengths[b].  A row that sees none gives zeros.
    max_length: a bound on the lengths that the caller knows; keys past it are
    not seen.  The launch and its workspace (4 bytes per query row and key for
    long sequences) are sized by it, or by the page table's width.
    Inference only: tensors that need gradients are refused."""
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(Q.size(-1))
    if torch.compiler.is_compiling():
        from . import library
        return library.cache_attention(cache, Q, page_table, lengths, Q_idx, float(alpha),
                                       float(sm_scale), max_length)
    return attend(cache, Q, page_table, lengths, Q_idx, float(alpha), float(sm_scale), max_length)

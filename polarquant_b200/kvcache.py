"""Compressed key-value cache for a language model's attention.

The keys and values of past tokens are what Quantizer compresses everywhere
else in this package: vectors, stored as a norm and packed Lloyd-Max codes of
the rotated unit vector.  ``KVCache`` keeps them in pages, ``append`` writes
tokens, ``attend`` computes the attention of one new token of each sequence
without decompressing the cache (scores are the ADC inner product with the
rotated query), ``evict`` cuts sequences down to their most attended tokens and
``read`` gives tokens back as vectors.  No counterpart in the reference.

Every method enqueues kernels on the current stream of the cache's device and
returns without waiting; all can be captured into a CUDA graph.  Calls that
write pages (``append``, ``evict``, ``attend(accumulate=True)``) are ordered by
the caller against other calls on the same pages, as one stream does.
"""

from __future__ import annotations

import ctypes
import math
from typing import Dict, Optional, Tuple, Union

import numpy as np
import torch

from . import _lib
from .core import Quantizer
from .device import ptr, require_cuda, row_stride, stream_ptr, to_device_f32, workspace

MAX_D = 256
BITS = (2, 4, 8)
TURN_ROWS = 131072  # the encoder's chunk: a call of no more rows stays on the caller's stream
PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class KVCodec:
    """One side's tables (rotation, boundaries, centroids) on a device.

    rotation: (d, d), orthonormal rows (to 1e-2 in every entry of R R^T, so one
    rounded to bf16 is taken); boundaries: (2^bits - 1,) ascending; centroids:
    (2^bits,); arrays or tensors.  bits is 2, 4 or 8 and d at most 256.

    Making one checks and lays out the tables and waits for the device: once for
    a model's rotation, not once a cache or a step."""

    def __init__(self, rotation, boundaries, centroids, device: Optional[torch.device] = None):
        if device is None:
            device = rotation.device if isinstance(rotation, torch.Tensor) and rotation.is_cuda \
                else require_cuda()
        self.device = _device(device)
        shape = tuple(np.shape(rotation))
        if len(shape) != 2 or shape[0] != shape[1] or not 1 <= shape[0] <= MAX_D:
            raise ValueError(f"rotation must be (d, d) with 1 <= d <= {MAX_D}, got {shape}")
        self.d = int(shape[0])
        levels = int(np.prod(np.shape(centroids)))
        if len(np.shape(centroids)) != 1 or levels not in [1 << b for b in BITS]:
            raise ValueError(f"centroids must hold 4, 16 or 256 values (bits 2, 4 or 8), got "
                             f"{tuple(np.shape(centroids))}")
        self.bits = levels.bit_length() - 1
        if tuple(np.shape(boundaries)) != (levels - 1,):
            raise ValueError(f"boundaries must hold {levels - 1} values, got "
                             f"{tuple(np.shape(boundaries))}")
        # (copies: what was given may be used for something else afterwards)
        self.rotation = to_device_f32(rotation, self.device).detach().clone()
        self.boundaries = to_device_f32(boundaries, self.device).detach().clone()
        self.centroids = to_device_f32(centroids, self.device).detach().clone()
        if not bool((self.boundaries[1:] >= self.boundaries[:-1]).all()):
            raise ValueError("boundaries must ascend")
        if not bool(self.rotation.isfinite().all() & self.centroids.isfinite().all()):
            raise ValueError("rotation and centroids must be finite")
        # Codes are exact within a bound on sums of rows of length 1, and R^T turns back.
        r = self.rotation.cpu().double().numpy()
        off = np.abs(r @ r.T - np.eye(self.d)).max()
        if not off <= 1e-2:
            raise ValueError(f"rotation's rows must be orthonormal (an entry of R R^T is off by {off:.3g})")
        nbytes = _lib.query("pq_kv_codec_bytes", self.d, self.bits)
        self.tables = workspace(nbytes, self.device)
        with torch.cuda.device(self.device):
            _lib.call("pq_kv_prepare_codec", ptr(self.rotation), ptr(self.boundaries),
                      ptr(self.centroids), self.d, self.bits, ptr(self.tables), nbytes,
                      stream_ptr(self.device))
            torch.cuda.current_stream(self.device).synchronize()  # usable on every stream

    @classmethod
    def from_quantizer(cls, q: Quantizer, device: Optional[torch.device] = None) -> "KVCodec":
        """The tables of a Quantizer (2, 4 or 8 bits, d <= 256)."""
        if q.bits not in BITS:
            raise ValueError(f"a key-value cache holds 2, 4 or 8 bits, got bits={q.bits}")
        if q.d > MAX_D:
            raise ValueError(f"a key-value cache holds d <= {MAX_D}, got d={q.d}")
        return cls(q.R, q.boundaries, q.centroids, device)


def _device(device) -> torch.device:
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"the cache lives on a CUDA device, got {device}")
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


class KVCache:
    """Paged cache of compressed keys and values.

    key, value: a Quantizer or KVCodec each of the same d (``value`` defaults to
    ``key``; their bits may differ).  heads: key-value heads.  pages, page_size:
    the pool; page_size is a power of two from 16 to 1024.  buffers: existing
    tensors to use as the pool instead of new ones (``k_rows``, ``v_rows``,
    ``k_norms``, ``v_norms``, ``positions``, ``weights``, as the attributes of
    the same names).

    Pools are laid out [pages, heads, page_size]; rows have a fourth dimension,
    the packed row's stride (its bytes rounded up to 16).  A slot is
    ``page * page_size + offset``.  A sequence is a row of a page table and a
    length: token i lies in page ``table[i // page_size]`` at offset
    ``i % page_size``.  Which pages are free is the caller's to know."""

    def __init__(self, key: Union[Quantizer, KVCodec], value: Union[Quantizer, KVCodec, None] = None,
                 *, heads: int, pages: Optional[int] = None, page_size: int = 64,
                 device: Optional[torch.device] = None,
                 buffers: Optional[Dict[str, torch.Tensor]] = None):
        if device is None and buffers is not None and "k_rows" in buffers:
            device = buffers["k_rows"].device
        if isinstance(key, Quantizer):
            key = KVCodec.from_quantizer(key, device)
        if value is None:
            value = key
        elif isinstance(value, Quantizer):
            value = KVCodec.from_quantizer(value, key.device if isinstance(key, KVCodec) else device)
        for name, c in (("key", key), ("value", value)):
            if not isinstance(c, KVCodec):
                raise TypeError(f"{name} must be a Quantizer or KVCodec, got {type(c).__name__}")
        if key.d != value.d:
            raise ValueError(f"key and value sizes differ: {key.d} and {value.d}")
        if key.device != value.device or (device is not None and _device(device) != key.device):
            raise ValueError("key, value and the cache must be on the same device")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if int(heads) < 1:
            raise ValueError(f"heads must be at least 1, got {heads}")
        self.key, self.value = key, value
        self.d, self.heads, self.page_size = key.d, int(heads), int(page_size)
        self.device = key.device
        if buffers is None:
            if pages is None or int(pages) < 0:
                raise ValueError("pages must be given and at least 0")
            self.pages = int(pages)
        else:
            if "k_rows" not in buffers:
                raise ValueError("buffers lack k_rows")
            self.pages = int(buffers["k_rows"].shape[0])
            if pages is not None and int(pages) != self.pages:
                raise ValueError(f"buffers hold {self.pages} pages, not {pages}")
        if self.pages * self.page_size >= 1 << 31 or self.pages * self.heads >= 1 << 31 \
                or self.pages * self.heads * self.page_size >= 1 << 32:
            raise ValueError("a pool has fewer than 2^31 slots and 2^32 rows")
        pool = (self.pages, self.heads, self.page_size)
        kinds = {"k_rows": (pool + (row_stride(self.d, key.bits),), torch.uint8),
                 "v_rows": (pool + (row_stride(self.d, value.bits),), torch.uint8),
                 "k_norms": (pool, torch.float32), "v_norms": (pool, torch.float32),
                 "positions": (pool, torch.int32), "weights": (pool, torch.float32)}
        for name, (shape, dtype) in kinds.items():
            if buffers is None:
                t = torch.zeros(shape, dtype=dtype, device=self.device)
            else:
                if name not in buffers:
                    raise ValueError(f"buffers lack {name}")
                t = buffers[name]
                if tuple(t.shape) != shape or t.dtype != dtype or t.device != self.device \
                        or not t.is_contiguous() or t.data_ptr() % 16:
                    raise ValueError(f"buffer {name} must be a contiguous {dtype} tensor of shape "
                                     f"{shape} on {self.device}, 16-byte aligned")
            setattr(self, name, t)
        self._desc = _lib.KVCacheDesc(
            k_rows=self.k_rows.data_ptr(), v_rows=self.v_rows.data_ptr(),
            k_norms=self.k_norms.data_ptr(), v_norms=self.v_norms.data_ptr(),
            positions=self.positions.data_ptr(), weights=self.weights.data_ptr(),
            k_codec=key.tables.data_ptr(), v_codec=value.tables.data_ptr(),
            k_ldb=kinds["k_rows"][0][3], v_ldb=kinds["v_rows"][0][3], pages=self.pages,
            heads=self.heads, page_size=self.page_size, d=self.d, k_bits=key.bits,
            v_bits=value.bits)
        self._ref = ctypes.byref(self._desc)
        self._scale = 1.0 / math.sqrt(self.d)
        self._sizes: Dict[tuple, int] = {}

    @property
    def nbytes(self) -> int:
        """Bytes of the pool."""
        return sum(t.numel() * t.element_size() for t in
                   (self.k_rows, self.v_rows, self.k_norms, self.v_norms, self.positions,
                    self.weights))

    # -- checks ----------------------------------------------------------------
    # (A generation step calls attend and append once a layer, on work of a few
    # microseconds: sizes of workspaces are kept, and what is right is found right
    # in one comparison.)
    def _call(self, name: str, *args) -> None:
        """The entry point on the cache's device and its current stream."""
        index = self.device.index
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                _lib.call(name, self._ref, *args, stream_ptr(self.device))
        else:
            _lib.call(name, self._ref, *args, torch._C._cuda_getCurrentRawStream(index))

    def _workspace(self, name: str, *sizes: int) -> torch.Tensor:
        nbytes = self._sizes.get((name, sizes))
        if nbytes is None:
            nbytes = max(256, _lib.query(name, self._ref, *sizes))
            if len(self._sizes) >= 4096:
                self._sizes.clear()
            self._sizes[name, sizes] = nbytes
        return self.k_rows.new_empty(nbytes)

    def _tensor(self, name: str, t, dtype: torch.dtype, shape: Tuple[int, ...]) -> None:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.dtype is dtype and t.shape == shape and t.device == self.device:
            return
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")

    def _vectors(self, name: str, t, shape: Tuple[int, ...]) -> int:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        code = DTYPES.get(t.dtype)
        if code is None:
            raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if t.shape != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if self.d > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name}'s last dimension must be contiguous")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient, and a compressed cache has none: call "
                             f"under torch.no_grad() or detach it")
        return code

    def _vector(self, name: str, t, dtype: torch.dtype, n: int) -> None:
        self._tensor(name, t, dtype, (n,))
        if n > 1 and t.stride(0) != 1:
            raise ValueError(f"{name} must be contiguous")

    def _sequences(self, table, lengths) -> Tuple[int, int]:
        if not isinstance(table, torch.Tensor) or table.dim() != 2:
            raise ValueError("table must be a (sequences, pages) tensor")
        batch, width = shape = tuple(table.shape)
        self._tensor("table", table, torch.int32, shape)
        self._vector("lengths", lengths, torch.int32, batch)
        if width > 1 and table.stride(1) != 1:
            raise ValueError("table's last dimension must be contiguous")
        if width * self.page_size > 1 << 30:
            raise ValueError("a sequence has at most 2^30 tokens")
        return batch, width

    def _slots(self, slots) -> int:
        if not isinstance(slots, torch.Tensor) or slots.dim() != 1:
            raise ValueError("slots must be a 1-d tensor")
        n = slots.shape[0]
        self._vector("slots", slots, torch.int64, n)
        if n * self.heads >= 1 << 31:
            raise ValueError("a call takes fewer than 2^31 rows")
        return n

    # -- operators ---------------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               positions: torch.Tensor, weights: Optional[torch.Tensor] = None) -> None:
        """Compresses tokens into their slots.

        k, v: (n, heads, d) of one type (float32, float16 or bfloat16), any
        strides but the last.  slots: (n,) int64; a slot outside the pool (-1
        for the padding of a batch) skips its token.  The slots named in one
        call must differ: where two tokens name one slot, what it holds
        afterwards is not defined.  positions: (n,) int32, the tokens' places in
        their sequences, which ``evict`` goes by.  weights: (n, heads) float32,
        the accumulated attention they start with (0 by default).

        A row's norm and codes are Quantizer.encode's; vectors must be finite,
        and of norms below 2^100 for attend."""
        n = self._slots(slots)
        shape = (n, self.heads, self.d)
        code = self._vectors("k", k, shape)
        self._vectors("v", v, shape)
        if k.dtype != v.dtype:
            raise TypeError(f"k and v must have one type, got {k.dtype} and {v.dtype}")
        self._vector("positions", positions, torch.int32, n)
        if weights is not None:
            self._tensor("weights", weights, torch.float32, shape[:2])
            if not weights.is_contiguous():
                raise ValueError("weights must be contiguous")
        if n:
            self._call("pq_kv_append", k.data_ptr(), v.data_ptr(), code, n, k.stride(0), k.stride(1),
                       v.stride(0), v.stride(1), slots.data_ptr(), positions.data_ptr(),
                       0 if weights is None else weights.data_ptr())

    def read(self, slots: torch.Tensor, *, dtype: torch.dtype = torch.float32,
             rotated: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of slots as vectors, (n, heads, d) each of `dtype`.

        rotated=True leaves them in the codecs' rotated coordinates (norm times
        centroids), where attention can be computed with queries turned by
        ``key.rotation`` and outputs turned back by ``value.rotation``;
        otherwise they are turned back, as Quantizer.decode does.  Slots outside
        the pool give zeros."""
        n = self._slots(slots)
        if dtype not in DTYPES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        kind = dtype if rotated else torch.float32
        k, v = (self.weights.new_empty((n, self.heads, self.d), dtype=kind) for _ in range(2))
        if n:
            self._call("pq_kv_read", slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), DTYPES[kind])
        if not rotated:
            k, v = self._unrotate(k, self.key).to(dtype), self._unrotate(v, self.value).to(dtype)
        return k, v

    def _unrotate(self, x: torch.Tensor, codec: KVCodec) -> torch.Tensor:
        """x @ R for every vector, by the encoder's rotation kernel on R^T.

        In chunks of TURN_ROWS: calls of more rows are spread over streams that all
        encoders of the process share, which a capture would keep for itself."""
        rows = x.shape[0] * self.heads
        if not rows:
            return x
        y, size = torch.empty_like(x), self.d * x.element_size()
        with torch.cuda.device(self.device):
            st = stream_ptr(self.device)
            nb = _lib.query("pq_rotation_planes_bytes", self.d)
            planes = workspace(nb, self.device)
            turned = codec.rotation.t().contiguous()
            _lib.call("pq_prepare_rotation", ptr(turned), self.d, ptr(planes), nb, st)
            ws = workspace(_lib.query("pq_encode_workspace_bytes", min(rows, TURN_ROWS), self.d),
                           self.device)
            for at in range(0, rows, TURN_ROWS):
                _lib.call("pq_rotate_tc", x.data_ptr() + at * size, min(TURN_ROWS, rows - at), self.d,
                          ptr(planes), y.data_ptr() + at * size, ptr(ws), ws.numel(), st)
        return y

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
               scale: Optional[float] = None, accumulate: bool = False, return_lse: bool = False):
        """Attention of one token of each sequence over its cached tokens.

        q: (sequences, query heads, d), float32, float16 or bfloat16; the query
        heads are a multiple of the cache's heads, and query head h reads
        key-value head ``h // (query heads // heads)``.  table: (sequences,
        pages) int32, lengths: (sequences,) int32.  scale: 1/sqrt(d) by default.
        Returns (sequences, query heads, d) of q's type; with return_lse also
        the natural logarithm of each softmax's sum, (sequences, query heads)
        float32, by which the result can be joined with attention over tokens
        held elsewhere.  A sequence of length 0 gives 0 and -inf; tokens on
        pages outside the pool are passed over, and lengths above what the
        table has room for are taken as that.

        accumulate=True adds each token's softmax weight, summed over the query
        heads of its key-value head, to ``weights``, which ``evict`` goes by.
        (The sum of several sequences that share a page is taken in no fixed
        order.)  It takes 4 bytes of workspace for every query head and token that
        the table has room for, whatever the lengths: cut a wide table to the
        pages that the longest sequence needs.

        Scores are as exact as f32 allows for every type; values and their
        weights have 22 bits, for bfloat16 outputs 11."""
        batch, width = self._sequences(table, lengths)
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("q must be a (sequences, query heads, d) tensor")
        hq = q.shape[1]
        if hq == 0 or hq % self.heads:
            raise ValueError(f"query heads must be a multiple of the cache's {self.heads}, got {hq}")
        code = self._vectors("q", q, (batch, hq, self.d))
        if scale is None:
            scale = self._scale
        else:
            scale = float(scale)
            if not math.isfinite(scale):
                raise ValueError(f"scale must be finite, got {scale}")
        out = q.new_empty((batch, hq, self.d))
        lse = self.weights.new_empty((batch, hq)) if return_lse else None
        if batch:
            accumulate = int(bool(accumulate))
            ws = self._workspace("pq_kv_attend_workspace_bytes", batch, hq, width, accumulate)
            self._call("pq_kv_attend", q.data_ptr(), code, *q.stride()[:2], table.data_ptr(),
                       table.stride(0), width, lengths.data_ptr(), batch, hq, scale,
                       out.data_ptr(), lse.data_ptr() if return_lse else 0, accumulate,
                       ws.data_ptr(), ws.numel())
        return (out, lse) if return_lse else out

    def evict(self, table: torch.Tensor, lengths: torch.Tensor, budget: int, *, recent: int = 0,
              sinks: int = 0, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Cuts every longer sequence down to `budget` tokens, each head to its own.

        Kept are the tokens of positions below `sinks` and of the last `recent`
        positions (those after the largest position minus `recent`), then the
        ones of the largest accumulated ``weights``, ties to the lowest slot.
        Tokens kept from behind the budget take the places of evicted ones
        before it, in order; the others stay where they are.  Returns the new
        lengths, (sequences,) int32; pages behind them are free.  Tokens on pages
        outside the pool are not there: none is kept, and none is moved onto such
        a page, so that fewer than `budget` are left where the table has one (the
        new length counts such places).

        weights: (sequences, heads, tokens) float32 for prompts whose attention
        was computed elsewhere: token i has position i and this weight (the
        column sums of the prompt's attention, say), and the kept tokens'
        positions and weights are written to the cache.  A sequence longer than
        that is taken as that long.

        A page must belong to one sequence only: a shared prefix is copied, or
        left out of the table, before.  sequences * heads is below 65536.  (Wide
        tables get the kernel for long sequences: cut them as for ``attend``.)"""
        batch, table_width = self._sequences(table, lengths)
        for name, x in (("budget", budget), ("recent", recent), ("sinks", sinks)):
            if int(x) != x or not 0 <= x < 1 << 31:
                raise ValueError(f"{name} must be an integer in [0, 2^31), got {x}")
        given, width = (0, 0, 0), 0
        if weights is not None:
            if not isinstance(weights, torch.Tensor) or weights.dim() != 3:
                raise ValueError("weights must be a (sequences, heads, tokens) tensor")
            width = weights.shape[2]
            self._tensor("weights", weights, torch.float32, (batch, self.heads, width))
            if width > 1 and weights.stride(2) != 1:
                raise ValueError("weights' last dimension must be contiguous")
            given = (weights.data_ptr() or self.weights.data_ptr(), weights.stride(0),
                     weights.stride(1))
        new = self.positions.new_empty(batch)
        if batch:
            ws = self._workspace("pq_kv_evict_workspace_bytes", batch, table_width, int(budget))
            self._call("pq_kv_evict", table.data_ptr(), table.stride(0), table_width,
                       lengths.data_ptr(), batch, int(budget), int(recent), int(sinks), *given,
                       width, new.data_ptr(), ws.data_ptr(), ws.numel())
        return new

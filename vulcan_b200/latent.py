"""Rotary positions and the latent cache over the C ABI (include/vk_paged_kv.h).

* ``RotaryEmbedding`` — vk_rotary: q and k rotated in one launch, interleaved or
  half layout, the leading part of a head, frequencies scaled for long contexts.
* ``LatentKVPool`` — vk_latent: a paged cache of one latent vector and one shared
  rotary key part a token, its append (norm and rotation fused) and its
  attention in the absorbed form (decode) and the expanded form (prefill).  The
  page operations of ``PagedKVPool`` (alloc, free, copy, compaction, swap) work on it unchanged.

No reference counterpart: the reference has neither.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple

import torch

from . import _lib
from ._lib import check
from .paged_kv import PAGE_TOKENS, PagedKVPool

DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # VK_F16, VK_BF16, VK_F32
LAYOUTS = {"interleaved": 0, "half": 1}
SCALINGS = {None: 0, "linear": 1, "by_parts": 2, "by_wavelength": 3}


def _device(device) -> torch.device:
    if isinstance(device, torch.device) and device.index is not None:
        return device
    return torch.device("cuda", torch.cuda.current_device() if device is None or isinstance(device, torch.device)
                        else int(device))


# The calls below take a few microseconds of GPU time at their smallest, so the
# checks are kept to attribute reads.

def _stream_of(stream, index: int) -> int:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(index)
    return int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)


def _empty(shape, dtype, device: torch.device, stream) -> torch.Tensor:
    """Memory for a call on ``stream``: allocated on that stream, so the caching allocator hands it out again only
    behind the call (and a captured call keeps its own)."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(int(stream), device=device)
    with torch.cuda.stream(s):
        return torch.empty(shape, dtype=dtype, device=device)


def _on(t: torch.Tensor, dtype, name: str, index: int) -> None:
    if t.dtype is not dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if t.get_device() != index:
        raise ValueError("%s must be on cuda:%d, got %s" % (name, index, t.device))


def _workspace(given, need: int, like: torch.Tensor, index: int, stream) -> Tuple[torch.Tensor, int]:
    """(the call's scratch, its bytes): the caller's, or memory of its own."""
    if given is None:  # new_empty of a 16-bit tensor takes 1 us less than torch.empty
        return like.new_empty((need + 1 >> 1,)) if stream is None else _empty((need,), torch.uint8, like.device, stream), need
    if given.get_device() != index or not given.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor on cuda:%d" % index)
    return given, given.numel() * given.element_size()


def _i32(t: torch.Tensor, name: str, index: int, numel: int) -> int:
    _on(t, torch.int32, name, index)
    if t.numel() != numel or not t.is_contiguous():
        raise ValueError("%s must be contiguous with %d elements" % (name, numel))
    return t.data_ptr()


def _tables(t: torch.Tensor, index: int) -> Tuple[int, int]:
    """(batch, width) of the block tables."""
    _on(t, torch.int32, "block_tables", index)
    if t.dim() != 2 or not t.is_contiguous():
        raise ValueError("block_tables must be a contiguous [batch, width] tensor")
    return t.shape


def _token_head(t: torch.Tensor, name: str) -> Tuple[int, int]:
    """(token, head) strides of [tokens, heads, d] or [batch, tokens, heads, d] with unit stride along d and, in
    the second form, batches that follow one another."""
    s, shape = t.stride(), t.shape
    n = len(s)
    if n not in (3, 4) or (s[-1] != 1 and shape[-1] > 1):
        raise ValueError("%s must be [tokens, heads, d] or [batch, tokens, heads, d] with unit stride along d" % name)
    if n == 3:
        return s[0], s[1]
    if shape[1] == 1:
        return s[0], s[2]
    if s[0] != s[1] * shape[1] and shape[0] > 1 and shape[1]:
        raise ValueError("%s: the batches of a 4-D view must follow one another (stride 0 = stride 1 * tokens)" % name)
    return s[1], s[2]


class RotaryEmbedding:
    """Rotary positions (vk_rotary, see the C header for the scalings).

    ``rotary_dim`` leading elements of each head turn by position * f_i, with
    pairs (2i, 2i+1) (``layout="interleaved"``) or (i, i + rotary_dim/2)
    (``"half"``)."""

    def __init__(self, rotary_dim: int, theta: float = 10000.0, layout: str = "interleaved", scaling: Optional[str] = None,
                 factor: float = 1.0, original_len: float = 0.0, low: float = 1.0, high: float = 32.0,
                 magnitude: float = 0.0, device=None):
        if layout not in LAYOUTS:
            raise ValueError("layout must be one of %s" % sorted(LAYOUTS))
        if scaling not in SCALINGS:
            raise ValueError("scaling must be one of %s" % list(SCALINGS))
        self._lib = _lib.load()
        self.rotary_dim, self.layout, self.scaling = rotary_dim, layout, scaling
        # frequencies alone need no GPU: the device is looked up by the first apply
        self._cfg = _lib.VkRotaryCfg(rotary_dim, LAYOUTS[layout], SCALINGS[scaling], 0, theta, factor, original_len, low,
                                     high, magnitude)
        self.frequencies()
        self.handle = ctypes.c_void_p()
        self.device = _device(device) if torch.cuda.is_available() else torch.device("cpu")
        self._index = self._cfg.device = self.device.index or 0
        check(self._lib.vk_rotary_create(ctypes.byref(self._cfg), ctypes.byref(self.handle)), "vk_rotary_create")

    def frequencies(self) -> Tuple[List[float], float]:
        """(radians per position of each pair, factor on cos and sin), scaled, in double precision."""
        f = (ctypes.c_double * max(1, self.rotary_dim // 2))()
        m = ctypes.c_double()
        check(self._lib.vk_rotary_frequencies(ctypes.byref(self._cfg), f, ctypes.byref(m)), "vk_rotary_frequencies")
        return list(f), m.value

    def apply(self, q: torch.Tensor, positions: torch.Tensor, k: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None, stream=None):
        """q, k: [tokens, heads, D] (or [batch, tokens, heads, D]) fp16, bf16 or fp32, strided views allowed;
        positions: int32, one per token.  Returns the rotated q, or (q, k).  ``out``/``out_k`` may be q/k
        themselves: rotated in place (``out`` may not be k, nor ``out_k`` q)."""
        dev, index = self.device, self._index
        dtype, shape = q.dtype, q.shape
        if dtype not in DTYPES:
            raise TypeError("q must be fp16, bf16 or fp32, got %s" % dtype)
        d = shape[-1]
        y, view = self._view(q, out, "q", dtype, dev, index, stream)
        y_k = view_k = None
        if k is not None:
            if k.shape[:-2] != shape[:-2] or k.shape[-1] != d:
                raise ValueError("q and k must have the same tokens and head dimension")
            y_k, view_k = self._view(k, out_k, "k", dtype, dev, index, stream)
        tokens = shape[0] if len(shape) == 3 else shape[0] * shape[1]
        check(self._lib.vk_rotary_apply(self.handle, DTYPES[dtype], view, view_k, d, _i32(positions, "positions", index, tokens),
                                        tokens, _stream_of(stream, index)), "vk_rotary_apply")
        return y if k is None else (y, y_k)

    @staticmethod
    def _view(x, y, name, dtype, dev, index, stream):
        _on(x, dtype, name, index)
        token, head = _token_head(x, name)
        heads, d = x.shape[-2:]
        if y is None:
            y = torch.empty_like(x) if stream is None and x.is_contiguous() else _empty(x.shape, dtype, dev, stream)
            y_token, y_head = heads * d, d
        else:
            _on(y, dtype, "out", index)
            if y.shape != x.shape:
                raise ValueError("out must have the shape of its input")
            y_token, y_head = _token_head(y, "out")
        return y, _lib.VkRotaryView(x.data_ptr(), y.data_ptr(), token, head, y_token, y_head, heads)

    def close(self) -> None:
        if getattr(self, "handle", None) is not None and self.handle.value:
            self._lib.vk_rotary_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class LatentKVPool(PagedKVPool):
    """A paged cache of rows [latent | rotary key part] (vk_latent_pool_create).

    Storage: ``[num_layers, num_pages, page_tokens, latent_dim + rope_dim]`` of
    ``dtype`` (fp16 or bf16): a torch allocation, ``storage`` when given (a
    contiguous CUDA tensor of that size), or the library's own memory with
    ``own_memory``."""

    def __init__(self, num_layers: int, latent_dim: int, rope_dim: int, num_pages: int, page_tokens: int = PAGE_TOKENS,
                 dtype: torch.dtype = torch.float16, device=None, own_memory: bool = False, zero: bool = True,
                 storage: Optional[torch.Tensor] = None):
        self._lib = _lib.load()
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("dtype must be torch.float16 or torch.bfloat16")
        self.handle = None
        self.device = storage.device if storage is not None else _device(device)
        self._index = self.device.index
        self.num_layers, self.num_pages, self.page_tokens, self.dtype = num_layers, num_pages, page_tokens, dtype
        self.latent_dim, self.rope_dim, self.width = latent_dim, rope_dim, latent_dim + rope_dim
        self.num_kv_heads, self.head_dim, self.kv, self.kv_format = 1, self.width, False, "latent"
        self.block_bytes = 2 * page_tokens * self.width
        self.page_bytes = num_layers * self.block_bytes
        total = self.page_bytes * num_pages
        if storage is not None:
            if not storage.is_cuda or not storage.is_contiguous() or storage.numel() * storage.element_size() != total:
                raise ValueError("storage must be a contiguous CUDA tensor of %d bytes" % total)
            self.storage = storage
        elif own_memory:
            self.storage = None
        else:
            self.storage = (torch.zeros if zero else torch.empty)(max(0, total), dtype=torch.uint8, device=self.device)
        cfg = _lib.VkLatentCfg(num_layers, latent_dim, rope_dim, page_tokens, num_pages, self.device.index, DTYPES[dtype])
        handle = ctypes.c_void_p()
        check(self._lib.vk_latent_pool_create(ctypes.byref(cfg), None if own_memory and storage is None
                                              else ctypes.c_void_p(self.storage.data_ptr()), total, ctypes.byref(handle)),
              "vk_latent_pool_create")
        self.handle = handle

    def latent_view(self) -> torch.Tensor:
        """View [L, num_pages, page_tokens, latent_dim + rope_dim] of the pool."""
        if self.storage is None:
            raise RuntimeError("latent_view needs a torch-backed pool")
        return self.storage.view(torch.uint8).view(self.dtype).view(self.num_layers, self.num_pages, self.page_tokens, self.width)

    def append(self, layer: int, latent: torch.Tensor, k_rope: torch.Tensor, block_tables: torch.Tensor,
               positions: torch.Tensor, offsets: Optional[torch.Tensor] = None, norm_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-6, rope: Optional[RotaryEmbedding] = None, stream=None) -> None:
        """latent [tokens, latent_dim], k_rope [tokens, rope_dim] (row-strided views); sequence b takes the rows
        offsets[b]..offsets[b+1]-1 (None: the same number each; rows of no sequence are ignored) from position
        positions[b] on.  ``norm_weight``: root
        mean square norm of the latent first; ``rope``: k_rope rotated at its position."""
        index, dtype = self._index, self.dtype
        batch, width = _tables(block_tables, index)
        latent_rows, rope_rows = latent.stride(), k_rope.stride()
        for t, name, d, rows in ((latent, "latent", self.latent_dim, latent_rows), (k_rope, "k_rope", self.rope_dim, rope_rows)):
            if t.dtype is not dtype or t.get_device() != index:
                _on(t, dtype, name, index)
            if len(rows) != 2 or rows[1] != 1 or t.shape[1] != d:
                raise ValueError("%s must be [tokens, %d] with unit stride along its rows" % (name, d))
        tokens = latent.shape[0]
        if k_rope.shape[0] != tokens:
            raise ValueError("latent and k_rope must have the same tokens")
        weight = None
        if norm_weight is not None:
            _on(norm_weight, dtype, "norm_weight", index)
            if norm_weight.numel() != self.latent_dim or not norm_weight.is_contiguous():
                raise ValueError("norm_weight must be contiguous with %d elements" % self.latent_dim)
            weight = norm_weight.data_ptr()
        if rope is not None and not rope.handle.value:
            raise ValueError("rope is closed")
        check(self._lib.vk_latent_append(
            self.handle, layer, latent.data_ptr(), latent_rows[0], k_rope.data_ptr(), rope_rows[0], weight, eps,
            None if rope is None else rope.handle,
            block_tables.data_ptr(), width, _i32(positions, "positions", index, batch),
            None if offsets is None else _i32(offsets, "offsets", index, batch + 1), batch, tokens, _stream_of(stream, index)),
            "vk_latent_append")

    def decode_workspace_size(self, batch: int, tokens_per_seq: int, num_heads: int) -> int:
        return self._lib.vk_latent_decode_workspace_size(self.handle, batch, tokens_per_seq, num_heads)

    def decode(self, layer: int, q_latent: torch.Tensor, q_rope: torch.Tensor, block_tables: torch.Tensor,
               seq_lens: torch.Tensor, scale: float, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
               return_lse: bool = False, workspace: Optional[torch.Tensor] = None, stream=None):
        """Absorbed form.  q_latent [B, H, latent_dim] or [B, T, H, latent_dim], q_rope likewise with rope_dim
        (rotated; strided views allowed); seq_lens [B] int32: rows to attend, the T new ones included (query token t
        sees seq_lens[b] - (T-1-t)).  Returns out like q_latent, or (out, lse)."""
        dev, index = self.device, self._index
        batch, width = _tables(block_tables, index)
        _on(q_latent, self.dtype, "q_latent", index)
        _on(q_rope, self.dtype, "q_rope", index)
        shape = q_latent.shape
        if len(shape) not in (3, 4) or shape[:-1] != q_rope.shape[:-1] or shape[0] != batch or shape[-1] != self.latent_dim or \
                q_rope.shape[-1] != self.rope_dim:
            raise ValueError("q_latent must be [B, (T,) H, %d] and q_rope [B, (T,) H, %d]" % (self.latent_dim, self.rope_dim))
        tokens, heads = (shape[1] if len(shape) == 4 else 1), shape[-2]
        lt, lh = _token_head(q_latent, "q_latent")
        rt, rh = _token_head(q_rope, "q_rope")
        if out is None:
            out = torch.empty_like(q_latent) if stream is None and q_latent.is_contiguous() else _empty(shape, self.dtype, dev, stream)
        else:
            _on(out, self.dtype, "out", index)
            if out.shape != shape or not out.is_contiguous():
                raise ValueError("out must be contiguous with the shape of q_latent")
        if lse is not None:
            _on(lse, torch.float32, "lse", index)
            if lse.shape != shape[:-1] or not lse.is_contiguous():
                raise ValueError("lse must be contiguous [B, (T,) H]")
        elif return_lse:
            lse = q_latent.new_empty(shape[:-1], dtype=torch.float32) if stream is None else _empty(shape[:-1], torch.float32, dev, stream)
        ws, ws_bytes = _workspace(workspace, self.decode_workspace_size(batch, tokens, heads), q_latent, index, stream)
        check(self._lib.vk_latent_decode(
            self.handle, layer, q_latent.data_ptr(), lt, lh, q_rope.data_ptr(), rt, rh, out.data_ptr(),
            None if lse is None else lse.data_ptr(), block_tables.data_ptr(), width,
            _i32(seq_lens, "seq_lens", index, batch), batch, tokens, heads, scale, ws.data_ptr(), ws_bytes,
            _stream_of(stream, index)), "vk_latent_decode")
        return (out, lse) if return_lse else out

    def prefill_workspace_size(self, batch: int, max_seq_len: int, num_heads: int) -> int:
        return self._lib.vk_latent_prefill_workspace_size(self.handle, batch, max_seq_len, num_heads)

    def prefill(self, layer: int, q: torch.Tensor, w_kv: torch.Tensor, block_tables: torch.Tensor, positions: torch.Tensor,
                offsets: Optional[torch.Tensor] = None, max_tokens: Optional[int] = None, max_seq_len: Optional[int] = None,
                scale: float = 0.0, out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
        """Expanded form.  q [tokens, H, 128 + rope_dim] or [B, T, H, 128 + rope_dim] (rotary part rotated; strided
        views allowed), w_kv [H*256, latent_dim]: per head 128 rows of the key and 128 of the value up-projection.
        Sequence b's rows are offsets[b]..offsets[b+1]-1 (None: the same number each), from position positions[b] on.
        ``max_tokens`` bounds the longest chunk (default: without offsets the chunk, with them all tokens),
        ``max_seq_len`` the longest sequence after the chunk (default: what the tables hold).  Launches and
        workspace are sized by them: give both where the tables are wide.  Returns [..., H, 128]."""
        dev, index = self.device, self._index
        batch, width = _tables(block_tables, index)
        _on(q, self.dtype, "q", index)
        _on(w_kv, self.dtype, "w_kv", index)
        qt, qh = _token_head(q, "q")
        heads = q.shape[-2]
        if q.shape[-1] != 128 + self.rope_dim:
            raise ValueError("q must have %d elements a head" % (128 + self.rope_dim))
        if w_kv.dim() != 2 or w_kv.shape[0] != heads * 256 or w_kv.shape[1] != self.latent_dim or w_kv.stride(1) != 1:
            raise ValueError("w_kv must be [%d, %d] with unit stride along its rows" % (heads * 256, self.latent_dim))
        tokens = q.shape[0] if q.dim() == 3 else q.shape[0] * q.shape[1]
        if max_tokens is None:
            max_tokens = tokens if offsets is not None else tokens // max(1, batch)
        if max_seq_len is None:
            max_seq_len = block_tables.shape[1] * self.page_tokens
        shape = q.shape[:-1] + (128,)
        if out is None:
            out = _empty(shape, self.dtype, dev, stream)
        else:
            _on(out, self.dtype, "out", index)
            if out.shape != shape or not out.is_contiguous():
                raise ValueError("out must be contiguous with shape %s" % (tuple(shape),))
        ws, ws_bytes = _workspace(workspace, self.prefill_workspace_size(batch, max_seq_len, heads), q, index, stream)
        check(self._lib.vk_latent_prefill(
            self.handle, layer, q.data_ptr(), qt, qh, w_kv.data_ptr(), w_kv.stride(0), out.data_ptr(),
            block_tables.data_ptr(), width, _i32(positions, "positions", index, batch),
            None if offsets is None else _i32(offsets, "offsets", index, batch + 1), batch, tokens, max_tokens, max_seq_len,
            heads, scale, ws.data_ptr(), ws_bytes, _stream_of(stream, index)), "vk_latent_prefill")
        return out

    def plan(self, *args, **kwargs):
        raise TypeError("a latent pool has no planned decode: use decode")

    workspace = workspace_size = pages_per_split = set_split = set_rope = set_plan_workers = set_prefill_path = plan

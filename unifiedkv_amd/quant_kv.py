"""An 8-bit paged KV cache: rows quantised into 16-token pages, read back, and attended.

The cache of one layer (``QuantLayer``) keeps the Page16 layout of core/pool.py:67-71 with one byte an
element, int8 or float8_e4m3fn, and one power-of-two exponent byte for every 32 dims of a token's head
(``include/ukv.h`` states the format). Values read back exactly as they are attended, in fp16 or bf16:
quantising rounds once, nothing after it does. The calls mirror those of the 16-bit pool:

* ``write_chunk_kv`` / ``append_kv``   a prefill chunk's, a decode step's K/V into the pages
* ``read_kv``                          tokens back as packed 16-bit rows
* ``decode_attention``                 ``page16_native.page16_decode_attention`` over the cache
* ``prefill_attention``, ``chunked_prefill``   ``prefill``'s over the cache

``QuantizedKVPool`` is the pool of such layers; ``DecodeBatch`` and ``PrefillPages`` take it like the
16-bit one. Every function enqueues on the current stream and returns without a host synchronisation
(unless a length that it needs on the host is on the device only), and needs libukv.so: there is no fallback.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import _ext, page_ops
from .page16_native import _current_stream, _workspace
from .pool import PagedKVPool
from .prefill import _chunk_lens_on_host, _i32, _longest_pages, _max_chunk

FORMATS = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
QUANT_BLOCK = 32  # dims that share an exponent

_FORMAT_CODES = {torch.int8: _ext.UKV_CACHE_INT8, torch.float8_e4m3fn: _ext.UKV_CACHE_FP8}
_DTYPE_CODES = {torch.float16: _ext.UKV_DTYPE_F16, torch.bfloat16: _ext.UKV_DTYPE_BF16}


def _refuse(what: str):
    raise RuntimeError(f"quant_kv_shape_unsupported:{what}")


class QuantLayer:
    """One layer of the cache: codes ``k``, ``v`` [N, 16, H, D] (int8 or float8_e4m3fn) and exponent bytes
    ``k_scale``, ``v_scale`` [N, H, ceil(D / 32), 16] (uint8), last dimensions contiguous, other strides free."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "num_pages", "num_heads", "head_dim", "format_code", "device",
                 "strides", "pointers")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        # (each attribute is read once: a program without a pool may build one per call, 3 us)
        shape, dtype, dev = k.shape, k.dtype, k.device
        if len(shape) != 4 or shape[1] != 16:
            _refuse("cache")
        code = _FORMAT_CODES.get(dtype)
        if code is None or v.dtype != dtype:
            _refuse("cache_dtype")
        N, _, H, D = shape
        if v.shape != shape:
            _refuse("v_cache")
        want = (N, H, -(-D // QUANT_BLOCK), 16)
        if k_scale.shape != want or v_scale.shape != want:
            _refuse("scale")
        if k_scale.dtype != torch.uint8 or v_scale.dtype != torch.uint8:
            _refuse("scale_dtype")
        ks, vs, kss, vss = k.stride(), v.stride(), k_scale.stride(), v_scale.stride()
        if ks[3] != 1 or vs[3] != 1 or kss[3] != 1 or vss[3] != 1:
            _refuse("cache_stride")
        if v.device != dev or k_scale.device != dev or v_scale.device != dev:
            raise RuntimeError("quant_kv_unavailable:device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.num_heads, self.head_dim = N, H, D
        self.format_code = code
        self.device = dev
        self.strides = _ext.i64_tuple(ks[:3] + vs[:3] + kss[:3] + vss[:3])
        self.pointers = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())


def _check_rows(layer: QuantLayer, k: torch.Tensor, v: torch.Tensor) -> None:
    """K and V rows [total, H, D] of one 16-bit type on the cache's GPU."""
    shape = k.shape
    if len(shape) != 3 or v.shape != shape or shape[1] != layer.num_heads or shape[2] != layer.head_dim:
        _refuse("rows")
    if k.dtype not in _DTYPE_CODES or v.dtype != k.dtype:
        _refuse("dtype")
    if k.stride(2) != 1 or v.stride(2) != 1:
        _refuse("stride")
    _check_device(layer, k, v)


def _check_device(layer: QuantLayer, *tensors: torch.Tensor) -> None:
    dev = layer.device
    if dev.type != "cuda":
        raise RuntimeError("quant_kv_unavailable:device")
    for t in tensors:
        if t.device != dev:
            raise RuntimeError("quant_kv_unavailable:device")


_device_now = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(entry, layer: QuantLayer, *args) -> None:
    """A C entry's call with the layer's device as the current one, which is where it launches."""
    if layer.device.index == _device_now():
        code = entry(*args)
    else:
        with torch.cuda.device(layer.device):
            code = entry(*args)
    if code != _ext.UKV_OK:
        if code == _ext.UKV_ERR_HEAD_DIM:
            _refuse(f"head_dim_{layer.head_dim}")
        raise RuntimeError(f"quant_kv_error:{_ext.status_string(code)}")


def _batch(cu, lens, table) -> int:
    B, shape = lens.numel(), table.shape
    if len(shape) != 2 or shape[0] != B or (cu is not None and cu.numel() != B + 1):
        _refuse("batch")
    return B


def _write(layer, k, v, bt, cu, lens, lens_add, batch, max_chunk) -> None:
    _launch(
        _ext.load().ukv_quant_kv_write, layer,
        *layer.pointers, layer.strides, layer.num_pages, k.data_ptr(), v.data_ptr(),
        _ext.i64_tuple(k.stride()[:2] + v.stride()[:2]), bt.data_ptr(), int(bt.shape[1]),
        None if cu is None else cu.data_ptr(), None if lens is None else lens.data_ptr(), lens_add, batch, max_chunk,
        layer.num_heads, layer.head_dim, layer.format_code, _DTYPE_CODES[k.dtype], _current_stream(layer.device))


def _read(layer, k, v, bt, cu, lens, batch, max_chunk) -> None:
    _launch(
        _ext.load().ukv_quant_kv_read, layer,
        *layer.pointers, layer.strides, layer.num_pages, k.data_ptr(), v.data_ptr(),
        _ext.i64_tuple(k.stride()[:2] + v.stride()[:2]), bt.data_ptr(), int(bt.shape[1]),
        None if cu is None else cu.data_ptr(), None if lens is None else lens.data_ptr(), batch, max_chunk,
        layer.num_heads, layer.head_dim, layer.format_code, _DTYPE_CODES[k.dtype], _current_stream(layer.device))


def write_chunk_kv(layer: QuantLayer, k_new: torch.Tensor, v_new: torch.Tensor, block_table: torch.Tensor,
                   cu_seqlens_q, kv_lens, *, max_chunk: Optional[int] = None) -> None:
    """Row cu[b] + i of k_new / v_new ([total, H, D]) -> position kv_lens[b] - C_b + i of sequence b, quantised.

    ``max_chunk``, the longest chunk, saves the synchronisation that reading device ``cu_seqlens_q`` back would
    cost; a chunk longer than it is written all the same. Positions without a page are not written."""
    _check_rows(layer, k_new, v_new)
    chunk_lens = _chunk_lens_on_host(cu_seqlens_q)
    if chunk_lens is not None and sum(chunk_lens) > int(k_new.shape[0]):
        _refuse("rows")
    dev = layer.device
    cu, lens, bt = _i32(cu_seqlens_q, dev), _i32(kv_lens, dev), _i32(block_table, dev)
    B = _batch(cu, lens, bt)
    mc = _max_chunk(cu_seqlens_q, max_chunk, chunk_lens)
    if chunk_lens is None:
        mc = max(mc, 1)  # (sizes the launch alone: rows beyond it are written too)
    _write(layer, k_new, v_new, bt, cu, lens, 0, B, mc)


def append_kv(layer: QuantLayer, k_new: torch.Tensor, v_new: torch.Tensor, block_table: torch.Tensor,
              old_lens: torch.Tensor) -> None:
    """The decode token of each sequence, [B, H, D] (or [B, 1, H, D]), quantised to position old_lens[b]."""
    if k_new.dim() == 4:
        if int(k_new.shape[1]) != 1 or v_new.dim() != 4 or int(v_new.shape[1]) != 1:
            _refuse("rows")
        k_new, v_new = k_new[:, 0], v_new[:, 0]
    _check_rows(layer, k_new, v_new)
    dev = layer.device
    lens, bt = _i32(old_lens, dev), _i32(block_table, dev)
    B = _batch(None, lens, bt)
    if int(k_new.shape[0]) != B:
        _refuse("batch")
    _write(layer, k_new, v_new, bt, None, lens, 1, B, 1)


def read_kv(layer: QuantLayer, block_table: torch.Tensor, cu_seqlens, kv_lens, *, dtype: torch.dtype,
            max_chunk: Optional[int] = None, total: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(K, V) [total, H, D] in ``dtype``: row cu[b] + i is the token at position kv_lens[b] - C_b + i of sequence b.

    The counterpart of ``write_chunk_kv``; cu = cumulated kv_lens reads whole sequences. A position without a
    page reads as zeros. ``max_chunk`` and ``total`` save the synchronisation that reading device ``cu_seqlens``
    back would cost; ``total`` must be cu[B] (rows behind it are not written)."""
    if dtype not in _DTYPE_CODES:
        _refuse("dtype")
    _check_device(layer)
    chunk_lens = _chunk_lens_on_host(cu_seqlens)
    if chunk_lens is None and (total is None or max_chunk is None):
        cu_host = cu_seqlens.tolist()  # host sync
        chunk_lens = [cu_host[i + 1] - cu_host[i] for i in range(len(cu_host) - 1)]
    if chunk_lens is not None:
        if total is not None and int(total) != sum(chunk_lens):
            _refuse("rows")
        total = sum(chunk_lens)
    dev = layer.device
    cu, lens, bt = _i32(cu_seqlens, dev), _i32(kv_lens, dev), _i32(block_table, dev)
    B = _batch(cu, lens, bt)
    mc = _max_chunk(cu_seqlens, max_chunk, chunk_lens)
    if mc * B < int(total):
        _refuse("max_chunk")
    _check_device(layer, cu, lens, bt)
    k = torch.empty((int(total), layer.num_heads, layer.head_dim), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if k.numel():
        _read(layer, k, v, bt, cu, lens, B, mc)
    return k, v


def _check_queries(q: torch.Tensor, layer: QuantLayer, n_rep: int) -> None:
    if q.dim() != 3:
        _refuse(f"q_dim_{q.dim()}")
    if q.dtype not in _DTYPE_CODES:
        _refuse("dtype")
    if int(q.shape[2]) != layer.head_dim:
        _refuse("cache")
    if int(n_rep) < 1 or int(q.shape[1]) > int(n_rep) * layer.num_heads:
        _refuse("gqa")


def decode_attention(q: torch.Tensor, layer: QuantLayer, block_table: torch.Tensor, cache_seqlens: torch.Tensor, *,
                     softmax_scale: float, n_rep: int) -> torch.Tensor:
    """``page16_native.page16_decode_attention`` over an 8-bit layer: one query token per sequence.

    q [B, H_q, D] fp16 / bf16, cache_seqlens [B] with the current token; q head h reads KV head h // n_rep.
    Returns [B, H_q, D] in q's type; a sequence without a key gives NaN."""
    _check_queries(q, layer, n_rep)
    dev = layer.device
    _check_device(layer, q, block_table, cache_seqlens)
    if not q.is_contiguous():
        q = q.contiguous()
    bt, lens = _i32(block_table, dev), _i32(cache_seqlens, dev)
    B, Hq, D = q.shape
    if _batch(None, lens, bt) != B:
        _refuse("batch")
    if B == 0 or Hq == 0 or D == 0:
        _refuse("empty")
    out = torch.empty_like(q)
    stream = _current_stream(dev)
    width = int(bt.shape[1])
    ws = _workspace(B, Hq, D, width, dev, stream)
    _launch(
        _ext.load().ukv_quant_decode, layer,
        q.data_ptr(), *layer.pointers, layer.strides, layer.num_pages, bt.data_ptr(), lens.data_ptr(), out.data_ptr(),
        B, Hq, layer.num_heads, D, int(n_rep), width, _ext.i64_tuple(q.stride()[:2]), float(softmax_scale),
        layer.format_code, _DTYPE_CODES[q.dtype], ws.data_ptr(), ws.numel(), stream)
    return out


def prefill_attention(q: torch.Tensor, layer: QuantLayer, block_table: torch.Tensor, cu_seqlens_q, kv_lens, *,
                      softmax_scale: float, n_rep: int, max_chunk: Optional[int] = None, host_lens=None
                      ) -> torch.Tensor:
    """``prefill.paged_prefill_attention`` over an 8-bit layer: causal attention of packed chunk queries.

    q [total_q, H_q, D]; query i of sequence b is at position kv_lens[b] - C_b + i and sees the keys up to it.
    Rows behind the last sequence are not written. ``max_chunk`` and ``host_lens`` as there: a chunk longer than a
    ``max_chunk`` given with device lengths comes back as NaN."""
    _check_queries(q, layer, n_rep)
    if q.stride(2) != 1:
        _refuse("stride")
    _check_device(layer, q)
    dev = layer.device
    cu, lens, bt = _i32(cu_seqlens_q, dev), _i32(kv_lens, dev), _i32(block_table, dev)
    B = _batch(cu, lens, bt)
    total_q, Hq, D = (int(x) for x in q.shape)
    mc = _max_chunk(cu_seqlens_q, max_chunk, None if host_lens is None else host_lens[0])
    out = torch.empty((total_q, Hq, D), dtype=q.dtype, device=dev)
    lib = _ext.load()
    width = int(bt.shape[1])
    shape = (B, total_q, mc, Hq, layer.num_heads, D, int(n_rep))
    need = lib.ukv_quant_prefill_workspace_bytes(*shape, width)
    if need:
        # (a table wider than its sequences: where the host knows the lengths, a call without scratch may do)
        pages = _longest_pages(kv_lens, host_lens)
        if pages is not None and pages < width and not lib.ukv_quant_prefill_workspace_bytes(*shape, pages):
            need = 0
    ws = None
    if need:
        try:
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
        except torch.OutOfMemoryError:  # without scratch the keys stay in one part
            need = 0
    _launch(
        lib.ukv_quant_prefill, layer,
        q.data_ptr(), *layer.pointers, layer.strides, layer.num_pages, bt.data_ptr(), cu.data_ptr(), lens.data_ptr(),
        out.data_ptr(), B, total_q, mc, Hq, layer.num_heads, D, int(n_rep), width, _ext.i64_tuple(q.stride()[:2]),
        float(softmax_scale), layer.format_code, _DTYPE_CODES[q.dtype], ws.data_ptr() if ws is not None else None,
        need, _current_stream(dev))
    return out


def chunked_prefill(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, layer: QuantLayer,
                    block_table: torch.Tensor, cu_seqlens_q, kv_lens, *, softmax_scale: float, n_rep: int,
                    max_chunk: Optional[int] = None) -> torch.Tensor:
    """Quantise the chunk's K/V into its pages, then causal attention of its queries over prefix and chunk."""
    mc = _max_chunk(cu_seqlens_q, max_chunk)
    write_chunk_kv(layer, k_new, v_new, block_table, cu_seqlens_q, kv_lens, max_chunk=mc)
    return prefill_attention(q, layer, block_table, cu_seqlens_q, kv_lens, softmax_scale=softmax_scale, n_rep=n_rep,
                             max_chunk=mc)


class QuantizedKVPool(PagedKVPool):
    """``PagedKVPool`` whose pages hold 8-bit codes: the same constructor, allocation and token I/O.

    ``dtype`` is the type of the rows that go in and come out, ``cache_format`` "int8" or "fp8". A page takes
    (1 + 1/32) bytes an element instead of two, so the same memory holds 1.94 times the pages. ``layer(l)`` is a
    layer's ``QuantLayer``. What moves or scores 16-bit pages (``k_cache``, SnapKV scores, token-granular
    compaction, offload) refuses this pool; ``copy_pages`` and with it ``compaction.compact`` take it."""

    def __init__(self, block_size: int, num_layers: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, gpu_mem_frac: float = 0.75, cpu_mem_gb: float = 48.0, *,
                 cache_format: str = "int8", num_blocks: Optional[int] = None, device=None):
        if cache_format not in FORMATS:
            raise ValueError(f"cache_format must be one of {sorted(FORMATS)}, got {cache_format!r}")
        if block_size != 16:
            _refuse(f"block_size_{block_size}")
        if dtype not in _DTYPE_CODES:
            _refuse("dtype")
        self.cache_format = cache_format
        self._layers: List[QuantLayer] = []
        super().__init__(block_size, num_layers, num_kv_heads, head_dim, dtype, gpu_mem_frac, cpu_mem_gb,
                         num_blocks=num_blocks, device=device)

    def _bytes_per_block(self) -> int:
        blocks = -(-self.head_dim // QUANT_BLOCK)
        return 2 * self.num_layers * self.B * self.num_kv_heads * (self.head_dim + blocks)

    # ------------------------------------------------------------------ storage
    def ensure_allocated(self) -> None:
        if self.is_allocated:
            return
        L, N, H, D = self.num_layers, self.N_total, self.num_kv_heads, self.head_dim
        of = FORMATS[self.cache_format]
        codes = [torch.zeros((L, N, 16, H, D), dtype=torch.uint8, device=self.device).view(of) for _ in range(2)]
        scales = [torch.zeros((L, N, H, -(-D // QUANT_BLOCK), 16), dtype=torch.uint8, device=self.device)
                  for _ in range(2)]
        self._layers = [QuantLayer(codes[0][i], codes[1][i], scales[0][i], scales[1][i]) for i in range(L)]
        self.k_scale, self.v_scale = scales
        self._k_cache, self._v_cache = codes

    def release_if_empty(self) -> bool:
        with self.lock:
            empty = len(self.used_blocks) == 0
        if not empty or not self.is_allocated:
            return False
        self._layers = []
        self.k_scale = self.v_scale = None
        return super().release_if_empty()

    @property
    def k_cache(self) -> torch.Tensor:
        raise RuntimeError("quant_kv_shape_unsupported:k_cache")

    @property
    def v_cache(self) -> torch.Tensor:
        raise RuntimeError("quant_kv_shape_unsupported:v_cache")

    def layer(self, layer_id: int) -> QuantLayer:
        self.ensure_allocated()
        layer_id = int(layer_id)
        if not 0 <= layer_id < self.num_layers:
            raise IndexError(f"layer {layer_id} is outside the pool's {self.num_layers} layers")
        return self._layers[layer_id]

    # ---------------------------------------------------------------- token I/O
    def write_kv_to_blocks(self, layer_id: int, block_ids: List[int], K: torch.Tensor, V: torch.Tensor):
        """K/V [h_kv, T, d]: token t -> page block_ids[t // 16], slot t % 16, quantised (core/pool.py:127-141)."""
        n = min(int(K.shape[1]), 16 * len(block_ids))
        if n <= 0:
            return
        layer = self.layer(layer_id)
        k, v = (self._as_pool_rows(x)[:, :n].transpose(0, 1) for x in (K, V))
        _check_rows(layer, k, v)
        _write(layer, k, v, self._device_ids(block_ids)[None], None, None, 0, 1, n)

    def write_one_token(self, layer_id: int, block_id: int, pos_in_block: int, k_tok: torch.Tensor,
                        v_tok: torch.Tensor):
        if not (0 <= int(block_id) < self.N_total and 0 <= int(pos_in_block) < 16):
            raise IndexError(f"page {block_id}, slot {pos_in_block}: outside the pool")
        at = torch.tensor([[int(block_id)], [int(pos_in_block)]], dtype=torch.int32, device=self.device)
        append_kv(self.layer(layer_id), self._as_pool_rows(k_tok.squeeze(1))[None],
                  self._as_pool_rows(v_tok.squeeze(1))[None], at[:1], at[1])

    def read_kv_from_blocks(self, layer_id: int, block_ids: List[int], seq_len: int
                            ) -> Tuple[torch.Tensor, torch.Tensor]:
        """[h_kv, min(seq_len, 16 * len(block_ids)), d] K and V (core/pool.py:154-172)."""
        n = max(0, min(int(seq_len), 16 * len(block_ids)))
        if n == 0:
            K = torch.empty(self.num_kv_heads, 0, self.head_dim, dtype=self.dtype, device=self.device)
            return K, torch.empty_like(K)
        layer = self.layer(layer_id)
        _check_device(layer)
        K = torch.empty((self.num_kv_heads, n, self.head_dim), dtype=self.dtype, device=self.device)
        V = torch.empty_like(K)
        _read(layer, K.transpose(0, 1), V.transpose(0, 1), self._device_ids(block_ids)[None], None, None, 1, n)
        return K, V

    def build_block_table(self, layer_id: int, seq_block_ids_list: List[List[int]]
                          ) -> Tuple[QuantLayer, torch.Tensor]:
        """(layer, int32 [batch, max_blocks]): ``layer(layer_id)`` and ``block_table_for``'s table."""
        return self.layer(layer_id), self.block_table_for(seq_block_ids_list)

    def append_decode_tokens(self, layer_id: int, block_table: torch.Tensor, old_lens: torch.Tensor,
                             k_new: torch.Tensor, v_new: torch.Tensor) -> torch.Tensor:
        """Token b, quantised, to page block_table[b, len // 16], slot len % 16; returns old_lens + 1."""
        append_kv(self.layer(layer_id), self._as_pool_rows(k_new), self._as_pool_rows(v_new), block_table, old_lens)
        return old_lens.to(torch.int32) + 1

    def copy_pages(self, src_ids, dst_ids) -> None:
        """Codes and exponents of page src_ids(l)[j] -> page dst_ids(l)[j] for every layer l, bit for bit."""
        self.ensure_allocated()
        for k, v in ((self._k_cache, self._v_cache), (self.k_scale, self.v_scale)):
            # (the copy kernel moves pages of any sixteen-byte multiple, as 16-bit elements)
            pages = [x.view(torch.uint8).flatten(2).view(torch.float16) for x in (k, v)]
            page_ops.page_copy(pages, pages, src_ids, dst_ids)


__all__ = ["FORMATS", "QuantLayer", "QuantizedKVPool", "append_kv", "chunked_prefill", "decode_attention",
           "prefill_attention", "read_kv", "write_chunk_kv"]

"""The paged key-value cache of a causal model and the operators on it: append of new tokens,
attention of a ragged batch of new tokens (prompts) and of one new token per sequence.

The tensors belong to the caller (a page allocator, a scheduler); ``PagedKVCache`` checks them
once and passes their addresses to the C ABI, so a serving loop writes ``page_table`` and
``kv_lens`` in place and calls::

    cache.append(k_new, v_new, offsets)         # after kv_lens counts the new tokens
    y = cache.prefill(q, offsets, window=1024, sinks=4)
    y = cache.decode(q)

Every call is stream-ordered on the current stream of the cache's device and can be captured
into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import check, lib
from .ops import _DTYPES, _on, _raw_stream


class PagedKVCache:
    """Keys and values in pages (see ``lsc_paged_kv``).

    k, v: [pages, page_size, kv_heads, head_dim] f16 or bf16 CUDA tensors, views of any strides
    that both share (head_dim contiguous); page_size a power of two from 8 to 256, head_dim 64 or
    128.  page_table: [batch, max_pages] int32; kv_lens: [batch] int32, the tokens of each
    sequence.  Both are read on the device when a kernel runs.
    """

    def __init__(self, k, v, page_table, kv_lens):
        if k.dim() != 4 or not k.is_cuda or k.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"k: expected a [pages, page_size, heads, head_dim] CUDA f16 or bf16 tensor, got "
                             f"{k.dtype} {tuple(k.shape)} on {k.device}")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device or v.stride() != k.stride():
            raise ValueError("v: expected k's shape, type, device and strides")
        if k.stride(3) != 1:
            raise ValueError("k, v: head_dim must be contiguous")
        for name, t, dim in (("page_table", page_table, 2), ("kv_lens", kv_lens, 1)):
            if t.dim() != dim or t.dtype != torch.int32 or t.device != k.device or (t.numel() and t.stride(-1) != 1):
                raise ValueError(f"{name}: expected a {dim}-D int32 tensor on {k.device} with contiguous rows")
        if page_table.shape[0] != kv_lens.shape[0]:
            raise ValueError(f"page_table and kv_lens: {page_table.shape[0]} and {kv_lens.shape[0]} sequences")
        self.k, self.v, self.page_table, self.kv_lens = k, v, page_table, kv_lens
        self.device, self._index, self._dtype = k.device, k.get_device(), k.dtype
        self.batch = kv_lens.shape[0]
        pages, page_size, self.kv_heads, self.head_dim = k.shape
        self._desc = _lib.lsc_paged_kv(
            k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype], page_size, self.kv_heads, self.head_dim, pages,
            *k.stride()[:3], page_table.data_ptr(), page_table.stride(0), kv_lens.data_ptr(), page_table.shape[1],
            self.batch)
        self._ref = C.byref(self._desc)
        self._scale = self.head_dim ** -0.5
        self._offsets_shape = torch.Size([self.batch + 1])
        self._workspace_bytes = {}  # by query heads
        # sequences that cannot grow long enough to be cut need no workspace
        self._cut = lib().lsc_paged_attention_decode_workspace_size(self._ref, self.kv_heads) > 0

    def _heads(self, t, name):
        """Checks a [tokens, heads, head_dim] tensor of the cache's type with contiguous heads; its shape and
        strides."""
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or t.dtype is not self._dtype or t.get_device() != self._index or \
                shape[2] != self.head_dim or stride[2] != 1:
            raise ValueError(f"{name}: expected a [tokens, heads, {self.head_dim}] {self._dtype} tensor on "
                             f"{self.device} with contiguous heads, got {t.dtype} {tuple(shape)} on {t.device}")
        return shape, stride

    def _offsets(self, t):
        if t.dtype is not torch.int32 or t.get_device() != self._index or t.shape != self._offsets_shape or \
                not t.is_contiguous():
            raise ValueError(f"q_offsets: expected {self.batch + 1} contiguous int32 values on {self.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def append(self, k_new, v_new, q_offsets):
        """Writes the new tokens' keys and values ([tokens, kv_heads, head_dim]; views of a fused
        projection can be given in place) behind the tokens already held: rows
        q_offsets[b] .. q_offsets[b + 1] - 1 become the last of sequence b's kv_lens[b] tokens."""
        shape, stride = self._heads(k_new, "k_new")
        if v_new.shape != shape or v_new.dtype is not self._dtype or v_new.get_device() != self._index or \
                v_new.stride() != stride:
            raise ValueError("v_new: expected k_new's shape, type, device and strides")
        if shape[1] != self.kv_heads:
            raise ValueError(f"k_new: {shape[1]} heads, the cache has {self.kv_heads}")
        offsets = self._offsets(q_offsets)
        with _on(self._index):
            check(lib().lsc_kv_cache_append(self._ref, k_new.data_ptr(), v_new.data_ptr(), shape[0], stride[0],
                                            stride[1], offsets, _raw_stream(self._index)))

    def _outputs(self, q, shape, out, out_i8):
        if out is None and out_i8 is None:
            out = torch.empty(shape, dtype=q.dtype, device=q.device)
        for name, t, dtype in (("out", out, self._dtype), ("out_i8", out_i8, torch.int8)):
            if t is not None and (t.dtype is not dtype or t.get_device() != self._index or t.shape != shape or
                                  not t.is_contiguous()):
                raise ValueError(f"{name}: expected a contiguous {dtype} tensor of {tuple(shape)} on {self.device}, "
                                 f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        return out, None if out is None else out.data_ptr(), None if out_i8 is None else out_i8.data_ptr()

    def prefill(self, q, q_offsets, alpha=None, window=0, sinks=0, out=None, out_i8=None, s_out=1.0,
                rounding=_lib.ROUND_HALF_AWAY):
        """Causal attention of new tokens (see ``lsc_paged_attention_prefill``).  q: [tokens,
        q_heads, head_dim]; rows q_offsets[b] .. q_offsets[b + 1] - 1 are the last tokens of sequence
        b, already appended.  ``window`` > 0: a sliding window of that many tokens beside the first
        ``sinks`` ones.  alpha defaults to 1 / sqrt(head_dim).  Writes ``out`` (allocated when neither
        output is given) and / or ``out_i8`` quantized with ``s_out``; returns out or out_i8."""
        shape, stride = self._heads(q, "q")
        offsets = self._offsets(q_offsets)
        out, p_out, p_i8 = self._outputs(q, shape, out, out_i8)
        with _on(self._index):
            check(lib().lsc_paged_attention_prefill(
                self._ref, q.data_ptr(), shape[0], shape[1], stride[0], stride[1], offsets,
                self._scale if alpha is None else alpha, window, sinks, p_out, p_i8, s_out, rounding,
                _raw_stream(self._index)))
        return out if out is not None else out_i8

    def decode_workspace(self, q_heads):
        """A workspace for ``decode`` with that many query heads."""
        n = self._workspace_bytes.get(q_heads)
        if n is None:
            n = lib().lsc_paged_attention_decode_workspace_size(self._ref, q_heads)
            self._workspace_bytes[q_heads] = n
        return torch.empty(n, dtype=torch.uint8, device=self.device)

    def decode(self, q, alpha=None, window=0, sinks=0, out=None, out_i8=None, s_out=1.0,
               rounding=_lib.ROUND_HALF_AWAY, workspace=None):
        """Attention of one new token per sequence (see ``lsc_paged_attention_decode``).  q: [batch,
        q_heads, head_dim]; the other arguments as for ``prefill``.  ``workspace``
        (``decode_workspace``) is allocated for the call when it is not given; calls that share one
        must be ordered on one stream."""
        shape, stride = self._heads(q, "q")
        if shape[0] != self.batch:
            raise ValueError(f"q: {shape[0]} rows, the cache has {self.batch} sequences")
        out, p_out, p_i8 = self._outputs(q, shape, out, out_i8)
        if workspace is None:
            workspace = self.decode_workspace(shape[1]) if self._cut else None
        elif not workspace.is_contiguous() or workspace.get_device() != self._index:
            raise ValueError(f"workspace: expected a contiguous tensor on {self.device}")
        with _on(self._index):
            check(lib().lsc_paged_attention_decode(
                self._ref, q.data_ptr(), shape[1], stride[0], stride[1], self._scale if alpha is None else alpha, window,
                sinks, p_out, p_i8, s_out, rounding, None if workspace is None else workspace.data_ptr(),
                0 if workspace is None else workspace.nbytes, _raw_stream(self._index)))
        return out if out is not None else out_i8

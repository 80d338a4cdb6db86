"""The paged int8 key/value cache of a decoder layer and the calls around it.

What a serving program does between the fused QKV projection and the output projection, for a ragged batch of
sequences whose tokens lie in pages of one pool::

    cache = PagedKvInt8(ops, ops.KaioDevice(0), num_pages=4096, heads=64, kv_heads=8, head_dim=128)
    cache.append(q, k, v, q_rot, cos, sin, block_table, q_start, kv_len)       # rotate, quantise, append
    cache.attend(q_rot, out, block_table, q_start, kv_len, max_new=1)          # the new tokens attend to the cache

``block_table`` int32 ``[batch, max_pages]``, ``q_start`` int32 ``[batch + 1]`` (the rows of q, k and v that belong to
each sequence) and ``kv_len`` int32 ``[batch]`` (tokens in the cache with this call's) live on the device and are read
when the work runs, so a captured CUDA graph follows them.  Which pages a sequence has is the caller's business; no
two sequences may append to one page, but they may read one (a shared prefix of whole pages).
The buffers and the arithmetic are described in ``include/kaio_b200.h``.
"""
from __future__ import annotations

import torch

BLOCK = 16  # tokens that share a scale


def _rows(t: torch.Tensor, name: str, columns: int):
    """(buffer, rows, row stride) of a matrix that is dense along its rows, as the ops take it: a flat tensor from the matrix's
    first element to its last."""
    shape = t.shape
    if len(shape) != 2 or shape[1] != columns:
        raise ValueError(f"{name}: expected a matrix of {columns} columns, got shape {tuple(shape)}")
    if t.is_contiguous():
        return t, shape[0], columns
    stride, inner = t.stride()
    if inner != 1 or stride < columns:
        raise ValueError(f"{name}: expected a matrix whose rows are contiguous, got shape {tuple(shape)} strides {(stride, inner)}")
    return t.as_strided(((shape[0] - 1) * stride + columns,), (1,)), shape[0], stride


class PagedKvInt8:
    """``num_pages`` pages of ``page_size`` tokens for ``kv_heads`` heads of ``head_dim``, read by ``heads`` query heads.

    ``storage``: the four tensors ``(k, v, k_scale, v_scale)`` to use instead of new ones (int8 ``[num_pages, kv_heads,
    page_size, head_dim]`` twice, float32 ``[num_pages, kv_heads, page_size/16]`` twice).
    """

    def __init__(self, ops, device, num_pages: int, heads: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 storage=None):
        self.ops, self.device = ops, device
        self.num_pages, self.heads, self.kv_heads = num_pages, heads, kv_heads
        self.head_dim, self.page_size = head_dim, page_size
        values, scales = (num_pages, kv_heads, page_size, head_dim), (num_pages, kv_heads, page_size // BLOCK)
        if storage is None:
            dev = torch.device("cuda", device.ordinal)
            storage = tuple(torch.zeros(values, dtype=torch.int8, device=dev) for _ in range(2)) + \
                tuple(torch.zeros(scales, dtype=torch.float32, device=dev) for _ in range(2))
        for name, t, shape in zip(("k", "v", "k_scale", "v_scale"), storage, (values, values, scales, scales)):
            if tuple(t.shape) != shape:
                raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")
        self.k, self.v, self.k_scale, self.v_scale = storage
        self._width, self._q_width = kv_heads * head_dim, heads * head_dim

    def _batch(self, block_table, start, name):
        shape = block_table.shape
        if len(shape) != 2 or len(start) != shape[0] + 1:
            raise ValueError(f"block_table [batch, max_pages] and {name} [batch + 1] do not fit: {tuple(shape)}, {tuple(start.shape)}")
        return shape

    def append(self, q, k, v, q_out, cos, sin, block_table, q_start, kv_len, *, rot_dim=None, interleaved=False):
        """Rotates ``q`` ``[tokens, heads*head_dim]`` into ``q_out`` and appends ``k``, ``v`` ``[tokens, kv_heads*head_dim]``;
        the three may be column ranges of one matrix.  ``cos``, ``sin``: float32 ``[positions, rot_dim/2]``;
        ``rot_dim`` defaults to what they hold, 0 (both ``None``) for no rotation.  ``q`` and ``q_out`` may be ``None``."""
        batch, max_pages = self._batch(block_table, q_start, "q_start")
        k, tokens, kv_stride = _rows(k, "k", self._width)
        v, v_tokens, v_stride = _rows(v, "v", self._width)
        if v_tokens != tokens or (v_stride != kv_stride and tokens > 1):
            raise ValueError(f"k and v must have one shape and one row stride, got {(tokens, kv_stride)} and {(v_tokens, v_stride)}")
        q_stride = 0
        if q is not None:
            out_shape = q.shape
            q, q_tokens, q_stride = _rows(q, "q", self._q_width)
            if q_tokens != tokens or q_out is None or q_out.shape != out_shape:
                raise ValueError("q, k and q_out must have the same number of rows, and q_out the shape of q")
        positions = half = 0
        if cos is not None:
            positions, half = cos.shape
        if rot_dim is None:
            rot_dim = 2 * half
        if rot_dim and (2 * half != rot_dim or sin is None or sin.shape != cos.shape):
            raise ValueError(f"cos and sin must both be [positions, {rot_dim // 2}]")
        self.ops.rope_append_kv_int8(
            self.device, q, k, v, cos, sin, q_out, self.k, self.v, self.k_scale, self.v_scale, block_table, q_start, kv_len,
            batch, tokens, self.heads, self.kv_heads, self.head_dim, q_stride, kv_stride, rot_dim, interleaved, positions,
            self.page_size, self.num_pages, max_pages)

    def gather(self, k_out, v_out, block_table, kv_start):
        """Sequence ``b``'s cached tokens as the rows ``[kv_start[b], kv_start[b + 1])`` of ``k_out`` and ``v_out``, float16
        ``[total, kv_heads*head_dim]``."""
        batch, max_pages = self._batch(block_table, kv_start, "kv_start")
        self.ops.gather_kv_int8(self.device, self.k, self.v, self.k_scale, self.v_scale, block_table, kv_start, k_out,
                                v_out, batch, k_out.shape[0], self.kv_heads, self.head_dim, self.page_size,
                                self.num_pages, max_pages)

    def scratch(self, batch: int, tokens: int, max_new: int):
        """A scratch tensor for :meth:`attend` calls of these sizes (or ``None`` where they need none).  Calls that may run at the
        same time, two replayed graphs among them, need one each."""
        n = self.ops.attention_paged_int8_scratch(batch, tokens, max_new, self.heads, self.kv_heads, self.head_dim)
        return torch.empty(n, dtype=torch.float32, device=self.k.device) if n else None

    def attend(self, q, out, block_table, q_start, kv_len, max_new, *, causal=True, scratch=None):
        """``out[tokens, heads*head_dim]``: attention of the (rotated) ``q`` to the cache; ``max_new`` is the most new tokens a
        sequence has.  ``scratch`` (see :meth:`scratch`) is allocated per call when it is not given, on the stream that
        the call runs on."""
        batch, max_pages = self._batch(block_table, q_start, "q_start")
        if out.shape != q.shape:
            raise ValueError(f"out must have the shape of q, {tuple(q.shape)}, got {tuple(out.shape)}")
        q, tokens, q_stride = _rows(q, "q", self._q_width)
        if scratch is None:
            stream = getattr(self.device, "_stream", None)
            if stream is None:
                scratch = self.scratch(batch, tokens, max_new)
            else:
                with torch.cuda.stream(stream):
                    scratch = self.scratch(batch, tokens, max_new)
        self.ops.attention_paged_int8(
            self.device, q, self.k, self.v, self.k_scale, self.v_scale, block_table, q_start, kv_len, out, scratch,
            batch, tokens, max_new, self.heads, self.kv_heads, self.head_dim, q_stride, causal, self.page_size,
            self.num_pages, max_pages)

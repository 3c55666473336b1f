"""A paged KV cache held in NVFP4 and the attention that reads it (csrc/mtq_kvcache.hip).

The cache stores what ``NVFP4_KV_CFG`` simulates: every 16 values of a K / V row as E2M1 codes with an
E4M3 scale, under a global scale ``amax / 2688`` per tensor -- 9 / 16 byte a value.  Where the
reference's ``attention()`` takes 16-bit paged caches (triton_fa.py:1221-1390, ``k_cache`` / ``v_cache`` /
``block_table``), this one computes straight from the 4-bit pages.
"""

from __future__ import annotations

import torch

from ....._ext import ops
from ...quantization.mx import check_device, refuse_grad

__all__ = ["NVFP4KVCache"]


class NVFP4KVCache:
    """Pages of K and V rows in NVFP4.

    ``k_data`` / ``v_data`` ``uint8 [num_pages, num_kv_heads, page_size, head_dim / 2]`` (two codes a byte,
    the even column low), ``k_scale`` / ``v_scale`` ``float8_e4m3fn [..., head_dim / 16]``, ``k_amax`` /
    ``v_amax`` one fp32 value each on the device (the calibrated amax of ``k_bmm_quantizer`` /
    ``v_bmm_quantizer``).  ``page_size`` is a power of two from 16 to 32768, ``head_dim`` 64, 128 or 256.

    Every call names its sequences as ``attention()`` does: ``b_start_loc`` / ``b_seq_len`` (int32 ``[batch]``)
    are the rows of a sequence's new tokens in the flat ``[tokens, heads, head_dim]`` tensors,
    ``b_seq_len_k`` its length in the cache with them (the new tokens are its last positions), and
    ``block_table`` (int32 ``[batch, pages per sequence]``) the page of every ``page_size`` positions;
    ``max_input_len`` bounds ``b_seq_len`` (tokens from it on are left out).  All of them stay on the device: no call synchronises, and each can
    be captured into a graph.  An entry outside ``[0, num_pages)`` stands for no page: rows for it are
    dropped, read as zeros and not seen by the attention.  A page that ``append`` writes must belong to one
    sequence; pages that are only read may be shared.
    """

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *, k_amax=2688.0, v_amax=2688.0,
                 device="cuda"):
        self._check_head_dim(head_dim)
        shape = (num_pages, num_kv_heads, page_size)

        def scalar(v):
            return torch.as_tensor(v, dtype=torch.float32, device=device).detach().reshape(1)

        data = [torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device) for _ in range(2)]
        scale = [torch.zeros(*shape, head_dim // 16, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        self._set(data[0], scale[0], data[1], scale[1], scalar(k_amax), scalar(v_amax))

    @staticmethod
    def _check_head_dim(head_dim):
        if head_dim not in (64, 128, 256):
            raise NotImplementedError(f"head_dim {head_dim} is not supported (supported: 64, 128, 256)")

    @classmethod
    def from_tensors(cls, k_data, k_scale, v_data, v_scale, k_amax, v_amax) -> "NVFP4KVCache":
        """A cache over tensors that the caller holds (any strides over pages, heads and places; rows contiguous, of
        codes at multiples of 16 bytes, of scales at multiples of ``head_dim / 16``)."""
        self = cls.__new__(cls)
        self._set(k_data, k_scale, v_data, v_scale, k_amax, v_amax)
        return self

    def _set(self, k_data, k_scale, v_data, v_scale, k_amax, v_amax):
        if k_data.dim() != 4 or v_data.shape != k_data.shape:
            raise ValueError("k_data and v_data must both be [num_pages, num_kv_heads, page_size, head_dim / 2]")
        self._check_head_dim(2 * k_data.shape[3])
        page_size = k_data.shape[2]
        if not 16 <= page_size <= 32768 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 32768, got {page_size}")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float8_e4m3fn or t.shape != (*k_data.shape[:3], k_data.shape[3] // 8):
                raise ValueError(f"{name} must be float8_e4m3fn [num_pages, num_kv_heads, page_size, head_dim / 16]")
        self.k_data, self.k_scale, self.v_data, self.v_scale = k_data, k_scale, v_data, v_scale
        self.k_amax, self.v_amax = k_amax, v_amax
        self.num_pages, self.num_kv_heads, self.page_size = k_data.shape[:3]
        self.head_dim = 2 * k_data.shape[3]

    def _tensors(self):
        return [self.k_data, self.k_scale, self.v_data, self.v_scale, self.k_amax, self.v_amax]

    def append(self, k, v, b_start_loc, b_seq_len, b_seq_len_k, block_table, max_input_len: int) -> None:
        """Quantise the new tokens' rows ``k`` / ``v [tokens, num_kv_heads, head_dim]`` (bf16, fp16 or fp32)
        into their pages."""
        check_device("NVFP4KVCache.append", k)
        refuse_grad("NVFP4KVCache.append", k, v)
        ops().kv_append(self._tensors(), k, v, b_start_loc, b_seq_len, b_seq_len_k, block_table, max_input_len)

    def read(self, b_start_loc, b_seq_len, b_seq_len_k, block_table, max_input_len: int, total_tokens: int, *,
             dtype=torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows of those positions as ``(k, v)``, ``[total_tokens, num_kv_heads, head_dim]`` of
        ``dtype`` (rows of no sequence are not written)."""
        shape = (total_tokens, self.num_kv_heads, self.head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=self.k_data.device) for _ in range(2))
        check_device("NVFP4KVCache.read", k)
        ops().kv_read(self._tensors(), k, v, b_start_loc, b_seq_len, b_seq_len_k, block_table, max_input_len)
        return k, v

    def attention(self, q, b_start_loc, b_seq_len, b_seq_len_k, block_table, max_input_len: int, max_kv_len: int | None = None,
                  *, is_causal: bool = True, softmax_scale: float | None = None) -> torch.Tensor:
        """``softmax(q k^T * softmax_scale) v`` over the cached keys for ``q [tokens, num_q_heads, head_dim]``
        (bf16 or fp16; ``num_q_heads`` a multiple of ``num_kv_heads``).

        Causal: a query sees the keys up to its own position.  A query that sees no key gives zeros; rows of
        no sequence are not written, as ``attention()``.  ``max_kv_len`` (a bound of ``b_seq_len_k``, default what
        ``block_table`` can hold) sizes the split over the keys.  ``softmax_scale`` is positive (default
        ``head_dim ** -0.5``)."""
        check_device("NVFP4KVCache.attention", q)
        refuse_grad("NVFP4KVCache.attention", q)
        if max_kv_len is None:
            max_kv_len = block_table.shape[1] * self.page_size
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ops().kv_attention(self._tensors(), q, o, b_start_loc, b_seq_len, b_seq_len_k, block_table, max_input_len, max_kv_len,
                           is_causal, self.head_dim ** -0.5 if softmax_scale is None else softmax_scale)
        return o

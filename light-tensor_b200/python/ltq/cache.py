"""``ltq_kv_cache``: keys and values of an attention layer in 8 bits, with one scale per block of tokens and head."""
import ctypes as C

import torch

from . import tokens as _tokens
from ._binding import KVCacheDesc, check, lib


class KVCache:
    """A paged cache over tensors that stay the caller's: codes ``k``, ``v`` uint8 CUDA [blocks, kv_heads, block_tokens, head_dim] and
    their parameters ``k_qparams``, ``v_qparams`` uint8 CUDA [blocks, kv_heads, 8] (a QParams each).  ``KVCache.empty`` makes
    them.  block_tokens 16, 32, 64 or 128; head_dim 32, 64, 96, 128, 192 or 256.

    A batch of sequences is described by int32 CUDA tensors: ``lengths`` [seqs] (tokens in all, the new ones included),
    ``offsets`` [seqs + 1] (sequence b's new tokens are rows offsets[b] .. offsets[b + 1] - 1) and ``table`` [seqs, width] (block ids);
    ``max_new`` is a host bound on the new tokens of a sequence, at most the rows there are.  The kernels read these tensors when they run, so a captured
    call follows their contents.  A sequence or block id that contradicts the bounds is left out and makes the next
    ``check()`` raise."""

    def __init__(self, k, k_qparams, v, v_qparams):
        for t in (k, v):
            if not (t.is_cuda and t.dtype == torch.uint8 and t.dim() == 4 and t.is_contiguous() and t.shape == k.shape and t.device == k.device):
                raise ValueError("codes must be contiguous uint8 CUDA tensors [blocks, kv_heads, block_tokens, head_dim] of one shape and device")
        self.blocks, self.kv_heads, self.block_tokens, self.head_dim = k.shape
        for t in (k_qparams, v_qparams):
            _tokens.check_qparams(t, self.blocks * self.kv_heads, k.device.index)
        self.k, self.k_qparams, self.v, self.v_qparams = k, k_qparams, v, v_qparams
        self.device, self._index = k.device, k.device.index
        self._desc = KVCacheDesc(k.data_ptr(), k_qparams.data_ptr(), v.data_ptr(), v_qparams.data_ptr(), self.blocks, self.kv_heads,
                                 self.block_tokens, self.head_dim)
        self._ref = C.byref(self._desc)
        self._last = None, 0

    @classmethod
    def empty(cls, blocks, kv_heads, block_tokens, head_dim, device="cuda"):
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        codes = [torch.full((blocks, kv_heads, block_tokens, head_dim), 128, dtype=torch.uint8, device=device) for _ in range(2)]
        qparams = [torch.zeros((blocks, kv_heads, 8), dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(codes[0], qparams[0], codes[1], qparams[1])

    def _batch(self, table, lengths, offsets):
        dev, i32 = self._index, torch.int32
        if not (table.dtype is i32 and lengths.dtype is i32 and offsets.dtype is i32 and
                table.get_device() == dev and lengths.get_device() == dev and offsets.get_device() == dev):
            raise ValueError(f"table, lengths and offsets must be int32 tensors on {self.device}")
        if not (table.is_contiguous() and lengths.is_contiguous() and offsets.is_contiguous()):
            raise ValueError("table, lengths and offsets must be contiguous")
        seqs = lengths.numel()
        if not (table.dim() == 2 and table.shape[0] == seqs and lengths.dim() == 1 and offsets.dim() == 1 and offsets.numel() == seqs + 1):
            raise ValueError("table [seqs, width], lengths [seqs] and offsets [seqs + 1] are expected")
        return seqs, table.shape[1]

    def _rows(self, t, heads, what):
        """(tokens, heads, elements between the tokens) of a [tokens, heads, head_dim] tensor whose tokens are contiguous."""
        if not (t.get_device() == self._index and t.dim() == 3 and t.shape[2] == self.head_dim and (heads is None or t.shape[1] == heads)):
            raise ValueError(f"{what} must be a tensor [tokens, heads, {self.head_dim}] on {self.device}")
        tokens, heads, D = t.shape
        pitch, between, step = t.stride()
        n = heads * D
        if step != 1 or (heads > 1 and between != D) or (tokens > 1 and pitch < n):
            raise ValueError(f"the heads of a token of {what} must be contiguous")
        return tokens, heads, pitch if tokens > 1 else n

    def append(self, k, v, table, lengths, offsets, max_new):
        """Quantises new keys and values [tokens, kv_heads, head_dim] (float32 / float16 / bfloat16; token stride free) into the
        cache.  See ltq_cache_append for the scales."""
        tokens, _, ld = self._rows(k, self.kv_heads, "k")
        if v.dtype is not k.dtype or self._rows(v, self.kv_heads, "v") != (tokens, self.kv_heads, ld):
            raise ValueError("k and v must have the same type, shape and strides")
        seqs, width = self._batch(table, lengths, offsets)
        check(lib().ltq_cache_append(self._ref, k.data_ptr(), v.data_ptr(), _tokens.dtype_code(k.dtype), ld, tokens, offsets.data_ptr(),
                                     lengths.data_ptr(), table.data_ptr(), seqs, width, max_new, self._index, _tokens.raw_stream(self._index)))

    def attention(self, q, table, lengths, offsets, max_new, scale=None, out=None, workspace=None):
        """Causal attention of the new tokens' queries [tokens, q_heads, head_dim] over the cache, which holds their keys already.
        Returns the same shape and type (`out`, contiguous, if given).  scale: default head_dim ** -0.5.  workspace: uint8
        CUDA tensor of at least ``attention_workspace`` bytes; made here if not given."""
        tokens, heads, ld = self._rows(q, None, "q")
        code = _tokens.dtype_code(q.dtype)
        seqs, width = self._batch(table, lengths, offsets)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif not (out.get_device() == self._index and out.dtype is q.dtype and out.shape == q.shape and out.is_contiguous()):
            raise ValueError("out must be a contiguous tensor of q's shape, type and device")
        if workspace is None:
            sizes = (tokens, heads, seqs, width, max_new)
            last = self._last   # sizes and bytes of a call before: a decode loop's calls have the same ones
            if last[0] != sizes:
                last = self._last = sizes, self.attention_workspace(*sizes)
            if last[1]:
                workspace = q.new_empty(last[1], dtype=torch.uint8)
        elif not (workspace.get_device() == self._index and workspace.dtype is torch.uint8 and workspace.is_contiguous()):
            raise ValueError("workspace must be a contiguous uint8 tensor on q's device")
        check(lib().ltq_cache_attention(self._ref, q.data_ptr(), code, ld, tokens, heads, offsets.data_ptr(), lengths.data_ptr(),
                                        table.data_ptr(), seqs, width, max_new, self.head_dim ** -0.5 if scale is None else scale,
                                        out.data_ptr(), workspace.data_ptr() if workspace is not None else None,
                                        workspace.numel() if workspace is not None else 0, self._index, _tokens.raw_stream(self._index)))
        return out

    def attention_workspace(self, tokens, q_heads, seqs, width, max_new):
        """Bytes of workspace that ``attention`` needs for these sizes."""
        return lib().ltq_cache_attention_workspace(self._ref, tokens, q_heads, seqs, width, max_new, self._index)

    def values(self, dtype=torch.float32):
        """Keys and values of all slots as numbers: two tensors [blocks, kv_heads, block_tokens, head_dim] of `dtype`."""
        code, shape = _tokens.dtype_code(dtype), self.k.shape
        rows, row, stream = self.blocks * self.kv_heads, self.block_tokens * self.head_dim, _tokens.raw_stream(self._index)
        out = self.k.new_empty(*shape, dtype=dtype), self.k.new_empty(*shape, dtype=dtype)
        for o, codes, qparams in zip(out, (self.k, self.v), (self.k_qparams, self.v_qparams)) if rows else ():
            check(lib().ltq_dequantize_tokens_u8(o.data_ptr(), code, row, codes.data_ptr(), qparams.data_ptr(), rows, row, self._index, stream))
        return out

    def check(self):
        """Waits for the stream and raises if a cache call met a sequence or block id outside its bounds since the last check."""
        check(lib().ltq_device_check(self._index, _tokens.raw_stream(self._index)))

"""Append attention of the LLM backbone on the B200 kernels
(``dllm_append_attention``, ``include/dllm.h``).

The reference prefills through flash-attn's variable-length call
(``nanovllm_dots/layers/attention.py:66-86``): the new tokens of every sequence,
packed, over the paged cache that already holds their K/V.
``B200AppendAttention.append`` is that call with capped scores, a distance bias,
sliding windows, bidirectional prefixes and packed documents; one new token a
sequence is the decode step under the same options.  ``verify`` attends for
trees of drafted tokens.  ``install_append_attention`` routes a reference
``Attention`` module's prefill through it.  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .llm_rotary import overlap

_DTYPES = {torch.bfloat16: _lib.DLLM_BF16, torch.float16: _lib.DLLM_FP16}
_pack = _lib.packer(_lib.DllmAppend)
TREE_MAX = 64     # drafted tokens of one sequence


def tree_masks(parents) -> torch.Tensor:
    """The masks ``verify`` takes, int64 [tokens], from each sequence's list of
    parents: ``parents[i][t]`` is the drafted token that token t continues, or -1
    for one that continues the history.  Bit u of a token's mask is set where
    token u is the token itself or one of its ancestors."""
    out = []
    for i, row in enumerate(parents):
        if len(row) > TREE_MAX:
            raise ValueError(f"sequence {i}: {len(row)} drafted tokens (at most {TREE_MAX})")
        bits = []
        for t, up in enumerate(row):
            if not -1 <= up < t:
                raise ValueError(f"sequence {i}: parent {up} of token {t} does not come before it")
            bits.append((bits[up] if up >= 0 else 0) | 1 << t)
        out += [b - (1 << 64) if b >> 63 else b for b in bits]
    return torch.tensor(out, dtype=torch.int64)


class B200AppendAttention:
    """Append attention of one model: heads, cache geometry and score options,
    with a workspace for up to ``max_tokens`` new tokens of ``max_seqs``
    sequences.

    The workspace serves one call at a time.  Calls on one stream follow each
    other; a call on another stream waits for the last one's stream, which has to
    exist until then.  A captured graph keeps using the workspace: replay graphs of
    one object, and call it, on one stream at a time, or give each an object of its
    own, as threads need that call at the same time.
    """

    def __init__(self, num_heads: int, head_dim: int, scale: float, num_kv_heads: int, *,
                 max_tokens: int, max_seqs: int, max_blocks: int, block_size: int = 256,
                 dtype: torch.dtype = torch.bfloat16, causal: bool = True, window: int = 0,
                 softcap: float = 0.0, slopes: torch.Tensor | None = None,
                 device: torch.device | str = "cuda"):
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("B200AppendAttention runs on a CUDA device only (no CPU path)")
        if dtype not in _DTYPES:
            raise RuntimeError(f"unsupported append-attention type {dtype}")
        if block_size < 16 or block_size % 16:
            raise RuntimeError(f"block_size {block_size}: expected a multiple of 16")
        if not 0 < scale < 3e38 or not 0 <= softcap < 3e38 or not 0 <= window < 1 << 31 or max_blocks < 1:
            raise RuntimeError("expected a positive scale and max_blocks, no negative softcap or window, "
                               "all finite and the window below 2^31")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.scale, self.softcap, self.window = float(scale), float(softcap), int(window)
        self.causal, self.dtype = bool(causal), dtype
        self.max_tokens, self.max_seqs = max_tokens, max_seqs
        self.max_blocks, self.block_size = max_blocks, block_size
        if slopes is not None:
            if slopes.shape != (num_heads,):
                raise RuntimeError(f"slopes: expected one for each of {num_heads} heads")
            slopes = slopes.to(device=self.device, dtype=torch.float32).contiguous()
        self.slopes = slopes
        self.L = _lib.lib()
        with torch.cuda.device(self.device):
            self.ws_bytes = int(self.L.dllm_append_workspace_size(max_tokens, max_seqs, num_heads,
                                                                  num_kv_heads, head_dim))
        if self.ws_bytes == 0:
            raise RuntimeError("unsupported append-attention shape")
        self.workspace = torch.empty(self.ws_bytes, dtype=torch.uint8, device=self.device)
        self.workspace[:256].zero_()
        torch.cuda.current_stream(self.device).synchronize()   # graphs may be replayed on any stream
        self._index = self.device.index
        self._dtype = _DTYPES[dtype]
        self._call = _lib.packed("dllm_append_attention", _lib.c_void_p, _lib.c_size_t, _lib.c_void_p)
        self._workspace = self.workspace.data_ptr()
        self._slopes = 0 if slopes is None else slopes.data_ptr()
        self._stream = _lib.raw_stream(self._index)   # the last one used: that of the zero-fill

    def _ints(self, name, t, dtype, shape):
        if t.dtype is not dtype or t.get_device() != self._index or t.shape != shape or not t.is_contiguous():
            raise RuntimeError(f"{name}: expected a contiguous {dtype} tensor of shape {shape} on "
                               f"{self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def _run(self, q, k_cache, v_cache, cu, ctx, table, prefix, first, tree, out, stream):
        H, D, index, dtype = self.num_heads, self.head_dim, self._index, self.dtype
        shape, rows, seqs = q.shape, table.shape, ctx.shape
        if len(shape) != 3 or shape[1] != H or shape[2] != D or q.dtype is not dtype or q.get_device() != index:
            raise RuntimeError(f"q: expected a {dtype} tensor [tokens, {H}, {D}] on {self.device}, "
                               f"got {q.dtype} {tuple(shape)} on {q.device}")
        T, n = shape[0], seqs[0] if seqs else 0
        if T > self.max_tokens or not 1 <= n <= self.max_seqs:
            raise RuntimeError(f"append of {T} tokens of {n} sequences "
                               f"(at most {self.max_tokens} of {self.max_seqs})")
        st, sh, sd = q.stride()
        if sd != 1 or T > 1 and (st % 8 or st < D) or H > 1 and (sh % 8 or sh < D) or q.data_ptr() % 16:
            raise RuntimeError("q: expected contiguous head dims and 16-byte aligned heads that share no memory")
        geometry = (k_cache.shape[0], self.block_size, self.num_kv_heads, D)
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            if c.dtype is not dtype or c.get_device() != index or c.shape != geometry or \
                    geometry[0] < 1 or not c.is_contiguous():
                raise RuntimeError(f"{name}: expected a contiguous {dtype} tensor [num_blocks, "
                                   f"{', '.join(map(str, geometry[1:]))}] on {self.device}, both caches alike")
        if len(rows) != 2 or not 1 <= rows[1] <= self.max_blocks:
            raise RuntimeError(f"block_tables: expected [{n}, 1..{self.max_blocks}]")
        if out is None:
            if stream is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
            else:     # owned by the stream that writes it
                with torch.cuda.stream(stream):
                    out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.dtype is not dtype or out.get_device() != index or out.shape != (T, H, D) or \
                not out.is_contiguous():
            raise RuntimeError(f"out: expected a contiguous {dtype} tensor {(T, H, D)} on {self.device}")
        elif out.data_ptr() % 32:
            raise RuntimeError("out: expected 32-byte alignment")
        elif overlap(q, out) and not (out.data_ptr() == q.data_ptr() and q.is_contiguous()):
            raise RuntimeError("out: overlaps q without being q")
        elif T and any(c.data_ptr() < out.data_ptr() + out.nbytes and out.data_ptr() < c.data_ptr() + c.nbytes
                       for c in (k_cache, v_cache)):
            raise RuntimeError("out: overlaps a cache")
        i32, width = torch.int32, rows[1]
        plain = tree is None
        a = _pack(
            self._dtype, T, n, H, self.num_kv_heads, D, geometry[0], self.block_size, width, self.causal,
            self.window if plain else 0, self.scale, self.softcap, q.data_ptr(), st, sh,
            k_cache.data_ptr(), v_cache.data_ptr(), self._ints("cu_seqlens_q", cu, i32, (n + 1,)),
            self._ints("context_lens", ctx, i32, (n,)), self._ints("block_tables", table, i32, (n, width)),
            0 if prefix is None else self._ints("prefix_lens", prefix, i32, (n,)),
            0 if first is None else self._ints("first_keys", first, i32, (T,)),
            0 if plain else self._ints("tree_masks", tree, torch.int64, (T,)),
            self._slopes if plain else 0, out.data_ptr())
        if T == 0:
            return out
        handle = _lib.raw_stream(index) if stream is None else stream.cuda_stream
        if handle != self._stream:
            self._follow(handle)
        rc = _lib.call_on(index, self._call, a, self._workspace, self.ws_bytes, handle)
        if rc:
            _lib.check(rc, "dllm_append_attention")
        return out

    def _follow(self, handle: int) -> None:
        """The workspace may still be in use on the stream of the last call.  (A
        capture cannot wait for one outside it.)"""
        def stream(h):
            return torch.cuda.ExternalStream(h, device=self.device) if h else \
                torch.cuda.default_stream(self.device)

        with torch.cuda.stream(stream(handle)):
            if torch.cuda.is_current_stream_capturing():
                return
        stream(handle).wait_stream(stream(self._stream))
        self._stream = handle

    def append(self, q, k_cache, v_cache, cu_seqlens_q, context_lens, block_tables, *,
               prefix_lens: torch.Tensor | None = None, first_keys: torch.Tensor | None = None,
               out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """q [tokens, H, D]: the newest tokens of n sequences, packed; int32
        cu_seqlens_q [n + 1] where each sequence's begin; int32 context_lens [n]
        cached positions, the new tokens included; int32 block_tables [n, width].
        prefix_lens [n]: leading positions every token of the sequence sees,
        whatever its own; first_keys [tokens]: the first position a token sees
        (its document's).  -> [tokens, H, D] (``out=q`` overwrites a contiguous
        q); zeros where a token sees nothing, rows past cu_seqlens_q[n] as they
        were (in an ``out`` of its own: undefined)."""
        return self._run(q, k_cache, v_cache, cu_seqlens_q, context_lens, block_tables, prefix_lens,
                         first_keys, None, out, stream)

    def verify(self, q, k_cache, v_cache, cu_seqlens_q, context_lens, block_tables,
               tree_masks: torch.Tensor, *, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """``append`` for trees of drafted tokens, at most 64 a sequence, whose
        K/V stand in the cache in the order of q.  A token sees the history
        before them and the drafted tokens whose bits are set in its int64 mask
        (``tree_masks(parents)``).  ``causal`` plays no part."""
        if self.slopes is not None or self.window:
            raise RuntimeError("verify: not supported with slopes or a window")
        return self._run(q, k_cache, v_cache, cu_seqlens_q, context_lens, block_tables, None, None,
                         tree_masks, out, stream)

    def check_errors(self) -> None:
        """Wait for the device (calls and replayed graphs may be on any stream) and
        raise if a kernel reported an error."""
        torch.cuda.synchronize(self.device)
        v = _lib.c_uint32(0)
        s = torch.cuda.current_stream(self.device)
        with torch.cuda.device(self.device):
            _lib.check(self.L.dllm_read_error(_lib.ptr(self.workspace), _lib.c_void_p(s.cuda_stream), v),
                       "dllm_read_error")
        if v.value:
            names = [nm for bit, nm in _lib.DEVERR_BITS.items() if v.value & bit]
            raise RuntimeError(f"append attention device error: {', '.join(names)} (0x{v.value:x})")


def install_append_attention(module, get_context, att: B200AppendAttention, store_kvcache) -> None:
    """Route a reference ``Attention`` module's prefill over the paged cache through ``att``.

    ``get_context`` and ``store_kvcache`` are the reference's own
    (``nanovllm_dots.utils.context.get_context``, ``layers/attention.py:33-47``),
    passed in so that this package does not import the reference.  When the
    context is a prefill with block tables (``attention.py:66-86``) the module's
    forward stores this call's k and v at ``slot_mapping`` and becomes
    ``att.append`` over ``cu_seqlens_q`` and the lengths in ``cu_seqlens_k``;
    every other call keeps the forward that was there, so that
    ``install_decode_attention`` may come before or after."""
    original = module.forward

    def forward(q, k, v):
        ctx = get_context()
        if not getattr(module, "is_causal", True) or not ctx.is_prefill or ctx.block_tables is None \
                or not module.k_cache.numel():
            return original(q, k, v)
        store_kvcache(k.view(-1, module.num_kv_heads, module.head_dim),
                      v.view(-1, module.num_kv_heads, module.head_dim), module.k_cache, module.v_cache,
                      ctx.slot_mapping)
        lens = ctx.cu_seqlens_k[1:] - ctx.cu_seqlens_k[:-1]
        return att.append(q.view(-1, module.num_heads, module.head_dim), module.k_cache, module.v_cache,
                          ctx.cu_seqlens_q, lens, ctx.block_tables)

    module.forward = forward

"""Rotary positions of the LLM backbone on the B200 kernels (``dllm_rotary``,
``include/dllm.h``).

The reference rotates whole heads in the half layout at unscaled frequencies
(``nanovllm_dots/layers/rotary_embedding.py:6-47``) and stores k and v with a
kernel of its own (``layers/attention.py:10-47``).  ``B200Rotary`` does both in
one launch, in either pair layout, over part of a head, at frequencies scaled
for contexts longer than the trained one.  There is no CPU path.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DLLM_BF16, torch.float16: _lib.DLLM_FP16,
           torch.float32: _lib.DLLM_FP32}
_pack = _lib.packer(_lib.DllmRotary)
KINDS = ("linear", "ntk", "bands", "yarn")
LAYOUTS = ("half", "interleaved")


@dataclass(frozen=True)
class RotaryScaling:
    """How the frequencies w_i = theta^(-2i / rot_dim) change for a context
    ``factor`` times the ``original_max`` positions of training:

    * ``linear``: w_i / factor;
    * ``ntk``: theta becomes theta * factor^(rot_dim / (rot_dim - 2));
    * ``bands``: waves that turn at least ``high_freq`` times in the original
      context keep w_i, those below ``low_freq`` turns get w_i / factor, and the
      turns between blend the two linearly;
    * ``yarn`` (Peng et al., 2023): the blend runs over the pair index between
      the pairs that turn ``beta_fast`` and ``beta_slow`` times, and cos and sin
      are multiplied by 0.1 ln(factor) + 1 (``attention_factor`` overrides).
    """
    kind: str
    factor: float
    original_max: int = 0
    low_freq: float = 1.0
    high_freq: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None


def rotary_frequencies(rot_dim: int, theta: float, scaling: RotaryScaling | None = None
                       ) -> tuple[torch.Tensor, float]:
    """(radians a position of each pair, in float64 [rot_dim / 2]; factor on cos and sin)."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim {rot_dim}: expected an even number of dims")
    if not theta > 1.0 or not math.isfinite(theta):
        raise ValueError(f"theta {theta}: expected a finite base above 1")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    inv = theta ** (-i / rot_dim)
    if scaling is None:
        return inv, 1.0
    s = scaling
    if s.kind not in KINDS:
        raise ValueError(f"rotary scaling {s.kind!r}: expected one of {KINDS}")
    if not s.factor >= 1.0 or not math.isfinite(s.factor):
        raise ValueError(f"rotary scaling factor {s.factor}: expected at least 1")
    if s.kind in ("bands", "yarn") and s.original_max < 1:
        raise ValueError(f"rotary scaling {s.kind!r} needs original_max")
    factor = 1.0 if s.attention_factor is None else float(s.attention_factor)
    if s.kind == "linear":
        return inv / s.factor, factor
    if s.kind == "ntk":
        if rot_dim == 2:
            raise ValueError("rotary scaling 'ntk' needs rot_dim above 2")
        return (theta * s.factor ** (rot_dim / (rot_dim - 2))) ** (-i / rot_dim), factor
    if s.kind == "bands":
        if not s.high_freq > s.low_freq:
            raise ValueError("rotary scaling 'bands': expected high_freq above low_freq")
        turns = s.original_max * inv / (2 * math.pi)
        keep = ((turns - s.low_freq) / (s.high_freq - s.low_freq)).clamp(0, 1)
    else:
        if not s.beta_fast > s.beta_slow > 0:
            raise ValueError("rotary scaling 'yarn': expected beta_fast above beta_slow above 0")

        def pair(turns):    # the (fractional) pair that turns so often in the original context
            return rot_dim * math.log(s.original_max / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low = max(math.floor(pair(s.beta_fast)), 0)
        high = min(math.ceil(pair(s.beta_slow)), rot_dim - 1)
        keep = 1 - ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        if s.attention_factor is None:
            factor = 0.1 * math.log(s.factor) + 1.0
    return inv / s.factor * (1 - keep) + inv * keep, factor


def _two_pi(bits: int) -> int:
    """2 pi * 2^bits as an integer (Machin: pi = 16 arctan(1/5) - 4 arctan(1/239))."""
    one = 1 << (bits + 16)

    def arctan(n):
        term, total, k = one // n, 0, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total

    return (32 * arctan(5) - 8 * arctan(239)) >> 16


_TWO_PI = _two_pi(192)


def _turns(inv: torch.Tensor) -> torch.Tensor:
    """Frequencies as turns a position, a binary fraction of 2^64 in int64: each
    float64 frequency by 2 pi in integer arithmetic, rounded once."""
    out = []
    for w in inv.tolist():
        n, d = w.as_integer_ratio()
        scaled, by = n << (64 + 192), d * _TWO_PI
        bits = (2 * scaled + by) // (2 * by) & ((1 << 64) - 1)
        out.append(bits - (1 << 64) if bits >> 63 else bits)
    return torch.tensor(out, dtype=torch.int64)


class B200Rotary:
    """Rotary of one model: head size, layout and frequencies.  Rotated values
    are computed in fp32 and rounded once; the angle is that of the frequencies
    in float64 to 2^-31 turns, at every int32 position."""

    def __init__(self, head_dim: int, *, theta: float = 10000.0, rot_dim: int | None = None,
                 layout: str = "half", scaling: RotaryScaling | None = None,
                 device: torch.device | str = "cuda"):
        if layout not in LAYOUTS:
            raise ValueError(f"rotary layout {layout!r}: expected one of {LAYOUTS}")
        rot_dim = head_dim if rot_dim is None else rot_dim
        if head_dim < 2 or head_dim % 2 or rot_dim > head_dim:
            raise ValueError(f"head_dim {head_dim}, rot_dim {rot_dim}: expected even sizes, "
                             "rot_dim at most head_dim")
        inv, factor = rotary_frequencies(rot_dim, theta, scaling)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("B200Rotary runs on a CUDA device only (no CPU path)")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.head_dim, self.rot_dim, self.layout, self.factor = head_dim, rot_dim, layout, factor
        self.L = _lib.lib()
        self.turns = _turns(inv).to(self.device)
        self.err = torch.zeros(64, dtype=torch.int32, device=self.device)
        torch.cuda.current_stream(self.device).synchronize()   # calls may come on any stream
        self._size = {_lib.DLLM_BF16: 2, _lib.DLLM_FP16: 2, _lib.DLLM_FP32: 4}
        self._index, self._inter = self.device.index, layout == "interleaved"
        self._call = _lib.packed("dllm_rotary", _lib.c_void_p)
        self._turns, self._err = self.turns.data_ptr(), self.err.data_ptr()

    def _heads(self, name, t, dtype, tokens):
        """[tokens, heads, head_dim] with contiguous head dims -> its heads and strides."""
        shape = t.shape
        if len(shape) != 3 or shape[2] != self.head_dim or t.get_device() != self._index:
            raise RuntimeError(f"{name}: expected [tokens, heads, {self.head_dim}] on {self.device}, "
                               f"got {tuple(shape)} on {t.device}")
        if t.dtype is not dtype:
            raise RuntimeError(f"{name}: expected {dtype}, got {t.dtype}")
        if shape[0] != tokens:
            raise RuntimeError(f"{name}: expected {tokens} tokens, got {shape[0]}")
        ts, hs, one = t.stride()
        if one != 1:
            raise RuntimeError(f"{name}: expected contiguous head dims")
        return shape[1], ts, hs

    def _ints(self, name, t, tokens):
        if t.dtype is not torch.int32 or t.get_device() != self._index or t.shape != (tokens,) or \
                not t.is_contiguous():
            raise RuntimeError(f"{name}: expected a contiguous int32 [{tokens}] on {self.device}")
        return t.data_ptr()

    def _check_apart(self, read, out, T, size, kc, vc, room):
        """Raises where the store's outputs share memory with each other or with what
        the call reads (out may be q).  Tensors come with address, token and head
        strides and heads: where their spans cross, slices of one packed row are
        apart by their places in it, heads that take turns by theirs, and else every
        row is looked at (milliseconds)."""
        D = self.head_dim
        if abs(kc - vc) < room:
            raise RuntimeError("k_cache and v_cache overlap")
        for t, p, ts, hs, n in read if out is None else (*read, out):
            end = p + ((T - 1) * ts + (n - 1) * hs + D) * size
            if (p < kc + room and end > kc and meets(t, kc, kc + room)) or \
                    (p < vc + room and end > vc and meets(t, vc, vc + room)):
                raise RuntimeError("q, k, v or out overlaps a cache")
        if out is None:
            return
        t, p, ts, hs, n = out
        row, wide = ts * size, ((n - 1) * hs + D) * size
        for other, p2, ts2, hs2, n2 in read[1:]:
            wide2 = ((n2 - 1) * hs2 + D) * size
            if p2 + (T - 1) * ts2 * size + wide2 <= p or p + (T - 1) * row + wide <= p2 or \
                    (ts == ts2 and row and wide <= (p2 - p) % row <= row - wide2) or \
                    (hs == hs2 and hs and ts % hs == ts2 % hs == 0 and
                     D * size <= (p2 - p) % (hs * size) <= (hs - D) * size):
                continue
            if shared(t, other):
                raise RuntimeError("out: overlaps k or v")

    def _run(self, q, positions, out, stream, store):
        dtype, given = _DTYPES.get(q.dtype), out is not None
        if dtype is None:
            raise RuntimeError(f"q: unsupported type {q.dtype}")
        T = q.shape[0]
        heads, qt, qh = self._heads("q", q, q.dtype, T)
        pos = self._ints("positions", positions, T)
        if out is None:
            if stream is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
            else:       # owned by the stream that writes it
                with torch.cuda.stream(stream):
                    out = torch.empty_like(q, memory_format=torch.contiguous_format)
            ot, oh = heads * self.head_dim, self.head_dim
        else:
            oheads, ot, oh = self._heads("out", out, q.dtype, T)
            if oheads != heads:
                raise RuntimeError(f"out: expected shape {tuple(q.shape)}")
            if out.data_ptr() == q.data_ptr():
                if (qt, qh) != (ot, oh):
                    raise RuntimeError("out: rotating in place needs q's own strides")
            elif overlap(q, out):
                raise RuntimeError("out: overlaps q without being q")
            if not _apart(out):
                raise RuntimeError("out: rows share memory")
        kvh = kt = kh = vt = vh = slots = places = kp = vp = kcp = vcp = 0
        if store is not None:
            k, v, slot_mapping, k_cache, v_cache = store
            kvh, kt, kh = self._heads("k", k, q.dtype, T)
            vheads, vt, vh = self._heads("v", v, q.dtype, T)
            if kvh != vheads or kvh < 1:
                raise RuntimeError("k and v have different heads, or none")
            places = self._ints("slot_mapping", slot_mapping, T)
            shape, cache_type = k_cache.shape, q.dtype
            good = len(shape) == 4 and shape[0] and shape[1] and shape[2] == kvh and shape[3] == self.head_dim
            for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
                if not good or c.dtype is not cache_type or c.get_device() != self._index or \
                        c.shape != shape or not c.is_contiguous():
                    raise RuntimeError(f"{name}: expected a contiguous {q.dtype} [num_blocks, block_size, "
                                       f"{kvh}, {self.head_dim}] on {self.device}, and both caches alike")
            slots = shape[0] * shape[1]
            kp, vp, qp = k.data_ptr(), v.data_ptr(), q.data_ptr()
            kcp, vcp = k_cache.data_ptr(), v_cache.data_ptr()
            D, size, t1 = self.head_dim, self._size[dtype], T - 1
            room = slots * kvh * D * size
            kce, vce, qe = kcp + room, vcp + room, qp + (t1 * qt + (heads - 1) * qh + D) * size
            ke, ve = kp + (t1 * kt + (kvh - 1) * kh + D) * size, vp + (t1 * vt + (kvh - 1) * vh + D) * size
            if T and (given or kcp < vce and vcp < kce or qp < kce and kcp < qe or qp < vce and vcp < qe or
                      kp < kce and kcp < ke or kp < vce and vcp < ke or vp < kce and kcp < ve or
                      vp < vce and vcp < ve):
                self._check_apart(((q, qp, qt, qh, heads), (k, kp, kt, kh, kvh), (v, vp, vt, vh, kvh)),
                                  (out, out.data_ptr(), ot, oh, heads) if given else None, T, size, kcp, vcp, room)
        if T == 0 or heads == 0 and store is None:
            return out
        a = _pack(dtype, T, heads, kvh, self.head_dim, self.rot_dim, self._inter, self.factor,
                  self._turns, pos, q.data_ptr(), out.data_ptr(), kp, vp, kcp, vcp, places,
                  qt, qh, ot, oh, kt, kh, vt, vh, slots, self._err)
        handle = _lib.raw_stream(self._index) if stream is None else stream.cuda_stream
        rc = _lib.call_on(self._index, self._call, a, handle)
        if rc:
            _lib.check(rc, "dllm_rotary")
        return out

    def rotate(self, q, positions, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """q [tokens, heads, head_dim] (any token and head strides) at int32
        positions [tokens] -> out (``out=q`` rotates in place)."""
        return self._run(q, positions, out, stream, None)

    def rotate_store(self, q, k, v, positions, slot_mapping, k_cache, v_cache,
                     out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """Rotates q as ``rotate`` does and writes rotated k and unrotated v
        [tokens, kv_heads, head_dim] into the paged caches [num_blocks,
        block_size, kv_heads, head_dim] at int32 slot_mapping [tokens] (block *
        block_size + offset; -1 stores nothing).  Two tokens must not share a
        slot.  A slot past the cache is not stored and reported by
        ``check_errors``.  The caches share no memory with each other nor with q,
        k or v, and out none with k, v and the caches."""
        return self._run(q, positions, out, stream, (k, v, slot_mapping, k_cache, v_cache))

    def check_errors(self) -> None:
        """Wait for the device (calls and replayed graphs may be on any stream) and
        raise if a slot past the cache was met."""
        torch.cuda.synchronize(self.device)
        v = _lib.c_uint32(0)
        s = torch.cuda.current_stream(self.device)
        with torch.cuda.device(self.device):
            _lib.check(self.L.dllm_read_error(_lib.ptr(self.err), _lib.c_void_p(s.cuda_stream), v),
                       "dllm_read_error")
        if v.value:
            names = [nm for bit, nm in _lib.DEVERR_BITS.items() if v.value & bit]
            raise RuntimeError(f"rotary device error: {', '.join(names)} (0x{v.value:x})")


def _span(t):
    """First byte of a tensor's elements and the one behind the last."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def overlap(a, b) -> bool:
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _starts(t):
    """First bytes of the rows of [tokens, heads, dims], sorted, and a row's length."""
    size = t.element_size()
    token, head = (torch.arange(n, device="cpu") for n in t.shape[:2])
    at = (token[:, None] * t.stride(0) + head * t.stride(1)) * size
    return (at.flatten() + t.data_ptr()).sort().values, t.shape[2] * size


def meets(t, lo: int, hi: int) -> bool:
    """Whether a row of [tokens, heads, dims] reaches into the bytes [lo, hi)."""
    at, room = _starts(t)
    return bool(((at < hi) & (at + room > lo)).any())


def shared(a, b) -> bool:
    """Whether two tensors [tokens, heads, dims] have elements in common, which
    spans that cross do not say: heads of a packed row may take turns."""
    if not overlap(a, b):
        return False
    (x, wx), (y, wy) = _starts(a), _starts(b)
    # rows of y before the end of a row of x, of which the last reaches into it
    i = torch.searchsorted(y, x + wx) - 1
    return bool(((i >= 0) & (y[i.clamp(min=0)] + wy > x)).any())


def _apart(t) -> bool:
    """Whether no two elements of [tokens, heads, dims] share memory."""
    if not t.numel():
        return True
    room = t.shape[2]
    for n, stride in sorted(((t.shape[0], t.stride(0)), (t.shape[1], t.stride(1))), key=lambda x: x[1]):
        if n > 1:
            if stride < room:
                return False
            room = (n - 1) * stride + room
    return True

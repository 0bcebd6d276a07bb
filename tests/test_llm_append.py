"""Rotary and append attention without a GPU: the C ABI's layouts and refusals,
frequency scalings, tree masks, and the oracle against plain attention."""
from __future__ import annotations

import ctypes
import math
import os
import shutil
import subprocess
from fractions import Fraction

import pytest
import torch

from nanovllm_dots_b200 import _lib
from nanovllm_dots_b200.llm_append import B200AppendAttention, tree_masks
from nanovllm_dots_b200.llm_rotary import B200Rotary, RotaryScaling, _turns, meets, rotary_frequencies, shared
from oracle import llm_append_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4


# ------------------------------------------------------------------ ABI
@pytest.mark.parametrize("name", ["DllmRotary", "DllmAppend"])
def test_struct_matches_header(name, tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    cls = getattr(_lib, name)
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "dllm.h"\nint main(void) {\n'
                   + f'printf("%zu\\n", sizeof({name}));\n'
                   + "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f, _ in cls._fields_)
                   + "return 0; }\n")
    subprocess.run([cc, "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src),
                    "-o", str(exe)], check=True, capture_output=True, text=True)
    said = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True,
                                           text=True).stdout.split()]
    assert said == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]


@pytest.mark.parametrize("args", [_lib.DllmRotary, _lib.DllmAppend])
def test_packed_arguments_are_the_structure(args):
    values = [i + 0.5 if t is ctypes.c_float else (1 << 40) + i if ctypes.sizeof(t) == 8 else -i
              for i, (_, t) in enumerate(args._fields_)]
    assert _lib.packer(args)(*values) == bytes(args(*values))


# pointers of refused calls are never followed: the checks come first
A = 1 << 12


def rotary(**over):
    a = dict(dtype=0, tokens=3, q_heads=2, kv_heads=1, head_dim=64, rot_dim=64, interleaved=0,
             factor=1.0, turns=A, positions=A, q=A, q_out=2 * A, k=A, v=A, k_cache=A, v_cache=A,
             slot_mapping=A, q_token_stride=128, q_head_stride=64, out_token_stride=128,
             out_head_stride=64, k_token_stride=64, k_head_stride=64, v_token_stride=64,
             v_head_stride=64, num_slots=16, err_word=A)
    a.update(over)
    return _lib.lib().dllm_rotary(_lib.DllmRotary(**a), None)


@pytest.mark.parametrize("over,code", [
    (dict(dtype=3), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED), (dict(tokens=-1), INVALID),
    (dict(q_heads=0), INVALID), (dict(head_dim=63), INVALID), (dict(rot_dim=0), INVALID),
    (dict(rot_dim=3), INVALID), (dict(rot_dim=66), INVALID), (dict(turns=None), INVALID),
    (dict(positions=None), INVALID), (dict(q=None), INVALID), (dict(q_out=None), INVALID),
    (dict(v=None), INVALID), (dict(k_cache=None), INVALID), (dict(v_cache=None), INVALID),
    (dict(slot_mapping=None), INVALID), (dict(err_word=None), INVALID), (dict(kv_heads=0), INVALID),
    (dict(num_slots=0), INVALID), (dict(q_out=A, out_token_stride=256), INVALID),
    (dict(tokens=0), OK)])
def test_rotary_refusals(over, code):
    assert rotary(**over) == code


def append(ws=1 << 12, size=1 << 30, **over):
    a = dict(dtype=0, tokens=8, n=2, num_heads=12, num_kv_heads=2, head_dim=128, num_blocks=4,
             block_size=256, max_blocks=4, causal=1, window=0, scale=0.1, softcap=0.0, q=A,
             q_token_stride=1536, q_head_stride=128, k_cache=A, v_cache=A, cu_seqlens_q=A,
             context_lens=A, block_table=A, prefix_lens=None, first_keys=None, tree_masks=None,
             slopes=None, out=A)
    a.update(over)
    return _lib.lib().dllm_append_attention(_lib.DllmAppend(**a), ctypes.c_void_p(ws), size, None)


@pytest.mark.parametrize("over,code", [
    (dict(ws=0), INVALID), (dict(ws=(1 << 12) + 16), INVALID), (dict(size=1 << 16), WORKSPACE),
    (dict(dtype=2), UNSUPPORTED), (dict(n=0), UNSUPPORTED), (dict(tokens=-1), UNSUPPORTED),
    (dict(num_heads=13), UNSUPPORTED), (dict(num_heads=258), UNSUPPORTED),
    (dict(num_kv_heads=0), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED),
    (dict(tokens=2 ** 31 - 1, num_heads=256), WORKSPACE),
    (dict(block_size=24), UNSUPPORTED), (dict(block_size=8), UNSUPPORTED),
    (dict(block_size=1 << 16, max_blocks=1 << 15), UNSUPPORTED),
    (dict(num_blocks=0), INVALID), (dict(max_blocks=0), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=math.nan), INVALID), (dict(scale=math.inf), INVALID), (dict(softcap=-1.0), INVALID),
    (dict(softcap=math.nan), INVALID), (dict(softcap=1e-39), UNSUPPORTED), (dict(window=-1), INVALID),
    (dict(max_blocks=1 << 22, tokens=100000, size=1 << 40), UNSUPPORTED), (dict(q_token_stride=1540), INVALID),
    (dict(q_head_stride=4), INVALID), (dict(q_head_stride=64), INVALID), (dict(q_token_stride=0), INVALID),
    (dict(q_head_stride=-128), INVALID), (dict(q=A + 2), INVALID), (dict(k_cache=A + 8), INVALID),
    (dict(out=A + 8), INVALID), (dict(tree_masks=A, slopes=A), UNSUPPORTED),
    (dict(tree_masks=A, window=3), UNSUPPORTED), (dict(tree_masks=A, prefix_lens=A), UNSUPPORTED),
    (dict(tree_masks=A, first_keys=A), UNSUPPORTED), (dict(tokens=0), OK)]
    + [({f: None}, INVALID) for f in ("q", "k_cache", "v_cache", "cu_seqlens_q", "context_lens",
                                      "block_table", "out")])
def test_append_refusals(over, code):
    assert append(**over) == code


@pytest.mark.parametrize("scale,softcap,code", [
    (0.1, 1e16, OK), (0.1, 1e18, UNSUPPORTED), (0.1, 3e38, UNSUPPORTED), (1e-30, 1e15, UNSUPPORTED),
    (1e-20, 3e38, UNSUPPORTED), (1e-12, 1.0, OK)])
def test_append_refuses_caps_beyond_its_arithmetic(scale, softcap, code):
    """The square of a score below the cap, and the cap's constants, have to fit fp32."""
    assert append(scale=scale, softcap=softcap, tokens=0) == code


def test_append_workspace_size():
    size = _lib.lib().dllm_append_workspace_size
    assert size(8, 2, 12, 2, 128) > size(8, 2, 12, 2, 64) > 0
    assert size(100000, 2, 12, 2, 64) > size(8, 2, 12, 2, 64)
    assert size(8, 2, 12, 2, 96) == size(8, 2, 12, 5, 64) == size(8, 0, 12, 2, 64) == 0
    assert size(8, 2, 129, 1, 64) == 0 < size(8, 2, 128, 1, 64)


# ------------------------------------------------------------------ host side
def test_classes_refuse_what_they_cannot_do():
    with pytest.raises(RuntimeError, match="CUDA"):
        B200Rotary(64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        B200AppendAttention(12, 128, 0.1, 2, max_tokens=8, max_seqs=1, max_blocks=1, device="cpu")
    for kw in (dict(layout="pairs"), dict(rot_dim=66), dict(rot_dim=3), dict(theta=1.0), dict(theta=math.inf),
               dict(scaling=RotaryScaling("cubic", 2.0)), dict(scaling=RotaryScaling("linear", 0.5)),
               dict(scaling=RotaryScaling("yarn", 2.0)), dict(scaling=RotaryScaling("bands", 2.0)),
               dict(rot_dim=2, scaling=RotaryScaling("ntk", 2.0)),
               dict(scaling=RotaryScaling("bands", 2.0, 4096, low_freq=4.0)),
               dict(scaling=RotaryScaling("yarn", 2.0, 4096, beta_fast=1.0))):
        with pytest.raises(ValueError):
            B200Rotary(64, **kw)
    for kw in (dict(dtype=torch.float32), dict(block_size=40), dict(scale=0.0), dict(softcap=-1.0),
               dict(window=-1), dict(max_blocks=0)):
        kw = {"scale": 0.1, "max_blocks": 1, **kw}
        with pytest.raises(RuntimeError):
            B200AppendAttention(12, 128, kw.pop("scale"), 2, max_tokens=8, max_seqs=1, device="cuda:0", **kw)


@pytest.mark.parametrize("kw", [dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e39), dict(softcap=math.nan),
                                dict(softcap=math.inf), dict(softcap=1e39), dict(window=1 << 31), dict(window=1 << 70)])
def test_options_beyond_their_fields_are_refused_at_once(kw):
    kw = {"scale": 0.1, **kw}
    with pytest.raises(RuntimeError, match="expected a positive scale"):
        B200AppendAttention(12, 128, kw.pop("scale"), 2, max_tokens=8, max_seqs=1, max_blocks=1, device="cuda:0", **kw)


def test_frequencies():
    plain, one = rotary_frequencies(128, 1e6)
    assert one == 1.0 and plain.dtype == torch.float64
    # the reference's table (rotary_embedding.py:26-27)
    assert torch.allclose(plain.float(), 1.0 / 1e6 ** (torch.arange(0, 128, 2).float() / 128), rtol=1e-6)
    assert torch.equal(rotary_frequencies(128, 1e6, RotaryScaling("linear", 4.0))[0], plain / 4)
    ntk, _ = rotary_frequencies(128, 1e6, RotaryScaling("ntk", 4.0))
    assert ntk[0] == 1.0 and abs(float(ntk[-1] / plain[-1]) - 0.25) < 1e-12    # slowest pair: all of the factor
    bands, _ = rotary_frequencies(128, 1e6, RotaryScaling("bands", 4.0, 8192))
    turns = 8192 * plain / (2 * math.pi)
    assert torch.equal(bands[turns >= 4], plain[turns >= 4]) and torch.equal(bands[turns <= 1], plain[turns <= 1] / 4)
    assert (bands <= plain).all() and (bands >= plain / 4).all() and (bands.diff() < 0).all()
    yarn, f = rotary_frequencies(128, 1e6, RotaryScaling("yarn", 4.0, 8192))
    assert f == 0.1 * math.log(4.0) + 1.0
    assert torch.equal(yarn[turns >= 33], plain[turns >= 33]) and torch.equal(yarn[turns < 0.8], plain[turns < 0.8] / 4)
    assert rotary_frequencies(128, 1e6, RotaryScaling("yarn", 4.0, 8192, attention_factor=1.0))[1] == 1.0


def test_turns_keep_the_angle_at_far_positions():
    """position * turns modulo 2^64 is the angle: against exact integer arithmetic."""
    inv, _ = rotary_frequencies(64, 10000.0)
    for w, t in zip(inv.tolist(), _turns(inv).tolist()):
        for pos in (1, 12345, 2 ** 31 - 1):
            got = (pos * (t & (1 << 64) - 1)) % (1 << 64) / 2.0 ** 64 * 2 * math.pi
            gap = abs(math.remainder(got - math.fmod(pos * w, 2 * math.pi), 2 * math.pi))
            # the fraction of 2^64 is rounded: half a unit a position, in radians
            assert gap <= pos * (w * 2.0 ** -51 + math.pi * 2.0 ** -64) + 1e-12


def exact_two_pi():
    """2 pi as a fraction, from Euler's pi = 20 arctan(1/7) + 8 arctan(3/79)."""
    def arctan(x):
        total, power, k = Fraction(0), x, 1
        while abs(power) > Fraction(1, 1 << 220):
            total += power / k if k % 4 == 1 else -power / k
            power, k = power * x * x, k + 2
        return total

    return 2 * (20 * arctan(Fraction(1, 7)) + 8 * arctan(Fraction(3, 79)))


@pytest.mark.parametrize("rot,theta,scaling", [(128, 1e6, None), (64, 10000.0, None), (2, 5e4, None),
                                               (64, 1e6, RotaryScaling("yarn", 16.0, 4096)),
                                               (128, 5e5, RotaryScaling("bands", 8.0, 8192))])
def test_turns_are_rounded_to_the_last_bit(rot, theta, scaling):
    """Against rational arithmetic: half a unit of 2^-64 turns a position, which is
    |position| 2^-65 turns of the angle."""
    inv, _ = rotary_frequencies(rot, theta, scaling)
    period = exact_two_pi()
    for w, t in zip(inv.tolist(), _turns(inv).tolist()):
        off = Fraction(t % (1 << 64)) - Fraction(w) / period * (1 << 64)
        assert abs(off) <= Fraction(1, 2) + Fraction(1, 1 << 100)


def test_shared_memory_is_found_element_by_element():
    """Against the sets of the elements' addresses, for views of one buffer at random."""
    import random

    r = random.Random(0)
    room = torch.zeros(4000, dtype=torch.bfloat16)

    def view():
        n, heads, dims = r.randint(0, 5), r.randint(1, 4), r.choice((2, 4, 8))
        ts, hs = r.choice((0, 8, 24, 40, 96, 97)), r.choice((0, 2, 8, 10, 24))
        return room.as_strided((n, heads, dims), (ts, hs, 1), r.randint(0, 300))

    def bytes_of(t):
        return {t.data_ptr() + 2 * (i * t.stride(0) + j * t.stride(1) + d) for i in range(t.shape[0])
                for j in range(t.shape[1]) for d in range(t.shape[2])}

    seen = set()
    for _ in range(3000):
        a, b = view(), view()
        want = bool(bytes_of(a) & bytes_of(b))
        assert shared(a, b) == want == shared(b, a)
        lo = room.data_ptr() + 2 * r.randint(0, 400)
        hi = lo + 2 * r.randint(1, 60)
        inside = any(lo <= x < hi for x in bytes_of(a))
        assert meets(a, lo, hi) == inside
        seen.add((want, inside))
    assert len(seen) == 4
    packed = torch.zeros(7, 16, 8)           # a packed projection, and one interleaved by heads
    assert not shared(packed[:, :12], packed[:, 12:14]) and shared(packed[:, :13], packed[:, 12:14])
    assert not shared(packed[:, 0::2], packed[:, 1::2]) and shared(packed[:, 0::2], packed[:, 0::4])


def test_store_check_refuses_exactly_what_shares_memory():
    """The strides' short cuts and the search behind them against sets of addresses."""
    import random
    from types import SimpleNamespace as NS

    r, room = random.Random(1), torch.zeros(6000, dtype=torch.bfloat16)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        T, D = r.randint(1, 4), r.choice((2, 4))
        ts, hs = r.choice((12, 24, 48, 96, 40)), r.choice((D, 2 * D, 3 * D, 12, 24, 96))

        def view(heads):
            t, h = (ts, hs) if r.random() < 0.7 else (r.choice((8, 24, 50)), r.choice((D, 6, 16)))
            return room.as_strided((T, heads, D), (t, h, 1), r.randint(0, 250))

        q, k, v, out = view(3), view(2), view(2), view(3)
        if r.random() < 0.3:
            out = q
        # mostly behind the views, sometimes among them
        kc, vc = (room.data_ptr() + 2 * r.choice((r.randint(0, 300), r.randint(700, 2500))) for _ in range(2))
        n = 2 * r.randint(8, 200)

        def of(t):
            return {t.data_ptr() + 2 * (i * t.stride(0) + j * t.stride(1) + d) + b for i in range(T)
                    for j in range(t.shape[1]) for d in range(D) for b in range(2)}

        caches = [set(range(c, c + n)) for c in (kc, vc)]
        bad = bool(caches[0] & caches[1]) or any(of(t) & c for t in (q, k, v, out) for c in caches) or \
            bool(of(out) & (of(k) | of(v)))
        at = lambda t: (t, t.data_ptr(), t.stride(0), t.stride(1), t.shape[1])  # noqa: E731
        try:
            B200Rotary._check_apart(NS(head_dim=D), (at(q), at(k), at(v)), at(out), T, 2, kc, vc, n)
            refused = False
        except RuntimeError:
            refused = True
        assert refused == bad
        seen[bad] += 1
    assert min(seen.values()) > 300, seen


def test_tree_masks():
    got = tree_masks([[-1, 0, 0, -1, 2], [-1]])
    assert got.tolist() == [0b1, 0b11, 0b101, 0b1000, 0b10101, 0b1]
    long = tree_masks([list(range(-1, 63))])
    assert long[-1].item() == -1 and long[62].item() == (1 << 63) - 1
    for bad in ([[0]], [[-1, 1]], [[-2]], [[-1] * 65]):
        with pytest.raises(ValueError):
            tree_masks(bad)


# ------------------------------------------------------------------ the oracle
def test_oracle_is_plain_attention():
    g = torch.Generator().manual_seed(0)
    q, K, V = (torch.randn(*s, generator=g).bfloat16() for s in ((6, 4, 64), (20, 2, 64), (20, 2, 64)))
    got, tol = O.attend(q, K, V, O.visible(6, 20), 0.125)
    up = lambda x: x.double().repeat_interleave(2, 1).transpose(0, 1)  # noqa: E731
    want = torch.nn.functional.scaled_dot_product_attention(
        q.double().transpose(0, 1), up(K), up(V), attn_mask=O.visible(6, 20), scale=0.125).transpose(0, 1)
    assert torch.allclose(got, want, atol=1e-12) and (tol > 0).all() and tol.max() < 0.05
    # a chain of drafted tokens is the causal mask
    assert torch.equal(O.visible(6, 20, tree=tree_masks([list(range(-1, 5))])), O.visible(6, 20))
    # rows without keys are zeros
    none, _ = O.attend(q, K, V, torch.zeros(6, 20, dtype=torch.bool), 0.125)
    assert (none == 0).all()


def test_oracle_rotary_turns_pairs():
    x = torch.randn(3, 2, 8, dtype=torch.float32)
    inv, pos = torch.tensor([0.5, 0.25]), torch.tensor([0, 1, 7], dtype=torch.int32)
    for layout, (a, b) in (("half", (1, 3)), ("interleaved", (2, 3))):
        y, _ = O.rotate(x, pos, inv, 2.0, 4, layout)
        z = torch.complex(x[..., a].double(), x[..., b].double()) * torch.polar(
            torch.full((3, 1), 2.0, dtype=torch.float64), pos.double()[:, None] * 0.25)
        assert torch.allclose(y[..., a], z.real) and torch.allclose(y[..., b], z.imag)
        assert torch.equal(y[..., 4:], x[..., 4:].double())


def test_install_routes_prefill_over_the_paged_cache():
    """Prefill with block tables stores and appends; every other call keeps the module's forward."""
    from types import SimpleNamespace as NS

    from nanovllm_dots_b200.llm_append import install_append_attention
    calls = []
    module = NS(num_heads=4, num_kv_heads=2, head_dim=64, is_causal=True, k_cache=torch.zeros(2, 16, 2, 64),
                v_cache=torch.zeros(2, 16, 2, 64), forward=lambda q, k, v: calls.append("own") or "own")
    att = NS(append=lambda *a: calls.append(a) or "append")
    ctx = NS(is_prefill=True, block_tables=torch.zeros(2, 1, dtype=torch.int32),
             cu_seqlens_q=torch.tensor([0, 3, 5], dtype=torch.int32),
             cu_seqlens_k=torch.tensor([0, 10, 12], dtype=torch.int32), slot_mapping=torch.arange(5))
    stored = []
    install_append_attention(module, lambda: ctx, att, lambda *a: stored.append(a))
    q, k = torch.zeros(5, 4 * 64), torch.ones(5, 2 * 64)
    assert module.forward(q, k, k) == "append"
    a = calls.pop()
    assert a[0].shape == (5, 4, 64) and a[1] is module.k_cache and a[2] is module.v_cache
    assert a[3] is ctx.cu_seqlens_q and a[4].tolist() == [10, 2] and a[4].dtype == torch.int32
    assert a[5] is ctx.block_tables
    assert stored[0][0].shape == (5, 2, 64) and stored[0][4] is ctx.slot_mapping
    for change in (dict(is_prefill=False), dict(block_tables=None)):
        kept = dict(vars(ctx))
        vars(ctx).update(change)
        assert module.forward(q, k, k) == "own"
        vars(ctx).update(kept)
    module.is_causal = False
    assert module.forward(q, k, k) == "own" and len(stored) == 1

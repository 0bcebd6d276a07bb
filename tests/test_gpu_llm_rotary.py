"""Rotary positions with the cache store (``dllm_rotary`` through ``B200Rotary``)
against a float64 oracle; the bound of every element is derived in
``llm_append_oracle.rotate`` (fp32 products and sums, one rounding)."""
from __future__ import annotations

import pytest
import torch

from nanovllm_dots_b200.llm_rotary import B200Rotary, RotaryScaling, rotary_frequencies
from oracle import llm_append_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def positions(T, seed=0):
    """Positions over the whole int32 range, the ends among them."""
    g = torch.Generator().manual_seed(seed)
    p = (2.0 ** (torch.rand(T, generator=g, dtype=torch.float64) * 31)).long() - 1
    p[0] = 0
    if T > 2:
        p[1], p[2] = 2 ** 31 - 1, 1
    return p.to(torch.int32)


def data(T, H, D, dtype, seed=0):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


def close(got, ref, tol):
    over = (got.double().cpu() - ref).abs() - tol
    assert over.max() <= 0, f"{int((over > 0).sum())} of {over.numel()} are off, by up to {over.max():.3g}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 128, 128), (5, 12, 128, 64), (64, 3, 64, 64), (7, 2, 64, 16),
                                       (3, 2, 80, 20), (2, 1, 6, 2), (9000, 12, 128, 128), (4001, 16, 64, 32)])
def test_rotate(T, H, D, rot, layout, dtype):
    x, pos = data(T, H, D, dtype), positions(T)
    inv, f = rotary_frequencies(rot, 10000.0)
    ref, tol = O.rotate(x, pos, inv, f, rot, layout)
    r = B200Rotary(D, rot_dim=rot, layout=layout, device=DEV)
    xd, pd = x.to(DEV), pos.to(DEV)
    got = r.rotate(xd, pd)
    close(got, ref, tol)
    assert torch.equal(xd.cpu(), x)
    assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
    assert r.rotate(xd, pd, out=xd) is xd and torch.equal(xd, got)     # in place


@pytest.mark.parametrize("scaling", [RotaryScaling("linear", 4.0), RotaryScaling("ntk", 8.0),
                                     RotaryScaling("bands", 8.0, 8192), RotaryScaling("yarn", 16.0, 4096),
                                     RotaryScaling("yarn", 2.0, 32768, attention_factor=0.5)])
def test_scaled_frequencies(scaling):
    x, pos = data(300, 4, 128, torch.float32), torch.arange(100000, 100300, dtype=torch.int32)
    inv, f = rotary_frequencies(128, 1e6, scaling)
    ref, tol = O.rotate(x, pos, inv, f, 128, "half")
    got = B200Rotary(128, theta=1e6, scaling=scaling, device=DEV).rotate(x.to(DEV), pos.to(DEV))
    close(got, ref, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,KVH,D,rot,bs", [(1, 12, 2, 128, 128, 256), (64, 12, 2, 128, 128, 256),
                                              (333, 8, 8, 64, 32, 16), (5000, 12, 2, 128, 64, 256),
                                              (17, 3, 1, 20, 10, 48)])
def test_rotate_and_store(T, H, KVH, D, rot, bs, dtype):
    """q, k, v as slices of the packed projection; -1 slots store nothing; other slots stay."""
    packed = data(T, H + 2 * KVH, D, dtype)
    pos, blocks = positions(T, 1), -(-T // bs) + 2
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(2))[:T].to(torch.int32)
    slots[T // 2] = -1 if T > 1 else slots[0]
    K0, V0 = data(blocks * bs, KVH, D, dtype, 5), data(blocks * bs, KVH, D, dtype, 6)
    inv, f = rotary_frequencies(rot, 5e4)
    r = B200Rotary(D, theta=5e4, rot_dim=rot, device=DEV)
    p = packed.to(DEV)
    K, V = (c.view(blocks, bs, KVH, D).to(DEV) for c in (K0, V0))
    q = r.rotate_store(p[:, :H], p[:, H:H + KVH], p[:, H + KVH:], pos.to(DEV), slots.to(DEV), K, V)
    r.check_errors()
    close(q, *O.rotate(packed[:, :H], pos, inv, f, rot, "half"))
    kr, kt = O.rotate(packed[:, H:H + KVH], pos, inv, f, rot, "half")
    live = slots >= 0
    at = slots[live].long()
    close(K.view(-1, KVH, D)[at.to(DEV)], kr[live], kt[live])
    assert torch.equal(V.view(-1, KVH, D).cpu()[at], packed[live, H + KVH:])
    rest = torch.ones(blocks * bs, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(K.view(-1, KVH, D).cpu()[rest], K0[rest])
    assert torch.equal(V.view(-1, KVH, D).cpu()[rest], V0[rest])


def test_odd_strides_and_alignment():
    """Rows that are not 16-byte aligned take the element-wise kernel: same values."""
    T, H, D = 50, 3, 64
    x, pos = data(T, H, D, torch.bfloat16), positions(T)
    r = B200Rotary(D, device=DEV)
    want = r.rotate(x.to(DEV), pos.to(DEV))
    base = torch.zeros(T, H, D + 3, dtype=torch.bfloat16, device=DEV)
    base[..., 1:D + 1] = x.to(DEV)
    odd = base[..., 1:D + 1]
    assert torch.equal(r.rotate(odd, pos.to(DEV)), want)
    flipped = x.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(H, T, D, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    assert torch.equal(r.rotate(flipped, pos.to(DEV), out=out), want)
    shared = x[:, :1].to(DEV).expand(T, H, D)        # one head read for all
    assert torch.equal(r.rotate(shared, pos.to(DEV)), want[:, :1].expand(T, H, D))


def test_slot_past_the_cache_is_reported():
    r = B200Rotary(128, device=DEV)
    qkv = data(4, 4, 128, torch.bfloat16).to(DEV)
    K = torch.zeros(2, 16, 1, 128, dtype=torch.bfloat16, device=DEV)
    V = torch.zeros_like(K)
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    slots = torch.tensor([0, 32, 5, 31], dtype=torch.int32, device=DEV)
    r.rotate_store(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], pos, slots, K, V)
    with pytest.raises(RuntimeError, match="page"):
        r.check_errors()
    r.check_errors()
    assert int((V.view(32, -1) != 0).any(1).sum()) == 3


def test_no_tokens_graph_and_stream():
    r = B200Rotary(64, device=DEV)
    x, pos = data(40, 2, 64, torch.float16).to(DEV), positions(40).to(DEV)
    assert r.rotate(x[:0], pos[:0]).shape == (0, 2, 64)
    want = r.rotate(x, pos)
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r.rotate(x, pos, out=out)
    out.zero_()
    g.replay()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = r.rotate(x, pos, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(other, want)


@pytest.mark.parametrize("how", ["stream argument", "current stream", "replayed graph"])
def test_errors_on_other_streams_are_reported(how):
    """A slot past the cache met on a stream that is still busy when the error is asked for."""
    r = B200Rotary(128, device=DEV)
    qkv = data(4, 4, 128, torch.bfloat16).to(DEV)
    K = torch.zeros(2, 16, 1, 128, dtype=torch.bfloat16, device=DEV)
    V = torch.zeros_like(K)
    pos, slots = torch.arange(4, dtype=torch.int32, device=DEV), torch.tensor([0, 32, 5, 31], dtype=torch.int32, device=DEV)
    args = (qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], pos, slots, K, V)
    out = torch.empty(4, 2, 128, dtype=torch.bfloat16, device=DEV)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    if how == "replayed graph":
        with torch.cuda.graph(g):
            r.rotate_store(*args, out=out)
    for _ in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(100_000_000)
            if how == "replayed graph":
                g.replay()
            elif how == "current stream":
                r.rotate_store(*args, out=out)
        if how == "stream argument":
            r.rotate_store(*args, out=out, stream=s)
        with pytest.raises(RuntimeError, match="page"):
            r.check_errors()
        r.check_errors()


def test_store_refuses_memory_that_its_outputs_share():
    """out over k, v or a cache, caches over each other or over what is read; slices of one
    packed projection, out=q among them, are apart."""
    T, D = 40, 64
    r = B200Rotary(D, device=DEV)
    packed = data(T, 16, D, torch.bfloat16).to(DEV)
    pos, slots = positions(T).to(DEV), torch.arange(T, dtype=torch.int32, device=DEV)
    pool = torch.zeros(6, 48, 2, D, dtype=torch.bfloat16, device=DEV)
    K, V, more = pool[:2], pool[2:4], pool[4:]
    q, k, v = packed[:, :12], packed[:, 12:14], packed[:, 14:]

    def call(q=q, k=k, v=v, K=K, V=V, out=None):
        return r.rotate_store(q, k, v, pos, slots, K, V, out=out)

    want = call().clone()
    kept = K.clone(), V.clone()
    rows = more.view(-1, 2, D)[:T]
    for bad in (dict(out=packed[:, 1:13]), dict(out=packed[:, 2:14]), dict(out=packed[:, 4:16]),
                dict(V=K), dict(V=pool[1:3]), dict(k=K.view(-1, 2, D)[:T]), dict(v=V.view(-1, 2, D)[:T]),
                dict(q=V.view(-1, 2, D)[:T]), dict(q=rows, out=K.view(-1, 2, D)[:T]),
                dict(q=rows, out=pool.view(-1, 2, D)[90:90 + T])):
        with pytest.raises(RuntimeError, match="overlap|share no memory"):
            call(**bad)
    torch.cuda.synchronize()
    assert torch.equal(K, kept[0]) and torch.equal(V, kept[1])
    K.zero_(), V.zero_()
    assert torch.equal(call(out=torch.empty_like(want)), want)
    assert call(out=q) is q and torch.equal(q, want)          # in place, next to k and v
    assert torch.equal(K, kept[0]) and torch.equal(V, kept[1])
    mixed = packed[:, :12].view(T, 2, 6, D)                    # heads of q, k and v interleaved
    qi, ki, vi = (mixed[:, :, i] for i in range(3))
    got = call(q=qi, k=ki, v=vi)
    again = call(q=qi.clone(), k=ki.clone(), v=vi.clone())
    assert torch.equal(got, again)
    assert torch.equal(call(q=qi, k=ki, v=vi, out=qi), again)
    r.check_errors()


def test_usual_layouts_are_told_apart_by_their_strides(monkeypatch):
    """In place in a packed row, in one whose heads are interleaved, and in a buffer with
    the heads in front: no row by row search."""
    from nanovllm_dots_b200 import llm_rotary

    def search(*_):
        raise AssertionError("searched row by row")

    monkeypatch.setattr(llm_rotary, "shared", search)
    monkeypatch.setattr(llm_rotary, "meets", search)
    T, D = 300, 64
    r = B200Rotary(D, device=DEV)
    pos, slots = positions(T).to(DEV), torch.arange(T, dtype=torch.int32, device=DEV)
    x = data(T, 12, D, torch.bfloat16).to(DEV)
    K = torch.zeros(2, 160, 4, D, dtype=torch.bfloat16, device=DEV)
    V = torch.zeros_like(K)
    want = r.rotate_store(x[:, :4], x[:, 4:8], x[:, 8:], pos, slots, K, V)
    kept = K.clone()
    for layout in ("packed", "interleaved", "heads in front"):
        buffer = torch.empty(12 * T * D, dtype=torch.bfloat16, device=DEV)
        if layout == "packed":
            q, k, v = buffer.view(T, 12, D).split(4, dim=1)
        elif layout == "interleaved":
            q, k, v = buffer.view(T, 4, 3, D).unbind(2)
        else:
            q, k, v = buffer.view(12, T, D).transpose(0, 1).split(4, dim=1)
        for to, at in ((q, 0), (k, 4), (v, 8)):
            to.copy_(x[:, at:at + 4])
        K.zero_()
        assert r.rotate_store(q, k, v, pos, slots, K, V, out=q) is q
        assert torch.equal(q, want) and torch.equal(K, kept)

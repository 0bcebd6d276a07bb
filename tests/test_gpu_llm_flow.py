"""Rotary, append, decode and verify together over one paged cache, as a serving
loop uses them: two prompts are prefilled in chunks, one token is decoded, a tree
of drafted tokens is verified, its accepted path is kept and the next token
follows.  At every step the rotated queries and the whole cache are checked
against the unrotated projections, and the attention against float64 attention
over the sequence so far."""
from __future__ import annotations

import pytest
import torch

from nanovllm_dots_b200.llm_append import B200AppendAttention, tree_masks
from nanovllm_dots_b200.llm_attention import B200DecodeAttention
from nanovllm_dots_b200.llm_rotary import B200Rotary, rotary_frequencies
from oracle import llm_append_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
H, KVH, D, BS, THETA = 12, 2, 128, 256, 1e6
BF = torch.bfloat16


class Loop:
    def __init__(self):
        self.g = torch.Generator().manual_seed(7)
        self.rotary = B200Rotary(D, theta=THETA, device=DEV)
        self.append = B200AppendAttention(H, D, D ** -0.5, KVH, max_tokens=600, max_seqs=2, max_blocks=4,
                                          block_size=BS, device=DEV)
        self.decode = B200DecodeAttention(H, D, D ** -0.5, KVH, max_batch=2, max_blocks=4, block_size=BS,
                                          device=DEV)
        self.table = torch.tensor([[5, 1, 7, 2], [0, 6, 3, 4]], dtype=torch.int32)
        self.K = torch.full((8, BS, KVH, D), float("nan"), dtype=BF, device=DEV)
        self.V = self.K.clone()
        self.kept = [[], []]         # what the cache holds: per sequence [(k unrotated, v, position)]

    def project(self, counts):
        """Packed projections of new tokens and, per sequence, their rows."""
        return torch.randn(sum(counts), (H + 2 * KVH), D, generator=self.g).to(BF)

    def slots(self, seq, first, n):
        p = torch.arange(first, first + n)
        return self.table[seq, p // BS].long() * BS + p % BS

    def place(self, packed, counts, positions):
        """Rotates and stores new tokens behind each sequence's cached ones."""
        slots = torch.cat([self.slots(i, len(self.kept[i]), m) for i, m in enumerate(counts)]).to(torch.int32)
        p = packed.to(DEV)
        q = self.rotary.rotate_store(p[:, :H], p[:, H:H + KVH], p[:, H + KVH:],
                                     torch.tensor(positions, dtype=torch.int32, device=DEV), slots.to(DEV),
                                     self.K, self.V)
        at = 0
        for i, m in enumerate(counts):
            self.kept[i] += [(packed[at + j, H:H + KVH], packed[at + j, H + KVH:], positions[at + j])
                             for j in range(m)]
            at += m
        return q, slots.to(DEV)

    def lens(self, counts):
        d = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        return d([0, counts[0], sum(counts)]), d([len(k) for k in self.kept]), self.table.to(DEV)

    def check(self, got, q, packed, counts, positions, see):
        """q and the cache against the rotary's bound, got against attention in
        float64 of what q and the cache then hold."""
        inv, _ = rotary_frequencies(D, THETA)
        q, at = q.cpu(), 0
        for i, m in enumerate(counts):
            ref, tol = O.rotate(packed[at:at + m, :H], torch.tensor(positions[at:at + m]), inv, 1.0, D, "half")
            assert ((q[at:at + m].double() - ref).abs() <= tol).all()
            K, V = (O.gather(c.cpu(), self.table[i], len(self.kept[i])) for c in (self.K, self.V))
            k = torch.stack([x[0] for x in self.kept[i]])
            ref, tol = O.rotate(k, torch.tensor([x[2] for x in self.kept[i]]), inv, 1.0, D, "half")
            assert ((K.double() - ref).abs() <= tol).all()
            assert torch.equal(V, torch.stack([x[1] for x in self.kept[i]]))
            ref, tol = O.attend(q[at:at + m], K, V, see[i], D ** -0.5)
            off = (got[at:at + m].double().cpu() - ref).abs() - tol
            assert off.max() <= 0, f"sequence {i}: off by {off.max():.3g} over its bound"
            at += m


def test_serving_loop():
    s = Loop()
    # prompts in two chunks each
    for counts in ([300, 40], [77, 200]):
        packed = s.project(counts)
        first = [len(k) for k in s.kept]
        pos = [first[i] + j for i, m in enumerate(counts) for j in range(m)]
        q, _ = s.place(packed, counts, pos)
        got = s.append.append(q, s.K, s.V, *s.lens(counts))
        s.check(got, q, packed, counts, pos, [O.visible(m, len(s.kept[i])) for i, m in enumerate(counts)])
    # one decoded token each: append and the decode attention agree
    counts = [1, 1]
    packed = s.project(counts)
    pos = [len(k) for k in s.kept]
    q, slots = s.place(packed, counts, pos)
    cu, ctx, table = s.lens(counts)
    got = s.append.append(q, s.K, s.V, cu, ctx, table)
    see = [O.visible(1, len(k)) for k in s.kept]
    s.check(got, q, packed, counts, pos, see)
    s.check(s.decode.decode(q, None, None, s.K, s.V, None, ctx, table), q, packed, counts, pos, see)
    # trees of drafted tokens: positions by depth, keys in the order of the draft
    parents = [[-1, 0, 0, 1, 1, 2, 3], [-1, -1, 0, 1]]
    counts = [len(p) for p in parents]
    base = [len(k) for k in s.kept]
    pos = []
    for i, up in enumerate(parents):
        depth = []
        for t in up:
            depth.append(0 if t < 0 else depth[t] + 1)
        pos += [base[i] + d for d in depth]
    packed = s.project(counts)
    q, _ = s.place(packed, counts, pos)
    masks = tree_masks(parents)
    got = s.append.verify(q, s.K, s.V, *s.lens(counts), masks.to(DEV))
    s.check(got, q, packed, counts, pos, [O.visible(m, len(s.kept[i]), tree=masks[sum(counts[:i]):][:m])
                                       for i, m in enumerate(counts)])
    # the accepted paths move to the front, the rest is forgotten
    for i, path in enumerate(([0, 2, 5], [1])):
        src, dst = s.slots(i, base[i], counts[i])[path].to(DEV), s.slots(i, base[i], len(path)).to(DEV)
        for c in (s.K, s.V):
            flat = c.view(-1, KVH, D)
            flat[dst] = flat[src]
        s.kept[i] = s.kept[i][:base[i]] + [s.kept[i][base[i] + t] for t in path]
    # and the next token sees them
    counts = [1, 1]
    packed = s.project(counts)
    pos = [len(k) for k in s.kept]
    q, _ = s.place(packed, counts, pos)
    got = s.append.append(q, s.K, s.V, *s.lens(counts))
    s.check(got, q, packed, counts, pos, [O.visible(1, len(k)) for k in s.kept])
    s.append.check_errors()
    s.rotary.check_errors()
    s.decode.check_errors()


@pytest.mark.parametrize("decode_first", [True, False])
def test_installed_module_over_a_packed_projection(decode_first):
    """The two hooks on a module of the engine's shape: its forward gets the projection's slices
    ([tokens, heads * D], the values still inside the packed row), prefills two chunks of
    two prompts over the paged cache and decodes one token each.  Calls outside the
    hooks' conditions reach the module's own forward."""
    from types import SimpleNamespace as NS

    from nanovllm_dots_b200.llm_append import install_append_attention
    from nanovllm_dots_b200.llm_attention import install_decode_attention

    s, own = Loop(), []
    module = NS(num_heads=H, num_kv_heads=KVH, head_dim=D, is_causal=True, k_cache=s.K, v_cache=s.V,
                forward=lambda q, k, v: own.append(q.shape))
    ctx = NS()

    def store(k, v, k_cache, v_cache, slots):
        k_cache.view(-1, KVH, D)[slots.long()] = k
        v_cache.view(-1, KVH, D)[slots.long()] = v

    hooks = [lambda: install_decode_attention(module, lambda: ctx, s.decode),
             lambda: install_append_attention(module, lambda: ctx, s.append, store)]
    for hook in hooks if decode_first else hooks[::-1]:
        hook()

    def forward(counts, prefill):
        packed = s.project(counts)
        base = [len(k) for k in s.kept]
        pos = [base[i] + j for i, m in enumerate(counts) for j in range(m)]
        d = packed.to(DEV).view(sum(counts), -1)
        q, k, v = d.split([H * D, KVH * D, KVH * D], dim=1)
        at = torch.tensor(pos, dtype=torch.int32, device=DEV)
        q, k = (s.rotary.rotate(x.view(x.shape[0], -1, D), at).flatten(1) for x in (q, k))
        ctx.slot_mapping = torch.cat([s.slots(i, base[i], m) for i, m in enumerate(counts)]).to(torch.int32).to(DEV)
        i = 0
        for n, m in enumerate(counts):
            s.kept[n] += [(packed[i + j, H:H + KVH], packed[i + j, H + KVH:], pos[i + j]) for j in range(m)]
            i += m
        ctx.is_prefill = prefill
        ctx.cu_seqlens_q, ctx.context_lens, ctx.block_tables = s.lens(counts)
        ctx.cu_seqlens_k = torch.nn.functional.pad(ctx.context_lens.cumsum(0, dtype=torch.int32), (1, 0))
        got = module.forward(q, k if prefill else k.contiguous(), v if prefill else v.contiguous())
        s.check(got, q.view(-1, H, D), packed, counts, pos,
                [O.visible(m, len(s.kept[i])) for i, m in enumerate(counts)])

    for counts, prefill in (([300, 40], True), ([77, 200], True), ([1, 1], False), ([3, 1], True)):
        forward(counts, prefill)
    s.append.check_errors()
    s.decode.check_errors()
    assert not own
    ctx.is_prefill, ctx.block_tables = True, None
    q = torch.zeros(5, H * D, dtype=BF, device=DEV)
    module.forward(q, q[:, :KVH * D], q[:, :KVH * D])
    assert own == [q.shape]

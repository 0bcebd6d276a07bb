"""Append attention and tree verification (``dllm_append_attention`` through
``B200AppendAttention``) against a float64 oracle.

The bound of every output element is derived in ``llm_append_oracle.attend``:
one rounding of each probability to the cache's 16-bit type (half a step, in the
mean of |v|), one of the result, and the fp32 errors of scores, cap, bias and
exponential.  Every cache row that no token sees holds NaN."""
from __future__ import annotations

import random

import pytest
import torch

from nanovllm_dots_b200.llm_append import B200AppendAttention, tree_masks
from oracle import llm_append_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF, FP = torch.bfloat16, torch.float16


class Case:
    """n sequences of (new tokens, positions before them) over a shuffled paged cache."""

    def __init__(self, lens, H=12, KVH=2, D=128, bs=256, dtype=BF, seed=0, spread=1.5, **opts):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.KVH, self.D, self.bs, self.dtype = lens, H, KVH, D, bs, dtype
        self.causal = opts.pop("causal", True)
        self.window, self.softcap = opts.pop("window", 0), opts.pop("softcap", 0.0)
        self.slopes, self.prefix = opts.pop("slopes", None), opts.pop("prefix", None)
        self.first, self.tree = opts.pop("first", None), opts.pop("tree", None)
        assert not opts
        self.cu = torch.tensor([0] + [m for m, _ in lens], dtype=torch.int32).cumsum(0).to(torch.int32)
        self.ctx = torch.tensor([m + p for m, p in lens], dtype=torch.int32)
        need = [-(-int(c) // bs) for c in self.ctx]
        blocks = sum(need) + 3
        perm = torch.randperm(blocks, generator=g).tolist()
        self.table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
        at = 0
        for i, b in enumerate(need):
            self.table[i, :b] = torch.tensor(perm[at:at + b], dtype=torch.int32)
            at += b
        T = int(self.cu[-1])
        self.q = (torch.randn(T, H, D, generator=g) * spread).to(dtype)
        self.K = torch.full((blocks, bs, KVH, D), float("nan"), dtype=dtype)
        self.V = self.K.clone()
        self.see = []
        for i, (m, p) in enumerate(lens):
            a = int(self.cu[i])
            see = O.visible(m, m + p, self.causal, self.window, self.prefix[i] if self.prefix else 0,
                            None if self.first is None else self.first[a:a + m],
                            None if self.tree is None else self.tree[a:a + m])
            self.see.append(see)
            k = torch.arange(m + p)
            live = see.any(0) if m else torch.zeros(m + p, dtype=torch.bool)
            blk, row = self.table[i, k // bs].long(), k % bs
            self.K[blk[live], row[live]] = torch.randn(int(live.sum()), KVH, D, generator=g).to(dtype)
            self.V[blk[live], row[live]] = torch.randn(int(live.sum()), KVH, D, generator=g).to(dtype)

    def attention(self, **over):
        kw = dict(max_tokens=max(1, self.q.shape[0]), max_seqs=len(self.lens),
                  max_blocks=self.table.shape[1], block_size=self.bs, dtype=self.dtype,
                  causal=self.causal, window=self.window, softcap=self.softcap, slopes=self.slopes,
                  device=DEV)
        kw.update(over)
        return B200AppendAttention(self.H, self.D, self.D ** -0.5, self.KVH, **kw)

    def device(self):
        d = lambda t: t.to(DEV)  # noqa: E731
        self.qd, self.Kd, self.Vd = d(self.q), d(self.K), d(self.V)
        self.cud, self.ctxd, self.tabled = d(self.cu), d(self.ctx), d(self.table)
        self.prefixd = None if self.prefix is None else torch.tensor(self.prefix, dtype=torch.int32, device=DEV)
        self.firstd = None if self.first is None else d(self.first)
        self.treed = None if self.tree is None else d(self.tree)
        return self

    def call(self, att, **kw):
        if self.tree is not None:
            return att.verify(self.qd, self.Kd, self.Vd, self.cud, self.ctxd, self.tabled, self.treed, **kw)
        return att.append(self.qd, self.Kd, self.Vd, self.cud, self.ctxd, self.tabled,
                          prefix_lens=self.prefixd, first_keys=self.firstd, **kw)

    def reference(self):
        outs, tols = [], []
        for i, (m, p) in enumerate(self.lens):
            a = int(self.cu[i])
            K, V = (O.gather(c, self.table[i], m + p) for c in (self.K, self.V))
            o, t = O.attend(self.q[a:a + m], K, V, self.see[i], self.D ** -0.5, self.softcap, self.slopes)
            outs.append(o)
            tols.append(t)
        return torch.cat(outs), torch.cat(tols)


def check(got, ref, tol):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{(~torch.isfinite(got)).sum()} values are not finite"
    over = ((got - ref).abs() - tol).flatten()
    worst = int(over.argmax())
    assert over[worst] <= 0, (f"element {worst} of {over.numel()}: {got.flatten()[worst]:.6g}, expected "
                              f"{ref.flatten()[worst]:.6g} within {tol.flatten()[worst]:.3g}; "
                              f"{int((over > 0).sum())} are off")


def run(case):
    att = case.attention()
    got = case.device().call(att)
    att.check_errors()
    check(got, *case.reference())
    return got


def slopes_of(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])


RAGGED = [(1, 0), (1, 127), (1, 128), (5, 0), (22, 300), (43, 85), (130, 1), (300, 513)]


def test_one_token_alone():
    run(Case([(1, 0)]))


def test_one_token_over_history():
    run(Case([(1, 300)]))


def test_one_row_tile_two_key_tiles():
    run(Case([(21, 200)]))


def test_two_row_tiles():
    run(Case([(42, 200)]))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("H,KVH,D,bs", [(12, 2, 128, 256), (16, 16, 64, 16), (8, 1, 64, 48),
                                        (14, 2, 128, 64), (3, 1, 128, 16), (32, 2, 64, 256),
                                        (128, 1, 64, 32)])
def test_ragged_causal(H, KVH, D, bs, dtype):
    run(Case(RAGGED, H, KVH, D, bs, dtype))


@pytest.mark.parametrize("opts", [
    dict(window=1), dict(window=7), dict(window=300), dict(causal=False),
    dict(causal=False, window=40), dict(prefix=[0, 128, 50, 3, 322, 100, 131, 700]),
    dict(prefix=[0, 128, 50, 3, 322, 100, 131, 700], window=90)])
def test_masks(opts):
    run(Case(RAGGED, dtype=FP, **opts))


def documents(lens, seed):
    r = random.Random(seed)
    first = []
    for m, p in lens:
        cuts = sorted({0, *(r.randrange(m + p) for _ in range(3))})
        first += [max(c for c in cuts if c <= p + j) for j in range(m)]
    return torch.tensor(first, dtype=torch.int32)


@pytest.mark.parametrize("opts", [dict(), dict(window=64), dict(softcap=20.0)])
def test_documents(opts):
    run(Case(RAGGED, 16, 16, 64, 16, first=documents(RAGGED, 3), **opts))


@pytest.mark.parametrize("n", [40, 200, 300])
def test_documents_of_many_sequences(n):
    """Units planned by the CTAs themselves, and by the kernel in front of them: more
    units, and more sequences (some of them empty)."""
    r = random.Random(n)
    lens = [(r.choice((0, 1, 9, 33, 65)), r.randrange(1, 300)) for _ in range(n)]
    run(Case(lens, 8, 1, 64, 64, first=documents(lens, n), slopes=slopes_of(8)))


def test_rows_that_see_nothing_are_zero():
    """Every third token's document begins behind it; one sequence is all such tokens."""
    lens = [(70, 100), (3, 40), (64, 0)]
    first, at = torch.zeros(137, dtype=torch.int32), 0
    for i, (m, p) in enumerate(lens):
        for j in range(m):
            first[at + j] = p + j + 1 if i == 1 or j % 3 == 0 else 0
        at += m
    got = run(Case(lens, first=first)).cpu()
    assert (got[0] == 0).all() and (got[70:73] == 0).all() and (got[1] != 0).any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("opts", ["cap", "slopes", "both", "both prefix"])
def test_caps_and_distance_bias(opts, D):
    kw = {}
    if "cap" in opts or "both" in opts:
        kw["softcap"] = 4.0
    if "slopes" in opts or "both" in opts:
        kw["slopes"] = slopes_of(12)
    if "prefix" in opts:
        kw["prefix"] = [0, 128, 50, 3, 322, 100, 131, 700]
    run(Case(RAGGED, D=D, spread=4.0, **kw))


def test_peaked_scores_move_the_maximum():
    """Scores that grow by hundreds from the newest key to the oldest."""
    c = Case([(30, 700), (1, 900)], spread=8.0, dtype=FP)
    for i, (m, p) in enumerate(c.lens):
        k = torch.arange(m + p)
        c.K[c.table[i, k // c.bs].long(), k % c.bs] *= torch.linspace(4.0, 0.1, m + p)[:, None, None].half()
    run(c)


@pytest.mark.parametrize("lens", [[(3, 70000)], [(1, 40000), (64, 33333), (1, 0)], [(200, 20000)]])
def test_long_history_is_split(lens):
    run(Case(lens, 4, 1, 64, 256))


def test_many_sequences():
    r = random.Random(5)
    run(Case([(r.randint(0, 3), r.randint(1, 200)) for _ in range(1500)], 2, 1, 64, 16))


def trees(lens, seed):
    r = random.Random(seed)
    return tree_masks([[r.randint(max(-1, t - 5), t - 1) for t in range(m)] for m, _ in lens])


TREES = [(1, 0), (8, 300), (64, 0), (64, 1000), (17, 111), (33, 128), (5, 123), (64, 65)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("H,KVH,D,bs", [(12, 2, 128, 256), (16, 4, 64, 16), (2, 2, 128, 48)])
def test_trees(H, KVH, D, bs, dtype):
    run(Case(TREES, H, KVH, D, bs, dtype, tree=trees(TREES, 1)))


def test_tree_with_cap_and_with_empty_masks():
    t = trees(TREES, 2)
    t[0] = 0                     # sees nothing at all
    t[9] = 0                     # sees the history of 300
    run(Case(TREES, softcap=5.0, tree=t))


def test_chain_tree_is_causal():
    """A tree without branches gives what the causal mask gives, bit for bit."""
    lens = [(20, 333), (1, 7)]
    a = Case(lens)
    b = Case(lens, tree=tree_masks([list(range(-1, m - 1)) for m, _ in lens]))
    assert torch.equal(run(a), run(b))


@pytest.mark.parametrize("special", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["K", "V"])
def test_special_values_reach_only_rows_that_see_them(where, special):
    """A drafted branch with a NaN or an infinity does not reach the other
    branches, a document's does not reach the next document."""

    def spoilt(c, token):        # [heads]: a score of -inf (an infinite key, a negative q) only has no weight
        return (c.q[token, :, 5] > 0) if where == "K" and special > 0 else torch.ones(12, dtype=torch.bool)

    masks = tree_masks([[-1, 0, -1, 2, 3, 1]])
    c = Case([(6, 150)], tree=masks)
    clean = run(c)
    k = 150 + 1                  # drafted token 1: seen by tokens 1 and 5
    getattr(c, where)[int(c.table[0, k // c.bs]), k % c.bs, :, 5] = special
    got = c.device().call(c.attention())
    sees = torch.tensor([False, True, False, False, False, True])
    assert torch.equal(got[~sees], clean[~sees])
    for t in (1, 5):
        assert torch.equal(~torch.isfinite(got[t].float()).all(dim=-1).cpu(), spoilt(c, t))
    first = torch.tensor([0] * 30 + [100] * 30, dtype=torch.int32)
    c = Case([(60, 70)], first=first, bs=64)
    clean = run(c)
    getattr(c, where)[int(c.table[0, 99 // c.bs]), 99 % c.bs, :, 5] = special
    got = c.device().call(c.attention())
    sees = torch.arange(60) == 29            # position 99 itself: the document's last token
    assert torch.equal(got[~sees], clean[~sees])
    assert torch.equal(~torch.isfinite(got[29].float()).all(dim=-1).cpu(), spoilt(c, 29))


def test_pages_behind_the_window_may_be_gone():
    c = Case([(40, 1000), (1, 777)], window=100, bs=16)
    full = run(c)
    for i, (m, p) in enumerate(c.lens):
        c.table[i, :max(0, p - 99) // 16] = -1
    att = c.attention()
    got = c.device().call(att)
    att.check_errors()
    assert torch.equal(got, full)


def test_empty_sequences_and_rows_behind_the_last():
    c = Case([(0, 50), (4, 60), (0, 0), (2, 0), (0, 9)])
    run(c)
    att = c.attention(max_tokens=20)
    q = torch.cat([c.qd, torch.full((9, 12, 128), float("nan"), dtype=BF, device=DEV)])
    out = torch.full_like(q, 7.0)
    att.append(q, c.Kd, c.Vd, c.cud, c.ctxd, c.tabled, out=out)
    att.check_errors()
    check(out[:6], *c.reference())
    assert (out[6:] == 7).all()
    none = att.append(q[:0], c.Kd, c.Vd, torch.zeros_like(c.cud), c.ctxd, c.tabled)
    assert none.shape == (0, 12, 128)


def test_strided_queries():
    """q as a slice of the packed projection, and as a transposed tensor."""
    c = Case([(50, 100), (3, 3)]).device()
    att = c.attention()
    want = c.call(att)
    T = c.q.shape[0]
    packed = torch.randn(T, 16, 128, device=DEV).to(BF)
    packed[:, :12] = c.qd
    c.qd = packed[:, :12]
    assert torch.equal(c.call(att), want)
    flipped = torch.empty(12, T, 128, dtype=BF, device=DEV)
    flipped.copy_(packed[:, :12].transpose(0, 1))
    c.qd = flipped.transpose(0, 1)
    assert torch.equal(c.call(att), want)


def test_one_token_or_head_has_any_stride():
    c = Case([(1, 300)]).device()
    att = c.attention()
    want = c.call(att)
    c.qd = c.qd.as_strided((1, 12, 128), (7, 128, 1))
    assert torch.equal(c.call(att), want)
    c = Case([(9, 300)], 1, 1).device()
    att = c.attention()
    want = c.call(att)
    c.qd = c.qd.as_strided((9, 1, 128), (128, 5, 1))
    assert torch.equal(c.call(att), want)


def test_out_may_be_q_and_nothing_near_it():
    """Units of one and of several shares, narrow and wide, written over their queries."""
    c = Case([(200, 3000), (1, 5000), (64, 100), (7, 0)], 8, 2).device()
    att = c.attention()
    want, q = c.call(att), c.qd
    for _ in range(3):
        c.qd = q.clone()
        assert c.call(att, out=c.qd) is c.qd and torch.equal(c.qd, want)
    T = q.shape[0]
    room = torch.zeros(T + 1, 8, 128, dtype=BF, device=DEV)
    c.qd = room[:T]
    with pytest.raises(RuntimeError, match="overlaps"):
        c.call(att, out=room[1:])
    with pytest.raises(RuntimeError, match="32-byte"):
        c.call(att, out=room.flatten()[8:8 + T * 1024].view(T, 8, 128))
    c.qd = room[:1].expand(T, 8, 128)
    with pytest.raises(RuntimeError, match="share no memory"):
        c.call(att)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [2.0, 12.0, 60.0])
def test_cap_of_unmasked_tiles(cap, D):
    """Scores mostly past the cap, around half of it, and far below."""
    run(Case([(30, 900), (1, 1100), (70, 600)], D=D, softcap=cap, spread=2.0))


@pytest.mark.parametrize("spread", [0.0, 1.0])
def test_cap_far_below_the_scores(spread):
    """Every score is capped to nothing: the mean of V, also where the scores are zero."""
    run(Case([(30, 900), (1, 100)], softcap=1e-8, spread=spread))


@pytest.mark.parametrize("n", [3, 300])
def test_no_sequence_has_tokens(n):
    c = Case([(2, 30)] + [(0, 20)] * (n - 1)).device()
    att = c.attention()
    c.cud.zero_()
    out = torch.full_like(c.qd, 3.0)
    c.call(att, out=out)
    att.check_errors()
    assert (out == 3.0).all()


def test_bad_block_id_is_reported_and_read_as_zeros():
    c = Case([(5, 600), (3, 20)])
    c.device()
    c.tabled[0, 1] = 10_000
    att = c.attention()
    got = c.call(att)
    with pytest.raises(RuntimeError, match="page"):
        att.check_errors()
    att.check_errors()           # read and cleared
    k = torch.arange(256, 512)
    blk = c.table[0, 1].long()
    c.K[blk], c.V[blk] = 0, 0
    c.table[0, 1] = blk
    check(got, *c.reference())


def test_lengths_that_make_no_sense_are_reported():
    c = Case([(5, 60), (3, 20), (4, 9)]).device()
    att = c.attention()
    want = c.call(att)
    att.check_errors()
    c.ctxd = torch.tensor([65, 2, 100_000], dtype=torch.int32, device=DEV)   # below its tokens; past the table
    got = c.call(att)
    with pytest.raises(RuntimeError, match="len"):
        att.check_errors()
    assert torch.equal(got[:5], want[:5]) and (got[5:] == 0).all()
    c.ctxd = c.ctx.to(DEV)
    for cu in ([0, 5, 3, 12], [0, 5, 8, 4000], [-3, 5, 8, 12], [0, 12, 0, 12]):
        c.cud = torch.tensor(cu, dtype=torch.int32, device=DEV)
        c.call(att)
        with pytest.raises(RuntimeError, match="len"):
            att.check_errors()
    c.cud = c.cu.to(DEV)
    assert torch.equal(c.call(att), want)
    att.check_errors()
    t = Case([(65, 0)], tree=torch.zeros(65, dtype=torch.int64)).device()
    att = t.attention()
    assert (t.call(att) == 0).all()
    with pytest.raises(RuntimeError, match="len"):
        att.check_errors()


def test_graph_replays_follow_the_lengths():
    """One captured call serves other lengths of the same buffers; two graphs of one object take turns."""
    a, b = Case([(9, 500), (30, 41)], seed=1).device(), Case([(9, 300), (30, 200)], seed=1).device()
    wide = max(a.table.shape[1], b.table.shape[1])
    att = a.attention(max_blocks=wide)
    want = [x.call(att).clone() for x in (a, b)]
    q, cu, ctx = a.qd.clone(), a.cud.clone(), a.ctxd.clone()
    table = torch.full((2, wide), -1, dtype=torch.int32, device=DEV)
    blocks = max(a.Kd.shape[0], b.Kd.shape[0])
    K = torch.zeros(blocks, 256, 2, 128, dtype=BF, device=DEV)
    V = torch.zeros_like(K)
    out = torch.empty_like(q)
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            att.append(q, K, V, cu, ctx, table, out=out)
        graphs.append(g)
    for g, x, w in zip(graphs * 2, (a, b, b, a), (want[0], want[1], want[1], want[0])):
        q.copy_(x.qd)
        ctx.copy_(x.ctxd)
        table.fill_(-1)
        table[:, :x.table.shape[1]] = x.tabled
        K[:x.Kd.shape[0]] = x.Kd
        V[:x.Vd.shape[0]] = x.Vd
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    att.check_errors()


def test_streams_take_turns_and_results_repeat():
    c = Case([(200, 3000), (1, 5000), (64, 100)], 8, 2).device()
    att = c.attention()
    want = c.call(att)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [c.call(att, stream=s) for s in streams * 4]
    with torch.cuda.stream(streams[1]):
        outs.append(c.call(att))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_offsets_past_32_bits():
    """Blocks whose elements lie past 2^32 bytes and 2^31 elements of the cache."""
    c = Case([(7, 500), (1, 255)])
    blocks = (1 << 31) // (256 * 2 * 128) + 40
    K = torch.empty(blocks, 256, 2, 128, dtype=BF, device=DEV)
    V = torch.empty_like(K)
    want = run(c)
    shift = blocks - c.K.shape[0]
    K[shift:], V[shift:] = c.Kd, c.Vd
    c.Kd, c.Vd = K, V
    c.tabled = torch.where(c.tabled >= 0, c.tabled + shift, c.tabled)
    att = c.attention()
    assert torch.equal(c.call(att), want)
    att.check_errors()


# Bit-for-bit tests: enough sequences that a share has several key tiles of a unit, over
# which a row's maximum rises, by less and by more than what is put off.
MANY = [(9, 1900), (3, 2000), (1, 1800), (60, 1500)] * 12


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("opts", [dict(), dict(slopes=True), dict(tree=True)])
def test_a_row_depends_on_its_own_query_alone(opts, D):
    """Queries of other tokens of the sequence, and of the sequence packed behind it,
    whose rows fill up the row tile, have no say."""
    kw = dict(slopes=slopes_of(12)) if "slopes" in opts else \
        dict(tree=trees(MANY, 4)) if "tree" in opts else {}
    c = Case(MANY, D=D, **kw)
    att = c.attention()
    want, q = c.device().call(att), c.q
    r = random.Random(D)
    for by in (8.0, 0.0, 30.0, 0.01):
        rows = [t for t in range(q.shape[0]) if r.random() < 0.3]
        c.q = q.clone()
        c.q[rows] *= by
        others = torch.ones(q.shape[0], dtype=torch.bool)
        others[rows] = False
        assert torch.equal(c.device().call(att).cpu()[others], want.cpu()[others])


def test_what_the_shared_memory_held_has_no_say():
    """Six heads to a kv head are 126 rows of 128: the last two hold what was there, here
    queries of another call's, large and small."""
    c = Case([(21, 1900), (42, 1700), (20, 2100)] * 12).device()
    att = c.attention()
    want = c.call(att)
    fill = Case([(64, 1200)] * 8, 2, 2).device()
    other, q = fill.attention(), fill.qd
    for by in (60.0, 1e-3, 0.0, 8.0):
        fill.qd = q * by
        fill.call(other)
        assert torch.equal(c.call(att), want)


@pytest.mark.parametrize("ctx", [40, 1500])
@pytest.mark.parametrize("cap", [1e-3, 1.0, 1e5])
def test_caps_far_above_the_scale(ctx, cap):
    """Queries and keys of 60000 under a small scale: scores near 0.46 caps, where tanh's
    higher terms count (the cap in units of the raw product is 10^12).  Half of the keys
    have positive scores and values of 1, half negative ones and zeros."""
    scale = cap * 1e-12
    q = torch.full((3, 2, 128), 6e4, dtype=FP)
    sign = torch.where(torch.arange(ctx) % 2 == 0, 1.0, -1.0)
    K = (sign * 6e4)[:, None, None].expand(ctx, 2, 128).to(FP).contiguous()
    V = (sign > 0).to(FP)[:, None, None].expand(ctx, 2, 128).contiguous()
    att = B200AppendAttention(2, 128, scale, 2, max_tokens=3, max_seqs=1, max_blocks=1, block_size=1536,
                              dtype=FP, softcap=cap, device=DEV)
    pages = torch.zeros(2, 1, 1536, 2, 128, dtype=FP, device=DEV)
    pages[0, 0, :ctx], pages[1, 0, :ctx] = K.to(DEV), V.to(DEV)
    d = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = att.append(q.to(DEV), pages[0], pages[1], d(0, 3), d(ctx), d(0)[None])
    att.check_errors()
    check(got, *O.attend(q, K, V, O.visible(3, ctx), scale, cap))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("opts", [dict(softcap=30.0), dict(softcap=6.0), dict(softcap=1e4),
                                  dict(softcap=30.0, slopes=slopes_of(12))])
def test_a_capped_row_depends_on_its_query_and_the_keys_it_sees(opts, D):
    """Bit for bit, for caps whose scores lie below and around half of them: other tokens'
    queries, what stands in cache rows that no token sees, and the key of a drafted
    token that only it sees, choose no other token's way to compute tanh."""
    c = Case(MANY, D=D, **opts)
    att = c.attention()
    want, q, K = c.device().call(att).cpu(), c.q, c.K
    r = random.Random(D)
    for by in (8.0, 0.0, 30.0):
        rows = [t for t in range(q.shape[0]) if r.random() < 0.3]
        c.q = q.clone()
        c.q[rows] *= by
        others = torch.ones(q.shape[0], dtype=torch.bool)
        others[rows] = False
        assert torch.equal(c.device().call(att).cpu()[others], want[others])
    c.q = q
    for fill in (0.0, 1.0, 1e4, 1e38, float("inf")):
        c.K = torch.where(K.isnan(), fill, K)
        assert torch.equal(c.device().call(att).cpu(), want)
    if "slopes" in opts:
        return
    c = Case(TREES * 6, D=D, tree=trees(TREES * 6, 5), **opts)
    att = c.attention()
    want = c.device().call(att).cpu()
    others = torch.ones(c.q.shape[0], dtype=torch.bool)
    for i, (m, p) in enumerate(c.lens):      # the last drafted token is nobody's parent
        others[int(c.cu[i]) + m - 1] = False
        c.K[c.table[i, (p + m - 1) // c.bs].long(), (p + m - 1) % c.bs] *= 64
    assert torch.equal(c.device().call(att).cpu()[others], want[others])


SPECIALS = [  # sequences (new, before), their options, special rows of V (sequence, position, value)
    ("tree", [(6, 150), (64, 300)], dict(tree=[[-1, 0, -1, 2, 3, 1], list(range(-1, 31)) + list(range(-1, 31))]),
     [(0, 151, 1), (0, 154, -1), (1, 320, 0), (1, 350, 1), (1, 351, -1)]),
    ("causal", [(9, 200), (70, 90)], dict(),
     [(0, 203, 1), (0, 205, 0), (0, 206, -1), (1, 100, 1), (1, 101, -1), (1, 140, 0), (1, 3, 1)]),
    ("split", [(30, 40000), (3, 30000)], dict(), [(0, 40010, 1), (0, 40020, -1), (1, 30001, 0), (1, 20000, 1)]),
    ("window", [(40, 1000), (1, 777)], dict(window=100), [(0, 905, 1), (0, 930, -1), (0, 1010, 1), (1, 700, 0)]),
    ("prefix", [(150, 300), (20, 0)], dict(prefix=[400, 9]), [(0, 390, 1), (0, 420, -1), (0, 449, 0), (1, 7, 1), (1, 15, -1)]),
]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name,lens,opts,rows", SPECIALS, ids=[x[0] for x in SPECIALS])
def test_special_values_of_v_reach_their_own_dims(name, lens, opts, rows, D, dtype):
    """An infinity or a NaN at one dim of a V row, in tiles with masks and without, in
    units of one share and of several: the tokens that see it have the sum of what they see
    at that dim, and every other value is, bit for bit, as it is with zeros there."""
    opts = dict(opts)
    if "tree" in opts:
        opts["tree"] = tree_masks(opts["tree"])
    c = Case(lens, D=D, dtype=dtype, spread=0.3, **opts)
    value = {1: float("inf"), -1: float("-inf"), 0: float("nan")}
    T = c.q.shape[0]
    expect = torch.zeros(T, D, dtype=torch.float64)
    for x, (i, at, kind) in enumerate(rows):
        dims = [(7 * x) % D, 11]         # one of its own, one that the special rows share
        a = int(c.cu[i])
        see = c.see[i][:, at]
        assert see.any()
        for d in dims:
            expect[a:a + lens[i][0], d] += torch.where(see, value[kind], 0.0).double()
            c.V[int(c.table[i, at // c.bs]), at % c.bs, :, d] = 0
    att = c.attention()
    want = c.device().call(att).cpu()
    for x, (i, at, kind) in enumerate(rows):
        for d in ((7 * x) % D, 11):
            c.V[int(c.table[i, at // c.bs]), at % c.bs, :, d] = value[kind]
    got = c.device().call(att).cpu()
    att.check_errors()
    expect = expect[:, None].expand(T, 12, D)
    plain = expect == 0
    assert torch.equal(got[plain], want[plain])
    assert torch.equal(got[~plain].double().nan_to_num(7.0), expect[~plain].nan_to_num(7.0))


def test_errors_of_a_graph_on_another_stream_are_reported():
    """A bad block id met by a graph that is replayed on a busy stream."""
    c = Case([(5, 600), (3, 20)]).device()
    c.tabled[0, 1] = 10_000
    att, out = c.attention(), torch.empty_like(c.qd)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        c.call(att, out=out)
    for _ in range(2):
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(100_000_000)
            g.replay()
        with pytest.raises(RuntimeError, match="page"):
            att.check_errors()
        att.check_errors()


def test_out_over_a_cache_is_refused():
    c = Case([(20, 300), (3, 40)], 8, 8, D=64, bs=16).device()
    att = c.attention()
    want, K, V = c.call(att), c.Kd.clone(), c.Vd.clone()
    T = c.q.shape[0]
    for cache in (c.Kd, c.Vd):
        for at in (0, cache.numel() - T * 512):
            with pytest.raises(RuntimeError, match="overlaps a cache"):
                c.call(att, out=cache.flatten()[at:at + T * 512].view(T, 8, 64))
    both = torch.zeros(c.Kd.numel() + T * 512, dtype=BF, device=DEV)      # right behind a cache is free
    both[:c.Kd.numel()] = c.Kd.flatten()
    c.Kd, out = both[:c.Kd.numel()].view_as(c.Kd), both[c.Kd.numel():].view(T, 8, 64)
    assert torch.equal(c.call(att, out=out), want)
    assert torch.equal(c.Kd.nan_to_num(9.0), K.nan_to_num(9.0)) and torch.equal(c.Vd.nan_to_num(9.0), V.nan_to_num(9.0))


LONG = [[(3, 70000)], [(1, 40000), (64, 33333), (1, 0)], [(200, 20000)], [(1, 9000), (2, 12345), (40, 6000)] * 7]


@pytest.mark.parametrize("D,bs,H,KVH", [(64, 256, 4, 1), (128, 256, 12, 2), (64, 16, 4, 4), (128, 48, 6, 2)])
@pytest.mark.parametrize("lens,opts", [(x, {}) for x in LONG] + [
    (LONG[0], dict(window=30011)), (LONG[1], dict(causal=False)), (LONG[3], dict(window=5000)),
    ([(25, 40000), (64, 17000), (7, 999)], dict(tree=True)), (LONG[1], dict(softcap=10.0))])
def test_every_key_counts_once(lens, opts, D, bs, H, KVH):
    """Zero queries weigh all keys alike; the values say which 16 keys they belong to (a
    one at that number modulo D), so that the output counts the keys of each: a box of
    16 that is left out, read twice or taken from elsewhere changes a dim by one part
    in as many boxes as share it, several times the rounding of the result.  (Sums of
    ones are exact, the probabilities of the fp32 pipe 1e-7 off.)"""
    opts = dict(opts)
    if "tree" in opts:
        opts["tree"] = trees(lens, 6)
    c = Case(lens, H, KVH, D, bs, **opts)
    c.q.zero_()
    ref = []
    for i, (m, p) in enumerate(lens):
        k = torch.arange(m + p)
        live = c.see[i].any(0)
        code = torch.nn.functional.one_hot(k // 16 % D, D)
        c.V[c.table[i, k[live] // bs].long(), k[live] % bs] = code[live, None].to(BF).expand(-1, KVH, D)
        see = c.see[i].double()
        ref.append(see @ code.double() / see.sum(1, keepdim=True))
        assert -(-(m + p) // 16) / D < 1 / (2 * O.HALF_STEP[BF]) - 1      # (a box is seen in the result)
    att = c.attention()
    got = c.device().call(att)
    att.check_errors()
    ref = torch.cat(ref)[:, None].expand(-1, H, D)
    check(got, ref, ref * (O.HALF_STEP[BF] + 2.0 ** -21))

"""Kernels for trees of drafted tokens against 64-bit references: masks, attention, the walk, the commit, and a step."""
import pytest
import torch

from nanovllm_self_b200.ops import torch_ref as R
from test_tree_cpu import make_ctx, random_parents

pytestmark = pytest.mark.gpu

DEV = "cuda"
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from nanovllm_self_b200.ops import get_ops
    return get_ops(DEV)


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    from nanovllm_self_b200.ops._ext import load
    torch.cuda.synchronize()
    assert load().tree_error(True) == 0


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------------------------- masks
@pytest.mark.parametrize("ns,rows", [([1], 0), ([8], 3), ([5, 1, 3, 64, 2], 0), ([65, 0, 2], 5), ([256, 255, 200], 1),
                                     ([130] * 3, 0), (list(range(1, 40)), 2)])
def test_mask(ops, ns, rows):
    ctx, _ = make_ctx(ns, [max(1, n) for n in ns], device=DEV)
    parents = torch.cat([random_parents(ns, len(ns)), torch.zeros(rows, dtype=torch.int32)])
    parents[-1] = 1 << 20
    want = R.tree_mask(parents, ctx.cu_seqlens_q.tolist(), ctx.max_seqlen_q)
    got = ops.tree_mask(parents.to(DEV), ctx)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_mask_of_a_chain_and_of_more_nodes_than_the_largest_tree(ops):
    ctx, _ = make_ctx([256, 100], [256, 100], device=DEV)
    parents = torch.cat([torch.arange(256) - 1, torch.arange(100) - 1]).int()
    for most in (256, 64, 1):
        ctx.max_seqlen_q = most
        want = R.tree_mask(parents, ctx.cu_seqlens_q.tolist(), most)
        got = ops.tree_mask(parents.to(DEV), ctx)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


# --------------------------------------------------------------------------------- attention
class Case:
    """Trees over a paged cache, and their attention in 64 bits with the bound of its error."""

    def __init__(self, ns, ks, nq, nkv, bs, dtype=torch.bfloat16, seed=0, spread=1.5, rows=0, mask=None):
        g = _gen(seed)
        self.ns, self.ks, self.nq, self.nkv, self.bs, self.dtype = ns, ks, nq, nkv, bs, dtype
        self.ctx, nb = make_ctx(ns, ks, bs, device=DEV)
        perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).int().to(DEV)
        self.ctx.block_tables = perm[self.ctx.block_tables.long()]
        self.T = sum(ns) + rows
        self.scale = 128 ** -0.5
        self.q = (spread * torch.randn(self.T, nq * 128, device=DEV, generator=g)).bfloat16()
        shape = (nb, nkv, bs, 128)
        self.ks_, self.vs_ = None, None
        if dtype == F8:
            # scales that differ by two orders of magnitude between blocks
            self.ks_, self.vs_ = (torch.exp(1.5 * torch.randn(shape[:2], device=DEV, generator=g)) / 60 for _ in range(2))
            self.k, self.v = ((60 * torch.randn(shape, device=DEV, generator=g)).clamp(-448, 448).to(F8) for _ in range(2))
            self.ks_.clamp_(1e-3, 0.05)
        else:
            self.k, self.v = (torch.randn(shape, device=DEV, generator=g).bfloat16() for _ in range(2))
        parents = random_parents(ns, seed + 1)
        self.mask = R.tree_mask(torch.cat([parents, torch.zeros(rows, dtype=torch.int32)]),
                                self.ctx.cu_seqlens_q.tolist(), max(ns))[0].to(DEV) if mask is None else mask

    def run(self, ops, q=None):
        return ops.attention_tree(self.q if q is None else q, self.k, self.v, self.ctx, self.mask, self.scale, self.ks_, self.vs_)

    def oracle(self):
        """(outputs, bound of the error) in 64 bits; what a row does not see is left out of its sums."""
        out = torch.zeros(self.T, self.nq, 128, dtype=torch.float64, device=DEV)
        bound = torch.zeros_like(out)
        at, g = 0, self.nq // self.nkv
        for b, (n, kl) in enumerate(zip(self.ns, self.ks)):
            if n and kl > 0:
                ids = self.ctx.block_tables[b, :-(-kl // self.bs)].long()
                k, v = self.k[ids].double(), self.v[ids].double()
                if self.dtype == F8:
                    k, v = k * self.ks_[ids].double()[..., None, None], v * self.vs_[ids].double()[..., None, None]
                k, v = (x.transpose(0, 1).reshape(self.nkv, -1, 128)[:, :kl] for x in (k, v))
                q = self.q[at:at + n].double().view(n, self.nkv, g, 128)
                j = torch.arange(kl, device=DEV) - (kl - n)
                see = (j < 0) | (self.mask[at:at + n][:, j.clamp(min=0) // 64] >> (j.clamp(min=0) % 64) & 1).bool()
                s = torch.einsum("nhgd,hkd->hgnk", q, k) * self.scale
                size = torch.einsum("nhgd,hkd->hgnk", q.abs(), k.abs()).amax() * self.scale
                s = s.masked_fill(~see, float("-inf"))
                a = torch.softmax(s, -1).nan_to_num(0.0)
                out[at:at + n] = torch.einsum("hgnk,hkd->nhgd", a, v).reshape(n, self.nq, 128)
                aabs = torch.einsum("hgnk,hkd->nhgd", a, v.abs()).reshape(n, self.nq, 128)
                # a score: 128 rounded sums and 4 products of it, exp2 to 2^-22, the sums over at most 2^15 keys in
                # tiles: 600 roundings; each weight (8-bit caches: times V's scale) is rounded to bf16, half a step
                # of which is 2^-8 of it
                e = 2 * (float(size) * 132 * 2.0 ** -24 + 2.0 ** -21) + 600 * 2.0 ** -24
                bound[at:at + n] = aabs * (e + 2.0 ** -8)
            at += n
        return out, bound + out.abs() * 2.0 ** -8 + 1e-30

    def check(self, got):
        want, bound = self.oracle()
        n = sum(self.ns)
        err = (got.view(self.T, self.nq, 128).double() - want).abs()
        worst = float((err[:n] / bound[:n]).nan_to_num(1e30).max())
        assert worst <= 1


KV = pytest.mark.parametrize("dtype", [torch.bfloat16, F8])


@KV
@pytest.mark.parametrize("nq,nkv", [(32, 8), (16, 8), (8, 1), (4, 4), (15, 3), (20, 1)])
@pytest.mark.parametrize("ns,ks", [([8], [600]), ([1], [1]), ([5, 1, 16, 3], [70, 1, 16, 1000]), ([17, 64], [64, 321])])
def test_attention(ops, dtype, nq, nkv, ns, ks):
    c = Case(ns, ks, nq, nkv, 16, dtype)
    c.check(c.run(ops))


@KV
@pytest.mark.parametrize("bs", [16, 32, 64, 256])
@pytest.mark.parametrize("k", [62, 63, 64, 65, 127, 128, 129, 256, 257])
def test_attention_at_the_edges_of_tiles_and_blocks(ops, dtype, bs, k):
    c = Case([7, 2, 33], [k, k + 1, k + 31], 8, 2, bs, dtype, seed=k)
    c.check(c.run(ops))


@KV
@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 9, 16, 17, 63, 64, 65, 130, 256])
def test_attention_over_tree_sizes(ops, dtype, n):
    c = Case([n, max(1, n // 3)], [n + 300, n + 5], 8, 2, 64, dtype, seed=n)
    c.check(c.run(ops))


@KV
def test_attention_ragged_batch(ops, dtype):
    g = torch.Generator().manual_seed(5)
    ns = torch.randint(0, 17, (61,), generator=g).tolist()
    ks = [n + int(torch.randint(0, 3000, (), generator=g)) for n in ns]
    ks[3] = ns[3]
    c = Case(ns, ks, 32, 8, 64, dtype, rows=3)
    c.check(c.run(ops))


@KV
def test_attention_long_context_and_no_context(ops, dtype):
    c = Case([12, 1, 6], [32768 + 12, 1, 6], 8, 2, 256, dtype)
    c.check(c.run(ops))


@KV
@pytest.mark.parametrize("longer", [0, 1, 7])
def test_attention_many_items_of_one_tile(ops, dtype, longer):
    """Between 64 and 128 rows over contexts of up to a tile, some ten items per CTA: one of the two groups has no step
    in them, but in the contexts of a few tiles among them."""
    g = torch.Generator().manual_seed(longer)
    ns = torch.randint(17, 33, (200,), generator=g).tolist()
    ks = [n + int(torch.randint(0, 128 - n + 1, (), generator=g)) for n in ns]
    for i in range(longer):
        ks[29 * i + 3] = 128 * (i + 1) + 1
    c = Case(ns, ks, 32, 8, 16, dtype, seed=longer)
    first = c.run(ops)
    c.check(first)
    for _ in range(5):
        assert torch.equal(c.run(ops), first)


@KV
def test_attention_is_the_same_on_every_run(ops, dtype):
    """Fewer tiles than CTAs, and more; memory that the allocator hands out again holds other sums, or NaN."""
    for c in (Case([8], [600], 8, 2, 16, dtype), Case([8, 3, 16], [2000, 70, 512], 32, 8, 64, dtype)):
        first = c.run(ops)
        c.check(first)
        for fill in (float("nan"), float("inf"), 1e30):
            junk = [torch.full((1 << 22,), fill, device=DEV) for _ in range(8)]
            del junk
            assert torch.equal(c.run(ops), first)


@KV
def test_attention_rows_without_anything_to_see(ops, dtype):
    """Empty mask rows behind a context see the context; without one they give zeros, as padding sequences do."""
    c = Case([4, 3, 2], [4, 40, 0], 8, 2, 16, dtype)
    c.mask[1] = 0
    c.mask[5] = 0
    got = c.run(ops)
    c.check(got)
    assert (got[1] == 0).all() and (got[7:] == 0).all()


@KV
def test_attention_masked_infinities_and_nan_take_no_part(ops, dtype):
    c = Case([9, 70], [50, 300], 8, 2, 16, dtype)
    clean = c.run(ops)
    bad = float("nan")

    def rows(b, pos):
        return int(c.ctx.block_tables[b, pos // 16]), pos % 16

    # node 5 of the first tree and node 66 of the second, and all that lies behind the contexts
    hit = []
    for b, node in ((0, 5), (1, 66)):
        n, k = c.ns[b], c.ks[b]
        blk, off = rows(b, k - n + node)
        c.k.view(torch.uint8)[blk, :, off] = 0xff        # a NaN in both types
        c.v[blk, 0, off, 3] = bad
        c.v[blk, 1, off, ::7] = bad if dtype == F8 else float("-inf")
        hit.append(node)
        for p in range(k, -(-k // 16) * 16):
            blk, off = rows(b, p)
            c.k.view(torch.uint8)[blk, :, off] = 0xff
            c.v.view(torch.uint8)[blk, :, off] = 0x7f if dtype == F8 else 0xff
    got = c.run(ops)
    at = 0
    for n, node in zip(c.ns, hit):
        sees = (c.mask[at:at + n, node // 64] >> (node % 64) & 1).bool()
        assert torch.equal(got[at:at + n][~sees], clean[at:at + n][~sees]) and (~sees).any()
        assert got[at:at + n][sees].isnan().all(-1).all()  # its score is a NaN
        at += n


@KV
def test_attention_visible_infinite_values_reach_their_rows(ops, dtype):
    """A value that is not finite, under a finite score: the dims that hold it in the rows that see it, no others."""
    c = Case([6], [37], 4, 2, 16, dtype)
    clean = c.run(ops).view(6, 4, 128)
    blk = int(c.ctx.block_tables[0, (31 + 2) // 16])
    c.v[blk, 1, (31 + 2) % 16, 17] = float("nan") if dtype == F8 else float("inf")
    got = c.run(ops).view(6, 4, 128)
    sees = (c.mask[:, 0] >> 2 & 1).bool()
    want = clean.clone()
    want[sees, 2:, 17] = float("nan") if dtype == F8 else float("inf")
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("ns,ks,nq,nkv", [([20, 3], [52, 40], 2, 2), ([20], [308], 4, 2), ([20, 9], [52, 300], 6, 2),
                                          ([20, 7], [52, 800], 32, 4), ([200], [232], 2, 2)])
def test_attention_masked_scales_take_no_part(ops, ns, ks, nq, nkv, bad):
    """Scales of blocks behind the contexts, and of blocks that hold nodes which some rows do not see."""
    c = Case(ns, ks, nq, nkv, 16, F8)
    c.mask[:16, 0] &= 0xffff                    # the first tree's first 16 nodes see none of the others, which
    base, nb = ks[0] - ns[0], c.k.shape[0]      # lie in blocks of their own
    assert base % 16 == 0
    # behind the contexts the tables name a block that nobody owns
    extra = torch.full((1, nkv, 16, 128), 0x38, dtype=torch.uint8, device=DEV)
    c.k, c.v = (torch.cat([x.view(torch.uint8), extra]).view(F8) for x in (c.k, c.v))
    c.ks_, c.vs_ = (torch.cat([s, torch.ones(1, nkv, device=DEV)]) for s in (c.ks_, c.vs_))
    t = torch.full((len(ns), c.ctx.block_tables.shape[1] + 8), nb, dtype=torch.int32, device=DEV)
    for b, k in enumerate(ks):
        t[b, :-(-k // 16)] = c.ctx.block_tables[b, :-(-k // 16)]
    c.ctx.block_tables = t
    clean = c.run(ops)
    c.check(clean)
    for s in (c.ks_, c.vs_):
        s[nb] = bad
    assert torch.equal(c.run(ops), clean)
    late = t[0, (base + 16) // 16:-(-ks[0] // 16)].long()
    sees = torch.zeros(c.T, dtype=torch.bool, device=DEV)
    sees[:ns[0]] = torch.stack([(c.mask[:ns[0], i // 64] >> (i % 64) & 1).bool() for i in range(16, ns[0])]).any(0)
    assert sees.any() and not sees[:16].any()
    for s in (c.vs_, c.ks_):
        keep = s.clone()
        s[late] = bad
        got = c.run(ops)
        s.copy_(keep)
        assert torch.equal(got[~sees], clean[~sees])
        assert s is c.ks_ or not got[sees].isfinite().any()


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("nq,nkv", [(2, 2), (16, 4)])
def test_attention_visible_scales_reach_their_rows(ops, nq, nkv, bad):
    """A scale that is not finite over the last cached tokens and the first nodes, or over the last nodes: infinite or NaN
    where the values times their scale, added up over what a row sees, are."""
    c = Case([20], [53], nq, nkv, 16, F8)
    for place in (2, 3):
        keep = c.vs_.clone()
        c.vs_[int(c.ctx.block_tables[0, place])] = bad
        got = c.run(ops).view(20, nq, 128)
        want = R.tree_attention(c.q.view(20, nq, 128), c.k, c.v, c.ns, c.ks, c.ctx.block_tables.tolist(), c.mask, c.scale,
                                c.ks_, c.vs_)
        c.vs_.copy_(keep)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        assert torch.equal(got[got.isinf()], want[want.isinf()]) and (want.isinf().any() or bad != bad)
        assert not want[0].isfinite().any() if place == 2 else want[0].isfinite().all()


def test_attention_bad_blocks_read_as_zeros(ops):
    c = Case([5], [200], 8, 2, 16)
    t = c.ctx.block_tables
    bad = t.clone()
    bad[0, 2], bad[0, 5], bad[0, 12] = -1, c.k.shape[0], 1 << 30
    c.ctx.block_tables = bad
    got = c.run(ops)
    for i in (2, 5, 12):
        c.k[int(t[0, i])], c.v[int(t[0, i])] = 0, 0
    c.ctx.block_tables = t
    c.check(got)
    c.ctx.block_tables = t[:, :11].contiguous()     # a table that ends early
    got = c.run(ops)
    c.ctx.block_tables = t
    for i in range(11, t.shape[1]):
        c.k[int(t[0, i])], c.v[int(t[0, i])] = 0, 0
    c.check(got)


@KV
def test_attention_large_and_small_magnitudes(ops, dtype):
    """Scores of some hundreds (one key takes all), and queries far from 1 in both directions."""
    for spread in (40.0, 1e-4):
        c = Case([8], [500], 8, 2, 16, dtype, spread=spread)
        c.check(c.run(ops))
    c = Case([8], [300], 8, 2, 16, dtype)
    if dtype == F8:
        # q's range is bf16's: the cache's scales bring the scores back
        c.q = (c.q.float() * 2.0 ** 30).bfloat16()
        c.ks_ = c.ks_ * 2.0 ** -30
        c.check(c.run(ops))


@KV
@pytest.mark.parametrize("ns,ks,nq,nkv", [([256], [700], 2, 2), ([40, 9], [300, 77], 16, 4), ([8, 5], [300, 500], 8, 2)])
def test_attention_with_a_negative_scale(ops, dtype, ns, ks, nq, nkv):
    """Scores of some hundreds of both signs: weights are relative to the largest of scale q k, not of q k."""
    c = Case(ns, ks, nq, nkv, 16, dtype, spread=40.0)
    c.check(ops.attention_tree(-c.q, c.k, c.v, c.ctx, c.mask, -c.scale, c.ks_, c.vs_))


def test_attention_strided_operands(ops):
    c = Case([8, 5], [300, 77], 8, 2, 16)
    want = c.run(ops)
    wide = torch.randn(13, 8 * 128 + 512, device=DEV).bfloat16()
    wide[:, 256:256 + 1024] = c.q
    assert torch.equal(c.run(ops, wide[:, 256:256 + 1024]), want)
    assert torch.equal(c.run(ops, c.q.view(13, 8, 128)), want)
    big = torch.zeros(2, c.ctx.block_tables.shape[1] + 3, dtype=torch.int32, device=DEV)
    big[:, :-3] = c.ctx.block_tables
    c.ctx.block_tables = big[:, :-3]
    m = torch.full((13, 3), -1, dtype=torch.int64, device=DEV)
    m[:, :1] = c.mask
    c.mask = m[:, :2]
    assert torch.equal(c.run(ops), want)


def test_attention_cache_rows_past_2_31_bytes(ops):
    c = Case([8], [500], 4, 1, 256)
    nb = (5 << 30) // (256 * 256)           # 5 GiB of keys
    k = torch.zeros(nb, 1, 256, 128, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    ids = torch.tensor([nb - 1, nb // 2 + 1], device=DEV)
    k[ids], v[ids] = c.k[c.ctx.block_tables[0].long()], c.v[c.ctx.block_tables[0].long()]
    c.k, c.v = k, v
    c.ctx.block_tables = ids.int()[None]
    c.check(c.run(ops))


def test_attention_on_a_side_stream_and_in_graphs(ops):
    """Two captured graphs of different trees replayed on two streams at once: each has a workspace of its own."""
    cases = [Case([8, 3], [2000, 900], 32, 8, 64, seed=1), Case([16] * 4, [1500] * 4, 32, 8, 64, seed=2)]
    want = [c.run(ops).clone() for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(cases[0].run(ops), want[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c.run(ops)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out, w)
    # new lengths in the captured tensors
    c = cases[0]
    c.ks = [1200, 300]
    c.ctx.context_lens.copy_(torch.tensor(c.ks))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    c.check(graphs[0][1])


def test_an_expired_wait_reaches_the_caller(ops):
    """The code of a wait that runs out is what device_error gives once the stream is synchronised, and only until it is
    cleared; calls behind it are as they were."""
    c = Case([8], [600], 8, 2, 16)
    want = c.run(ops)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    ops.C.tree_wait_check(1000000)     # nothing ends this wait: given up after a millisecond
    got = c.run(ops)
    torch.cuda.synchronize()
    assert ops.device_error() == 699 and ops.C.tree_error() == 699 and torch.equal(got, want)
    assert ops.C.tree_error(True) == 699 and ops.device_error() == 0


# ------------------------------------------------------------------------------ verification
class Walk:
    def __init__(self, ns, v, dtype=torch.bfloat16, draft=False, seed=0, temps=(1.0, 0.7, 0.0), spread=2.0):
        g = torch.Generator().manual_seed(seed)
        self.ns, t, b = ns, sum(ns), len(ns)
        self.ctx, _ = make_ctx(ns, [max(n, 1) for n in ns], device=DEV)
        self.parents = random_parents(ns, seed + 1)
        x = spread * torch.randn(t, v, generator=g)
        likely = torch.randint(0, v, (t, 4), generator=g)
        x.scatter_(1, likely, x.amax(-1, keepdim=True) + torch.tensor([3.0, 2.5, 1.5, 1.0]))
        self.logits = x.to(dtype)
        self.temps = torch.tensor([temps[i % len(temps)] for i in range(b)])
        start = torch.repeat_interleave(torch.tensor([0] + ns[:-1]).cumsum(0), torch.tensor(ns))
        above = (start + self.parents).clamp(min=0, max=max(t - 1, 0))
        rank = torch.randint(0, 4, (t,), generator=g)
        self.draft = torch.softmax(x + 0.7 * torch.randn(t, v, generator=g), -1) if draft else None
        if draft:
            self.tokens = torch.multinomial(self.draft[above], 1, generator=g)[:, 0].int()
        else:
            self.tokens = likely[above, rank].int()
        self.u, self.ud = torch.rand(t, generator=g), torch.rand(b, generator=g)

    def operands(self):
        return (self.logits, self.tokens, self.parents, self.temps, self.u, self.ud, self.draft)

    def want(self):
        x, tok, par, temps, u, ud, draft = self.operands()
        return R.tree_verify(x, tok, par, self.ns, self.ctx.max_seqlen_q, temps, u, ud, draft)

    def run(self, ops):
        x, tok, par, temps, u, ud, draft = (None if o is None else o.to(DEV) for o in self.operands())
        return ops.verify_tree(x, tok, par, self.ctx, temps, u, ud, draft)

    def check(self, ops):
        for got, want in zip(self.run(ops), self.want()):
            assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ns,v", [([1], 1), ([8], 17), ([3, 0, 9], 1000), ([16] * 9, 1024), ([5, 64, 1], 4099),
                                  ([12] * 40, 2050), ([8] * 3, 37987), ([256, 2], 333)])
def test_walk(ops, draft, dtype, ns, v):
    Walk(ns, v, dtype, draft, seed=v).check(ops)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("b", [1, 5, 20, 32, 33, 80, 170])
def test_walk_over_cluster_sizes(ops, draft, b):
    """A tree takes up to 16 CTAs where trees are few, up to 8 smaller ones where they are many."""
    Walk([3] * b, 20001, torch.bfloat16, draft, seed=b).check(ops)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("b", [3, 40])
def test_walk_with_numbers_next_to_the_borders(ops, b, draft):
    """Random numbers that are the fp32 values next to a probability (tests) or to a border of the cumulative sum (draws),
    on either side: within 1e-7 of it, and by the widths of these distributions never within the 1e-11 of 64-bit sums."""
    for seed in range(4):
        w = Walk([4] * b, 20011, torch.float32, draft, seed, temps=(1.0, 0.6, 1.4), spread=1.0)
        start = torch.arange(b).repeat_interleave(4) * 4
        above = start + w.parents.clamp(min=0)
        p = torch.softmax(w.logits.double() / w.temps.double().repeat_interleave(4)[:, None], -1)
        tok = w.tokens.long()
        near = p[above, tok] / (w.draft[above, tok].double() if draft else 1.0)
        w.u = near.clamp(max=1.0).float()
        pick = torch.randint(0, 20011, (b,), generator=torch.Generator().manual_seed(seed))
        w.ud = p[::4].cumsum(-1)[torch.arange(b), pick].float()  # of the root, where its children are rejected or none
        if seed % 2:
            w.u, w.ud = torch.nextafter(w.u, torch.ones(())), torch.nextafter(w.ud, torch.zeros(()))
        w.parents[torch.arange(0, 4 * b, 4 * 3)[:, None] + torch.arange(1, 4)] = -1  # every third tree: the draw alone
        w.check(ops)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_walk_full_vocabulary_flat_and_peaked(ops, dtype):
    for spread, seed in ((0.0, 1), (0.1, 2), (8.0, 3)):
        Walk([4, 6, 2, 5, 3, 4], 151936, dtype, False, seed, (1.0, 2.5, 0.3), spread).check(ops)
    Walk([4, 6, 2], 151936, dtype, True, 4).check(ops)


def test_walk_long_vocabulary(ops):
    Walk([3, 2], 1200003, torch.bfloat16, True, 7).check(ops)


def test_walk_many_rejections(ops):
    """A root with 40 children, none of which is taken: the residual is taken from 40 times; draws from what is left."""
    for draft in (False, True):
        w = Walk([41, 41, 41], 300, torch.float32, draft, 3, (1.0,))
        w.parents = torch.tensor([-1] + [0] * 40, dtype=torch.int32).repeat(3)
        w.u = torch.full_like(w.u, 1 - 2.0 ** -24)
        w.ud = torch.tensor([0.0, 0.5, 1 - 2.0 ** -24])
        w.check(ops)


def test_walk_where_the_draft_is_the_target(ops):
    """p = q: every child is taken at u < 1 and nothing is left behind one that is not (u = 1)."""
    w = Walk([4, 4], 512, torch.float32, True, 5, (1.0,))
    w.draft = torch.softmax(w.logits.double(), -1).float()
    w.draft[:4] = 0
    w.draft[torch.arange(4), w.logits[:4].argmax(-1)] = 1.0
    w.logits[:4] = float("-inf")
    w.logits[torch.arange(4), w.draft[:4].argmax(-1)] = 3.0
    w.parents = torch.tensor([-1, 0, 0, 0] * 2, dtype=torch.int32)
    w.tokens[:4] = int(w.draft[0].argmax())
    w.u[:4] = 1.0
    w.check(ops)
    assert w.want()[1][0] == 1


@pytest.mark.parametrize("v", [301, 1303])
@pytest.mark.parametrize("b", [9, 24, 40])
def test_walk_behind_rejections_of_a_draft_near_the_target(ops, b, v):
    """q = p (1 +- 2^-21): a rejection leaves 2.4e-7 of p and multiplies its relative error by 2^21, a second one by 2.
    p is within 1e-13 of itself, so the cumulative shares within 1e-13 2^22 / 2 = 2.1e-7 (an error e of each term moves
    a share c by 2 c (1 - c) e at most); the draws are 2.4e-7 and more from a border, the tests 3e-7 of p."""
    w = Walk([3] * b, v, torch.float32, True, b, temps=(1.0, 0.6, 1.4), spread=1.0)
    g = torch.Generator().manual_seed(b)
    p = torch.softmax(w.logits.double() / w.temps.double().repeat_interleave(3)[:, None], -1)
    more = torch.rand(3 * b, v, generator=g) < 0.5
    w.draft = (p * torch.where(more, 1 + 2.0 ** -21, 1 - 2.0 ** -21)).float()
    w.parents = torch.tensor([-1, 0, 0] * b, dtype=torch.int32)
    w.parents[2::6] = -1                                  # one rejection in every other tree, two in the rest
    above = (torch.arange(b) * 3).repeat_interleave(3)
    w.tokens = torch.multinomial(p[above] * more[above], 1, generator=g)[:, 0].int()
    w.u = torch.full_like(w.u, 1 - 2.0 ** -24)            # u q is above p
    for i in range(b):
        r, q = p[3 * i], w.draft[3 * i].double()
        for _ in range(1 + int(w.parents[3 * i + 2] == 0)):
            r = (r - q).clamp(min=0.0)
            r = r / r.sum()
        c = r.cumsum(0)
        # next to a border below a quarter, where fp32 numbers are 1.5e-8 apart at most, on either side of it
        at = int(torch.randint(0, int((c < 0.25).sum()), (), generator=g))
        share = float(c[at]) + (1 if i % 2 else -1) * (2.5e-7 + 5e-8 * int(torch.randint(0, 3, (), generator=g)))
        w.ud[i] = max(share, 0.0)
    w.check(ops)
    assert (w.want()[1] == 1).all()


@pytest.mark.parametrize("b", [12, 40])  # 40: summed in fp32 first
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_walk_infinities_nan_and_odd_numbers(ops, dtype, b):
    inf, nan = float("inf"), float("nan")
    for v in (5, 3001):
        w = Walk([3] * b, v, dtype, False, v, (1.0,))
        x = w.logits
        x[0] = -inf
        x[3, ::2] = nan
        x[6] = nan
        x[9, 2:4] = inf
        x[12, 1:] = -inf
        x[15, : v // 2] = -inf
        x[18] = x[18].abs() * 1e30
        w.temps[:12] = torch.tensor([1.0, 1, 1, 1, 1, 1, 1, 1e-30, 1e30, inf, nan, -1])
        w.tokens[1:3] = torch.tensor([-1, v])
        w.tokens[9:12] = torch.tensor([0, 2, 3])
        w.ud[:7] = torch.tensor([0.5, 1.0, nan, 0.7, -2.0, 1.0, 3.0])
        w.u[20], w.u[23] = nan, -1.0
        w.check(ops)


def test_walk_draft_probabilities_that_are_none(ops):
    w = Walk([6, 6], 700, torch.float32, True, 11, (1.0, 0.8))
    w.draft[:, ::3] = float("nan")
    w.draft[:, 1::5] = -1.0
    w.draft[7, 4] = float("inf")
    w.check(ops)


def test_walk_ties_take_the_lowest_index(ops):
    w = Walk([2] * 4, 70000, torch.bfloat16, False, 1, (0.0,))
    w.logits[:] = 1.0
    w.logits[2, 40000:] = 2.0
    w.logits[4, [69999, 1025, 5]] = 3.0
    w.check(ops)


def test_walk_rows_of_any_alignment(ops):
    for dtype in (torch.bfloat16, torch.float32):
        w = Walk([5, 3], 5001, dtype, True, 2)
        want = w.run(ops)
        t, v = w.logits.shape
        for off in (1, 2, 3, 5):
            big = torch.zeros(t, v + 9, dtype=dtype, device=DEV)[:, off:off + v]
            big.copy_(w.logits)
            d = torch.zeros(t, v + 6, device=DEV)[:, off:off + v]
            d.copy_(w.draft)
            got = ops.verify_tree(big, w.tokens.to(DEV), w.parents.to(DEV), w.ctx, w.temps.to(DEV), w.u.to(DEV), w.ud.to(DEV), d)
            assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("draft", [False, True])
def test_walk_many_trees_in_rows_of_any_alignment(ops, draft):
    """More trees than get a CTA of 512 threads, rows of an odd length; a vocabulary in chunks longer than 512 tokens."""
    Walk([2] * 70, 9001, torch.bfloat16, draft, 3, (1.0, 0.5, 2.0), spread=3.0).check(ops)
    Walk([1] * 34, 270001, torch.bfloat16, draft, 4, (1.0, 0.5), spread=3.0).check(ops)


def test_walk_in_a_graph(ops):
    w = Walk([8] * 6, 3000, torch.bfloat16, True, 9)
    dev = [None if o is None else o.to(DEV) for o in w.operands()]
    x, tok, par, temps, u, ud, draft = dev
    ops.verify_tree(x, tok, par, w.ctx, temps, u, ud, draft)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.verify_tree(x, tok, par, w.ctx, temps, u, ud, draft)
    w2 = Walk([8] * 6, 3000, torch.bfloat16, True, 10)
    for dst, src in zip(dev, w2.operands()):
        dst.copy_(src)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(out, w2.want()))


# ------------------------------------------------------------------------------------ commit
def _commit_case(ns, ks, bs, dtype, L=3, nkv=2, seed=0, width=None):
    g = _gen(seed)
    ctx, nb = make_ctx(ns, ks, bs, device=DEV)
    shape = (2, L, nb, nkv, bs, 128)
    kv = (30 * torch.randn(shape, device=DEV, generator=g)).clamp(-448, 448).to(dtype)
    s = torch.exp(torch.randn(shape[:4], device=DEV, generator=g)) / 30 if dtype == F8 else None
    h = torch.Generator().manual_seed(seed + 1)
    width = width or max(ns)
    path = torch.full((len(ns), width), -1, dtype=torch.int32)
    length = []
    for b, n in enumerate(ns):
        k = int(torch.randint(0, min(n, width), (), generator=h)) if n else 0
        nodes = sorted((torch.randperm(n - 1, generator=h)[:k] + 1).tolist()) if n > 1 else []
        path[b, :1 + len(nodes)] = torch.tensor([0] + nodes)
        length.append(1 + len(nodes) if n else 0)
    return ctx, kv, s, path.to(DEV), torch.tensor(length, dtype=torch.int32, device=DEV)


def _check_commit(ops, ctx, kv, s, path, length):
    # the oracle on the GPU too: there a division by 448 is a product with its reciprocal, as where K/V is stored
    kv2, s2 = kv.clone(), None if s is None else s.clone()
    R.tree_commit(kv2, ctx.host_q_lens, ctx.host_k_lens, ctx.block_tables.tolist(), path.cpu(), length.cpu(), s2)
    ops.commit_tree(kv, ctx, path, length, s)
    assert torch.equal(kv.view(torch.uint8), kv2.view(torch.uint8))  # the same fp32 operations: bit for bit
    assert s is None or torch.equal(s, s2)


@KV
@pytest.mark.parametrize("bs", [1, 4, 16, 256])
@pytest.mark.parametrize("ns,ks", [([1], [1]), ([8], [600]), ([16, 5, 0, 64], [40, 5, 0, 130]), ([256, 31], [300, 64])])
def test_commit(ops, dtype, bs, ns, ks):
    for seed in range(3):
        _check_commit(ops, *_commit_case(ns, ks, bs, dtype, seed=seed))


@KV
def test_commit_many_layers_heads_and_narrow_paths(ops, dtype):
    _check_commit(ops, *_commit_case([20] * 9, list(range(20, 29)), 16, dtype, L=36, nkv=8, width=6))
    _check_commit(ops, *_commit_case([7] * 5, [30] * 5, 16, dtype, L=5, nkv=1))


@KV
def test_commit_paths_that_end_early_and_bad_blocks(ops, dtype):
    ctx, kv, s, path, length = _commit_case([9] * 6, [40] * 6, 16, dtype)
    path[:, :] = torch.tensor([[0, 2, 4, 4, 6, 7, 8, -1, -1], [0, 3, 9, 5, 6, 7, 8, -1, -1], [0, 5, 3, 6, 7, 8, -1, -1, -1],
                               [-1, 3, 4, 5, 6, 7, 8, -1, -1], [2, 3, 4, 5, 6, 7, 8, -1, -1], [0, 4, 5, 6, 7, 8, -1, -1, -1]])
    length[:] = torch.tensor([7, 7, 6, 7, 7, 100])
    ctx.block_tables[4, 2] = -1
    ctx.block_tables[5, 1] = kv.shape[2] + 7
    _check_commit(ops, ctx, kv, s, path, length)
    # a context that is shorter than the tree: nothing moves
    ctx, kv, s, path, length = _commit_case([9], [40], 16, dtype)
    ctx.context_lens[0], ctx.host_k_lens[0] = 4, 4
    _check_commit(ops, ctx, kv, s, path, length)


def test_commit_scales_of_any_size(ops):
    """Quotients by scales far from 1, where the remainder of a quotient would fall below fp32's smallest."""
    for size in (1e-30, 1e-12, 1e12, 1e30):
        ctx, kv, s, path, length = _commit_case([16, 9], [40, 30], 16, F8, seed=4)
        s *= size
        _check_commit(ops, ctx, kv, s, path, length)


@pytest.mark.parametrize("bs", [4, 16])
def test_commit_between_scales_of_different_sizes(ops, bs):
    """Every pair of sizes as source and destination: quotients past fp32's range saturate, ones below the format vanish."""
    sizes = torch.tensor([1e-38, 2e-20, 1e-8, 1.0, 5e19, 1e30], device=DEV)
    for seed in range(4):
        ctx, kv, s, path, length = _commit_case([16] * 12, [37 + i for i in range(12)], bs, F8, L=4, seed=seed)
        pick = torch.randint(0, len(sizes), s.shape, device=DEV, generator=_gen(seed))
        s = sizes[pick] * (1 + torch.rand(s.shape, device=DEV, generator=_gen(seed)))
        _check_commit(ops, ctx, kv, s, path, length)


@KV
def test_commit_of_a_range_of_layers(ops, dtype):
    ctx, kv, s, path, length = _commit_case([12, 12], [40, 29], 16, dtype, L=6)
    kv0, s0 = kv.clone(), None if s is None else s.clone()
    _check_commit(ops, ctx, kv[:, 2:4], None if s is None else s[:, 2:4], path, length)
    for i in (0, 1, 4, 5):
        assert torch.equal(kv[:, i].view(torch.uint8), kv0[:, i].view(torch.uint8)) and (s is None or torch.equal(s[:, i], s0[:, i]))


# ------------------------------------------------------------------------- a step of a model
@pytest.mark.parametrize("kv", ["none", "fp8"])
def test_steps_of_drafted_trees_equal_steps_of_single_tokens(kv):
    """The operators in a row on the engine's model and pool: a tree around the tokens that single steps choose is
    accepted as they are, and the cache that the commit leaves gives the logits that theirs gives."""
    from nanovllm_self_b200 import LLM
    from nanovllm_self_b200.utils.context import Context
    llm = LLM("tiny-gpu", block_size=16, max_model_len=512, num_blocks=64, kv_cache_quant_mode=kv, enforce_eager=True)
    run, ops = llm.model_runner, llm.model_runner.ops
    table = torch.arange(3, 3 + run.max_blocks_per_seq, dtype=torch.int32, device=DEV)[None]

    def forward(tokens, positions, start, n, mask=None, decode=0):
        ctx = Context(cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device=DEV),
                      context_lens=torch.tensor([start + n], dtype=torch.int32, device=DEV), block_tables=table,
                      num_seqs=1, num_tokens=n, max_seqlen_q=n, max_seqlen_k=start + n, num_decode_seqs=decode,
                      host_q_lens=[n], host_k_lens=[start + n], tree_mask=mask)
        pos = torch.arange(start, start + n, device=DEV)
        ctx.slot_mapping = (table[0, pos // 16] * 16 + pos % 16).int()
        ctx.logits_indices = torch.arange(n, dtype=torch.int32, device=DEV)
        return ctx, run.model.forward(torch.tensor(tokens, dtype=torch.int32, device=DEV), positions, ctx, run.kv_layers,
                                      run.kv_scale_layers)

    def lin(a, n):
        return torch.arange(a, a + n, dtype=torch.int32, device=DEV)

    prompt = torch.randint(3, 2000, (27,), generator=torch.Generator().manual_seed(0)).tolist()
    # single steps, and what they choose
    forward(prompt[:-1], lin(0, 26), 0, 26)
    line, rows = list(prompt), []
    for i in range(9):
        _, x = forward([line[-1]], lin(26 + i, 1), 26 + i, 1, decode=1)
        rows.append(x[0].float())
        line.append(int(x[0].argmax()))
    forward(prompt[:-1], lin(0, 26), 0, 26)
    tokens = list(prompt)
    for step in range(3):
        start = len(tokens) - 1
        good = line[start + 1:start + 4]
        tree = [tokens[-1], good[0] ^ 1, good[0], 11, good[1], good[1] ^ 1, 12]
        par = torch.tensor([-1, 0, 0, 1, 2, 2, 4], dtype=torch.int32, device=DEV)
        from types import SimpleNamespace
        cu = torch.tensor([0, 7], dtype=torch.int32, device=DEV)
        mask, depth = ops.tree_mask(par, SimpleNamespace(cu_seqlens_q=cu, num_seqs=1, max_seqlen_q=7))
        ctx, x = forward(tree, depth + start, start, 7, mask)
        # the three nodes on the line see what the single steps saw: bf16 activations, and an 8-bit cache that
        # rounds rows again where they change blocks
        for node, k in ((0, 0), (2, 1), (4, 2)):
            ref = rows[start - 26 + k]
            assert (x[node].float() - ref).abs().max() <= (0.05 if kv == "none" else 0.3) * ref.std()
        one = torch.zeros(1, device=DEV)
        path, n, nxt = ops.verify_tree(x, torch.tensor(tree, dtype=torch.int32, device=DEV), par, ctx, one,
                                       torch.rand(7, device=DEV), one)
        taken = [tree[i] for i in path[0, 1:int(n)].tolist()] + [int(nxt)]
        if kv == "none":
            assert taken == good
        taken = good  # the next tree starts from the line whatever a near tie chose
        path = torch.tensor([[0, 2, 4]], dtype=torch.int32, device=DEV)
        ops.commit_tree(run.kv_cache, ctx, path, torch.tensor([3], dtype=torch.int32, device=DEV), run.kv_scale_cache)
        tokens += taken


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kv", ["none", "fp8"])
def test_whole_steps_of_several_sequences(kv, captured):
    """Masks, forward pass, walk and commit in a row, of three sequences at once, eagerly or as one graph that is replayed
    with new inputs: what each operator leaves is what its plain form makes of what the one before left, and the cache
    behind the last commit is that of the tokens that the steps added."""
    from nanovllm_self_b200 import LLM
    from nanovllm_self_b200.utils.context import Context
    llm = LLM("tiny-gpu", block_size=16, max_model_len=512, num_blocks=64, kv_cache_quant_mode=kv, enforce_eager=True)
    run, ops = llm.model_runner, llm.model_runner.ops
    i32 = dict(dtype=torch.int32, device=DEV)
    ns, B, T = [7, 4, 1], 3, 12
    par = torch.tensor([-1, 0, 0, 1, 2, 2, 4, -1, 0, 1, 2, -1], **i32)
    tables = torch.randperm(48, generator=torch.Generator().manual_seed(1)).int().view(6, 8).to(DEV)  # the last 3: see below
    g = torch.Generator().manual_seed(0)
    lines = [torch.randint(3, 2000, (n,), generator=g).tolist() for n in (27, 40, 5)]

    def slots(row, start, n):
        pos = torch.arange(start, start + n)
        return tables[row].cpu()[pos // 16] * 16 + pos % 16

    def forward(rows, tokens, starts, mask=None, decode=0):
        """New tokens per sequence behind `starts` cached ones, in the blocks of the tables' `rows`."""
        n = [len(t) for t in tokens]
        ctx, _ = make_ctx(n, [s + k for s, k in zip(starts, n)], device=DEV, tables=tables[rows].cpu())
        ctx.num_decode_seqs, ctx.tree_mask = decode, mask
        ctx.slot_mapping = torch.cat([slots(r, s, k) for r, s, k in zip(rows, starts, n)]).int().to(DEV)
        ctx.logits_indices = torch.arange(sum(n), **i32)
        pos = torch.cat([torch.arange(s, s + k) for s, k in zip(starts, n)]).int().to(DEV)
        return run.model.forward(torch.tensor(sum(tokens, []), **i32), pos, ctx, run.kv_layers, run.kv_scale_layers)

    # what single greedy steps of the first sequence choose, to draft from
    for r in range(B):
        forward([r], [lines[r][:-1]], [0])
    good = list(lines[0])
    for _ in range(12):
        good.append(int(forward([0], [[good[-1]]], [len(good) - 1], decode=1)[0].argmax()))
    for r in range(B):
        forward([r], [lines[r][:-1]], [0])

    tokens, u, base = torch.zeros(T, **i32), torch.zeros(T, device=DEV), torch.zeros(T, **i32)
    ud, temps = torch.zeros(B, device=DEV), torch.tensor([0.0, 0.8, 0.9], device=DEV)
    ctx, _ = make_ctx(ns, [64] * B, device=DEV, tables=tables[:B].cpu())
    ctx.slot_mapping, ctx.logits_indices = torch.zeros(T, **i32), torch.arange(T, **i32)

    def pass_through(x):
        ctx.tree_mask = x["mask"]
        return run.model.forward(tokens, base + x["depth"], ctx, run.kv_layers, run.kv_scale_layers)

    def step():
        x = dict(zip(("mask", "depth"), ops.tree_mask(par, ctx)))
        x["logits"] = pass_through(x)
        x["path"], x["length"], x["next"] = ops.verify_tree(x["logits"], tokens, par, ctx, temps, u, ud)
        ops.commit_tree(run.kv_cache, ctx, x["path"], x["length"], run.kv_scale_cache)
        return x

    pool = [t for t in (run.kv_cache, run.kv_scale_cache) if t is not None]
    graph, x = None, None
    lengths = []
    for number in range(4):
        starts = [len(l) - 1 for l in lines]
        nxt = good[starts[0] + 1:starts[0] + 4]
        trees = [[lines[0][-1], nxt[0] ^ 1, nxt[0], 11, nxt[1], nxt[1] ^ 1, 12],
                 [lines[1][-1]] + torch.randint(3, 2000, (3,), generator=g).tolist(), [lines[2][-1]]]
        tokens.copy_(torch.tensor(sum(trees, [])))
        base.copy_(torch.repeat_interleave(torch.tensor(starts), torch.tensor(ns)))
        ctx.host_k_lens = [s + n for s, n in zip(starts, ns)]
        ctx.context_lens.copy_(torch.tensor(ctx.host_k_lens))
        ctx.slot_mapping.copy_(torch.cat([slots(r, s, n) for r, (s, n) in enumerate(zip(starts, ns))]))
        # the second sequence's chain is taken up to node `number`: a child at u = 0 is, at u = 1 - 2^-24 it is not
        u.copy_(torch.rand(T, generator=g))
        u[7:11] = torch.tensor([0.0 if i <= number else 1 - 2.0 ** -24 for i in range(4)])
        ud.copy_(torch.rand(B, generator=g))
        before = [t.clone() for t in pool]
        if not captured:
            x = step()
        else:
            if graph is None:
                step()                      # plans and workspaces
                torch.cuda.synchronize()
                for t, b in zip(pool, before):
                    t.copy_(b)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    x = step()
            graph.replay()
        torch.cuda.synchronize()
        after = [t.clone() for t in pool]
        # each operator by its plain form
        mask, depth = R.tree_mask(par.cpu(), [0, 7, 11, 12], 7)
        assert torch.equal(x["mask"].cpu(), mask) and torch.equal(x["depth"].cpu(), depth)
        for t, b in zip(pool, before):
            t.copy_(b)
        assert torch.equal(pass_through(x), x["logits"])
        path, length, token = R.tree_verify(x["logits"].cpu(), tokens.cpu(), par.cpu(), ns, 7, temps.cpu(), u.cpu(), ud.cpu())
        assert torch.equal(x["path"].cpu(), path) and torch.equal(x["length"].cpu(), length) and torch.equal(x["next"].cpu(), token)
        R.tree_commit(run.kv_cache, ns, ctx.host_k_lens, tables[:B].tolist(), path, length, run.kv_scale_cache)
        for t, a in zip(pool, after):
            assert torch.equal(t.view(torch.uint8) if t.element_size() == 1 else t, a.view(torch.uint8) if a.element_size() == 1 else a)
        lengths.append(length.tolist())
        for b in range(B):
            lines[b] += [trees[b][i] for i in path[b, 1:length[b]].tolist()] + [int(token[b])]
    assert [n[1:] for n in lengths] == [[min(i, 3) + 1, 1] for i in range(4)]
    if kv == "none":
        assert lines[0] == good[:len(lines[0])] and [n[0] for n in lengths] == [3] * 4
    # the next tokens' logits behind the committed cache, and behind a cache that the whole lines are written to at once:
    # bf16 activations, and an 8-bit cache that rounds rows again where they change blocks
    got = forward([0, 1, 2], [[l[-1]] for l in lines], [len(l) - 1 for l in lines], decode=3)
    for b in range(B):
        want = forward([3 + b], [lines[b]], [0])[-1].float()
        assert (got[b].float() - want).abs().max() <= (0.05 if kv == "none" else 0.3) * want.std()

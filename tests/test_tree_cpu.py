"""Trees of drafted tokens on CPU: the plain operators against brute force, a whole step of a model, and refusals."""
import math

import pytest
import torch

from nanovllm_self_b200 import LLM
from nanovllm_self_b200.models.reference import dense_logits, greedy_generate
from nanovllm_self_b200.ops import get_ops, torch_ref as R
from nanovllm_self_b200.utils.context import Context

U32 = 2.0 ** -24  # half a step of fp32, relative


def make_ctx(ns, ks, bs=16, device="cpu", tables=None, W=None):
    """A step's Context for trees of ``ns`` nodes over ``ks`` cached tokens; blocks in falling order."""
    cu = [0]
    for n in ns:
        cu.append(cu[-1] + n)
    per = [max(1, -(-k // bs)) for k in ks]
    W = W or max(per)
    if tables is None:
        tables = torch.zeros(len(ns), W, dtype=torch.int32)
        at = sum(per)
        for b, c in enumerate(per):
            tables[b, :c] = torch.arange(at - 1, at - 1 - c, -1)
            at -= c
    i32 = dict(dtype=torch.int32, device=device)
    return Context(cu_seqlens_q=torch.tensor(cu, **i32), context_lens=torch.tensor(ks, **i32),
                   block_tables=tables.to(device), num_seqs=len(ns), num_tokens=cu[-1], max_seqlen_q=max(ns),
                   max_seqlen_k=max(ks), host_q_lens=list(ns), host_k_lens=list(ks)), sum(per)


def random_parents(ns, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in ns:
        for i in range(n):
            out.append(-1 if i == 0 else i - 1 if torch.rand((), generator=g) < 0.5 else
                       int(torch.randint(0, i, (), generator=g)))
    return torch.tensor(out, dtype=torch.int32)


def ancestors(parents, i):
    out = {i}
    while 0 <= parents[i] < i:
        i = parents[i]
        out.add(i)
    return out


# ------------------------------------------------------------------------------------- masks
@pytest.mark.parametrize("ns", [[1], [5, 1, 3], [64], [65, 2], [256]])
def test_mask_is_the_set_of_ancestors(ns):
    ctx, _ = make_ctx(ns, ns)
    parents = random_parents(ns, sum(ns))
    mask, depth = get_ops("cpu").tree_mask(parents, ctx)
    assert mask.shape == (sum(ns), -(-max(ns) // 64)) and mask.dtype == torch.int64 and depth.dtype == torch.int32
    at = 0
    for n in ns:
        host = parents[at:at + n].tolist()
        for i in range(n):
            want = ancestors(host, i)
            got = {j for j in range(64 * mask.shape[1]) if int(mask[at + i, j // 64]) >> (j % 64) & 1}
            assert got == want and depth[at + i] == len(want) - 1
        at += n


def test_mask_of_nodes_without_a_parent_and_of_rows_behind_the_sequences():
    ctx, _ = make_ctx([4], [4])
    mask, depth = get_ops("cpu").tree_mask(torch.tensor([-1, 7, 2, 1, 0, 0], dtype=torch.int32), ctx)
    assert mask[:, 0].tolist() == [1, 2, 4, 10, 0, 0] and depth.tolist() == [0, 0, 0, 1, 0, 0]


# --------------------------------------------------------------------------------- attention
def attention_oracle(q, k, v, ctx, mask, scale, nkv):
    """64-bit outputs, and the sums of |a v| that errors are relative to, of caches given per sequence."""
    out, size, at = [], [], 0
    for b, n in enumerate(ctx.host_q_lens):
        kl = ctx.host_k_lens[b]
        for r in range(n):
            seen = [p for p in range(kl) if p < kl - n or int(mask[at + r, (p - kl + n) // 64]) >> ((p - kl + n) % 64) & 1]
            for h in range(q.shape[1]):
                kk, vv = k[b][seen, h * nkv // q.shape[1]].double(), v[b][seen, h * nkv // q.shape[1]].double()
                a = torch.softmax(kk @ q[at + r, h].double() * scale, 0)
                out.append(a @ vv if seen else torch.zeros(q.shape[2], dtype=torch.float64))
                size.append(a @ vv.abs() if seen else torch.zeros(q.shape[2], dtype=torch.float64))
        at += n
    return torch.stack(out).view(q.shape), torch.stack(size).view(q.shape)


def test_attention_is_that_of_the_formula():
    torch.manual_seed(0)
    ns, ks, bs, nkv, nq, d = [5, 1, 3], [40, 1, 3], 16, 2, 4, 32
    ctx, nb = make_ctx(ns, ks, bs)
    ops = get_ops("cpu")
    mask, _ = ops.tree_mask(random_parents(ns, 1), ctx)
    mask[2] = 0                                        # sees the context alone
    mask[6] = 0                                        # a whole context of its own tree: sees nothing
    k, v = torch.randn(nb, nkv, bs, d), torch.randn(nb, nkv, bs, d)
    q = torch.randn(sum(ns), nq, d)
    seqs = [[R.gather_kv(c, ctx.block_tables[b].tolist(), ks[b]) for b in range(3)] for c in (k, v)]
    want, size = attention_oracle(q, *seqs, ctx, mask, 0.3, nkv)
    got = ops.attention_tree(q.view(9, -1), k, v, ctx, mask, 0.3).view(9, nq, d)
    # fp32: 40 keys and 32 dims of rounded sums, scores below 30
    assert ((got - want).abs() <= (40 + 2 * (32 + 2) * 30) * U32 * size).all()
    assert (got[6] == 0).all()
    # the caches' own attention agrees where the tree is a line
    line = torch.tensor([-1, 0, 1, 2, 3, -1, -1, 0, 1], dtype=torch.int32)
    got = ops.attention_tree(q.view(9, -1), k, v, ctx, ops.tree_mask(line, ctx)[0], 0.3).view(9, nq, d)
    assert torch.allclose(got, ops.attention(q, k, v, ctx, 0.3), rtol=0, atol=1e-5)


def test_what_a_node_does_not_see_has_no_part_in_it():
    torch.manual_seed(0)
    ctx, nb = make_ctx([4], [20], 16)
    ops = get_ops("cpu")
    mask, _ = ops.tree_mask(torch.tensor([-1, 0, 0, 2], dtype=torch.int32), ctx)
    k, v, q = torch.randn(nb, 1, 16, 32), torch.randn(nb, 1, 16, 32), torch.randn(4, 32)
    want = ops.attention_tree(q, k, v, ctx, mask, 0.2)
    blk = int(ctx.block_tables[0, 1])
    k[blk, 0, 1], v[blk, 0, 1, 3] = float("nan"), float("inf")        # node 1 (position 17)
    k[blk, 0, 4:], v[blk, 0, 4:] = float("nan"), float("nan")         # behind the context
    got = ops.attention_tree(q, k, v, ctx, mask, 0.2)
    assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]]) and got[1].isnan().any()


def test_blocks_outside_of_the_pool_read_as_zeros():
    torch.manual_seed(0)
    ctx, nb = make_ctx([2], [40], 16)
    ops = get_ops("cpu")
    mask, _ = ops.tree_mask(torch.tensor([-1, 0], dtype=torch.int32), ctx)
    k, v, q = torch.randn(nb, 1, 16, 32), torch.randn(nb, 1, 16, 32), torch.randn(2, 32)
    k0, v0 = k.clone(), v.clone()
    for c in (k0, v0):
        c[int(ctx.block_tables[0, 0])] = 0
    want = ops.attention_tree(q, k0, v0, ctx, mask, 0.2)
    for bad in (-1, nb, 1 << 30):
        ctx.block_tables[0, 0] = bad
        assert torch.equal(ops.attention_tree(q, k, v, ctx, mask, 0.2), want)


# ------------------------------------------------------------------------------ verification
def test_walk_keeps_the_target_distribution():
    """Over many random numbers, the first token that a step adds is distributed as the target's probabilities,
    whatever the draft proposes."""
    torch.manual_seed(0)
    v, trials = 6, 20000
    logits = torch.randn(3, v)
    p = torch.softmax(logits[0].double(), 0)
    q = torch.softmax(torch.randn(3, v), -1)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32)
    for draft in (None, q):
        counts = torch.zeros(v)
        kids = torch.multinomial(q[0], 2 * trials, replacement=True).view(trials, 2) if draft is not None else None
        u, ud = torch.rand(trials, 3), torch.rand(trials)
        for i in range(trials // 10 if draft is None else trials // 10):
            tokens = torch.tensor([0, 1, 4]) if kids is None else torch.cat([torch.zeros(1, dtype=torch.long), kids[i]])
            path, n, nxt = R.tree_verify(logits, tokens.int(), parents, [3], 3, torch.ones(1), u[i], ud[i:i + 1], draft)
            counts[int(tokens[path[0, 1]]) if n[0] > 1 else int(nxt[0])] += 1
        got = counts.double() / counts.sum()
        # five standard deviations of a share of 2000 draws
        assert ((got - p).abs() <= 5 * (p * (1 - p) / (trials // 10)).sqrt()).all()


@pytest.mark.parametrize("draft", [True, False])
def test_walk_keeps_the_distribution_of_the_second_token(draft):
    """Behind an accepted child the next token, taken from the tree or drawn, is distributed as the target's
    probabilities behind that child's token."""
    torch.manual_seed(1)
    v, trials = 3, 4000
    first, second = torch.randn(v), torch.randn(v, v)         # the target's logits: of the first token, and behind each
    q0, q1 = torch.softmax(torch.randn(v), 0), torch.softmax(torch.randn(v, v), -1)
    parents = torch.tensor([-1, 0, 1], dtype=torch.int32)
    counts = torch.zeros(v, v)
    for _ in range(trials):
        x = int(torch.multinomial(q0, 1)) if draft else int(torch.randint(0, v, ()))
        y = int(torch.multinomial(q1[x], 1)) if draft else 1
        path, n, nxt = R.tree_verify(torch.stack([first, second[x], second[x]]), torch.tensor([0, x, y], dtype=torch.int32),
                                     parents, [3], 3, torch.ones(1), torch.rand(3), torch.rand(1),
                                     torch.stack([q0, q1[x], q1[x]]) if draft else None)
        if n[0] > 1:
            counts[x, y if n[0] > 2 else int(nxt[0])] += 1
    for x in range(v):
        p, k = torch.softmax(second[x].double(), 0), float(counts[x].sum())
        assert k > 200
        # five standard deviations of a share of k draws
        assert ((counts[x].double() / k - p).abs() <= 5 * (p * (1 - p) / k).sqrt()).all()


def test_greedy_walk_follows_the_first_maximum():
    logits = torch.tensor([[0.0, 2, 2, 1], [5, 0, 0, 0], [0, 0, 0, 9], [0, 0, 7, 7]])
    parents = torch.tensor([-1, 0, 0, 2], dtype=torch.int32)
    tokens = torch.tensor([3, 2, 1, 3], dtype=torch.int32)
    path, n, nxt = R.tree_verify(logits, tokens, parents, [4], 4, torch.zeros(1), torch.rand(4), torch.rand(1))
    assert path[0].tolist() == [0, 2, 3, -1] and n[0] == 3 and nxt[0] == 2


def test_walk_at_the_borders():
    inf = float("inf")
    logits = torch.tensor([[0.0, math.log(3.0), -inf, float("nan")], [-inf] * 4, [0.0, inf, -inf, inf]])
    one = torch.ones(1)

    def step(row, token, u, ud):
        path, n, nxt = R.tree_verify(logits[[row, 0]], torch.tensor([0, token], dtype=torch.int32),
                                     torch.tensor([-1, 0], dtype=torch.int32), [2], 2, one, torch.tensor([0.0, u]),
                                     torch.tensor([ud]))
        return int(n[0]), int(nxt[0])

    assert step(0, 1, 0.7499, 0.0)[0] == 2 and step(0, 1, 0.7501, 0.0) == (1, 0)   # p = 3/4
    assert step(0, 0, 0.9, 0.0) == (1, 1)                                           # 1/4: the rest is all of p
    assert step(0, 2, 0.0, 0.2499) == (1, 0) and step(0, 3, 0.0, 0.2501) == (1, 1)  # no weight
    assert step(0, 4, 0.0, 1.0) == (1, 1) and step(0, -1, 0.0, -3.0) == (1, 0)      # no such token; clamped
    assert step(0, 2, 0.5, float("nan")) == (1, 0)
    assert step(1, 1, 0.0, 0.5) == (1, 0)                                           # nothing above -inf
    assert step(2, 1, 0.499, 0.5)[0] == 2 and step(2, 1, 0.501, 0.5) == (1, 3)      # two infinities share it


# ------------------------------------------------------------------------------------ commit
@pytest.mark.parametrize("dtype", [torch.float32, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("bs", [4, 16])
def test_commit_gives_what_storing_in_order_gives(dtype, bs):
    torch.manual_seed(0)
    ns, ks = [7, 3, 5], [9, 35, 21]
    ctx, nb = make_ctx(ns, ks, bs)
    shape = (2, 2, nb, 2, bs, 32)
    pool = torch.randn(shape) if dtype == torch.float32 else torch.randint(-40, 40, shape).to(dtype)
    scale = None
    if dtype != torch.float32:
        scale = torch.rand(shape[:4] if dtype == torch.float8_e4m3fn else shape[:5]) + 0.5
    path = torch.tensor([[0, 2, 3, 6, -1], [0, -1, -1, -1, -1], [0, 1, 4, 4, 2]], dtype=torch.int32)
    lengths = torch.tensor([4, 1, 5], dtype=torch.int32)

    def values(pool, scale, b, pos):
        blk, off = int(ctx.block_tables[b, pos // bs]), pos % bs
        x = pool[:, :, blk, :, off].float()
        return x if scale is None else x * (scale[:, :, blk] if scale.dim() == 4 else scale[:, :, blk, :, off])[..., None]

    before = [[values(pool, scale, b, p) for p in range(k)] for b, k in enumerate(ks)]
    new, sc = pool.clone(), None if scale is None else scale.clone()
    get_ops("cpu").commit_tree(new, ctx, path, lengths, sc)
    for b, nodes in enumerate([[0, 2, 3, 6], [0], [0, 1, 4]]):  # a path ends where it stops to increase
        base = ks[b] - ns[b]
        for p in range(base + len(nodes)):
            want = before[b][p if p < base else base + nodes[p - base]]
            got = values(new, sc, b, p)
            if dtype == torch.float8_e4m3fn:
                # rounded at most once more: half a step of e4m3, 2^-10 of the scale at the least
                s = sc[:, :, int(ctx.block_tables[b, p // bs])][..., None]
                assert ((got - want).abs() <= want.abs() * (2.0 ** -4 + 2 * U32) + s * 2.0 ** -10).all()
            else:
                assert torch.equal(got, want)


# ------------------------------------------------------------------------- a step of a model
def _tree_step(llm, prompt, tokens, parents):
    """Runs a tree behind a cached prompt through the model; (ctx, logits)."""
    run = llm.model_runner
    n, kl, bs = len(tokens), len(prompt) - 1 + len(tokens), run.block_size
    ctx, _ = make_ctx([n], [kl], bs, tables=torch.arange(run.max_blocks_per_seq, dtype=torch.int32)[None])
    par = torch.tensor(parents, dtype=torch.int32)
    ctx.tree_mask, depth = run.ops.tree_mask(par, ctx)
    ctx.slot_mapping = torch.arange(kl - n, kl, dtype=torch.int32)
    ctx.logits_indices = torch.arange(n, dtype=torch.int32)
    logits = run.model.forward(torch.tensor(tokens, dtype=torch.int32), depth + (kl - n), ctx, run.kv_layers,
                               run.kv_scale_layers)
    return ctx, par, logits


def _prefill(llm, tokens):
    run = llm.model_runner
    n = len(tokens)
    ctx, _ = make_ctx([n], [n], run.block_size, tables=torch.arange(run.max_blocks_per_seq, dtype=torch.int32)[None])
    ctx.slot_mapping = torch.arange(n, dtype=torch.int32)
    ctx.logits_indices = torch.tensor([n - 1], dtype=torch.int32)
    return run.model.forward(torch.tensor(tokens, dtype=torch.int32), torch.arange(n, dtype=torch.int32), ctx,
                             run.kv_layers, run.kv_scale_layers)


def test_steps_of_drafted_trees_generate_what_greedy_decoding_does():
    llm = LLM("tiny", device="cpu", dtype="fp32", block_size=16, max_model_len=256, num_blocks=32)
    prompt = torch.randint(3, 1000, (29,), generator=torch.Generator().manual_seed(3)).tolist()
    want = greedy_generate(llm.model_runner.model, prompt, 12)
    _prefill(llm, prompt[:-1])
    tokens, ops = list(prompt), llm.model_runner.ops
    lengths = []
    while len(tokens) < len(prompt) + 9:
        done = len(tokens) - len(prompt)
        # two right guesses behind a wrong branch, and wrong leaves
        nxt = want[done:done + 3]
        tree = [tokens[-1], nxt[0] ^ 1, nxt[0], 5, nxt[1], nxt[1] ^ 1, 7]
        parents = [-1, 0, 0, 1, 2, 2, 4]
        ctx, par, logits = _tree_step(llm, tokens, tree, parents)
        path, n, nxt_tok = ops.verify_tree(logits, torch.tensor(tree, dtype=torch.int32), par, ctx, torch.zeros(1),
                                           torch.rand(7), torch.rand(1))
        ops.commit_tree(llm.model_runner.kv_cache, ctx, path, n, llm.model_runner.kv_scale_cache)
        lengths.append(int(n[0]))
        tokens += [tree[i] for i in path[0, 1:n[0]].tolist()] + [int(nxt_tok[0])]
        # the logits of an accepted node are those of its own line of tokens
        line = tokens[:len(tokens) - 1]
        assert torch.allclose(logits[path[0, n[0] - 1]], dense_logits(llm.model_runner.model, line), atol=1e-3)
    assert tokens[len(prompt):] == want[:len(tokens) - len(prompt)] and lengths == [3, 3, 3]


# ---------------------------------------------------------------------------------- refusals
def test_the_plain_operators_refuse_bad_sizes():
    ops = get_ops("cpu")
    ctx, _ = make_ctx([257], [257])
    parents = torch.zeros(257, dtype=torch.int32)
    with pytest.raises(ValueError, match="256 nodes"):
        ops.tree_mask(parents, ctx)
    ctx, nb = make_ctx([65], [65])
    q, kv = torch.randn(65, 32), torch.randn(nb, 1, 16, 32)
    for mask in (torch.zeros(65, 1, dtype=torch.int64), torch.zeros(65, 2, dtype=torch.int32),
                 torch.zeros(64, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="mask"):
            ops.attention_tree(q, kv, kv, ctx, mask, 1.0)


def _refused(f, *args, **kw):
    with pytest.raises(RuntimeError) as e:
        f(*args, **kw)
    return str(e.value)


def test_the_kernels_refuse_bad_arguments():
    from nanovllm_self_b200.ops._ext import available, load
    if not available():
        pytest.skip("extension not built")
    C = load()
    i32 = dict(dtype=torch.int32)
    ctx, nb = make_ctx([3, 2], [40, 20])
    par, cu = torch.zeros(5, **i32), ctx.cu_seqlens_q
    assert "nodes" in _refused(C.tree_mask, par, cu, 2, 257) and "nodes" in _refused(C.tree_mask, par, cu, 2, 0)
    assert "cu_seqlens_q" in _refused(C.tree_mask, par, cu, 3, 3)
    assert "cu_seqlens_q" in _refused(C.tree_mask, par, cu.long(), 2, 3)
    assert "parents" in _refused(C.tree_mask, par.long(), cu, 2, 3)
    assert "CUDA" in _refused(C.tree_mask, par, cu, 2, 3)

    def attend(**kw):
        a = dict(q=torch.zeros(5, 512, dtype=torch.bfloat16), k=torch.zeros(nb, 2, 16, 128, dtype=torch.bfloat16),
                 v=None, ks=None, vs=None, mask=torch.zeros(5, 1, dtype=torch.int64), bt=ctx.block_tables, cu=cu,
                 lens=ctx.context_lens, n=2, m=3)
        a.update(kw)
        a["v"] = a["k"] if a["v"] is None else a["v"]
        return _refused(C.tree_attention, a["q"], a["k"], a["v"], a["ks"], a["vs"], a["mask"], a["bt"], a["cu"],
                        a["lens"], a["n"], a["m"], 1.0)

    bf16, f8 = dict(dtype=torch.bfloat16), dict(dtype=torch.float8_e4m3fn)
    assert "CUDA" in attend()
    assert "bfloat16" in attend(q=torch.zeros(5, 512)) and "cache" in attend(k=torch.zeros(nb, 2, 16, 128))
    assert "one type" in attend(v=torch.zeros(nb, 2, 32, 128, **bf16))
    assert "head dim" in attend(k=torch.zeros(nb, 2, 16, 64, **bf16))
    for bs in (8, 48):
        assert "power of two" in attend(k=torch.zeros(nb, 2, bs, 128, **bf16))
    assert "query heads" in attend(q=torch.zeros(5, 384, **bf16)) and "heads" in attend(q=torch.zeros(5, 500, **bf16))
    assert "contiguous" in attend(q=torch.zeros(512, 5, **bf16).t())
    assert "mask" in attend(mask=torch.zeros(5, 1, **i32)) and "mask" in attend(mask=torch.zeros(4, 1, dtype=torch.int64))
    assert "mask" in attend(m=65) and "nodes" in attend(m=300)
    assert "block_tables" in attend(bt=ctx.block_tables[:1]) and "context_lens" in attend(lens=ctx.context_lens[:1])
    assert "context_lens" in attend(lens=ctx.context_lens.long())
    k8, s = torch.zeros(nb, 2, 16, 128, **f8), torch.ones(nb, 2)
    assert "scales" in attend(k=k8) and "scales" in attend(k=k8, ks=s, vs=s[:1]) and "CUDA" in attend(k=k8, ks=s, vs=s)

    def verify(**kw):
        a = dict(logits=torch.zeros(5, 50), tokens=par, parents=par, cu=cu, temps=torch.ones(2), u=torch.rand(5),
                 ud=torch.rand(2), draft=None, n=2, m=3)
        a.update(kw)
        return _refused(C.tree_verify, *a.values())

    assert "CUDA" in verify() and "CUDA" in verify(draft=torch.zeros(5, 50))
    assert "logits" in verify(logits=torch.zeros(5, 50).half()) and "logits" in verify(logits=torch.zeros(50, 5).t())
    assert "tokens" in verify(tokens=par[:4]) and "parents" in verify(parents=par.long())
    assert "temperatures" in verify(temps=torch.ones(3)) and "uniforms" in verify(u=torch.rand(5).double())
    assert "draw_uniforms" in verify(ud=torch.rand(1)) and "draft_probs" in verify(draft=torch.zeros(5, 51))
    assert "draft_probs" in verify(draft=torch.zeros(5, 50).bfloat16()) and "nodes" in verify(m=257)
    assert "4194303" in verify(logits=torch.empty(5, 1 << 22, dtype=torch.bfloat16))

    def commit(**kw):
        a = dict(kv=torch.zeros(2, 3, nb, 2, 16, 128, **bf16), path=torch.zeros(2, 3, **i32),
                 length=torch.ones(2, **i32), bt=ctx.block_tables, cu=cu, lens=ctx.context_lens, scale=None, n=2, m=3)
        a.update(kw)
        return _refused(C.tree_commit, *a.values())

    assert "CUDA" in commit()
    assert "cache" in commit(kv=torch.zeros(3, nb, 2, 16, 128, **bf16)) and "cache" in commit(kv=torch.zeros(2, 3, nb, 2, 16, 128))
    assert "head dim" in commit(kv=torch.zeros(2, 3, nb, 2, 16, 64, **bf16))
    assert "contiguous" in commit(kv=torch.zeros(2, 3, nb, 2, 128, 16, **bf16).transpose(4, 5))
    assert "path" in commit(path=torch.zeros(3, 3, **i32)) and "lengths" in commit(length=torch.ones(1, **i32))
    kv8 = torch.zeros(2, 3, nb, 2, 16, 128, **f8)
    assert "scales" in commit(kv=kv8) and "scales" in commit(kv=kv8, scale=torch.ones(2, 3, nb, 1))
    assert "CUDA" in commit(kv=kv8, scale=torch.ones(2, 3, nb, 2))


def test_an_expired_wait_of_a_tree_ends_the_engines_step(monkeypatch):
    from nanovllm_self_b200 import SamplingParams
    llm = LLM("tiny", device="cpu", dtype="fp32", block_size=16, max_model_len=128, num_blocks=16, weight_quant_mode="fp8")
    monkeypatch.setattr(llm.model_runner.ops, "device_error", lambda: 613)
    with pytest.raises(RuntimeError, match="a kernel gave up on a bounded wait .code 613"):
        llm.generate([[1, 2, 3]], SamplingParams(temperature=0, max_tokens=2, ignore_eos=True))

"""Plain-PyTorch implementations of every hot op.

These run the tiny CPU model (fp32) and are the numerics oracle for the CUDA kernels
(each GPU kernel test compares against these evaluated in fp32).  They mirror the
reference's eager semantics:

* RMSNorm in fp32, cast back (``nanovllm/layers/RMSNorm.py:11-17``);
* NeoX rotate-half RoPE in fp32 with a ``[max_pos, D]`` cos‖sin table
  (``nanovllm/layers/RoPE.py:5-55``);
* KV store by slot ``block * BS + offset`` (``nanovllm/layers/attention.py:139-189``),
  with the cache laid out ``[num_blocks, kv_heads, block_size, head_dim]`` per layer;
* causal attention whose mask is offset by ``k_len - q_len`` so that a chunk or a
  prefix-hit prefill sees all cached tokens (``attention.py:378-498``);
* sampler: greedy for temperature <= 0, else softmax(logits / T) sampling, with an
  optional top-p filter (``nanovllm/layers/sampler.py:9-43``).
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

FP8_MAX = 448.0
FP8_HEADROOM = 4.0


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * r * w.float()).to(x.dtype)


def add_rmsnorm(x: torch.Tensor, residual: torch.Tensor | None, w: torch.Tensor, eps: float):
    """residual' = x + residual (or x); returns (rmsnorm(residual'), residual')."""
    r = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    return rmsnorm(r, w, eps), r


def rope_cos_sin(head_dim: int, max_pos: int, theta: float, device=None) -> torch.Tensor:
    """fp32 table [max_pos, head_dim]: first half cos, second half sin."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    t = torch.arange(max_pos, dtype=torch.float64)
    f = torch.outer(t, inv)
    return torch.cat([f.cos(), f.sin()], dim=-1).float().to(device)


def apply_rope(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor) -> torch.Tensor:
    """x [T, H, D] rotated by the NeoX rule at ``positions`` [T]."""
    d2 = x.shape[-1] // 2
    cs = cos_sin[positions.long()]
    cos, sin = cs[:, None, :d2], cs[:, None, d2:]
    x1, x2 = x.float()[..., :d2], x.float()[..., d2:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(x.dtype)


def fp8_block_scale(first_token_absmax: torch.Tensor) -> torch.Tensor:
    return torch.clamp(first_token_absmax.float() * FP8_HEADROOM / FP8_MAX, min=1e-8)


def store_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             slot_mapping: torch.Tensor, k_scale: torch.Tensor | None = None,
             v_scale: torch.Tensor | None = None) -> None:
    """Scatter k, v [T, Hkv, D] into caches [NB, Hkv, BS, D] at ``slot_mapping`` [T].

    Negative slots are skipped (padding rows).  For fp8 caches the per-(block, head)
    scale is set by the step that writes the block's first token: absmax of that token
    times a headroom of 4, divided by 448; later tokens in the block reuse it.
    """
    bs = k_cache.shape[2]
    slots = slot_mapping.long()
    keep = slots >= 0
    if not bool(keep.all()):
        k, v, slots = k[keep], v[keep], slots[keep]
    blk, off = slots // bs, slots % bs
    if k_cache.dtype == torch.float8_e4m3fn:
        for cache, x, sc in ((k_cache, k, k_scale), (v_cache, v, v_scale)):
            first = off == 0
            if bool(first.any()):
                amax = x[first].float().abs().amax(dim=-1)  # [n_first, Hkv]
                sc[blk[first]] = fp8_block_scale(amax)
            s = sc[blk]  # [T, Hkv]
            q = torch.clamp(x.float() / s[..., None], -FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
            cache[blk, :, off] = q
    elif k_cache.dtype == torch.int8:
        for cache, x, sc in ((k_cache, k, k_scale), (v_cache, v, v_scale)):
            amax = x.float().abs().amax(dim=-1)
            s = torch.clamp(amax / 127.0, min=1e-6)
            qv = torch.clamp(torch.round(x.float() / s[..., None]), -127, 127).to(torch.int8)
            cache[blk, :, off] = qv
            sc[blk, :, off] = s
    else:
        k_cache[blk, :, off] = k.to(k_cache.dtype)
        v_cache[blk, :, off] = v.to(v_cache.dtype)


def gather_kv(cache: torch.Tensor, block_table, k_len: int, scale: torch.Tensor | None = None) -> torch.Tensor:
    """Return [k_len, Hkv, D] fp32 for one sequence."""
    bs = cache.shape[2]
    nb = (k_len + bs - 1) // bs
    ids = torch.as_tensor(list(block_table[:nb]), dtype=torch.long, device=cache.device)
    x = cache[ids].float()  # [nb, Hkv, BS, D]
    if cache.dtype == torch.float8_e4m3fn:
        x = x * scale[ids][:, :, None, None].float()
    elif cache.dtype == torch.int8:
        x = x * scale[ids][..., None].float()
    return x.permute(0, 2, 1, 3).reshape(nb * bs, x.shape[1], x.shape[3])[:k_len]


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    q_lens: list, k_lens: list, block_tables: list, scale: float,
                    k_scale=None, v_scale=None) -> torch.Tensor:
    """q [T, Hq, D] (sequences packed in order) -> out [T, Hq, D]."""
    out = torch.empty_like(q)
    hq, hkv = q.shape[1], k_cache.shape[1]
    g = hq // hkv
    t0 = 0
    for i, (ql, kl) in enumerate(zip(q_lens, k_lens)):
        if ql == 0:
            continue
        qi = q[t0:t0 + ql].float()  # [ql, Hq, D]
        k = gather_kv(k_cache, block_tables[i], kl, k_scale).repeat_interleave(g, dim=1)
        v = gather_kv(v_cache, block_tables[i], kl, v_scale).repeat_interleave(g, dim=1)
        s = torch.einsum("qhd,khd->hqk", qi, k) * scale
        qpos = torch.arange(ql, device=q.device)[:, None] + (kl - ql)
        kpos = torch.arange(kl, device=q.device)[None, :]
        s = s.masked_fill((kpos > qpos)[None], float("-inf"))
        p = torch.softmax(s, dim=-1)
        out[t0:t0 + ql] = torch.einsum("hqk,khd->qhd", p, v).to(q.dtype)
        t0 += ql
    return out


def silu_mul(x: torch.Tensor) -> torch.Tensor:
    """x [T, 2I] = gate ‖ up -> silu(gate) * up [T, I]."""
    i = x.shape[-1] // 2
    g, u = x[..., :i].float(), x[..., i:].float()
    return (F.silu(g) * u).to(x.dtype)


GATE_UP_GROUP = 16


def interleave_gate_up(g: torch.Tensor, u: torch.Tensor, group: int = GATE_UP_GROUP) -> torch.Tensor:
    """[I, H] gate and up weights -> [2I, H] with rows interleaved in groups of ``group``:
    rows 2·group·j .. +group-1 are gate features group·j.., the next ``group`` rows the
    matching up features.  Every tile of 32 output columns of ``x @ W^T`` then holds 16
    gates and their 16 ups, which lets the GEMM apply SiLU-and-mul in its epilogue."""
    i, h = g.shape
    if i % group:
        raise ValueError(f"intermediate size {i} is not a multiple of {group}")
    return torch.stack([g.reshape(i // group, group, h), u.reshape(i // group, group, h)], 1).reshape(2 * i, h)


def silu_mul_interleaved(y: torch.Tensor, group: int = GATE_UP_GROUP) -> torch.Tensor:
    """y [T, 2I] in the interleaved layout of :func:`interleave_gate_up` -> silu(gate) * up [T, I]."""
    t, n = y.shape
    y = y.float().reshape(t, n // (2 * group), 2, group)
    return (F.silu(y[:, :, 0]) * y[:, :, 1]).reshape(t, n // 2)


def linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return F.linear(x, w)


FP8_GROUP = 128        # channels of one activation scale; side of one weight scale's block
FP8_AMAX_MIN = 1e-30


def _fp8_scale(a: torch.Tensor):
    """(scale, its inverse) of groups with largest magnitude ``a`` (fp32)."""
    a = a.clamp(min=FP8_AMAX_MIN)
    m = torch.full_like(a, FP8_MAX)  # a tensor: IEEE divisions, no multiplication by a reciprocal
    return a / m, m / a


def quant_fp8(x: torch.Tensor):
    """x [T, K] -> (q [T, K] e4m3, s [T, ceil(K / 128)] fp32), x ~ q * s per group of 128 channels:
    s = max |x| / 448 (at least 1e-30 / 448), q = e4m3(x * (448 / max |x|)), saturating."""
    t, k = x.shape
    kb = -(-k // FP8_GROUP)
    p = x.new_zeros(t, kb * FP8_GROUP, dtype=torch.float32)
    p[:, :k] = x
    p = p.view(t, kb, FP8_GROUP)
    s, inv = _fp8_scale(p.abs().amax(-1))
    q = torch.clamp(p * inv[..., None], -FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q.view(t, kb * FP8_GROUP)[:, :k].contiguous(), s


def dequant_fp8(q: torch.Tensor, s: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    return q.to(dtype) * s.to(dtype).repeat_interleave(FP8_GROUP, 1)[:, :q.shape[1]]


def quant_fp8_weight(w: torch.Tensor):
    """w [N, K] -> (q [N, K] e4m3, s [ceil(N / 128), ceil(K / 128)] fp32): one scale per block of
    128 x 128, by the rule of :func:`quant_fp8`."""
    n, k = w.shape
    g = FP8_GROUP
    nb, kb = -(-n // g), -(-k // g)
    p = w.new_zeros(nb * g, kb * g, dtype=torch.float32)
    p[:n, :k] = w
    p = p.view(nb, g, kb, g)
    s, inv = _fp8_scale(p.abs().amax(dim=(1, 3)))
    q = torch.clamp(p * inv[:, None, :, None], -FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q.view(nb * g, kb * g)[:n, :k].contiguous(), s


def dequant_fp8_weight(q: torch.Tensor, s: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    g = FP8_GROUP
    s = s.to(dtype).repeat_interleave(g, 0)[:q.shape[0]].repeat_interleave(g, 1)[:, :q.shape[1]]
    return q.to(dtype) * s


def group_gate_up(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    """[I, H] gate and up weights -> [2 * 128 * ceil(I / 128), H]: blocks of 128 gate rows and the
    128 matching up rows in turn, the last pair of blocks filled up with zero rows.  No block of
    128 x 128 then mixes gate and up rows, and 256 output columns are one group of 128 of
    silu(gate) * up."""
    i, h = g.shape
    b = -(-i // FP8_GROUP)
    out = g.new_zeros(b, 2, FP8_GROUP, h)
    for j, x in enumerate((g, u)):
        p = g.new_zeros(b * FP8_GROUP, h)
        p[:i] = x
        out[:, j] = p.view(b, FP8_GROUP, h)
    return out.view(2 * b * FP8_GROUP, h)


def linear_fp8(x, w) -> torch.Tensor:
    """x and w as (values, scales) -> fp32 x @ w^T."""
    return F.linear(dequant_fp8(*x), dequant_fp8_weight(*w))


def linear_silu_fp8(x, w, features: int):
    """silu(gate) * up of x @ w^T, quantised; w in the layout of :func:`group_gate_up`."""
    y = linear_fp8(x, w)
    y = y.view(y.shape[0], -1, 2, FP8_GROUP)
    h = (F.silu(y[:, :, 0]) * y[:, :, 1]).reshape(y.shape[0], -1)
    return quant_fp8(h[:, :features])


def embedding(ids: torch.Tensor, w: torch.Tensor, vocab_start: int = 0) -> torch.Tensor:
    """Rows of the (possibly vocab-sharded) table; ids outside the shard give zeros."""
    local = ids.long() - vocab_start
    ok = (local >= 0) & (local < w.shape[0])
    out = w[torch.where(ok, local, torch.zeros_like(local))]
    return out * ok[:, None].to(out.dtype)


def sample(logits: torch.Tensor, temperatures: torch.Tensor, top_p: torch.Tensor | None = None,
           generator: torch.Generator | None = None, batch_greedy_compat: bool = False) -> torch.Tensor:
    """Per-row: argmax if T <= 0 else sample softmax(logits / T) restricted to top-p."""
    logits = logits.float()
    greedy = logits.argmax(dim=-1)
    t = temperatures.float()
    if batch_greedy_compat and bool((t <= 0).any()):
        return greedy
    if bool((t <= 0).all()):
        return greedy
    probs = torch.softmax(logits / torch.where(t > 0, t, torch.ones_like(t))[:, None], dim=-1)
    if top_p is not None and bool((top_p < 1.0).any()):
        sp, si = probs.sort(dim=-1, descending=True)
        cum = sp.cumsum(-1)
        drop = (cum - sp) > top_p[:, None].float()
        sp = sp.masked_fill(drop, 0.0)
        probs = torch.zeros_like(probs).scatter_(-1, si, sp)
    drawn = torch.multinomial(probs, 1, generator=generator).squeeze(-1)
    return torch.where(t > 0, drawn, greedy)


# ------------------------------------------------------------------ trees of drafted tokens
# A step that checks drafted tokens gives each sequence the nodes of a tree as its new tokens: node 0 is the
# root (the last token that is known), ``parents`` holds each node's parent by its index within the tree, which
# lies below the node's own, and node i's K/V lies at position context_len - nodes + i.  A node whose parent is no
# index below its own has none.
TREE_MAX_NODES = 256


def tree_words(max_nodes: int) -> int:
    """Words of a mask row for trees of up to ``max_nodes`` nodes (bit j % 64 of word j / 64 is node j)."""
    if not 1 <= max_nodes <= TREE_MAX_NODES:
        raise ValueError(f"trees have 1 to {TREE_MAX_NODES} nodes, got max_seqlen_q = {max_nodes}")
    return -(-max_nodes // 64)


def tree_mask(parents: torch.Tensor, cu_q: list, max_nodes: int):
    """(mask int64 [T, words]: the ancestors of each node and itself; depth int32 [T]: how many ancestors)."""
    words, t = tree_words(max_nodes), parents.shape[0]
    mask = torch.zeros(t, words, dtype=torch.int64)
    depth = torch.zeros(t, dtype=torch.int32)
    host = parents.tolist()
    for t0, t1 in zip(cu_q[:-1], cu_q[1:]):
        see: list[int] = []
        for i in range(min(t1 - t0, max_nodes)):
            p = host[t0 + i]
            see.append((see[p] if 0 <= p < i else 0) | 1 << i)
            for w in range(words):
                x = see[i] >> 64 * w & (1 << 64) - 1
                mask[t0 + i, w] = x - (1 << 64) if x >> 63 else x
            depth[t0 + i] = bin(see[i]).count("1") - 1
    return mask.to(parents.device), depth.to(parents.device)


def _gather_pages(cache: torch.Tensor, table: list, k_len: int, scale: torch.Tensor | None) -> torch.Tensor:
    """``gather_kv`` with blocks outside of the pool or of the table read as zeros."""
    nb = -(-k_len // cache.shape[2])
    ids = (list(table) + [-1] * nb)[:nb]
    ok = torch.tensor([0 <= i < cache.shape[0] for i in ids], device=cache.device)
    x = gather_kv(cache, [i if 0 <= i < cache.shape[0] else 0 for i in ids], k_len, scale)
    return torch.where(ok.repeat_interleave(cache.shape[2])[:k_len, None, None], x, 0.0)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, q_lens: list, k_lens: list,
                   block_tables: list, mask: torch.Tensor, scale: float, k_scale=None, v_scale=None) -> torch.Tensor:
    """q [T, Hq, D] (each sequence's tree nodes) -> out [T, Hq, D]: node r sees the positions before the tree and
    the nodes of its mask; a node that sees nothing gives zeros, and what a node does not see has no part in it,
    an infinity or a NaN included."""
    out = torch.zeros_like(q)
    g = q.shape[1] // k_cache.shape[1]
    t0 = 0
    for b, (n, kl) in enumerate(zip(q_lens, k_lens)):
        if n and kl > 0:
            k = _gather_pages(k_cache, block_tables[b], kl, k_scale).repeat_interleave(g, dim=1)
            v = _gather_pages(v_cache, block_tables[b], kl, v_scale).repeat_interleave(g, dim=1)
            j = torch.arange(kl, device=q.device) - (kl - n)
            word = mask[t0:t0 + n][:, (j // 64).clamp(0, mask.shape[1] - 1)]
            see = (j < 0) | ((word >> (j % 64) & 1 == 1) & (j < 64 * mask.shape[1]))     # [n, kl]
            s = torch.einsum("qhd,khd->hqk", q[t0:t0 + n].to(k.dtype), k) * scale
            s = s.masked_fill(~see, float("-inf"))
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m.masked_fill(m == float("-inf"), 0.0))
            z = p.sum(-1, keepdim=True)
            p = p / torch.where(z == 0, 1.0, z)
            fine = torch.isfinite(v)
            o = torch.einsum("hqk,khd->qhd", p, torch.where(fine, v, 0.0))
            for i in torch.nonzero(~fine.all(-1).all(-1)).flatten().tolist():
                part = p[:, :, i].t()[..., None] * torch.where(fine[i], 0.0, v[i])
                o = o + torch.where(see[:, i, None, None], part, 0.0)
            out[t0:t0 + n] = o.to(q.dtype)
        t0 += n
    return out


def _tree_probs(row: torch.Tensor, temperature: float) -> torch.Tensor:
    """float64 probabilities of a row of logits; all zero where no logit is above -inf (a NaN counts as -inf; less than
    2^-900 of the largest as nothing).  A temperature that is not above 0 puts all of it on the first maximum."""
    z = row.double()
    z = torch.where(torch.isnan(z), float("-inf"), z)
    top = z.max()
    if top == float("-inf"):
        return torch.zeros_like(z)
    if not temperature > 0:
        p = torch.zeros_like(z)
        p[int((z == top).int().argmax())] = 1.0
        return p
    w = (z == top).double() if top == float("inf") else torch.exp((z - top) / temperature)
    w = torch.where(w < 2.0 ** -900, 0.0, w)
    return w / w.sum()


def tree_verify(logits, tokens, parents, q_lens: list, max_nodes: int, temperatures, uniforms, draw_uniforms,
                draft_probs=None):
    """(path int32 [B, max_nodes], length int32 [B], next token int32 [B]) by the walk through each tree.

    At a node with the target's probabilities p = softmax(logits / temperature), its children are tried in order.
    Child c with token x is taken if ``uniforms[c] * q(x) < p(x)``, and the walk goes on there; else p becomes
    ``max(p - q, 0)`` over its sum (p stays where that is nothing), and the next child is tried.  q is the node's
    row of ``draft_probs``, from which its children were drawn independently, or, without them, 1 at x alone (p
    loses x).  Behind the last child the next token is drawn from p: the first x whose cumulative sum is
    above ``draw_uniforms[b]`` times the total.  At temperatures of 0 and below, a child is taken if its
    token is the first maximum of the logits, which is the next token too.

    ``path`` holds the nodes of the walk, the root first, then -1; ``length`` counts them: the tokens that the step
    adds are those of path[1:] and the next one.  Without any logit above -inf the next token is 0; a sequence
    without nodes has length 0 and next token -1."""
    tree_words(max_nodes)
    b, v = len(q_lens), logits.shape[1]
    path = torch.full((b, max_nodes), -1, dtype=torch.int32)
    length = torch.zeros(b, dtype=torch.int32)
    draws = torch.full((b,), -1, dtype=torch.int32)
    par, tok, u = parents.tolist(), tokens.tolist(), uniforms.double().tolist()
    t0 = 0
    for i, n in enumerate(q_lens):
        n, step = min(n, max_nodes), n
        temperature, node, walk = float(temperatures[i]), 0, [0]
        while n:
            p = _tree_probs(logits[t0 + node], temperature)
            greedy, q = not temperature > 0, None
            if draft_probs is not None and not greedy:
                q = draft_probs[t0 + node].double()
                q = torch.where(q > 0, q, 0.0)
            took = None
            for c in (c for c in range(node + 1, n) if par[t0 + c] == node):
                x = tok[t0 + c]
                if not 0 <= x < v:
                    took_it = False
                elif greedy:
                    took_it = float(p[x]) > 0
                else:
                    took_it = u[t0 + c] * (1.0 if q is None else float(q[x])) < float(p[x])
                if took_it:
                    took = c
                    break
                if greedy:
                    continue
                if q is None:
                    r = p.clone()
                    if 0 <= x < v:
                        r[x] = 0.0
                else:
                    r = (p - q).clamp(min=0.0)
                if float(r.sum()) > 0:
                    p = r / r.sum()
            if took is None:
                break
            node = took
            walk.append(node)
        if n:
            total = p.cumsum(0)
            share = min(max(float(draw_uniforms[i].nan_to_num(0.0)), 0.0), 1.0)
            above = torch.nonzero(total > share * total[-1]).flatten()
            held = torch.nonzero(p > 0).flatten()
            draws[i] = int(above[0]) if len(above) else int(held[-1]) if len(held) else 0
            path[i, :len(walk)] = torch.tensor(walk, dtype=torch.int32)
            length[i] = len(walk)
        t0 += step
    return tuple(x.to(logits.device) for x in (path, length, draws))


def tree_commit(kv_cache: torch.Tensor, q_lens: list, k_lens: list, block_tables: list, path: torch.Tensor,
                lengths: torch.Tensor, kv_scale_cache: torch.Tensor | None = None) -> None:
    """Moves the K/V of each sequence's path to consecutive positions, in every layer of the pool [2, L, blocks,
    heads, block size, D]: row ``context_len - nodes + path[j]`` to ``context_len - nodes + j``.

    The path ends at ``lengths``, or at an entry that is not above the one before it or no node of the tree.  fp8:
    a block whose first row is moved takes that row's scale (as :func:`store_kv` gives a first token); a row is
    rounded again where the scales differ.  int8: rows move with their scales."""
    bs, nb = kv_cache.shape[4], kv_cache.shape[2]
    fp8 = kv_cache.dtype == torch.float8_e4m3fn
    raw = kv_cache.view(torch.uint8) if fp8 else kv_cache
    for b, (n, kl) in enumerate(zip(q_lens, k_lens)):
        base, table = kl - n, block_tables[b]
        nodes: list[int] = []
        for i in path[b, :max(0, min(int(lengths[b]), path.shape[1]))].tolist():
            if not (nodes[-1] if nodes else -1) < i < n:
                break
            nodes.append(i)
        if base < 0:
            continue

        def at(pos):
            blk = table[pos // bs] if pos // bs < len(table) else -1
            return (blk, pos % bs) if 0 <= blk < nb else None

        rows = []
        for i in nodes:
            w = at(base + i)
            x = s = None
            if w is not None:
                x = raw[:, :, w[0], :, w[1]].clone()
                if kv_scale_cache is not None:
                    s = (kv_scale_cache[:, :, w[0]] if fp8 else kv_scale_cache[:, :, w[0], :, w[1]]).clone()
            rows.append((x, s))
        for j, (i, (x, s)) in enumerate(zip(nodes, rows)):
            w = at(base + j)
            if i == j or x is None or w is None:
                continue
            if fp8:
                f = x.view(kv_cache.dtype).float() * s[..., None]
                if w[1] == 0:
                    kv_scale_cache[:, :, w[0]] = fp8_block_scale(f.abs().nan_to_num(0.0).amax(-1))
                now = kv_scale_cache[:, :, w[0]][..., None]
                y = torch.clamp(f / now, -FP8_MAX, FP8_MAX).to(kv_cache.dtype).view(torch.uint8)
                x = torch.where(now == s[..., None], x, y)
            elif s is not None:
                kv_scale_cache[:, :, w[0], :, w[1]] = s
            raw[:, :, w[0], :, w[1]] = x


def dense_causal_attention(q, k, v, scale):
    """No-cache attention for one sequence: q [L, Hq, D], k/v [L, Hkv, D]."""
    g = q.shape[1] // k.shape[1]
    k = k.repeat_interleave(g, dim=1).float()
    v = v.repeat_interleave(g, dim=1).float()
    s = torch.einsum("qhd,khd->hqk", q.float(), k) * scale
    L = q.shape[0]
    mask = torch.triu(torch.ones(L, L, dtype=torch.bool, device=q.device), 1)
    s = s.masked_fill(mask[None], float("-inf"))
    return torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).to(q.dtype)


def softmax_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)

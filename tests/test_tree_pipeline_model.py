"""CPU models of the synchronisation in the kernels for trees of drafted tokens (no GPU).

As in the model of the fp8 products' roles, coroutines run under random interleavings."""
import os
import random

import pytest

from test_fp8_pipeline_model import Bar, run, wait


def _source(name):
    with open(os.path.join(os.path.dirname(__file__), "..", "csrc", name)) as f:
        return f.read()


# ------------------------------------------------------------------------------ the walk's cluster
class ClusterBarrier:
    def __init__(self, ctas):
        self.ctas, self.phase, self.at = ctas, 0, 0

    def arrive(self):
        self.at += 1
        if self.at == self.ctas:
            self.at, self.phase = 0, self.phase + 1


def walk_cluster(rng, ctas, passes, start_barrier=True):
    """tree_verify_kernel: in each pass a CTA stores its sums into the chunk buffer (two, in turn) of every CTA, meets the
    cluster's barrier and reads the buffer.  A CTA's shared memory is there from its start to its end, and CTAs start
    when they start; CTA 0 alone goes on behind the last pass (the draw)."""
    bar = ClusterBarrier(ctas)
    started, ended = [False] * ctas, [False] * ctas
    chunk = [[[None] * ctas for _ in range(2)] for _ in range(ctas)]

    def cta(me):
        for _ in range(rng.randrange(1, 60)):  # until it starts
            yield "went on"
        started[me] = True
        due = bar.phase + 1
        if start_barrier:
            bar.arrive()
            yield "went on"
            while bar.phase < due:
                yield "blocked"
        for p in range(passes):
            for to in range(ctas):
                assert started[to], "a store ahead of its target's start"
                assert not ended[to], "a store behind its target's end"
                chunk[to][p & 1][me] = p
                yield "went on"
            due = bar.phase + 1
            bar.arrive()
            while bar.phase < due:
                yield "blocked"
            for k in range(ctas):
                assert chunk[me][p & 1][k] == p
                yield "went on"
        ended[me] = True

    return [cta(i) for i in range(ctas)]


@pytest.mark.parametrize("ctas", [1, 2, 4, 8, 16])
def test_walk_stores_into_ctas_that_have_started(ctas):
    for seed in range(30):
        rng = random.Random(seed)
        run(walk_cluster(rng, ctas, 1 + seed % 5), rng, [])


def test_model_finds_stores_ahead_of_a_start():
    """Without a barrier behind the start the first sums go to CTAs that may not run yet."""
    found = 0
    for seed in range(20):
        rng = random.Random(seed)
        try:
            run(walk_cluster(rng, 4, 2, start_barrier=False), rng, [])
        except AssertionError as e:
            assert "ahead of its target's start" in str(e)
            found += 1
    assert found


def test_walk_waits_for_its_cluster_ahead_of_the_first_store():
    s = _source("tree_verify.cu")
    body = s[s.index("tree_verify_kernel(TreeVerify a, int len)"):s.index("cudaError_t launch_tree_verify")]
    loop = body.index("  while (true) {\n    const int64_t r")
    # arrived once by every thread on entry, ahead of any way out ...
    head = body[:loop]
    entry = head.index("tc::cluster_arrive();")
    assert entry < head.index("pdl_wait()") < head.index("return;")
    # ... waited for on the way out of an empty tree, and on the way to the first pass; the other pair is the pass's own
    empty = head[head.index("if (n <= 0)"):head.index("return;")]
    assert empty.count("tc::cluster_wait();") == 1
    assert head.rstrip().endswith("tc::cluster_wait();  // every CTA of the cluster has started")
    assert body.count("tc::cluster_arrive();") == 2 and body.count("tc::cluster_wait();") == 3


# --------------------------------------------------------------- attention of more than 64 rows
class Named:
    """A named barrier: `count` arrivals end a phase; who syncs waits for the end of the phase that it arrived in."""

    def __init__(self, count):
        self.count, self.at, self.phase = count, 0, 0

    def arrive(self):
        due = self.phase + 1
        self.at += 1
        if self.at == self.count:
            self.at, self.phase = 0, due
        return due

    def sync(self):
        due = self.arrive()
        while self.phase < due:
            yield "blocked"
        yield "went on"


def wide_kernel(items, slots, warps=2, group_barriers=True):
    """tree_attn_kernel on a bf16 cache: `items` is a list of (tiles, more than 128 rows?).  Two softmax groups of `warps`
    warps (the kernel's have four), an MMA warp for each, a producer with a ring of `slots` tiles (K and V in turn).  Without
    group_barriers one q_full announces an item's queries to both MMA warps."""
    q_full = [Bar(2 * warps) for _ in range(2)]
    full, empty = [Bar(1) for _ in range(slots)], [Bar(2) for _ in range(slots)]
    s_full, p_ready, o_done = [Bar(1) for _ in range(2)], [Bar(warps) for _ in range(2)], [Bar(1) for _ in range(2)]
    o_empty = Bar(2 * warps)
    turn, both = [Named(2 * warps) for _ in range(2)], Named(2 * warps)
    ring, q = [None] * slots, [[None] * warps for _ in range(2)]
    scores, weights, out = [None] * 2, [[None] * warps for _ in range(2)], [None] * 2

    def producer():
        c = 0
        for it, (n, _) in enumerate(items):
            for t in range(n):
                for kv in "kv":
                    s = c % slots
                    yield from wait(empty[s], ((c // slots) & 1) ^ 1)
                    ring[s] = (it, t, kv)
                    full[s].arrive()
                    c += 1

    def softmax(g, w):
        if g == 1:
            turn[0].arrive()
        n_done = tile0 = 0
        q[g][w] = 0
        for it, (n, two) in enumerate(items):
            steps = 2 * n if two else n
            q_full[0].arrive()
            yield "went on"
            if group_barriers and steps > 1:
                q_full[1].arrive()
            mine = 0
            for st in range(g, steps, 2):
                j = st >> 1 if two else st
                yield from wait(s_full[g], n_done & 1)
                yield from turn[g].sync()
                assert scores[g] == (it, st)
                turn[1 - g].arrive()
                weights[g][w] = (it, st)
                c = 2 * (tile0 + j) + 1
                yield from wait(full[c % slots], (c // slots) & 1)
                assert ring[c % slots] == (it, j, "v")
                p_ready[g].arrive()
                mine += 1
                n_done += 1
            if g == 1 and not two and n & 1:
                yield from turn[g].sync()
                turn[1 - g].arrive()
            if mine:
                yield from wait(o_done[g], (n_done - 1) & 1)
                assert out[g] == (it, steps - 1 - (steps - 1 - g) % 2)
            yield from both.sync()
            q[g][w] = it + 1
            yield "went on"
            assert not mine or out[g][0] == it     # read to the end
            yield from both.sync()
            o_empty.arrive()
            tile0 += n

    def mma(g):
        done = q_items = 0
        begin = 0
        for it, (n, two) in enumerate(items):
            mine, by = (n, 2) if two else ((n + 1 - g) >> 1, 4)
            k_at = begin + (2 if not two and g else 0)
            v_at = k_at + 1
            if group_barriers:
                if mine:
                    yield from wait(q_full[g], q_items & 1)
                    q_items += 1
            else:
                yield from wait(q_full[0], it & 1)
            for i in range(mine + 1):
                st = (i - 1) * 2 + g
                if i > 0:
                    yield from wait(p_ready[g], (done - 1) & 1)
                    yield from wait(full[v_at % slots], (v_at // slots) & 1)
                    if i == 1 and it > 0:
                        yield from wait(o_empty, (it - 1) & 1)
                    assert weights[g] == [(it, st)] * warps and ring[v_at % slots] == (it, st >> 1 if two else st, "v")
                    out[g] = (it, st)
                    yield "went on"
                    o_done[g].arrive()
                    for _ in range(1 if two else 2):
                        empty[v_at % slots].arrive()
                    v_at += by
                if i < mine:
                    st += 2
                    yield from wait(full[k_at % slots], (k_at // slots) & 1)
                    if done:
                        yield from wait(o_done[g], (done - 1) & 1)
                    assert q == [[it] * warps] * 2 and ring[k_at % slots] == (it, st >> 1 if two else st, "k")
                    scores[g] = (it, st)
                    yield "went on"
                    s_full[g].arrive()
                    for _ in range(1 if two else 2):
                        empty[k_at % slots].arrive()
                    k_at += by
                    done += 1
            begin += 2 * n

    return [producer()] + [softmax(g, w) for g in range(2) for w in range(warps)] + [mma(g) for g in range(2)]


def run_unevenly(roles, rng):
    """Random interleavings in which a role may be far slower than the others."""
    speed = {id(r): rng.choice([1.0, 1.0, 0.1, 0.003]) for r in roles}
    live, idle = list(roles), 0
    while live:
        r = rng.choices(live, [speed[id(x)] for x in live])[0]
        try:
            idle = idle + 1 if next(r) == "blocked" else 0
        except StopIteration:
            live.remove(r)
            idle = 0
        if idle >= 200:  # everyone twice: a step that ends in a wait may have let others go on
            idle = 0
            stuck = True
            for r in live * 2:
                try:
                    stuck = (r not in live or next(r) == "blocked") and stuck
                except StopIteration:
                    live.remove(r)
                    stuck = False
            assert not stuck, "nobody can go on"


def _items(rng):
    kind = rng.randrange(3)
    return [(1 if kind == 0 or rng.random() < 0.6 else rng.randrange(1, 6), kind == 2 and rng.random() < 0.4)
            for _ in range(rng.randrange(1, 14))]


@pytest.mark.parametrize("slots", [4, 5, 6])
def test_wide_kernel_roles(slots):
    for seed in range(60):
        rng = random.Random(seed)
        run_unevenly(wide_kernel(_items(rng), slots), rng)


def test_model_finds_an_item_that_a_group_without_steps_has_missed():
    """With one barrier for both groups' queries, a slow MMA warp loses items of one tile and waits for ever."""
    found = 0
    for seed in range(60):
        rng = random.Random(seed)
        try:
            run_unevenly(wide_kernel([(1, False)] * 8 + [(2, False)], 6, group_barriers=False), rng)
        except AssertionError as e:
            assert "nobody can go on" in str(e)
            found += 1
    assert found


def test_wide_kernel_has_the_barriers_of_the_model():
    s = _source("tree_attention.cu")
    wide = s[s.index("tree_attn_kernel(const __grid_constant__"):s.index("struct Few {")]
    assert "mbar_init(bar(sh.q_full[g]), 8)" in wide
    assert "mbar_arrive_release(bar(sh.q_full[0]));\n        if (steps > 1) tc::mbar_arrive_release(bar(sh.q_full[1]));" in wide
    assert "if (mine > 0) ok = wait(sh.q_full[g], q_items++ & 1, 2);" in wide and wide.count("q_items++") == 1

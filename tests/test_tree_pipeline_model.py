"""CPU models of the synchronisation in the kernels for trees of drafted tokens (no GPU).

As in the model of the fp8 products' roles, coroutines run under random interleavings."""
import os
import random

import pytest

from test_fp8_pipeline_model import run


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

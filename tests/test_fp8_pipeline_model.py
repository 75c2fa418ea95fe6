"""CPU model of the barriers between the roles of the fp8 products (no GPU).

The roles of one CTA run as coroutines under random interleavings.  A read of shared memory is allowed to be
performed late: at the latest when its thread next releases (a releasing arrival) or stores a value made from
it.  A relaxed arrival, which carries the accumulator's hand-over, performs nothing.  Every read checks that it
sees the k-block it was meant for, every landed copy that it was asked for, and the run that it ends."""
import random

import pytest


class Bar:
    def __init__(self, count):
        self.count, self.pending, self.phase = count, count, 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def passed(self, parity):
        """mbarrier.try_wait.parity: the phase of this parity has completed."""
        return (self.phase & 1) != parity


class Thread:
    """Reads that are issued and not yet performed."""

    def __init__(self, rng):
        self.rng, self.late = rng, []

    def read(self, where, index, expected):
        self.late.append((where, index, expected))

    def perform(self):
        for where, index, expected in self.late:
            assert where[index] == expected, f"read {where[index]} in place of {expected}"
        self.late.clear()

    def maybe(self):
        if self.late and self.rng.random() < 0.1:
            where, index, expected = self.late.pop(0)
            assert where[index] == expected, f"read {where[index]} in place of {expected}"


def run(roles, rng, threads):
    live = list(roles)
    idle = 0
    while live:
        r = rng.choice(live)
        try:
            idle = idle + 1 if next(r) == "blocked" else 0
        except StopIteration:
            live.remove(r)
            idle = 0
        for t in threads:
            t.maybe()
        assert idle < 5000, "nobody can go on"
    for t in threads:
        t.perform()


def wait(bar, parity):
    while not bar.passed(parity):
        yield "blocked"
    yield "went on"


def tokens_kernel(rng, n, stages, bufs, blocks, warps, prods, product_barriers=True):
    """gemm_fp8_tokens_kernel: n k-blocks through `stages` operand stages (with a slot of scales each), `bufs`
    accumulators, `blocks` scale warps and `warps` epilogue warps; the products of scales are given back by
    halves of `prods` k-blocks.  Without those barriers the scale warps wait for the product `bufs` k-blocks back
    to have landed, which says that the epilogue has handed over the accumulator before it."""
    half = prods // 2
    go = [Bar(1 + warps) for _ in range(stages)]
    empty = [Bar(1 + blocks) for _ in range(stages)]
    sfull = [Bar(1) for _ in range(stages)]
    tfull = [Bar(1 + blocks) for _ in range(prods if product_barriers else bufs)]
    pempty = [Bar(warps) for _ in range(2)]
    slot, product = [None] * stages, [[None] * prods for _ in range(blocks)]
    acc, stage = [None] * bufs, [None] * stages
    scale = [Thread(rng) for _ in range(blocks)]
    epi = [Thread(rng) for _ in range(warps)]
    ring = len(tfull)

    def producer():
        for it in range(n):
            s = it % stages
            yield from wait(empty[s], ((it // stages) & 1) ^ 1)
            stage[s] = it
            go[s].arrive()
            yield "went on"
            slot[s] = it
            sfull[s].arrive()

    def mma():
        for it in range(n):
            s = it % stages
            yield from wait(go[s], (it // stages) & 1)
            assert stage[s] == it
            acc[it % bufs] = it
            empty[s].arrive()
            yield "went on"
            tfull[it % ring].arrive()

    def scales(b):
        for it in range(n):
            s = it % stages
            if not product_barriers:
                if it >= bufs:
                    yield from wait(tfull[it % bufs], (it // bufs - 1) & 1)
            elif it % half == 0:
                yield from wait(pempty[it // half & 1], ((it // prods) & 1) ^ 1)
            yield from wait(sfull[s], (it // stages) & 1)
            scale[b].read(slot, s, it)
            yield "went on"
            scale[b].perform()          # the product is made from it
            product[b][it % prods] = it
            tfull[it % ring].arrive()   # releases
            yield "went on"
            empty[s].arrive()

    def epilogue(w):
        for b in range(bufs):
            go[b].arrive()
        for it in range(n):
            yield from wait(tfull[it % ring], (it // ring) & 1)
            assert acc[it % bufs] == it
            for b in range(blocks):
                epi[w].read(product[b], it % prods, it)
            yield "went on"
            go[(it + bufs) % stages].arrive()   # relaxed: the reads above may still be under way
            if product_barriers and it % half == half - 1:
                yield "went on"
                epi[w].perform()
                pempty[it // half & 1].arrive()

    return [producer(), mma()] + [scales(b) for b in range(blocks)] + [epilogue(w) for w in range(warps)], scale + epi


def weights_kernel(rng, n, stages, bufs, warps, slot_barriers=True):
    """gemm_fp8_weights_kernel: the epilogue warps read the activation scales themselves."""
    slots = stages + bufs + 1
    go = [Bar(1 + warps) for _ in range(stages)]
    empty = [Bar(1) for _ in range(stages)]
    tfull = [Bar(1) for _ in range(bufs)]
    sfull = [Bar(1) for _ in range(slots)]
    sempty = [Bar(warps) for _ in range(slots)]
    slot, acc, stage = [None] * slots, [None] * bufs, [None] * stages
    epi = [Thread(rng) for _ in range(warps)]

    def producer():
        for it in range(n):
            s, l = it % stages, it % slots
            yield from wait(empty[s], ((it // stages) & 1) ^ 1)
            if slot_barriers:
                yield from wait(sempty[l], ((it // slots) & 1) ^ 1)
            stage[s] = it
            go[s].arrive()
            yield "went on"
            slot[l] = it
            sfull[l].arrive()

    def mma():
        for it in range(n):
            s = it % stages
            yield from wait(go[s], (it // stages) & 1)
            assert stage[s] == it
            acc[it % bufs] = it
            empty[s].arrive()
            yield "went on"
            tfull[it % bufs].arrive()

    def epilogue(w):
        for b in range(bufs):
            go[b].arrive()
        for it in range(n):
            yield from wait(sfull[it % slots], (it // slots) & 1)
            yield from wait(tfull[it % bufs], (it // bufs) & 1)
            assert acc[it % bufs] == it
            go[(it + bufs) % stages].arrive()   # relaxed
            yield "went on"
            epi[w].read(slot, it % slots, it)
            yield "went on"
            if slot_barriers:
                epi[w].perform()
                sempty[it % slots].arrive()

    return [producer(), mma()] + [epilogue(w) for w in range(warps)], epi


# stages, accumulators, blocks of W of the three tile shapes (fewer epilogue warps than the kernel's 8)
TOKENS = [(4, 2, 2), (6, 2, 2), (6, 4, 1)]
WEIGHTS = [(5, 4), (4, 4), (3, 2)]


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 40, 100])
@pytest.mark.parametrize("stages,bufs,blocks", TOKENS)
def test_tokens_kernel_roles(stages, bufs, blocks, n):
    for seed in range(20):
        rng = random.Random(seed)
        roles, threads = tokens_kernel(rng, n, stages, bufs, blocks, 3, 8)
        run(roles, rng, threads)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 40, 100])
@pytest.mark.parametrize("stages,bufs", WEIGHTS)
def test_weights_kernel_roles(stages, bufs, n):
    for seed in range(20):
        rng = random.Random(seed)
        roles, threads = weights_kernel(rng, n, stages, bufs, 3)
        run(roles, rng, threads)


@pytest.mark.parametrize("kernel", ["tokens", "weights"])
def test_model_finds_reads_that_only_relaxed_arrivals_follow(kernel):
    """Without barriers of their own the scales' places rest on reads being performed before a relaxed arrival."""
    found = 0
    for seed in range(20):
        rng = random.Random(seed)
        roles, threads = (tokens_kernel(rng, 60, 4, 2, 2, 3, 4, product_barriers=False) if kernel == "tokens"
                          else weights_kernel(rng, 60, 3, 2, 3, slot_barriers=False))
        try:
            run(roles, rng, threads)
        except AssertionError as e:
            assert "in place of" in str(e)
            found += 1
    assert found


def _source():
    import os
    with open(os.path.join(os.path.dirname(__file__), "..", "csrc", "gemm_fp8.cu")) as f:
        return f.read()


def test_kernel_has_the_barriers_of_the_model():
    """Each place of scales or products that is written again is waited for, and given back by a releasing arrival."""
    s = _source()
    tokens, weights = s[s.index("gemm_fp8_tokens_kernel(const"):s.index("template <int NP, int MW>\n__global__")], \
        s[s.index("gemm_fp8_weights_kernel(const"):]
    assert "mbar_init(empty(s), 1 + C::BLOCKS)" in tokens and "mbar_arrive_release(empty(s))" in tokens
    assert "warp_wait(pempty(" in tokens and "mbar_arrive_release(pempty(" in tokens
    assert "mbar_wait(sempty(l)" in weights and "mbar_arrive_release(sempty(l))" in weights

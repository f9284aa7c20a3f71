"""The paged attention kernel's barriers (wpt_b200/csrc/paged.cuh), modelled on
the CPU: the warps that bring tiles, bring scales, issue products and take the
softmax, and the tensor pipe, which completes what was issued in order but at
any time. A segment's results may be read, and the weights' buffers be written
over with them, only once all of its products O^T += V^T P^T are complete. The
model waits for that as the source does (the barrier that the softmax waits on
after its loop over a segment's tiles is read there); with the parity of o_done,
which cannot tell a segment's last product from the one two before it, it must
find a schedule that reads too early, which shows that it can."""

import os
import random
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Barrier:
    """An mbarrier of `count` arrivals a phase; a wait names a phase by its parity only."""

    def __init__(self, count=1):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left = self.count
            self.phase += 1

    def passed(self, parity):
        return self.phase % 2 != parity % 2


def _run(segments, final, seed, raises=0.3):
    """One schedule; what was read too early."""
    rnd = random.Random(seed)
    k_full, k_empty, v_full, v_empty = ([Barrier() for _ in range(2)] for _ in range(4))
    s_full, p_ready = [Barrier(2) for _ in range(2)], [Barrier() for _ in range(2)]
    q_full, o_done, o_final = Barrier(), Barrier(), Barrier()
    tiles, pipe, arriving, complete, early = sum(segments), [], [], [0], []

    def bring():
        for j in range(tiles):
            while j >= 2 and not k_empty[j % 2].passed(j // 2 + 1):
                yield
            arriving.append(k_full[j % 2])
            while j >= 2 and not v_empty[j % 2].passed(j // 2 + 1):
                yield
            arriving.append(v_full[j % 2])
            yield

    def lands():  # copies complete in any order
        while True:
            if arriving:
                arriving.pop(rnd.randrange(len(arriving))).arrive()
            yield

    def scales():
        for j in range(tiles):
            while j >= 2 and not v_empty[(j - 2) % 2].passed((j - 2) // 2):
                yield
            s_full[j % 2].arrive()
            yield

    def issue():
        j = 0
        for number, n in enumerate(segments):
            while not q_full.passed(number):
                yield
            for i in range(n + 1):
                if i < n:
                    while not k_full[j % 2].passed(j // 2):
                        yield
                    pipe.append((None, [s_full[j % 2], k_empty[j % 2]]))
                    j += 1
                    yield
                if i > 0:
                    jp = j - 2 if i < n else j - 1
                    while not v_full[jp % 2].passed(jp // 2):
                        yield
                    while not p_ready[jp % 2].passed(jp // 2):
                        yield
                    pipe.append((jp, [v_empty[jp % 2], o_done] + ([o_final] if i == n else [])))
                    yield

    def compute():
        while True:
            if pipe:
                product, commits = pipe.pop(0)
                if product is not None:
                    assert product == complete[0]
                    complete[0] += 1
                for barrier in commits:
                    barrier.arrive()
            yield

    def softmax():
        j = 0
        for number, n in enumerate(segments):
            q_full.arrive()
            for i in range(n):
                while not s_full[j % 2].passed(j // 2):
                    yield
                if i > 0 and rnd.random() < raises:  # a base is raised: O up to the tile before is rescaled
                    while not o_done.passed(j - 1):
                        yield
                    if complete[0] < j:
                        early.append(("raise", j))
                yield
                p_ready[j % 2].arrive()
                j += 1
                yield
            while not (o_final.passed(number) if final == "o_final" else o_done.passed(j - 1)):
                yield
            if complete[0] < j:
                early.append(("result", number))
            yield

    main = softmax()
    others = [f() for f in (bring, lands, scales, issue, compute)]
    weights = [rnd.choice((0.05, 0.3, 1.0, 3.0)) for _ in range(6)]  # some agents are held up
    for _ in range(20000):
        at = rnd.choices(range(len(others) + 1), weights[:len(others)] + weights[5:])[0]
        agent = main if at == len(others) else others[at]
        try:
            next(agent)
        except StopIteration:
            if agent is main:
                return early
            weights[at] = 0.0
    raise AssertionError("the segments did not end")


SEGMENTS = ([1], [2], [3], [4], [7], [1, 1, 1], [2, 2], [1, 2, 1, 3], [5, 2, 6, 1])


def _waited_for():
    """The barrier that the softmax waits on between a segment's tiles and its results."""
    source = open(os.path.join(ROOT, "wpt_b200", "csrc", "paged.cuh")).read()
    after = source.split("more = nx.next();\n      if (more) load_ahead();")
    assert len(after) == 2
    return re.search(r"mbar_wait\((\w+),", after[1]).group(1)


@pytest.mark.parametrize("segments", SEGMENTS)
def test_results_are_read_after_a_segments_last_product(segments):
    for seed in range(400):
        assert not _run(segments, _waited_for(), seed), seed


def test_o_dones_parity_is_not_enough():
    assert any(("result", 0) in _run([2], "o_done", seed) for seed in range(400))
    assert any(("result", 0) in _run([3], "o_done", seed) for seed in range(400))
    # the wait before a raised base's rescaling is sound: that tile's scores were issued after the product before last
    assert not any(kind == "raise" for seed in range(400) for kind, _ in _run([5, 2, 6, 1], "o_final", seed, 1.0))

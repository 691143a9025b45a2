"""The expert layer cuts a phase's units into an equal run for each CTA
(MoeRuns).  Its shared memory holds the maxima of four experts of a run: no run
meets more as long as there are at most three experts in use for each CTA."""
import random


def _most_experts(experts, units, ctas):
    """The most experts that a run meets: `experts` of `units` units each, one after another."""
    total = experts * units
    ctas = min(ctas, total)
    q, r = divmod(total, ctas)
    begin = lambda c: c * q + min(c, r)  # noqa: E731
    return max((begin(c + 1) - 1) // units - begin(c) // units + 1 for c in range(ctas))


def test_a_run_meets_four_experts_at_most():
    rng = random.Random(1)
    for ctas in (1, 7, 86, 108, 132, 148, 160):
        for _ in range(200):
            experts, units = rng.randint(1, min(256, 3 * ctas)), rng.choice((1, 2, 3, rng.randint(1, 64), rng.randint(1, 5000)))
            assert _most_experts(experts, units, ctas) <= 4
    assert _most_experts(256, 2, 86) <= 4  # 256 experts, the most there are
    assert _most_experts(256, 7, 62) > 4   # refused: more than three experts a CTA

"""Which tokens a position sees: the host build of the function the kernels use, against the definition."""
import random

import flashoverlap_b200  # noqa: F401
import torch

OPS = torch.ops.flashoverlap_op


def test_visible_tokens():
    rng = random.Random(1)
    for _ in range(3000):
        i, length = rng.randrange(0, 60), rng.randrange(0, 60)
        window, sinks = rng.choice([0, 1, 2, 17, 2 ** 31 - 1]), rng.choice([0, 1, 5, 70, 2 ** 31 - 1])
        want = [j for j in range(i + 1) if window == 0 or j > i - window or j < sinks] if i < length else []
        assert OPS.seen_tokens(i, length, window, sinks) == want, (i, length, window, sinks)

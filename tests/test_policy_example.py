"""The hover example (examples/hover_policy.py): environments, advantages,
log probabilities and the optimiser together learn the task."""
import os
import sys

import pytest

from b3test import ROOT

sys.path.insert(0, os.path.join(ROOT, "examples"))


@pytest.mark.gpu
@pytest.mark.parametrize("state_bits", [32, 8])
def test_hover_policy_learns(state_bits):
    """The reward of a step is 1 - min(e, 2) with e = |y - target| + 0.1 |v|:
    a policy of even chances falls or climbs away, one that holds the height
    gets close to 1.  Four rollouts are one episode."""
    from hover_policy import train
    got = train(envs=1024, steps=64, updates=24, state_bits=state_bits)
    first, last = sum(got[:4]) / 4, sum(got[-4:]) / 4
    assert last > first + 0.3 and last > 0.5, got

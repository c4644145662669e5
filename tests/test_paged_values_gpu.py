"""The paged cache on the GPU where values, lengths and timing are unkind."""
import numpy as np
import pytest

import saetta_macqwen_b200 as sa
from test_paged_gpu import Case

pytestmark = pytest.mark.gpu


def test_a_cta_that_joins_an_item_and_goes_on_to_another():
    """Verify rows of ragged sequences: a CTA joins an item's parts and then begins another, whose statistics lie where the joined sums
    were.  Half of a row tile's warps have no live rows and do not wait for the others' stores."""
    import torch

    rng = np.random.default_rng(11)
    c = Case(16, 2, 256, 64, [(int(kv), 4) for kv in rng.integers(200, 3000, 24)], sa.BF16, sa.F32, True, seed=11)
    op = c.op()
    c.record(op)
    c.check()
    first = c.out.clone()
    for _ in range(200):
        c.record(op)
        torch.cuda.synchronize()
        assert torch.equal(first, c.out)
    assert op.device_status() == 0

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


@pytest.mark.parametrize("dt", [sa.F32, sa.BF16])
def test_short_runs_that_raise_a_scale_read_it_before_it_is_written(dt):
    """One lane writes a block's scale that all lanes of the warp have read: single rows of as many sequences, each larger than what its
    block holds."""
    import torch

    from paged_util import ref_store
    from test_paged_gpu import Pool, i32, tdt

    p = Pool(2, 256, 64, 300, seed=3)
    rng = np.random.default_rng(3)
    slots = [b * 64 + int(rng.integers(1, 64)) for b in range(300)]
    k, v = (torch.from_numpy((rng.normal(size=(300, 2, 256)) * 2.0 ** rng.integers(-3, 9, (300, 1, 1))).astype(np.float32)).to(tdt(dt)) for _ in range(2))
    p.cache.store(k.cuda(), v.cuda(), i32(slots), 300, dtype=dt)
    torch.cuda.synchronize()
    ref_store(*p.codes, p.scales, k.double().numpy(), v.double().numpy(), slots, 64)
    p.same()


FRESH = """
import sys
sys.path[:0] = {path!r}
import torch
from test_paged_gpu import Step
for seqs in (3046, 3047, 3071, 3073, 8192):
    st = Step([5] * seqs, [1] * seqs, None, [0] * 4, 4, [[0]] * seqs, 16, seqs)
    st.run()
    torch.cuda.synchronize()
    assert st.status.item() == 0 and st.starts[-1].item() == seqs and st.slots.cpu().tolist() == [5] * seqs, seqs
print("done")
"""


def test_assign_of_every_number_of_sequences_in_a_process_that_made_no_larger_call():
    """Its scan's shared memory passes what a launch has without asking at 3047 sequences."""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FRESH.format(path=[here, os.path.dirname(here)])], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("rows", [1, 20])
def test_lengths_that_are_cut_off_are_reported(rows):
    """A length behind its row of the block table, rows behind the call's, falling row starts: cut off as before, and said."""
    import torch

    from test_paged_gpu import i32

    def run(change):
        c = Case(16, 2, 256, 16, [(90, rows), (64, rows)], sa.BF16, sa.F32, seed=2)
        change(c)
        op = c.op()
        c.record(op)
        torch.cuda.synchronize()
        return op.device_status()

    assert run(lambda c: None) == 0
    longest = lambda c: c.dev.__setitem__(3, i32([90, c.width * 16]))  # noqa: E731 (its last pages lie outside the cache)
    assert run(longest) & 32 == 0
    assert run(lambda c: c.dev.__setitem__(3, i32([90, c.width * 16 + 1]))) & 32
    assert run(lambda c: (c.dev.__setitem__(2, i32([0, rows, rows])), c.dev.__setitem__(3, i32([90, 1 << 30])))) == 0  # no rows: its length is not read
    assert run(lambda c: c.dev.__setitem__(2, i32([0, rows, 2 * rows + 1]))) & 32
    assert run(lambda c: c.dev.__setitem__(2, i32([0, rows, rows - 1]))) & 32


@pytest.mark.parametrize("q_dt", [sa.BF16, sa.F16])
@pytest.mark.parametrize("dim", [128, 256])
def test_row_tiles_of_one_key_tile_behind_one_another(q_dt, dim):
    """Short prompts: every item of a CTA is one tile, and its products are under way when the next one is at hand."""
    import torch

    rng = np.random.default_rng(dim)
    c = Case(16, 2, dim, 16, [(int(kv), int(n)) for kv, n in zip(rng.integers(5, 120, 500), rng.integers(3, 6, 500))], q_dt, sa.F32, seed=dim)
    op = c.op()
    c.record(op)
    c.check()
    first = c.out.clone()
    for _ in range(100):
        c.record(op)
        torch.cuda.synchronize()
        assert torch.equal(first, c.out)
    assert op.device_status() == 0

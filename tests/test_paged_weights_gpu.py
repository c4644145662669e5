"""Attention over the paged cache on the GPU, for keys, values and scores that models have and random ones do not."""
import numpy as np
import pytest

import saetta_macqwen_b200 as sa
from paged_values import Sequences, bf16, off

pytestmark = pytest.mark.gpu

# The yardstick: the same softmax in 64 bits with its weights rounded to bfloat16, as an ordinary kernel has them.  The kernels may be
# off by twice that as a whole, and by what f32 scores make of the weights: a score is a running sum of some 2 * dim / 32 steps (three terms: 3),
# each off by at most 2^-22 of the largest partial sum, which the tests keep near the score itself.

HEADS, DIM = 8, 128


def parts(q_dt):
    return 2 if q_dt == sa.BF16 else 3


def allowed(s, want, absv, top):
    coarse = s.exact(bf16)[0]
    return 2 * np.linalg.norm(coarse - want) + np.linalg.norm(absv * (parts(s.q_dt) * s.dim / 32 * 2.0 ** -22 * (top[..., None] + 1)))


def near(s, got):
    want, absv, top, _ = s.exact()
    lim = allowed(s, want, absv, top)
    assert np.linalg.norm(got - want) <= lim, (np.linalg.norm(got - want) / np.linalg.norm(want), lim / np.linalg.norm(want))


def plain(rng, n, kv, dim=DIM, heads=HEADS, mean=1.0):
    """Scores of one nat's spread once scaled by dim ** -0.5; dim 0 of q is 1 and of k is 0: for offsets."""
    q, k, v = rng.normal(size=(n, heads, dim)), rng.normal(size=(kv, 1, dim)), rng.normal(size=(kv, 1, dim)) + mean
    q[..., 0], k[..., 0] = 1.0, 0.0
    return q, k, v


ROWS = [(2, "few"), (24, "many")]  # rows of a sequence: 16 and 192 rows of a tile


@pytest.mark.parametrize("rows,kernel", ROWS)
@pytest.mark.parametrize("q_dt", [sa.BF16, sa.F16])
@pytest.mark.parametrize("kv,share", [(100, 0.9), (4096, 0.5), (4096, 0.9), (32768, 0.3), (32768, 0.5), (32768, 0.9)])
def test_a_key_that_holds_much_of_the_weight(rows, kernel, q_dt, kv, share):
    """An attention sink: the first key, of a value near zero, has a given share of every row's weight."""
    rng = np.random.default_rng(kv)
    q, k, v = plain(rng, rows, kv)
    k[0], v[0] = 0, rng.normal(size=DIM) * 0.01
    k[0, 0, 0] = (np.log(kv * np.exp(0.5) * share / (1 - share))) * DIM ** 0.5
    s = Sequences([(q, k, v)], 64, q_dt, DIM ** -0.5)
    near(s, s.run())


@pytest.mark.parametrize("rows,kernel", ROWS)
@pytest.mark.parametrize("q_dt", [sa.BF16, sa.F16])
@pytest.mark.parametrize("nats", [400, 700, 1500, -700, -1500, 6000])
def test_an_offset_of_all_scores_changes_nothing(rows, kernel, q_dt, nats):
    rng = np.random.default_rng(5)
    q, k, v = plain(rng, rows, 1500)
    q[..., 0] = nats / 16
    k[..., 0] = 16 * DIM ** 0.5
    s = Sequences([(q, k, v)], 64, q_dt, DIM ** -0.5)
    near(s, s.run())
@pytest.mark.parametrize("rows,kernel", ROWS)
@pytest.mark.parametrize("q_dt", [sa.BF16, sa.F16])
@pytest.mark.parametrize("doublings", [6, 10, 20, 40])
@pytest.mark.parametrize("nats", [-40, -80])
def test_a_block_of_large_values_and_little_weight(rows, kernel, q_dt, doublings, nats):
    """One block's values are larger than the others', and its keys have next to no weight."""
    rng = np.random.default_rng(doublings)
    q, k, v = plain(rng, rows, 1500)
    k[128:192, 0, 0] = nats * DIM ** 0.5
    v[128:192] *= 2.0 ** doublings
    s = Sequences([(q, k, v)], 64, q_dt, DIM ** -0.5)
    near(s, s.run())


@pytest.mark.parametrize("q_dt", [sa.BF16, sa.F16])
@pytest.mark.parametrize("doublings", [10, 20, 40])
@pytest.mark.parametrize("kv,rows", [(200, 200), (130, 3), (500, 400)])
def test_a_later_block_of_large_values_leaves_the_rows_before_it_alone(q_dt, doublings, kv, rows):
    """Every row by itself: those that do not see the large block are as exact as without it."""
    rng = np.random.default_rng(doublings + kv)
    q, k, v = plain(rng, rows, kv, heads=8)
    v[kv - 70:] *= 2.0 ** doublings
    s = Sequences([(q, k, v)], 16, q_dt, DIM ** -0.5)
    want, absv, top, edge = s.exact()
    got = s.run(max_rows=rows if rows > 3 else 2)
    # Twice bfloat16's step for each weight; and what the weights' terms end at: the largest weight (times value scale) of a tile is kept at 2^-2 at least (it
    # may stand 8 doublings below what weights are kept against, 2^6), and no weight is off by more than 2^-14 (two terms) or 2^-17 beside its step.
    lim = np.linalg.norm(absv * (2.0 ** -7 + 1e-4) + 2.0 ** (-12 if parts(q_dt) == 2 else -15) * edge, axis=-1)
    err = np.linalg.norm(got - want, axis=-1)
    assert (err <= lim).all(), (err / lim).max()


@pytest.mark.parametrize("rows", [1, 2, 24])
@pytest.mark.parametrize("q_dt", [sa.F32, sa.BF16, sa.F16])
@pytest.mark.parametrize("kv,sign", [(1, 1.0), (1, -1.0), (40, -1.0)])
def test_an_infinite_query_gives_nan_whatever_the_keys_signs(rows, q_dt, kv, sign):
    """All scores at minus infinity are not a row without keys; rows beside it, and rows that see no key, stay as they are."""
    rng = np.random.default_rng(3)
    q, k, v = plain(rng, rows, kv)
    k[..., 5] = np.abs(k[..., 5]) + 1
    q[:, 3, 5] = sign * np.inf
    s = Sequences([(q, k, v)], 16, q_dt, DIM ** -0.5)
    got = s.run()
    s.q[0][:, 3, 5] = 0
    want = s.exact()[0]
    sees = np.arange(rows) >= rows - kv
    assert np.isnan(got[sees, 3]).all() and (got[~sees] == 0).all()
    rest = [h for h in range(HEADS) if h != 3]
    assert off(got[:, rest], want[:, rest]) < 2.0 ** -7


NANS = [  # few rows; heads, dim, block, keys, rows, the keys that hold NaN
    (2, 128, 16, 6, 6, [2, 4]),
    (2, 128, 16, 300, 8, [295, 298]),
    (4, 256, 64, 130, 4, [127, 129]),
    (8, 256, 32, 700, 2, [699]),
    (1, 128, 128, 200, 16, [190, 199]),
    (8, 128, 16, 5000, 2, [10, 4999]),
    (3, 256, 64, 64, 5, [60, 62]),
    # many rows
    (8, 128, 16, 200, 200, [0, 50, 130]),
    (2, 256, 64, 300, 70, [231, 299, 257]),
    (1, 128, 32, 700, 400, [300, 511, 512, 600, 699]),
    (16, 256, 128, 1000, 40, [961, 999, 5]),
    (8, 128, 64, 9000, 20, [8981, 8999, 4000]),
    (3, 128, 16, 50, 90, [10, 49]),
    (12, 256, 16, 130, 130, [126, 127, 128, 129]),
]


@pytest.mark.parametrize("q_dt", [sa.BF16, sa.F16])
@pytest.mark.parametrize("heads,dim,block,kv,rows,keys", NANS)
def test_nan_reaches_the_rows_that_see_it_and_no_other(q_dt, heads, dim, block, kv, rows, keys):
    """NaN in a few dims of some rows' values, the others' among the same keys: in the dims that have it for the rows that see the key, and
    nowhere for those before it.  The same for a NaN key, which takes the whole row."""
    rng = np.random.default_rng(kv + rows)
    for side in (2, 1):
        x = list(plain(rng, rows, kv, dim=dim, heads=heads))
        for i, key in enumerate(keys):
            x[side][key, 0, [3 + i, dim - 1]] = np.nan
        s = Sequences([tuple(x)], block, q_dt, dim ** -0.5, seed=kv)
        got = s.run()
        for i in range(2):
            s.kv[i][0] = np.nan_to_num(s.kv[i][0])
        want = s.exact()[0]
        nan = np.zeros(want.shape, bool)
        for i, key in enumerate(keys):
            sees = np.arange(rows) + kv - rows >= key
            if side == 1:
                nan[sees] = True
            else:
                nan[np.ix_(sees, np.arange(heads), [3 + i, dim - 1])] = True
        assert np.array_equal(np.isnan(got), nan), np.argwhere(np.isnan(got) != nan)[:5]
        err = np.abs(np.where(nan, 0, got - want)).max((1, 2))
        assert (err < 2.0 ** -5).all(), err.max()


@pytest.mark.parametrize("dim,q_dt", [(128, sa.F16), (256, sa.BF16)])
@pytest.mark.parametrize("doublings,nats,share", [(10, -40, 0), (20, -40, 0), (40, -80, 0), (60, -80, 0), (-140, 0, 0), (0, 0, 0.99), (0, 0, 0.9999)])
def test_long_shares_of_a_decode_batch(dim, q_dt, doublings, nats, share):
    """So many sequences that a warp goes through several tiles of each: a block of large values and little weight, zeros, or a first key of
    much weight takes nothing from what the warp meets after it."""
    rng = np.random.default_rng(dim + 200 + doublings)
    seqs = []
    for i in range(37):
        kv = int(rng.integers(2500, 4500))
        q, k, v = plain(rng, 2, kv, dim=dim)
        at = 64 * int(rng.integers(0, 4))
        k[at:at + 64, 0, 0] = nats * dim ** 0.5
        v[at:at + 64] *= 2.0 ** doublings if doublings > -100 else 0
        if share:
            k[0], v[0] = 0, rng.normal(size=dim) * 0.01
            k[0, 0, 0] = np.log(kv * np.exp(0.5) * share / (1 - share)) * dim ** 0.5
        seqs.append((q, k, v))
    s = Sequences(seqs, 64, q_dt, dim ** -0.5)
    near(s, s.run())


@pytest.mark.parametrize("dim,q_dt", [(128, sa.F16), (128, sa.BF16), (256, sa.F16), (256, sa.BF16)])
@pytest.mark.parametrize("doublings,nats,share", [(10, -40, 0), (40, -80, 0), (-140, 0, 0), (0, 0, 0.9), (0, 700, 0), (0, -30, 0), (-20, 0, 0)])
def test_long_shares_of_prompts(dim, q_dt, doublings, nats, share):
    """The same for the many-rows kernel: so many prompts that a CTA goes through all tiles of a row tile, and its weights' reference goes up and
    down on the way: 192 keys of other scores and values, or a first key of much weight."""
    rng = np.random.default_rng(dim + 300 + doublings + int(share * 10))
    seqs = []
    for i in range(30):
        kv = int(rng.integers(900, 1700))
        q, k, v = plain(rng, 32, kv, dim=dim)
        at = 64 * int(rng.integers(0, 8))
        k[at:at + 192, 0, 0] = nats * dim ** 0.5
        v[at:at + 192] *= 2.0 ** doublings if doublings > -100 else 0
        if share:
            k[0], v[0] = 0, rng.normal(size=dim) * 0.01
            k[0, 0, 0] = np.log(kv * np.exp(0.5) * share / (1 - share)) * dim ** 0.5
        seqs.append((q, k, v))
    s = Sequences(seqs, 64, q_dt, dim ** -0.5)
    near(s, s.run())


@pytest.mark.parametrize("rows,kernel", ROWS)
@pytest.mark.parametrize("q_dt", [sa.BF16, sa.F16, sa.F32])
@pytest.mark.parametrize("size,nan", [(2.0 ** 12, False), (2.0 ** 24, True), (2.0 ** 34, True)])
def test_scores_past_what_f32_resolves(rows, kernel, q_dt, size, nan):
    """One key's score stands out by far.  Up to 2^20 both kernels return its value; past that a difference of two scores has no fraction left: the few-rows
    kernel still does, the many-rows kernel returns NaN and never another key's value."""
    rng = np.random.default_rng(4)
    q, k, v = plain(rng, rows, 700)
    k[..., 0] = 1.0
    k[300, 0, 0] = 1.5
    q[..., 0] = 2.0 ** 12
    s = Sequences([(q, k, v)], 64, q_dt, DIM ** -0.5 * size / 2.0 ** 12)
    got, want = s.run(), np.broadcast_to(s.kv[1][0][0][300], (rows, HEADS, DIM))
    if nan and kernel == "many":
        assert np.isnan(got).all()
    else:
        # The one weight is 2 to the power of a difference of two f32 numbers of 1.44 * 1.5 * 4096 = 2^13.1, rounded to 2^-10 each, and its sum has what the products'
        # first term rounds away: off by 2 * 2^-11 * ln 2 < 2^-10 at most.  (The few-rows kernel subtracts after rounding: exact.)
        assert (np.abs(got - want) <= (2.0 ** -10 * np.abs(want) if kernel == "many" else 0)).all()

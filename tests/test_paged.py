"""The paged cache without a GPU: refusals come back before any device work, and the plain restatements hold."""
import ctypes as C
import functools
import os

import numpy as np
import pytest

import saetta_macqwen_b200 as sa
from paged_util import TABLE, e4m3_encode, pow2_scale

FAKE = 4096  # a non-null, 16-byte aligned address that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(sa.LIB_PATH):
        sa.build()
    return sa.lib()


def refused(code, fn, *args, **kw):
    with pytest.raises(sa.SaettaError) as e:
        fn(*args, **kw)
    assert e.value.code == code, str(e.value)
    return str(e.value)


def wrap(kv_heads=2, head_dim=256, block=64, blocks=8, k=FAKE, v=FAKE, s=FAKE):
    return sa.PagedKvCache.wrap(0, kv_heads, head_dim, block, blocks, k, v, s)


def test_cache_refusals(lib):
    refused(sa.BAD_SHAPE, wrap, head_dim=64)
    refused(sa.BAD_SHAPE, wrap, kv_heads=0)
    for block in (0, 8, 48, 256):
        refused(sa.BAD_SHAPE, wrap, block=block)
    refused(sa.BAD_SHAPE, wrap, blocks=0)
    refused(sa.BAD_SHAPE, wrap, blocks=1 << 24)  # 2 * 64 * 2^24 rows: the copies' row coordinate is 32-bit
    refused(sa.BAD_ARG, wrap, k=None)
    refused(sa.BAD_ARG, wrap, s=FAKE + 4)
    assert lib.saetta_paged_cache_create(0, 2, 256, 64, 8, None) == sa.BAD_ARG
    assert lib.saetta_paged_cache_buffers(None, None, None, None) == sa.BAD_ARG
    lib.saetta_paged_cache_destroy(None)
    c = wrap()
    assert c.buffers() == (FAKE, FAKE, FAKE)


def test_store_refusals(lib):
    c = wrap()
    store = functools.partial(c.store, stream=0)
    refused(sa.BAD_ARG, store, FAKE, FAKE, FAKE, 1, dtype=7)
    refused(sa.BAD_ARG, store, None, FAKE, FAKE, 1)
    refused(sa.BAD_ARG, store, FAKE, FAKE, None, 1)
    refused(sa.BAD_SHAPE, store, FAKE, FAKE, FAKE, 1, k_stride=511)
    refused(sa.BAD_ARG, store, FAKE + 8, FAKE, FAKE, 1)
    refused(sa.BAD_ARG, store, FAKE, FAKE, FAKE, 1, v_stride=514, dtype=sa.F16)
    refused(sa.BAD_SHAPE, store, FAKE, FAKE, FAKE, 1 << 30)
    store(None, None, None, 0)  # no rows: nothing to do
    assert lib.saetta_paged_store(None, FAKE, FAKE, 0, 1, 512, 512, FAKE, None, None) == sa.BAD_ARG


def test_assign_refusals(lib):
    ok = dict(device=0, seqs=2, block_tokens=16, kv_lens=FAKE, new_tokens=FAKE, free_blocks=FAKE, free_cap=8, free_count=FAKE, block_tables=FAKE,
              table_stride=4, row_starts=FAKE, slots=FAKE, positions=None, rows_cap=4, kv_lens_out=FAKE, free_count_out=FAKE, status=FAKE, stream=0)
    for name in ("kv_lens", "new_tokens", "free_blocks", "free_count", "block_tables", "row_starts", "slots", "kv_lens_out", "free_count_out", "status"):
        assert "null" in refused(sa.BAD_ARG, sa.paged_assign, **{**ok, name: None})
    for bad in (dict(block_tokens=20), dict(seqs=8193), dict(table_stride=0), dict(table_stride=1 << 28), dict(free_cap=1 << 28), dict(rows_cap=1 << 31)):
        refused(sa.BAD_SHAPE, sa.paged_assign, **{**ok, **bad})


def test_attend_refusals(lib):
    h = C.c_void_p()
    for heads, kv, dim in ((16, 2, 64), (15, 2, 256), (34, 2, 256), (0, 2, 256), (16, 0, 256)):
        assert lib.saetta_paged_attention_create(0, heads, kv, dim, C.byref(h)) == sa.BAD_SHAPE
    assert lib.saetta_paged_attention_create(0, 16, 2, 256, None) == sa.BAD_ARG
    batch = sa.PagedBatch(1, 1, 1, 1, FAKE, FAKE, FAKE)
    assert lib.saetta_paged_attend(None, wrap().h, batch, FAKE, 0, 4096, None, FAKE, 0, 1.0, None) == sa.BAD_ARG
    assert lib.saetta_paged_attention_status(None, None, C.byref(C.c_uint32())) == sa.BAD_ARG
    lib.saetta_paged_attention_destroy(None)


def test_e4m3_restatement_against_torch():
    import torch

    rng = np.random.default_rng(3)
    grid = TABLE[:127]
    y = np.concatenate([grid, (grid[1:] + grid[:-1]) / 2, rng.uniform(-448, 448, 5000), rng.normal(0, 0.01, 5000)])
    y = np.concatenate([y, -y]).astype(np.float32)
    want = torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(e4m3_encode(y), want)
    assert np.array_equal(TABLE[want], torch.from_numpy(y).to(torch.float8_e4m3fn).double().numpy())


def test_scale_is_the_smallest_power_of_two_that_fits():
    for amax in (448.0, 448.0 * (1 + 2.0 ** -23), 1.0, 1.75, 3.5e-30, 3.0e38, 1e-44):
        s = float(pow2_scale(amax))
        assert amax <= 448 * s and (amax > 448 * s / 2 or s == 2.0 ** -126)
    assert float(pow2_scale(0.0)) == 2.0 ** -126

"""The paged 8-bit cache on the GPU: block assignment, the quantising append and attention, each against its plain
64-bit restatement, and a run of them together."""
import numpy as np
import pytest

import saetta_macqwen_b200 as sa
from paged_util import TABLE, ref_assign, ref_attend, ref_store

pytestmark = pytest.mark.gpu

U = {sa.F32: 2.0 ** -24, sa.F16: 2.0 ** -11, sa.BF16: 2.0 ** -8}


def tdt(dt):
    import torch

    return {sa.F32: torch.float32, sa.F16: torch.float16, sa.BF16: torch.bfloat16}[dt]


def i32(x):
    import torch

    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------- assign


class Step:
    """Device buffers of one assign call."""

    def __init__(self, lens, new, fin, free, count, tables, block, rows_cap, cap=None):
        import torch

        self.n, self.block, self.rows_cap, self.width = len(lens), block, rows_cap, len(tables[0]) if tables else 0
        self.cap = len(free) if cap is None else cap
        self.lens, self.new, self.fin = i32(lens), i32(new), (i32(fin) if fin is not None else None)
        self.free, self.count, self.tables = i32(free), i32([count]), i32(tables)
        z = lambda n: torch.full((n,), -77, dtype=torch.int32, device="cuda")  # noqa: E731
        self.starts, self.slots, self.pos, self.out_lens, self.out_count, self.status = z(self.n + 1), z(rows_cap), z(rows_cap), z(self.n), z(1), z(1)

    def run(self, in_place=False, positions=True, stream=None):
        sa.paged_assign(0, self.n, self.block, self.lens, self.new, self.free, self.cap, self.count, self.tables, self.width, self.starts,
                        self.slots, self.pos if positions else None, self.rows_cap, self.lens if in_place else self.out_lens,
                        self.count if in_place else self.out_count, self.status, finished=self.fin, stream=stream)


def random_step(rng, seqs, block, len_hi, new_hi, done, pad):
    lens = [int(x) for x in rng.integers(0, len_hi + 1, seqs)]
    new = [int(x) for x in rng.integers(0, new_hi + 1, seqs)]
    fin = [int(x) for x in rng.random(seqs) < done]
    width = max(1, max((n + m + block - 1) // block for n, m in zip(lens, new)))
    have = [(n + block - 1) // block for n in lens]
    pool = sum((n + m + block - 1) // block + 1 for n, m in zip(lens, new)) + 3
    ids = [int(x) for x in rng.permutation(pool)]
    tables, at = [], 0
    for h in have:
        tables.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    free = ids[at:] + [-5] * at
    return lens, new, fin, free, pool - at, tables, sum(new) + pad


@pytest.mark.parametrize("seqs,block,len_hi,new_hi,done,pad", [
    (1, 64, 700, 1, 0.0, 0), (1, 16, 0, 0, 0.0, 2), (3, 16, 40, 40, 0.5, 5), (257, 32, 500, 1, 0.2, 7), (1025, 16, 64, 9, 0.3, 100),
    (8192, 128, 300, 2, 0.1, 1), (40, 128, 4000, 900, 0.5, 0), (1, 16, 5, 20000, 0.0, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_assign_is_the_plain_step(seqs, block, len_hi, new_hi, done, pad, in_place):
    import torch

    lens, new, fin, free, count, tables, cap = random_step(np.random.default_rng(seqs + block), seqs, block, len_hi, new_hi, done, pad)
    st = Step(lens, new, fin, free, count, tables, block, cap)
    st.run(in_place)
    torch.cuda.synchronize()
    want_tables, want_free = [list(t) for t in tables], list(free)
    starts, slots, pos, want_lens, want_count = ref_assign(lens, new, fin, want_free, count, want_tables, block, cap)
    got = lambda t: t.cpu().tolist()  # noqa: E731
    assert got(st.status) == [0]
    assert got(st.starts) == starts and got(st.slots) == slots and got(st.pos) == pos
    assert got(st.tables) == want_tables and got(st.free) == want_free
    assert got(st.lens if in_place else st.out_lens) == want_lens and got(st.count if in_place else st.out_count) == [want_count]
    if not in_place:
        assert got(st.lens) == lens and got(st.count) == [count]


def test_assign_refuses_whole_steps_on_the_device():
    import torch

    base = dict(lens=[20, 0], new=[30, 5], fin=[0, 0], free=[9, 8, 7, 6], count=4, tables=[[1, 2, -1, -1], [-1, -1, -1, -1]], block=16, rows_cap=40)
    for change, bit in ((dict(count=2), sa.PAGED_NO_BLOCKS), (dict(new=[50, 5]), sa.PAGED_TABLE_FULL), (dict(rows_cap=34), sa.PAGED_ROWS_FULL),
                        (dict(cap=3), sa.PAGED_NO_BLOCKS), (dict(new=[2**31 - 1, 5]), sa.PAGED_TABLE_FULL), (dict(lens=[2**31 - 1, 0]), sa.PAGED_TABLE_FULL)):
        st = Step(**{**base, **change})
        before = st.tables.cpu().tolist(), st.free.cpu().tolist()
        st.run(positions=False)
        torch.cuda.synchronize()
        assert st.status.item() & bit, (change, st.status.item())
        assert (st.tables.cpu().tolist(), st.free.cpu().tolist()) == before
        assert st.starts.cpu().tolist() == [0, 0, 0] and set(st.slots.cpu().tolist()) == {-1}
        assert st.out_lens.cpu().tolist() == st.lens.cpu().tolist() and st.out_count.item() == st.count.item()
        assert set(st.pos.cpu().tolist()) == {-77}  # not asked for


def test_assign_without_sequences():
    import torch

    st = Step([], [], None, [3, 4], 2, [], 16, 3)
    st.run()
    torch.cuda.synchronize()
    assert st.status.item() == 0 and st.starts.cpu().tolist() == [0] and st.slots.cpu().tolist() == [-1] * 3 and st.out_count.item() == 2


# ----------------------------------------------------------------- store


class Pool:
    """A cache over torch buffers, with its plain twin."""

    def __init__(self, kv_heads, dim, block, blocks, seed=0, nan=False):
        import torch

        rng = np.random.default_rng(seed)
        self.kv, self.dim, self.block, self.blocks = kv_heads, dim, block, blocks
        shape = (blocks, kv_heads, block, dim)
        self.codes = [rng.integers(0, 256, shape, dtype=np.uint8) for _ in range(2)]
        if not nan:
            for c in self.codes:
                c[(c & 127) == 127] = 0x30
        self.scales = 2.0 ** rng.integers(-9, -6, (blocks, kv_heads, 2)).astype(np.float64)
        self.keys, self.values = (torch.from_numpy(c.copy()).cuda() for c in self.codes)
        self.sc = torch.from_numpy(self.scales.astype(np.float32)).cuda()
        self.cache = sa.PagedKvCache.wrap(0, kv_heads, dim, block, blocks, self.keys, self.values, self.sc)

    def same(self):
        for t, c in zip((self.keys, self.values), self.codes):
            got = t.cpu().numpy()
            nan = (got & 127) == 127
            assert np.array_equal(nan, (c & 127) == 127)
            bad = np.argwhere((got != c) & ~nan)
            assert not len(bad), (len(bad), bad[:3], got[tuple(bad[0])], c[tuple(bad[0])])
        assert np.array_equal(self.sc.cpu().numpy().astype(np.float64), self.scales)


STORES = [  # dtype, kv heads, dim, block, [(block id, offset, rows)] or a negative number of skipped rows
    (sa.F32, 2, 256, 64, [(3, 5, 1)]),
    (sa.F32, 1, 128, 16, [(0, 0, 16), (5, 0, 16), (2, 0, 3)]),
    (sa.BF16, 2, 256, 64, [(1, 63, 1), (4, 0, 64), (0, 0, 7), (2, 9, 55)]),
    (sa.F16, 8, 128, 32, [-2, (6, 31, 1), -1, (7, 1, 2), (0, 0, 1), -3]),
    (sa.BF16, 3, 128, 128, [(1, 0, 128), (0, 100, 28), (2, 0, 90)]),
    (sa.F16, 1, 256, 128, [(1, 37, 70)]),
]


@pytest.mark.parametrize("dt,kv,dim,block,runs", STORES)
@pytest.mark.parametrize("grow", [1.0, 40.0, 0.01])
def test_store_is_the_plain_append(dt, kv, dim, block, runs, grow):
    import torch

    p = Pool(kv, dim, block, 8, seed=block)
    slots = []
    for r in runs:
        slots += [-1] * -r if isinstance(r, int) else [r[0] * block + r[1] + j for j in range(r[2])]
    rng = np.random.default_rng(7)
    k, v = (torch.from_numpy((rng.normal(size=(len(slots), kv, dim)) * grow).astype(np.float32)).to(tdt(dt)) for _ in range(2))
    status = i32([0])
    p.cache.store(k.cuda(), v.cuda(), i32(slots), len(slots), dtype=dt, status=status)
    torch.cuda.synchronize()
    ref_store(*p.codes, p.scales, k.double().numpy(), v.double().numpy(), slots, block)
    p.same()
    assert status.item() == 0


def test_store_strided_rows_of_a_fused_projection():
    import torch

    p = Pool(2, 128, 16, 4)
    fused = torch.randn((9, 1000), device="cuda")  # k at 8, v at 520 of each row
    slots = list(range(20, 29))
    p.cache.store(fused.data_ptr() + 8 * 4, fused.data_ptr() + 520 * 4, i32(slots), 9, k_stride=1000, v_stride=1000)
    torch.cuda.synchronize()
    f = fused.cpu().double().numpy()
    ref_store(*p.codes, p.scales, f[:, 8:264].reshape(9, 2, 128), f[:, 520:776].reshape(9, 2, 128), slots, 16)
    p.same()


def test_store_of_extreme_values():
    import torch

    p = Pool(1, 128, 16, 3)
    k = torch.zeros((6, 1, 128))
    k[0, 0, :8] = torch.tensor([float("inf"), -float("inf"), float("nan"), 3.0, -448.0, 1e-30, 0.0, -0.0])
    k[1] = 3.0e38  # with the row before: the scale follows the finite values
    k[2] = 1.0e-41  # a block of values below the smallest scale
    v = torch.zeros((6, 1, 128))  # a block of zeros
    slots = [0, 1, 16, 17, 40, 41]
    p.cache.store(k.cuda(), v.cuda(), i32(slots), 6)
    torch.cuda.synchronize()
    ref_store(*p.codes, p.scales, k.double().numpy(), v.double().numpy(), slots, 16)
    p.same()


def test_store_reports_and_skips_bad_slots():
    import torch

    p = Pool(2, 128, 16, 4)
    k, v = torch.randn((6, 2, 128), device="cuda"), torch.randn((6, 2, 128), device="cuda")
    slots = [64, 5, 5, 7, 1 << 30, 20]  # outside; fine; the same again; out of order; outside; fine
    status = i32([0])
    p.cache.store(k, v, i32(slots), 6, status=status)
    torch.cuda.synchronize()
    assert status.item() == sa.PAGED_BAD_SLOT
    keep = [1, 5]
    ref_store(*p.codes, p.scales, k.cpu().double().numpy()[keep], v.cpu().double().numpy()[keep], [5, 20], 16)
    p.same()


# ----------------------------------------------------------------- attend


def bound(out_dt, q_dt, out, b, kv_max, dim, many):
    """What the arithmetic allows, per value: the output's rounding; each probability's, and what an error of its score makes of
    it, weighted like the values; the f32 sums' own.  A score's error: f32 queries enter with 11 bits; each of dim additions may
    be off by one part in 2^23 of the sum of |q k|; scale factors and the exponential, a few parts in 2^23 of |s|.  Few rows: a
    probability is a binary16 (2^-11).  Many rows: q and the probabilities are sums of e4m3 values, two (2^-8 of the value) for bfloat16 q,
    three (2^-12) else; below e4m3's normal range a term is off by up to 2^-10 of its unit, where a row's largest q is 2^7 units at least and
    the largest weight 2^4.75 of the largest value scale's (it is kept times 2^5.5, under a maximum with half a doubling to spare that is
    rounded up to bfloat16: |s| < 64 here)."""
    ds = (dim * 2.0 ** -23 + (2.0 ** -11 if q_dt == sa.F32 else 0.0)) * b["mag"] + 8 * 2.0 ** -23 * (b["top"] + 1)
    p_step, floor = 2.0 ** -11, 0.0
    if many:
        ds = ds + 2.0 ** -17 * b["qwide"]
        p_step = 2.0 ** -8 if q_dt == sa.BF16 else 2.0 ** -12 + 2.0 ** -24
        floor = 2.0 ** -14.75 * b["wide"]
    rel = p_step + 2 * ds + kv_max * 2.0 ** -23 + 2.0 ** -18
    return (U[out_dt] * np.abs(out) + (rel[..., None] * b["absv"] + floor) * (1 + U[out_dt]) + 2.0 ** -24 * (out_dt == sa.F16) + 1e-30)


class Case:
    def __init__(self, heads, kv_heads, dim, block, seqs, q_dt=sa.BF16, out_dt=sa.BF16, gate=False, seed=0, pad=0, tail_nan=True, peaky=1.0):
        """seqs: [(kv_len, rows)]."""
        import torch

        rng = np.random.default_rng(seed)
        need = [(kv + block - 1) // block for kv, _ in seqs]
        self.width = max(max(need), 1) + 1
        pool = sum(need) + 2
        self.p = Pool(kv_heads, dim, block, pool, seed=seed)
        ids = rng.permutation(pool)
        self.tables = np.full((len(seqs), self.width), -1, np.int64)
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = ids[at:at + n]
            at += n
        x = [rng.normal(size=(pool, kv_heads, block, dim)) * s for s in (peaky, 1.0)]
        from paged_util import e4m3_encode, pow2_scale

        for i in range(2):
            self.p.scales[..., i] = pow2_scale(np.abs(x[i]).max((2, 3))) * 2.0 ** rng.integers(0, 3, (pool, kv_heads))
            self.p.codes[i][:] = e4m3_encode(x[i] / self.p.scales[..., i][:, :, None, None])
        dirty = [c.copy() for c in self.p.codes]
        if tail_nan:  # what was never written may be anything
            for s, (kv, _) in enumerate(seqs):
                if kv % block:
                    for c in dirty:
                        c[self.tables[s, kv // block], :, kv % block:] = 0x7F
            used = set(self.tables[self.tables >= 0].tolist())
            for b in range(pool):
                if b not in used:
                    for c in dirty:
                        c[b] = 0xFF
        self.p.keys.copy_(torch.from_numpy(dirty[0])), self.p.values.copy_(torch.from_numpy(dirty[1]))
        self.p.sc.copy_(torch.from_numpy(self.p.scales.astype(np.float32)))
        self.kv_lens = [kv for kv, _ in seqs]
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in seqs])]).tolist()
        self.rows = self.starts[-1] + pad
        self.heads, self.kv_heads, self.dim, self.block, self.q_dt, self.out_dt = heads, kv_heads, dim, block, q_dt, out_dt
        self.q = torch.from_numpy(rng.normal(size=(self.rows, heads, dim)).astype(np.float32)).to(tdt(q_dt))
        self.gate = torch.from_numpy(rng.normal(size=(self.rows, heads, 2 * dim)).astype(np.float32)) if gate else None
        self.max_rows = max([n for _, n in seqs] + [0])
        self.scale = dim ** -0.5
        self.out = torch.full((self.rows, heads, dim), 7.0, dtype=tdt(out_dt), device="cuda")
        self.dev = [self.q.cuda(), self.gate.cuda() if gate else None, i32(self.starts), i32(self.kv_lens), i32(self.tables)]

    def record(self, op, q=None, q_stride=None, stream=None, out=None):
        d = self.dev
        op.record(self.p.cache, d[0] if q is None else q, self.q_dt, self.rows, len(self.kv_lens), d[2], d[3], d[4], self.width, self.max_rows,
                  self.scale, self.out if out is None else out, self.out_dt, q_and_gate=d[1], q_stride=q_stride, stream=stream)

    def op(self):
        return sa.PagedAttention(0, self.heads, self.kv_heads, self.dim)

    def ref(self):
        gate = self.gate[..., self.dim:].double().numpy() if self.gate is not None else None
        return ref_attend(self.q.double().numpy(), *self.p.codes, self.p.scales, self.tables, self.starts, self.kv_lens, self.block, self.scale, gate)

    def check(self, out=None):
        import torch

        torch.cuda.synchronize()
        got = (self.out if out is None else out).cpu().double().numpy()
        want, b = self.ref()
        total = self.starts[-1]
        assert np.isfinite(got[:total]).all()
        many = self.max_rows * (self.heads // self.kv_heads) > 16
        lim = bound(self.out_dt, self.q_dt, want, b, max(self.kv_lens), self.dim, many)
        off = np.abs(got - want)[:total] / lim[:total]
        assert off.size == 0 or off.max() <= 1.0, (off.max(), np.unravel_index(off.argmax(), off.shape))
        assert (got[total:] == 7.0).all()  # rows of no sequence


DECODES = [
    # heads, kv heads, dim, block, [(kv_len, rows)]
    (16, 2, 256, 64, [(1, 1)]),
    (16, 2, 256, 64, [(701, 1)]),
    (16, 2, 256, 16, [(64, 1), (65, 1), (63, 1), (0, 0), (16, 1), (17, 1)]),
    (32, 8, 128, 32, [(300, 1), (0, 1), (5, 0), (1999, 1)]),
    (8, 8, 128, 128, [(129, 1), (128, 1), (1000, 1)]),
    (14, 2, 128, 16, [(77, 1), (200, 2)]),
    (16, 1, 256, 32, [(500, 1), (33, 1)]),
    (16, 1, 128, 64, [(90, 3)]),
    (12, 2, 256, 128, [(1025, 1), (127, 1)]),
    (16, 2, 256, 64, [(9000, 1)]),
    (40, 8, 128, 16, [(333, 4), (4, 4), (50, 1)]),
    (16, 2, 256, 32, [(3, 5), (2, 2), (700, 8)]),  # more rows than keys: the first rows see nothing
]


@pytest.mark.parametrize("heads,kv,dim,block,seqs", DECODES)
@pytest.mark.parametrize("q_dt,out_dt,gate", [(sa.BF16, sa.BF16, True), (sa.F16, sa.F16, False), (sa.F32, sa.F32, True)])
def test_few_rows(heads, kv, dim, block, seqs, q_dt, out_dt, gate):
    c = Case(heads, kv, dim, block, seqs, q_dt, out_dt, gate, seed=len(seqs) + block, pad=2)
    op = c.op()
    c.record(op)
    c.check()
    assert op.device_status() == 0


PROMPTS = [
    (16, 2, 256, 64, [(128, 128)]),
    (16, 2, 256, 64, [(5, 5)]),
    (16, 2, 256, 16, [(300, 300), (17, 1), (40, 33), (0, 0)]),
    (8, 8, 128, 32, [(257, 129), (127, 127)]),
    (32, 8, 128, 128, [(500, 100), (130, 130), (77, 0)]),
    (28, 4, 128, 16, [(211, 200), (19, 19)]),
    (10, 2, 256, 32, [(400, 64)]),
    (16, 1, 256, 64, [(90, 61), (1000, 3)]),
    (16, 1, 128, 16, [(1500, 40)]),
    (12, 2, 128, 64, [(30, 50), (64, 64)]),  # more rows than keys
    (2, 2, 256, 128, [(700, 290)]),
]


@pytest.mark.parametrize("heads,kv,dim,block,seqs", PROMPTS)
@pytest.mark.parametrize("q_dt,out_dt,gate", [(sa.BF16, sa.BF16, True), (sa.F16, sa.F16, False), (sa.F32, sa.F32, True)])
def test_prompts(heads, kv, dim, block, seqs, q_dt, out_dt, gate):
    c = Case(heads, kv, dim, block, seqs, q_dt, out_dt, gate, seed=len(seqs) + block, pad=3)
    op = c.op()
    c.record(op)
    c.check()
    assert op.device_status() == 0


def test_a_chunk_far_into_a_sequence_is_split_and_joined():
    for q_dt in (sa.BF16, sa.F16):
        c = Case(16, 2, 256, 64, [(5000, 40)], q_dt, q_dt, True, seed=4)
        op = c.op()
        c.record(op)
        c.check()
        first = c.out.clone()
        c.record(op)
        c.check()
        assert (first == c.out).all() and op.device_status() == 0


def test_many_sequences_in_one_call():
    rng = np.random.default_rng(5)
    seqs = [(int(kv), int(kv > 0)) for kv in rng.integers(0, 200, 700)]
    c = Case(8, 4, 128, 16, seqs, sa.F16, sa.F16, seed=9)
    op = c.op()
    c.record(op)
    c.check()
    first = c.out.clone()
    c.record(op)  # the same call again gives the same bits
    c.check()
    assert (first == c.out).all()


def test_rows_of_q_with_a_stride():
    import torch

    c = Case(16, 2, 256, 32, [(90, 1), (300, 1)], sa.BF16, sa.BF16, seed=3)
    wide = torch.zeros((2, 16 * 256 + 264), dtype=torch.bfloat16, device="cuda")
    wide[:, 8:8 + 4096] = c.dev[0].reshape(2, -1)
    op = c.op()
    c.record(op, q=wide.data_ptr() + 16, q_stride=wide.shape[1])
    c.check()


@pytest.mark.parametrize("rows", [1, 20])
def test_value_scales_of_every_size(rows):
    """Blocks of zeros (their scale is the smallest) beside ordinary ones, and sequences whose values are all tiny or all huge."""
    import torch

    for kind in range(3):
        c = Case(16, 2, 256, 16, [(200, rows), (90, rows)], sa.BF16, sa.F32, seed=kind)
        if kind == 0:
            for b in c.tables[0, ::3][:3]:
                c.p.codes[1][b] = 0
                c.p.scales[b, :, 1] = 2.0 ** -126
        else:
            c.p.scales[..., 1] *= 2.0 ** (-100 if kind == 1 else 60)
        c.p.values.copy_(torch.from_numpy(np.where(np.isnan(TABLE[c.p.values.cpu().numpy()]), 0x7F, c.p.codes[1])))
        c.p.sc.copy_(torch.from_numpy(c.p.scales.astype(np.float32)))
        op = c.op()
        c.record(op)
        c.check()


@pytest.mark.parametrize("rows", [1, 30])
def test_a_table_entry_outside_the_cache_is_reported_and_left_out(rows):
    import torch

    c = Case(16, 2, 256, 32, [(300, rows)], sa.BF16, sa.BF16, seed=2)
    hole = 3  # this block's keys take no part: the same as the sequence without them
    c.dev[4][0, hole] = c.p.blocks + 7
    op = c.op()
    c.record(op)
    torch.cuda.synchronize()
    assert op.device_status() == 16
    got = c.out.cpu().double().numpy()
    q = c.q.double().numpy()
    k, v = ((TABLE[side[c.tables[0, :10]]] * c.p.scales[c.tables[0, :10], :, i][:, :, None, None]).transpose(1, 0, 2, 3).reshape(2, 320, 256)
            for i, side in enumerate(c.p.codes))
    for i in range(rows):
        seen = np.array([j for j in range(300 - rows + i + 1) if not hole * 32 <= j < hole * 32 + 32])
        for h in (0, 9):
            w = k[h // 8][seen] @ q[i, h] * c.scale
            w = np.exp(w - w.max())
            want = w @ v[h // 8][seen] / w.sum()
            assert np.abs(got[i, h] - want).max() < 2.0 ** -7 * np.abs(v[h // 8][seen]).max()  # bfloat16 weights and output, each 2^-8 of the largest value


def test_long_prompt_tails_are_joined_in_two_rounds():
    """Few rows over many keys: an item lies in more CTAs than one joins by itself."""
    c = Case(8, 1, 128, 128, [(30000, 16)], sa.F16, sa.F32, seed=1)
    c.max_rows = 64  # the many-rows kernel
    op = c.op()
    c.record(op)
    c.check()
    c.max_rows = 2
    c.record(op)
    c.max_rows = 16  # (which bound holds)
    first = c.out.clone()
    c.record(op)
    c.check()
    assert op.device_status() == 0 and first.isfinite().all()


def test_offsets_beyond_32_bits():
    import torch

    blocks = (1 << 32) // (2 * 64 * 256) + 9  # 4 GB of keys and a little more
    cache = sa.PagedKvCache(0, 2, 256, 64, blocks)
    rng = np.random.default_rng(0)
    n = 130
    k, v = (torch.from_numpy(rng.normal(size=(n, 2, 256)).astype(np.float32)) for _ in range(2))
    table = [blocks - 1, 3, blocks - 2]
    slots = [table[j // 64] * 64 + j % 64 for j in range(n)]
    cache.store(k.cuda(), v.cuda(), i32(slots), n)
    codes = [np.zeros((3, 2, 64, 256), np.uint8) for _ in range(2)]
    scales = np.full((3, 2, 2), 1.0)
    ref_store(*codes, scales, k.double().numpy(), v.double().numpy(), list(range(n)), 64)
    for rows in (1, 3):
        q = torch.from_numpy(rng.normal(size=(rows, 16, 256)).astype(np.float32)).to(torch.bfloat16)
        out = torch.zeros((rows, 16, 256), dtype=torch.bfloat16, device="cuda")
        op = sa.PagedAttention(0, 16, 2, 256)
        op.record(cache, q.cuda(), sa.BF16, rows, 1, i32([0, rows]), i32([n]), i32([table]), 3, rows, 1 / 16, out, sa.BF16)
        torch.cuda.synchronize()
        want, b = ref_attend(q.double().numpy(), *codes, scales, np.array([[0, 1, 2]]), [0, rows], [n], 64, 1 / 16)
        lim = bound(sa.BF16, sa.BF16, want, b, n, 256, rows * 8 > 16)
        assert (np.abs(out.cpu().double().numpy() - want) <= lim).all()


def test_two_ops_on_two_streams_at_once():
    import torch

    cases = [Case(16, 2, 256, 64, [(3000, 1), (500, 1)], sa.BF16, sa.BF16, seed=1), Case(16, 2, 256, 64, [(900, 120)], sa.BF16, sa.BF16, seed=2)]
    ops = [c.op() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, op, s in zip(cases, ops, streams):
            c.record(op, stream=s)
    for c, op in zip(cases, ops):
        c.check()
        assert op.device_status() == 0


# ----------------------------------------------------------------- together


class Server:
    """A small server's buffers: requests of one layer, three launches a step, all lengths on the device."""

    def __init__(self, heads=16, kv=2, dim=256, block=16, blocks=64, seqs=5, width=12, rows_cap=40, seed=0):
        import torch

        self.rng = np.random.default_rng(seed)
        self.heads, self.kv, self.dim, self.block, self.seqs, self.width, self.cap = heads, kv, dim, block, seqs, width, rows_cap
        self.cache = sa.PagedKvCache(0, kv, dim, block, blocks)
        self.op = sa.PagedAttention(0, heads, kv, dim)
        self.free = [int(x) for x in self.rng.permutation(blocks)]
        self.count, self.lens, self.tables = blocks, [0] * seqs, [[-1] * width for _ in range(seqs)]
        self.codes = [np.zeros((blocks, kv, block, dim), np.uint8) for _ in range(2)]
        self.scales = np.zeros((blocks, kv, 2))
        z = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.d = dict(lens=i32(self.lens), new=z(seqs), fin=z(seqs), free=i32(self.free), count=i32([self.count]), tables=i32(self.tables), starts=z(seqs + 1),
                      slots=z(rows_cap), pos=z(rows_cap), status=z(1), store_status=z(1))
        self.k, self.v = (torch.zeros((rows_cap, kv, dim), device="cuda") for _ in range(2))
        self.q = torch.zeros((rows_cap, heads, dim), dtype=torch.bfloat16, device="cuda")
        self.gate = torch.zeros((rows_cap, heads, 2 * dim), device="cuda")
        self.out = torch.zeros((rows_cap, heads, dim), dtype=torch.bfloat16, device="cuda")

    def launch(self, max_rows, stream=None):
        d = self.d
        sa.paged_assign(0, self.seqs, self.block, d["lens"], d["new"], d["free"], len(self.free), d["count"], d["tables"], self.width, d["starts"], d["slots"], d["pos"],
                        self.cap, d["lens"], d["count"], d["status"], finished=d["fin"], stream=stream)
        self.cache.store(self.k, self.v, d["slots"], self.cap, status=d["store_status"], stream=stream)
        self.op.record(self.cache, self.q, sa.BF16, self.cap, self.seqs, d["starts"], d["lens"], d["tables"], self.width, max_rows, self.dim ** -0.5, self.out, sa.BF16,
                       q_and_gate=self.gate, stream=stream)

    def feed(self, new, fin):
        import torch

        self.new, self.fin = new, fin
        self.d["new"].copy_(i32(new)), self.d["fin"].copy_(i32(fin))
        for t in (self.k, self.v, self.q, self.gate):
            t.copy_(torch.from_numpy(self.rng.normal(size=tuple(t.shape)).astype(np.float32)))
        self.out.fill_(5.0)

    def check(self, max_rows):
        import torch

        torch.cuda.synchronize()
        starts, slots, pos, self.lens, self.count = ref_assign(self.lens, self.new, self.fin, self.free, self.count, self.tables, self.block, self.cap)
        assert self.d["status"].item() == 0 and self.d["store_status"].item() == 0 and self.op.device_status() == 0
        assert self.d["slots"].cpu().tolist() == slots and self.d["pos"].cpu().tolist() == pos and self.d["tables"].cpu().tolist() == self.tables
        ref_store(*self.codes, self.scales, self.k.cpu().double().numpy(), self.v.cpu().double().numpy(), slots, self.block)
        want, b = ref_attend(self.q.cpu().double().numpy(), *self.codes, self.scales, np.array(self.tables), starts, self.lens, self.block, self.dim ** -0.5,
                             self.gate[..., self.dim:].cpu().double().numpy())
        got, total = self.out.cpu().double().numpy(), starts[-1]
        lim = bound(sa.BF16, sa.BF16, want, b, max(self.lens + [1]), self.dim, max_rows * self.heads // self.kv > 16)
        assert (np.abs(got - want) <= lim)[:total].all() and (got[total:] == 5.0).all()


STEPS = [([7, 0, 19, 1, 3], [0] * 5), ([1, 16, 1, 1, 1], [0] * 5), ([1, 1, 1, 1, 1], [0, 0, 0, 1, 0]), ([0, 1, 1, 9, 1], [1, 0, 0, 0, 0]), ([12, 1, 1, 1, 1], [0, 0, 1, 0, 0]),
         ([1] * 5, [0] * 5), ([0] * 5, [0] * 5), ([0, 2, 0, 0, 1], [1, 0, 0, 0, 0])]


def test_steps_of_a_server():
    srv = Server()
    for new, fin in STEPS:
        srv.feed(new, fin)
        srv.launch(max(new))
        srv.check(max(new))


@pytest.mark.parametrize("max_rows", [2, 19])
def test_a_recorded_step_serves_other_lengths(max_rows):
    """One capture replayed for every step, lengths and tables read on the device; more rows than the hint only cost time."""
    import torch

    srv = Server(seed=max_rows)
    srv.feed([1] * 5, [0] * 5)
    srv.launch(max_rows)
    srv.check(max_rows)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        srv.launch(max_rows)
    for new, fin in STEPS:
        srv.feed(new, fin)
        graph.replay()
        srv.check(max_rows)


def test_a_step_that_does_not_fit_leaves_everything():
    import torch

    srv = Server(blocks=4)
    srv.feed([20, 20, 0, 0, 0], [0] * 5)
    srv.launch(20)
    srv.check(20)
    before = srv.d["tables"].clone(), srv.d["lens"].clone(), [t.clone() for t in (srv.out,)]
    srv.feed([20, 20, 0, 0, 0], [0] * 5)  # two more blocks are needed than there are
    srv.launch(20)
    torch.cuda.synchronize()
    assert srv.d["status"].item() == sa.PAGED_NO_BLOCKS
    assert (srv.d["tables"] == before[0]).all() and (srv.d["lens"] == before[1]).all()
    assert (srv.out == 5.0).all() and (srv.d["slots"] == -1).all()


def test_prep_paged_step_and_output_projection():
    """The framework's own layer around the cache: prep's f32 keys and queries in, the projection's f32 input out."""
    import torch

    H, KV, D, n = 16, 2, 256, 23
    srv = Server(blocks=8, seqs=1, rows_cap=n, width=4)
    rng = np.random.default_rng(8)
    qg, k, v = (torch.from_numpy(rng.normal(size=s).astype(np.float32)).cuda() for s in ((n, H, 2 * D), (n, KV, D), (n, KV, D)))
    ones = torch.ones(D, device="cuda")
    q, k_out, out = torch.zeros((n, H, D), device="cuda"), torch.zeros((n, KV, D), device="cuda"), torch.zeros((n, H, D), device="cuda")
    scratch = sa.GpuKvCache(0, 32, 128)
    sa.attention_prep(sa.PrepParams(H, KV, D, 64, 1.0e7, 1.0e-6), n, qg, k, v, ones, ones, q, sa.F32, scratch, pos=0, k_out=k_out)
    d = srv.d
    d["new"].copy_(i32([n]))
    sa.paged_assign(0, 1, 16, d["lens"], d["new"], d["free"], 8, d["count"], d["tables"], 4, d["starts"], d["slots"], d["pos"], n, d["lens"], d["count"], d["status"])
    srv.cache.store(k_out, v, d["slots"], n)
    srv.op.record(srv.cache, q, sa.F32, n, 1, d["starts"], d["lens"], d["tables"], 4, n, 1 / 16, out, sa.F32, q_and_gate=qg)
    words = torch.from_numpy(rng.integers(0, 2**31, (64, H * D // 4)).astype(np.int32)).cuda()  # 64 rows of an 8-bit matrix
    sc, bi = (torch.full((64, H * D // 64), x, dtype=torch.bfloat16, device="cuda") for x in (0.01, -1.28))
    y = torch.zeros((1, 64), device="cuda")
    sa.qmv_rows(0, words, sc, bi, 8, 64, H * D, 1, out[n - 1], y)
    torch.cuda.synchronize()
    kr, qr = k_out.cpu().double().numpy(), q.cpu().double().numpy()
    ref_store(*srv.codes, srv.scales, kr, v.cpu().double().numpy(), d["slots"].cpu().tolist(), 16)
    want, b = ref_attend(qr, *srv.codes, srv.scales, d["tables"].cpu().numpy(), [0, n], [n], 16, 1 / 16, qg[..., D:].cpu().double().numpy())
    assert (np.abs(out.cpu().double().numpy() - want) <= bound(sa.F32, sa.F32, want, b, n, D, True)).all()
    w = (words.cpu().numpy().view(np.uint8).astype(np.float64).reshape(64, H * D)) * float(sc[0, 0]) + float(bi[0, 0])
    row = out[n - 1].cpu().double().numpy().ravel()
    assert np.abs(y.cpu().double().numpy()[0] - w @ row).max() <= H * D * 2.0 ** -23 * (np.abs(w) @ np.abs(row)).max()


@pytest.mark.parametrize("rows", [1, 40])
def test_queries_of_every_size(rows):
    """Rows of q near the largest value, with keys that bring the scores back; an infinite and a NaN row, which reach no other."""
    import torch

    c = Case(16, 2, 256, 32, [(150, rows)], sa.BF16, sa.BF16, seed=6)
    c.q[:, 1] *= 2.0 ** 124
    c.q[:, 2] *= 2.0 ** -90
    c.p.scales[:, 0, 0] *= 2.0 ** -110
    c.p.sc.copy_(torch.from_numpy(c.p.scales.astype(np.float32)))
    c.scale = 2.0 ** -18  # of head 1 alone do the scores count
    clean = c.q.clone()
    clean[:, 12:14] = 0
    c.q[:, 12, 7], c.q[:, 13, 200] = float("inf"), float("nan")
    op = c.op()
    c.record(op, q=c.q.cuda())
    torch.cuda.synchronize()
    got = c.out.cpu().double().numpy()
    want, b = ref_attend(clean.double().numpy(), *c.p.codes, c.p.scales, c.tables, c.starts, c.kv_lens, c.block, c.scale)
    lim = bound(sa.BF16, sa.BF16, want, b, 150, 256, rows * 8 > 16)
    assert np.isnan(got[:, 12:14]).all()
    keep = [h for h in range(16) if h not in (12, 13)]
    assert (np.abs(got - want) <= lim)[:, keep].all() and op.device_status() == 0


@pytest.mark.parametrize("hint", [0, 1])
def test_a_hint_below_the_rows_costs_time_alone(hint):
    for heads, dim in ((16, 128), (9, 256)):
        c = Case(heads, 1, dim, 16, [(70, 5), (33, 1)], sa.F16, sa.F32, seed=heads)
        op = c.op()
        c.max_rows = hint
        c.record(op)
        c.max_rows = 1
        c.check()


@pytest.mark.parametrize("shift", [0, 1])
def test_assign_rows_at_any_address(shift):
    """slots and positions need no more than 4-byte alignment; runs of every length, and empty ones, side by side."""
    import torch

    rng = np.random.default_rng(shift)
    lens, new = [int(x) for x in rng.integers(0, 40, 300)], [int(x) for x in rng.integers(0, 7, 300)]
    tables = [[-1] * 4 for _ in lens]
    free = [int(x) for x in rng.permutation(1500)]
    count = len(free)
    for s, n in enumerate(lens):
        for j in range((n + 15) // 16):
            count -= 1
            tables[s][j] = free[count]
    cap = sum(new) + 3
    z = lambda *n: torch.full(n, 77, dtype=torch.int32, device="cuda")  # noqa: E731
    d = [i32(x) for x in (lens, new, free, [count], tables)]
    starts, slots, pos, status = z(301), z(cap + 2), z(cap + 2), z(1)
    sa.paged_assign(0, 300, 16, d[0], d[1], d[2], 1500, d[3], d[4], 4, starts, slots[shift:], pos[shift:], cap, d[0], d[3], status)
    torch.cuda.synchronize()
    w_starts, w_slots, w_pos, w_lens, w_count = ref_assign(lens, new, [0] * 300, free, count, tables, 16, cap)
    assert starts.cpu().tolist() == w_starts and d[0].cpu().tolist() == w_lens and d[3].item() == w_count and d[4].cpu().tolist() == tables
    for got, want in ((slots, w_slots), (pos, w_pos)):
        assert got.cpu().tolist() == [77] * shift + want + [77] * (2 - shift)


def test_a_plan_of_a_serving_step():
    """The framework's recorder: three kernels, run again for other lengths."""
    import torch

    srv = Server(seed=4)
    plan = sa.Plan(0)
    torch.cuda.synchronize()
    with plan.recording():
        srv.launch(1, stream=plan.stream)
    assert len(plan) == 3 and "paged_assign" in plan.kernels()[0][0]
    for new, fin in STEPS:
        srv.feed(new, fin)
        torch.cuda.synchronize()
        plan.set_params(0, 0)
        plan.run()
        torch.cuda.synchronize()
        srv.check(1)

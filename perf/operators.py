"""What is measured of the paged 8-bit cache: block assignment, the quantising append, and attention over its blocks.

Three operators, as a serving step uses them one after the other:

  assign   block tables and slot maps from request lengths (integers only)
  store    append of new key / value rows to e4m3 blocks with one scale for each (block, kv head, side)
  attend   causal attention of ragged query rows over those blocks: single tokens, verify rows, prompts

`run` computes them in elementary torch operations, or, where `own` is set, through saetta_macqwen_b200.
"""
import random

import torch

own = False

E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    # The sizes with 16 heads, 2 kv heads and dim 256 are this repository's model; the others are generic.
    return [
        # one request, one token: a scheduling step whose whole cost is latency
        dict(name="assign-1", op="assign", shape=1, seqs=1, block=64, len_lo=700, len_hi=700, new_lo=1, new_hi=1, done=0.0, pad=0),
        # a full decode batch: every request grows by a token, some end and give their blocks back, rows padded to the graph's size
        dict(name="assign-509-decode", op="assign", shape=2, seqs=509, block=16, len_lo=1, len_hi=8192, new_lo=1, new_hi=1, done=0.05, pad=3),
        # admission of prompts beside running requests: long slot maps
        dict(name="assign-1024-prompts", op="assign", shape=3, seqs=1024, block=32, len_lo=0, len_hi=4096, new_lo=0, new_hi=256, done=0.1, pad=100),
        # decode of one request: one row into a block that is partly full
        dict(name="store-1", op="store", shape=4, seqs=1, block=64, kv_heads=2, dim=256, len_lo=700, len_hi=700, new_lo=1, new_hi=1, dtype="f32", pad=0),
        # decode of a batch: one row each, every block partly full
        dict(name="store-253-decode", op="store", shape=5, seqs=253, block=16, kv_heads=8, dim=128, len_lo=0, len_hi=300, new_lo=1, new_hi=1, dtype="f16", pad=3),
        # prompts: whole blocks at a time, ragged ends
        dict(name="store-16k-prompts", op="store", shape=6, seqs=9, block=64, kv_heads=2, dim=256, len_lo=0, len_hi=200, new_lo=900, new_hi=2700, dtype="bf16", pad=0),
        # chat with one user: a short context, one token; latency
        dict(name="attend-1x701", op="attend", shape=7, seqs=1, block=64, heads=16, kv_heads=2, dim=256, kv_lo=701, kv_hi=701, new_lo=1, new_hi=1, dtype="bf16", gate=True, pad=0),
        # one request over a long document, one token: the cache's bandwidth
        dict(name="attend-1x131k", op="attend", shape=8, seqs=1, block=64, heads=16, kv_heads=2, dim=256, kv_lo=131072, kv_hi=131072, new_lo=1, new_hi=1, dtype="bf16", gate=True, pad=0),
        # a decode batch with ragged lengths, small blocks, head size 128
        dict(name="attend-61-ragged", op="attend", shape=9, seqs=61, block=16, heads=32, kv_heads=8, dim=128, kv_lo=1, kv_hi=8192, new_lo=1, new_hi=1, dtype="f16", gate=False, pad=3),
        # speculative decoding: four rows to be verified for each request
        dict(name="attend-24-verify", op="attend", shape=10, seqs=24, block=32, heads=16, kv_heads=2, dim=256, kv_lo=500, kv_hi=9000, new_lo=4, new_hi=4, dtype="bf16", gate=True, pad=0),
        # prompts of several requests in one call, some with a cached prefix
        dict(name="attend-7-prompts", op="attend", shape=11, seqs=7, block=16, heads=32, kv_heads=8, dim=128, kv_lo=40, kv_hi=3500, new_lo=33, new_hi=1500, dtype="f16", gate=False, pad=0),
        # a chunk of a long prompt, the size that this repository prefills by
        dict(name="attend-4096-at-28k", op="attend", shape=12, seqs=1, block=64, heads=16, kv_heads=2, dim=256, kv_lo=32768, kv_hi=32768, new_lo=4096, new_hi=4096, dtype="bf16", gate=True, pad=0),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    shape, block = rng.randrange(1 << 30), rng.choice([16, 32, 64, 128])
    kind = rng.choice(["assign", "store", "decode", "verify", "prompts", "prompts"])
    if kind == "assign":
        hi = _log(rng, 1, 256)
        return dict(op="assign", shape=shape, seqs=_log(rng, 1, 1024), block=block, len_lo=0, len_hi=_log(rng, 1, 4096), new_lo=rng.choice([0, 1]), new_hi=hi,
                    done=rng.choice([0.0, 0.1, 0.5]), pad=rng.randrange(64))
    heads, kv_heads, dim = rng.choice([(16, 2, 256), (32, 8, 128), (8, 8, 128), (12, 2, 256), (40, 8, 128), (16, 1, 256), (28, 4, 128)])
    if kind == "store":
        seqs = _log(rng, 1, 250)
        return dict(op="store", shape=shape, seqs=seqs, block=block, kv_heads=kv_heads, dim=dim, len_lo=0, len_hi=_log(rng, 1, 400), new_lo=1, new_hi=_log(rng, 1, 16000 // seqs),
                    dtype=rng.choice(["f32", "f16", "bf16"]), pad=rng.randrange(5))
    common = dict(op="attend", shape=shape, block=block, heads=heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["f16", "bf16"]), gate=rng.random() < 0.5, pad=rng.randrange(4))
    if kind == "prompts":
        seqs, new_hi = _log(rng, 1, 8), _log(rng, 17, 2000)
        kv_hi = max(new_hi, _log(rng, 100, 30000 // seqs))
        return dict(common, seqs=seqs, kv_lo=rng.randrange(1, 40), kv_hi=kv_hi, new_lo=rng.randrange(0, 17), new_hi=new_hi)
    seqs = _log(rng, 1, 200)
    new = 1 if kind == "decode" else rng.randrange(2, 9)
    return dict(common, seqs=seqs, kv_lo=rng.choice([0, 1, 300]), kv_hi=_log(rng, 400, max(500, min(130000, 400000 // seqs))), new_lo=rng.choice([0, new]), new_hi=new)


def _lengths(case):
    """Of each sequence: tokens cached before the call, new tokens, and whether it has ended.  Goes by the case alone."""
    r = random.Random(case["shape"])
    before, new, done = [], [], []
    for _ in range(case["seqs"]):
        n = r.randint(case["new_lo"], case["new_hi"])
        if case["op"] == "attend":
            kv = max(n, r.randint(case["kv_lo"], case["kv_hi"]))
            before.append(kv - n)
        else:
            before.append(r.randint(case["len_lo"], case["len_hi"]))
        new.append(n)
        done.append(case["op"] == "assign" and r.random() < case["done"])
    return before, new, done


def _blocks(tokens, block):
    return (tokens + block - 1) // block


def _sizes(case):
    before, new, done = _lengths(case)
    width = max(1, max(_blocks(b + n, case["block"]) for b, n in zip(before, new)))
    used = sum(_blocks(b + n, case["block"]) for b, n in zip(before, new))
    return dict(before=before, new=new, done=done, rows=sum(new) + case["pad"], width=width, pool=used + 5)


def _side(g, shape, spread):
    """Keys or values [blocks, kv heads, tokens, dim] in f32: unit values, some channels larger, as after a norm's weight."""
    x = torch.randn(shape, generator=g, device="cuda")
    wide = 1.0 + spread * (torch.rand((1, shape[1], 1, shape[3]), generator=g, device="cuda") > 0.97)
    return x.mul_(wide)


def _pow2_scale(amax):
    """The smallest power of two (2^-126 at least) by which amax lies within e4m3."""
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)  # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e, torch.full_like(e, -126))
    return ((e + 127) << 23).view(torch.float32)  # by its bits: a power function may be a place off


def _encode(x, scale):
    return (x * (1.0 / scale)).to(torch.float8_e4m3fn)


def prepare(case, seed):
    z = _sizes(case)
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["shape"] % 9973)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    S, B = case["seqs"], case["block"]
    st = dict(case=case, z=z)
    ids = torch.randperm(z["pool"], generator=g, device="cuda", dtype=torch.int32)  # a pool in use for a while has no order
    # tables as they stand before the call (assign) or with the call's own tokens (store, attend)
    own_blocks = [_blocks(b if case["op"] == "assign" else b + n, B) for b, n in zip(z["before"], z["new"])]
    have = torch.tensor(own_blocks, device="cuda")
    inside = torch.arange(z["width"], device="cuda")[None, :] < have[:, None]
    tables = torch.full((S, z["width"]), -1, dtype=torch.int32, device="cuda")
    tables[inside] = ids[: sum(own_blocks)]
    st["tables"] = tables
    st["row_starts"] = i32([sum(z["new"][:k]) for k in range(S + 1)]) if S < 64 else torch.cat([i32([0]), i32(z["new"]).cumsum(0).to(torch.int32)])
    if case["op"] == "assign":
        st["kv_lens"], st["new"], st["done"] = i32(z["before"]), i32(z["new"]), i32([int(d) for d in z["done"]])
        st["free"] = torch.full((z["pool"],), -1, dtype=torch.int32, device="cuda")
        left = ids[sum(own_blocks):]
        st["free"][: left.numel()] = left
        st["free_count"] = i32([left.numel()])
        st["out"] = dict(row_starts=torch.zeros(S + 1, dtype=torch.int32, device="cuda"), slots=torch.zeros(z["rows"], dtype=torch.int32, device="cuda"),
                         positions=torch.zeros(z["rows"], dtype=torch.int32, device="cuda"), kv_lens=torch.zeros(S, dtype=torch.int32, device="cuda"),
                         free_count=i32([0]), status=i32([0]))
        return st
    KV, D = case["kv_heads"], case["dim"]
    st["scales"] = torch.empty((z["pool"], KV, 2), device="cuda")
    for k, (side, spread) in enumerate((("keys", 3.0), ("values", 1.0))):
        x = _side(g, (z["pool"], KV, B, D), spread)
        scale = _pow2_scale(x.abs().amax((2, 3)))
        st["scales"][:, :, k] = scale
        st[side] = _encode(x, scale[:, :, None, None])
        del x
    kv = torch.tensor([b + n for b, n in zip(z["before"], z["new"])], device="cuda")
    st["kv_lens"] = kv.to(torch.int32)
    if case["op"] == "store":
        dt = DTYPES[case["dtype"]]
        # the new rows are now and then larger than what their block holds
        lift = 1.0 + 3.0 * (torch.rand((z["rows"], 1, 1), generator=g, device="cuda") > 0.9)
        st["k"] = (torch.randn((z["rows"], KV, D), generator=g, device="cuda") * lift).to(dt)
        st["v"] = (torch.randn((z["rows"], KV, D), generator=g, device="cuda") * lift).to(dt)
        row = torch.arange(z["rows"], device="cuda")
        total = sum(z["new"])
        seq = (torch.searchsorted(st["row_starts"].long(), row, right=True) - 1).clamp(max=S - 1)
        pos = torch.tensor(z["before"], device="cuda")[seq] + row - st["row_starts"].long()[seq]
        pos = torch.where(row < total, pos, 0)
        slots = tables[seq, pos // B].long() * B + pos % B
        st["slots"] = torch.where(row < total, slots, -1).to(torch.int32)
    else:
        # what lies behind a sequence's last token was never written: any byte may stand there, NaN too
        last = tables[torch.arange(S, device="cuda"), ((kv - 1).clamp(min=0)) // B].long()
        has = kv > 0
        tail = torch.arange(B, device="cuda")[None, :] >= (kv - (kv - 1) // B * B)[:, None]
        for side in ("keys", "values"):
            raw = st[side].view(torch.uint8)
            raw[last[has]] = torch.where(tail[has][:, None, :, None], torch.full_like(raw[last[has]], 0x7F), raw[last[has]])
        dt = DTYPES[case["dtype"]]
        st["q"] = (1.25 * torch.randn((z["rows"], case["heads"], D), generator=g, device="cuda")).to(dt)
        st["gate"] = torch.randn((z["rows"], case["heads"], 2 * D), generator=g, device="cuda") if case["gate"] else None
        st["out"] = torch.zeros_like(st["q"])
    if own:
        import saetta_macqwen_b200 as sa

        st["cache"] = sa.PagedKvCache.wrap(0, KV, D, B, z["pool"], st["keys"], st["values"], st["scales"])
        if case["op"] == "attend":
            st["op"] = sa.PagedAttention(0, case["heads"], KV, D)
    return st


def run(st):
    op = st["case"]["op"]
    if own:
        return {"assign": _own_assign, "store": _own_store, "attend": _own_attend}[op](st)
    return {"assign": _assign, "store": _store, "attend": _attend}[op](st)


def _own_assign(st):
    import saetta_macqwen_b200 as sa

    o = st["out"]
    sa.paged_assign(0, st["case"]["seqs"], st["case"]["block"], st["kv_lens"], st["new"], st["free"], st["z"]["pool"], st["free_count"], st["tables"], st["z"]["width"],
                    o["row_starts"], o["slots"], o["positions"], st["z"]["rows"], o["kv_lens"], o["free_count"], o["status"], finished=st["done"])
    return dict(o, tables=st["tables"], free=st["free"])


def _own_store(st):
    st["cache"].store(st["k"], st["v"], st["slots"], st["z"]["rows"], dtype={"f32": -1, "f16": 0, "bf16": 1}[st["case"]["dtype"]])
    return dict(keys=st["keys"], values=st["values"], scales=st["scales"])


def _own_attend(st):
    c, z = st["case"], st["z"]
    dt = {"f16": 0, "bf16": 1}[c["dtype"]]
    st["op"].record(st["cache"], st["q"], dt, z["rows"], c["seqs"], st["row_starts"], st["kv_lens"], st["tables"], z["width"], c["new_hi"],
                    c["dim"] ** -0.5, st["out"], dt, q_and_gate=st["gate"])
    return st["out"]


def _assign(st):
    c, z = st["case"], st["z"]
    S, B, W = c["seqs"], c["block"], z["width"]
    lens, new, done = st["kv_lens"].long(), st["new"].long(), st["done"] != 0
    tables, free, count = st["tables"], st["free"], st["free_count"].long()
    col = torch.arange(W, device="cuda")[None, :]
    # finished requests put their blocks on top of the free stack, in sequence and table order
    back = done[:, None] & (col < ((lens + B - 1) // B)[:, None])
    at = (count + back.reshape(-1).cumsum(0) - 1).reshape(S, W)
    stack = torch.cat([free, free.new_zeros(1)])  # the last place takes what is not given back
    stack.scatter_(0, torch.where(back, at, free.numel()).reshape(-1), tables.reshape(-1))
    free.copy_(stack[:-1])
    count = count + back.sum()
    lens = torch.where(done, 0, lens)
    have = (lens + B - 1) // B
    need = (lens + new + B - 1) // B - have
    first = need.cumsum(0) - need
    takes = (col >= have[:, None]) & (col < (have + need)[:, None])
    nth = first[:, None] + col - have[:, None]
    tables.copy_(torch.where(takes, free[(count - 1 - nth).clamp(0, free.numel() - 1)], tables))
    total = new.cumsum(0)
    starts = torch.cat([total.new_zeros(1), total])
    row = torch.arange(z["rows"], device="cuda")
    seq = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=S - 1)
    pos = lens[seq] + row - starts[seq]
    real = row < total[-1]
    slot = tables[seq, torch.where(real, pos // B, 0)].long() * B + pos % B
    i32 = torch.int32
    return dict(row_starts=starts.to(i32), slots=torch.where(real, slot, -1).to(i32), positions=torch.where(real, pos, -1).to(i32), kv_lens=(lens + new).to(i32),
                free_count=(count - need.sum()).to(i32), status=torch.zeros(1, dtype=i32, device="cuda"), tables=tables, free=free)


def _store(st):
    B, KV = st["case"]["block"], st["case"]["kv_heads"]
    slots = st["slots"].long()
    real = slots >= 0
    slots = slots[real]
    which, of_row = torch.unique(slots // B, return_inverse=True)
    off = slots % B
    first = torch.full_like(which, B).scatter_reduce_(0, of_row, off, "amin")  # the first offset written of each block
    for k, (x, pages) in enumerate(((st["k"], st["keys"]), (st["v"], st["values"]))):
        x = x[real].float()
        amax = x.abs().amax(2)
        amax = torch.zeros((which.numel(), KV), device="cuda").scatter_reduce_(0, of_row[:, None].expand(-1, KV), amax, "amax")
        was = st["scales"][which, :, k]
        scale = torch.where(first[:, None] == 0, _pow2_scale(amax), torch.maximum(was, _pow2_scale(amax)))
        codes = pages[which]
        old = torch.arange(B, device="cuda")[None, :] < first[:, None]
        again = (codes.float() * (was / scale)[:, :, None, None]).to(torch.float8_e4m3fn)
        codes = torch.where(old[:, None, :, None], again.view(torch.uint8), codes.view(torch.uint8))
        codes[of_row, :, off] = _encode(x, scale[of_row][:, :, None]).view(torch.uint8)
        pages.view(torch.uint8)[which] = codes
        st["scales"][which, :, k] = scale
    return dict(keys=st["keys"], values=st["values"], scales=st["scales"])


def _attend(st):
    c, z = st["case"], st["z"]
    S, B, H, KV, D = c["seqs"], c["block"], c["heads"], c["kv_heads"], c["dim"]
    G, N = H // KV, max(z["new"])
    rows, W = st["q"].shape[0], z["width"]
    if N == 0:
        return torch.zeros_like(st["q"])
    starts, kv = st["row_starts"].long(), st["kv_lens"].long()
    n = starts[1:] - starts[:-1]
    inside = torch.arange(W * B, device="cuda")[None, :] < kv[:, None]  # [S, L]
    page = st["tables"].long().clamp(min=0)

    def side(pages, k):
        x = pages[page].float() * st["scales"][page][:, :, :, k, None, None]  # [S, W, KV, B, D]
        x = x.transpose(1, 2).reshape(S, KV, W * B, D)
        return x.masked_fill_(~inside[:, None, :, None], 0.0)

    i = torch.arange(N, device="cuda")
    at = (starts[:-1, None] + i[None, :]).clamp(max=rows - 1)  # [S, N]
    q = st["q"][at].float().reshape(S, N, KV, G, D).transpose(1, 2).reshape(S, KV, N * G, D)
    s = (q @ side(st["keys"], 0).transpose(2, 3)).mul_(D ** -0.5)
    sees = torch.arange(W * B, device="cuda")[None, None, :] < (kv[:, None] - n[:, None] + i[None, :] + 1)[:, :, None]
    sees &= (i[None, :] < n[:, None])[:, :, None]
    s = s.reshape(S, KV, N, G, W * B).masked_fill_(~sees[:, None, :, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True).clamp_(min=-1e30)
    s = s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = s.reshape(S, KV, N * G, W * B) @ side(st["values"], 1)
    o = o.reshape(S, KV, N, G, D) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(S, N, H, D)
    row = torch.arange(rows, device="cuda")
    seq = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=S - 1)
    out = o[seq, (row - starts[seq]).clamp(max=N - 1)]
    if st["gate"] is not None:
        out = out / (1.0 + torch.exp(-st["gate"][:, :, D:]))
    return torch.where((row < starts[-1])[:, None, None], out, 0.0).to(st["q"].dtype)


def work(case):
    z = _sizes(case)
    B = case["block"]
    total = sum(z["new"])
    if case["op"] == "assign":
        back = sum(_blocks(b, B) for b, d in zip(z["before"], z["done"]) if d)
        start = [0 if d else b for b, d in zip(z["before"], z["done"])]
        taken = sum(_blocks(b + n, B) - _blocks(b, B) for b, n in zip(start, z["new"]))
        return {"bytes": 4 * (5 * case["seqs"] + 1) + 8 * (back + taken) + 8 * z["rows"] + 12, "flops": 0}
    KV, D = case["kv_heads"], case["dim"]
    if case["op"] == "store":
        return {"bytes": total * KV * D * 2 * ((4 if case["dtype"] == "f32" else 2) + 1) + 4 * z["rows"] + sum(_blocks(n, B) for n in z["new"]) * KV * 8, "flops": 0}
    H = case["heads"]
    kv = [b + n if n else 0 for b, n in zip(z["before"], z["new"])]  # a sequence without rows is not read
    pairs = sum(n * b + n * (n + 1) // 2 for b, n in zip(z["before"], z["new"]))
    moved = sum(kv) * KV * D * 2 + sum(_blocks(k, B) for k in kv) * (KV * 8 + 4) + total * H * D * (4 + (4 if case["gate"] else 0)) + 8 * case["seqs"]
    return {"bytes": max(moved, 64), "flops": 4 * D * H * pairs}


def exact(case, seed):
    if case["op"] == "assign":
        return None  # whole numbers
    st = prepare(case, seed)
    return _exact_store(st) if case["op"] == "store" else _exact_attend(st)


def _exact_round(y):
    """y in f64 to the nearest e4m3 value, ties to even: steps of 2^(floor(log2 |y|) - 3), of 2^-9 below 2^-6."""
    _, e = torch.frexp(y)
    step = _exact_pow2((e - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def _exact_pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_store(st):
    """Block by block: the run of new rows, its largest value, the block's scale, the codes."""
    B, KV = st["case"]["block"], st["case"]["kv_heads"]
    slots = st["slots"].tolist()
    scales = st["scales"].double()
    want = {"scales": scales}
    for k, (x, side) in enumerate((("k", "keys"), ("v", "values"))):
        new, pages = st[x].double(), st[side].double()
        r = 0
        while r < len(slots):
            if slots[r] < 0:
                r += 1
                continue
            end = r + 1
            while end < len(slots) and slots[end] >= 0 and slots[end] // B == slots[r] // B:
                end += 1
            b, off = slots[r] // B, slots[r] % B
            amax = new[r:end].abs().amax((0, 2))
            e = torch.ceil(torch.log2((amax / E4M3_MAX).clamp(min=2.0 ** -126)))
            e = torch.where(amax > E4M3_MAX * _exact_pow2(e), e + 1, e)  # log2 may be off by its last place at a power of two
            e = torch.where((amax <= E4M3_MAX * _exact_pow2(e - 1)) & (e > -126), e - 1, e)
            scale = _exact_pow2(e)
            if off:
                scale = torch.maximum(scale, scales[b, :, k])
                pages[b, :, :off] = _exact_round(pages[b, :, :off] * (scales[b, :, k] / scale)[:, None, None])
            pages[b, :, off:off + end - r] = _exact_round(new[r:end].transpose(0, 1) / scale[:, None, None])
            scales[b, :, k] = scale
            r = end
        want[side] = pages
    return want


def _exact_attend(st):
    """Sequence by sequence and kv head by kv head, a few rows at a time."""
    c, z = st["case"], st["z"]
    B, H, KV, D = c["block"], c["heads"], c["kv_heads"], c["dim"]
    G = H // KV
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for s in range(c["seqs"]):
        n, kv = z["new"][s], z["before"][s] + z["new"][s]
        if n:
            page = st["tables"][s, : _blocks(kv, B)].long()
            for h in range(KV):
                k, v = ((st[side][page, h].double() * st["scales"][page, h, i].double()[:, None, None]).reshape(-1, D)[:kv] for i, side in enumerate(("keys", "values")))
                q = st["q"][row:row + n, h * G:(h + 1) * G].double()
                for lo in range(0, n, 512):
                    hi = min(n, lo + 512)
                    w = torch.einsum("ngd,kd->ngk", q[lo:hi], k) / D ** 0.5
                    hidden = torch.arange(kv, device="cuda")[None, :] > (kv - n + torch.arange(lo, hi, device="cuda"))[:, None]
                    w = torch.softmax(w.masked_fill(hidden[:, None, :], float("-inf")), -1)
                    out[row + lo:row + hi, h * G:(h + 1) * G] = torch.einsum("ngk,kd->ngd", w, v)
        row += n
    if st["gate"] is not None:
        out[:row] *= torch.sigmoid(st["gate"][:row, :, D:].double())
    return out

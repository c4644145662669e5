"""Plain 64-bit restatements of the paged cache's operators, and inputs for their tests."""
import numpy as np


def e4m3_table():
    """The value of each of the 256 codes (sign, 4 exponent bits of bias 7, 3 mantissa bits; 0x7F and 0xFF are NaN)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


TABLE = e4m3_table()


def e4m3_encode(y):
    """f64 to codes: nearest, ties to the even code, saturating at 448; NaN to 0x7F."""
    y = np.asarray(y, np.float64)
    grid = TABLE[:127]
    mag = np.minimum(np.abs(y), 448.0)
    mag = np.where(np.isnan(y), 0.0, mag)
    hi = np.clip(np.searchsorted(grid, mag), 1, 126)
    lo = hi - 1
    dl, dh = mag - grid[lo], grid[hi] - mag
    code = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    code = np.where(np.isnan(y), 127, code)
    return (code | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def pow2_scale(amax):
    e = np.full(np.shape(amax), -126)
    m, x = np.frexp(np.asarray(amax, np.float64))
    e = np.where(np.asarray(amax) > 0, np.where(m > 0.875, x - 8, x - 9), e)
    return 2.0 ** np.maximum(e, -126).astype(np.float64)


def ref_store(keys, values, scales, k, v, slots, block):
    """keys, values: codes [blocks][kv][block][dim]; scales f64 [blocks][kv][2]; k, v [rows][kv][dim].  In place."""
    r = 0
    while r < len(slots):
        if slots[r] < 0:
            r += 1
            continue
        end = r + 1
        while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] // block == slots[r] // block:
            end += 1
        b, off = slots[r] // block, slots[r] % block
        for side, (x, pages) in enumerate(((k, keys), (v, values))):
            run = np.asarray(x[r:end], np.float64)
            fin = np.where(np.isfinite(run), np.abs(run), 0.0)
            s = pow2_scale(fin.max((0, 2)))
            if off:
                was = scales[b, :, side]
                s = np.maximum(s, was)
                for h in range(pages.shape[1]):
                    if s[h] != was[h]:
                        pages[b, h, :off] = e4m3_encode(TABLE[pages[b, h, :off]] * (was[h] / s[h]))
            pages[b, :, off:off + end - r] = e4m3_encode(run.transpose(1, 0, 2) / s[:, None, None])
            scales[b, :, side] = s
        r = end


def ref_assign(lens, new, finished, free, count, tables, block, rows_cap):
    """One scheduling step on Python lists; returns (row_starts, slots, positions, lens, count), tables and free in place."""
    blocks = lambda n: (n + block - 1) // block  # noqa: E731
    lens = list(lens)
    for s, f in enumerate(finished):
        if f:
            for j in range(blocks(lens[s])):
                free[count] = tables[s][j]
                count += 1
            lens[s] = 0
    starts, slots, pos = [0], [], []
    for s, n in enumerate(new):
        for j in range(blocks(lens[s]), blocks(lens[s] + n)):
            count -= 1
            tables[s][j] = free[count]
        for p in range(lens[s], lens[s] + n):
            slots.append(tables[s][p // block] * block + p % block)
            pos.append(p)
        lens[s] += n
        starts.append(len(slots))
    pad = rows_cap - len(slots)
    return starts, slots + [-1] * pad, pos + [-1] * pad, lens, count


def ref_attend(q, keys, values, scales, tables, starts, kv_lens, block, scale, gate=None):
    """q f64 [rows][heads][dim]; codes, scales as in ref_store.  Returns (out, bounds): `bounds` holds, per
    (row, head), what the error bounds of the kernels go by: absv (the average of |v| under the weights), mag (the largest scale * sum of
    |q k|), top (the largest |s|), wide (largest weight, times the
    sequence's largest value scale, times the sum of |code|), qwide (largest |q| times the largest
    scale * sum of |k|)."""
    rows, heads, dim = q.shape
    kv_heads = keys.shape[1]
    G = heads // kv_heads
    out, absv = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    mag, top, qwide, wide = (np.zeros((rows, heads)) for _ in range(4))
    wide = np.zeros((rows, heads, dim))
    for s in range(len(kv_lens)):
        lo, hi, kv = starts[s], starts[s + 1], kv_lens[s]
        n = hi - lo
        if not n or not kv:
            continue
        pages = tables[s][: (kv + block - 1) // block]
        for h in range(kv_heads):
            k, v = ((TABLE[side[pages, h]] * scales[pages, h, i][:, None, None]).reshape(-1, dim)[:kv] for i, side in enumerate((keys, values)))
            qs = q[lo:hi, h * G:(h + 1) * G]
            w = np.einsum("ngd,kd->ngk", qs, k) * scale
            hidden = np.arange(kv)[None, :] > (kv - n + np.arange(n))[:, None]
            a = np.einsum("ngd,kd->ngk", np.abs(qs), np.abs(k)) * scale
            a, aw = np.where(hidden[:, None], 0, a), np.where(hidden[:, None], 0, np.abs(w))
            w = np.where(hidden[:, None], -np.inf, w)
            m = w.max(-1, keepdims=True)
            p = np.exp(w - np.where(np.isfinite(m), m, 0.0))
            t = p.sum(-1, keepdims=True)
            p = p / np.where(t > 0, t, 1.0)
            out[lo:hi, h * G:(h + 1) * G] = np.einsum("ngk,kd->ngd", p, v)
            absv[lo:hi, h * G:(h + 1) * G] = np.einsum("ngk,kd->ngd", p, np.abs(v))
            at = (slice(lo, hi), slice(h * G, (h + 1) * G))
            mag[at], top[at] = a.max(-1), aw.max(-1)
            qwide[at] = np.abs(qs).max(-1) * scale * np.abs(k).sum(-1).max()
            vs = np.repeat(scales[pages, h, 1], block)[:kv]
            wide[at] = p.max(-1)[..., None] * vs.max() * np.einsum("ngk,kd->ngd", ~hidden[:, None] & np.ones((1, G, 1), bool), np.abs(v / vs[:, None]))
    if gate is not None:
        g = 1.0 / (1.0 + np.exp(-gate))
        out, absv, wide = out * g, absv * g, wide * g
    return out, dict(absv=absv, mag=mag, top=top, wide=wide, qwide=qwide)

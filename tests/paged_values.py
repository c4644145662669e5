"""Sequences of chosen keys, values and queries in a paged cache, and what attention over them is in 64 bits."""
import numpy as np

import saetta_macqwen_b200 as sa


def torch_type(dt):
    import torch

    return {sa.F32: torch.float32, sa.F16: torch.float16, sa.BF16: torch.bfloat16}[dt]


def rounded(x, dt):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch_type(dt)).double().numpy()


def bf16(p):
    """Nonnegative weights rounded to 8 significant bits."""
    m, e = np.frexp(p)
    return np.ldexp(np.rint(m * 256), e - 8)


class Sequences:
    """seqs: [(q [n][heads][dim], k [kv][kv_heads][dim], v)], f64; cached as e4m3 with a power-of-two scale for each block, head and side."""

    def __init__(self, seqs, block, q_dt, scale, seed=0, max_rows=None):
        import torch

        self.block, self.q_dt, self.scale = block, q_dt, scale
        self.heads, self.dim, self.kv_heads = seqs[0][0].shape[1], seqs[0][0].shape[2], seqs[0][1].shape[1]
        need = [-(-len(k) // block) for _, k, _ in seqs]
        pool, self.width = sum(need) + 1, max(need)
        ids = np.random.default_rng(seed).permutation(pool)
        tables = np.full((len(seqs), self.width), -1, np.int64)
        sides, self.kv = [np.zeros((pool, self.kv_heads, block, self.dim)) for _ in range(2)], []
        at = 0
        for s, (_, k, v) in enumerate(seqs):
            tables[s, :need[s]] = ids[at:at + need[s]]
            at += need[s]
            for side, x in zip(sides, (k, v)):
                for j in range(need[s]):
                    part = x[j * block:(j + 1) * block]
                    side[tables[s, j], :, :len(part)] = part.transpose(1, 0, 2)
        self.tables = tables
        self.scales = np.ones((pool, self.kv_heads, 2))
        self.codes = []
        for i, side in enumerate(sides):
            m, e = np.frexp(np.abs(np.where(np.isfinite(side), side, 0)).max((2, 3)))
            self.scales[..., i] = 2.0 ** np.maximum(np.where(m > 0.875, e - 8, e - 9), -126)
            y = torch.from_numpy((side / self.scales[..., i][:, :, None, None]).astype(np.float32))
            code = y.to(torch.float8_e4m3fn)
            self.codes.append(code)
            back = code.double().numpy() * self.scales[..., i][:, :, None, None]
            self.kv.append([back[tables[s, :need[s]]].transpose(1, 0, 2, 3).reshape(self.kv_heads, -1, self.dim)[:, :len(seqs[s][1])] for s in range(len(seqs))])
        self.q = [rounded(q, q_dt) for q, _, _ in seqs]
        self.lens = [len(k) for _, k, _ in seqs]
        self.starts = np.concatenate([[0], np.cumsum([len(q) for q in self.q])]).tolist()
        self.max_rows = max(len(q) for q in self.q) if max_rows is None else max_rows
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
        self.dev = [torch.from_numpy(np.concatenate(self.q).astype(np.float32)).to(torch_type(q_dt)).cuda(), i32(self.starts), i32(self.lens), i32(tables)]
        self.bufs = [c.view(torch.uint8).cuda() for c in self.codes] + [torch.from_numpy(self.scales.astype(np.float32)).cuda()]
        self.cache = sa.PagedKvCache.wrap(0, self.kv_heads, self.dim, block, pool, *self.bufs)

    def run(self, max_rows=None, op=None):
        """The kernel's output (f32) as f64, the few-rows or the many-rows kernel by max_rows."""
        import torch

        out = torch.full((self.starts[-1], self.heads, self.dim), 7.0, device="cuda")
        op = op or sa.PagedAttention(0, self.heads, self.kv_heads, self.dim)
        op.record(self.cache, self.dev[0], self.q_dt, self.starts[-1], len(self.lens), *self.dev[1:], self.width, self.max_rows if max_rows is None else max_rows,
                  self.scale, out, sa.F32)
        torch.cuda.synchronize()
        assert op.device_status() == 0
        return out.double().cpu().numpy()

    def exact(self, weights=lambda p: p):
        """softmax(scale q k) v; with the weights (the largest of a row is 1) rounded by `weights`.  Also the weighted average of |v|, the largest |score|,
        and `edge`: over tiles of 128 keys, the largest weight times value scale that the row sees there, times the sum of |code|."""
        out, absv, edge = np.zeros((3, self.starts[-1], self.heads, self.dim))
        top = np.zeros((self.starts[-1], self.heads))
        G = self.heads // self.kv_heads
        for s, q in enumerate(self.q):
            n, kv = len(q), self.lens[s]
            rows = slice(self.starts[s], self.starts[s + 1])
            for h in range(self.heads):
                k, v = self.kv[0][s][h // G], self.kv[1][s][h // G]
                vs = np.repeat(self.scales[self.tables[s, :-(-kv // self.block)], h // G, 1], self.block)[:kv]
                code = np.abs(v / vs[:, None])
                for i0 in range(0, n, 64):
                    i1 = min(n, i0 + 64)
                    w = q[i0:i1, h] @ k.T * self.scale
                    seen = np.arange(kv)[None, :] <= (kv - n + np.arange(i0, i1))[:, None]
                    w = np.where(seen, w, -np.inf)
                    m = w.max(1, keepdims=True)
                    p = np.exp(w - np.where(np.isfinite(m), m, 0))
                    t = p.sum(1, keepdims=True)
                    at = (slice(rows.start + i0, rows.start + i1), h)
                    out[at] = weights(p) @ v / np.where(t > 0, t, 1)
                    absv[at] = p @ np.abs(v) / np.where(t > 0, t, 1)
                    top[at] = np.where(seen, np.abs(w), 0).max(1)
                    for j in range(0, kv, 128):
                        t128 = slice(j, j + 128)
                        edge[at] += (p[:, t128] * vs[t128]).max(1, keepdims=True) * (seen[:, t128] @ code[t128]) / np.where(t > 0, t, 1)
        return out, absv, top, edge


def off(a, b):
    """How far a is from b, relative, as a whole."""
    return np.linalg.norm(a - b) / np.linalg.norm(b)

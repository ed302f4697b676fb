"""Plain 64-bit forms of the paged cache, the attention over it and the grouped router, and pages to run them on."""
import numpy as np

HALF_STEP = 2.0 ** -24  # an f32 rounding is off by at most this, relative to the value


def q8_levels(x):
    """Q8_0 of f32 rows, every step in f32 (src/backend/quant/q8k.zig:49-69): int8 levels and f16 scales."""
    b = np.ascontiguousarray(x, dtype=np.float32).reshape(-1, 32)
    d = np.abs(b).max(axis=1, keepdims=True) / np.float32(127)
    with np.errstate(divide="ignore"):
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d).astype(np.float32)
    y = (b * inv).astype(np.float32).astype(np.float64)
    q = np.clip(np.sign(y) * np.floor(np.abs(y) + 0.5), -127, 127).astype(np.int8)
    with np.errstate(over="ignore"):
        scale = d.astype(np.float16)
    return q.reshape(x.shape), scale.reshape(*x.shape[:-1], x.shape[-1] // 32)


def held(kind, x):
    """What a cache of this format holds of f32 rows, in 64 bits."""
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float64)
    q, s = q8_levels(x)
    return q.astype(np.float64) * np.repeat(s.astype(np.float64), 32, axis=-1)


def attention(q, keys, values, scale, window=0):
    """q [heads][d] against keys, values [len][kv_heads][d] (64-bit): out, stats, and sum p|v| / sum p per element."""
    heads, d = q.shape
    n, kv_heads, _ = keys.shape
    out, stats, weight = np.zeros((heads, d)), np.zeros((heads, 2)), np.zeros((heads, d))
    stats[:, 0] = -3.4e38
    first = max(0, n - window) if window else 0
    most = 0.0
    for h in range(heads):
        if n == 0:
            continue
        k, v = keys[first:, h // (heads // kv_heads)], values[first:, h // (heads // kv_heads)]
        x = (k @ q[h].astype(np.float64)) * scale
        most = max(most, float((np.abs(k) @ np.abs(q[h].astype(np.float64))).max() * abs(scale)))
        p = np.exp(x - x.max())
        out[h], weight[h] = (p @ v) / p.sum(), (p @ np.abs(v)) / p.sum()
        stats[h] = x.max(), p.sum()
    return out, stats, weight, most


def attention_slack(weight, most, d, n):
    """How far f32 arithmetic may be off, element by element. A score sums d products whose absolute sum is at most
    `most`: off by (d + 4) half steps of that (products, additions, the scale). exp turns a score's error into a relative
    one of the weight and adds 4 half steps; a weight enters numerator and denominator (factor 2), and the two sums over
    n keys add at most n + 8 half steps each, as do the joins of partial sums."""
    return (2 * ((d + 4) * most + 4) + 2 * (n + 8)) * HALF_STEP * weight + 1e-30


def router(logits, k, sigmoid=False, bias=None, groups=1, kept=1, top2=False, normalize=True, scale=1.0):
    x = logits.astype(np.float64)
    t, e = x.shape
    closed = np.isnan(x) | np.isneginf(x)
    if sigmoid:
        with np.errstate(over="ignore"):
            score = 1 / (1 + np.exp(-x))
    else:
        top = np.where(closed, -np.inf, x).max(axis=1, keepdims=True)
        with np.errstate(invalid="ignore"):
            score = np.where(x == top, 1.0, np.exp(x - top))
        score = np.where(closed, 0, score)
        total = score.sum(axis=1, keepdims=True)
        score = score / np.where(total > 0, total, 1)
    score = np.where(closed, 0, score)
    key = np.where(closed, -np.inf, score + (0 if bias is None else bias.astype(np.float64)))
    if groups > 1:
        size = e // groups
        best = -np.sort(-key.reshape(t, groups, size), axis=2)
        rank = best[:, :, :2].sum(axis=2) if top2 and size > 1 else best[:, :, 0]
        shut = np.argsort(-rank, axis=1, kind="stable")[:, kept:]
        view = key.reshape(t, groups, size)
        view[np.arange(t)[:, None], shut] = -np.inf
        key = view.reshape(t, e)
    chosen = np.argsort(-key, axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(score, chosen, axis=1)
    if normalize:
        total = w.sum(axis=1, keepdims=True)
        w = w / np.where(total > 0, total, 1)
    return chosen.astype(np.int32), w * scale


class Cache:
    """Pages on the GPU whose every slot starts as garbage (NaN where the type has one), with the rows written so far."""

    def __init__(self, P, kind, lens, page, kv_heads, d, rng, page_stride=0, scale_stride=0, spare=2):
        import torch

        self.P, self.kind, self.page, self.kv, self.d, self.lens = P, kind, page, kv_heads, d, list(lens)
        need = [-(-n // page) for n in lens]
        self.n_pages, self.max_pages = sum(need) + spare, max(max(need), 1)
        order = rng.permutation(self.n_pages)
        table = np.full((len(lens), self.max_pages), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.table_host = table
        self.table = torch.from_numpy(table).cuda()
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32).cuda()
        elems = kv_heads * page * d
        self.stride, self.sstride = page_stride or elems, scale_stride or elems // 32
        if kind == "f16":
            self.k = torch.full((self.n_pages * self.stride,), float("nan"), dtype=torch.float16).cuda()
            self.v, self.ks, self.vs = self.k.clone(), None, None
        else:
            self.k = torch.full((self.n_pages * self.stride,), -128, dtype=torch.int8).cuda()
            self.v = self.k.clone()
            self.ks = torch.full((self.n_pages * self.sstride,), float("nan"), dtype=torch.float16).cuda()
            self.vs = self.ks.clone()
        self.pages = P.KvPages(P.KV_F16 if kind == "f16" else P.KV_Q8_0, self.k, self.v, self.ks, self.vs, self.n_pages, page, kv_heads, d,
                               page_stride, scale_stride)
        torch.cuda.synchronize()

    def append(self, k, v, seq, pos, stream=0):
        """k, v f32 tensors or arrays [rows][kv_heads * d]; blocking."""
        import torch

        keep = [torch.as_tensor(x).cuda() for x in (k, v, np.asarray(seq, np.int32), np.asarray(pos, np.int32))]
        torch.cuda.synchronize()
        self.P.kv_append_dev(self.pages, *keep, len(seq), self.table, len(self.lens), self.max_pages, stream=stream)
        self.P.synchronize()

    def fill(self, rng, gain=1.0):
        """Every position of every sequence, in scattered order: the f32 rows as written, by sequence."""
        seq = np.repeat(np.arange(len(self.lens)), self.lens)
        pos = np.concatenate([np.arange(n) for n in self.lens]) if len(seq) else np.zeros(0, int)
        k = (rng.standard_normal((len(seq), self.kv * self.d)) * gain).astype(np.float32)
        v = (rng.standard_normal((len(seq), self.kv * self.d)) * gain).astype(np.float32)
        if len(seq):
            order = rng.permutation(len(seq))
            self.append(k[order], v[order], seq[order], pos[order])
        cut = np.cumsum([0] + self.lens)
        shape = (-1, self.kv, self.d)
        return [(k[a:b].reshape(shape), v[a:b].reshape(shape)) for a, b in zip(cut[:-1], cut[1:])]

    def attend(self, q, heads, scale, window=0, max_len=0, stats=False, workspace=True, stream=0):
        import torch

        n = len(self.lens)
        out = torch.full((n + 1, heads, self.d), float("nan")).cuda()  # a row behind the last sequence stays as it is
        st = torch.full((n, heads, 2), float("nan")).cuda() if stats else None
        q_dev = torch.as_tensor(q).cuda()
        size = self.P.attn_paged_workspace_bytes(self.pages, n, heads, max_len or self.max_pages * self.page)
        ws = torch.full((max(size, 16),), 0xFF, dtype=torch.uint8).cuda() if workspace else None
        torch.cuda.synchronize()
        self.P.attn_paged_dev(self.pages, q_dev, out, self.table, self.lens_dev, n, self.max_pages, heads, scale, window=window, max_len=max_len,
                              stats_dev=st, workspace=ws, workspace_bytes=size if workspace else 0, stream=stream)
        torch.cuda.synchronize()
        self.P.synchronize()
        assert bool(torch.isnan(out[n]).all())
        return out[:n].cpu().numpy(), st.cpu().numpy() if stats else None


def check_attention(cache, rows, q, got, scale, window=0, stats=None, heads=None):
    """Every element inside the f32 slack; all together within 48 half steps of the result's norm (independent roundings
    of a score, some sqrt(d) <= 16 half steps of a sum about three times its result, and a handful for the rest)."""
    err2 = ref2 = 0.0
    for s, (k, v) in enumerate(rows):
        want, st, weight, most = attention(q[s], held(cache.kind, k), held(cache.kind, v), scale, window)
        slack = attention_slack(weight, most, cache.d, len(k))
        assert np.all(np.abs(got[s] - want) <= slack), (s, len(k), float(np.max(np.abs(got[s] - want) / slack)))
        err2, ref2 = err2 + float(((got[s] - want) ** 2).sum()), ref2 + float((want ** 2).sum())
        if stats is not None:
            if len(k) == 0:
                assert np.all(stats[s] == np.array([-3.4e38, 0.0], np.float32))
            else:
                off = ((cache.d + 4) * most + 4) * HALF_STEP
                assert np.all(np.abs(stats[s][:, 0] - st[:, 0]) <= off + np.abs(st[:, 0]) * HALF_STEP)
                assert np.all(np.abs(stats[s][:, 1] / st[:, 1] - 1) <= 2 * off + (len(k) + 16) * HALF_STEP)
    if ref2:
        assert (err2 / ref2) ** 0.5 <= 48 * HALF_STEP, (err2 / ref2) ** 0.5

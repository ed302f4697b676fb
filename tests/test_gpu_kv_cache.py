"""Paged key-value cache on the GPU: rows written as f16 or Q8_0 and read back, against the formats' laws."""
import numpy as np
import pytest

from kv_reference import Cache, held, q8_levels

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    from fucina_b200 import provider

    provider.init(0)
    return provider


def read(P, cache, seq, pos, half=False, sides=(True, True), stream=0):
    import torch

    rows = (len(seq), cache.kv, cache.d)
    outs = [torch.full(rows, 7.0, dtype=torch.float16 if half else torch.float32).cuda() if s else None for s in sides]
    at = [torch.as_tensor(np.asarray(x, np.int32)).cuda() for x in (seq, pos)]
    torch.cuda.synchronize()
    P.kv_read_dev(cache.pages, outs[0], outs[1], half, at[0], at[1], len(seq), cache.table, len(cache.lens), cache.max_pages, stream=stream)
    torch.cuda.synchronize()
    P.synchronize()
    return [None if o is None else o.cpu().numpy() for o in outs]


@pytest.mark.parametrize("kind,lens,page,kv,d", [
    ("f16", [1], 16, 1, 16),
    ("f16", [37, 0, 130], 16, 3, 80),
    ("f16", [257, 64], 48, 2, 256),
    ("q8_0", [1], 16, 1, 32),
    ("q8_0", [63, 0, 65, 17], 64, 8, 128),
    ("q8_0", [300], 256, 5, 96),
    ("q8_0", [33, 1000], 32, 1, 256),
])
@pytest.mark.parametrize("half", [False, True])
def test_rows_come_back_as_the_format_holds_them(P, kind, lens, page, kv, d, half):
    rng = np.random.default_rng(len(lens) + d)
    cache = Cache(P, kind, lens, page, kv, d, rng)
    rows = cache.fill(rng)
    seq = np.repeat(np.arange(len(lens)), lens)
    pos = np.concatenate([np.arange(n) for n in lens])
    order = rng.permutation(len(seq))
    got = read(P, cache, seq[order], pos[order], half)
    for side in (0, 1):
        want = np.concatenate([held(kind, r[side]) for r in rows])[order]
        assert np.array_equal(got[side], want.astype(np.float16 if half else np.float32))


def test_q8_blocks_equal_the_library_encoder(P):
    import torch

    rng = np.random.default_rng(5)
    kv, d, n = 2, 128, 64
    x = (rng.standard_normal((n, kv * d)) * np.exp(rng.uniform(-12, 8, (n, 1)))).astype(np.float32)
    x[3] = 0
    x[4, 5] = 3e6  # its scale is still a finite f16
    cache = Cache(P, "q8_0", [n], 64, kv, d, rng)
    cache.append(x, x, np.zeros(n), np.arange(n))
    blocks = torch.zeros(n * kv * d // 32, 34, dtype=torch.uint8).cuda()
    src = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    P.quantize_acts_q8_0_dev(src, n, kv * d, blocks)
    P.synchronize()
    blocks = blocks.cpu().numpy().reshape(n, kv, d // 32, 34)
    page = int(cache.table_host[0, 0])
    k = cache.k.cpu().numpy().reshape(-1, kv, 64, d)[page].transpose(1, 0, 2).reshape(n, kv, d // 32, 32)
    s = cache.ks.cpu().numpy().reshape(-1, kv, 64, d // 32)[page].transpose(1, 0, 2)
    assert np.array_equal(k, blocks[..., 2:].view(np.int8))
    assert np.array_equal(s.view(np.uint16), np.ascontiguousarray(blocks[..., :2]).view(np.uint16)[..., 0])
    q, sc = q8_levels(x.reshape(n, kv, d))
    assert np.array_equal(k.reshape(n, kv, d), q) and np.array_equal(s, sc)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_padding_rows_strides_and_other_slots(P, kind):
    """Rows of a fused projection, padding rows between them, pages of two layers in one allocation: nothing but the
    named slots changes."""
    import torch

    rng = np.random.default_rng(8)
    kv, d, page = 2, 64, 16
    elems = kv * page * d
    cache = Cache(P, kind, [20, 9], page, kv, d, rng, page_stride=2 * elems, scale_stride=2 * elems // 32)
    before = [None if t is None else t.cpu().numpy().copy() for t in (cache.k, cache.v, cache.ks, cache.vs)]
    width = kv * d
    fused = torch.from_numpy(rng.standard_normal((5, 3 * width + 4)).astype(np.float32)).cuda()
    seq, pos = np.array([0, -1, 1, -3, 0], np.int32), np.array([19, 0, 8, 5, 2], np.int32)
    at = [torch.from_numpy(x).cuda() for x in (seq, pos)]
    torch.cuda.synchronize()
    P.kv_append_dev(cache.pages, fused[:, width:], fused[:, 2 * width:], at[0], at[1], 5, cache.table, 2, cache.max_pages, row_stride=3 * width + 4)
    P.synchronize()
    host = fused.cpu().numpy()
    after = [None if t is None else t.cpu().numpy() for t in (cache.k, cache.v, cache.ks, cache.vs)]
    named = set()
    for r in (0, 2, 4):
        pg, slot = int(cache.table_host[seq[r], pos[r] // page]), int(pos[r]) % page
        for h in range(kv):
            for side in (0, 1):
                x = host[r, (1 + side) * width + h * d:(1 + side) * width + (h + 1) * d]
                o = pg * cache.stride + (h * page + slot) * d
                if kind == "f16":
                    assert np.array_equal(after[side][o:o + d], x.astype(np.float16))
                else:
                    q, s = q8_levels(x[None])
                    assert np.array_equal(after[side][o:o + d], q[0])
                    so = pg * cache.sstride + (h * page + slot) * (d // 32)
                    assert np.array_equal(after[2 + side][so:so + d // 32], s[0])
                    named.update(("s", side, so + i) for i in range(d // 32))
                named.update((side, o + i) for i in range(d))
    for side in (0, 1):
        same = before[side].view(np.uint8) == after[side].view(np.uint8)
        changed = set(np.nonzero(~same)[0] // before[side].itemsize)
        assert changed <= {i for s, *i in named if s == side for i in i}
        if kind == "q8_0":
            same = before[2 + side].view(np.uint16) == after[2 + side].view(np.uint16)
            assert set(np.nonzero(~same)[0]) <= {n[2] for n in named if n[0] == "s" and n[1] == side}


def test_read_leaves_padding_rows_and_takes_one_side(P):
    rng = np.random.default_rng(9)
    cache = Cache(P, "q8_0", [40], 16, 1, 64, rng)
    rows = cache.fill(rng)
    k, v = read(P, cache, [0, -1, 0], [39, 0, 0], sides=(False, True))
    assert k is None
    assert np.all(v[1] == 7.0)
    assert np.array_equal(v[[0, 2]], held("q8_0", rows[0][1])[[39, 0]].astype(np.float32))


def test_rows_outside_the_cache_touch_nothing_and_are_reported(P):
    import torch

    rng = np.random.default_rng(10)
    cache = Cache(P, "f16", [30], 16, 1, 32, rng)
    before = cache.k.cpu().numpy().view(np.uint16).copy()
    x = np.ones((1, 32), np.float32)
    for seq, pos in ((0, 32), (0, -1), (1, 0), (5, 3), (0, 2**31 - 1)):
        with pytest.raises(P.DeviceError) as e:
            cache.append(x, x, [seq], [pos])
        assert e.value.code == -4
        with pytest.raises(P.DeviceError):
            read(P, cache, [seq], [pos])
    for entry in (-7, cache.n_pages, 2**31 - 1):
        cache.table[0, 1] = entry
        torch.cuda.synchronize()
        with pytest.raises(P.DeviceError):
            cache.append(x, x, [0], [17])
    assert np.array_equal(cache.k.cpu().numpy().view(np.uint16), before)
    P.synchronize()  # reported once


def test_values_beyond_f16_and_empty_calls(P):
    rng = np.random.default_rng(11)
    cache = Cache(P, "f16", [2], 16, 1, 16, rng)
    x = np.array([[1e6, -1e6, 65504, 1e-8] + [0.5] * 12, [np.nan, np.inf, -np.inf, 6e-8] + [1] * 12], np.float32)
    cache.append(x, -x, [0, 0], [0, 1])
    k, v = read(P, cache, [0, 0], [0, 1])
    with np.errstate(over="ignore"):
        assert np.array_equal(k.reshape(2, 16), x.astype(np.float16).astype(np.float32), equal_nan=True)
        assert np.array_equal(v.reshape(2, 16), (-x).astype(np.float16).astype(np.float32), equal_nan=True)
    cache.append(np.zeros((0, 16), np.float32), np.zeros((0, 16), np.float32), [], [])


def test_long_cache_past_32_bit_offsets(P):
    """Pages more than 2^32 bytes into the pool."""
    import torch

    kv, d, page = 8, 128, 64
    n_pages = (5 << 30) // (kv * page * d * 2)
    k = torch.empty(n_pages * kv * page * d, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    pages = P.KvPages(P.KV_F16, k, v, None, None, n_pages, page, kv, d)
    rng = np.random.default_rng(12)
    ids = [n_pages - 1, 0, n_pages - 2]
    table = torch.tensor([ids], dtype=torch.int32).cuda()
    n = 3 * page
    x = torch.from_numpy(rng.standard_normal((n, kv * d)).astype(np.float32)).cuda()
    seq, pos = torch.zeros(n, dtype=torch.int32).cuda(), torch.arange(n, dtype=torch.int32).cuda()
    out = torch.zeros(2, n, kv * d, device="cuda")
    q = torch.from_numpy(rng.standard_normal((1, kv, d)).astype(np.float32)).cuda()
    att = torch.zeros(1, kv, d, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    P.kv_append_dev(pages, x, -x, seq, pos, n, table, 1, 3)
    P.kv_read_dev(pages, out[0], out[1], False, seq, pos, n, table, 1, 3)
    P.attn_paged_dev(pages, q, att, table, lens, 1, 3, kv, d ** -0.5)
    P.synchronize()
    assert torch.equal(out[0], x.half().float()) and torch.equal(out[1], -out[0])
    kk = out[0].double().reshape(n, kv, d)
    p = torch.softmax(torch.einsum("hd,jhd->hj", q[0].double(), kk) * d ** -0.5, dim=1)
    want = -torch.einsum("hj,jhd->hd", p, kk)
    assert float((att[0] - want).norm() / want.norm()) <= 48 * 2.0 ** -24

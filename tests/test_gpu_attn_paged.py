"""Attention of one new token per sequence over paged keys and values, against the 64-bit form."""
import numpy as np
import pytest

from kv_reference import Cache, check_attention, held

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    from fucina_b200 import provider

    provider.init(0)
    return provider


def run(P, kind, lens, page, heads, kv, d, window=0, seed=1, gain=1.0, max_len=0, **kw):
    rng = np.random.default_rng(seed)
    cache = Cache(P, kind, lens, page, kv, d, rng, **kw)
    rows = cache.fill(rng, gain)
    q = rng.standard_normal((len(lens), heads, d)).astype(np.float32)
    scale = float(np.float32(d ** -0.5))
    got, stats = cache.attend(q, heads, scale, window, stats=True, max_len=max_len)
    check_attention(cache, rows, q, got, scale, window, stats)
    return cache, rows, q, got


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("lens,page,heads,kv,d,window", [
    ([1], 16, 1, 1, 64, 0),
    ([0], 16, 4, 2, 64, 0),
    ([15, 16, 17], 16, 8, 2, 128, 0),
    ([31, 0, 33, 1, 0], 32, 5, 1, 96, 0),           # odd group, empty rows
    ([129, 7, 64], 64, 14, 2, 64, 0),               # seven heads to a kv head
    ([500, 499], 48, 16, 1, 128, 0),                # sixteen heads share one kv head, pages of 48
    ([70], 16, 36, 1, 64, 0),                       # thirty-six heads to a kv head
    ([200, 90], 16, 9, 1, 32, 0),
    ([300, 40], 16, 80, 1, 64, 0),                  # eighty heads to a kv head
    ([260], 256, 6, 3, 160, 0),
    ([5000, 20], 4096, 4, 1, 64, 0),                # pages longer than most sequences
    ([180, 5], 16, 17, 1, 160, 0),                  # seventeen heads of 160
    ([300, 290], 16, 31, 1, 192, 0),
    ([120, 300], 32, 4, 2, 256, 0),
    ([1000, 3, 40], 16, 8, 4, 128, 37),             # window starts inside a block of keys
    ([64, 65, 63], 16, 4, 4, 128, 64),
    ([90, 2], 16, 2, 2, 128, 1),                    # a window of the token itself
])
def test_against_64_bits(P, kind, lens, page, heads, kv, d, window):
    run(P, kind, lens, page, heads, kv, d, window)


@pytest.mark.parametrize("d", [16, 48, 80, 112, 176, 208])
def test_f16_head_sizes_that_are_odd_multiples_of_16(P, d):
    run(P, "f16", [77, 19], 16, 6, 2, d)


@pytest.mark.parametrize("d", [32, 96, 160, 192, 224])
def test_q8_head_sizes(P, d):
    run(P, "q8_0", [77, 19], 16, 6, 2, d)


@pytest.mark.parametrize("kind,lens,page,heads,kv,d,window", [
    ("f16", [20000], 64, 8, 2, 128, 0),             # one long sequence over the whole GPU
    ("q8_0", [20000], 16, 8, 2, 128, 0),
    ("q8_0", [9000, 100, 0, 5000, 1, 7000], 64, 8, 4, 128, 0),
    ("f16", [6000, 50, 9000], 32, 32, 2, 256, 4096),
    ("f16", [12000], 16, 4, 1, 64, 0),
    ("q8_0", [5000, 4999], 48, 40, 1, 64, 0),       # forty heads to a kv head
])
def test_long_and_uneven(P, kind, lens, page, heads, kv, d, window):
    run(P, kind, lens, page, heads, kv, d, window)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_many_sequences(P, kind):
    rng = np.random.default_rng(3)
    run(P, kind, [int(x) for x in rng.integers(0, 90, 700)], 16, 4, 2, 64)
    run(P, kind, [int(x) for x in rng.integers(0, 2500, 70)], 16, 4, 2, 64)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("gain", [1e-6, 1e-3, 60.0, 3000.0])
def test_values_of_other_magnitudes(P, kind, gain):
    """Keys and values far from one: tiny ones stay above f16's and the scales' smallest steps only in part, but the
    cache holds what it holds and the attention keeps f32 accuracy on that; large ones make the softmax a choice."""
    rng = np.random.default_rng(4)
    cache = Cache(P, kind, [400, 37], 16, 2, 128, rng)
    rows = cache.fill(rng, gain)
    q = (rng.standard_normal((2, 8, 128)) / max(gain, 1e-4)).astype(np.float32)
    got, _ = cache.attend(q, 8, 0.09)
    check_attention(cache, rows, q, got, float(np.float32(0.09)))


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_value_scales_that_grow_along_the_sequence(P, kind):
    rng = np.random.default_rng(14)
    n, kv, d = 700, 1, 64
    cache = Cache(P, kind, [n], 16, kv, d, rng)
    k = rng.standard_normal((n, d)).astype(np.float32)
    v = (rng.standard_normal((n, d)) * np.exp(np.linspace(-9, 9, n))[:, None]).astype(np.float32)
    cache.append(k, v, np.zeros(n), np.arange(n))
    q = rng.standard_normal((1, 3, d)).astype(np.float32)
    got, _ = cache.attend(q, 3, 0.125)
    check_attention(cache, [(k.reshape(n, kv, d), v.reshape(n, kv, d))], q, got, 0.125)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_queries_of_other_magnitudes(P, kind):
    rng = np.random.default_rng(15)
    cache = Cache(P, kind, [150], 16, 1, 64, rng)
    rows = cache.fill(rng)
    q = rng.standard_normal((1, 4, 64)).astype(np.float32) * np.array([1e-30, 1e-6, 1.0, 1e6], np.float32)[None, :, None]
    q[0, 2] = 0
    for scale in (0.125, 1e-7):
        got, _ = cache.attend(q, 4, scale)
        check_attention(cache, rows, q, got, float(np.float32(scale)))


def test_infinite_scores_and_values(P):
    """A key of -infinity closes its position; an infinite value comes out where it has weight."""
    rng = np.random.default_rng(16)
    d, n = 64, 40
    cache = Cache(P, "f16", [n], 16, 1, d, rng)
    k, v = rng.standard_normal((2, n, d)).astype(np.float32)
    k[5, 0] = -np.inf
    cache.append(k, v, np.zeros(n), np.arange(n))
    q = np.abs(rng.standard_normal((1, 2, d))).astype(np.float32)
    got, _ = cache.attend(q, 2, 0.125)
    keep = np.arange(n) != 5
    check_attention(cache, [(k[keep].reshape(-1, 1, d), v[keep].reshape(-1, 1, d))], q, got, 0.125)
    v[7, 3] = np.inf
    cache.append(k, v, np.zeros(n), np.arange(n))
    got, _ = cache.attend(q, 2, 0.125)
    assert np.all(np.isposinf(got[0, :, 3])) and np.all(np.isfinite(np.delete(got[0], 3, axis=1)))


def test_strided_queries_and_interleaved_pages(P):
    import torch

    rng = np.random.default_rng(17)
    kv, d, page, heads = 2, 128, 16, 8
    elems = kv * page * d
    for kind in ("f16", "q8_0"):
        cache = Cache(P, kind, [100, 33], page, kv, d, rng, page_stride=3 * elems, scale_stride=elems // 32 + 8)
        rows = cache.fill(rng)
        fused = torch.from_numpy(rng.standard_normal((2, heads * d + 2 * kv * d)).astype(np.float32)).cuda()
        out = torch.empty(2, heads, d, device="cuda")
        torch.cuda.synchronize()
        P.attn_paged_dev(cache.pages, fused, out, cache.table, cache.lens_dev, 2, cache.max_pages, heads, 0.0625, q_stride=fused.shape[1])
        P.synchronize()
        q = fused[:, : heads * d].reshape(2, heads, d).cpu().numpy()
        check_attention(cache, rows, q, out.cpu().numpy(), 0.0625)


def test_shared_prefix_pages(P):
    """Two sequences whose tables begin with the same pages."""
    import torch

    rng = np.random.default_rng(18)
    cache = Cache(P, "q8_0", [80, 96], 16, 2, 64, rng)
    rows = cache.fill(rng)
    cache.table[1, :5] = cache.table[0, :5]
    torch.cuda.synchronize()
    mixed = [rows[0], tuple(np.concatenate([rows[0][i], rows[1][i][80:]]) for i in (0, 1))]
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    got, _ = cache.attend(q, 4, 0.125)
    check_attention(cache, mixed, q, got, 0.125)


@pytest.mark.parametrize("kind,heads,kv,d", [("q8_0", 2, 1, 128), ("f16", 16, 1, 128), ("q8_0", 20, 1, 64), ("f16", 32, 1, 64), ("f16", 12, 1, 256)])
@pytest.mark.parametrize("rings", [2, 4, 6, 8, 11, 12])
@pytest.mark.parametrize("over", [1, 2, 3, 5])
def test_last_chunks_of_every_size(P, kind, heads, kv, d, rings, over):
    """Very short sequences under a table for long ones: work is handed out in chunks of three units (a unit per sequence),
    and the last chunk has one, two or three, for whatever number of rings an SM holds."""
    import torch

    rng = np.random.default_rng(24)
    n = P.sm_count() * rings * 3 + over
    lens = [int(x) for x in rng.integers(0, 4, n)]
    cache = Cache(P, kind, lens, 16, kv, d, rng)
    rows = cache.fill(rng)
    wide = torch.full((n, 128), -1, dtype=torch.int32).cuda()
    wide[:, :1] = cache.table
    cache.table, cache.max_pages = wide, 128
    q = rng.standard_normal((n, heads, d)).astype(np.float32)
    got, _ = cache.attend(q, heads, 0.125)
    for s in range(n):
        if lens[s] == 0:
            assert not got[s].any()
    some = [0, 1, 2, n - 1, n - 2, n - 3] + [int(x) for x in rng.integers(0, n, 60)]
    sub = Cache.__new__(Cache)
    sub.kind, sub.d = kind, d
    check_attention(sub, [rows[s] for s in some], q[some], got[some], 0.125)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 31, 32, 33, 100])
def test_pages_behind_the_window_may_be_gone(P, kind, window):
    """A sliding window's user hands pages that lie wholly before the window to other sequences."""
    import torch

    rng = np.random.default_rng(23)
    lens = [130, 129, 145, 4000]
    cache = Cache(P, kind, lens, 16, 1, 64, rng)
    rows = cache.fill(rng)
    for s, n in enumerate(lens):
        cache.table[s, : (n - window) // 16] = -1
    torch.cuda.synchronize()
    q = rng.standard_normal((len(lens), 3, 64)).astype(np.float32)
    got, _ = cache.attend(q, 3, 0.125, window)
    check_attention(cache, rows, q, got, 0.125, window)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("lens", [[500], [9000], [3000, 200, 6000]])
def test_bad_pages_and_lengths_are_reported_and_left_out(P, kind, lens):
    import torch

    rng = np.random.default_rng(19)
    cache = Cache(P, kind, lens, 16, 1, 64, rng)
    rows = cache.fill(rng)
    q = rng.standard_normal((len(lens), 4, 64)).astype(np.float32)
    good = cache.table.clone()
    for entry in (-1, cache.n_pages, 2**31 - 1):
        cache.table.copy_(good)
        cache.table[0, 3] = entry
        out = torch.full((len(lens), 4, 64), float("nan")).cuda()
        qd = torch.from_numpy(q).cuda()
        torch.cuda.synchronize()
        P.attn_paged_dev(cache.pages, qd, out, cache.table, cache.lens_dev, len(lens), cache.max_pages, 4, 0.125)
        with pytest.raises(P.DeviceError) as e:
            P.synchronize()
        assert e.value.code == -4
        keep = np.ones(lens[0], bool)
        keep[48:64] = False
        check_attention(cache, [tuple(x[keep] for x in rows[0])] + rows[1:], q, out.cpu().numpy(), 0.125)
    cache.table.copy_(good)
    cut = lens[0] - 5
    for bad, seen in ((lens[0] + 100000, cut), (-3, 0)):
        cache.lens_dev[0] = bad
        out = torch.full((len(lens), 4, 64), float("nan")).cuda()
        qd = torch.from_numpy(q).cuda()
        torch.cuda.synchronize()
        P.attn_paged_dev(cache.pages, qd[:1], out, cache.table, cache.lens_dev, 1, cache.max_pages, 4, 0.125, max_len=cut)
        with pytest.raises(P.DeviceError):
            P.synchronize()
        check_attention(cache, [tuple(x[:seen] for x in rows[0])], q, out.cpu().numpy(), 0.125)
    P.synchronize()


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_same_bits_alone_and_among_others(P, kind):
    """A call's result does not depend on workspace contents, the stream, or how often it ran."""
    import torch

    rng = np.random.default_rng(20)
    cache = Cache(P, kind, [7000, 30, 4000], 16, 2, 128, rng)
    cache.fill(rng)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    first, _ = cache.attend(q, 8, 0.09)
    for kw in ({}, {"workspace": False}, {"stream": torch.cuda.Stream().cuda_stream}):
        again, _ = cache.attend(q, 8, 0.09, **kw)
        assert np.array_equal(first.view(np.uint32), again.view(np.uint32))


def test_captured_steps_follow_the_lengths(P):
    """Two graphs of append + attention replayed in turn, each with its own workspace, while the lengths grow."""
    import torch

    rng = np.random.default_rng(21)
    kv, d, heads, page, cap = 2, 128, 8, 16, 3000
    worlds = []
    for kind in ("q8_0", "f16"):
        cache = Cache(P, kind, [cap, cap], page, kv, d, rng)
        full = rng.standard_normal((2, 2, cap, kv, d)).astype(np.float32)  # [k or v][seq]
        start = [2990, 5]
        for s in (0, 1):
            cache.append(full[0, s, :start[s]].reshape(-1, kv * d), full[1, s, :start[s]].reshape(-1, kv * d), np.full(start[s], s), np.arange(start[s]))
        w = {"cache": cache, "full": full, "lens": list(start), "new": torch.zeros(2, 2, kv * d).cuda(), "q": torch.zeros(2, heads, d).cuda(),
             "out": torch.zeros(2, heads, d).cuda(), "seq": torch.arange(2, dtype=torch.int32).cuda(), "pos": torch.zeros(2, dtype=torch.int32).cuda()}
        size = P.attn_paged_workspace_bytes(cache.pages, 2, heads, cap)
        w["ws"] = torch.empty(max(size, 16), dtype=torch.uint8).cuda()
        torch.cuda.synchronize()
        with P.capture() as cap_:
            P.kv_append_dev(cache.pages, w["new"][0], w["new"][1], w["seq"], w["pos"], 2, cache.table, 2, cache.max_pages)
            P.attn_paged_dev(cache.pages, w["q"], w["out"], cache.table, cache.lens_dev, 2, cache.max_pages, heads, 0.09, max_len=cap,
                             workspace=w["ws"], workspace_bytes=size)
        w["graph"] = cap_.graph
        worlds.append(w)
    for step in range(3):
        for w in worlds:
            lens = w["lens"]
            w["new"].copy_(torch.from_numpy(np.stack([[w["full"][i, s, lens[s]].reshape(-1) for s in (0, 1)] for i in (0, 1)])))
            w["pos"].copy_(torch.tensor(lens, dtype=torch.int32))
            w["lens"] = [n + 1 for n in lens]
            w["cache"].lens_dev.copy_(torch.tensor(w["lens"], dtype=torch.int32))
            w["qh"] = rng.standard_normal((2, heads, d)).astype(np.float32)
            w["q"].copy_(torch.from_numpy(w["qh"]))
        torch.cuda.synchronize()
        for w in worlds:
            w["graph"].launch()
        P.synchronize()
        for w in worlds:
            rows = [(w["full"][0, s, :w["lens"][s]], w["full"][1, s, :w["lens"][s]]) for s in (0, 1)]
            check_attention(w["cache"], rows, w["qh"], w["out"].cpu().numpy(), float(np.float32(0.09)))
    for w in worlds:
        w["graph"].destroy()


def test_a_captured_call_needs_a_workspace_of_its_own(P):
    import torch

    rng = np.random.default_rng(25)
    cache = Cache(P, "f16", [9000], 64, 1, 128, rng)
    q, out = torch.zeros(1, 4, 128).cuda(), torch.zeros(1, 4, 128).cuda()
    size = P.attn_paged_workspace_bytes(cache.pages, 1, 4, 9000)
    assert size > 0
    ws = torch.empty(size, dtype=torch.uint8).cuda()
    torch.cuda.synchronize()
    args = (cache.pages, q, out, cache.table, cache.lens_dev, 1, cache.max_pages, 4, 0.1)
    with P.capture() as cap:
        with pytest.raises(P.Declined):
            P.attn_paged_dev(*args)
        with pytest.raises(P.Declined):
            P.attn_paged_dev(*args, workspace=ws, workspace_bytes=size - 16)
        P.attn_paged_dev(*args, workspace=ws, workspace_bytes=size)
    cap.graph.launch()
    P.synchronize()
    cap.graph.destroy()


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_two_streams_at_once(P, kind):
    """Calls on two streams without an order between them, each with its own workspace or the library's."""
    import torch

    rng = np.random.default_rng(26)
    cache = Cache(P, kind, [6000, 40, 3000], 16, 2, 128, rng)
    cache.fill(rng)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    want, _ = cache.attend(q, 8, 0.09)
    qd = torch.from_numpy(q).cuda()
    size = P.attn_paged_workspace_bytes(cache.pages, 3, 8, cache.max_pages * 16)
    streams = [torch.cuda.Stream().cuda_stream for _ in range(2)]
    outs = [torch.zeros(3, 8, 128).cuda() for _ in range(8)]
    spaces = [torch.empty(max(size, 16), dtype=torch.uint8).cuda() for _ in range(2)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        kw = {"workspace": spaces[i % 2], "workspace_bytes": size} if i < 4 else {}
        P.attn_paged_dev(cache.pages, qd, out, cache.table, cache.lens_dev, 3, cache.max_pages, 8, 0.09, stream=streams[i % 2], **kw)
    torch.cuda.synchronize()
    for out in outs:
        assert np.array_equal(out.cpu().numpy().view(np.uint32), want.view(np.uint32))


def test_long_sums_keep_f32_accuracy(P):
    """A batch whose chunks are hundreds of units long, all keys of nearly equal weight: what the sums lose per unit must not
    add up. Compared in 64 bits on the GPU, one head of each sequence."""
    import torch

    n, length, kv, d, page = 40, 16384, 2, 128, 64
    gen = torch.Generator(device="cuda").manual_seed(27)
    pages_per = length // page
    k = torch.randn(n * pages_per, kv, page, d, generator=gen, device="cuda").half()
    v = (torch.randn(n * pages_per, kv, page, d, generator=gen, device="cuda") + 0.25).half()
    table = torch.arange(n * pages_per, dtype=torch.int32, device="cuda").reshape(n, pages_per).contiguous()
    lens = torch.full((n,), length, dtype=torch.int32, device="cuda")
    q = torch.randn(n, 8, d, generator=gen, device="cuda") * 0.3
    out = torch.empty(n, 8, d, device="cuda")
    pages = P.KvPages(P.KV_F16, k, v, None, None, n * pages_per, page, kv, d)
    torch.cuda.synchronize()
    P.attn_paged_dev(pages, q, out, table, lens, n, pages_per, 8, d ** -0.5)
    P.synchronize()
    err = ref = 0.0
    for s in range(0, n, 7):
        kk = k[table[s].long()].transpose(0, 1).reshape(kv, length, d).double()
        vv = v[table[s].long()].transpose(0, 1).reshape(kv, length, d).double()
        x = torch.einsum("gd,jd->gj", q[s, :4].double(), kk[0]) * d ** -0.5
        want = torch.softmax(x, dim=1) @ vv[0]
        err, ref = err + float((out[s, :4].double() - want).square().sum()), ref + float(want.square().sum())
    assert (err / ref) ** 0.5 <= 48 * 2.0 ** -24


def test_prompt_chunk_reads_its_cache_for_the_dense_attention(P):
    """A prompt in two chunks: append, read back as f16, attend with the dense entry; then one decode step over the pages
    gives the row that the dense entry gives for the same token."""
    import torch

    rng = np.random.default_rng(22)
    heads, kv, d, n, page = 8, 2, 128, 90, 32
    for kind in ("f16", "q8_0"):
        cache = Cache(P, kind, [n], page, kv, d, rng)
        k, v = rng.standard_normal((2, n, kv, d)).astype(np.float32)
        q = rng.standard_normal((n, heads, d)).astype(np.float32)
        qd = torch.from_numpy(q).cuda()
        kvmap = torch.tensor([h // (heads // kv) for h in range(heads)], dtype=torch.int32).cuda()
        outs = []
        for a, b in ((0, 50), (50, n)):
            cache.append(k[a:b].reshape(b - a, -1), v[a:b].reshape(b - a, -1), np.zeros(b - a), np.arange(a, b))
            kd, vd = torch.empty(2, b, kv, d, dtype=torch.float16, device="cuda")
            seq, pos = torch.zeros(b, dtype=torch.int32).cuda(), torch.arange(b, dtype=torch.int32).cuda()
            out = torch.empty(b - a, heads, d, device="cuda")
            torch.cuda.synchronize()
            P.kv_read_dev(cache.pages, kd, vd, True, seq, pos, b, cache.table, 1, cache.max_pages)
            P.attn_fwd_dev(qd[a:b], kd, vd, True, out, kvmap, b - a, b, heads, kv, d, a, d ** -0.5)
            P.synchronize()
            outs.append(out.cpu().numpy())
        dense = np.concatenate(outs)
        # the dense entry's own bound (its weights are f16, and a Q8_0 value rounds to f16 on the way)
        step, _ = cache.attend(q[n - 1:], heads, d ** -0.5)
        assert np.all(np.abs(step[0] - dense[n - 1]) <= np.maximum(2e-3 * np.abs(step[0]), 2e-3))
        check_attention(cache, [(k, v)], q[n - 1:], step, d ** -0.5)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_thousands_of_sequences_of_every_length(P, kind):
    """More sequences than a ring adds up by itself, a few long ones among them."""
    rng = np.random.default_rng(28)
    lens = [int(x) for x in rng.integers(0, 40, 1500)]
    lens[7], lens[800], lens[1499] = 3000, 1700, 900
    cache = Cache(P, kind, lens, 16, 1, 64, rng)
    rows = cache.fill(rng)
    q = rng.standard_normal((len(lens), 3, 64)).astype(np.float32)
    got, stats = cache.attend(q, 3, 0.125, stats=True)
    check_attention(cache, rows, q, got, 0.125, stats=stats)

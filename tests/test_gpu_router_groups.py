"""Router with score kinds, balance bias and expert groups, against the 64-bit form, and in front of the expert layer."""
import numpy as np
import pytest

from kv_reference import Cache, attention, held, router

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    from fucina_b200 import provider

    provider.init(0)
    return provider


def route(P, logits, k, sigmoid=False, bias=None, groups=1, kept=1, top2=False, normalize=True, scale=1.0, stream=0):
    import torch

    t, e = logits.shape
    x = torch.from_numpy(np.ascontiguousarray(logits)).cuda()
    b = None if bias is None else torch.from_numpy(bias).cuda()
    sel, w = torch.full((t + 1, k), -9, dtype=torch.int32).cuda(), torch.full((t + 1, k), -9.0).cuda()
    torch.cuda.synchronize()
    P.router_groups_dev(x, t, e, k, sel, w, score=P.SCORE_SIGMOID if sigmoid else P.SCORE_SOFTMAX, bias_dev=b, n_group=groups, topk_group=kept,
                        group_score=P.GROUP_TOP2 if top2 else P.GROUP_MAX, normalize=normalize, scale=scale, stream=stream)
    torch.cuda.synchronize()
    P.synchronize()
    assert bool((sel[t] == -9).all()) and bool((w[t] == -9).all())
    return sel[:t].cpu().numpy(), w[:t].cpu().numpy()


def check(P, logits, k, **kw):
    sel, w = route(P, logits, k, **kw)
    want_sel, want_w = router(logits, k, **kw)
    assert np.array_equal(sel, want_sel)
    # 64-bit arithmetic, one rounding to f32 at the end
    assert np.all(np.abs(w - want_w) <= (2.0 ** -24 + 1e-12) * np.abs(want_w) + 1e-44)


@pytest.mark.parametrize("t,e,k,groups,kept", [
    (1, 1, 1, 1, 1), (1, 8, 2, 1, 1), (3, 60, 6, 1, 1), (7, 128, 8, 1, 1), (129, 256, 8, 8, 4), (5, 160, 6, 8, 3), (33, 64, 6, 4, 4),
    (2, 100, 32, 1, 1), (4, 96, 32, 3, 2), (9, 512, 10, 64, 8), (3, 64, 5, 64, 5), (2, 1023, 7, 1, 1), (2, 4096, 8, 16, 3), (65, 33, 3, 11, 2),
    (2, 1536, 4, 2, 1),
])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_against_64_bits(P, t, e, k, groups, kept, sigmoid, biased):
    rng = np.random.default_rng(t * e + k)
    logits = (rng.standard_normal((t, e)) * 2).astype(np.float32)
    bias = (rng.standard_normal(e) * 0.1).astype(np.float32) if biased else None
    for top2 in (False, True):
        for normalize in (False, True):
            check(P, logits, k, sigmoid=sigmoid, bias=bias, groups=groups, kept=kept, top2=top2, normalize=normalize, scale=2.5 if normalize else 1.0)


def test_large_batch(P):
    rng = np.random.default_rng(2)
    check(P, (rng.standard_normal((20000, 256)) * 1.5).astype(np.float32), 8, sigmoid=True, bias=(rng.standard_normal(256) * 0.05).astype(np.float32),
          groups=8, kept=4, top2=True, scale=2.5)
    check(P, (rng.standard_normal((20000, 128)) * 1.5).astype(np.float32), 8)


def test_ties_go_to_the_lowest_index(P):
    logits = np.zeros((3, 64), np.float32)
    logits[1, 40:] = 1
    logits[2, ::2] = -1
    for kw in ({}, {"sigmoid": True}, {"groups": 8, "kept": 3}, {"groups": 8, "kept": 3, "top2": True, "sigmoid": True}):
        check(P, logits, 6, **kw)


def test_neighbours_closer_than_f32_resolves(P):
    """Logits one f32 step apart under a sigmoid that maps them to the same f32 score, with and without a bias."""
    rng = np.random.default_rng(3)
    base = np.float32(6.0)
    steps = rng.permutation(96)
    logits = (base.view(np.int32) + steps).astype(np.int32).view(np.float32)[None]
    assert len(set((1 / (1 + np.exp(-logits[0]))).astype(np.float32))) < 96
    check(P, logits, 12, sigmoid=True)
    check(P, logits, 12, sigmoid=True, bias=np.full(96, 0.25, np.float32))
    check(P, logits, 12, sigmoid=True, bias=np.full(96, 0.25, np.float32), groups=4, kept=2, top2=True)
    check(P, np.tile(logits, (50, 1)), 12)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_closed_experts(P, sigmoid):
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((6, 32)).astype(np.float32)
    logits[0, 5:] = -np.inf
    logits[1, :] = -np.inf
    logits[2, ::2] = np.nan
    logits[3, 1:] = -np.inf
    logits[4, 7] = np.inf
    logits[5, 16:] = -np.inf
    for kw in ({}, {"groups": 4, "kept": 2}, {"groups": 4, "kept": 2, "top2": True}, {"bias": rng.standard_normal(32).astype(np.float32)}):
        check(P, logits, 8, sigmoid=sigmoid, **kw)


def test_extreme_logits(P):
    rng = np.random.default_rng(5)
    logits = (rng.standard_normal((40, 48)) * 100).astype(np.float32)
    logits[0, 3] = 3e38
    logits[1] = -3e38
    for sigmoid in (False, True):
        check(P, logits, 5, sigmoid=sigmoid)
        check(P, logits, 5, sigmoid=sigmoid, bias=(rng.standard_normal(48) * 10).astype(np.float32), groups=6, kept=3)


def test_same_bits_on_another_stream_and_in_a_graph(P):
    import torch

    rng = np.random.default_rng(6)
    logits = rng.standard_normal((50, 256)).astype(np.float32)
    kw = {"sigmoid": True, "groups": 8, "kept": 4, "top2": True}
    a = route(P, logits, 8, **kw)
    b = route(P, logits, 8, stream=torch.cuda.Stream().cuda_stream, **kw)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    x = torch.from_numpy(logits).cuda()
    sel, w = torch.zeros(50, 8, dtype=torch.int32).cuda(), torch.zeros(50, 8).cuda()
    torch.cuda.synchronize()
    with P.capture() as cap:
        P.router_groups_dev(x, 50, 256, 8, sel, w, score=P.SCORE_SIGMOID, n_group=8, topk_group=4, group_score=P.GROUP_TOP2)
    cap.graph.launch()
    P.synchronize()
    assert np.array_equal(sel.cpu().numpy(), a[0]) and np.array_equal(w.cpu().numpy(), a[1])
    cap.graph.destroy()


def test_decode_step_append_attend_route_experts(P):
    """The middle of a decode step as it is used: the new token's keys and values into the cache, attention over it, a
    router product, expert choice, the expert layer, all on the library stream."""
    import torch

    import oracle
    from parity import assert_close, make_weights

    rng = np.random.default_rng(7)
    n_seqs, heads, kv, d, page, n_expert, top_k, hidden, out_pe = 3, 4, 2, 64, 16, 8, 2, 256, 256
    lens = [33, 1, 120]
    cache = Cache(P, "q8_0", lens, page, kv, d, rng)
    rows = [tuple(rng.standard_normal((n, kv, d)).astype(np.float32) for _ in (0, 1)) for n in lens]
    for s, (k, v) in enumerate(rows):
        if lens[s] > 1:
            cache.append(k[:-1].reshape(lens[s] - 1, -1), v[:-1].reshape(lens[s] - 1, -1), np.full(lens[s] - 1, s), np.arange(lens[s] - 1))
    fmt = oracle.FORMATS["q5_k"]
    blocks = [make_weights("q5_k", n_expert * n, k, 30 + i) for i, (n, k) in enumerate(((out_pe, hidden), (out_pe, hidden), (hidden, out_pe)))]
    experts = [P.Weights.upload(fmt, b, n, k, n_expert) for b, (n, k) in zip(blocks, ((out_pe, hidden), (out_pe, hidden), (hidden, out_pe)))]
    rw_blocks = make_weights("q8_0", n_expert, hidden, 40)
    rw = P.Weights.upload(oracle.FORMATS["q8_0"], rw_blocks, n_expert, hidden)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    fused = rng.standard_normal((n_seqs, (heads + 2 * kv) * d)).astype(np.float32)
    for s, (k, v) in enumerate(rows):
        fused[s, heads * d:] = np.concatenate([k[-1].reshape(-1), v[-1].reshape(-1)])
    bias = (rng.standard_normal(n_expert) * 0.1).astype(np.float32)
    fd, bd = dev(fused), dev(bias)
    seq, pos = dev(np.arange(n_seqs, dtype=np.int32)), dev(np.array(lens, np.int32) - 1)
    att, logits, out = torch.empty(n_seqs, heads * d).cuda(), torch.empty(n_seqs, n_expert).cuda(), torch.empty(n_seqs, hidden).cuda()
    sel, w = torch.empty(n_seqs, top_k, dtype=torch.int32).cuda(), torch.empty(n_seqs, top_k).cuda()
    torch.cuda.synchronize()
    P.kv_append_dev(cache.pages, fd[:, heads * d:], fd[:, (heads + kv) * d:], seq, pos, n_seqs, cache.table, n_seqs, cache.max_pages,
                    row_stride=fused.shape[1])
    P.attn_paged_dev(cache.pages, fd, att, cache.table, cache.lens_dev, n_seqs, cache.max_pages, heads, 0.125, q_stride=fused.shape[1])
    P.gemm_quant_nt_dev(rw, att, logits, n_seqs)
    P.router_groups_dev(logits, n_seqs, n_expert, top_k, sel, w, score=P.SCORE_SIGMOID, bias_dev=bd, n_group=4, topk_group=2, group_score=P.GROUP_TOP2)
    P.moe_layer_dev(*experts, att, n_seqs, top_k, sel, w, out)
    P.synchronize()
    q = fused[:, : heads * d].reshape(n_seqs, heads, d)
    want = np.stack([attention(q[s], held("q8_0", k), held("q8_0", v), 0.125)[0] for s, (k, v) in enumerate(rows)]).reshape(n_seqs, -1)
    assert np.linalg.norm(att.cpu().numpy() - want) <= 48 * 2.0 ** -24 * np.linalg.norm(want)
    got_logits = logits.cpu().numpy()
    assert_close(got_logits, oracle.matmul(oracle.FORMATS["q8_0"], rw_blocks, att.cpu().numpy()), 1e-3, "router product")
    want_sel, want_w = router(got_logits, top_k, sigmoid=True, bias=bias, groups=4, kept=2, top2=True)
    assert np.array_equal(sel.cpu().numpy(), want_sel)
    assert np.all(np.abs(w.cpu().numpy() - want_w) <= 2.0 ** -23 * want_w)
    ref = oracle.moe_ffn(fmt, *blocks, att.cpu().numpy(), want_sel, w.cpu().numpy(), n_expert, out_pe)
    assert_close(out.cpu().numpy(), ref, 5e-3, "expert layer")
    for h in experts + [rw]:
        h.free()

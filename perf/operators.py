"""Cases of the paged key-value cache (write, read back), of attention over it, and of the expert router.

`run` computes a case in its plain form, elementary torch operations, or (with `own`) through this library's entries.
"""
import math

import torch

if __name__ == "__main__":
    raise SystemExit("a list of cases: nothing to run")

own = False

BLOCK = 32  # values that share one scale in the 8-bit cache


# ---- the cases ------------------------------------------------------------------------------------------------------
# store: rows of new tokens are written into pages, and rows are read back from them
#   seqs sequences of lo..hi tokens; the last `new` tokens of each are written (0: all of them) and all are read back as
#   f32 or f16; with `back` 0 only the new ones are read back. `pad` rows of the batch belong to no sequence.
# attend: one new token of each sequence attends to its pages
# route: tokens choose experts
def _store(name, kind, seqs, lo, hi, new, back, kv, d, page, half, pad=0):
    return {"name": name, "op": "store", "kind": kind, "seqs": seqs, "lo": lo, "hi": hi, "new": new, "back": back, "kv": kv, "d": d, "page": page,
            "half": half, "pad": pad}


def _attend(name, kind, seqs, lo, hi, heads, kv, d, page, window=0):
    return {"name": name, "op": "attend", "kind": kind, "seqs": seqs, "lo": lo, "hi": hi, "heads": heads, "kv": kv, "d": d, "page": page, "window": window}


def _route(name, tokens, experts, k, sigmoid, bias, groups, kept, best2, renorm, scale, masked=0):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "k": k, "sigmoid": sigmoid, "bias": bias, "groups": groups, "kept": kept,
            "best2": best2, "renorm": renorm, "scale": scale, "masked": masked}


def listed():
    return [
        # a decode step of 32 sequences puts one token each into an 8-bit cache
        _store("store_step_q8", "q8_0", 32, 400, 1200, 1, 0, 8, 128, 16, False),
        # a prompt batch goes into an 8-bit cache and comes back as the f16 rows that the dense attention reads
        _store("store_prompt_q8", "q8_0", 5, 1200, 4000, 0, 1, 8, 128, 64, True, pad=7),
        # the next chunk of each prompt on an f16 cache with an odd head count and size, everything read back as f32
        _store("store_chunk_f16", "f16", 3, 700, 2900, 511, 1, 5, 80, 48, False),
        # one short conversation: latency of a single small call
        _attend("attend_one_short_f16", "f16", 1, 517, 517, 32, 8, 128, 16),
        # one very long document, 8-bit
        _attend("attend_one_long_q8", "q8_0", 1, 131072, 131072, 32, 8, 128, 64),
        # one long document in f16
        _attend("attend_one_8k_f16", "f16", 1, 8192, 8192, 32, 8, 128, 64),
        # a serving batch of uneven lengths, both formats
        _attend("attend_batch_f16", "f16", 64, 300, 8000, 32, 8, 128, 16),
        _attend("attend_batch_q8", "q8_0", 64, 300, 8000, 32, 8, 128, 64),
        # wide heads, sixteen to one shared key head, a sliding window
        _attend("attend_wide_window_f16", "f16", 24, 900, 9000, 32, 2, 256, 32, window=4096),
        # a padded batch of short sequences, some empty; seven heads to a key head
        _attend("attend_ragged_q8", "q8_0", 100, 0, 300, 28, 4, 64, 16),
        # one token through the softmax router of a 128-expert layer
        _route("route_token_softmax", 1, 128, 8, False, False, 1, 1, False, True, 1.0),
        # a prompt batch through a sigmoid router with a balance bias and expert groups
        _route("route_batch_sigmoid", 4099, 256, 8, True, True, 8, 4, True, True, 2.5),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "route"])
    if op == "route":
        experts = _spread(rng, 8, 512)
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if experts % g == 0 and experts // g >= 2])
        kept = rng.randint(1, groups)
        masked = rng.choice([0, 0, rng.randint(0, experts // 4)])
        k = rng.randint(1, min(16, max(1, kept * (experts // groups) - masked)))
        sigmoid = rng.random() < 0.6
        return _route("", _spread(rng, 1, 8192), experts, k, sigmoid, rng.random() < 0.6, groups, kept, rng.random() < 0.5, rng.random() < 0.7,
                      rng.choice([1.0, 2.5]), masked) | {"name": "drawn"}
    kind = rng.choice(["f16", "q8_0"])
    d = rng.choice([64, 96, 128, 128, 128, 160, 256] if kind == "q8_0" else [48, 64, 80, 128, 128, 128, 192, 256])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    if op == "store":
        kv = rng.randint(1, 8)
        seqs = _spread(rng, 1, 48)
        hi = _spread(rng, 1, max(2, min(8192, 20_000_000 // (seqs * kv * d))))
        lo = rng.randint(0, hi)
        new = rng.choice([0, 1, _spread(rng, 1, hi)])
        return _store("drawn", kind, seqs, lo, hi, new, rng.choice([0, 1]), kv, d, page, rng.random() < 0.5, pad=rng.choice([0, 5]))
    kv = rng.randint(1, 8)
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 12, 16])
    seqs = _spread(rng, 1, 160)
    hi = _spread(rng, 1, max(2, min(131072, 250_000_000 // (seqs * kv * d * max(1, group // 4)))))
    lo = rng.choice([0, hi, rng.randint(0, hi)])
    window = rng.choice([0, 0, 0, _spread(rng, 1, hi)])
    return _attend("drawn", kind, seqs, lo, hi, kv * group, kv, d, page, window)


def _lengths(case):
    """The sequences' lengths, spread evenly over lo..hi in a scattered order."""
    lo, hi = case["lo"], case["hi"]
    return [lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + 0.5) % 1.0)) for i in range(case["seqs"])]


def _rows(case):
    """The (sequence, position) rows that a store case writes and reads."""
    wrote, read = [], []
    for s, n in enumerate(_lengths(case)):
        first = max(0, n - case["new"]) if case["new"] else 0
        wrote += [(s, p) for p in range(first, n)]
        read += [(s, p) for p in range(0 if case["back"] else first, n)]
    return wrote, read


def _row_bytes(case):
    """Bytes of one token's keys (or values) of all heads in the cache."""
    return case["kv"] * (case["d"] * 2 if case["kind"] == "f16" else case["d"] + case["d"] // BLOCK * 2)


def work(case):
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        return {"bytes": 4 * t * e + 8 * t * k + (4 * e if case["bias"] else 0), "flops": 4 * t * e}
    lens = _lengths(case)
    if case["op"] == "store":
        first = [max(0, n - case["new"]) if case["new"] else 0 for n in lens]
        wrote = sum(n - f for n, f in zip(lens, first))
        read = sum(lens) if case["back"] else wrote
        width = case["kv"] * case["d"]
        moved = wrote * (8 * width + 2 * _row_bytes(case)) + read * (2 * _row_bytes(case) + width * (4 if case["half"] else 8))
        return {"bytes": moved + 8 * (wrote + read) + 16, "flops": 4 * (wrote + read) * width}
    seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
    heads, d = case["heads"], case["d"]
    return {"bytes": seen * 2 * _row_bytes(case) + 8 * case["seqs"] * heads * d + 16, "flops": 4 * seen * heads * d + 16}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _quantise(x):
    """8-bit blocks of 32 values (last axis) as the framework's Q8_0 has them: whole levels and f16 scales, all steps in f32."""
    x = x.unflatten(-1, (-1, BLOCK))
    step = x.abs().amax(-1, keepdim=True) / torch.full_like(x[..., :1], 127.0)
    inverse = torch.where(step == 0, 0.0, torch.ones_like(step) / step)
    a = (x * inverse).abs()
    level = torch.where(a - a.trunc() >= 0.5, a.trunc() + 1, a.trunc()).clamp(max=127)  # halves go away from zero
    return (level * x.sign()).to(torch.int8).flatten(-2), step.squeeze(-1).half()


def _table(case, gen, lens):
    """The table that names each sequence's pages, in scattered order."""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1)
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")  # entries behind a sequence's end name no page
    inside = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[inside] = order[: sum(need)]
    return {"table": table, "n_pages": total}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        s["logits"] = torch.randn(t, e, generator=gen, device="cuda") * 1.5
        if case["masked"]:  # experts that pad the layer to its size
            s["logits"][:, e - case["masked"]:] = -math.inf
        s["bias"] = torch.randn(e, generator=gen, device="cuda") * 0.05 if case["bias"] else None
        return s
    lens = _lengths(case)
    s |= _table(case, gen, lens)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for side in ("k", "v"):  # what the pages hold before the call
        x = torch.randn(s["n_pages"], case["kv"], case["page"], case["d"], generator=gen, device="cuda")
        s[side], s[side + "_scale"] = (x.half(), None) if case["kind"] == "f16" else _quantise(x)
    if case["op"] == "attend":
        s["q"] = torch.randn(case["seqs"], case["heads"], case["d"], generator=gen, device="cuda") * 1.5
        return s
    wrote, read = _rows(case)
    wrote = wrote + [(-1, 0)] * case["pad"]
    for what, rows in (("wrote", wrote), ("read", read)):
        at = torch.tensor(rows, dtype=torch.int32).reshape(-1, 2).cuda()
        s[what + "_seq"], s[what + "_pos"] = at[:, 0].contiguous(), at[:, 1].contiguous()
    # keys and values as they leave a fused projection: neighbours in one wider row
    width = case["kv"] * case["d"]
    s["fused"] = torch.randn(len(wrote), 2 * width, generator=gen, device="cuda")
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _at(s, seq, pos):
    """Page and slot of every (sequence, position)."""
    page = s["case"]["page"]
    return s["table"][seq.long(), pos.long() // page].long(), pos.long() % page


def _held(s, side, where, slot):
    """What the cache holds at these slots, in f32."""
    x = s[side][where, :, slot].float()
    if s[side + "_scale"] is None:
        return x
    return (x.unflatten(-1, (-1, BLOCK)) * s[side + "_scale"][where, :, slot].float()[..., None]).flatten(-2)


def _plain_store(s):
    case = s["case"]
    live = s["wrote_seq"] >= 0
    where, slot = _at(s, s["wrote_seq"][live], s["wrote_pos"][live])
    new = s["fused"][live].reshape(-1, 2, case["kv"], case["d"])
    if case["kind"] == "f16":
        s["k"][where, :, slot] = new[:, 0].half()
        s["v"][where, :, slot] = new[:, 1].half()
    else:
        s["k"][where, :, slot], s["k_scale"][where, :, slot] = _quantise(new[:, 0])
        s["v"][where, :, slot], s["v_scale"][where, :, slot] = _quantise(new[:, 1])
    where, slot = _at(s, s["read_seq"], s["read_pos"])
    out = torch.float16 if case["half"] else torch.float32
    return {"k": _held(s, "k", where, slot).to(out), "v": _held(s, "v", where, slot).to(out)}


def _plain_attend(s):
    case = s["case"]
    n, heads, kv, d = case["seqs"], case["heads"], case["kv"], case["d"]
    lens = s["lens"].long()[:, None]
    pos = torch.arange(max(case["hi"], 1), device="cuda")[None].expand(n, -1)
    seen = pos < lens
    if case["window"]:
        seen = seen & (pos >= lens - case["window"])
    where, slot = _at(s, torch.arange(n, device="cuda")[:, None], torch.where(seen, pos, 0))
    where = where.clamp(min=0)
    k = _held(s, "k", where, slot).permute(0, 2, 1, 3)
    q = s["q"].reshape(n, kv, heads // kv, d)
    x = (q @ k.transpose(-1, -2)) * d ** -0.5
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    high = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(high == -math.inf, 0.0, high))
    total = p.sum(-1, keepdim=True)
    v = _held(s, "v", where, slot).permute(0, 2, 1, 3)
    return ((p @ v) / torch.where(total == 0, 1.0, total)).reshape(n, heads, d)


def _plain_route(s):
    """Scores in 64 bits: two experts may lie closer than 32 bits tell."""
    case = s["case"]
    t, e, g = case["tokens"], case["experts"], case["groups"]
    x = s["logits"].double()
    if case["sigmoid"]:
        score = 1 / (1 + torch.exp(-x))
    else:
        score = torch.exp(x - x.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    key = score + s["bias"].double() if case["bias"] else score
    key = key.masked_fill(x == -math.inf, -math.inf)
    if g > 1:
        best = torch.sort(key.reshape(t, g, e // g), dim=-1, descending=True).values
        rank = best[..., 0] + best[..., 1] if case["best2"] else best[..., 0]
        kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, : case["kept"]]
        open_ = torch.zeros(t, g, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        key = key.masked_fill(~open_[..., None].expand(t, g, e // g).reshape(t, e), -math.inf)
    chosen = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, : case["k"]]
    weight = score.gather(1, chosen)
    if case["renorm"]:
        weight = weight / weight.sum(-1, keepdim=True)
    return {"selected": chosen.to(torch.int32), "weights": (weight * case["scale"]).float()}


# ---- the library's entries ------------------------------------------------------------------------------------------
def _keep(s):
    """What a program makes once and keeps: the description of its pages, its output buffers, the workspace."""
    from fucina_b200 import provider as P

    case = s["case"]
    s["P"] = P
    P.init(0)
    if case["op"] == "route":
        s["out"] = {"selected": torch.empty(case["tokens"], case["k"], dtype=torch.int32, device="cuda"),
                    "weights": torch.empty(case["tokens"], case["k"], device="cuda")}
        return
    s["pages"] = P.KvPages(P.KV_F16 if case["kind"] == "f16" else P.KV_Q8_0, s["k"], s["v"], s["k_scale"], s["v_scale"], s["n_pages"], case["page"],
                           case["kv"], case["d"])
    if case["op"] == "attend":
        s["out"] = torch.empty_like(s["q"])
        size = P.attn_paged_workspace_bytes(s["pages"], case["seqs"], case["heads"], case["hi"])
        s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    else:
        rows = (s["read_seq"].numel(), case["kv"], case["d"])
        s["out"] = {x: torch.empty(rows, dtype=torch.float16 if case["half"] else torch.float32, device="cuda") for x in ("k", "v")}
        s["value_rows"] = s["fused"][:, case["kv"] * case["d"]:]


def _own(s):
    if "P" not in s:
        _keep(s)
    P, case = s["P"], s["case"]
    if case["op"] == "route":
        P.router_groups_dev(s["logits"], case["tokens"], case["experts"], case["k"], s["out"]["selected"], s["out"]["weights"],
                            score=P.SCORE_SIGMOID if case["sigmoid"] else P.SCORE_SOFTMAX, bias_dev=s["bias"], n_group=case["groups"],
                            topk_group=case["kept"], group_score=P.GROUP_TOP2 if case["best2"] else P.GROUP_MAX, normalize=case["renorm"],
                            scale=case["scale"])
    elif case["op"] == "attend":
        P.attn_paged_dev(s["pages"], s["q"], s["out"], s["table"], s["lens"], case["seqs"], s["table"].shape[1], case["heads"], case["d"] ** -0.5,
                         window=case["window"], max_len=case["hi"], workspace=s["workspace"], workspace_bytes=s["workspace"].numel())
    else:
        n, width = s["table"].shape
        P.kv_append_dev(s["pages"], s["fused"], s["value_rows"], s["wrote_seq"], s["wrote_pos"], s["wrote_seq"].numel(), s["table"], n, width,
                        row_stride=s["fused"].shape[1])
        P.kv_read_dev(s["pages"], s["out"]["k"], s["out"]["v"], case["half"], s["read_seq"], s["read_pos"], s["read_seq"].numel(), s["table"], n, width)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "attend": _plain_attend, "route": _plain_route}[state["case"]["op"]](state)


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------
def _exact_blocks(rows):
    """Q8_0 of numpy f32 rows: the format fixes its steps in f32, so each is taken there; the values are given in 64 bits."""
    import numpy as np

    b = rows.reshape(-1, BLOCK)
    step = np.max(np.abs(b), axis=1, keepdims=True) / np.float32(127)
    with np.errstate(divide="ignore"):
        inverse = np.where(step > 0, np.float32(1) / step, np.float32(0)).astype(np.float32)
    y = (b * inverse).astype(np.float64)
    level = np.minimum(np.floor(np.abs(y) + 0.5), 127) * np.sign(y)
    return (level * step.astype(np.float16).astype(np.float64)).reshape(rows.shape)


def _dense(s, side):
    """All pages of one side as f64 numpy rows [page][slot][head][d]."""
    x = s[side].double()
    if s[side + "_scale"] is not None:
        x = x * s[side + "_scale"].double().repeat_interleave(BLOCK, dim=-1)
    return x.transpose(1, 2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        t, e, g, k = case["tokens"], case["experts"], case["groups"], case["k"]
        x = s["logits"].cpu().double().numpy()
        import numpy as np

        if case["sigmoid"]:
            score = 0.5 * (1 + np.tanh(0.5 * x))
        else:
            score = np.exp(x - np.logaddexp.reduce(x, axis=1, keepdims=True))
        key = score + (s["bias"].cpu().double().numpy() if case["bias"] else 0.0)
        key[np.isneginf(x)] = -np.inf
        if g > 1:
            best = -np.sort(-key.reshape(t, g, e // g), axis=2)
            rank = best[:, :, :2].sum(2) if case["best2"] else best[:, :, 0]
            shut = np.argsort(-rank, axis=1, kind="stable")[:, case["kept"]:]
            blocks = key.reshape(t, g, e // g)
            blocks[np.arange(t)[:, None], shut] = -np.inf
        chosen = np.argsort(-key, axis=1, kind="stable")[:, :k]
        weight = np.take_along_axis(score, chosen, 1)
        if case["renorm"]:
            weight = weight / weight.sum(1, keepdims=True)
        return {"selected": None, "weights": torch.from_numpy(weight * case["scale"])}
    page = case["page"]
    if case["op"] == "store":
        import numpy as np

        sides = []
        live = (s["wrote_seq"] >= 0).cpu()
        for i, side in enumerate(("k", "v")):
            held = _dense(s, side).cpu()
            new = s["fused"].cpu()[live].reshape(-1, 2, case["kv"], case["d"])[:, i].contiguous().numpy()
            new = new.astype(np.float16).astype(np.float64) if case["kind"] == "f16" else _exact_blocks(new)
            table = s["table"].cpu()
            seq, pos = s["wrote_seq"].cpu()[live].long(), s["wrote_pos"].cpu()[live].long()
            held[table[seq, pos // page].long(), pos % page] = torch.from_numpy(new)
            seq, pos = s["read_seq"].cpu().long(), s["read_pos"].cpu().long()
            sides.append(held[table[seq, pos // page].long(), pos % page])
        return {"k": sides[0], "v": sides[1]}
    # one sequence after the other, over its own pages
    out = torch.zeros(case["seqs"], case["heads"], case["d"], dtype=torch.float64, device="cuda")
    if sum(_lengths(case)) * case["heads"] * case["d"] > 4e9:
        return None
    group = case["heads"] // case["kv"]
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        used = s["table"][i, : -(-n // page)].long()
        first = max(0, n - case["window"]) if case["window"] else 0
        k, v = ({"k": s["k"][used], "k_scale": None if s["k_scale"] is None else s["k_scale"][used]},
                {"v": s["v"][used], "v_scale": None if s["v_scale"] is None else s["v_scale"][used]})
        k = _dense(k, "k").reshape(-1, case["kv"], case["d"])[first:n].repeat_interleave(group, dim=1)
        v = _dense(v, "v").reshape(-1, case["kv"], case["d"])[first:n].repeat_interleave(group, dim=1)
        x = torch.einsum("hd,jhd->hj", s["q"][i].double(), k) / math.sqrt(case["d"])
        out[i] = torch.einsum("hj,jhd->hd", torch.softmax(x, dim=1), v)
    return out

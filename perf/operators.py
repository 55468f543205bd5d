"""Cases, plain forms and 64-bit values of the operators around attention: rotary
positions with several axes (training, and the serving form that appends to a cache),
attention of a batch that shares a long prefix, and eviction from a cache by the
attention weight its entries received.

``run`` computes an operator in elementary torch operations in 32 bits, or, where ``own``
is true, through the framework's public entry points; ``exact`` gives the values that the
definitions have in 64 bits, by another route.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One user's decode step: a token is rotated and joins a cache of 4096 slots.
        dict(name="append one", op="append", dtype="bf16", layout="bshd", B=1, T=1, Hq=32, Hk=8, D=128, C=4096, pairing="half", sections="16,24,24", base=1e6),
        # A serving batch's decode step, ragged cache lengths.
        dict(name="append batch", op="append", dtype="fp16", layout="bhsd", B=160, T=1, Hq=32, Hk=8, D=128, C=257, pairing="adjacent", sections="16,24,24", base=1e4),
        # Training at the sequence length and heads of the framework's headline benchmark.
        dict(name="rotary train 8192", op="rotary", dtype="bf16", layout="bhsd", B=1, T=8192, Hq=32, Hk=8, D=128, pairing="half", sections="16,24,24", base=1e6),
        # A video's patches in one long sequence, wide heads, odd length.
        dict(name="rotary train video", op="rotary", dtype="fp16", layout="bshd", B=2, T=16385, Hq=16, Hk=8, D=256, pairing="adjacent", sections="32,48,48", base=1e4),
        # One user after a system prompt: the step's latency.
        dict(name="attend one", op="attend", dtype="bf16", layout="bshd", B=1, T=1, Hq=32, Hk=8, D=128, P=1024, C=512, low=300, high=300, mask=False, weights=False),
        # A chat server's batch behind one system prompt, weights kept for eviction.
        dict(name="attend chat", op="attend", dtype="bf16", layout="bshd", B=32, T=1, Hq=32, Hk=8, D=128, P=4096, C=2048, low=1, high=2048, mask=False, weights=True),
        # One key head for all queries, narrow heads, an odd prefix.
        dict(name="attend one key head", op="attend", dtype="fp16", layout="bhsd", B=48, T=1, Hq=64, Hk=1, D=64, P=8191, C=1024, low=17, high=1023, mask=False, weights=False),
        # Draft trees verified in one step: several new tokens under a mask, wide heads.
        dict(name="attend draft trees", op="attend", dtype="bf16", layout="bhsd", B=16, T=6, Hq=16, Hk=4, D=256, P=2050, C=777, low=6, high=770, mask=True, weights=True),
        # A large batch over a long shared document, each request with a long history.
        dict(name="attend large", op="attend", dtype="bf16", layout="bshd", B=128, T=1, Hq=32, Hk=8, D=128, P=32768, C=4096, low=512, high=4096, mask=False, weights=True),
        # One user's cache halved.
        dict(name="evict one", op="evict", dtype="bf16", layout="bshd", B=1, Hk=8, D=128, C=1024, keep=512, sinks=4, recent=64, low=1024, high=1024),
        # A batch brought back to its budget; some requests are still below it.
        dict(name="evict batch", op="evict", dtype="bf16", layout="bshd", B=32, Hk=8, D=128, C=2304, keep=1536, sinks=4, recent=256, low=1100, high=2304),
        # Few long caches, narrow heads.
        dict(name="evict long", op="evict", dtype="fp16", layout="bhsd", B=4, Hk=8, D=64, C=65536, keep=32768, sinks=1, recent=1024, low=50001, high=65536),
    ]


HEADS = [(8, 2, 64), (32, 8, 128), (64, 1, 64), (16, 16, 96), (16, 4, 256), (28, 4, 128), (12, 3, 64)]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _sections(rng, pairs):
    """A split of the pairs over two to four axes, in whole pairs."""
    axes = rng.choice([2, 3, 3, 4])
    cuts = sorted(rng.sample(range(1, pairs), axes - 1))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))


def draw(rng):
    op = rng.choice(["append", "rotary", "attend", "attend", "evict"])
    Hq, Hk, D = rng.choice(HEADS)
    case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), layout=rng.choice(["bshd", "bhsd"]))
    if op in ("append", "rotary"):
        case.update(Hq=Hq, Hk=Hk, D=D, pairing=rng.choice(["half", "adjacent"]), sections=_sections(rng, D // 2), base=rng.choice([1e4, 5e5, 1e6]))
    if op == "append":
        case.update(B=_between(rng, 1, 200), T=rng.choice([1, 1, 1, 2, 5]), C=_between(rng, 64, 1024))
    elif op == "rotary":
        case.update(B=rng.choice([1, 1, 2, 3]), T=_between(rng, 256, 40000))
        while work(case)["bytes"] > 2e9:
            case["T"] = case["T"] * 2 // 3
    elif op == "attend":
        T = rng.choice([1, 1, 1, 1, 3, 7])
        C = _between(rng, 64, 4096)
        case.update(B=_between(rng, 1, 160), T=T, Hq=Hq, Hk=Hk, D=D, P=_between(rng, 128, 40000), C=C, low=rng.randint(T, min(C, 512)), high=C, mask=T > 1 and rng.random() < 0.5, weights=rng.random() < 0.6)
        case["low"] = min(case["low"], case["high"])
        while work(case)["bytes"] > 2e9 or work(case)["flops"] > 7e10 or case["B"] * T * Hq * case["P"] > 2 ** 28:
            case["B"], case["P"] = (case["B"] + 1) // 2, case["P"] * 3 // 4 + 1
    else:
        C = _between(rng, 300, 65536)
        keep = max(2, int(C * rng.uniform(0.3, 0.9)))
        case.update(B=_between(rng, 1, 48), Hk=Hk, D=D, C=C, keep=keep, sinks=rng.choice([0, 1, 4]) if keep > 8 else 0, recent=int(keep * rng.uniform(0, 0.6)), low=rng.randint(C // 2, C), high=C)
        while work(case)["bytes"] > 2e9 or case["B"] * Hk * C * D > 2 ** 29:
            case["B"] = case["B"] // 2 or 1
            if case["B"] == 1:
                case["Hk"] = 1
    return case


def _lengths(case):
    """Cache lengths of the batch: even steps from low to high (a seed only shuffles them)."""
    return [int(round(case["low"] + (case["high"] - case["low"]) * i / max(1, case["B"] - 1))) for i in range(case["B"])]


def _positions(T, offset):
    """[3, T]: a text part, where all axes count alike, then a video's patches."""
    text = T // 4
    i = np.arange(T - text)
    h, w = 18, 32
    grid = np.stack([i // (h * w), i // w % h, i % w]) + text
    return torch.from_numpy(np.concatenate([np.tile(np.arange(text), (3, 1)), grid], 1) + offset)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op, B, D = DTYPES[case["dtype"]], case["op"], case["B"], case["D"]
    seq_first = case["layout"] == "bshd"

    def randn(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if math.prod(shape) < 1 << 26 else dt).mul_(scale).to(dt)

    def tokens(n, heads, scale=1.0):
        return randn(B, n, heads, D, scale=scale) if seq_first else randn(B, heads, n, D, scale=scale)

    state = dict(case)
    if op in ("append", "rotary"):
        sections = [int(x) for x in case["sections"].split(",")]
        axes = len(sections)
        state["half"] = D // 2
        state["axis"] = torch.repeat_interleave(torch.arange(axes), torch.tensor(sections)).cuda()
        state["inv_freq"] = (case["base"] ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)).float().cuda()
        if own:
            import tilelang_fa2_4d_mask as api

            state["rotary"] = api.MultiAxisRotary(D, sections, base=case["base"], pairing=case["pairing"])
        T, Hq, Hk = case["T"], case["Hq"], case["Hk"]
        state["q"], state["k"] = tokens(T, Hq), tokens(T, Hk)
    if op == "rotary":
        pos = torch.cat([_positions(T, seed % 17 + 7 * b)[None] for b in range(B)])  # [B, 3, T]
        state["positions"] = pos[:, torch.arange(axes) % 3].transpose(0, 1).contiguous().cuda()  # [axes, B, T]
        state["dq"], state["dk"] = tokens(T, Hq), tokens(T, Hk)
        state["q"].requires_grad_(own), state["k"].requires_grad_(own)
    elif op == "append":
        C = case["C"]
        state["v"] = tokens(T, Hk)
        state["k_cache"], state["v_cache"] = tokens(C, Hk), tokens(C, Hk)
        state["weights"] = torch.rand((B, Hk, C), generator=g, device="cuda")
        state["lengths"] = torch.randint(0, C - T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        start = 2000 + state["lengths"].long()
        state["positions"] = (start[None, :, None] + torch.arange(T, device="cuda")).expand(axes, B, T).contiguous()
    elif op == "attend":
        T, Hq, Hk, P, C = case["T"], case["Hq"], case["Hk"], case["P"], case["C"]
        state["q"] = tokens(T, Hq, scale=1.5)
        state["k"], state["v"] = tokens(C, Hk), tokens(C, Hk)
        state["pk"], state["pv"] = (randn(P, Hk, D) if seq_first else randn(Hk, P, D) for _ in range(2))
        order = torch.randperm(B, generator=g, device="cuda")
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32).cuda()[order]
        # Weight gathered so far, of the size of what one step adds.
        state["weights"] = torch.rand((B, Hk, C), generator=g, device="cuda").mul_(2 * T * Hq / (Hk * (P + C))) if case["weights"] else None
        state["mask"] = None
        if case["mask"]:
            # Each request's new tokens form a tree: a token sees its ancestors and itself.
            rng = np.random.RandomState(seed % (1 << 31))
            sees = np.zeros((B, T, T), bool)
            for t in range(T):
                if t:
                    sees[:, t] = sees[np.arange(B), rng.randint(0, t, B)]
                sees[:, t, t] = True
            mask = torch.ones((B, 1, T, C), dtype=torch.bool, device="cuda")
            at = (state["lengths"].long() - T)[:, None] + torch.arange(T, device="cuda")
            state["mask"] = mask.scatter_(3, at[:, None, None].expand(B, 1, T, T), torch.from_numpy(sees).cuda()[:, None])
    elif op == "evict":
        Hk, C = case["Hk"], case["C"]
        state["k"], state["v"] = tokens(C, Hk), tokens(C, Hk)
        order = torch.randperm(B, generator=g, device="cuda")
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32).cuda()[order]
        # Few entries gather most of the weight, and some none at all.
        w = torch.randn((B, Hk, C), generator=g, device="cuda").mul_(2).exp_()
        state["weights"] = w * (torch.rand((B, Hk, C), generator=g, device="cuda") > 0.1)
    return state


# ---------------------------------------------------------------------------- plain forms


def _rotate(x, cos, sin, pairing):
    """x [..., D] in 32 bits, cos/sin broadcast over its last but one axes."""
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if pairing == "half" else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([a, b], -1) if pairing == "half" else torch.stack([a, b], -1).flatten(-2)


def _angles(s):
    """cos, sin [B, T, D/2], with an axis for the heads where the layout has it."""
    phi = s["positions"].float()[s["axis"]].permute(1, 2, 0) * s["inv_freq"]
    phi = phi.unsqueeze(2 if s["layout"] == "bshd" else 1)
    return phi.cos(), phi.sin()


def _plain_rotary(s):
    cos, sin = _angles(s)
    q, k = (_rotate(s[n].float(), cos, sin, s["pairing"]).to(s[n].dtype) for n in ("q", "k"))
    dq, dk = (_rotate(s[n].float(), cos, -sin, s["pairing"]).to(s[n].dtype) for n in ("dq", "dk"))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _plain_append(s):
    cos, sin = _angles(s)
    q, k = (_rotate(s[n].float(), cos, sin, s["pairing"]).to(s[n].dtype) for n in ("q", "k"))
    seq = 1 if s["layout"] == "bshd" else 2
    slots = s["lengths"].long()[:, None] + torch.arange(s["T"], device="cuda")
    rows = torch.arange(s["B"], device="cuda")[:, None]
    s["k_cache"].transpose(1, seq)[rows, slots] = k.transpose(1, seq)
    s["v_cache"].transpose(1, seq)[rows, slots] = s["v"].transpose(1, seq)
    s["weights"].transpose(1, 2)[rows, slots] = 0.0
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"], "weights": s["weights"], "lengths": s["lengths"] + s["T"]}


def _plain_attend(s):
    B, T, Hq, Hk, D, C = s["B"], s["T"], s["Hq"], s["Hk"], s["D"], s["C"]
    heads_first = s["layout"] == "bhsd"
    q = s["q"].float() if heads_first else s["q"].float().transpose(1, 2)
    k, v = (s[n].float() if heads_first else s[n].float().transpose(1, 2) for n in ("k", "v"))
    pk, pv = (s[n].float() if heads_first else s[n].float().transpose(0, 1) for n in ("pk", "pv"))
    q = q.reshape(B, Hk, Hq // Hk * T, D) * D ** -0.5  # rows (head of the group, token)
    shared = torch.matmul(q.transpose(0, 1).reshape(Hk, -1, D), pk.transpose(1, 2)).reshape(Hk, B, -1, pk.shape[1])
    each = torch.matmul(q, k.transpose(2, 3)).reshape(B, Hk, Hq // Hk, T, C)
    j = torch.arange(C, device="cuda")
    t = torch.arange(T, device="cuda")
    see = j <= s["lengths"].long()[:, None, None] - T + t[:, None]  # [B, T, C]
    if s["mask"] is not None:
        see = see & s["mask"][:, 0]
    each = each.masked_fill(~see[:, None, None], -math.inf).flatten(2, 3)
    m = torch.maximum(shared.amax(-1).transpose(0, 1), each.amax(-1)).unsqueeze(-1)
    shared, each = (shared - m.transpose(0, 1)).exp(), (each - m).exp()
    total = shared.sum(-1).transpose(0, 1) + each.sum(-1)
    out = torch.matmul(shared.reshape(Hk, -1, pk.shape[1]), pv).reshape(Hk, B, -1, D).transpose(0, 1) + torch.matmul(each, v)
    out = (out / total.unsqueeze(-1)).reshape(B, Hq, T, D).to(s["q"].dtype)
    found = {"out": out if heads_first else out.transpose(1, 2)}
    if s["weights"] is not None:
        found["weights"] = s["weights"].add_((each / total.unsqueeze(-1)).sum(2))
    return found


def _plain_evict(s):
    keep, C, heads_first = s["keep"], s["C"], s["layout"] == "bhsd"
    n = s["lengths"].long()[:, None, None]
    j = torch.arange(C, device="cuda")
    worth = torch.where((j < s["sinks"]) | (j >= n - s["recent"]), math.inf, s["weights"])
    worth = torch.where(j < n, worth, -math.inf)
    index = worth.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(dim=-1).values
    live = torch.arange(keep, device="cuda") < n
    at = index.unsqueeze(-1).expand(-1, -1, -1, s["D"])
    if not heads_first:
        at = at.transpose(1, 2)
    gone = ~live.unsqueeze(-1) if heads_first else ~live.transpose(1, 2).unsqueeze(-1)
    seq = 2 if heads_first else 1
    k, v = (s[x].gather(seq, at).masked_fill(gone, 0.0) for x in ("k", "v"))
    weights = s["weights"].gather(2, index).masked_fill(~live, 0.0)
    return {"k": k, "v": v, "weights": weights, "lengths": s["lengths"].clamp(max=keep), "index": index.masked_fill(~live, -1).int()}


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}


def _own(s):
    import tilelang_fa2_4d_mask as api

    op, layout = s["op"], s["layout"]
    if op == "rotary":
        q, k = s["rotary"](s["q"], s["k"], s["positions"], layout=layout)
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if op == "append":
        q, lengths = s["rotary"].append(s["q"], s["k"], s["v"], s["positions"], s["k_cache"], s["v_cache"], s["lengths"], weights=s["weights"], layout=layout)
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"], "weights": s["weights"], "lengths": lengths}
    if op == "attend":
        out = api.shared_prefix_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lengths"], mask=s["mask"], weights=s["weights"], layout=layout)
        return {"out": out} if s["weights"] is None else {"out": out, "weights": s["weights"]}
    k, v, weights, lengths, index = api.evict_by_weight(s["k"], s["v"], s["weights"], s["lengths"], keep=s["keep"], sinks=s["sinks"], recent=s["recent"], layout=layout)
    return {"k": k, "v": v, "weights": weights, "lengths": lengths, "index": index}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


def work(case):
    op, B, D, Hk = case["op"], case["B"], case["D"], case["Hk"]
    if op == "rotary":
        moved = B * case["T"] * (case["Hq"] + Hk) * D
        return {"bytes": 2 * (2 * moved * 2) + 8 * 3 * B * case["T"], "flops": 2 * 3 * moved}
    if op == "append":
        n = B * case["T"]
        return {"bytes": n * (2 * case["Hq"] * D * 2 + 2 * 2 * Hk * D * 2 + 4 * Hk + 24) + 8 * B, "flops": 3 * n * (case["Hq"] + Hk) * D}
    if op == "attend":
        T, Hq, P, own_keys = case["T"], case["Hq"], case["P"], sum(_lengths(case))
        size = 2 * 2 * B * T * Hq * D + 2 * 2 * P * Hk * D + 2 * 2 * own_keys * Hk * D
        size += (2 * 4 * own_keys * Hk if case["weights"] else 0) + (T * own_keys if case["mask"] else 0)
        return {"bytes": size, "flops": 4 * D * Hq * T * (B * P + own_keys)}
    lengths = _lengths(case)
    kept = sum(min(n, case["keep"]) for n in lengths)
    return {"bytes": Hk * (4 * sum(lengths) + kept * (2 * 2 * 2 * D + 4 + 4)), "flops": 0}


# ---------------------------------------------------------------------------- 64 bits


def _exact_turn(x, s, sign):
    """Each pair as a complex number times e^(i phi), phi in 64 bits."""
    D, layout = s["D"], s["layout"]
    x = x.detach().double()
    half = D // 2
    sections = [int(n) for n in s["sections"].split(",")]
    axis = sum(([a] * n for a, n in enumerate(sections)), [])
    theta = torch.tensor([s["base"] ** (-2.0 * i / D) for i in range(half)], dtype=torch.float64, device="cuda")
    phi = torch.stack([s["positions"][a].double() for a in axis], -1) * theta
    turn = torch.polar(torch.ones_like(phi), sign * phi)
    turn = turn[:, :, None] if layout == "bshd" else turn[:, None]
    pair = torch.stack([x[..., :half], x[..., half:]], -1) if s["pairing"] == "half" else x.unflatten(-1, (half, 2))
    y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    return torch.cat([y[..., 0], y[..., 1]], -1) if s["pairing"] == "half" else y.flatten(-2)


def _exact_attend(s):
    """Request by request: softmax over the prefix's and the request's own keys together."""
    B, T, Hq, Hk, D, P = s["B"], s["T"], s["Hq"], s["Hk"], s["D"], s["P"]
    bshd = s["layout"] == "bshd"
    pk, pv = (x.permute(1, 0, 2) if bshd else x for x in (s["pk"], s["pv"]))
    pk, pv = pk.double(), pv.double()
    outs, weights = [], None if s["weights"] is None else s["weights"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        q, k, v = (x[b].transpose(0, 1) if bshd else x[b] for x in (s["q"], s["k"], s["v"]))
        q = q.double().reshape(Hk, Hq // Hk, T, D)
        k, v = torch.cat([pk, k[:, :n].double()], 1), torch.cat([pv, v[:, :n].double()], 1)
        logits = torch.einsum("hgtd,hjd->hgtj", q, k) / math.sqrt(D)
        late = torch.ones(T, n, dtype=torch.bool, device="cuda").triu(n - T + 1)
        if s["mask"] is not None:
            late |= ~s["mask"][b, 0, :, :n]
        logits[..., P:][late.expand(Hk, Hq // Hk, T, n)] = -math.inf
        p = torch.softmax(logits, -1)
        out = torch.einsum("hgtj,hjd->hgtd", p, v).reshape(Hq, T, D)
        outs.append(out.transpose(0, 1) if bshd else out)
        if weights is not None:
            weights[b, :, :n] += p[..., P:].sum((1, 2))
    found = {"out": torch.stack(outs)}
    return found if weights is None else dict(found, weights=weights)


def _exact_evict(s):
    """numpy, head by head: the entries in order of (weight, index)."""
    B, Hk, keep = s["B"], s["Hk"], s["keep"]
    w, lengths = s["weights"].double().cpu().numpy(), s["lengths"].tolist()
    index = np.full((B, Hk, keep), -1, np.int32)
    kept = np.zeros((B, Hk, keep))
    for b, n in enumerate(lengths):
        for h in range(Hk):
            if n <= keep:
                chosen = np.arange(n)
            else:
                middle = np.arange(s["sinks"], n - s["recent"])
                best = middle[np.lexsort((middle, -w[b, h, middle]))][: keep - s["sinks"] - s["recent"]]
                chosen = np.sort(np.concatenate([np.arange(s["sinks"]), best, np.arange(n - s["recent"], n)]))
            index[b, h, : len(chosen)] = chosen
            kept[b, h, : len(chosen)] = w[b, h, chosen]
    at = torch.from_numpy(index).long().cuda()
    live = (at >= 0).unsqueeze(-1)
    rows, heads = torch.arange(B, device="cuda")[:, None, None], torch.arange(Hk, device="cuda")[:, None]
    k, v = (torch.where(live, (x.transpose(1, 2) if s["layout"] == "bshd" else x)[rows, heads, at.clamp(min=0)].double(), 0.0) for x in (s["k"], s["v"]))
    if s["layout"] == "bshd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return {"k": k, "v": v, "weights": kept, "lengths": np.minimum(lengths, keep), "index": index}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return {"q": _exact_turn(s["q"], s, 1), "k": _exact_turn(s["k"], s, 1), "dq": _exact_turn(s["dq"], s, -1), "dk": _exact_turn(s["dk"], s, -1)}
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "evict":
        return _exact_evict(s)
    # append: the caches change at the new tokens' slots only.
    q, k = _exact_turn(s["q"], s, 1), _exact_turn(s["k"], s, 1)
    kc, vc, weights = s["k_cache"].double(), s["v_cache"].double(), s["weights"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        at = (b, slice(n, n + case["T"])) if case["layout"] == "bshd" else (b, slice(None), slice(n, n + case["T"]))
        kc[at], vc[at] = k[b], s["v"][b].double()
        weights[b, :, n : n + case["T"]] = 0.0
    return {"q": q, "k_cache": kc, "v_cache": vc, "weights": weights, "lengths": s["lengths"] + case["T"]}

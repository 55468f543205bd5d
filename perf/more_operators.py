"""Cases, plain forms and 64-bit values of the operators of models that normalise queries and
keys and keep their caches in 8 bits: the norm of each head with the rotary turn in the same
pass (training, and the serving form that appends to a cache), caches of 8-bit codes with a
power-of-two scale for each block of 64 tokens and head, and attention over them.

``run`` computes an operator in elementary torch operations in 32 bits, or, where ``own``
is true, through the framework's public entry points; ``exact`` gives the values that the
definitions have in 64 bits, by another route.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MOST = {"e4m3": 448.0, "int8": 127.0}  # the largest value of a code
BLOCK = 64  # tokens that share a scale
EPS = 1e-6


def listed():
    return [
        # A short fine-tuning step of a small model with narrow heads.
        dict(name="norm train short", op="norm", dtype="fp16", layout="bshd", B=2, T=384, Hq=8, Hk=2, D=64, pairing="adjacent", sections="8,12,12", base=1e4, weight="same"),
        # Training at the sequence length and heads of the framework's headline benchmark, master weights.
        dict(name="norm train 8192", op="norm", dtype="bf16", layout="bhsd", B=1, T=8192, Hq=32, Hk=8, D=128, pairing="half", sections="16,24,24", base=1e6, weight="fp32"),
        # A video's patches in one long sequence, wide heads, odd length.
        dict(name="norm train video", op="norm", dtype="fp16", layout="bshd", B=2, T=16385, Hq=16, Hk=8, D=256, pairing="adjacent", sections="32,48,48", base=1e4, weight="same"),
        # One user's decode step into an 8-bit cache, which is then read back (it becomes a prefix, say).
        dict(name="append one", op="append", cache="e4m3", norm=True, dtype="bf16", layout="bshd", B=1, T=1, Hq=32, Hk=8, D=128, C=1024, pairing="half", sections="16,24,24", base=1e6, weight="same"),
        # A serving batch's decode step of a model without norms, caches that end inside a block.
        dict(name="append batch", op="append", cache="int8", norm=False, dtype="fp16", layout="bhsd", B=64, T=1, Hq=32, Hk=8, D=128, C=300, pairing="adjacent", sections="16,24,24", base=1e4, weight="same"),
        # Two prompts of odd length join caches that hold something already.
        dict(name="append prompt", op="append", cache="e4m3", norm=True, dtype="bf16", layout="bshd", B=2, T=4097, Hq=32, Hk=8, D=128, C=6000, pairing="half", sections="16,24,24", base=1e6, weight="same"),
        # The decode step of a model with norms whose cache stays in 16 bits.
        dict(name="append 16 bits", op="append", cache="same", norm=True, dtype="bf16", layout="bshd", B=160, T=1, Hq=16, Hk=4, D=256, C=64, pairing="half", sections="32,48,48", base=1e6, weight="fp32"),
        # One user with a conversation of some thousand tokens: the step's latency.
        dict(name="attend one", op="attend", cache="e4m3", dtype="bf16", layout="bshd", B=1, T=1, Hq=32, Hk=8, D=128, P=0, C=4096, low=4000, high=4000, mask=False),
        # A chat server's batch behind one system prompt.
        dict(name="attend chat", op="attend", cache="e4m3", dtype="bf16", layout="bshd", B=32, T=1, Hq=32, Hk=8, D=128, P=4096, C=4096, low=1, high=4096, mask=False),
        # One key head for all queries, narrow heads.
        dict(name="attend one key head", op="attend", cache="int8", dtype="fp16", layout="bhsd", B=48, T=1, Hq=64, Hk=1, D=64, P=0, C=8191, low=17, high=8191, mask=False),
        # Draft trees verified in one step: several new tokens under a mask, wide heads.
        dict(name="attend draft trees", op="attend", cache="int8", dtype="bf16", layout="bhsd", B=16, T=6, Hq=16, Hk=4, D=256, P=0, C=2050, low=6, high=2050, mask=True),
        # A large batch, each request with a long history.
        dict(name="attend large", op="attend", cache="e4m3", dtype="bf16", layout="bshd", B=64, T=1, Hq=32, Hk=8, D=128, P=0, C=16384, low=2048, high=16384, mask=False),
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
    op = rng.choice(["norm", "append", "attend", "attend"])
    Hq, Hk, D = rng.choice(HEADS)
    case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), layout=rng.choice(["bshd", "bhsd"]))
    if op in ("norm", "append"):
        case.update(Hq=Hq, Hk=Hk, D=D, pairing=rng.choice(["half", "adjacent"]), sections=_sections(rng, D // 2), base=rng.choice([1e4, 5e5, 1e6]), weight=rng.choice(["same", "fp32"]))
    if op == "norm":
        case.update(B=rng.choice([1, 1, 2, 3]), T=_between(rng, 100, 30000))
        while work(case)["bytes"] > 2e9:
            case["T"] = case["T"] * 2 // 3
    elif op == "append":
        cache = rng.choice(["e4m3", "e4m3", "int8", "int8", "same"])
        T = rng.choice([1, 1, 1, 2, 7, _between(rng, 30, 4500)])
        case.update(cache=cache, norm=cache == "same" or rng.random() < 0.7, B=_between(rng, 1, 160), T=T, C=T + _between(rng, 1, 2000))
        while case["B"] > 1 and case["B"] * (case["C"] * Hk + T * Hq) * D > 1 << 26:
            case["B"] //= 2
    else:
        T = rng.choice([1, 1, 1, 1, 3, 7])
        C = _between(rng, 64, 16384)
        case.update(cache=rng.choice(["e4m3", "int8"]), B=_between(rng, 1, 100), T=T, Hq=Hq, Hk=Hk, D=D, P=rng.choice([0, 0, _between(rng, 100, 8000)]), C=C, low=rng.randint(T, C), high=C, mask=T > 1 and rng.random() < 0.5)
        while case["B"] > 1 and (case["B"] * Hk * C * D > 1 << 28 or work(case)["flops"] > 2e10 or case["B"] * T * Hq * (case["P"] + C) > 1 << 26):
            case["B"] //= 2
    return case


def _lengths(case):
    """Cache lengths of the batch: even steps from low to high (a seed only shuffles them)."""
    return [int(round(case["low"] + (case["high"] - case["low"]) * i / max(1, case["B"] - 1))) for i in range(case["B"])]


def _positions(T, offset):
    """[3, T]: a text part, where all axes count alike, then a video's patches."""
    text = T // 4
    i = torch.arange(T - text)
    h, w = 18, 32
    grid = torch.stack([i // (h * w), i // w % h, i % w]) + text
    return torch.cat([torch.arange(text).expand(3, -1), grid], 1) + offset


def _by_block(x, C):
    """[..., blocks] to [..., C]: each token's."""
    return x.repeat_interleave(BLOCK, -1)[..., :C]


def _least_scale(most, cache):
    """The least power of two, from 2^-126 up, under which `most` does not pass the largest code."""
    m, e = torch.frexp(most.double() / MOST[cache])
    return torch.exp2(torch.where(m > 0.5, e, e - 1).clamp(min=-126).float())


def _codes(x, cache):
    return x.round().to(torch.int8) if cache == "int8" else x.to(torch.float8_e4m3fn)


def _fill(case, g, C):
    """Codes and scales of a cache that holds keys or values: some channels and some blocks are larger."""
    B, Hk, D, cache = case["B"], case["Hk"], case["D"], case["cache"]
    seq = 1 if case["layout"] == "bshd" else 2
    codes = torch.empty((B, C, Hk, D) if seq == 1 else (B, Hk, C, D), dtype=CODES[cache], device="cuda")
    scales = torch.empty((B, Hk, -(-C // BLOCK)), device="cuda")
    channel = 1 + 3 * (torch.rand(D, generator=g, device="cuda") < 0.05)
    for b in range(B):  # request by request, so that large caches need little beside themselves
        size = torch.exp2(torch.rand((Hk, scales.shape[2]), generator=g, device="cuda") * 2 - 1)
        x = torch.randn((Hk, C, D), generator=g, device="cuda").mul_(channel).mul_(_by_block(size, C).unsqueeze(-1))
        pad = torch.nn.functional.pad(x.abs().amax(-1), (0, scales.shape[2] * BLOCK - C))
        scales[b] = _least_scale(pad.view(Hk, -1, BLOCK).amax(-1), cache)
        codes[b] = _codes(x / _by_block(scales[b], C).unsqueeze(-1), cache).transpose(0, 2 - seq)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op, B, D = DTYPES[case["dtype"]], case["op"], case["B"], case["D"]
    T, Hq, Hk = case["T"], case["Hq"], case["Hk"]
    seq_first = case["layout"] == "bshd"

    def randn(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dt)

    def tokens(n, heads, scale=1.0):
        return randn(B, n, heads, D, scale=scale) if seq_first else randn(B, heads, n, D, scale=scale)

    state = dict(case)
    state["q"] = tokens(T, Hq, scale=1.5)
    if op in ("norm", "append"):
        sections = [int(x) for x in case["sections"].split(",")]
        axes = len(sections)
        state["axis"] = torch.repeat_interleave(torch.arange(axes), torch.tensor(sections)).cuda()
        state["inv_freq"] = (case["base"] ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)).cuda()
        if own:
            import tilelang_fa2_4d_mask as api

            state["rotary"] = api.MultiAxisRotary(D, sections, base=case["base"], pairing=case["pairing"])
        state["k"] = tokens(T, Hk, scale=0.7)
        wide = torch.float32 if case["weight"] == "fp32" else dt
        state["wq"], state["wk"] = (torch.randn(D, generator=g, device="cuda").mul_(0.2).add_(1.0).to(wide) for _ in range(2))
    if op == "norm":
        pos = torch.cat([_positions(T, seed % 17 + 7 * b)[None] for b in range(B)])  # [B, 3, T]
        state["positions"] = pos[:, torch.arange(axes) % 3].transpose(0, 1).contiguous().cuda()  # [axes, B, T]
        state["dq"], state["dk"] = tokens(T, Hq), tokens(T, Hk)
        for n in ("q", "k", "wq", "wk"):
            state[n].requires_grad_(own)
    elif op == "append":
        C = case["C"]
        state["v"] = tokens(T, Hk)
        if case["cache"] == "same":
            state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"] = tokens(C, Hk), tokens(C, Hk), None, None
        else:
            (state["k_cache"], state["k_scale"]), (state["v_cache"], state["v_scale"]) = _fill(case, g, C), _fill(case, g, C)
        state["lengths"] = torch.randint(0, C - T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        start = 2000 + state["lengths"].long()
        state["positions"] = (start[None, :, None] + torch.arange(T, device="cuda")).expand(axes, B, T).contiguous()
    else:
        P, C = case["P"], case["C"]
        (state["k"], state["k_scale"]), (state["v"], state["v_scale"]) = _fill(case, g, C), _fill(case, g, C)
        state["pk"], state["pv"] = ((randn(P, Hk, D) if seq_first else randn(Hk, P, D)) if P else None for _ in range(2))
        order = torch.randperm(B, generator=g, device="cuda")
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32).cuda()[order]
        state["mask"] = None
        if case["mask"]:
            # Each request's new tokens form a tree: a token sees its ancestors and itself.
            parent = (torch.rand((B, T), generator=g, device="cuda") * torch.arange(T, device="cuda")).long()
            sees = torch.eye(T, dtype=torch.bool, device="cuda").repeat(B, 1, 1)
            rows = torch.arange(B, device="cuda")
            for t in range(1, T):
                sees[:, t] |= sees[rows, parent[:, t]]
            at = (state["lengths"].long() - T)[:, None] + torch.arange(T, device="cuda")
            mask = torch.ones((B, 1, T, C), dtype=torch.bool, device="cuda")
            state["mask"] = mask.scatter_(3, at[:, None, None].expand(B, 1, T, T), sees[:, None])
    return state


# ---------------------------------------------------------------------------- plain forms


def _turned(x, cos, sin, pairing):
    """x [..., D] in 32 bits, cos/sin broadcast over its last but one axes."""
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if pairing == "half" else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([a, b], -1) if pairing == "half" else torch.stack([a, b], -1).flatten(-2)


def _angles(s):
    """cos, sin [B, T, D/2], with an axis for the heads where the layout has it; angles in 64 bits."""
    phi = s["positions"].double()[s["axis"]].permute(1, 2, 0) * s["inv_freq"]
    phi = phi.unsqueeze(2 if s["layout"] == "bshd" else 1)
    return phi.cos().float(), phi.sin().float()


def _plain_norm(s):
    cos, sin = _angles(s)

    def both(x, w, dy):
        x, w = x.float(), w.float()
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        n = x * r
        y = _turned(n * w, cos, sin, s["pairing"])
        g = _turned(dy.float(), cos, -sin, s["pairing"])
        dw = (g * n).sum((0, 1, 2))
        g = g * w
        return y, r * (g - n * (g * n).mean(-1, keepdim=True)), dw

    q, dq, dwq = both(s["q"], s["wq"], s["dq"])
    k, dk, dwk = both(s["k"], s["wk"], s["dk"])
    dt, wide = s["q"].dtype, s["wq"].dtype
    return {"q": q.to(dt), "k": k.to(dt), "dq": dq.to(dt), "dk": dk.to(dt), "dwq": dwq.to(wide), "dwk": dwk.to(wide)}


def _plain_append(s):
    cos, sin = _angles(s)

    def normed(x, w):
        x = x.float()
        return x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float() if s["norm"] else x

    q = _turned(normed(s["q"], s["wq"]), cos, sin, s["pairing"]).to(s["q"].dtype)
    k = _turned(normed(s["k"], s["wk"]), cos, sin, s["pairing"])
    found = {"q": q, "lengths": s["lengths"] + s["T"]}
    B, C, T, cache = s["B"], s["C"], s["T"], s["cache"]
    seq = 1 if s["layout"] == "bshd" else 2
    had = s["lengths"].long()
    slots = had[:, None] + torch.arange(T, device="cuda")
    rows = torch.arange(B, device="cuda")[:, None]
    if cache == "same":
        s["k_cache"].transpose(1, seq)[rows, slots] = k.to(q.dtype).transpose(1, seq)
        s["v_cache"].transpose(1, seq)[rows, slots] = s["v"].transpose(1, seq)
        return dict(found, k=s["k_cache"], v=s["v_cache"])

    def store(x, codes, scale):
        x = x.float() if seq == 2 else x.float().transpose(1, 2)  # [B, Hk, T, D]
        blocks = scale.shape[2]
        most = torch.full_like(scale, -1.0)  # the largest magnitude that joins each block
        most.scatter_reduce_(2, (slots // BLOCK)[:, None].expand(-1, x.shape[1], -1), x.abs().amax(-1), "amax")
        start = torch.arange(blocks, device="cuda") * BLOCK
        least = _least_scale(most.clamp(min=0), cache)
        new = torch.where(start < had[:, None, None], torch.maximum(scale, least), least)
        new = torch.where(most >= 0, new, scale)
        before = torch.arange(C, device="cuda") < had[:, None, None]
        factor = torch.where(before, _by_block(scale / new, C), torch.ones((), device="cuda"))
        view = codes if seq == 2 else codes.transpose(1, 2)
        value = view.float() * factor.unsqueeze(-1)
        at = slots[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3])
        value.scatter_(2, at, x / torch.gather(_by_block(new, C), 2, at[..., 0]).unsqueeze(-1))
        view.copy_(_codes(value, cache))
        scale.copy_(new)
        value = view.float() * _by_block(new, C).unsqueeze(-1)
        value = value.masked_fill((torch.arange(C, device="cuda") >= had[:, None, None] + T).unsqueeze(-1), 0.0).to(q.dtype)
        return value if seq == 2 else value.transpose(1, 2)

    return dict(found, k=store(k, s["k_cache"], s["k_scale"]), v=store(s["v"], s["v_cache"], s["v_scale"]))


def _plain_attend(s):
    B, T, Hq, Hk, D, C = s["B"], s["T"], s["Hq"], s["Hk"], s["D"], s["C"]
    heads_first = s["layout"] == "bhsd"
    q = s["q"].float() if heads_first else s["q"].float().transpose(1, 2)
    k, v = ((s[n].float() if heads_first else s[n].float().transpose(1, 2)) * _by_block(s[n + "_scale"], C).unsqueeze(-1) for n in ("k", "v"))
    q = q.reshape(B, Hk, Hq // Hk * T, D) * D ** -0.5  # rows (head of the group, token)
    logits = torch.matmul(q, k.transpose(2, 3)).reshape(B, Hk, Hq // Hk, T, C)
    j = torch.arange(C, device="cuda")
    t = torch.arange(T, device="cuda")
    see = j <= s["lengths"].long()[:, None, None] - T + t[:, None]  # [B, T, C]
    if s["mask"] is not None:
        see = see & s["mask"][:, 0]
    logits = logits.masked_fill(~see[:, None, None], -math.inf).flatten(2, 3)
    m = logits.amax(-1)
    if s["pk"] is not None:
        pk, pv = (s[n].float() if heads_first else s[n].float().transpose(0, 1) for n in ("pk", "pv"))
        shared = torch.matmul(q.transpose(0, 1).reshape(Hk, -1, D), pk.transpose(1, 2)).reshape(Hk, B, -1, pk.shape[1])
        m = torch.maximum(m, shared.amax(-1).transpose(0, 1))
    p = (logits - m.unsqueeze(-1)).exp()
    total, out = p.sum(-1), torch.matmul(p, v)
    if s["pk"] is not None:
        shared = (shared - m.transpose(0, 1).unsqueeze(-1)).exp()
        total = total + shared.sum(-1).transpose(0, 1)
        out = out + torch.matmul(shared.reshape(Hk, -1, pk.shape[1]), pv).reshape(Hk, B, -1, D).transpose(0, 1)
    out = (out / total.unsqueeze(-1)).reshape(B, Hq, T, D).to(s["q"].dtype)
    return {"out": out if heads_first else out.transpose(1, 2)}


PLAIN = {"norm": _plain_norm, "append": _plain_append, "attend": _plain_attend}


def _own(s):
    import tilelang_fa2_4d_mask as api

    op, layout = s["op"], s["layout"]
    if op == "norm":
        q, k = s["rotary"](s["q"], s["k"], s["positions"], query_norm=s["wq"], key_norm=s["wk"], eps=EPS, layout=layout)
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if op == "append":
        norms = dict(query_norm=s["wq"], key_norm=s["wk"], eps=EPS) if s["norm"] else {}
        scales = {} if s["cache"] == "same" else dict(key_scale=s["k_scale"], value_scale=s["v_scale"])
        q, lengths = s["rotary"].append(s["q"], s["k"], s["v"], s["positions"], s["k_cache"], s["v_cache"], s["lengths"], layout=layout, **norms, **scales)
        if s["cache"] == "same":
            return {"q": q, "lengths": lengths, "k": s["k_cache"], "v": s["v_cache"]}
        k, v = (api.cache_values(s[n + "_cache"], s[n + "_scale"], lengths, dtype=q.dtype, layout=layout) for n in ("k", "v"))
        return {"q": q, "lengths": lengths, "k": k, "v": v}
    out = api.shared_prefix_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lengths"], mask=s["mask"], key_scale=s["k_scale"], value_scale=s["v_scale"], layout=layout)
    return {"out": out}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


def work(case):
    op, B, T, D, Hq, Hk = case["op"], case["B"], case["T"], case["D"], case["Hq"], case["Hk"]
    if op == "norm":
        moved, wide = B * T * (Hq + Hk) * D, 4 if case["weight"] == "fp32" else 2
        return {"bytes": 5 * moved * 2 + 8 * len(case["sections"].split(",")) * B * T + 4 * wide * D, "flops": 25 * moved}
    if op == "append":
        n, wide = B * T, 4 if case["weight"] == "fp32" else 2
        size = n * (2 * Hq * D * 2 + 2 * Hk * D * 2 + 8 * len(case["sections"].split(","))) + 8 * B
        size += 2 * wide * D if case["norm"] else 0
        stored = 2 * n * Hk * D
        if case["cache"] == "same":
            return {"bytes": size + 2 * stored, "flops": 10 * n * (Hq + Hk) * D}
        # On average half of what the capacity leaves is held before; all of it is read back.
        live = 2 * B * Hk * (T + (case["C"] - T) / 2)
        return {"bytes": size + stored + live * (D + 4 / BLOCK) + 2 * B * Hk * case["C"] * D * 2, "flops": 10 * n * (Hq + 2 * Hk) * D + live * D}
    P, own_keys = case["P"], sum(_lengths(case))
    size = 2 * 2 * B * T * Hq * D + 2 * 2 * P * Hk * D + 2 * own_keys * Hk * (D + 4 / BLOCK)
    return {"bytes": size + (T * own_keys if case["mask"] else 0), "flops": 4 * D * Hq * T * (B * P + own_keys)}


# ---------------------------------------------------------------------------- 64 bits


def _exact_turn(x, s, sign=1):
    """Each pair as a complex number times e^(i phi)."""
    D, layout = s["D"], s["layout"]
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


def _exact_norm(x, w):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w


def _exact_train(s):
    """The forward from its definition, the gradients by differentiating it in 64 bits."""
    found = {}
    for n in ("q", "k"):
        x, w = (s[i].detach().double().requires_grad_() for i in (n, "w" + n))
        y = _exact_turn(_exact_norm(x, w), s)
        found["d" + n], found["dw" + n] = torch.autograd.grad(y, (x, w), s["d" + n].double())
        found[n] = y.detach()
    return found


def _power(e):
    """2^e for whole e, without the last place's error that exp2 has in 64 bits."""
    return torch.exp2(e.float()).double()


def _to_grid(x, cache):
    """The nearest value of a code, ties to even."""
    if cache == "int8":
        return torch.round(x)
    step = _power(torch.frexp(x.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return torch.round(x / step) * step


def _exact_append(s):
    B, T, C, cache = s["B"], s["T"], s["C"], s["cache"]
    seq = 1 if s["layout"] == "bshd" else 2
    q, k = s["q"].double(), s["k"].double()
    if s["norm"]:
        q, k = _exact_norm(q, s["wq"].double()), _exact_norm(k, s["wk"].double())
    q, k, v = _exact_turn(q, s), _exact_turn(k, s), s["v"].double()
    found = {"q": q, "lengths": s["lengths"] + T}
    for name, x in (("k", k), ("v", v)):
        codes = s[name + "_cache"].to(torch.float64)
        x, codes = (i.transpose(1, 2) if seq == 1 else i for i in (x, codes))
        for b, n in enumerate(s["lengths"].tolist()):
            if cache == "same":
                codes[b, :, n : n + T] = x[b]
                continue
            scale = s[name + "_scale"][b].double()  # [Hk, blocks]
            codes[b, :, n + T :] = 0.0
            for j in range(n // BLOCK, (n + T - 1) // BLOCK + 1):
                held, first, last = slice(j * BLOCK, max(n, j * BLOCK)), max(n, j * BLOCK), min(n + T, (j + 1) * BLOCK)
                fresh = x[b, :, first - n : last - n]
                to = _power(torch.tensor([max(-126, math.frexp(a / MOST[cache])[1] - (math.frexp(a / MOST[cache])[0] == 0.5)) for a in fresh.abs().amax((1, 2)).tolist()], device="cuda"))
                if first > j * BLOCK:
                    to = torch.maximum(to, scale[:, j])
                codes[b, :, held] = _to_grid(codes[b, :, held] * (scale[:, j] / to)[:, None, None], cache)
                codes[b, :, first:last] = _to_grid(fresh / to[:, None, None], cache)
                scale[:, j] = to
            codes[b, :, : n + T] *= _by_block(scale, C)[:, : n + T, None]
        found[name] = codes.transpose(1, 2) if seq == 1 else codes
    return found


def _exact_attend(s):
    """Request by request: softmax over the prefix's and the request's own keys together."""
    B, T, Hq, Hk, D = s["B"], s["T"], s["Hq"], s["Hk"], s["D"]
    bshd, P = s["layout"] == "bshd", s["P"]
    outs = []
    for b, n in enumerate(s["lengths"].tolist()):
        q = (s["q"][b].transpose(0, 1) if bshd else s["q"][b]).double().reshape(Hk, Hq // Hk, T, D)
        k, v = (((s[i][b, :n].transpose(0, 1) if bshd else s[i][b, :, :n]).to(torch.float64)) * _by_block(s[i + "_scale"][b].double(), n).unsqueeze(-1) for i in ("k", "v"))
        if P:
            pk, pv = ((s[i].permute(1, 0, 2) if bshd else s[i]).double() for i in ("pk", "pv"))
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        logits = torch.einsum("hgtd,hjd->hgtj", q, k) / math.sqrt(D)
        late = torch.ones(T, n, dtype=torch.bool, device="cuda").triu(n - T + 1)
        if s["mask"] is not None:
            late |= ~s["mask"][b, 0, :, :n]
        logits[..., P:][late.expand(Hk, Hq // Hk, T, n)] = -math.inf
        out = torch.einsum("hgtj,hjd->hgtd", torch.softmax(logits, -1), v).reshape(Hq, T, D)
        outs.append(out.transpose(0, 1) if bshd else out)
    return {"out": torch.stack(outs)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"norm": _exact_train, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)

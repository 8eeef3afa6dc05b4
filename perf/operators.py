"""Measured cases of the serving operators: the 8-bit paged KV cache (write, read), attention of a
batch over a shared prefix and its own pages, and the verification of drafted tokens.

With ``own`` false ``run`` computes an operator from elementary torch operations in 32 bits; with
``own`` true it makes the calls of ``dotllm_b200.serving`` that a serving loop makes.

Data layout (both forms): a pool of pages of 64 positions, codes ``[n_pages][heads_kv][64][dim]``
(int8 or e4m3) and one fp32 scale per position and head.  ``pages[b]`` lists sequence b's pages,
``seq_len[b]`` its positions, and rows ``row_start[b] .. row_start[b + 1]`` of a call are the last
positions of sequence b.
"""
import torch

own = False

PAGE = 64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TOP = {"i8": 127.0, "e4m3": 448.0}  # the largest magnitude a code stands for


def listed():
    return [
        # the K/V rows of one decode step of a few sessions (1B shape: 8 kv heads of 64): latency
        {"name": "write step", "op": "write", "fmt": "i8", "type": "f32", "heads_kv": 8, "dim": 64,
         "batch": 8, "rows": 1, "ragged": 0, "len_lo": 1, "len_hi": 600},
        # the K/V of a long prompt (8B shape)
        {"name": "write prompt", "op": "write", "fmt": "e4m3", "type": "bf16", "heads_kv": 8, "dim": 128,
         "batch": 2, "rows": 8191, "ragged": 1, "len_lo": 8191, "len_hi": 8192},
        # the last positions of a few sessions, read back (Phi-3-mini heads: 32 of 96)
        {"name": "read tails", "op": "read", "fmt": "e4m3", "type": "f16", "heads_kv": 32, "dim": 96,
         "batch": 5, "rows": 97, "ragged": 1, "len_lo": 130, "len_hi": 1100},
        # a whole long cache handed to a consumer of fp32 rows
        {"name": "read cache", "op": "read", "fmt": "i8", "type": "f32", "heads_kv": 8, "dim": 128,
         "batch": 4, "rows": 4000, "ragged": 1, "len_lo": 4000, "len_hi": 4096},
        # one session behind a system prompt (1B shape): latency
        {"name": "attend one", "op": "attend", "fmt": "i8", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 64,
         "batch": 1, "rows": 1, "ragged": 0, "prefix": 512, "len_lo": 70, "len_hi": 70, "window": 0, "cap": 0.0, "lse": 0},
        # an ordinary decode step: 32 sessions, one token each, behind one prompt (8B shape)
        {"name": "attend step", "op": "attend", "fmt": "i8", "type": "bf16", "heads": 32, "heads_kv": 8, "dim": 128,
         "batch": 32, "rows": 1, "ragged": 0, "prefix": 2048, "len_lo": 33, "len_hi": 1500, "window": 0, "cap": 0.0, "lse": 0},
        # drafted tokens of 16 sessions, no head sharing (Phi-3-mini heads)
        {"name": "attend drafts", "op": "attend", "fmt": "e4m3", "type": "f16", "heads": 32, "heads_kv": 32, "dim": 96,
         "batch": 16, "rows": 5, "ragged": 1, "prefix": 1021, "len_lo": 6, "len_hi": 700, "window": 0, "cap": 0.0, "lse": 1},
        # sliding window, capped scores, wide heads, fp32 activations (Gemma-2-2B heads)
        {"name": "attend window", "op": "attend", "fmt": "i8", "type": "f32", "heads": 8, "heads_kv": 4, "dim": 256,
         "batch": 4, "rows": 4, "ragged": 1, "prefix": 6144, "len_lo": 100, "len_hi": 999, "window": 4096, "cap": 50.0, "lse": 1},
        # many sessions with drafts behind a long shared context (8B shape): the largest
        {"name": "attend many", "op": "attend", "fmt": "i8", "type": "bf16", "heads": 32, "heads_kv": 8, "dim": 128,
         "batch": 96, "rows": 5, "ragged": 1, "prefix": 8192, "len_lo": 64, "len_hi": 2048, "window": 0, "cap": 0.0, "lse": 0},
        # one session's drafts over a 32000-token vocabulary: latency
        {"name": "verify one", "op": "verify", "batch": 1, "drafts": 4, "vocab": 32000, "ragged": 0, "probs": 1},
        # an ordinary speculative step; the odd vocabulary leaves rows unaligned
        {"name": "verify step", "op": "verify", "batch": 24, "drafts": 5, "vocab": 128255, "ragged": 1, "probs": 1},
        # many sessions, the widest vocabulary
        {"name": "verify many", "op": "verify", "batch": 96, "drafts": 7, "vocab": 256000, "ragged": 1, "probs": 1},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(["write", "read", "attend", "attend", "attend", "verify", "verify"])
    if op == "verify":
        vocab = rng.choice([log(1000, 256000), 32000, 32064, 50257, 128256, 256000])
        return {"op": op, "batch": log(1, 96), "drafts": rng.randint(1, 7), "vocab": vocab, "ragged": rng.randint(0, 1),
                "probs": rng.choice([1, 1, 1, 0])}
    case = {"op": op, "fmt": rng.choice(["i8", "e4m3"]), "type": rng.choice(["f32", "f16", "bf16"])}
    case["dim"] = rng.choice([64, 96, 128, 256])
    if op in ("write", "read"):
        case["heads_kv"] = rng.choice([1, 2, 4, 8, 32])
        most = 16384 * 8 * 128 // (case["heads_kv"] * case["dim"])
        case["batch"] = log(1, 64)
        case["rows"] = log(1, max(1, min(8192, most // case["batch"])))
        case["ragged"] = rng.randint(0, 1)
        case["len_lo"] = case["rows"] + rng.randint(0, 100)
        case["len_hi"] = case["len_lo"] + rng.randint(0, 500)
        return case
    case["heads_kv"] = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 2, 4, 8])
    if rng.random() < 0.2:
        case["heads_kv"], group = 32, 1
    case["heads"] = case["heads_kv"] * group
    case["batch"] = log(1, 96)
    case["rows"] = rng.choice([1, 1, rng.randint(2, 8)])
    case["ragged"] = rng.randint(0, 1)
    case["prefix"] = rng.choice([0, log(16, 8192), log(16, 8192)])
    case["len_lo"] = rng.randint(1, 64)
    case["len_hi"] = case["len_lo"] + log(1, 2048)
    # no more key/value values, nor more products, than the largest listed case has
    while (case["prefix"] + case["batch"] * case["len_hi"]) * case["heads_kv"] * case["dim"] > 150e6 or \
            case["batch"] * case["rows"] * case["heads"] * (case["prefix"] + case["len_hi"]) * case["dim"] > 15e9:
        case["batch"] = max(1, case["batch"] // 2)
        case["len_hi"] = max(case["len_lo"], case["len_hi"] * 3 // 4)
    case["window"] = rng.choice([0, 0, log(64, 8192)])
    case["cap"] = rng.choice([0.0, 0.0, 50.0])
    case["lse"] = rng.randint(0, 1)
    return case


def lengths(case):
    """Rows and positions of each sequence: fixed by the case, spread over its range in a mixed order."""
    B = case["batch"]
    at = [(i * 37) % B for i in range(B)] if B % 37 else list(range(B))
    span = case["len_hi"] - case["len_lo"]
    lens = [case["len_lo"] + at[i] * span // max(1, B - 1) for i in range(B)]
    rows = [max(1, case["rows"] - (i % 3 if case["ragged"] else 0)) for i in range(B)]
    return rows, lens


def quantise(x, fmt):
    """(codes, scales) of the rows of x (last axis)."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(top) & (top >= 1e-30)
    y = torch.where(ok, x * (TOP[fmt] / top), 0.0)
    scale = torch.where(ok, top / TOP[fmt], torch.where(top < 1e-30, 0.0, float("nan"))).squeeze(-1)
    if fmt == "i8":
        return torch.round(y).clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def generator(seed, n=0):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + n)


def prepare(case, seed):
    return prepare_verify(case, seed) if case["op"] == "verify" else prepare_cache(case, seed)


def prepare_verify(case, seed):
    B, k, V = case["batch"], case["drafts"], case["vocab"]
    g = generator(seed)
    # the target's probabilities, and a draft model's that mostly agrees with it
    x = torch.randn(B, k + 1, V, device="cuda", generator=g).mul_(3.0)
    y = torch.randn(B, k, V, device="cuda", generator=g).mul_(1.2).add_(x[:, :k], alpha=0.9)
    p, q = torch.softmax(x, -1), torch.softmax(y, -1)
    del x
    noise = torch.rand(B, k, V, device="cuda", generator=g).clamp_min_(1e-12)
    drafts = (y - noise.log_().neg_().log_()).argmax(-1).to(torch.int32)  # sampled from q
    n = [max(0, k - i % 3) if case["ragged"] else k for i in range(B)]
    return {"case": case, "p": p, "q": q if case["probs"] else None, "drafts": drafts,
            "u": torch.rand(B, k + 1, device="cuda", generator=g),
            "n_draft": torch.tensor(n, dtype=torch.int32, device="cuda")}


def prepare_cache(case, seed):
    g = generator(seed)
    rows, lens = lengths(case)
    B, Hk, D, P = case["batch"], case["heads_kv"], case["dim"], case.get("prefix", 0)
    need = [-(-n // PAGE) for n in lens]
    prefix_pages, most = -(-P // PAGE), max(need)
    n_pages = sum(need) + prefix_pages + 3  # a pool is not exactly full
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    ends = torch.tensor(need).cumsum(0)
    slot = torch.arange(most)[None] + (ends - torch.tensor(need))[:, None]
    valid = torch.arange(most)[None] < torch.tensor(need)[:, None]
    pages = torch.where(valid.cuda(), order[slot.clamp(max=n_pages - 1).cuda()], 0).to(torch.int32).contiguous()
    state = {"case": case, "pages": pages, "max_rows": max(rows),
             "prefix_pages": order[int(ends[-1]):int(ends[-1]) + prefix_pages].contiguous(),
             "row_start": torch.tensor([0] + rows).cumsum(0).to(torch.int32).cuda(),
             "seq_len": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    R = sum(rows)

    def filled(n):
        k = torch.randn(n_pages, Hk, PAGE, D, device="cuda", generator=generator(seed, n))
        # K has a few wide channels, as keys after rotary positions have
        return quantise(k * (1.0 + 2.0 * (torch.arange(D, device="cuda") % 32 == 5)) if n == 1 else k, case["fmt"])

    (state["k"], state["k_scale"]), (state["v"], state["v_scale"]) = filled(1), filled(2)
    t = TYPES[case["type"]]
    if case["op"] == "write":
        # K and V are slices of one projection's output, as a fused QKV product leaves them
        kv = torch.randn(R, 2, Hk, D, device="cuda", generator=g).to(t)
        state["new_k"], state["new_v"] = kv[:, 0], kv[:, 1]
    if case["op"] == "attend":
        state["q"] = torch.randn(R, case["heads"], D, device="cuda", generator=g).to(t)
    return state


def run(state):
    if own:
        return run_own(state)
    return {"write": plain_write, "read": plain_read, "attend": plain_attend, "verify": plain_verify}[state["case"]["op"]](state)


def run_own(s):
    from dotllm_b200 import serving

    case = s["case"]
    if case["op"] == "verify":
        tokens, accepted = serving.verify_draft(s["p"], s["q"], s["drafts"], s["u"], s["n_draft"])
        return {"tokens": tokens, "accepted": accepted}
    pool = serving.KvqPool(s["k"], s["v"], s["k_scale"], s["v_scale"])
    batch = serving.KvqBatch(s["row_start"], s["seq_len"], s["pages"], s["max_rows"])
    if case["op"] == "write":
        serving.kvq_write(pool, batch, s["new_k"], s["new_v"])
        return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if case["op"] == "read":
        k, v = serving.kvq_read(pool, batch, sum(lengths(case)[0]), TYPES[case["type"]])
        return {"k": k, "v": v}
    got = serving.kvq_attention(pool, batch, s["q"], prefix_pages=s["prefix_pages"], prefix_len=case["prefix"],
                                softcap=case["cap"], window=case["window"], return_lse=bool(case["lse"]))
    return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}


# ---------------------------------------------------------------- plain forms
def row_places(s, n_rows):
    """For each row: its sequence, its position, and the pool page and slot of that position."""
    r = torch.arange(n_rows, device="cuda")
    b = torch.searchsorted(s["row_start"][1:].long(), r, right=True)
    pos = s["seq_len"].long()[b] - s["row_start"].long()[b + 1] + r
    page = s["pages"].long()[b, pos.clamp(min=0) // PAGE]
    return b, pos, page, pos % PAGE


def plain_write(s):
    case = s["case"]
    _, _, page, at = row_places(s, s["new_k"].shape[0])
    for codes, scales, x in (("k", "k_scale", "new_k"), ("v", "v_scale", "new_v")):
        c, sc = quantise(s[x], case["fmt"])
        s[codes].view(torch.int8)[page, :, at] = c.view(torch.int8)
        s[scales][page, :, at] = sc
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def plain_read(s):
    case = s["case"]
    _, _, page, at = row_places(s, sum(lengths(case)[0]))
    t = TYPES[case["type"]]

    def back(codes, scales):
        c = s[codes].view(torch.int8)[page, :, at].view(s[codes].dtype)
        return (c.float() * s[scales][page, :, at][..., None]).to(t)

    return {"k": back("k", "k_scale"), "v": back("v", "v_scale")}


def plain_attend(s):
    case = s["case"]
    q, Hk, D, P = s["q"], case["heads_kv"], case["dim"], case["prefix"]
    R, H = q.shape[0], q.shape[1]
    G, B = H // Hk, s["seq_len"].shape[0]
    n_max, neg = s["max_rows"], float("-inf")

    def values(codes, scales, pages):  # [..., positions, Hk, D] in 32 bits
        c = s[codes].view(torch.int8)[pages].view(s[codes].dtype).float() * s[scales][pages][..., None]
        return c.transpose(-3, -2).flatten(-4, -3)

    b, pos, _, _ = row_places(s, R)
    i = torch.arange(R, device="cuda") - s["row_start"].long()[b]
    seen = P + pos  # a row sees the positions up to its own
    first = seen - case["window"] + 1 if case["window"] else torch.zeros_like(seen)
    qf = q.float().view(R, Hk, G, D)

    def capped(x):
        x = x * D ** -0.5
        return case["cap"] * torch.tanh(x / case["cap"]) if case["cap"] else x

    # the shared prefix, every row at once
    pp = s["prefix_pages"].long()
    kp, vp = values("k", "k_scale", pp)[:P], values("v", "v_scale", pp)[:P]
    j = torch.arange(P, device="cuda")
    sp = capped(torch.einsum("rhgd,jhd->rhgj", qf, kp))
    sp = sp.masked_fill(((j[None] > seen[:, None]) | (j[None] < first[:, None]))[:, None, None], neg)
    # each sequence's own positions
    ks, vs = values("k", "k_scale", s["pages"].long()), values("v", "v_scale", s["pages"].long())
    S = ks.shape[1]
    qs = torch.zeros(B, n_max, Hk, G, D, device="cuda")
    qs[b, i] = qf
    j = P + torch.arange(S, device="cuda")
    ss = capped(torch.einsum("bnhgd,bjhd->bnhgj", qs, ks))[b, i]
    ss = ss.masked_fill(((j[None] > seen[:, None]) | (j[None] < first[:, None]))[:, None, None], neg)
    m = torch.cat([sp, ss], -1).amax(-1, keepdim=True)
    m0 = torch.where(m == neg, 0.0, m)
    ep, es = torch.exp(sp - m0), torch.exp(ss - m0)
    total = ep.sum(-1, keepdim=True) + es.sum(-1, keepdim=True)
    ws = torch.zeros(B, n_max, Hk, G, S, device="cuda")
    ws[b, i] = es
    out = torch.einsum("rhgj,jhd->rhgd", ep, vp) + torch.einsum("bnhgj,bjhd->bnhgd", ws, vs)[b, i]
    out = torch.where(total > 0, out / total, 0.0).view(R, H, D).to(q.dtype)
    if not case["lse"]:
        return {"out": out}
    return {"out": out, "lse": (m0 + torch.log(total)).view(R, H)}


def plain_verify(s):
    p, q, x, u, n = s["p"], s["q"], s["drafts"].long(), s["u"], s["n_draft"].long()
    B, k, V = p.shape[0], p.shape[1] - 1, p.shape[2]
    inside = (x >= 0) & (x < V)
    at = x.clamp(0, V - 1)[..., None]
    px = p[:, :k].gather(2, at)[..., 0]
    qx = q.gather(2, at)[..., 0] if q is not None else torch.ones_like(px)
    ok = (u[:, :k] * qx < px) & inside & (torch.arange(k, device="cuda")[None] < n[:, None])
    acc = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device="cuda")
    row, last = p[b, acc], acc.clamp(max=k - 1)
    if q is not None:
        less = q[b, last]
    else:
        less = torch.zeros_like(row).scatter_(1, at[b, last], inside[b, last].float()[:, None])
    rest = torch.where((acc < n)[:, None], row - less, row)
    rest = torch.clamp(torch.nan_to_num(rest, 0.0, 1.0, 0.0), 0.0, 1.0)
    w = (rest * 2.0 ** 40).long()
    plain = (torch.clamp(torch.nan_to_num(row, 0.0, 1.0, 0.0), 0.0, 1.0) * 2.0 ** 40).long()
    w = torch.where(w.sum(1, keepdim=True) > 0, w, plain)
    total = w.sum(1)
    m = (u[:, k] * 2.0 ** 24).long()
    t = (total >> 24) * m + (((total & 0xFFFFFF) * m) >> 24)
    pick = torch.where(total > 0, (w.cumsum(1) <= t[:, None]).sum(1), 0)
    j = torch.arange(k + 1, device="cuda")[None]
    tokens = torch.where(j < acc[:, None], torch.nn.functional.pad(x, (0, 1)), -1)
    tokens = torch.where(j == acc[:, None], pick[:, None], tokens)
    return {"tokens": tokens.to(torch.int32), "accepted": acc.to(torch.int32)}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    """Sequence by sequence and position by position from the formulas; whole numbers have no such value."""
    if case["op"] == "verify":
        return None
    s = prepare(case, seed)
    rows, lens = lengths(case)
    Hk, D, P = case["heads_kv"], case["dim"], case.get("prefix", 0)
    pages = s["pages"].tolist()

    def held(codes, scales, list_of_pages, n):  # [n][Hk][D]
        at = torch.tensor(list_of_pages, dtype=torch.long, device="cuda")
        c = s[codes].view(torch.int8)[at].view(s[codes].dtype).double() * s[scales][at].double()[..., None]
        return c.permute(0, 2, 1, 3).reshape(-1, Hk, D)[:n]

    if case["op"] == "write":
        out = {"k": None, "v": None}
        for scales, x in (("k_scale", "new_k"), ("v_scale", "new_v")):
            got, r = s[scales].double(), 0
            for b in range(case["batch"]):
                pos = torch.arange(lens[b] - rows[b], lens[b], device="cuda")
                page = s["pages"][b].long()[pos // PAGE]
                got[page, :, pos % PAGE] = s[x][r:r + rows[b]].double().abs().amax(-1) / TOP[case["fmt"]]
                r += rows[b]
            out[scales] = got
        return out
    if case["op"] == "read":
        out = {}
        for name, scales in (("k", "k_scale"), ("v", "v_scale")):
            out[name] = torch.cat([held(name, scales, pages[b], lens[b])[lens[b] - rows[b]:] for b in range(case["batch"])])
        return out
    G = case["heads"] // Hk
    shared = [held(c, sc, s["prefix_pages"].tolist(), P) for c, sc in (("k", "k_scale"), ("v", "v_scale"))]
    outs, lses, r = [], [], 0
    for b in range(case["batch"]):
        k = torch.cat([shared[0], held("k", "k_scale", pages[b], lens[b])]).permute(1, 0, 2)
        v = torch.cat([shared[1], held("v", "v_scale", pages[b], lens[b])]).permute(1, 0, 2)
        n, T = rows[b], P + lens[b]
        q = s["q"][r:r + n].double().view(n, Hk, G, D).permute(1, 0, 2, 3).reshape(Hk, n * G, D)
        x = q @ k.transpose(1, 2) / D ** 0.5
        if case["cap"]:
            x = case["cap"] * torch.tanh(x / case["cap"])
        p = T - n + torch.arange(n, device="cuda").repeat_interleave(G)[:, None]
        j = torch.arange(T, device="cuda")[None]
        x = x.masked_fill((j > p) | (j <= p - (case["window"] or T + n)), float("-inf"))
        lse = torch.logsumexp(x, -1)
        o = torch.exp(x - torch.where(torch.isinf(lse), 0.0, lse)[..., None]) @ v
        outs.append(o.view(Hk, n, G, D).permute(1, 0, 2, 3).reshape(n, Hk * G, D))
        lses.append(lse.view(Hk, n, G).permute(1, 0, 2).reshape(n, Hk * G))
        r += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)} if case["lse"] else {"out": torch.cat(outs)}


def work(case):
    if case["op"] == "verify":
        # one row of p; one of q too where a draft is refused (about three in four sequences)
        return {"bytes": case["batch"] * case["vocab"] * 4 * (1.75 if case["probs"] else 1.0), "flops": 0}
    rows, lens = lengths(case)
    R, Hk, D = sum(rows), case["heads_kv"], case["dim"]
    if case["op"] != "attend":
        return {"bytes": R * Hk * 2 * (D * SIZE[case["type"]] + D + 4), "flops": 0}
    P, win = case["prefix"], case["window"]
    seen, own_first, shared_first = 0, [], P
    for n, length in zip(rows, lens):
        first = P + length - n  # the first row's position; rows before position 0 see nothing
        own_first.append(max(0, first - win + 1 - P) if win else 0)
        shared_first = min(shared_first, max(0, first - win + 1) if win else 0)
        for i in range(n):
            seen += max(0, min(first + i + 1, win) if win else first + i + 1)
    held = P - shared_first + sum(max(0, length - f) for length, f in zip(lens, own_first))
    return {"bytes": held * Hk * 2 * (D + 4) + R * case["heads"] * D * 2 * SIZE[case["type"]],
            "flops": 4 * D * case["heads"] * seen}

"""The serving operators: cases, plain forms and their definition in 64 bits.

A case is a dict of plain values; ``kind`` names the operator:

  append     per-head norm + rotation of a ragged batch's new tokens, K and V into the paged cache
  attention  attention of a ragged batch's new tokens over the paged cache
  logprobs   log probabilities of given tokens with entropy, rank and top alternatives

Ragged batches are drawn from the seed between the case's bounds: sequence s has ``qlo..qhi`` new
tokens over ``clo..chi`` cached ones.  Pages are handed out in a random order, as a running server's are,
and every table ends in entries that name no page.  Head counts are those of the Bonsai 1.7B / 4B / 8B
layers of this repository and of its tiny decoder, plus ungrouped heads.
"""
import math
import random

import numpy as np
import torch

own = False

NO_PAGE = 0xFFFFFFFF
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
THETA, EPS = 1.0e6, 1e-6
_dev = None


def listed():
    return [
        # one token of one chat on the 1.7B layer: the append of a decode step on its own (bound by the call)
        dict(name="append_one", kind="append", seqs=1, qlo=1, qhi=1, clo=700, chi=700, hq=16, hkv=8, d=128, page=16,
             type="f16", norm=True, halves=False, pad=0),
        # a decode step of 256 running sequences on the 8B layer, some of them far into long documents
        dict(name="append_decode_256", kind="append", seqs=256, qlo=1, qhi=1, clo=0, chi=131000, hq=32, hkv=8, d=128,
             page=16, type="bf16", norm=True, halves=True, pad=0),
        # prompts of odd lengths that enter together, in a buffer that is padded behind them
        dict(name="append_prompts", kind="append", seqs=7, qlo=150, qhi=1100, clo=0, chi=900, hq=32, hkv=8, d=128,
             page=64, type="f16", norm=True, halves=False, pad=61),
        # one token over the benchmark's 512-token prompt (bound by the call and one round to memory)
        dict(name="decode_one_513", kind="attention", seqs=1, qlo=1, qhi=1, clo=512, chi=512, hq=16, hkv=8, d=128,
             page=16, type="f16", cap=0.0, window=0, bias=False, prefix=0, pad=0),
        # one token over a very long document: the split of one sequence over the chip
        dict(name="decode_one_131k", kind="attention", seqs=1, qlo=1, qhi=1, clo=131071, chi=131071, hq=32, hkv=8,
             d=128, page=64, type="bf16", cap=0.0, window=0, bias=False, prefix=0, pad=0),
        # a decode step of 64 chats of all lengths on the 8B layer
        dict(name="decode_64_chats", kind="attention", seqs=64, qlo=1, qhi=1, clo=3, chi=8191, hq=32, hkv=8, d=128,
             page=16, type="f16", cap=0.0, window=0, bias=False, prefix=0, pad=0),
        # a chunk of a long prompt over what the chunks before it left in the cache (1.7B heads)
        dict(name="chunk_2048_on_8k", kind="attention", seqs=1, qlo=2048, qhi=2048, clo=8192, chi=8192, hq=16, hkv=8,
             d=128, page=16, type="f16", cap=0.0, window=0, bias=False, prefix=0, pad=0),
        # prompts' chunks with running chats between them, capped scores within a sliding window
        dict(name="mixed_capped_window", kind="attention", seqs=24, qlo=1, qhi=700, clo=1, chi=1500, hq=16, hkv=4, d=64,
             page=32, type="bf16", cap=30.0, window=512, bias=False, prefix=0, pad=13),
        # whole prompts with a prefix that all of their tokens see, ungrouped heads, distance bias
        dict(name="prefix_biased", kind="attention", seqs=5, qlo=200, qhi=1300, clo=0, chi=0, hq=16, hkv=16, d=64,
             page=16, type="f16", cap=0.0, window=0, bias=True, prefix=100, pad=0),
        # the token that a decode step drew, with its 20 best alternatives (vocabulary of the Bonsai presets)
        dict(name="logprobs_one", kind="logprobs", rows=1, vocab=151669, type="f32", top=20, temperature=1.0, pad=0),
        # a long prompt's chunk scored against a 151936-word vocabulary
        dict(name="logprobs_2048", kind="logprobs", rows=2048, vocab=151936, type="f32", top=5, temperature=1.0, pad=0),
        # odd vocabulary in padded rows of 16-bit logits, at a chat's temperature
        dict(name="logprobs_333_bf16", kind="logprobs", rows=333, vocab=50257, type="bf16", top=8, temperature=0.7,
             pad=47),
    ]


def draw(rng):
    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "append", "attention", "attention", "attention", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = logint(100, 160000)
        return dict(kind=kind, rows=logint(1, max(1, min(4096, 300_000_000 // vocab))), vocab=vocab,
                    type=rng.choice(["f32", "f16", "bf16"]), top=rng.choice([0, 1, 5, 20, 64]),
                    temperature=rng.choice([1.0, 0.6, 1.7]), pad=rng.choice([0, 0, 5, 64]))
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([2, 4, 8, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 8] if hkv < 8 else [1, 2, 4])
    c = dict(kind=kind, hq=hq, hkv=hkv, d=d, page=rng.choice([16, 16, 32, 64, 128]), type=rng.choice(["f16", "bf16"]),
             pad=rng.choice([0, 0, 7]))
    if kind == "append":
        seqs = logint(1, 300)
        qhi = logint(1, max(1, min(4096, 8192 // seqs)))
        chi = rng.choice([0, logint(1, 2000), logint(1000, 131000)])
        return dict(c, seqs=seqs, qlo=rng.choice([0, 1, qhi]) if seqs > 1 else qhi, qhi=qhi, clo=chi // 3, chi=chi,
                    norm=rng.random() < 0.7, halves=rng.random() < 0.5)
    shape = rng.choice(["decode", "few", "prompts", "mixed"])
    if shape == "decode":
        seqs = logint(1, 128)
        chi = logint(8, min(100000, 500_000 // seqs))
        q = (1, 1)
    elif shape == "few":     # drafts that are checked together
        seqs = logint(1, 64)
        chi = logint(8, min(32000, 300_000 // seqs))
        q = (2, rng.randint(2, 9))
    elif shape == "prompts":
        seqs = logint(1, 8)
        qhi = logint(16, 1500 // seqs + 16)
        chi = rng.choice([0, logint(1, 4000)])
        q = (max(1, qhi // 3), qhi)
    else:
        seqs = rng.randint(3, 20)
        chi = logint(16, 2000)
        q = (1, logint(8, 600))
    c.update(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), window=rng.choice([0, 0, 0, 64, 1000]), bias=rng.random() < 0.25,
             prefix=rng.choice([0, 0, 0, 33]))
    return dict(c, seqs=seqs, qlo=q[0], qhi=q[1], clo=max(chi // 8, 0), chi=chi)


def _batch(case):
    """Lengths of the case's ragged batch: new tokens and cached tokens of each sequence.  They belong to the
    case, not to the seed, so that every seed asks for the same work."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = [r.randint(case["qlo"], case["qhi"]) for _ in range(case["seqs"])]
    if case["qlo"] != case["qhi"] and case["seqs"] > 1:
        n[0], n[-1] = case["qhi"], case["qlo"]
    if case["kind"] == "attention" and case["qlo"] == 1 and case["qhi"] > 64:   # chats between the chunks
        n = [x if i % 4 == 0 else 1 for i, x in enumerate(n)]
    ctx = [r.randint(case["clo"], case["chi"]) for _ in range(case["seqs"])]
    return n, [a + b for a, b in zip(n, ctx)]


def _pages(case, n, lens, g):
    """A page table with the pages in random order.  The append needs only the pages that it writes."""
    P = case["page"]
    width = max(1, max((l + P - 1) // P for l in lens) + 1)
    table = np.full((len(lens), width), NO_PAGE, dtype=np.uint32)
    first = [(l - m) // P if case["kind"] == "append" else 0 for m, l in zip(n, lens)]
    used = [max(0, (l + P - 1) // P - f) for l, f in zip(lens, first)]
    total = max(1, sum(used)) + 3
    order = np.random.default_rng(g).permutation(total).astype(np.uint32)
    at = 0
    for s, (f, u) in enumerate(zip(first, used)):
        table[s, f:f + u] = order[at:at + u]
        at += u
    return table, total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]
    if case["kind"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        buf = torch.empty(R, V + case["pad"], dtype=dt, device="cuda")
        # logits of a trained head: a bulk of width 2.5 and a few ids that stand out
        buf.copy_(torch.randn(R, V + case["pad"], generator=g, device="cuda").mul_(2.5))
        hot = torch.randint(0, V, (R, 12), generator=g, device="cuda")
        up = torch.rand(R, 12, generator=g, device="cuda") * 12 + 6
        buf.scatter_(1, hot, up.to(dt))
        tokens = torch.where(torch.rand(R, generator=g, device="cuda") < 0.7, hot[:, 0],
                             torch.randint(0, V, (R,), generator=g, device="cuda")).to(torch.int32)
        new = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        return dict(case=case, logits=buf[:, :V], tokens=tokens, lp=new(R), lse=new(R), entropy=new(R),
                    rank=new(R, t=torch.int32), top_ids=new(R, case["top"], t=torch.int32),
                    top_lp=new(R, case["top"]), ready={})
    n, lens = _batch(case)
    hq, hkv, d, P = case["hq"], case["hkv"], case["d"], case["page"]
    table, total = _pages(case, n, lens, seed)
    T = sum(n) + case["pad"]
    starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    st = dict(case=case, n=n, lens=lens, T=T, rows=sum(n), max_q=max(n), max_kv=max(lens), pages=total, ready={},
              starts=torch.from_numpy(starts).cuda(), kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              table=torch.from_numpy(table.view(np.int32)).cuda())

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    if case["kind"] == "append":
        qkv = normal(T, (hq + 2 * hkv) * d)     # one row per token, as the projections of a token lie together
        st["q"] = qkv[:, :hq * d].view(T, hq, d)
        st["k"] = qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d)
        st["v"] = qkv[:, (hq + hkv) * d:].view(T, hkv, d)
        st["q_out"] = torch.zeros(T, hq, d, dtype=dt, device="cuda")
        st["k_pages"] = torch.zeros(total, hkv, P, d, dtype=dt, device="cuda")
        st["v_pages"] = torch.zeros(total, hkv, d, P, dtype=dt, device="cuda")
        if case["norm"]:
            st["q_scale"] = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
            st["k_scale"] = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
        else:
            st["q_scale"] = st["k_scale"] = None
        # where each row's token stands, for the plain form
        seq = np.repeat(np.arange(len(n)), n)
        pos = np.concatenate([np.arange(l - m, l) for m, l in zip(n, lens)]) if sum(n) else np.zeros(0, np.int64)
        st["pos"] = torch.from_numpy(pos).cuda()
        st["page_of"] = torch.from_numpy(table[seq, pos // P].astype(np.int64)).cuda()
    else:
        st["q"] = normal(T, hq, d)
        st["k_pages"] = normal(total, hkv, P, d)
        st["v_pages"] = normal(total, hkv, d, P)
        st["out"] = torch.zeros(T, hq, d, dtype=dt, device="cuda")
        st["lse"] = torch.zeros(T, hq, device="cuda")
        st["slopes"] = (2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq)).float() if case["bias"] else None
        st["prefix"] = (torch.tensor([min(case["prefix"], l) for l in lens], dtype=torch.int32, device="cuda")
                        if case["prefix"] else None)
        seq = np.repeat(np.arange(len(n)), n)
        off = np.concatenate([np.arange(m) for m in n]) if sum(n) else np.zeros(0, np.int64)
        st["seq"], st["off"] = torch.from_numpy(seq).cuda(), torch.from_numpy(off).cuda()
    return st


# ------------------------------------------------------------------ the framework's calls
def _device():
    """The context that every case runs on (a program keeps one per GPU)."""
    global _dev
    if _dev is None:
        from nnzap_amd import ops
        _dev = ops.Device(0)
    return _dev


def _plan(st):
    """The cache and batch objects and the workspace that a serving program keeps."""
    r = st["ready"]
    if not r:
        from nnzap_amd import ops
        dev = r["dev"] = _device()
        c = st["case"]
        if c["kind"] == "logprobs":
            n = ops.token_logprobs_workspace_bytes(c["rows"], c["vocab"], c["top"])
            r["ws"] = torch.empty(max(1, n), dtype=torch.uint8, device="cuda")
        else:
            r["kv"] = ops.PagedKVCache(dev, st["k_pages"], st["v_pages"])
            r["batch"] = ops.PagedBatch(st["table"], st["starts"], st["kv_lens"], st["T"], st["max_q"], st["max_kv"])
            if c["kind"] == "attention":
                n = ops.paged_attention_workspace_bytes(r["kv"], r["batch"], c["hq"])
                r["ws"] = torch.empty(max(1, n), dtype=torch.uint8, device="cuda")
    return r


def _run_own(st):
    from nnzap_amd import ops
    c, r = st["case"], _plan(st)
    if c["kind"] == "logprobs":
        ops.dispatch_token_logprobs(r["dev"], st["logits"], st["tokens"], st["lp"], r["ws"], lse=st["lse"],
                                    entropy=st["entropy"], rank=st["rank"],
                                    top_ids=st["top_ids"] if c["top"] else None,
                                    top_logprobs=st["top_lp"] if c["top"] else None, temperature=c["temperature"])
        return [st["lp"], st["lse"], st["entropy"], st["rank"], st["top_ids"], st["top_lp"]]
    if c["kind"] == "append":
        ops.dispatch_paged_append(r["dev"], r["kv"], r["batch"], st["q"], st["k"], st["v"], st["q_out"],
                                  q_scale=st["q_scale"], k_scale=st["k_scale"], eps=EPS, theta=THETA,
                                  halves=c["halves"])
        return [st["q_out"], st["k_pages"], st["v_pages"]]
    ops.dispatch_paged_attention(r["dev"], r["kv"], r["batch"], st["q"], st["out"], r["ws"], lse=st["lse"],
                                 softcap=c["cap"], window=c["window"], slopes=st["slopes"], prefix_lens=st["prefix"])
    return [st["out"], st["lse"]]


# ------------------------------------------------------------------ plain forms
def _append_plain(st):
    c = st["case"]
    n, d, P = st["rows"], c["d"], c["page"]
    ang = st["pos"].double()[:, None] * THETA ** (-torch.arange(0, d, 2, device="cuda").double() / d)
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def turn(x, w):
        x = x[:n].float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        if c["halves"]:
            a, b = x[..., :d // 2], x[..., d // 2:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

    slot = st["pos"] % P
    st["q_out"][:n] = turn(st["q"], st["q_scale"]).to(st["q_out"].dtype)
    st["k_pages"][st["page_of"], :, slot] = turn(st["k"], st["k_scale"]).to(st["k_pages"].dtype)
    st["v_pages"][st["page_of"], :, :, slot] = st["v"][:n]
    return [st["q_out"], st["k_pages"], st["v_pages"]]


def _attention_plain(st):
    c = st["case"]
    B, hq, hkv, d, P = c["seqs"], c["hq"], c["hkv"], c["d"], c["page"]
    G, mq, W = hq // hkv, st["max_q"], st["table"].shape[1]
    S = W * P
    page = st["table"].long().clamp(0, st["pages"] - 1)
    k = st["k_pages"][page].float().permute(0, 2, 1, 3, 4).reshape(B, hkv, S, d)
    v = st["v_pages"][page].float().permute(0, 2, 1, 4, 3).reshape(B, hkv, S, d)
    q = torch.zeros(B, mq, hq, d, device="cuda")
    q[st["seq"], st["off"]] = st["q"][:st["rows"]].float()
    q = q.view(B, mq, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * mq, d)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(d)).view(B, hkv, G, mq, S)
    if c["cap"]:
        s = s.div_(c["cap"]).tanh_().mul_(c["cap"])
    lens = st["kv_lens"].long()
    new = st["starts"][1:].long() - st["starts"][:-1].long()
    p = ((lens - new)[:, None] + torch.arange(mq, device="cuda"))[:, :, None]        # [B, mq, 1]
    j = torch.arange(S, device="cuda")
    if c["bias"]:
        s -= st["slopes"].view(1, hkv, G, 1, 1) * (p - j).abs().float()[:, None, None]
    see = j <= p
    if c["prefix"]:
        see |= j < st["prefix"].long()[:, None, None]
    if c["window"]:
        see &= j > p - c["window"]
    see &= j < lens[:, None, None]
    s.masked_fill_(~see[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(-3e38)
    s = s.sub_(m).exp_()
    l = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, hkv, G * mq, S), v).view(B, hkv, G, mq, d) / l.clamp_min(1e-38)
    lse = torch.where(l > 0, m + l.log(), -math.inf).squeeze(-1)
    st["out"][:st["rows"]] = o.permute(0, 3, 1, 2, 4).reshape(B, mq, hq, d)[st["seq"], st["off"]].to(st["out"].dtype)
    st["lse"][:st["rows"]] = lse.permute(0, 3, 1, 2).reshape(B, mq, hq)[st["seq"], st["off"]]
    return [st["out"], st["lse"]]


def _logprobs_plain(st):
    c = st["case"]
    x = st["logits"].float()
    tok = st["tokens"].long()[:, None]
    xt = x.gather(1, tok)
    ids = torch.arange(c["vocab"], device="cuda")
    rank = ((x > xt) | ((x == xt) & (ids < tok))).sum(1).to(torch.int32)
    top = torch.sort(x, dim=1, descending=True, stable=True)
    top_x, top_ids = top.values[:, :c["top"]], top.indices[:, :c["top"]].to(torch.int32)
    m = x.amax(1, keepdim=True)
    e = (x - m) / c["temperature"]
    p = e.exp()
    total = p.sum(1, keepdim=True)
    log_total = total.log()
    entropy = log_total - torch.where(p > 0, p * e, 0.0).sum(1, keepdim=True) / total
    lse = m / c["temperature"] + log_total
    lp = (xt - m) / c["temperature"] - log_total
    return [lp[:, 0], lse[:, 0], entropy[:, 0], rank, top_ids, (top_x - m) / c["temperature"] - log_total]


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "append":
        return _append_plain(state)
    return _attention_plain(state) if kind == "attention" else _logprobs_plain(state)


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logprobs":
        return _logprobs_exact(st)
    return _append_exact(st) if case["kind"] == "append" else _attention_exact(st)


def _logprobs_exact(st):
    c = st["case"]
    T, tok = c["temperature"], st["tokens"].long()
    out = [[], [], [], []]
    for a in range(0, c["rows"], 256):      # the rows in pieces: 64-bit copies are large
        x = st["logits"][a:a + 256].double() / T
        lse = torch.logsumexp(x, 1)
        lp = x - lse[:, None]
        out[0].append(lp[torch.arange(len(x)), tok[a:a + 256]])
        out[1].append(lse)
        out[2].append(-(lp.exp() * lp).sum(1))
        out[3].append(lp.topk(c["top"], dim=1).values if c["top"] else lp[:, :0])
    lp, lse, entropy, top = (torch.cat(v) for v in out)
    return [lp, lse, entropy, None, None, top]


def _append_exact(st):
    c = st["case"]
    d, P, n = c["d"], c["page"], st["rows"]
    half = d // 2
    z = torch.polar(torch.ones(n, half, dtype=torch.float64, device="cuda"),
                    st["pos"].double()[:, None] / THETA ** (torch.arange(half, device="cuda").double() / half))

    def turn(x, w):
        x = x[:n].double()
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        pairs = x.unflatten(-1, (2, half)).transpose(-1, -2) if c["halves"] else x.unflatten(-1, (half, 2))
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z[:, None])
        return (y.transpose(-1, -2) if c["halves"] else y).flatten(-2)

    q_out = torch.zeros(st["q_out"].shape, dtype=torch.float64, device="cuda")
    k_pages = torch.zeros(st["k_pages"].shape, dtype=torch.float64, device="cuda")
    v_pages = torch.zeros(st["v_pages"].shape, dtype=torch.float64, device="cuda")
    q_out[:n] = turn(st["q"], st["q_scale"])
    k = turn(st["k"], st["k_scale"])
    heads = torch.arange(c["hkv"], device="cuda")[None]
    at = (st["page_of"][:, None], heads, (st["pos"] % P)[:, None])
    k_pages[at] = k
    v_pages.transpose(2, 3)[at] = st["v"][:n].double()
    return [q_out, k_pages, v_pages]


def _attention_exact(st):
    c = st["case"]
    hq, hkv, d, P = c["hq"], c["hkv"], c["d"], c["page"]
    G = hq // hkv
    out = torch.zeros(st["T"], hq, d, dtype=torch.float64, device="cuda")
    lses = torch.zeros(st["T"], hq, dtype=torch.float64, device="cuda")
    row = 0
    for s, (n, L) in enumerate(zip(st["n"], st["lens"])):
        if n == 0:
            continue
        used = st["table"][s, :(L + P - 1) // P].long()
        p = torch.arange(L - n, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None]
        hide = j > p
        if c["prefix"]:
            hide = hide & (j >= st["prefix"][s].long())
        if c["window"]:
            hide = hide | (p - j >= c["window"])
        for h in range(hkv):
            k = st["k_pages"][used, h].double().reshape(-1, d)[:L]
            v = st["v_pages"][used, h].double().transpose(1, 2).reshape(-1, d)[:L]
            for e in range(G):
                x = (st["q"][row:row + n, h * G + e].double() @ k.T.contiguous()) / math.sqrt(d)
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                if c["bias"]:
                    x = x - st["slopes"][h * G + e].double() * (p - j).abs()
                x = x.masked_fill(hide, -math.inf)
                lse = torch.logsumexp(x, 1)
                out[row:row + n, h * G + e] = torch.exp(x - lse[:, None]) @ v
                lses[row:row + n, h * G + e] = lse
        row += n
    return [out, lses]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "logprobs":
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 5 * 4 + 8 * case["top"]),
                "flops": 4.0 * case["rows"] * case["vocab"]}
    n, lens = _batch(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    rows = sum(n)
    if case["kind"] == "append":
        return {"bytes": 2 * 2 * rows * (hq + 2 * hkv) * d + 8 * d, "flops": 10.0 * rows * (hq + hkv) * d}
    seen, keys = 0, 0
    for m, L in zip(n, lens):
        p = np.arange(L - m, L)
        hi = np.minimum(np.maximum(p + 1, min(case["prefix"], L)), L)
        lo = np.maximum(p + 1 - case["window"], 0) if case["window"] else np.zeros_like(p)
        seen += int((hi - lo).sum())
        keys += int(hi.max() - lo.min()) if m else 0
    return {"bytes": 2 * 2 * rows * hq * d + 4 * rows * hq + 2 * 2 * keys * hkv * d, "flops": 4.0 * d * hq * seen}

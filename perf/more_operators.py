# SPDX-License-Identifier: MIT
"""The operators that continue and score requests, and how a program calls each of them.

  chunk     new tokens of requests that have tokens in the paged bf16 cache already: attention of every new token over its
            request's cache up to itself (`ops.paged_attn_chunk`)
  chunk4    the same over the 4-bit cache (`ops.paged_attn_chunk_q4`)
  logprobs  log probabilities of given tokens, the entropy of the distribution and its most likely tokens
            (`ops.token_logprobs`)

With `own` false `run` states the same in elementary torch operations.  The 4-bit cache holds keys and values in groups of 32
dimensions of a head: a group's lowest element `low` and `step` = bf16((highest - low) / 15) stand beside its codes
rint((x - low) / step), 0 to 15; a code reads as bf16(low + step * code), and attention is over what is read.
"""
import math

import torch

own = False

GROUP = 32
# (query heads, KV heads, head dim): the 7B and 32B decoder shapes whole, the 7B shape as two ranks hold it, the tiny
# decoder's, one KV head with few and with many query heads, no shared heads
HEADS = [(28, 4, 128), (40, 8, 128), (14, 2, 128), (8, 2, 64), (7, 1, 128), (16, 1, 128), (4, 4, 128), (12, 1, 64)]
# what a drawn case may cost: (new token, query head, key) triples and (request, KV head, token) triples
MOST_PAIRS, MOST_KEYS = 2048 * 40 * 16383, 2 * 8 * 100000


def listed():
    return [
        # an interactive request whose draft tokens are checked: latency counts
        dict(name="chunk_b1_5x333", op="chunk", heads=0, batch=1, new=5, ctx=333, block=16),
        # a serving batch with draft tokens, lengths as continuous batching has them
        dict(name="chunk_b64_8x1100", op="chunk", heads=0, batch=64, new=8, ctx=1100, block=16),
        # further turns of some conversations on the 7B shape as two ranks hold it
        dict(name="chunk_b9_700x5001", op="chunk", heads=2, batch=9, new=700, ctx=5001, block=16),
        # a piece of a long prompt on the 32B shape
        dict(name="chunk_b1_2048x16383", op="chunk", heads=1, batch=1, new=2048, ctx=16383, block=32),
        # the interactive request and the serving batch on the 4-bit cache
        dict(name="chunk4_b1_4x900", op="chunk4", heads=0, batch=1, new=4, ctx=900, block=16),
        dict(name="chunk4_b64_6x1100", op="chunk4", heads=0, batch=64, new=6, ctx=1100, block=16),
        # two very long conversations get a short turn
        dict(name="chunk4_b2_13x100000", op="chunk4", heads=1, batch=2, new=13, ctx=100000, block=32),
        # a piece of a long prompt
        dict(name="chunk4_b1_1500x9000", op="chunk4", heads=0, batch=1, new=1500, ctx=9000, block=16),
        # the token that a request has produced, with the alternatives that a client asks for
        dict(name="logprobs_b1", op="logprobs", rows=1, vocab=152064, top=20, ids=1, fp32=False),
        # a serving batch
        dict(name="logprobs_b64", op="logprobs", rows=64, vocab=152064, top=5, ids=1, fp32=False),
        # a prompt scored
        dict(name="logprobs_2000", op="logprobs", rows=2000, vocab=152064, top=0, ids=1, fp32=False),
        # answers of one token each compared under a few questions: fp32, odd vocabulary
        dict(name="logprobs_33_fp32", op="logprobs", rows=33, vocab=32003, top=8, ids=4, fp32=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "chunk4", "chunk4", "logprobs"])
    if op == "logprobs":
        vocab = _log(rng, 500, 152064)
        return dict(op=op, rows=_log(rng, 1, 2000), vocab=vocab, top=rng.choice([0, 1, 5, 8, 20, rng.randint(2, 20)]), ids=rng.choice([1, 1, rng.randint(2, 8)]),
                    fp32=rng.random() < 0.3)
    heads = rng.randrange(len(HEADS))
    nq, nkv, _ = HEADS[heads]
    batch = _log(rng, 1, 96)
    new = _log(rng, 1, min(2048, max(1, MOST_PAIRS // (batch * nq * 400))))
    ctx = _log(rng, new, max(new, min(100000, MOST_KEYS // (batch * nkv), MOST_PAIRS // (batch * nq * new))))
    return dict(op=op, heads=heads, batch=batch, new=new, ctx=ctx, block=rng.choice([16, 16, 32, 64]))


# ---------------------------------------------------------------- inputs, from the seed alone
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)


def _ints(g, lo, hi, *shape):
    """int32 in [lo, hi]"""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _new_lens(case):
    """From case["new"] tokens down to next to none, evenly spread: a step has the same number of rows whichever request has how many."""
    return [case["new"] - (case["new"] + 1) * i // case["batch"] for i in range(case["batch"])] if case["new"] > 1 else [1] * case["batch"]


def _chunk_inputs(case, seed):
    nq, nkv, hd = HEADS[case["heads"]]
    g, b, bs = _gen(seed), case["batch"], case["block"]
    new = torch.tensor(_new_lens(case), dtype=torch.int32, device="cuda")[torch.randperm(b, generator=g, device="cuda")]
    lens = torch.maximum(_ints(g, 0, case["ctx"], b), new)
    lens[new.argmax()] = case["ctx"]
    cu = torch.zeros(b + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(new, 0)
    per = -(-case["ctx"] // bs)  # blocks of a request
    n_blocks = b * per + 3
    table = torch.randperm(n_blocks, generator=g, device="cuda")[: b * per].to(torch.int32).view(b, per).contiguous()
    # keys with channels of their own size and offset, as projections with a bias give them; values around zero
    size, off = 0.5 + torch.rand(nkv, 1, hd, generator=g, device="cuda"), torch.randn(nkv, 1, hd, generator=g, device="cuda")
    k = (torch.randn(n_blocks, nkv, bs, hd, generator=g, device="cuda") * size + off).bfloat16()
    v = torch.randn(n_blocks, nkv, bs, hd, generator=g, device="cuda").bfloat16()
    # (the rows of the QKV linear: the queries are their first columns)
    qkv = torch.randn(int(cu[-1]), (nq + 2 * nkv) * hd, generator=g, device="cuda").bfloat16()
    return dict(nq=nq, nkv=nkv, hd=hd, bs=bs, cu=cu, lens=lens, table=table, k=k, v=v, qkv=qkv, most=case["new"], scale=1.0 / math.sqrt(hd))


def _logits_inputs(case, seed):
    g, rows, vocab = _gen(seed), case["rows"], case["vocab"]
    # some rows are sure of their token, others are not
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * (1 + 3 * torch.rand(rows, 1, generator=g, device="cuda"))
    ids = _ints(g, 0, vocab - 1, rows, case["ids"])
    # a token that the model expected: the row's most likely one
    ids[:, 0] = torch.where(_ints(g, 0, 1, rows) == 0, ids[:, 0], logits.argmax(1).to(torch.int32))
    return dict(logits=logits if case["fp32"] else logits.bfloat16(), ids=ids[:, 0].contiguous() if case["ids"] == 1 else ids, top=case["top"])


def prepare(case, seed):
    if case["op"] == "logprobs":
        return _logits_inputs(case, seed)
    s = _chunk_inputs(case, seed)
    if case["op"] == "chunk4":
        if own:
            from barlink_sm86_b200 import ops

            n_blocks, nkv, bs, hd = s["k"].shape
            rows = n_blocks * bs
            cache = ops.kv4_cache(n_blocks, nkv, hd, bs, "cuda")
            kv = torch.cat([s["k"].transpose(1, 2), s["v"].transpose(1, 2)], 2).reshape(rows, -1)
            # (position 0: kept as they are)
            ops.rope_kv_write_q4(kv, torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.arange(rows, dtype=torch.int32, device="cuda"), cache, 0,
                                 nkv, hd, bs, 1e6)
            s["cache"] = cache
        else:
            s["kc"], s["vc"] = _quantise(s["k"]), _quantise(s["v"])
        del s["k"], s["v"]
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from barlink_sm86_b200 import ops

    if "logits" in s:
        r = ops.token_logprobs(s["logits"], s["ids"], top=s["top"])
        return [r.logprobs, r.entropy, r.top_ids, r.top_logprobs] if s["top"] else [r.logprobs, r.entropy]
    if "cache" in s:
        return ops.paged_attn_chunk_q4(s["qkv"], s["cache"], s["table"], s["cu"], s["lens"], s["nq"], s["nkv"], s["hd"], s["scale"])
    return ops.paged_attn_chunk(s["qkv"], s["k"], s["v"], s["table"], s["cu"], s["lens"], s["nq"], s["nkv"], s["hd"], s["scale"])


def _run_plain(s):
    return _plain_logprobs(s) if "logits" in s else _plain_chunk(s)


def _quantise(x):
    """[..., hd] bf16 values -> (codes uint8, low, step), a group's low and step once a group."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low = x.amin(-1, keepdim=True)
    step = ((x.amax(-1, keepdim=True) - low) / 15).bfloat16().float()
    codes = torch.where(step > 0, torch.round((x - low) / step), torch.zeros_like(x)).clamp(0, 15)
    return codes.to(torch.uint8), low.bfloat16(), step.bfloat16()


def _gathered(s, name):
    """Keys or values of every request's pages, fp32 [batch, nkv, tokens, hd]."""
    table = s["table"].long()
    if name in s:
        x = s[name][table].float()
    else:
        codes, low, step = (t[table] for t in s[name + "c"])
        x = (low.float() + step.float() * codes.float()).flatten(-2).bfloat16().float()
    return x.transpose(1, 2).flatten(2, 3)  # [batch, pages, nkv, block, hd] -> [batch, nkv, pages * block, hd]


def _plain_chunk(s):
    nq, nkv, hd, most = s["nq"], s["nkv"], s["hd"], s["most"]
    b, tokens, cu = s["table"].shape[0], s["qkv"].shape[0], s["cu"].long()
    new, lens = cu[1:] - cu[:-1], s["lens"].long()
    # queries padded to the longest chunk: [batch, nkv, new * group, hd]
    i = torch.arange(most, device="cuda")
    there = i < new[:, None]
    at = (cu[:-1, None] + i).clamp(max=tokens - 1)
    q = s["qkv"][:, : nq * hd].float()[at].view(b, most, nkv, nq // nkv, hd).permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, hd)
    k, v = _gathered(s, "k"), _gathered(s, "v")
    x = (q @ k.transpose(2, 3)) * s["scale"]
    pos = (lens - new)[:, None] + i
    seen = (torch.arange(k.shape[2], device="cuda") <= torch.where(there, pos, -1)[:, :, None])
    seen = seen[:, None, :, None].expand(b, 1, most, nq // nkv, -1).reshape(b, 1, -1, k.shape[2])
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    # (blocks behind a request's last token are another's, or nobody's)
    v = torch.where((torch.arange(v.shape[2], device="cuda") < lens[:, None])[:, None, :, None], v, 0.0)
    o = torch.where(total > 0, (p @ v) / total, 0.0)
    o = o.view(b, nkv, most, nq // nkv, hd).permute(0, 2, 1, 3, 4).reshape(b, most, nq * hd)
    return o[there].bfloat16()  # request by request, as the rows were


def _plain_logprobs(s):
    x = s["logits"].float()
    t = x - x.amax(-1, keepdim=True)
    e = torch.exp(t)
    total = e.sum(-1, keepdim=True)
    entropy = torch.log(total[:, 0]) - (t * e).sum(-1) / total[:, 0]
    logp = t - torch.log(total)
    ids = s["ids"].long()
    given = logp.gather(1, ids.view(ids.shape[0], -1)).view(ids.shape)
    if not s["top"]:
        return [given, entropy]
    # ties go to the lowest index
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : s["top"]]
    return [given, entropy, order.to(torch.int32), logp.gather(1, order)]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["fp32"] else 2) + case["rows"] * (8 * case["ids"] + 4 + 8 * case["top"]), "flops": 5 * n}
    nq, nkv, hd = HEADS[case["heads"]]
    held = 4 * hd if case["op"] == "chunk" else 2 * (hd // 2 + 4 * (hd // GROUP))  # bytes of a token and head
    # requests without the longest chunk have up to ctx tokens, and no less than their new ones
    new, ctx = _new_lens(case), case["ctx"]
    keys, pairs = 0.0, 0.0
    for i, n in enumerate(new):
        mean = ctx if i == 0 else (n * n + ctx * ctx) / (2 * ctx)
        keys += mean if n else 0
        pairs += n * (mean - (n - 1) / 2)
    rows = sum(new)
    return {"bytes": keys * nkv * held + rows * nq * hd * 4, "flops": 4 * pairs * nq * hd}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_cache(x):
    """What the 4-bit cache reads as for bf16 values, in 64 bits."""
    shape = x.shape
    x = x.double().reshape(-1, GROUP)
    low, high = x.min(1).values[:, None], x.max(1).values[:, None]
    step = ((high - low) / 15).to(torch.bfloat16).double()
    return (low + step * torch.round((x - low) / step.clamp(min=1e-300)).clamp(0, 15)).reshape(shape).to(torch.bfloat16)


def exact(case, seed):
    if case["op"] == "logprobs":
        s = _logits_inputs(case, seed)
        x = s["logits"].double()
        x -= torch.logsumexp(x, 1)[:, None]
        given = torch.stack([x[torch.arange(x.shape[0], device="cuda"), i] for i in s["ids"].long().view(x.shape[0], -1).unbind(1)], 1)
        best = x.topk(s["top"]).values if s["top"] else None
        entropy = -torch.special.xlogy(torch.exp(x), torch.exp(x)).sum(1)
        return [given.view(s["ids"].shape), entropy] + ([None, best] if s["top"] else [])
    s = _chunk_inputs(case, seed)
    nq, nkv, hd, bs = s["nq"], s["nkv"], s["hd"], s["bs"]
    out = torch.zeros(s["qkv"].shape[0], nkv, nq // nkv, hd, dtype=torch.float64, device="cuda")
    cu = s["cu"].tolist()
    for i, n in enumerate(s["lens"].tolist()):
        m = cu[i + 1] - cu[i]
        if not m:
            continue
        pages = s["table"][i, : -(-n // bs)].long()
        hidden = torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + 1)
        for h in range(nkv):
            k, v = (t[pages, h].reshape(-1, hd)[:n] for t in (s["k"], s["v"]))
            if case["op"] == "chunk4":
                k, v = _exact_cache(k), _exact_cache(v)
            q = s["qkv"][cu[i]: cu[i + 1], : nq * hd].view(m, nkv, nq // nkv, hd)[:, h].double()
            for j in range(q.shape[1]):
                x = (q[:, j] @ k.double().T).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
                out[cu[i]: cu[i + 1], h, j] = torch.softmax(x, 1) @ v.double()
    return out.flatten(1)

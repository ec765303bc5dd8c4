# SPDX-License-Identifier: MIT
"""The operators that serve ragged requests from a key/value cache held in 4 bits, and how a program calls each of them.

  attn    one query token per request against the paged 4-bit cache (`ops.paged_attn_decode_q4`)
  write   RoPE on a step's queries and keys; its keys and values are quantised into the cache
          (`ops.rope_kv_write_q4`), then read back from it (`ops.kv4_read`)
  layout  request lengths to block tables, row offsets, positions and slots (`ops.paged_layout`)
  logits  penalties for repeated tokens, biases and a grammar mask on the logits, and the arg max of the
          result (`ops.logits_argmax`, `ops.logits_process`)
  count   token histories to the tables that the penalties read (`ops.count_tokens`)

With `own` false `run` states the same in elementary torch operations.  What the cache holds: keys after RoPE and values, both
rounded to bf16, in groups of 32 dimensions of a head; a group's lowest element `low` and `step` = bf16((highest - low) / 15)
stand beside its codes rint((x - low) / step), 0 to 15; a code stands for low + step * code.
"""
import math

import torch

own = False

GROUP = 32
# (query heads, KV heads, head dim): the 7B and 32B decoder shapes whole, the 7B shape as two ranks hold it, the tiny
# decoder's, one KV head with few and with many query heads, no shared heads
HEADS = [(28, 4, 128), (40, 8, 128), (14, 2, 128), (8, 2, 64), (7, 1, 128), (16, 1, 128), (4, 4, 128), (12, 1, 64)]


def listed():
    return [
        # an interactive request: little to read, latency counts
        dict(name="attn_b1_333", op="attn", heads=0, batch=1, ctx=333, block=16),
        # the serving batch of the headline shape, lengths as continuous batching has them
        dict(name="attn_b64_1100", op="attn", heads=0, batch=64, ctx=1100, block=16),
        # a few very long conversations on the 32B shape
        dict(name="attn_b4_32k", op="attn", heads=1, batch=4, ctx=32767, block=32),
        # a decode step's new tokens: k-split slabs of the QKV linear with its bias
        dict(name="write_decode_64", op="write", heads=0, rows=64, splits=3, pos=32000, block=16),
        # the largest prefill pass of the engine, odd by one row
        dict(name="write_prefill_8191", op="write", heads=0, rows=8191, splits=0, pos=8000, block=16),
        # every request of a batch gets one token
        dict(name="layout_decode_64", op="layout", batch=64, new=1, past=4000, block=16),
        # prompts come in, others go on, some requests end
        dict(name="layout_mixed_700", op="layout", batch=700, new=90, past=3000, block=32),
        # one interactive request with all rules
        dict(name="logits_b1", op="logits", rows=1, vocab=152064, hist=900, bias=8, mask=True, pick=True, fp32=False),
        # a serving batch: greedy tokens under all rules
        dict(name="logits_b64", op="logits", rows=64, vocab=152064, hist=1500, bias=16, mask=True, pick=True, fp32=False),
        # logits for a sampler behind: fp32, odd vocabulary
        dict(name="logits_process_33", op="logits", rows=33, vocab=32003, hist=700, bias=0, mask=True, pick=False, fp32=True),
        # a single request resumed with its history
        dict(name="count_b1", op="count", rows=1, vocab=152064, hist=2000),
        # a whole batch set up
        dict(name="count_b64", op="count", rows=64, vocab=152064, hist=3000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "write", "write", "layout", "logits", "logits", "count"])
    block = rng.choice([16, 16, 32, 64])
    if op == "attn":
        heads = rng.randrange(len(HEADS))
        batch = _log(rng, 1, 96)
        # cost: (request, KV head, token) triples, up to those of the largest listed case
        most = min(32767, (4 * 32767 * 8) // (batch * HEADS[heads][1]))
        return dict(op=op, heads=heads, batch=batch, ctx=_log(rng, 1, most), block=block)
    if op == "write":
        splits = rng.choice([0, 0, rng.randint(1, 8)])
        return dict(op=op, heads=rng.choice([0, 2, 3, 4, 5, 6, 7]), rows=_log(rng, 1, 128 if splits else 8191), splits=splits,
                    pos=_log(rng, 1, 130000), block=block)
    if op == "layout":
        batch = _log(rng, 1, 1500)
        return dict(op=op, batch=batch, new=_log(rng, 1, max(2, 63000 // batch)), past=_log(rng, 1, 9000), block=block)
    vocab = _log(rng, 500, 152064)
    if op == "logits":
        return dict(op=op, rows=_log(rng, 1, 64), vocab=vocab, hist=_log(rng, 1, 1500), bias=rng.choice([0, 1, 7, 16]), mask=rng.random() < 0.7,
                    pick=rng.random() < 0.6, fp32=rng.random() < 0.3)
    return dict(op=op, rows=_log(rng, 1, 64), vocab=vocab, hist=_log(rng, 1, 3000))


# ---------------------------------------------------------------- inputs, from the seed alone
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)


def _ints(g, lo, hi, *shape):
    """int32 in [lo, hi]"""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _kv(g, rows, nkv, hd):
    """Keys with channels of their own size and offset, as projections with a bias give them; values around zero."""
    size = 0.5 + torch.rand(nkv, hd, generator=g, device="cuda")
    off = torch.randn(nkv, hd, generator=g, device="cuda")
    k = torch.randn(rows, nkv, hd, generator=g, device="cuda") * size + off
    v = torch.randn(rows, nkv, hd, generator=g, device="cuda")
    return k.bfloat16(), v.bfloat16()


def _attn_inputs(case, seed):
    nq, nkv, hd = HEADS[case["heads"]]
    g, b, bs = _gen(seed), case["batch"], case["block"]
    lens = _ints(g, 0, case["ctx"], b)
    lens[0] = case["ctx"]
    per = -(-case["ctx"] // bs)  # blocks of a request
    n_blocks = b * per + 3
    table = torch.randperm(n_blocks, generator=g, device="cuda")[: b * per].to(torch.int32).view(b, per).contiguous()
    k, v = _kv(g, n_blocks * bs, nkv, hd)
    qkv = torch.randn(b, (nq + 2 * nkv) * hd, generator=g, device="cuda").bfloat16()
    return dict(nq=nq, nkv=nkv, hd=hd, bs=bs, lens=lens, table=table, n_blocks=n_blocks, k=k, v=v, qkv=qkv, scale=1.0 / math.sqrt(hd))


def _write_inputs(case, seed):
    nq, nkv, hd = HEADS[case["heads"]]
    g, rows, bs = _gen(seed), case["rows"], case["block"]
    n_blocks = -(-rows // bs) + 5
    width = (nq + 2 * nkv) * hd
    if case["rows"] > 128:  # a prompt: neighbouring tokens stand in neighbouring slots of scattered blocks
        blocks = torch.randperm(n_blocks, generator=g, device="cuda")
        at = torch.arange(rows, device="cuda") + 3
        slots = (blocks[at // bs] * bs + at % bs).to(torch.int32)
        pos = ((case["pos"] + torch.arange(rows, device="cuda")) % 131072).to(torch.int32)
    else:
        slots = torch.randperm(n_blocks * bs, generator=g, device="cuda")[:rows].to(torch.int32)
        pos = _ints(g, 0, case["pos"], rows)
    slots = torch.where(_ints(g, 0, 40, rows) == 0, -1, slots)  # rows of padding are not kept
    x = torch.randn(rows, width, generator=g, device="cuda") * (0.5 + torch.rand(width, generator=g, device="cuda"))
    d = dict(nq=nq, nkv=nkv, hd=hd, bs=bs, n_blocks=n_blocks, slots=slots, pos=pos, bias=None, splits=case["splits"], theta=1e6)
    if case["splits"]:
        d["qkv"] = torch.randn(case["splits"], rows, width, generator=g, device="cuda") + x / case["splits"]
        d["bias"] = torch.randn(width, generator=g, device="cuda").bfloat16()
    else:
        d["qkv"] = x.bfloat16()
    return d


def _layout_inputs(case, seed):
    g, b, bs = _gen(seed), case["batch"], case["block"]
    new = _ints(g, 0, 2 * case["new"], b) if case["new"] > 1 else torch.ones(b, dtype=torch.int32, device="cuda")
    past = _ints(g, 0, case["past"], b)
    width = -(-(case["past"] + 2 * case["new"]) // bs)
    if case["new"] > 1:
        new = torch.where(_ints(g, 0, 20, b) == 0, -1, new)  # a request in 21 has ended
    n_blocks = b * width + 1
    ids = torch.randperm(n_blocks, generator=g, device="cuda").to(torch.int32)
    table = ids[: b * width].view(b, width)
    held = torch.arange(width, device="cuda")[None] < ((past + bs - 1) // bs)[:, None]
    # the ring of free blocks: those that no request holds, from somewhere inside it
    free = torch.cat([table[~held], ids[b * width:]])
    head = n_blocks // 3
    ring = torch.full((n_blocks,), -7, dtype=torch.int32, device="cuda")
    ring[(head + torch.arange(free.numel(), device="cuda")) % n_blocks] = free
    return dict(new=new, past=past, bs=bs, table=torch.where(held, table, -1).contiguous(), ring=ring, tokens=b * max(1, 2 * case["new"]),
                range=torch.tensor([head, free.numel(), 0], dtype=torch.int32, device="cuda"))


def _packed_ids(g, rows, vocab, hist):
    """Histories of 0..hist tokens, packed; frequent tokens are the low ids, as in text."""
    lens = _ints(g, 0, hist, rows)
    lens[0] = hist
    cu = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(lens, 0)
    u = torch.rand(rows * hist, generator=g, device="cuda")
    ids = (vocab * u ** 3).to(torch.int32).clamp_(0, vocab - 1)
    # (the buffer is as long as the longest histories would need; what stands behind the last one belongs to no request)
    return ids, cu, torch.minimum(lens, _ints(g, 0, hist, rows))


def _logits_inputs(case, seed):
    g, rows, vocab = _gen(seed), case["rows"], case["vocab"]
    logits = 3 * torch.randn(rows, vocab, generator=g, device="cuda")
    ids, cu, prompt = _packed_ids(g, rows, vocab, case["hist"])
    counts, seen = _plain_count(ids, cu, prompt, rows, vocab)
    pen = torch.rand(rows, 3, generator=g, device="cuda") * torch.tensor([0.5, 0.5, 0.3], device="cuda") + torch.tensor([1.0, 0.0, 0.0], device="cuda")
    d = dict(logits=logits if case["fp32"] else logits.bfloat16(), counts=counts, seen=seen, penalties=pen, bias_ids=None, bias=None, mask=None, pick=case["pick"])
    if case["bias"]:
        d["bias_ids"] = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda", dtype=torch.int32)
        d["bias_ids"] = ((d["bias_ids"] + 17 * torch.arange(case["bias"], device="cuda", dtype=torch.int32)) % vocab).contiguous()
        d["bias_ids"][:, case["bias"] // 2 + 1:] = -1  # lists end early
        d["bias"] = 5 * torch.randn(rows, case["bias"], generator=g, device="cuda")
    if case["mask"]:
        words = -(-vocab // 32)
        d["mask"] = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=g, device="cuda").to(torch.int32)
        d["mask"] &= torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=g, device="cuda").to(torch.int32)
        if rows > 2:
            d["mask"][2] = 0  # a grammar that allows nothing
    return d


def prepare(case, seed):
    if case["op"] == "attn":
        s = _attn_inputs(case, seed)
        if own:
            from barlink_sm86_b200 import ops

            rows = s["n_blocks"] * s["bs"]
            cache = ops.kv4_cache(s["n_blocks"], s["nkv"], s["hd"], s["bs"], "cuda")
            # (position 0: kept as they are)
            ops.rope_kv_write_q4(torch.cat([s["k"], s["v"]], 1).view(rows, -1), torch.zeros(rows, dtype=torch.int32, device="cuda"),
                                 torch.arange(rows, dtype=torch.int32, device="cuda"), cache, 0, s["nkv"], s["hd"], s["bs"], 1e6)
            s["cache"] = cache
        else:
            s["kc"], s["vc"] = _quantise(s["k"]), _quantise(s["v"])
        del s["k"], s["v"]
        return s
    if case["op"] == "write":
        s = _write_inputs(case, seed)
        if own:
            from barlink_sm86_b200 import ops

            s["cache"] = ops.kv4_cache(s["n_blocks"], s["nkv"], s["hd"], s["bs"], "cuda")
        else:
            n = s["n_blocks"] * s["bs"]
            s["kc"], s["vc"] = (_quantise(torch.zeros(n, s["nkv"], s["hd"], device="cuda")) for _ in range(2))
        s["out"] = torch.empty(case["rows"], (s["nq"] + 2 * s["nkv"]) * s["hd"], dtype=torch.bfloat16, device="cuda")
        return s
    if case["op"] == "layout":
        return _layout_inputs(case, seed)
    if case["op"] == "logits":
        s = _logits_inputs(case, seed)
        if own:
            from barlink_sm86_b200 import ops

            s["rules"] = ops.LogitRules(penalties=s["penalties"], counts=s["counts"], seen=s["seen"], bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"])
        return s
    ids, cu, prompt = _packed_ids(_gen(seed), case["rows"], case["vocab"], case["hist"])
    s = dict(ids=ids, cu=cu, prompt=prompt, rows=case["rows"], vocab=case["vocab"])
    if own:
        from barlink_sm86_b200 import ops

        s["rules"] = ops.LogitRules.empty(case["rows"], case["vocab"], "cuda")
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from barlink_sm86_b200 import ops

    if "table" in s and "qkv" in s:
        return ops.paged_attn_decode_q4(s["qkv"], s["cache"], s["table"], s["lens"], s["nq"], s["nkv"], s["hd"], s["scale"])
    if "qkv" in s:
        out = ops.rope_kv_write_q4(s["qkv"], s["pos"], s["slots"], s["cache"], s["nq"], s["nkv"], s["hd"], s["bs"], s["theta"], bias=s["bias"], out=s["out"])
        return [out, *ops.kv4_read(s["cache"], s["slots"], s["hd"], s["bs"])]
    if "ring" in s:
        r = ops.paged_layout(s["new"], s["past"], s["table"], s["ring"], s["range"], s["tokens"], s["bs"])
        return [r.cu, r.positions, r.slots, r.ctx_lens, r.free_range, s["table"], s["ring"]]
    if "logits" in s:
        return list(ops.logits_argmax(s["logits"], s["rules"])) if s["pick"] else ops.logits_process(s["logits"], s["rules"])
    ops.count_tokens(s["rules"], s["ids"], s["cu"], s["prompt"], reset=True)
    return [s["rules"].counts, s["rules"].seen]


def _run_plain(s):
    if "table" in s and "qkv" in s:
        return _plain_attn(s)
    if "qkv" in s:
        return _plain_write(s)
    if "ring" in s:
        return _plain_layout(s)
    if "logits" in s:
        x = _plain_rules(s)
        if not s["pick"]:
            return x.to(s["logits"].dtype)
        val, idx = torch.where(x != x, -math.inf, x).max(-1)
        first = (x == val[:, None]).to(torch.int32).argmax(-1)  # ties go to the lowest index
        return [torch.where(val == -math.inf, -1, first).to(torch.int32), val]
    return list(_plain_count(s["ids"], s["cu"], s["prompt"], s["rows"], s["vocab"]))


def _quantise(x):
    """[..., hd] bf16 values -> (codes uint8, low, step), a group's low and step once a group."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low = x.amin(-1, keepdim=True)
    step = ((x.amax(-1, keepdim=True) - low) / 15).bfloat16().float()
    codes = torch.where(step > 0, torch.round((x - low) / step), torch.zeros_like(x)).clamp(0, 15)
    return codes.to(torch.uint8), low.bfloat16(), step.bfloat16()


def _values(c):
    return (c[1].float() + c[2].float() * c[0].float()).flatten(-2)


def _plain_attn(s):
    b, nq, nkv, hd, bs = s["qkv"].shape[0], s["nq"], s["nkv"], s["hd"], s["bs"]
    n = s["table"].shape[1] * bs
    at = (s["table"].long()[:, :, None] * bs + torch.arange(bs, device="cuda")).view(b, n)
    k, v = (_values([t[at] for t in c]).permute(0, 2, 1, 3) for c in (s["kc"], s["vc"]))  # [b, nkv, n, hd]
    q = s["qkv"][:, : nq * hd].float().view(b, nkv, nq // nkv, hd)
    x = (q @ k.transpose(2, 3)) * s["scale"]
    there = (torch.arange(n, device="cuda") < s["lens"][:, None])[:, None, None, :]
    x = torch.where(there, x, -math.inf)
    p = torch.where(there, torch.exp(x - x.amax(-1, keepdim=True)), 0.0)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, (p @ v) / total, 0.0)
    return o.reshape(b, nq * hd).bfloat16()


def _plain_write(s):
    nq, nkv, hd = s["nq"], s["nkv"], s["hd"]
    x = s["qkv"]
    if s["splits"]:
        total = x[0]
        for part in x[1:]:
            total = total + part
        x = (total + s["bias"].float()).bfloat16()
    rows = x.shape[0]
    x = x.float().view(rows, nq + 2 * nkv, hd)
    inv = s["theta"] ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = s["pos"].double()[:, None] * inv  # (in 64 bits: positions are far)
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[:, : nq + nkv, : hd // 2], x[:, : nq + nkv, hd // 2:]
    out = torch.cat([torch.cat([a * c - b * n, b * c + a * n], -1), x[:, nq + nkv:]], 1).bfloat16()
    keep = (s["slots"] >= 0).view(rows, 1, 1)
    at = torch.where(s["slots"] >= 0, s["slots"], 0).long()
    read = []
    for cache, new in ((s["kc"], out[:, nq: nq + nkv]), (s["vc"], out[:, nq + nkv:])):
        codes = _quantise(new)
        # (rows that are not kept go to a slot behind the cache)
        n_slots = cache[0].shape[0]
        to = torch.where(s["slots"] >= 0, s["slots"].long(), n_slots)
        for t, c2 in zip(cache, codes):
            wide = torch.cat([t, t[:1]])
            wide[to] = c2
            t.copy_(wide[:-1])
        read.append(torch.where(keep, _values([t[at] for t in cache]), 0.0).bfloat16())
    s["out"].copy_(out.view(rows, -1))
    return [s["out"], *read]


def _plain_layout(s):
    new, past, bs, table, ring, tokens = s["new"], s["past"], s["bs"], s["table"], s["ring"], s["tokens"]
    b, width = table.shape
    cap, dev = ring.numel(), ring.device
    head, free = s["range"][0].long(), s["range"][1].long()
    add = new.clamp(min=0).long()
    past = past.long()
    cu = torch.zeros(b + 1, dtype=torch.int64, device=dev)
    cu[1:] = torch.cumsum(add, 0)
    ended = new < 0
    had = ((past + bs - 1) // bs).clamp(max=width)
    want = torch.where(ended, had, ((past + add + bs - 1) // bs).clamp(max=width))
    page = torch.arange(width, device=dev)
    fresh = (page >= had[:, None]) & (page < want[:, None])
    nth = (torch.cumsum(fresh.reshape(-1).long(), 0) - 1).view(b, width)
    got = torch.where(nth < free, ring[(head + nth.clamp(min=0)) % cap], -1)
    need = fresh.sum()
    # blocks of requests that ended go to the end of the ring
    back = ended[:, None] & (page < had[:, None]) & (table >= 0)
    place = torch.cumsum(back.reshape(-1).long(), 0) - 1 + free
    place = torch.where(back.reshape(-1) & (place < cap), (head + place) % cap, cap)
    wide = torch.cat([ring, ring[:1]])
    wide[place] = table.reshape(-1)
    ring.copy_(wide[:-1])
    table.copy_(torch.where(fresh, got, table))
    taken = torch.minimum(need, free)
    given = torch.minimum(back.sum(), cap - free)
    left = torch.stack([(head + taken) % cap, free - taken + given, (need - free).clamp(min=0)]).to(torch.int32)
    row = torch.arange(tokens, device=dev)
    of = torch.searchsorted(cu, row, right=True) - 1
    there = of < b
    of = of.clamp(max=b - 1)
    pos = torch.where(there, past[of] + row - cu[of], 0)
    p = pos // bs
    blk = torch.where(p < width, table[of, p.clamp(max=width - 1)], -1)
    slot = torch.where(there & (blk >= 0), blk * bs + pos % bs, -1)
    return [cu.to(torch.int32), pos.to(torch.int32), slot.to(torch.int32), torch.where(ended, 0, past + add).to(torch.int32), left, table, ring]


def _bits(words, n):
    return ((words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1).flatten(1)[:, :n] != 0


def _plain_rules(s):
    x = s["logits"].float()
    n = x.shape[1]
    again, presence, frequency = (s["penalties"][:, i: i + 1] for i in range(3))
    x = torch.where(_bits(s["seen"], n), torch.where(x > 0, x / again, x * again), x)
    x = torch.where(s["counts"] > 0, (x - frequency * s["counts"].float()) - presence, x)
    if s["bias_ids"] is not None:
        there = s["bias_ids"] >= 0
        extra = torch.zeros(x.shape[0], n + 1, device=x.device)
        extra.scatter_add_(1, torch.where(there, s["bias_ids"], n).long(), s["bias"])
        x = x + extra[:, :n]
    if s["mask"] is not None:
        x = torch.where(_bits(s["mask"], n), x, -math.inf)
    return x


def _plain_count(ids, cu, prompt, rows, vocab):
    at = torch.arange(ids.numel(), device=ids.device)
    of = torch.searchsorted(cu.long(), at, right=True) - 1
    there = of < rows
    of = of.clamp(max=rows - 1)
    made = there & (at - cu.long()[of] >= prompt[of])
    slot = torch.where(there, of * vocab + ids, rows * vocab)
    counts = torch.zeros(rows * vocab + 1, dtype=torch.int32, device=ids.device)
    counts.scatter_add_(0, slot, made.to(torch.int32))
    words = -(-vocab // 32)
    hit = torch.zeros(rows * vocab + 1, dtype=torch.int32, device=ids.device)
    hit[slot] = 1
    hit = torch.nn.functional.pad(hit[:-1].view(rows, vocab), (0, words * 32 - vocab)).view(rows, words, 32)
    seen = (hit << torch.arange(32, device=ids.device, dtype=torch.int32)).sum(-1).to(torch.int32)  # (bit 31 wraps)
    return counts[:-1].view(rows, vocab), seen


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] in ("attn", "write"):
        nq, nkv, hd = HEADS[case["heads"]]
        held = 2 * nkv * (hd // 2 + 4 * (hd // GROUP))  # bytes of a token in the cache: codes, low and step, keys and values
    if case["op"] == "attn":
        # requests after the first are of 0..ctx tokens
        tokens = case["ctx"] + (case["batch"] - 1) * case["ctx"] / 2
        return {"bytes": tokens * held + case["batch"] * nq * hd * 4, "flops": 4 * tokens * nq * hd}
    if case["op"] == "write":
        width = (nq + 2 * nkv) * hd
        # QKV in, rotated QKV out, the cache written and read, values out
        return {"bytes": case["rows"] * (width * (4 * case["splits"] or 2) + 2 * width + 2 * held + 4 * nkv * hd), "flops": case["rows"] * (4 * width + 10 * nkv * hd)}
    if case["op"] == "layout":
        tokens = case["batch"] * case["new"]
        return {"bytes": 16 * case["batch"] + 8 * case["batch"] * max(1, 2 * case["new"]) + 8 * (tokens // case["block"] + 1), "flops": tokens + case["batch"]}
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        size = 4 if case["fp32"] else 2
        # counts are read where a token was seen
        return {"bytes": n * (size + 1 / 8 + (1 / 8 if case["mask"] else 0) + (0 if case["pick"] else size)) + 2 * case["rows"] * case["hist"], "flops": 4 * n}
    tokens = case["rows"] * case["hist"] / 2
    return {"bytes": 4 * tokens + case["rows"] * case["vocab"] * (4 + 1 / 8), "flops": tokens}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_cache(x):
    """What the cache holds of bf16 values, in 64 bits."""
    shape = x.shape
    x = x.double().reshape(-1, GROUP)
    low, high = x.min(1).values[:, None], x.max(1).values[:, None]
    step = ((high - low) / 15).to(torch.bfloat16).double()
    return (low + step * torch.round((x - low) / step.clamp(min=1e-300)).clamp(0, 15)).reshape(shape)


def exact(case, seed):
    if case["op"] == "attn":
        s = _attn_inputs(case, seed)
        nq, nkv, hd, bs = s["nq"], s["nkv"], s["hd"], s["bs"]
        out = []
        for i, n in enumerate(s["lens"].tolist()):
            if not n:
                out.append(torch.zeros(nq * hd, dtype=torch.float64, device="cuda"))
                continue
            at = (s["table"][i, : -(-n // bs), None].long() * bs + torch.arange(bs, device="cuda")).flatten()[:n]
            k, v = (_exact_cache(t[at]).transpose(0, 1) for t in (s["k"], s["v"]))
            q = s["qkv"][i, : nq * hd].double().view(nkv, nq // nkv, hd)
            out.append((torch.softmax(torch.einsum("hgd,htd->hgt", q, k) * s["scale"], -1) @ v).flatten())
        return torch.stack(out)
    if case["op"] == "write":
        s = _write_inputs(case, seed)
        nq, nkv, hd = s["nq"], s["nkv"], s["hd"]
        # (the rows that the QKV linear leaves are bf16)
        x = (s["qkv"].double().sum(0) + s["bias"].double()).bfloat16().double() if s["splits"] else s["qkv"].double()
        x = x.view(case["rows"], -1, hd)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           s["pos"].double()[:, None] * torch.exp(-math.log(s["theta"]) * torch.arange(hd // 2, device="cuda").double() * 2 / hd))[:, None]
        z = torch.complex(x[:, : nq + nkv, : hd // 2], x[:, : nq + nkv, hd // 2:]) * turn
        x = torch.cat([torch.cat([z.real, z.imag], -1), x[:, nq + nkv:]], 1)
        kept = (s["slots"] >= 0)[:, None, None]
        k, v = (torch.where(kept, _exact_cache(t.bfloat16()), 0.0) for t in (x[:, nq: nq + nkv], x[:, nq + nkv:]))
        return [x.flatten(1), k, v]
    if case["op"] == "logits":
        s = _logits_inputs(case, seed)
        x, bit = s["logits"].double(), torch.arange(s["logits"].shape[1], device="cuda")
        r, pres, freq = s["penalties"].double().unbind(1)
        hit = (s["seen"][:, bit // 32] >> (bit % 32).to(torch.int32)) & 1
        # x / r for x > 0, x * r otherwise
        x = x * torch.where(hit == 1, torch.where(x > 0, 1 / r[:, None], r[:, None]), 1.0)
        x = x - freq[:, None] * s["counts"] - pres[:, None] * (s["counts"] > 0)
        if s["bias"] is not None:
            for row in range(x.shape[0]):
                ids = s["bias_ids"][row]
                x[row].index_add_(0, ids[ids >= 0].long(), s["bias"][row][ids >= 0].double())
        if s["mask"] is not None:
            x[((s["mask"][:, bit // 32] >> (bit % 32).to(torch.int32)) & 1) == 0] = -math.inf
        return [None, x.amax(1)] if s["pick"] else x
    return None

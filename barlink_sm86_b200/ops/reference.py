# SPDX-License-Identifier: MIT
"""Plain PyTorch fp32 statements of every kernel in this library.

They serve two purposes: they are the oracles that the GPU numerics tests
compare against, and they are the CPU execution path that lets the models and
the tensor-parallel plumbing run (and be tested over gloo) on a machine
without a GPU.  Shapes and argument order match `barlink_sm86_b200.ops`.
"""
import functools
import math

import torch


def linear(x, weight, bias=None, residual=None, silu_mul=False, gelu=False):
    """y = x @ weight.T (+ bias) (tanh-GELU) (+ residual); silu_mul: rows of `weight` are
    interleaved (gate, up) pairs and y = silu(gate) * up has half the columns."""
    y = x.float() @ weight.float().t()
    if bias is not None:
        y = y + bias.float()
    if gelu:
        y = torch.nn.functional.gelu(y, approximate="tanh")
    if silu_mul:
        g, u = y[..., 0::2], y[..., 1::2]
        y = torch.nn.functional.silu(g) * u
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def rmsnorm(x, gamma, eps, residual=None):
    """Returns (normed, new_residual).  With a residual, x + residual is
    rounded to the storage dtype first and that rounded sum is normalised."""
    if residual is not None:
        s = (x.float() + residual.float()).to(x.dtype)
    else:
        s = x
    f = s.float()
    var = f.pow(2).mean(-1, keepdim=True)
    n = (f * torch.rsqrt(var + eps)).to(x.dtype)
    out = (n.float() * gamma.float()).to(x.dtype)
    return out, (s if residual is not None else None)


def _rope_angles(positions, dim, theta):
    inv = theta ** (-torch.arange(0, dim, 2, dtype=torch.float32, device=positions.device) / dim)
    ang = positions.float()[:, None] * inv[None, :]
    return ang.cos(), ang.sin()


def rope(x, positions, theta, axes=1):
    """Rotate-half RoPE on x [rows, heads, hd].  axes=2: positions [rows, 2]
    and each half of hd is rotated by its own coordinate."""
    rows, heads, hd = x.shape
    out = x.float().clone()
    sub = hd // axes
    pos = positions.view(rows, axes)
    for a in range(axes):
        cos, sin = _rope_angles(pos[:, a], sub, theta)
        seg = out[..., a * sub:(a + 1) * sub]
        x1, x2 = seg[..., : sub // 2], seg[..., sub // 2:]
        c, s = cos[:, None, :], sin[:, None, :]
        out[..., a * sub:(a + 1) * sub] = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)
    return out.to(x.dtype)


def qknorm_rope(qkv, gq, gk, positions, heads, eps=1e-6, theta=1e4, axes=2):
    """In place: per-head RMSNorm of the q and k heads at the start of each row
    of qkv [rows, width] (head_dim 128), then RoPE with `axes` coordinates."""
    rows = qkv.shape[0]
    qk = qkv[:, : 2 * heads * 128].reshape(rows, 2 * heads, 128).float()
    for lo, g in ((0, gq), (heads, gk)):
        if g is None:
            continue
        seg = qk[:, lo:lo + heads]
        n = (seg * torch.rsqrt(seg.pow(2).mean(-1, keepdim=True) + eps)).to(qkv.dtype).float()
        qk[:, lo:lo + heads] = n * g.float()
    rot = rope(qk.to(qkv.dtype), positions, theta, axes)
    qkv[:, : 2 * heads * 128] = rot.reshape(rows, 2 * heads * 128)
    return qkv


def layernorm_modulate(x, shift, scale, rows_per_batch, eps=1e-6):
    rows = x.numel() // x.shape[-1]
    f = x.reshape(rows, -1).float()
    n = torch.nn.functional.layer_norm(f, (f.shape[-1],), eps=eps)
    b = torch.arange(rows, device=x.device) // rows_per_batch
    out = n * (1.0 + scale.float()[b]) + shift.float()[b]
    return out.to(x.dtype).view_as(x)


def gate_residual(x, y, gate, rows_per_batch):
    rows = x.numel() // x.shape[-1]
    b = torch.arange(rows, device=x.device) // rows_per_batch
    x.copy_((x.reshape(rows, -1).float() + gate.float()[b] * y.reshape(rows, -1).float()).to(x.dtype).view_as(x))
    return x


def rope_kv_write(qkv, positions, slots, k_cache, v_cache, nq, nkv, hd, block_size, theta):
    """In place: rotate q and k inside qkv [rows, (nq+2nkv)*hd]; store k, v at
    slot (= block * block_size + offset) of caches [blocks, nkv, block_size, hd]."""
    rows = qkv.shape[0]
    v3 = qkv.view(rows, nq + 2 * nkv, hd)
    v3[:, : nq + nkv] = rope(v3[:, : nq + nkv], positions, theta)
    if slots is not None:
        for r in range(rows):
            s = int(slots[r])
            if s < 0:
                continue
            blk, off = divmod(s, block_size)
            k_cache[blk, :, off, :] = v3[r, nq:nq + nkv]
            v_cache[blk, :, off, :] = v3[r, nq + nkv:]
    return qkv


def silu_mul(gate_up, interleaved=False):
    if gate_up.dtype == torch.float32 and gate_up.dim() == 3:  # k-split slabs: summed first
        g, u = gate_up.sum(0)[..., 0::2], gate_up.sum(0)[..., 1::2]
        return (torch.nn.functional.silu(g) * u).to(torch.bfloat16)
    f = gate_up.float()
    if interleaved:
        g, u = f[..., 0::2], f[..., 1::2]
    else:
        h = f.shape[-1] // 2
        g, u = f[..., :h], f[..., h:]
    return (torch.nn.functional.silu(g) * u).to(gate_up.dtype)


def embedding(ids, table, vocab_lo=0):
    out = torch.zeros(ids.numel(), table.shape[1], dtype=table.dtype, device=table.device)
    loc = ids.long() - vocab_lo
    ok = (loc >= 0) & (loc < table.shape[0])
    out[ok] = table[loc[ok]]
    return out


def argmax(logits, offset=0):
    val, idx = logits.float().max(-1)
    return (idx + offset).to(torch.int32), val


def paged_attn_decode(q, k_cache, v_cache, block_tables, ctx_lens, nq, nkv, hd, scale):
    """q [batch, >= nq*hd] (first nq*hd columns are the query heads)."""
    batch = q.shape[0]
    bs = k_cache.shape[2]
    G = nq // nkv
    out = torch.zeros(batch, nq * hd, dtype=q.dtype, device=q.device)
    for b in range(batch):
        n = int(ctx_lens[b])
        if n == 0:
            continue
        nb = (n + bs - 1) // bs
        blks = block_tables[b, :nb].long()
        k = k_cache[blks].permute(1, 0, 2, 3).reshape(nkv, nb * bs, hd)[:, :n].float()
        v = v_cache[blks].permute(1, 0, 2, 3).reshape(nkv, nb * bs, hd)[:, :n].float()
        qq = q[b, : nq * hd].view(nkv, G, hd).float()
        s = torch.einsum("hgd,htd->hgt", qq, k) * scale
        p = torch.softmax(s, -1)
        o = torch.einsum("hgt,htd->hgd", p, v)
        out[b] = o.reshape(nq * hd).to(q.dtype)
    return out


def attention(q, k, v, cu_q, cu_k, scale, causal):
    """Dense attention over packed sequences.  q [tq, nq, hd], k/v [tk, nkv, hd];
    cu_* are cumulative lengths (batch + 1).  causal aligns the last query of a
    sequence with its last key."""
    nq, nkv = q.shape[1], k.shape[1]
    G = nq // nkv
    out = torch.zeros_like(q)
    for b in range(len(cu_q) - 1):
        q0, q1, k0, k1 = int(cu_q[b]), int(cu_q[b + 1]), int(cu_k[b]), int(cu_k[b + 1])
        qq = q[q0:q1].float().permute(1, 0, 2)
        kk = k[k0:k1].float().permute(1, 0, 2).repeat_interleave(G, 0)
        vv = v[k0:k1].float().permute(1, 0, 2).repeat_interleave(G, 0)
        s = qq @ kk.transpose(1, 2) * scale
        if causal:
            lq, lk = q1 - q0, k1 - k0
            i = torch.arange(lq, device=q.device)[:, None] + (lk - lq)
            j = torch.arange(lk, device=q.device)[None, :]
            s = s.masked_fill(j > i, float("-inf"))
        o = torch.softmax(s, -1) @ vv
        out[q0:q1] = o.permute(1, 0, 2).to(q.dtype)
    return out


def quantize_w8(weight):
    """Symmetric per-output-channel int8: returns (wq int8 [n, k], scale bf16 [n])."""
    w = weight.float()
    amax = w.abs().amax(1).clamp_min(1e-12)
    scale = (amax / 127.0).to(torch.bfloat16)
    wq = torch.round(w / scale.float()[:, None]).clamp(-127, 127).to(torch.int8)
    return wq, scale


def w8_dequant(wq, scale):
    """int8 [n, k] with per-channel scales [n] or per-group scales [n, k/group] -> fp32 [n, k]."""
    if scale.dim() == 1:
        return wq.float() * scale.float()[:, None]
    n, k = wq.shape
    g = scale.shape[1]
    return (wq.float().view(n, g, k // g) * scale.float()[:, :, None]).view(n, k)


def quantize_w8_grouped(weight, group=128):
    """Symmetric int8 with one scale per (output channel, group of `group` inputs): the
    granularity of the reference's kernel (torch_ext/barlink_sm86/w8a16.cu:13-24)."""
    w = weight.float()
    n, k = w.shape
    wg = w.view(n, k // group, group)
    scale = (wg.abs().amax(2).clamp_min(1e-12) / 127.0).to(torch.bfloat16)
    wq = torch.round(wg / scale.float()[:, :, None]).clamp(-127, 127).to(torch.int8).view(n, k)
    return wq, scale


def w8a16_linear(x, wq, scale, bias=None, silu_mul=False):
    """y = x @ (wq * scale).T: bf16 activations, int8 weights widened exactly to
    bf16, fp32 accumulation; scale per output channel [n] (applied at the end) or
    per group [n, k/group] (applied to the weights)."""
    if scale.dim() == 2:
        y = x.float() @ w8_dequant(wq, scale).t()
    else:
        y = (x.float() @ wq.float().t()) * scale.float()[None, :]
    if bias is not None:
        y = y + bias.float()
    if silu_mul:
        g, u = y[..., 0::2], y[..., 1::2]
        y = torch.nn.functional.silu(g) * u
    return y.to(x.dtype)


def w8a8_dynamic_linear(x, wq, scale, bias=None, silu_mul=False):
    """The int8-activation form of `w8a16_linear`: per-token scale amax / 127, activations rounded to
    int8, exact integer products, result * scale[n] * xs[m] (torch_ext/barlink_sm86/w8a16.cu:37-150
    of the reference, with per-channel weight scales)."""
    xf = x.float()
    xs = (xf.abs().amax(dim=1) / 127.0).clamp_min(1e-12)
    xq = torch.round(xf / xs[:, None]).clamp(-127, 127)
    if scale.dim() == 2:
        # per-group weight scales: integer sums per group, scaled and added in fp32 (w8a16.cu:119-142 there)
        n, groups = scale.shape
        gk = wq.shape[1] // groups
        part = torch.einsum("mgk,ngk->mng", xq.double().view(-1, groups, gk), wq.double().view(n, groups, gk))
        y = (part * scale.double()[None, :, :]).sum(-1).float() * xs[:, None]
    else:
        y = (xq.double() @ wq.double().t()).float() * scale.float()[None, :] * xs[:, None]
    if bias is not None:
        y = y + bias.float()
    if silu_mul:
        g, u = y[..., 0::2], y[..., 1::2]
        y = torch.nn.functional.silu(g) * u
    return y.to(x.dtype)


def allreduce_rmsnorm(parts, residual, gamma, eps):
    """What the fused kernel computes on every rank, given all ranks' inputs:
    sum in fp32 in rank order, round, add the residual, round, normalise."""
    acc = torch.zeros_like(parts[0], dtype=torch.float32)
    for p in parts:
        acc = acc + p.float()
    s = acc.to(parts[0].dtype)
    if residual is not None:
        s = (s.float() + residual.float()).to(s.dtype)
    normed, _ = rmsnorm(s, gamma, eps)
    return normed, s


def default_scale(hd):
    return 1.0 / math.sqrt(hd)


def pack_int4(weight, group_size=128):
    """[n, k] weight -> GPTQ-v1 tensors (qweight int32 [k/8, n], scales fp16
    [k/group, n], qzeros int32 [k/group, n/8]), symmetric with zero point 8:
    the format of the reference's Int4Linear (demos/qwen_tp/int4linear.py:47-69)."""
    w = weight.float()
    n, k = w.shape
    assert k % group_size == 0 and n % 8 == 0 and k % 8 == 0
    groups = k // group_size
    wg = w.reshape(n, groups, group_size)
    scale = (wg.abs().amax(2) / 7.0).clamp(min=1e-8).half()            # [n, groups], as stored
    q = torch.round(wg / scale.float()[..., None] + 8.0).clamp(0, 15).to(torch.int64).reshape(n, k)
    qk = q.reshape(n, k // 8, 8)
    qw = sum(qk[..., j] << (4 * j) for j in range(8))
    qw = ((qw + 2 ** 31) % 2 ** 32 - 2 ** 31).to(torch.int32).t().contiguous()
    z = torch.full((groups, n // 8, 8), 8, dtype=torch.int64, device=w.device)
    qz = sum(z[..., j] << (4 * j) for j in range(8))
    qz = ((qz + 2 ** 31) % 2 ** 32 - 2 ** 31).to(torch.int32).contiguous()
    return qw, scale.t().contiguous(), qz


def w4_dequant(qweight, scales, qzeros, group_size=128):
    """GPTQ-v1 tensors -> fp32 [n, k]."""
    k, n = qweight.shape[0] * 8, qweight.shape[1]
    w = qweight.t().long() & 0xFFFFFFFF
    nib = torch.stack([(w >> (4 * j)) & 0xF for j in range(8)], 2).reshape(n, k)
    zz = qzeros.long() & 0xFFFFFFFF
    z = torch.stack([(zz >> (4 * j)) & 0xF for j in range(8)], 2).reshape(-1, n)     # [groups, n]
    z = z.repeat_interleave(group_size, 0)[:k].t()
    sc = scales.float().repeat_interleave(group_size, 0)[:k].t()
    return (nib - z).float() * sc


def w4a16_linear(x, qweight, scales, qzeros, group_size=128):
    return (x.float() @ w4_dequant(qweight, scales, qzeros, group_size).t()).to(x.dtype)


# ---------------------------------------------------------------- the key/value cache in 4 bits
# Layout (csrc/kv4.cuh): [blocks, nkv, block_size / 16, 20 * hd] bytes; a tile holds 16 tokens of a head.
KV4_GROUP = 32


@functools.lru_cache(maxsize=None)
def _kv4_maps(hd):
    """Byte and shift of every code of a tile, [16, hd] for keys and for values, and the bytes of the groups' step and low,
    [16, hd / 32]."""
    na = hd // KV4_GROUP
    r, d = torch.arange(16)[:, None], torch.arange(hd)[None]
    k = r * (hd // 2) + ((d // 8 % 4) * na + d // 32) * 4 + d % 8 // 2
    v = 8 * hd + (r // 2) * hd + (d // 4 % 8 * na + d // 32) * 4 + (r % 2) * 2 + d % 4 // 2
    a = torch.arange(na)[None]
    kp, vp = (at * hd + r * na * 4 + a * 2 for at in (16, 18))
    shift = (d % 2 * 4).expand(16, -1)
    return {"k": (k, shift, kp, kp + 2 * na), "v": (v, shift, vp, vp + 2 * na)}


def kv4_cache(n_blocks, nkv, hd, block_size, device):
    return torch.zeros(n_blocks, nkv, block_size // 16, 20 * hd, dtype=torch.uint8, device=device)


def kv4_quantise(x):
    """[..., hd] -> codes [..., hd / 32, 32] (int64), low and step (bf16) [..., hd / 32].  A group whose range is no finite number: step 0,
    low NaN."""
    x = x.to(torch.bfloat16).float().unflatten(-1, (-1, KV4_GROUP))
    low = x.amin(-1)
    step = ((x.amax(-1) - low) / 15).to(torch.bfloat16)
    fine = torch.isfinite(step.float()) & torch.isfinite(x).all(-1)
    step, low = torch.where(fine, step, torch.zeros_like(step)), torch.where(fine, low, torch.full_like(low, math.nan))
    codes = torch.where((step.float() > 0)[..., None], torch.round((x - low[..., None]) / step.float()[..., None]), torch.zeros_like(x))
    return codes.clamp(0, 15).long(), low.to(torch.bfloat16), step


def kv4_write(cache, slots, k, v, block_size):
    """Rows k, v [rows, nkv, hd] into the cache at their slots (below 0 or behind the cache: not kept)."""
    nkv, hd = k.shape[1:]
    maps, tiles = _kv4_maps(hd), cache.view(-1, 20 * hd)
    slots = slots.long()
    ok = (slots >= 0) & (slots < cache.shape[0] * block_size)
    slots, k, v = slots[ok], k[ok], v[ok]
    inb = slots % block_size
    tile = ((slots // block_size)[:, None] * nkv + torch.arange(nkv)) * (block_size // 16) + (inb // 16)[:, None]   # [rows, nkv]
    r = inb % 16
    for x, name in ((k, "k"), (v, "v")):
        codes, low, step = kv4_quantise(x)
        byte, shift, ps, pl = maps[name]
        val = codes.flatten(-2) << shift[r][:, None]
        rows = torch.zeros(*tile.shape, 20 * hd, dtype=torch.int64)
        rows.scatter_add_(2, byte[r][:, None].expand(-1, nkv, -1), val)   # (two codes to a byte)
        tiles[tile[:, :, None], byte[r][:, None]] = rows.gather(2, byte[r][:, None].expand(-1, nkv, -1)).to(torch.uint8)
        for t, at in ((step, ps), (low, pl)):
            b = t.contiguous().view(torch.uint8).view(*t.shape, 2)
            for j in range(2):
                tiles[tile[:, :, None], at[r][:, None] + j] = b[..., j]


def kv4_values(cache, slots, hd, block_size):
    """fp32 k, v [rows, nkv, hd] of the slots (all within the cache)."""
    nkv = cache.shape[1]
    maps, tiles = _kv4_maps(hd), cache.view(-1, 20 * hd)
    slots = slots.long()
    inb = slots % block_size
    tile = ((slots // block_size)[:, None] * nkv + torch.arange(nkv)) * (block_size // 16) + (inb // 16)[:, None]
    r, got = inb % 16, []
    for name in ("k", "v"):
        byte, shift, ps, pl = maps[name]
        codes = (tiles[tile[:, :, None], byte[r][:, None]].long() >> shift[r][:, None]) & 15
        par = []
        for at in (ps, pl):
            b = torch.stack([tiles[tile[:, :, None], at[r][:, None] + j] for j in range(2)], -1).contiguous()
            par.append(b.view(torch.bfloat16)[..., 0].float().repeat_interleave(KV4_GROUP, -1))
        got.append(par[1] + par[0] * codes.float())
    return got


def kv4_read(cache, slots, hd, block_size):
    ok = (slots >= 0) & (slots.long() < cache.shape[0] * block_size)
    k, v = kv4_values(cache, torch.where(ok, slots, torch.zeros_like(slots)), hd, block_size)
    return [torch.where(ok[:, None, None], t, torch.zeros_like(t)).to(torch.bfloat16) for t in (k, v)]


def rope_kv_write_q4(qkv, positions, slots, cache, nq, nkv, hd, block_size, theta, out):
    """Rotates q and k of qkv [rows, (nq + 2 nkv) * hd] into out, angles in 64 bits; k and v into the cache."""
    rows = qkv.shape[0]
    x = qkv.float().view(rows, nq + 2 * nkv, hd).clone()
    inv = theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    ang = positions.double()[:, None] * inv
    c, s = ang.cos().float()[:, None], ang.sin().float()[:, None]
    a, b = x[:, :nq + nkv, :hd // 2].clone(), x[:, :nq + nkv, hd // 2:].clone()
    x[:, :nq + nkv, :hd // 2], x[:, :nq + nkv, hd // 2:] = a * c - b * s, b * c + a * s
    out.copy_(x.view(rows, -1).to(out.dtype))
    if slots is not None:
        o = out.view(rows, nq + 2 * nkv, hd)
        kv4_write(cache, slots, o[:, nq:nq + nkv], o[:, nq + nkv:], block_size)
    return out


def paged_attn_decode_q4(q, cache, block_tables, ctx_lens, nq, nkv, hd, scale):
    """As paged_attn_decode, on the 4-bit cache; tokens of table entries that name no block are left out."""
    bs, G = cache.shape[2] * 16, nq // nkv
    out = torch.zeros(q.shape[0], nq * hd, dtype=q.dtype)
    for b in range(q.shape[0]):
        t = torch.arange(min(int(ctx_lens[b]), block_tables.shape[1] * bs))
        blk = block_tables[b].long()[t // bs]
        slots = (blk * bs + t % bs)[(blk >= 0) & (blk < cache.shape[0])]
        if len(slots) == 0:
            continue
        k, v = kv4_values(cache, slots, hd, bs)
        p = torch.softmax(torch.einsum("hgd,thd->hgt", q[b, :nq * hd].view(nkv, G, hd).float(), k) * scale, -1)
        out[b] = torch.einsum("hgt,thd->hgd", p, v).reshape(-1).to(q.dtype)
    return out


def _paged_attn_chunk(q, n_blocks, bs, block_tables, cu_q, ctx_lens, nq, nkv, hd, scale, out, read):
    """read(slots) -> k, v [rows, nkv, hd]"""
    G = nq // nkv
    for b in range(ctx_lens.numel()):
        lo = min(max(int(cu_q[b]), 0), q.shape[0])
        n = min(max(int(cu_q[b + 1]), lo), q.shape[0]) - lo
        ctx = max(int(ctx_lens[b]), 0)
        t = torch.arange(min(ctx, block_tables.shape[1] * bs))
        blk = block_tables[b].long()[t // bs] if len(t) else t
        ok = (blk >= 0) & (blk < n_blocks)
        t, slots = t[ok], (blk * bs + t % bs)[ok]
        k, v = (x.float() for x in read(slots))
        qq = q[lo:lo + n, :nq * hd].reshape(n, nkv, G, hd).float()
        s = torch.einsum("nhgd,thd->hgnt", qq, k) * scale
        seen = t <= (ctx - n + torch.arange(n))[:, None]
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        p = torch.where(seen.any(-1)[:, None], torch.softmax(s, -1), torch.zeros_like(s))
        o = torch.einsum("hgnt,thd->nhgd", p, v)
        if not torch.isfinite(v).all():
            # (0 x infinity is NaN: a row is made from the values that it sees)
            for i in range(n):
                o[i] = torch.einsum("hgt,thd->hgd", p[:, :, i, seen[i]], v[seen[i]])
        out[lo:lo + n] = o.reshape(n, nq * hd).to(q.dtype)
    return out


def paged_attn_chunk(q, k_cache, v_cache, block_tables, cu_q, ctx_lens, nq, nkv, hd, scale, out):
    bs = k_cache.shape[2]

    def read(slots):
        return [c[slots // bs, :, slots % bs] for c in (k_cache, v_cache)]

    return _paged_attn_chunk(q, k_cache.shape[0], bs, block_tables, cu_q, ctx_lens, nq, nkv, hd, scale, out, read)


def paged_attn_chunk_q4(q, cache, block_tables, cu_q, ctx_lens, nq, nkv, hd, scale, out):
    bs = cache.shape[2] * 16
    return _paged_attn_chunk(q, cache.shape[0], bs, block_tables, cu_q, ctx_lens, nq, nkv, hd, scale, out,
                             lambda slots: kv4_read(cache, slots, hd, bs))


# ---------------------------------------------------------------- serving steps
def paged_layout(new_lens, past_lens, block_tables, free_list, free_range, tokens, block_size, rows_per_request=0, lost=None):
    """See ops.paged_layout; block_tables, free_list and lost are updated in place."""
    width, cap = block_tables.shape[1], free_list.numel()
    head, free, _ = (int(v) for v in free_range)
    free = min(max(free, 0), cap)
    cu, ctx, need, back = [0], [], 0, []
    pos = torch.zeros(tokens, dtype=torch.int32)
    slots = torch.full((tokens,), -1, dtype=torch.int32)
    for b, (n, past) in enumerate(zip(new_lens.tolist(), past_lens.tolist())):
        past = max(past, 0)
        had = min(-(-past // block_size), width)
        if n < 0:
            back += [i for i in block_tables[b, :had].tolist() if i >= 0]
            cu.append(cu[-1])
            ctx.append(0)
            continue
        for page in range(had, min(-(-(past + n) // block_size), width)):
            block_tables[b, page] = free_list[(head + need) % cap] if need < free else -1
            need += 1
        for i in range(min(n, rows_per_request) if rows_per_request else n):
            row, p = (b * rows_per_request if rows_per_request else cu[-1]) + i, past + i
            if row >= tokens:
                break
            pos[row] = p
            blk = int(block_tables[b, p // block_size]) if p // block_size < width else -1
            slots[row] = blk * block_size + p % block_size if blk >= 0 else -1
            if blk < 0 and lost is not None:
                lost += 1
        cu.append(cu[-1] + n)
        ctx.append(past + n)
    taken, given = min(need, free), min(len(back), cap - free)
    for i, blk in enumerate(back[:given]):
        free_list[(head + free + i) % cap] = blk
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return [i32(cu), pos, slots, i32(ctx), i32([(head + taken) % cap, free - taken + given, max(need - free, 0)])]


def count_tokens(counts, seen, ids, cu=None, prompt_lens=None, reset=False):
    rows, vocab = counts.shape
    if reset:
        counts.zero_()
        seen.zero_()
    for r in range(rows):
        lo, hi = (max(int(cu[r]), 0), min(int(cu[r + 1]), ids.numel())) if cu is not None else (r, r + 1)
        h = ids[lo:hi].long()
        ok = (h >= 0) & (h < vocab)
        made = torch.arange(len(h)) >= (int(prompt_lens[r]) if prompt_lens is not None else 0)
        counts[r].scatter_add_(0, h[ok & made], torch.ones(int((ok & made).sum()), dtype=torch.int32))
        for i in set(h[ok].tolist()):
            w = (int(seen[r, i // 32]) & 0xffffffff) | 1 << (i % 32)
            seen[r, i // 32] = w - (1 << 32) if w >= 1 << 31 else w


def _word_bits(words, ids):
    return (words[:, ids // 32] >> (ids % 32).to(torch.int32)) & 1 != 0


def logit_rules(logits, vocab, offset=0, penalties=None, counts=None, seen=None, bias_ids=None, bias=None, mask=None):
    """fp32 logits [rows, n] under the rules; column i is token i + offset."""
    x = logits.float().clone()
    ids = torch.arange(x.shape[1]) + offset
    known = ids < vocab
    at = torch.where(known, ids, torch.zeros_like(ids))
    if penalties is not None:
        again, presence, frequency = (penalties[:, i:i + 1] for i in range(3))
        hit = _word_bits(seen, at) & known
        c = torch.where(hit, counts[:, at], torch.zeros_like(counts[:, at])).float()
        x = torch.where(hit, torch.where(x > 0, x / again, x * again), x)
        x = torch.where(c > 0, x - frequency * c - presence, x)
    if bias_ids is not None:
        for j in range(bias_ids.shape[1]):
            x = torch.where((bias_ids[:, j:j + 1] == ids) & (bias_ids[:, j:j + 1] >= 0), x + bias[:, j:j + 1], x)
    ok = known if mask is None else _word_bits(mask, at) & known
    return torch.where(ok, x, torch.full_like(x, -math.inf))


def pick(x, offset=0):
    """(token int32, value fp32) of every row's greatest (the first of equals, NaN passed over); token -1 where all are -inf."""
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    val = x.amax(-1)
    idx = (x == val[:, None]).int().argmax(-1) + offset
    return torch.where(val == -math.inf, torch.full_like(idx, -1), idx).to(torch.int32), val


def token_logprob_parts(logits, ids, top=0, offset=0, vocab=2 ** 31 - 1):
    """(logits of ids, parts fp32 [rows, 3] = m, S, T, top_ids, top logits), see ops.token_logprobs."""
    n = max(0, min(logits.shape[1], vocab - offset))
    x = logits[:, :n].double()
    rows = x.shape[0]
    m = torch.where(torch.isnan(x), -math.inf, x).amax(-1) if n else torch.full((rows,), -math.inf, dtype=torch.float64)
    t = x - torch.where(m == -math.inf, 0.0, m)[:, None]
    e = torch.exp(t)
    parts = torch.stack([m, e.sum(-1), torch.where(t == -math.inf, 0.0, t * e).sum(-1)], 1).float()
    wide = ids.reshape(rows, 1 if ids.dim() == 1 else ids.shape[1])
    at = wide.long() - offset
    ok = (wide >= 0) & (at >= 0) & (at < n)
    given = torch.where(ok, x.gather(1, torch.where(ok, at, 0)), -math.inf) if n else torch.full(at.shape, -math.inf, dtype=torch.float64)
    order = torch.sort(torch.where(torch.isnan(x), -math.inf, x), dim=-1, descending=True, stable=True)
    val = torch.nn.functional.pad(order.values[:, :top], (0, max(0, top - n)), value=-math.inf)
    idx = torch.nn.functional.pad(order.indices[:, :top] + offset, (0, max(0, top - n)), value=-1)
    return given.view(ids.shape).float(), parts, torch.where(val == -math.inf, -1, idx).to(torch.int32), val.float()


def token_logprobs_of(given, parts, top_ids, top_val):
    """(logprobs, entropy, top_ids, top_logprobs) from what token_logprob_parts leaves."""
    m, s, t = parts.double().unbind(-1)
    none = (m == -math.inf) & (s == 0)

    def logp(x):
        rows = (-1,) + (1,) * (x.dim() - 1)
        y = (x.double() - m.view(rows)) - torch.log(s).view(rows)
        return torch.where(none.view(rows), -math.inf, y).float()

    top = torch.where((top_ids < 0) & ~torch.isnan(s)[:, None], -math.inf, logp(top_val))
    return logp(given), torch.where(none, 0.0, torch.log(s) - t / s).float(), top_ids, top


def join_token_logprobs(shards):
    """What token_logprob_parts leaves, of the shards of a vocabulary in their order -> the same of the whole."""
    given = torch.stack([s[0] for s in shards]).amax(0)
    parts = torch.stack([s[1] for s in shards]).double()
    m = parts[..., 0].amax(0)
    # (the distance of an empty shard is of no account: its sums are zero)
    d = torch.where(parts[..., 0] == -math.inf, 0.0, parts[..., 0] - torch.where(m == -math.inf, 0.0, m))
    e = torch.exp(d)
    s = (e * parts[..., 1]).sum(0)
    t = (e * (parts[..., 2] + torch.where(d == -math.inf, 0.0, d) * parts[..., 1])).sum(0)
    top = shards[0][2].shape[-1]
    order = torch.sort(torch.cat([x[3] for x in shards], 1), dim=-1, descending=True, stable=True)
    ids = torch.cat([x[2] for x in shards], 1).gather(1, order.indices[:, :top])
    return given, torch.stack([m, s, t], 1).float(), ids, order.values[:, :top]

"""PyTorch reference implementations of every decoder op.

These are the arithmetic of the CPU engine (fp32 on CPU, the reference tier and the
CPU/gloo configuration) and the numerical oracle of the sm_100a kernels: each kernel's test
compares against the function here evaluated in fp32.

Conventions shared with the kernels:
  * RMSNorm: ``y = x * rsqrt(mean(x^2) + eps) * w`` in fp32, one rounding to the output dtype;
    with a residual, ``r = round(x + r)`` is stored first and then normalised.
  * RoPE: rotate-half pairs (i, i + d/2), angles from a precomputed fp32 ``cos_sin`` table
    ``[max_pos, d]`` holding cos in the first half and sin in the second.
  * KV cache of one layer: ``[num_blocks, 2, kv_heads, block_size, head_dim]``; slot = block *
    block_size + offset; a negative slot is a padding token and is not written.

Reference parity: HF-convention rms_norm / rope / llama3 inverse frequencies of
core/everserve/reference/arith/ops.py:17-73.
"""

from __future__ import annotations

import math

import torch


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, residual: torch.Tensor | None = None) -> torch.Tensor:
    if residual is not None:
        s = (x.float() + residual.float()).to(residual.dtype)
        residual.copy_(s)
        x = s
    xf = x.float()
    inv = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * inv * w.float()).to(x.dtype)


def inverse_frequencies(head_dim: int, theta: float, scaling: dict | None = None) -> torch.Tensor:
    """Rotary inverse frequencies, with the llama3 long-context scaling when ``scaling`` asks."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    if scaling and scaling.get("rope_type", scaling.get("type")) == "llama3":
        factor = scaling["factor"]
        lo, hi = scaling.get("low_freq_factor", 1.0), scaling.get("high_freq_factor", 4.0)
        old_ctx = scaling.get("original_max_position_embeddings", 8192)
        lo_wl, hi_wl = old_ctx / lo, old_ctx / hi
        wl = 2 * math.pi / inv
        smooth = (old_ctx / wl - lo) / (hi - lo)
        scaled = torch.where(wl > lo_wl, inv / factor, inv)
        mid = (wl <= lo_wl) & (wl >= hi_wl)
        scaled = torch.where(mid, (1 - smooth) * inv / factor + smooth * inv, scaled)
        inv = scaled
    return inv.float()


def cos_sin_table(head_dim: int, max_pos: int, theta: float, scaling: dict | None = None) -> torch.Tensor:
    inv = inverse_frequencies(head_dim, theta, scaling).double()
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None, :]
    return torch.cat([torch.cos(ang), torch.sin(ang)], dim=-1).float()


def rope(x: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    """x: [T, H, d] (fp32), cs: [T, d] cos|sin rows for each token."""
    half = x.shape[-1] // 2
    c, s = cs[:, None, :half], cs[:, None, half:]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def rope_kv_write(qkv, bias, positions, cos_sin, slots, cache, hq: int, hkv: int, block_size: int) -> torch.Tensor:
    """Rotate q and k, write k and v into the paged cache; return q as [T, hq, d]."""
    T = qkv.shape[0]
    d = cos_sin.shape[1]
    x = qkv.float()
    if bias is not None:
        x = x + bias.float()
    x = x.view(T, hq + 2 * hkv, d)
    cs = cos_sin[positions]
    q = rope(x[:, :hq], cs)
    k = rope(x[:, hq : hq + hkv], cs)
    v = x[:, hq + hkv :]
    valid = slots >= 0
    if bool(valid.any()):
        sl = slots[valid]
        blk, off = sl // block_size, sl % block_size
        cache[blk, 0, :, off] = k[valid].to(cache.dtype)
        cache[blk, 1, :, off] = v[valid].to(cache.dtype)
    return q.to(qkv.dtype)


def gather_kv(cache: torch.Tensor, block_table: torch.Tensor, n: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The first n positions of one sequence: k, v as [n, kv_heads, d]."""
    bs = cache.shape[3]
    nb = (n + bs - 1) // bs
    blocks = cache[block_table[:nb].long()]  # [nb, 2, Hkv, bs, d]
    k = blocks[:, 0].permute(0, 2, 1, 3).reshape(nb * bs, cache.shape[2], cache.shape[4])[:n]
    v = blocks[:, 1].permute(0, 2, 1, 3).reshape(nb * bs, cache.shape[2], cache.shape[4])[:n]
    return k, v


def paged_attention(q, cache, block_tables, ctx_lens, q_seq, q_pos, scale: float) -> torch.Tensor:
    """Causal attention of query rows against their sequence's paged history.

    q: [T, hq, d]; q_seq[t] is the row's sequence index into block_tables/ctx_lens, q_pos[t] its
    position (it sees positions 0..q_pos[t]). Returns [T, hq, d] in q's dtype (fp32 inside).
    """
    T, hq, d = q.shape
    hkv = cache.shape[2]
    g = hq // hkv
    out = torch.empty_like(q)
    seqs = q_seq.tolist()
    pos = q_pos.tolist()
    start = 0
    while start < T:
        s = seqs[start]
        end = start
        while end < T and seqs[end] == s:
            end += 1
        n = int(ctx_lens[s])
        k, v = gather_kv(cache, block_tables[s], n)
        kf = k.float().repeat_interleave(g, dim=1)  # [n, hq, d]
        vf = v.float().repeat_interleave(g, dim=1)
        qf = q[start:end].float()
        scores = torch.einsum("thd,nhd->htn", qf, kf) * scale
        p_idx = torch.tensor(pos[start:end], device=q.device)
        mask = torch.arange(n, device=q.device)[None, :] > p_idx[:, None]
        scores = scores.masked_fill(mask[None], float("-inf"))
        prob = torch.softmax(scores, dim=-1)
        out[start:end] = torch.einsum("htn,nhd->thd", prob, vf).to(q.dtype)
        start = end
    return out


# ---- the paged cache held in 4 bits (one layer: uint8 [num_blocks, kv_heads, record]) ---------------
#
# A group is 64 channels, or the whole head, of one row (one token's K or V of one kv head). With mn and
# mx its smallest and largest value: scale = bf16((mx - mn) / 15), zero = bf16(mn), code =
# clamp(round((x - zero) / scale), 0, 15), and the value held is scale * code + zero (a group of equal
# values has scale 0). So a value is held within half a scale, or 2^-8 (|mn| + mx - mn) where that is more. A
# group holding a value that is not finite, or whose range passes fp32's largest number, reads as NaN. A record
# holds the K codes [bs, d / 2], the V codes, the K pairs (scale, zero) [bs, groups, 2] in bf16, the V pairs.


def kv4_cache_shape(num_blocks: int, kv_heads: int, block_size: int, head_dim: int, group: int = 64) -> tuple[int, int, int]:
    """Shape of one layer's cache in 4 bits (uint8); `group`: channels that share a scale, 64 or head_dim."""
    if head_dim not in (64, 128) or group not in (64, head_dim) or block_size not in (16, 32):
        raise ValueError(f"no 4-bit cache of head_dim {head_dim}, group {group}, block_size {block_size}")
    return num_blocks, kv_heads, block_size * (head_dim + 8 * (head_dim // group))


def kv4_groups(cache: torch.Tensor, head_dim: int, block_size: int) -> int:
    """Groups of a row, from the size of the cache's records."""
    groups = (cache.shape[2] // block_size - head_dim) // 8
    if groups < 1 or kv4_cache_shape(cache.shape[0], cache.shape[1], block_size, head_dim, head_dim // groups) != tuple(cache.shape):
        raise ValueError(f"a record of {cache.shape[2]} bytes is not that of head_dim {head_dim}, block_size {block_size}")
    return groups


def kv4_order(head_dim: int, device=None) -> torch.Tensor:
    """The channel of each stored nibble of a row (byte by byte, the low nibble first)."""
    p = torch.arange(head_dim // 8, device=device)
    word = p // 2 + 8 * (p % 2) if head_dim == 128 else p
    return (8 * word[:, None] + torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=device)).reshape(-1)


def kv4_quantize(x: torch.Tensor, groups: int) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., d] -> (stored codes uint8 [..., d / 2], (scale, zero) bf16 [..., groups, 2])."""
    d = x.shape[-1]
    g = x.float().unflatten(-1, (groups, d // groups))
    mn, mx = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale, zero = ((mx - mn) * (1.0 / 15.0)).bfloat16(), mn.bfloat16()
    s = scale.float()
    code = torch.round((g - zero.float()) / torch.where(s > 0, s, torch.ones_like(s))).nan_to_num().clamp(0, 15)
    code = torch.where(s > 0, code, torch.zeros_like(code)).flatten(-2).to(torch.uint8)
    pair = code[..., kv4_order(d, x.device)].unflatten(-1, (d // 2, 2))
    scale = torch.where(torch.isfinite(g).all(-1, keepdim=True), scale, torch.full_like(scale, math.nan))
    return pair[..., 0] | (pair[..., 1] << 4), torch.cat([scale, zero], -1)


def kv4_parts(cache: torch.Tensor, head_dim: int, block_size: int) -> list[torch.Tensor]:
    """Views of the cache's bytes: K codes, V codes [nb, hkv, bs, d / 2], K pairs, V pairs [nb, hkv, bs, 4 * groups]."""
    n, m = block_size * head_dim // 2, 4 * block_size * kv4_groups(cache, head_dim, block_size)
    return [t.unflatten(-1, (block_size, -1)) for t in cache.split((n, n, m, m), -1)]


def kv4_values(codes: torch.Tensor, pairs: torch.Tensor) -> torch.Tensor:
    """The fp32 values of stored rows: codes [..., d / 2], pairs [..., 4 * groups] (bytes) -> [..., d]."""
    d = 2 * codes.shape[-1]
    nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    x = torch.empty_like(nib)
    x[..., kv4_order(d, codes.device)] = nib
    sz = pairs.contiguous().view(torch.bfloat16).unflatten(-1, (-1, 2)).float()
    groups = sz.shape[-2]
    return (x.unflatten(-1, (groups, d // groups)) * sz[..., :1] + sz[..., 1:]).flatten(-2)


def kv4_read(cache: torch.Tensor, slots: torch.Tensor, head_dim: int, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The fp32 rows at `slots` of a cache in 4 bits: k, v [n, hkv, d]; zeros for a negative slot."""
    kc, vc, kp, vp = kv4_parts(cache, head_dim, block_size)
    s = slots.clamp(min=0)
    blk, off = s // block_size, s % block_size
    keep = (slots >= 0)[:, None, None]
    zero = torch.zeros((), device=cache.device)
    return tuple(torch.where(keep, kv4_values(c[blk, :, off], p[blk, :, off]), zero) for c, p in ((kc, kp), (vc, vp)))


def kv4_cache_values(cache: torch.Tensor, head_dim: int, block_size: int) -> torch.Tensor:
    """Every value a cache in 4 bits holds, as an fp32 cache [num_blocks, 2, hkv, bs, d]."""
    kc, vc, kp, vp = kv4_parts(cache, head_dim, block_size)
    return torch.stack((kv4_values(kc, kp), kv4_values(vc, vp)), 1)


def rope_kv4_write(qkv, bias, positions, cos_sin, slots, cache, hq: int, hkv: int, block_size: int) -> torch.Tensor:
    """Rotate q and k, quantise k and v into the slots of a cache in 4 bits; return q as [T, hq, d]."""
    T, d = qkv.shape[0], cos_sin.shape[1]
    x = qkv.float()
    if bias is not None:
        x = x + bias.float()
    x = x.view(T, hq + 2 * hkv, d)
    qk = rope(x[:, : hq + hkv], cos_sin[positions])
    keep = slots >= 0
    blk, off = slots[keep] // block_size, slots[keep] % block_size
    kc, vc, kp, vp = kv4_parts(cache, d, block_size)
    groups = kv4_groups(cache, d, block_size)
    for rows, codes, pairs in ((qk[:, hq:], kc, kp), (x[:, hq + hkv :], vc, vp)):
        c, p = kv4_quantize(rows[keep], groups)
        codes[blk, :, off] = c
        pairs[blk, :, off] = p.flatten(-2).contiguous().view(torch.uint8)
    return qk[:, :hq].to(qkv.dtype)


def kv4_attention(q, cache, block_tables, ctx_lens, last_rows, scale: float, block_size: int) -> torch.Tensor:
    """Causal attention over a cache in 4 bits. q [T, hq, d]: sequence s owns the rows up to last_rows[s],
    and its last one sits at position ctx_lens[s] - 1; a row without a visible key is zero."""
    T, hq, d = q.shape
    out = torch.zeros_like(q)
    kc, vc, kp, vp = kv4_parts(cache, d, block_size)
    r0 = 0
    for s, (last, n) in enumerate(zip(last_rows.tolist(), ctx_lens.tolist())):
        r1 = last + 1
        if n > 0 and r1 > r0:
            blk = block_tables[s, : (n + block_size - 1) // block_size].long()
            k, v = (kv4_values(c[blk], p[blk]).transpose(1, 2).flatten(0, 1)[:n].repeat_interleave(hq // cache.shape[1], 1)
                    for c, p in ((kc, kp), (vc, vp)))
            score = torch.einsum("thd,nhd->htn", q[r0:r1].float(), k) * scale
            pos = torch.arange(n - (r1 - r0), n, device=q.device)
            score = score.masked_fill((torch.arange(n, device=q.device)[None] > pos[:, None])[None], float("-inf"))
            bad = ~torch.isfinite(v)  # reaches the rows that see it alone, not the others times zero
            o = torch.einsum("htn,nhd->thd", torch.softmax(score, -1), v.masked_fill(bad, 0.0))
            if bool(bad.any()):
                seen = (torch.arange(n, device=q.device)[None] <= pos[:, None]).float()
                o = o.masked_fill(torch.einsum("tn,nhd->thd", seen, bad.float()) > 0, math.nan)
            out[r0:r1] = torch.where((pos >= 0)[:, None, None], o, torch.zeros_like(o)).to(q.dtype)
        r0 = r1
    return out


def copy_pages(caches: list[torch.Tensor], pairs: torch.Tensor) -> None:
    """caches[l][to] = caches[l][from] for every layer and (from, to) of pairs [n, 2]; negative: padding."""
    p = pairs[(pairs >= 0).all(1)]
    for c in caches:
        c[p[:, 1]] = c[p[:, 0]]


def silu_mul(gu: torch.Tensor) -> torch.Tensor:
    inter = gu.shape[-1] // 2
    g, u = gu[..., :inter].float(), gu[..., inter:].float()
    return (g * torch.sigmoid(g) * u).to(gu.dtype)


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, scale: torch.Tensor | None = None,
           pre: torch.Tensor | None = None) -> torch.Tensor:
    """x . w^T * scale[m] + pre + bias + residual (fp32, one rounding): the GEMM epilogue's order."""
    y = x.float() @ w.float().t()
    if scale is not None:
        y = y * scale.float()[:, None]
    if pre is not None:
        y = y + pre.float()
    if bias is not None:
        y = y + bias.float()
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def moe_route(logits: torch.Tensor, k: int, e0: int, el: int) -> torch.Tensor:
    """Per-token weights of experts e0 .. e0 + el - 1: softmax, top k with ties to the lowest index,
    renormalised over the k; 0 for an expert not chosen. Returns fp32 [el, T]."""
    p = torch.softmax(logits.float(), dim=-1)
    order = torch.argsort(-p, dim=-1, stable=True)[:, :k]
    chosen = torch.zeros_like(p).scatter_(1, order, 1.0)
    w = p * chosen / (p * chosen).sum(-1, keepdim=True)
    return w[:, e0 : e0 + el].t().contiguous()


def moe_topk(logits: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Each token's top k experts by softmax probability (ties to the lowest index), in rank
    order, and their probabilities renormalised over the k: (int32 [T, k], fp32 [T, k])."""
    p = torch.softmax(logits.float(), dim=-1)
    ids = torch.argsort(-p, dim=-1, stable=True)[:, :k]
    w = p.gather(1, ids)
    return ids.to(torch.int32), w / w.sum(-1, keepdim=True)


def expert_places(ids: torch.Tensor, num_experts: int) -> torch.Tensor:
    """Where each (token, slot) row goes in its expert's segment from this sender: its rank among
    the sender's rows for the same expert in (token, slot) order. int32 like `ids`."""
    flat = ids.reshape(-1).long()
    onehot = torch.nn.functional.one_hot(flat, num_experts)
    before = onehot.cumsum(0) - onehot  # rows of each expert strictly before this one
    return before.gather(1, flat[:, None]).reshape(ids.shape).to(torch.int32)


def moe_a2a(xs: list[torch.Tensor], ids: list[torch.Tensor], weights: list[torch.Tensor], expert) -> list[torch.Tensor]:
    """Oracle of the expert-parallel all-to-all: for each member's tokens x [T, H], the sum over
    slots (in order, fp32) of weight * expert(e, x[t]); `expert(e, rows)` gives fp32 outputs."""
    outs = []
    for x, i, w in zip(xs, ids, weights):
        acc = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
        for j in range(i.shape[1]):
            for e in i[:, j].unique().tolist():
                rows = (i[:, j] == e).nonzero().flatten()
                acc[rows] += w[rows, j, None].float() * expert(int(e), x[rows]).float()
        outs.append(acc.to(x.dtype))
    return outs


def argmax(logits: torch.Tensor) -> torch.Tensor:
    return torch.argmax(logits.float(), dim=-1)


def member_sum(parts: list[torch.Tensor]) -> torch.Tensor:
    """Sum of the members' tensors in member order, fp32 accumulate, one rounding.

    The oracle of the failure-detecting all-reduce: the same order after a membership change
    gives the same bits (core/everserve/reference/arith/ops.py:63).
    """
    acc = torch.zeros_like(parts[0], dtype=torch.float32)
    for p in parts:
        acc = acc + p.float()
    return acc.to(parts[0].dtype)
